"""The host-side refusals of the paged-cache operators: nothing is launched, no GPU needed."""
import ctypes as C

import pytest

from nates_recipe_rs_b200 import _lib
from nates_recipe_rs_b200._lib import PagedKV, SeqBatch

P = 1 << 20  # an aligned address that is never followed
NAN, INF = float("nan"), float("inf")


def pool(**kw):
    d = dict(k_pages=P, v_pages=P, dtype=1, n_pages=4, page_size=16, n_kv_heads=2, head_dim=64, k_page_stride=0, v_page_stride=0, page_table=P,
             table_stride=4)
    d.update(kw)
    return PagedKV(**d)


def seqs(**kw):
    d = dict(cu_q=P, kv_len=P, n_seqs=2, total_q=0, max_q=1, max_kv=64)
    d.update(kw)
    return SeqBatch(**d)


def attn(kv=None, b=None, q=P, q_stride=512, out=2 * P, out_dtype=1, out_stride=512, scratch=P, nqh=8, window=0, scale=1.0, nbytes=None):
    L = _lib.lib()
    nbytes = max(L.qmm_attn_paged_scratch_bytes(1, 8, 2, 64), 0) if nbytes is None else nbytes
    return L.launch_attn_paged(q, q_stride, kv or pool(), b or seqs(), out, out_dtype, out_stride, scratch, nbytes, nqh, window, scale, None)


def append(kv=None, b=None, qkv=P, dtype=0, stride=768, q_out=2 * P, nqh=8, rot=64, theta=1e4):
    return _lib.lib().launch_rope_kv_append_paged(qkv, dtype, stride, q_out, kv or pool(), b or seqs(), nqh, rot, theta, None)


def packed(b=None, q=P, k=P, v=P, dtype=1, qs=512, ks=128, vs=128, out=2 * P, out_dtype=1, os=512, nqh=8, nkv=2, hd=64, window=0, scale=1.0):
    return _lib.lib().launch_attn_packed(q, k, v, dtype, qs, ks, vs, b or seqs(kv_len=None), out, out_dtype, os, nqh, nkv, hd, window, scale, None)


def test_no_rows_is_fine():
    assert attn() == 0 and append() == 0 and packed() == 0


@pytest.mark.parametrize("kw,status", [
    (dict(k_pages=None), -1), (dict(v_pages=None), -1), (dict(page_table=None), -1), (dict(dtype=0), -5), (dict(dtype=9), -5), (dict(n_pages=0), -2),
    (dict(page_size=0), -2), (dict(n_kv_heads=0), -2), (dict(head_dim=-64), -2), (dict(k_page_stride=100), -2), (dict(v_page_stride=-1), -2),
    (dict(k_pages=P + 2), -4), (dict(v_pages=P + 8), -4), (dict(k_page_stride=2052), -4), (dict(table_stride=-1), -2)])
def test_pools(kw, status):
    assert attn(pool(**kw)) == status
    assert append(pool(**kw)) == status


@pytest.mark.parametrize("kw,status", [(dict(cu_q=None), -1), (dict(kv_len=None), -1), (dict(n_seqs=0), -2), (dict(total_q=-1), -2), (dict(max_kv=-1), -2),
                                       (dict(max_q=-1), -2), (dict(n_seqs=1 << 21), -3)])
def test_batches(kw, status):
    assert attn(b=seqs(**kw)) == status
    assert append(b=seqs(**kw)) == status
    if "kv_len" not in kw and "max_kv" not in kw:
        assert packed(b=seqs(**kw)) == status


@pytest.mark.parametrize("kw,status", [
    (dict(q=None), -1), (dict(out=None), -1), (dict(scratch=None), -1), (dict(out_dtype=7), -5), (dict(q_stride=504), -2), (dict(out_stride=510), -2),
    (dict(nqh=7), -2), (dict(nqh=0), -2), (dict(window=-1), -2), (dict(scale=0.0), -2), (dict(scale=-1.0), -2), (dict(scale=NAN), -2),
    (dict(scale=INF), -2), (dict(out=P), -2), (dict(q=P + 8), -4), (dict(q_stride=516), -4), (dict(out=2 * P + 2), -4), (dict(out_stride=513), -4),
    (dict(scratch=P + 4), -4), (dict(nbytes=1000), -7), (dict(kv=pool(head_dim=80)), -3), (dict(kv=pool(page_size=12)), -3),
    (dict(nqh=2 * 65, q_stride=130 * 64, out_stride=130 * 64), -3), (dict(out_dtype=0, out=2 * P + 4), -4)])
def test_attention(kw, status):
    assert attn(**kw) == status


@pytest.mark.parametrize("kw,status", [
    (dict(qkv=None), -1), (dict(q_out=None), -1), (dict(dtype=3), -5), (dict(stride=760), -2), (dict(nqh=0), -2), (dict(rot=63), -2), (dict(rot=66), -2),
    (dict(rot=-2), -2), (dict(theta=0.0), -2), (dict(theta=NAN), -2), (dict(theta=INF), -2), (dict(q_out=P), -2), (dict(qkv=P + 2), -4),
    (dict(kv=pool(head_dim=512), rot=258, stride=12 * 512), -3)])
def test_append(kw, status):
    assert append(**kw) == status


@pytest.mark.parametrize("kw,status", [
    (dict(q=None), -1), (dict(k=None), -1), (dict(v=None), -1), (dict(out=None), -1), (dict(dtype=0), -5), (dict(out_dtype=5), -5), (dict(qs=500), -2),
    (dict(ks=120), -2), (dict(vs=120), -2), (dict(os=510), -2), (dict(nkv=3), -2), (dict(hd=48), -3), (dict(q=P + 8), -4), (dict(k=P + 8), -4),
    (dict(v=P + 2), -4), (dict(ks=132), -4), (dict(vs=132), -4), (dict(out=P), -2), (dict(scale=0.0), -2), (dict(window=-4), -2)])
def test_packed(kw, status):
    assert packed(**kw) == status


def test_scratch_sizes():
    L = _lib.lib()
    assert L.qmm_attn_paged_scratch_bytes(-1, 8, 2, 64) == -2
    assert L.qmm_attn_paged_scratch_bytes(1, 8, 3, 64) == -2
    assert L.qmm_attn_paged_scratch_bytes(1, 8, 2, 72) == -3
    for hd in (32, 64, 96, 128, 256):
        assert 0 < L.qmm_attn_paged_scratch_bytes(1, 8, 2, hd) < 1 << 27
        assert 0 < L.qmm_attn_paged_scratch_bytes(1000, 8, 2, hd) < 1 << 27


def test_structs_match_the_header():
    assert C.sizeof(SeqBatch) == 32 and C.sizeof(PagedKV) == 72
