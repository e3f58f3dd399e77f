"""The operators on a paged KV cache and on packed prompts at the ends of their ranges: the widest windows, the longest sequences,
bits that must not change, keys that are infinite, whole prompts through the cache.  References and bounds: paged_ref.py.
Needs a B200."""
import pytest
import torch

import paged_ref as ref
from test_gpu_paged import BF16, F16, F32, check, ops, pack, packed, paged  # noqa: F401 (ops is a fixture)

pytestmark = pytest.mark.gpu


# ---- windows ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("window", [(1 << 31) - 1, (1 << 31) - 2, 1 << 30])
@pytest.mark.parametrize("hd,q_len,kv", [(64, 4, 1), (128, 200, 130), (256, 60, 3)])
def test_windows_longer_than_any_sequence(ops, hd, q_len, kv, window):
    """They hide nothing, also where the first new tokens have no position (kv_len smaller than their number)."""
    b = ref.Batch([q_len, 3], [kv, 40], 8, 2, hd, 16, F16, seed=hd, spare_rows=1)
    assert torch.equal(check(ops, b, window=window), check(ops, b))


# ---- lengths ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("q_len", [1, 20])
def test_the_longest_sequences(ops, q_len):
    """2^31 - 4096 keys, every page of the table the same one, all scores 0 and all values 1: sums of ones below 2^24 are exact and
    those of the parts are rounded alike above and below the line, so the outputs are 1.  Longer ones are cut and reported."""
    page, longest = 1 << 16, (1 << 31) - 4096
    k = torch.zeros(1, page, 1, 32, dtype=F16, device="cuda")
    v = torch.ones_like(k)
    table = torch.zeros(1, 1 << 15, dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, q_len], dtype=torch.int32, device="cuda")
    q = torch.ones(q_len, 32, dtype=F16, device="cuda")
    for kv in (longest, longest + 1, (1 << 31) - 1):
        out = torch.full((q_len, 32), 77.0, dtype=F16, device="cuda")
        ops.gpu_gqa_attn_paged_into(q, k, v, table, cu, torch.tensor([kv], dtype=torch.int32, device="cuda"), out, 1, q_len, kv)
        if kv == longest:
            ops.check_launch()
            assert (out == 1).all()
        else:
            with pytest.raises(RuntimeError, match="status 7"):
                ops.check_launch()


# ---- what a row does not see -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("hd,nqh,nkv", [(128, 8, 2), (64, 7, 1), (256, 4, 4), (32, 12, 4)])
def test_a_large_later_key_changes_no_bit_of_the_rows_before(ops, hd, nqh, nkv):
    """The last key of a chunk takes all the weight of the last token; the rows of the tokens before share its tiles and warps."""
    b = ref.Batch([50, 50], [450, 333], nqh, nkv, hd, 16, BF16, seed=hd)
    one = paged(ops, b, out_dtype=F32).view(-1, nqh, hd)
    key = int(b.table[0, 449 // 16]), 449 % 16
    b.k[key] = 60.0 * torch.sign(b.q[49].view(nqh, hd)[::nqh // nkv]).to(BF16)
    two = paged(ops, b, out_dtype=F32).view(-1, nqh, hd)
    ops.check_launch()
    assert not torch.equal(one[49], two[49])
    assert torch.equal(one[:49], two[:49]) and torch.equal(one[50:], two[50:])


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_a_large_later_row_of_a_packed_prompt_changes_no_bit_of_the_rows_before(ops, hd):
    lens = [300, 90]
    qkv = torch.randn(390, 12 * hd, device="cuda", generator=torch.Generator(device="cuda").manual_seed(hd)).bfloat16()
    one = packed(ops, pack(qkv, lens, 8, 2, hd, BF16), qkv, out_dtype=F32)
    qkv[290, 8 * hd:10 * hd] *= 300
    two = packed(ops, pack(qkv, lens, 8, 2, hd, BF16), qkv, out_dtype=F32)
    ops.check_launch()
    assert not torch.equal(one[290:300], two[290:300])
    assert torch.equal(one[:290], two[:290]) and torch.equal(one[300:], two[300:])


@pytest.mark.parametrize("bad", [float("inf"), float("-inf")])
@pytest.mark.parametrize("hd,q_len", [(128, 1), (64, 2), (256, 3), (128, 100), (64, 300), (256, 80), (32, 70)])
def test_infinite_keys(ops, hd, q_len, bad):
    """Rows before it do not see it; a row that sees it is NaN where its score is +inf, and what it is without that key where its
    score is -inf."""
    kv = q_len + 77
    b = ref.Batch([q_len, 5], [kv, 9], 8, 2, hd, 16, BF16, seed=q_len + hd)
    b.q.view(-1, 8, hd)[:, 4:, 0] = torch.tensor([0.5, -0.5, 1.5, -2.0], device="cuda")  # heads of both signs
    want, tol = ref.expect(b, hd ** -0.5, 0, BF16)
    key = kv - max(q_len // 3, 1)
    page, slot = int(b.table[0, key // 16]), key % 16
    b.k[page, slot, 1, 0] = bad
    n = kv - key  # tokens that see it: the last ones
    rows = slice(q_len - n, q_len)
    keep = [t for t in range(kv) if t != key]
    want[rows], tol[rows] = (torch.cat([whole, gone[:, 4:]], dim=1) for whole, gone in zip(
        (want[rows][:, :4], tol[rows][:, :4]),
        ref.attention(b.q[rows].view(n, 8, hd), b.keys[0][keep], b.vals[0][keep], hd ** -0.5, 0, BF16, BF16)))
    got = paged(ops, b).view(-1, 8, hd)
    ops.check_launch()
    up = torch.zeros(b.total, 8, dtype=torch.bool, device="cuda")
    up[rows, 4:] = b.q.view(-1, 8, hd)[rows][:, 4:, 0] * bad > 0
    assert torch.isnan(got[up]).all()
    ref.near(torch.where(up[..., None], 0.0, got.double()), torch.where(up[..., None], 0.0, want), torch.where(up[..., None], 0.0, tol))


def test_values_near_the_end_of_a_bf16_cache(ops):
    """Sums of values of 1e30 with probabilities of up to 256 (scores that grow slowly from key to key) stay finite."""
    b = ref.Batch([1, 100], [900, 900], 8, 2, 64, 16, BF16, seed=31, values=1e30)
    ramp = torch.linspace(0, 30, 900).to(BF16).cuda()
    b.q.zero_()
    b.q.view(-1, 8, 64)[..., 0] = 1.0
    for s in range(2):
        b.keys[s][:] = 0
        b.keys[s][..., 0] = ramp[:, None]
        for t in range(900):
            b.k[int(b.table[s, t // 16]), t % 16] = b.keys[s][t]
    check(ops, b, scale=1.0)


def one_hot_batch(q_lens, kv_lens, hd, base, step, nqh=8, nkv=2, order=1):
    """Scores that f32 holds exactly: q = (base, step, 0 ..), key t = (base, +-t, 0 ..), so q . k = base^2 +- step t."""
    b = ref.Batch(q_lens, kv_lens, nqh, nkv, hd, 16, F16, seed=hd)
    b.q.zero_()
    b.q.view(-1, nqh, hd)[..., 0], b.q.view(-1, nqh, hd)[..., 1] = base, step
    for s, n in enumerate(kv_lens):
        b.keys[s].zero_()
        b.keys[s][..., 0], b.keys[s][..., 1] = base, order * torch.arange(n, device="cuda").half()[:, None]
        for t in range(n):
            b.k[int(b.table[s, t // 16]), t % 16] = b.keys[s][t]
    return b


@pytest.mark.parametrize("order", [1, -1])
@pytest.mark.parametrize("hd,q_len", [(64, 1), (128, 60), (64, 200), (256, 40), (32, 70)])
def test_scores_far_from_zero(ops, hd, q_len, order):
    """2^30 and more, whose differences decide.  With a scale of 1 the best key has all the weight; with 2^-6 the scores are 2^24
    +- 2 t, which f32 holds and the weights have to follow: exact scores leave the bound of the probabilities' rounding, of f32
    sums (600 keys) and of the output's rounding."""
    b = one_hot_batch([q_len, 3], [600, 50], hd, 32768.0, 128.0, order=order)
    for scale in (1.0, 2.0 ** -6):
        out = paged(ops, b, scale=scale, out_dtype=F32).view(-1, 8, hd)
        ops.check_launch()
        for s, (n, t) in enumerate(zip(b.q_lens, b.kv_lens)):
            pos, key = torch.arange(t - n, t, device="cuda")[:, None], torch.arange(t, device="cuda")[None]
            x = torch.where(key <= pos, scale * (2.0 ** 30 + order * 128.0 * key.double()), float("-inf"))
            p = torch.softmax(x, dim=1)
            v = b.vals[s].double().repeat_interleave(4, dim=1)
            want, size = torch.einsum("nt,thd->nhd", p, v), torch.einsum("nt,thd->nhd", p, v.abs())
            ref.near(out[b.rows(s)], want, size * (2.0 ** -11 + 2.0 ** -19 + 700 * 2.0 ** -23) + 2.0 ** -25 * t * v.abs().max(), f"scale {scale}")


# ---- long batches ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,nqh,nkv,q_lens,kv_lens", [
    (128, 8, 2, [1500], [1500]), (64, 14, 2, [1100, 3], [1100, 4000]), (256, 4, 2, [700], [700]), (96, 12, 4, [900], [2500]),
    (128, 16, 8, [30] * 60 + [1200], [300] * 60 + [1500]), (64, 16, 16, [17] * 150 + [600], [17] * 150 + [900]),
    (256, 8, 8, [40] * 50 + [500], [40] * 50 + [500]), (128, 32, 1, [1] * 40 + [1], [200] * 40 + [9000])])
def test_prompts_through_the_cache_and_batches_that_end_in_their_longest(ops, dtype, hd, nqh, nkv, q_lens, kv_lens):
    check(ops, ref.Batch(q_lens, kv_lens, nqh, nkv, hd, 32, dtype, seed=hd + len(q_lens), spare_rows=1))


@pytest.mark.parametrize("hd,nqh,nkv", [(128, 32, 8), (64, 4, 4), (256, 8, 4)])
def test_packed_batches_that_end_in_their_longest(ops, hd, nqh, nkv):
    lens = [30 + i % 50 for i in range(60)] + [1500]
    qkv = torch.randn(sum(lens), (nqh + 2 * nkv) * hd, device="cuda", generator=torch.Generator(device="cuda").manual_seed(hd)).half()
    b = pack(qkv, lens, nqh, nkv, hd, F16)
    out = packed(ops, b, qkv)
    ops.check_launch()
    ref.near(out, *ref.expect(b, hd ** -0.5, 0, F16))


# ---- tables and pages ------------------------------------------------------------------------------------------------
def test_page_tables_inside_wider_ones(ops):
    for q_lens, kv_lens in (([1, 1, 1], [100, 333, 7]), ([90, 7, 0], [100, 333, 20])):
        b = ref.Batch(q_lens, kv_lens, 8, 2, 64, 16, F16, seed=41)
        want = paged(ops, b)
        n = b.table.shape[1]
        wide = torch.full((3, n + 9), -5, dtype=torch.int32, device="cuda")
        wide[:, 4:4 + n] = b.table
        b.table = wide[:, 4:4 + n]
        assert torch.equal(check(ops, b), want)
        new = torch.randn(b.total, 12 * 64, device="cuda")
        k, v, q_out = b.k.clone(), b.v.clone(), [torch.empty(b.total, 512, dtype=F16, device="cuda") for _ in range(2)]
        ops.gpu_rope_kv_append_paged_into(new, q_out[0], b.k, b.v, b.table, b.cu, b.kv_len, 8, 1e4)
        ops.gpu_rope_kv_append_paged_into(new, q_out[1], k, v, b.table.contiguous(), b.cu, b.kv_len, 8, 1e4)
        ops.check_launch()
        for x, y in ((b.k, k), (b.v, v), q_out):
            assert torch.equal(x.view(torch.int16), y.view(torch.int16))
        b.max_kv = 16 * (n + 9)
        b.kv_len[1] = 16 * n + 1  # one more than the columns given have room for
        paged(ops, b)
        with pytest.raises(RuntimeError, match="status 7"):
            ops.check_launch()


def test_a_bad_page_takes_nothing(ops):
    """A new token whose table entry is no page of the pool is written nowhere: only the other sequence's pages change."""
    for bad in (-1, 1 << 30, -(1 << 31)):
        b = ref.Batch([1, 30], [50, 90], 8, 2, 128, 16, F16, seed=15, poison=False)
        own = set(b.table[1, :6].tolist())
        b.table[0, 3] = bad
        k, v = b.k.clone(), b.v.clone()
        ops.gpu_rope_kv_append_paged_into(torch.randn(31, 12 * 128, device="cuda"), torch.empty_like(b.q), b.k, b.v, b.table, b.cu, b.kv_len, 8, 1e4)
        with pytest.raises(RuntimeError, match="status 6"):
            ops.check_launch()
        for x, y in ((b.k, k), (b.v, v)):
            touched = set((x != y).flatten(1).any(dim=1).nonzero().flatten().tolist())
            assert touched and touched <= own
        assert len(own) < b.n_pages


def test_batches_without_rows_do_nothing(ops):
    k = torch.zeros(4, 16, 2, 64, dtype=F16, device="cuda")
    cu, kv, table = (torch.zeros(*n, dtype=torch.int32, device="cuda") for n in ((3,), (2,), (2, 2)))
    q = torch.empty(0, 512, dtype=F16, device="cuda")
    ops.gpu_rope_kv_append_paged_into(torch.empty(0, 768, device="cuda"), q, k, k, table, cu, kv, 8, 1e4)
    ops.gpu_gqa_attn_paged_into(q, k, k, table, cu, kv, torch.empty_like(q), 8, 0, 0)
    ops.gpu_gqa_attn_packed_into(q, q[:, :128], q[:, :128], cu, torch.empty_like(q), 8, 2, 64, 0)
    ops.check_launch()


@pytest.mark.parametrize("ws", [lambda n: torch.empty(2 * n, dtype=torch.uint8, device="cuda")[::2], lambda n: torch.empty(1, dtype=torch.uint8, device="cuda").expand(n)])
def test_workspaces_that_are_not_contiguous_are_refused(ops, ws):
    b = ref.Batch([1, 2], [9, 30], 8, 2, 64, 16, F16, seed=23, poison=False)
    n = ops.gpu_gqa_attn_paged_scratch(b.q, b.k, b.kv_len, 8, 2, 30).numel()
    with pytest.raises(ValueError, match="scratch"):
        paged(ops, b, scratch=ws(n))


# ---- streams ---------------------------------------------------------------------------------------------------------
def test_calls_at_the_same_time_on_two_streams(ops):
    """Each with a workspace of its own: decode, chunks and packed prompts side by side give what they give one after another."""
    a = ref.Batch([1] * 20, [300 * i + 1 for i in range(20)], 32, 8, 128, 16, F16, seed=51)
    b = ref.Batch([100, 30, 1], [3000, 700, 2000], 8, 2, 64, 16, BF16, seed=52)
    qkv = torch.randn(900, 12 * 256, device="cuda").half()
    c = pack(qkv, [600, 300], 8, 2, 256, F16)
    calls = [lambda ws: paged(ops, a, scratch=ws), lambda ws: paged(ops, b, scratch=ws), lambda ws: packed(ops, c, qkv)]
    spaces = [[ops.gpu_gqa_attn_paged_scratch(x.q, x.k, x.kv_len, x.nqh, x.max_q, x.max_kv) for x in (a, b)] + [None] for _ in range(2)]
    want = [f(ws) for f, ws in zip(calls, spaces[0])]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for i in range(12):
        for j, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                n = (i + j) % 3
                got.append((n, calls[n](spaces[j][n])))
    torch.cuda.synchronize()
    ops.check_launch()
    for n, out in got:
        assert torch.equal(out, want[n])
