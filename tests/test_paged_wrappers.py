"""The Python forms of the paged-cache operators without a GPU: what they refuse, and what they hand to the library.  Tensors in
host memory pass for tensors of device 0, and the launch is recorded instead of made."""
import pytest
import torch

from nates_recipe_rs_b200 import quant_ops as ops

F16, I32 = torch.float16, torch.int32


@pytest.fixture
def launches(monkeypatch):
    calls = []
    monkeypatch.setattr(torch.Tensor, "get_device", lambda self: 0)
    monkeypatch.setattr(ops, "_launch_on", lambda index, name, *args: calls.append((name, args)))
    return calls


def batch(**kw):
    d = dict(q=torch.zeros(3, 8 * 64, dtype=F16), kpages=torch.zeros(6, 16, 2, 64, dtype=F16), vpages=torch.zeros(6, 16, 2, 64, dtype=F16),
             page_table=torch.zeros(2, 3, dtype=I32), cu_q=torch.zeros(3, dtype=I32), kv_len=torch.zeros(2, dtype=I32), out=torch.zeros(3, 8 * 64),
             scratch=torch.empty(4096, dtype=torch.uint8), nqh=8, max_q=2, max_kv=30)
    d.update(kw)
    return d


def attn(**kw):
    ops.gpu_gqa_attn_paged_into(**batch(**kw))


def append(**kw):
    d = batch(**{"out": torch.zeros(3, 8 * 64, dtype=F16), **kw})
    ops.gpu_rope_kv_append_paged_into(d.get("qkv", torch.zeros(3, 12 * 64)), d["out"], d["kpages"], d["vpages"], d["page_table"], d["cu_q"], d["kv_len"], 8, 1e4)


def test_calls_reach_the_library(launches):
    attn()
    append()
    assert [c[0] for c in launches] == ["launch_attn_paged", "launch_rope_kv_append_paged"]


@pytest.mark.parametrize("ws", [lambda: torch.empty(1 << 13, dtype=torch.uint8)[::2], lambda: torch.empty(64, 64, dtype=torch.uint8)[:, 0],
                                lambda: torch.empty(1, dtype=torch.uint8).expand(1 << 20)])
def test_a_workspace_must_be_contiguous(launches, ws):
    """Its bytes are counted from the elements: those of a view with gaps are not all its own, an expanded one has only one."""
    with pytest.raises(ValueError, match="scratch"):
        attn(scratch=ws())
    assert not launches


@pytest.mark.parametrize("which", ["kpages", "vpages"])
def test_pages_must_not_share_memory(launches, which):
    """An expanded pool has a page stride of 0, which the library reads as 'back to back'; overlapping pages are no pool either."""
    for pages in (torch.zeros(1, 16, 2, 64, dtype=F16).expand(6, 16, 2, 64), torch.zeros(1 << 14, dtype=F16).as_strided((6, 16, 2, 64), (1024, 128, 64, 1))):
        for call in (attn, append):
            with pytest.raises(ValueError, match="pages"):
                call(**{which: pages})
    assert not launches


def packed(rows, cu):
    x = torch.zeros(rows, 12 * 64, dtype=F16)
    ops.gpu_gqa_attn_packed_into(x[:, :512], x[:, 512:640], x[:, 640:], cu, torch.zeros(rows, 512), 8, 2, 64, 0)


@pytest.mark.parametrize("n_seqs,rows", [(2, 0), (0, 0), (0, 3)])
def test_batches_without_rows_or_sequences_do_nothing(launches, n_seqs, rows):
    """A server's step without new tokens: tensors of no elements have no address to hand to the library."""
    kw = dict(q=torch.zeros(rows, 512, dtype=F16), cu_q=torch.zeros(n_seqs + 1, dtype=I32), kv_len=torch.zeros(n_seqs, dtype=I32),
              page_table=torch.zeros(n_seqs, 3, dtype=I32))
    attn(out=torch.zeros(rows, 512), **kw)
    append(qkv=torch.zeros(rows, 768), out=torch.zeros(rows, 512, dtype=F16), **kw)
    packed(rows, kw["cu_q"])
    assert not launches
    for kw in (dict(kw, page_table=kw["page_table"].long()), dict(kw, cu_q=kw["cu_q"].float()), dict(kw, q=kw["q"][:, :-1])):
        with pytest.raises(ValueError):
            attn(out=torch.zeros(rows, 512), **kw)
    with pytest.raises(ValueError, match="cu_q"):
        packed(rows, torch.zeros(0, dtype=I32))


def test_page_tables_inside_wider_ones(launches):
    """A server's table cut to the pages in use: its rows lie further apart than they are long, and no length reaches past the cut."""
    wide = torch.zeros(5, 40, dtype=I32)
    table = wide[1:3, 4:7]
    attn(page_table=table)
    attn(page_table=table, max_kv=1000)
    append(page_table=table)
    attn(page_table=wide[1:2, 4:7], q=torch.zeros(3, 512, dtype=F16), cu_q=torch.zeros(2, dtype=I32), kv_len=torch.zeros(1, dtype=I32))
    (_, a), (_, long), (_, b), (_, one) = launches
    for pool, batch in ((a[2], a[3]), (long[2], long[3]), (b[4], b[5])):
        assert pool.page_table == table.data_ptr() and pool.table_stride == 40 and batch.n_seqs == 2
    assert (a[3].max_kv, long[3].max_kv, b[5].max_kv, one[3].max_kv) == (30, 48, 48, 30)


@pytest.mark.parametrize("table", [lambda: torch.zeros(2, 6, dtype=I32)[:, ::2], lambda: torch.zeros(3, 2, dtype=I32).T, lambda: torch.zeros(1, 3, dtype=I32).expand(2, 3),
                                   lambda: torch.zeros(2, 3), lambda: torch.zeros(3, 3, dtype=I32), lambda: torch.zeros(6, dtype=I32)])
def test_page_tables_that_are_refused(launches, table):
    for call in (attn, append):
        with pytest.raises(ValueError, match="page_table"):
            call(page_table=table())
    assert not launches


@pytest.mark.parametrize("pool", [lambda: torch.zeros(6, 1, 16, 64, dtype=F16).transpose(1, 2), lambda: torch.zeros(6, 1, 64, dtype=F16).as_strided((6, 1, 1, 64), (64, 7, 9, 1)),
                                  lambda: torch.zeros(6, 2, 1, 64, dtype=F16).as_strided((6, 1, 2, 64), (128, 999, 64, 1))])
def test_strides_of_dimensions_of_one_element_do_not_matter(launches, pool):
    """One kv head kept heads first, or one slot a page: the pages are contiguous whatever such a dimension's stride says."""
    k, v = pool(), pool()
    page, nkv = k.shape[1:3]
    attn(kpages=k, vpages=v)
    append(kpages=k, vpages=v, qkv=torch.zeros(3, (8 + 2 * nkv) * 64))
    for _, args in launches:
        pool_arg = next(a for a in args if hasattr(a, "k_page_stride"))
        assert (pool_arg.page_size, pool_arg.n_kv_heads, pool_arg.k_page_stride) == (page, nkv, page * nkv * 64)
    assert len(launches) == 2
    for bad in (torch.zeros(6, 2, 16, 64, dtype=F16).transpose(1, 2), torch.zeros(6, 16, 1, 128, dtype=F16)[..., ::2]):
        with pytest.raises(ValueError, match="pages"):
            attn(kpages=bad, vpages=bad)


@pytest.mark.parametrize("window,given", [(0, 0), (7, 7), ((1 << 31) - 1, (1 << 31) - 1), (1 << 31, (1 << 31) - 1), ((1 << 32) + 5, (1 << 31) - 1), ((1 << 63) - 1, (1 << 31) - 1)])
def test_windows_past_32_bits_hide_nothing(launches, window, given):
    """The library takes 32 bits, and a number beyond them is not refused on the way there but loses its upper ones."""
    attn(window=window)
    x = torch.zeros(3, 768, dtype=F16)
    ops.gpu_gqa_attn_packed_into(x[:, :512], x[:, 512:640], x[:, 640:], torch.zeros(2, dtype=I32), torch.zeros(3, 512), 8, 2, 64, 3, window=window)
    assert [args[-2] for _, args in launches] == [given, given]
