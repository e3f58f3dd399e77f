"""The operators on a paged KV cache and on packed prompts against their plain 64-bit forms (tests/paged_ref.py, where the
tolerances are derived): lengths from none to many tokens, pages that end inside a tile, windows, rows that see nothing, groups
of every kind, strides, poison wherever the operators must not look.  Needs a B200."""
import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.fail("these tests need a CUDA device")
    from nates_recipe_rs_b200 import quant_ops
    return quant_ops


def paged(ops, b, out_dtype=None, window=0, scale=None, max_q=None, **kw):
    scale = b.hd ** -0.5 if scale is None else scale
    out = torch.full((b.total, b.nqh * b.hd), 77.0, dtype=out_dtype or b.dtype, device="cuda")
    ops.gpu_gqa_attn_paged_into(b.q, b.k, b.v, b.table, b.cu, b.kv_len, out, b.nqh, max_q or b.max_q, b.max_kv, scale, window=window, **kw)
    return out


def check(ops, b, out_dtype=None, window=0, scale=None, **kw):
    scale = b.hd ** -0.5 if scale is None else scale
    out = paged(ops, b, out_dtype, window, scale, **kw)
    ops.check_launch()
    want, tol = ref.expect(b, scale, window, out.dtype)
    ref.near(out, want, tol)
    assert (out[sum(b.q_lens):] == 77.0).all(), "rows behind the last sequence"
    return out


# ---- single tokens ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,nqh,nkv,page", [(128, 32, 8, 16), (64, 14, 2, 48), (96, 12, 4, 24), (256, 8, 4, 8), (32, 3, 1, 64), (128, 16, 1, 256),
                                             (64, 4, 4, 40)])
def test_decode(ops, dtype, hd, nqh, nkv, page):
    lens = [1, 2, 63, 64, 65, 127, 300, 1000, page, page + 1]
    check(ops, ref.Batch([1] * len(lens), lens, nqh, nkv, hd, page, dtype, seed=hd + page, spare_rows=3))


@pytest.mark.parametrize("hd,nqh,nkv,window", [(128, 8, 2, 1), (128, 8, 2, 100), (64, 7, 1, 64), (256, 4, 4, 1000)])
def test_decode_with_window(ops, hd, nqh, nkv, window):
    lens = [1, 64, 99, 100, 101, 1111, 5000]
    check(ops, ref.Batch([1] * len(lens), lens, nqh, nkv, hd, 16, F16, seed=window), window=window)


@pytest.mark.parametrize("n", [1, 3, 200, 700])
def test_decode_of_many_sequences(ops, n):
    """More sequences than a CTA has threads, lengths of all sizes, some without a new token."""
    lens = [(i * 37) % 400 + 1 for i in range(n)]
    check(ops, ref.Batch([0 if i % 5 == 3 else 1 for i in range(n)], lens, 8, 2, 64, 16, BF16, seed=n))


def test_decode_of_one_long_sequence(ops):
    """One sequence over all CTAs: many parts joined."""
    check(ops, ref.Batch([1], [50001], 32, 8, 128, 64, F16, seed=9))
    check(ops, ref.Batch([2], [30011], 4, 1, 256, 80, BF16, seed=10))


@pytest.mark.parametrize("out_dtype", [F16, BF16, F32])
def test_output_types(ops, out_dtype):
    check(ops, ref.Batch([1, 5, 40], [70, 5, 140], 8, 2, 128, 16, F16, seed=3), out_dtype)
    check(ops, ref.Batch([1, 1], [70, 500], 8, 2, 64, 16, BF16, seed=4), out_dtype)


# ---- pieces of prompts -----------------------------------------------------------------------------------------------
CHUNKS = [([3], [3]), ([2, 1, 0, 4], [900, 1, 17, 4]), ([17, 64, 65, 1, 0, 130], [17, 500, 129, 700, 0, 131]), ([300, 1, 31], [1500, 2000, 31])]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,nqh,nkv,page", [(128, 32, 8, 16), (64, 14, 2, 48), (96, 12, 4, 24), (256, 8, 4, 16), (32, 6, 2, 128), (128, 5, 5, 64),
                                             (64, 64, 1, 8)])
@pytest.mark.parametrize("lens", CHUNKS)
def test_chunks(ops, dtype, hd, nqh, nkv, page, lens):
    check(ops, ref.Batch(*lens, nqh, nkv, hd, page, dtype, seed=hd + page + len(lens[0]), spare_rows=2))


@pytest.mark.parametrize("hd,window", [(128, 1), (128, 33), (64, 128), (256, 200), (96, 5000), (32, 64)])
def test_chunks_with_window(ops, hd, window):
    check(ops, ref.Batch([200, 1, 37, 64], [900, 640, 37, 1000], 12, 4, hd, 16, BF16, seed=window), window=window)


@pytest.mark.parametrize("q_len", [1, 40, 300])
def test_rows_that_see_nothing_are_zero(ops, q_len):
    """kv_len of zero, and fewer keys than new tokens: the rows before position 0 see no key."""
    for hd in (64, 128, 256):
        b = ref.Batch([q_len, q_len, q_len], [0, max(q_len // 2, 1), 3 * q_len], 8, 2, hd, 16, F16, seed=q_len)
        out = check(ops, b)
        assert (out[:q_len] == 0).all()


@pytest.mark.parametrize("where", ["later", "before the window"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("hd,q_len", [(128, 100), (64, 300), (256, 80), (32, 70), (128, 3)])
def test_values_a_row_does_not_see_have_no_influence(ops, hd, q_len, bad, where):
    """A key or a value that is not finite reaches the rows that see it and no others."""
    kv = q_len + 77
    window = 0 if where == "later" else 30
    b = ref.Batch([q_len, 5], [kv, 9], 8, 2, hd, 16, BF16, seed=q_len)
    key = kv - q_len // 3 if where == "later" else kv - q_len + 2
    b.vals[0][key, 0, 3] = bad
    page, slot = int(b.table[0, key // 16]), key % 16
    b.v[page, slot, 0, 3] = bad
    scale = hd ** -0.5
    out = paged(ops, b, window=window)
    ops.check_launch()
    want, tol = ref.expect(b, scale, window, BF16)
    pos = torch.arange(kv - q_len, kv, device="cuda")
    sees = (pos >= key) & ((pos - key < window) if window else True)
    got = out.view(-1, 8, hd)
    assert not torch.isfinite(got[:q_len][sees][:, :4, 3]).any(), "rows that see it"
    mask = torch.ones_like(want, dtype=torch.bool)
    mask[:q_len][sees] = False
    ref.near(torch.where(mask, got.double(), 0.0), torch.where(mask, want, 0.0), tol)
    # the other elements of the rows that see it are what they were
    other = [d for d in range(hd) if d != 3]
    ref.near(got[:q_len][sees][..., other], want[:q_len][sees][..., other], tol[:q_len][sees][..., other])
    # a key that is not finite
    b.k[page, slot, 1, 0] = bad
    out = paged(ops, b, window=window)
    ops.check_launch()
    got = out.view(-1, 8, hd)
    assert torch.isnan(got[:q_len][sees][:, 4:]).any(dim=-1).all() or bad == float("inf")
    ref.near(torch.where(mask, got.double(), 0.0), torch.where(mask, want, 0.0), tol)


def test_large_scores(ops):
    """A scale that makes single keys take all the weight, and one that makes all equal."""
    for scale in (4.0, 1e-4):
        check(ops, ref.Batch([1, 1, 1], [1000, 64, 7], 8, 2, 128, 16, F16, seed=5), scale=scale, out_dtype=F32)
        check(ops, ref.Batch([100, 30], [400, 30], 8, 2, 128, 16, F16, seed=6), scale=scale, out_dtype=F32)


def test_growing_scores(ops):
    """Every later key beats the ones before by far: the running maximum moves all the time."""
    b = ref.Batch([1, 140], [700, 900], 4, 2, 64, 16, F16, seed=8)
    b.q.fill_(0.5)
    for s in range(2):
        n = b.kv_lens[s]
        ramp = torch.linspace(-4, 4, n, device="cuda").half()[:, None, None].expand(n, 2, 64)
        b.keys[s] = ramp.contiguous()
        for t in range(n):
            b.k[int(b.table[s, t // 16]), t % 16] = ramp[t]
    check(ops, b, scale=1.0, out_dtype=F32)


def test_strides_and_interleaved_pools(ops):
    """K and V pages side by side in one allocation, rows of q and out inside wider ones."""
    for q_lens, kv_lens in (([1, 1], [100, 333]), ([90, 7], [100, 333])):
        b = ref.Batch(q_lens, kv_lens, 8, 2, 128, 16, F16, seed=11)
        both = torch.empty(b.n_pages, 2, 16, 2, 128, dtype=F16, device="cuda")
        both[:, 0], both[:, 1] = b.k, b.v
        wide = torch.full((b.total, 8 * 128 + 40), float("nan"), dtype=F16, device="cuda")
        wide[:, 8:8 + 8 * 128] = b.q
        out = torch.full((b.total, 8 * 128 + 6), 77.0, dtype=F16, device="cuda")
        ops.gpu_gqa_attn_paged_into(wide[:, 8:8 + 8 * 128], both[:, 0], both[:, 1], b.table, b.cu, b.kv_len, out[:, 2:2 + 8 * 128], 8, b.max_q, b.max_kv,
                                    128 ** -0.5)
        ops.check_launch()
        assert torch.equal(out[:, 2:2 + 8 * 128], paged(ops, b))
        assert (out[:, :2] == 77.0).all() and (out[:, 2 + 8 * 128:] == 77.0).all()


def test_offsets_past_32_bits(ops):
    """Pages whose elements lie beyond 2^32 bytes and 2^31 elements of the pool."""
    nkv, hd, page = 8, 128, 256
    n_pages = (1 << 31) // (page * nkv * hd) + 9
    k = torch.empty(n_pages, page, nkv, hd, dtype=F16, device="cuda")
    v = torch.empty_like(k)
    for q_lens, kv_lens in (([1, 1], [300, 500]), ([40, 130], [300, 500])):
        b = ref.Batch(q_lens, kv_lens, 32, nkv, hd, page, F16, seed=12)
        table = torch.zeros_like(b.table)
        at = n_pages - 6
        for s, n in enumerate(kv_lens):
            for j in range(-(-n // page)):
                k[at], v[at] = b.k[int(b.table[s, j])], b.v[int(b.table[s, j])]
                table[s, j] = at
                at += 1
        b.k, b.v, b.table = k, v, table
        check(ops, b)
        new = torch.randn(b.total, 48 * 128, device="cuda", dtype=F16)
        q_out = torch.empty(b.total, 32 * 128, dtype=F16, device="cuda")
        ops.gpu_rope_kv_append_paged_into(new, q_out, k, v, table, b.cu, b.kv_len, 32, 1e4)
        ops.check_launch()
        last = kv_lens[1] - 1
        assert torch.equal(v[int(table[1, last // page]), last % page].reshape(-1), new[-1, 40 * 128:])


def test_reruns_are_bit_identical(ops):
    for q_lens, kv_lens in (([1] * 9, [5000, 3, 900, 64, 1, 777, 2048, 31, 4000]), ([300, 20], [3000, 2900])):
        b = ref.Batch(q_lens, kv_lens, 32, 8, 128, 16, BF16, seed=13)
        one = paged(ops, b)
        for _ in range(3):
            assert torch.equal(one, paged(ops, b))


@pytest.mark.parametrize("nqh,nkv", [(66, 2), (10, 2), (71, 1)])
def test_reruns_with_groups_that_leave_rows_unused(ops, nqh, nkv):
    """A group that does not divide a tile of rows leaves rows of it unused, whose shared memory holds anything."""
    nqh -= nqh % nkv + (7 if nqh == 71 else 0)
    b = ref.Batch([40 - i % 40 for i in range(130)], [300 - i for i in range(130)], nqh, nkv, 96, 256, BF16, seed=16)
    one = check(ops, b)
    for hd in (64, 128, 96):  # other kernels leave other contents behind
        paged(ops, ref.Batch([100], [700], 8, 2, hd, 16, F16, seed=hd, values=1e4))
        assert torch.equal(one, paged(ops, b))


def test_a_sequence_does_not_depend_on_its_neighbours_values(ops):
    b = ref.Batch([40, 40, 1], [200, 300, 90], 8, 2, 128, 16, F16, seed=14)
    one = paged(ops, b)
    for pg in b.table[1].tolist():
        if pg >= 0:
            b.v[pg], b.k[pg] = float("nan"), float("inf")
    two = paged(ops, b)
    ops.check_launch()
    assert torch.equal(one[:40], two[:40]) and torch.equal(one[80:], two[80:])


def test_bad_pages_and_lengths_are_reported(ops):
    b = ref.Batch([1, 30], [100, 90], 8, 2, 128, 16, F16, seed=15, poison=False)
    good = paged(ops, b)
    for bad in (-1, b.n_pages, 1 << 30):
        table = b.table.clone()
        b.table[0, 3] = bad
        out = paged(ops, b)
        with pytest.raises(RuntimeError, match="status 6"):
            ops.check_launch()
        assert torch.equal(out[1:], good[1:]), "the other sequence"
        qkv = torch.randn(31, 12 * 128, device="cuda")
        b.kv_len[0] = 50  # the new token's slot is in the bad page
        k, v = b.k.clone(), b.v.clone()
        ops.gpu_rope_kv_append_paged_into(qkv, torch.empty_like(b.q), b.k, b.v, b.table, b.cu, b.kv_len, 8, 1e4)
        with pytest.raises(RuntimeError, match="status 6"):
            ops.check_launch()
        touched = (b.k != k).flatten(1).any(dim=1).nonzero().flatten().tolist()
        assert set(touched) <= set(table[1].tolist())
        b.k.copy_(k), b.v.copy_(v)
        b.kv_len[0] = 100
        b.table.copy_(table)
    for name, t, i, x in (("kv_len", b.kv_len, 0, 1 << 20), ("kv_len", b.kv_len, 1, -5), ("cu_q", b.cu, 2, 1 << 20), ("cu_q", b.cu, 1, -3)):
        old = int(t[i])
        t[i] = x
        paged(ops, b)
        with pytest.raises(RuntimeError, match="status 7"):
            ops.check_launch()
        t[i] = old
    assert torch.equal(paged(ops, b), good)
    ops.check_launch()


# ---- whole prompts ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,nqh,nkv", [(128, 32, 8), (64, 14, 2), (96, 6, 2), (256, 4, 2), (32, 4, 4), (128, 3, 3), (64, 71, 71), (128, 48, 1)])
@pytest.mark.parametrize("lens", [[1], [0, 5, 0], [64, 1, 127, 128, 129, 0, 2], [700, 33]])
def test_packed_prompts(ops, dtype, hd, nqh, nkv, lens):
    g = torch.Generator(device="cuda").manual_seed(sum(lens) + hd)
    total = sum(lens) + 2
    qkv = torch.randn(total, (nqh + 2 * nkv) * hd, device="cuda", generator=g).to(dtype)
    qkv[sum(lens):] = float("nan")  # rows of no sequence
    b = pack(qkv, lens, nqh, nkv, hd, dtype)
    for window in (0, 40):
        out = packed(ops, b, qkv, window)
        ops.check_launch()
        want, tol = ref.expect(b, hd ** -0.5, window, dtype)
        ref.near(out, want, tol, f"window {window}")
        assert (out[sum(lens):] == 77.0).all()


def pack(qkv, lens, nqh, nkv, hd, dtype):
    b = ref.Batch(lens, [0] * len(lens), nqh, nkv, hd, 16, dtype, spare_rows=qkv.shape[0] - sum(lens))
    b.q = qkv[:, :nqh * hd]
    b.keys = [qkv[b.rows(s), nqh * hd:(nqh + nkv) * hd].reshape(-1, nkv, hd) for s in range(len(lens))]
    b.vals = [qkv[b.rows(s), (nqh + nkv) * hd:].reshape(-1, nkv, hd) for s in range(len(lens))]
    return b


def packed(ops, b, qkv, window=0, out_dtype=None):
    out = torch.full((b.total, b.nqh * b.hd), 77.0, dtype=out_dtype or b.dtype, device="cuda")
    n, m = b.nqh * b.hd, b.nkv * b.hd
    ops.gpu_gqa_attn_packed_into(b.q, qkv[:, n:n + m], qkv[:, n + m:], b.cu, out, b.nqh, b.nkv, b.hd, b.max_q, b.hd ** -0.5, window=window)
    return out


def test_packed_prompts_of_many_lengths(ops):
    lens = [(i * 29) % 90 for i in range(300)]
    qkv = torch.randn(sum(lens), 12 * 64, device="cuda").half()
    b = pack(qkv, lens, 8, 2, 64, F16)
    out = packed(ops, b, qkv)
    ops.check_launch()
    ref.near(out, *ref.expect(b, 64 ** -0.5, 0, F16))


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_packed_values_that_are_not_finite(ops, hd):
    """In one sequence: neither the other sequences nor its own earlier rows see them."""
    lens = [100, 150, 60]
    qkv = torch.randn(310, 12 * hd, device="cuda").bfloat16()
    b = pack(qkv, lens, 8, 2, hd, BF16)
    clean = packed(ops, b, qkv)
    qkv[190, 8 * hd:] = float("nan")
    out = packed(ops, b, qkv)
    ops.check_launch()
    want, tol = ref.expect(pack(qkv.nan_to_num(0.0), lens, 8, 2, hd, BF16), hd ** -0.5, 0, BF16)
    sees = torch.zeros(310, dtype=torch.bool, device="cuda")
    sees[190:250] = True
    assert torch.isnan(out[sees]).all()
    ref.near(out[~sees], want[~sees], tol[~sees])
    assert torch.equal(out[:100], clean[:100]) and torch.equal(out[250:], clean[250:])


# ---- the cache is filled ---------------------------------------------------------------------------------------------
def append(ops, qkv, b, theta=1e4, rot=None):
    q_out = torch.full((b.total, b.nqh * b.hd), 77.0, dtype=b.dtype, device="cuda")
    ops.gpu_rope_kv_append_paged_into(qkv, q_out, b.k, b.v, b.table, b.cu, b.kv_len, b.nqh, theta, rotary_dim=rot)
    return q_out


def check_append(ops, b, qkv, theta=1e4, rot=None):
    """A rotation is two products and a sum in f32 of a sine and a cosine off by at most 2^-22 (f32 function and the rounding of
    its reduced argument, which is at most pi: 2^-23), then one rounding."""
    k0, v0 = b.k.clone(), b.v.clone()
    q_out = append(ops, qkv, b, theta, rot)
    ops.check_launch()
    rot = b.hd if rot is None else rot
    x = qkv.reshape(b.total, b.nqh + 2 * b.nkv, b.hd)
    new = torch.zeros(b.n_pages, b.page, dtype=torch.bool, device="cuda")
    for s, (n, t) in enumerate(zip(b.q_lens, b.kv_lens)):
        if n == 0:
            continue
        pos = torch.arange(t - n, t, device="cuda")
        y = x[b.rows(s)]
        want = ref.rotate(y[:, :b.nqh + b.nkv], pos, rot, theta)
        size = torch.zeros_like(want)  # |a| + |b| of a pair
        size[..., :rot // 2] = size[..., rot // 2:rot] = y[:, :b.nqh + b.nkv, :rot // 2].double().abs() + y[:, :b.nqh + b.nkv, rot // 2:rot].double().abs()
        tol = size * 2.0 ** -20
        tol += ref.HALF[b.dtype] * (want.abs() + tol) + (2.0 ** -25 if b.dtype == F16 else 0.0)
        ref.near(q_out[b.rows(s)], want[:, :b.nqh].reshape(n, -1), tol[:, :b.nqh].reshape(n, -1), "q")
        fits = pos >= 0
        pos, y, want, tol = pos[fits], y[fits], want[fits], tol[fits]
        pages = b.table[s].long()[pos // b.page]
        ref.near(b.k[pages, pos % b.page], want[:, b.nqh:], tol[:, b.nqh:], "k")
        assert torch.equal(b.v[pages, pos % b.page], y[:, b.nqh + b.nkv:].to(b.dtype)), "v"
        new[pages, pos % b.page] = True
    same = lambda a, c: torch.equal(a[~new].view(torch.int16), c[~new].view(torch.int16))  # noqa: E731
    assert same(b.k, k0) and same(b.v, v0), "other slots are left as they were"
    assert (q_out[sum(b.q_lens):] == 77.0).all(), "rows behind the last sequence"


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("inp", [F32, F16, BF16])
@pytest.mark.parametrize("hd,rot,nqh,nkv,page", [(128, 128, 32, 8, 16), (96, 64, 12, 4, 24), (64, 64, 3, 1, 8), (256, 256, 4, 2, 80), (32, 0, 5, 5, 7),
                                                 (128, 36, 8, 2, 16), (80, 80, 4, 2, 3)])
def test_append(ops, dtype, inp, hd, rot, nqh, nkv, page):
    b = ref.Batch([1, 0, 70, 3, 1], [40, 5, 70, 100, 1], nqh, nkv, hd, page, dtype, seed=hd + rot, spare_rows=2)
    check_append(ops, b, torch.randn(b.total, (nqh + 2 * nkv) * hd, device="cuda").to(inp), rot=rot)


def test_append_to_many_sequences_and_far_positions(ops):
    b = ref.Batch([1] * 600, [i % 50 + 1 for i in range(600)], 4, 2, 64, 16, F16, seed=1)
    check_append(ops, b, torch.randn(600, 8 * 64, device="cuda"))
    b = ref.Batch([2000, 5], [131072, 100003], 4, 1, 64, 256, BF16, seed=2, poison=False)
    check_append(ops, b, torch.randn(b.total, 6 * 64, device="cuda"), theta=5e5)


def test_append_strided_rows_and_negative_positions(ops):
    b = ref.Batch([4, 9], [2, 30], 4, 2, 64, 16, F16, seed=3)
    wide = torch.randn(13, 8 * 64 + 24, device="cuda")
    check_append(ops, b, wide[:, 8:8 + 8 * 64])


# ---- together --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,nqh,nkv,page", [(128, 8, 2, 16), (64, 6, 2, 24), (256, 4, 4, 32)])
def test_serving_run(ops, dtype, hd, nqh, nkv, page):
    """Three sequences fed in pieces and token by token through the cache: every row as in one packed call over the whole
    prompts, whose keys were rotated the same way."""
    lens = [190, 75, 33]
    cuts = [[100, 1, 1, 60, 28], [64, 0, 9, 1, 1], [0, 31, 0, 1, 1]]
    x = [torch.randn(n, (nqh + 2 * nkv) * hd, device="cuda") for n in lens]
    b = ref.Batch([1, 1, 1], lens, nqh, nkv, hd, page, dtype, seed=7)
    b.k.fill_(float("nan")), b.v.fill_(float("nan"))
    scratch = ops.gpu_gqa_attn_paged_scratch(b.q, b.k, b.kv_len, nqh, 100, max(lens))
    got, done = [[] for _ in lens], [0, 0, 0]
    for step in range(5):
        n = [c[step] for c in cuts]
        rows = torch.cat([x[s][done[s]:done[s] + n[s]] for s in range(3)])
        done = [d + m for d, m in zip(done, n)]
        cu = torch.tensor([0, n[0], n[0] + n[1], sum(n)], dtype=torch.int32, device="cuda")
        kv = torch.tensor(done, dtype=torch.int32, device="cuda")
        q = torch.empty(sum(n), nqh * hd, dtype=dtype, device="cuda")
        out = torch.empty(sum(n), nqh * hd, dtype=dtype, device="cuda")
        ops.gpu_rope_kv_append_paged_into(rows, q, b.k, b.v, b.table, cu, kv, nqh, 1e4)
        ops.gpu_gqa_attn_paged_into(q, b.k, b.v, b.table, cu, kv, out, nqh, max(n), max(lens), hd ** -0.5, scratch=scratch)
        for s in range(3):
            got[s].append(out[int(cu[s]):int(cu[s + 1])])
    ops.check_launch()
    assert done == lens
    # the whole prompts, rotated by the same operator into a packed batch
    whole = torch.cat(x)
    cu = torch.tensor([0, lens[0], lens[0] + lens[1], sum(lens)], dtype=torch.int32, device="cuda")
    kv = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = torch.empty(sum(lens), nqh * hd, dtype=dtype, device="cuda")
    k2, v2 = torch.zeros_like(b.k), torch.zeros_like(b.v)
    ops.gpu_rope_kv_append_paged_into(whole, q, k2, v2, b.table, cu, kv, nqh, 1e4)
    ks, vs = [], []
    for s, n in enumerate(lens):
        pos = torch.arange(n, device="cuda")
        at = b.table[s].long()[pos // page]
        assert torch.equal(b.k[at, pos % page], k2[at, pos % page]) and torch.equal(b.v[at, pos % page], v2[at, pos % page])
        ks.append(k2[at, pos % page]), vs.append(v2[at, pos % page])
    out = torch.empty_like(q)
    ops.gpu_gqa_attn_packed_into(q, torch.cat(ks).view(-1, nkv * hd), torch.cat(vs).view(-1, nkv * hd), cu, out, nqh, nkv, hd, max(lens), hd ** -0.5)
    ops.check_launch()
    for s, n in enumerate(lens):
        a = int(cu[s])
        want, tol = ref.attention(q[a:a + n].view(n, nqh, hd), ks[s], vs[s], hd ** -0.5, 0, dtype, dtype)
        ref.near(torch.cat(got[s]), want.view(n, -1), tol.view(n, -1), "through the cache")
        ref.near(out[a:a + n], want.view(n, -1), tol.view(n, -1), "packed")


def test_captured_steps_follow_the_lengths(ops):
    """A decode step captured once and replayed while the sequences grow; two graphs on one workspace, replayed in turn."""
    nqh, nkv, hd, page, n = 8, 2, 128, 16, 4
    b = ref.Batch([1] * n, [200] * n, nqh, nkv, hd, page, F16, seed=21, poison=False)
    scratch = ops.gpu_gqa_attn_paged_scratch(b.q, b.k, b.kv_len, nqh, 1, 200)
    qkv = torch.empty(n, (nqh + 2 * nkv) * hd, device="cuda")
    q = torch.empty(n, nqh * hd, dtype=F16, device="cuda")
    out = torch.empty(n, nqh * hd, dtype=F16, device="cuda")
    kv_len = torch.tensor([150, 3, 64, 127], dtype=torch.int32, device="cuda")

    def step():
        kv_len.add_(1)
        ops.gpu_rope_kv_append_paged_into(qkv, q, b.k, b.v, b.table, b.cu, kv_len, nqh, 1e4)
        ops.gpu_gqa_attn_paged_into(q, b.k, b.v, b.table, b.cu, kv_len, out, nqh, 1, 200, hd ** -0.5, scratch=scratch)

    start, k0, v0 = kv_len.clone(), b.k.clone(), b.v.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for g in graphs:
        with torch.cuda.graph(g):
            step()
    xs = [torch.randn_like(qkv) for _ in range(6)]
    kv_len.copy_(start), b.k.copy_(k0), b.v.copy_(v0)
    eager = []
    for x in xs:
        qkv.copy_(x)
        step()
        eager.append(out.clone())
    kv_len.copy_(start), b.k.copy_(k0), b.v.copy_(v0)
    for i, x in enumerate(xs):
        qkv.copy_(x)
        graphs[i % 2].replay()
        assert torch.equal(out, eager[i]), f"step {i}"
    ops.check_launch()


def test_another_stream(ops):
    b = ref.Batch([1, 200], [3000, 900], 8, 2, 128, 16, F16, seed=22)
    want = paged(ops, b)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = paged(ops, b)
    side.synchronize()
    assert torch.equal(got, want)


def test_python_refusals(ops):
    b = ref.Batch([1, 2], [9, 30], 8, 2, 64, 16, F16, seed=23, poison=False)
    out = torch.empty_like(b.q)
    call = lambda **kw: ops.gpu_gqa_attn_paged_into(**{**dict(q=b.q, kpages=b.k, vpages=b.v, page_table=b.table, cu_q=b.cu, kv_len=b.kv_len, out=out,  # noqa: E731
                                                             nqh=8, max_q=2, max_kv=30), **kw})
    call()
    for kw in (dict(q=b.q.float()), dict(out=out.double()), dict(vpages=b.v.bfloat16())):
        with pytest.raises(TypeError):
            call(**kw)
    for kw in (dict(q=b.q.cpu()), dict(q=b.q[:, :-1]), dict(out=out[:-1]), dict(cu_q=b.cu.long()), dict(cu_q=b.cu[:-1]), dict(page_table=b.table[:1]),
               dict(kpages=b.k[:, :, :1]), dict(kpages=b.k.transpose(1, 2), vpages=b.v.transpose(1, 2)), dict(page_table=b.table.cpu())):
        with pytest.raises(ValueError):
            call(**kw)
    from nates_recipe_rs_b200._lib import QmmError
    for kw in (dict(kq_scale=0.0), dict(window=-1), dict(scratch=torch.empty(64, dtype=torch.uint8, device="cuda")), dict(out=b.q)):
        with pytest.raises(QmmError):
            call(**kw)
    with pytest.raises(TypeError):
        ops.gpu_gqa_attn_packed_into(b.q, b.q[:, :128].float(), b.q[:, :128], b.cu, out, 8, 2, 64, 2)
    with pytest.raises(TypeError):
        ops.gpu_rope_kv_append_paged_into(torch.zeros(3, 12 * 64, device="cuda"), out.bfloat16(), b.k, b.v, b.table, b.cu, b.kv_len, 8, 1e4)
    ops.check_launch()
