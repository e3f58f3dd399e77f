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
