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
