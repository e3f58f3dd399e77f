"""The ends of the argument ranges of the paged-cache operators, refused on the host: nothing is launched, no GPU needed."""
import pytest

from test_paged_args import append, attn, packed, pool


@pytest.mark.parametrize("nqh,nkv", [(8, 1 << 30), (8, (1 << 31) - 1), ((1 << 31) - 1, 2), ((1 << 31) - 8, 1 << 30)])
def test_numbers_of_heads_whose_sum_passes_32_bits(nqh, nkv):
    assert append(pool(n_kv_heads=nkv), nqh=nqh) == -2
    assert append(pool(n_kv_heads=nkv), nqh=nqh, stride=1 << 50) == -3
