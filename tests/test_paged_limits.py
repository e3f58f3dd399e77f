"""The ends of the argument ranges of the paged-cache operators, refused on the host: nothing is launched, no GPU needed."""
import pytest

from test_paged_args import append, attn, packed, pool


@pytest.mark.parametrize("nqh,nkv", [(8, 1 << 30), (8, (1 << 31) - 1), ((1 << 31) - 1, 2), ((1 << 31) - 8, 1 << 30)])
def test_numbers_of_heads_whose_sum_passes_32_bits(nqh, nkv):
    assert append(pool(n_kv_heads=nkv), nqh=nqh) == -2
    assert append(pool(n_kv_heads=nkv), nqh=nqh, stride=1 << 50) == -3


@pytest.mark.parametrize("scale", [2.4e38, 3.4e38])
def test_scales_whose_product_with_log2_e_overflows(scale):
    """exp(x) is computed as exp2(x log2(e)): the factor has to be finite too."""
    assert attn(scale=scale) == -2 and packed(scale=scale) == -2
    assert attn(scale=2.3e38) == 0 and packed(scale=2.3e38) == 0 and attn(scale=1e-45) == 0
