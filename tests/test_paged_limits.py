"""The ends of the argument ranges of the paged-cache operators, refused on the host: nothing is launched, no GPU needed."""
import pytest

from nates_recipe_rs_b200._lib import lib
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


@pytest.mark.parametrize("hd", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("nqh,nkv", [(8, 2), (64, 1), (4, 4), (17, 1)])
def test_a_workspace_for_more_tokens_serves_fewer(hd, nqh, nkv):
    sizes = [lib().qmm_attn_paged_scratch_bytes(n, nqh, nkv, hd) for n in (0, 1, 2, 4, 16, 17, 1000, 1 << 20)]
    assert sizes[0] > 0 and sizes == sorted(sizes)
