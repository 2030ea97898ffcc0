"""Sizes at the limits of the products with 4-bit weights: a plan that is selected can
be run (no GPU)."""
import pytest

from baracuda_amd import ffi, w4
from baracuda_amd.plans import Unsupported


def _moe(experts, topk, pairs, n, k):
    return w4.MoeW4GroupedPlan.select(w4.MoeW4GroupedDescriptor(experts, topk, pairs, n, k))


# rows of x times K at and past 2^30
@pytest.mark.parametrize("experts,topk,pairs,k", [(8, 1, 2 ** 20, 4096), (8, 1, 2 ** 18, 4096), (8, 2, 2 ** 19, 4096),
                                                  (8, 8, 2 ** 20, 8192), (8, 2, 2 ** 18 + 1, 8192), (4, 3, 2 ** 20, 4096)])
def test_select_refuses_x_past_31_bits(experts, topk, pairs, k):
    with pytest.raises(Unsupported):
        _moe(experts, topk, pairs, 64, k)


@pytest.mark.parametrize("experts,topk,pairs,k", [(8, 1, 2 ** 18 - 1, 4096), (8, 2, 2 ** 19 - 2, 4096), (8, 8, 2 ** 20, 4096),
                                                  (8, 2, 2 ** 18 - 3, 8192), (4, 3, 2 ** 20, 2880), (4, 4, 0, 4096)])
def test_select_takes_x_of_31_bits(experts, topk, pairs, k):
    _moe(experts, topk, pairs, 64, k)


def test_run_refuses_the_rows_that_weights_ask_for():
    """Before any launch: x has a row for each pair where router weights are given."""
    L, p = ffi.lib(), 1 << 20     # an aligned address that nothing reads
    assert L.moe_w4_grouped_gfx950_can_implement(8, 8, 2 ** 18, 64, 4096, 2, 0) == 0
    assert L.moe_w4_grouped_gfx950_run(8, 8, 2 ** 18, 64, 4096, 2, 0, p, p, p, p, p, None, p, p, p, None, 0, None) == 3
