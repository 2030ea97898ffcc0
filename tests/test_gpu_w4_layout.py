"""The packed bytes of 4-bit weights as the products read them, beyond what a plan packs."""
import pytest
import torch

from baracuda_amd import w4
from tests import w4_plain as plain
from tests.test_gpu_w4 import BF, F16, KIND, _gen, _packed, _randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, F16], ids=str)
@pytest.mark.parametrize("m", [1, 3, 8, 16, 33, 300])
@pytest.mark.parametrize("n,k", [(50, 32), (33, 96), (70, 160), (64, 352)])
def test_padding_scales_of_zero(gpu, dtype, m, n, k):
    """Bytes 0 for the scales past N and K in place of 2: the same results."""
    g = _gen(m + n)
    codes, scales = plain.checkpoint(g, 1, n, k)
    held = _packed(codes, scales)
    real = plain.packed(torch.full_like(codes, 0xff), torch.full_like(scales, 7)) != plain.packed(
        torch.zeros_like(codes), torch.full_like(scales, 9))          # what is no padding
    zeros = torch.where(real, held, 0)
    assert bool((held[~real] != 0).any())
    x = _randn(g, m, k).to(dtype)
    plan = w4.W4LinearPlan.select(w4.W4LinearDescriptor(m, n, k, element=KIND[dtype]))
    outs = [torch.empty(m, n, dtype=dtype, device=gpu) for _ in range(2)]
    plan.run(x, held, outs[0])
    plan.run(x, zeros, outs[1])
    assert torch.equal(*outs)
    ok, why = plain.close(outs[1], *plain.product(x, plain.values(codes, scales)[0]))
    assert ok, why
