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


@pytest.mark.parametrize("m,gated", [(1, False), (17, False), (17, True)])
def test_scales_past_31_bits(gpu, m, gated):
    """More than 2^31 bytes of scales: weights are zero but in a few blocks of 32 rows, the
    first and last of them and those where the scales pass 2^31."""
    n, k, g = 16646592, 4128, _gen(m)
    blocks, codes_of, scales_of = n // 32, -(-k // 128) * 2048, -(-k // 256) * 256
    assert blocks * scales_of > 2 ** 31 and n * k <= 2 ** 36
    edge = 2 ** 31 // scales_of
    some = [0, 1, blocks // 2 - 1, blocks // 2, blocks // 2 + 1, edge - 1, edge, edge + 1, blocks - 2, blocks - 1]
    codes, scales = plain.checkpoint(g, 1, 32 * len(some), k)
    part = _packed(codes, scales)[0]
    packed = torch.zeros(w4.packed_bytes(n, k), dtype=torch.uint8, device=gpu)
    c, s = packed[:blocks * codes_of].view(blocks, -1), packed[blocks * codes_of:].view(blocks, -1)
    at = torch.tensor(some, device=gpu)
    c[at], s[at] = part[:len(some) * codes_of].view(len(some), -1), part[len(some) * codes_of:].view(len(some), -1)
    x = _randn(g, m, k).to(BF)
    out = torch.full((m, n // 2 if gated else n), 3.0, dtype=BF, device=gpu)
    w4.W4LinearPlan.select(w4.W4LinearDescriptor(m, n, k, gated=gated)).run(x, packed, out)
    w = dict(zip(some, plain.values(codes, scales)[0].view(len(some), 32, k)))
    none = torch.zeros(32, k, dtype=torch.float64, device=gpu)
    half = blocks // 2
    for b in sorted({b % half if gated else b for b in some} | {5, half - 3}):
        rows = torch.cat((w.get(b, none), w.get(b + half, none))) if gated else w.get(b, none)
        ok, why = plain.close(out[:, 32 * b:32 * b + 32], *plain.product(x, rows, None, gated))
        assert ok, (b, why)
    written = torch.zeros(out.shape[1] // 32, dtype=torch.bool, device=gpu)
    written[torch.tensor([b % half if gated else b for b in some], device=gpu)] = True
    assert not bool(out.view(m, -1, 32)[:, ~written].any())


@pytest.mark.parametrize("dtype", [BF, F16], ids=str)
@pytest.mark.parametrize("m", [1, 3, 16, 20, 90, 300])
def test_every_scale_rounds_to_the_element(gpu, dtype, m):
    """Scales beyond those with which weights are elements, one of 256 a row: a weight enters
    as its value rounded to the element, infinite past its range.  x is one power of two
    and zeros, so that each result is one product, rounded once."""
    n, k, g = 256, 32, _gen(m)
    some = torch.randint(0, 256, (1, n, k // 2), generator=g, device=gpu, dtype=torch.uint8)
    scales = torch.arange(256, device=gpu).to(torch.uint8).view(1, n, 1).contiguous()
    plan = w4.W4LinearPlan.select(w4.W4LinearDescriptor(m, n, k, element=KIND[dtype]))
    for power in (-14, 0, 12) if dtype == F16 else (-40, 0, 20):
        for at in (0, 7, 31):
            codes = torch.zeros_like(some)                  # no zero of x meets an infinity
            codes[..., at // 2] = some[..., at // 2] & (0xf0 if at % 2 else 0x0f)
            x = torch.zeros(m, k, dtype=dtype, device=gpu)
            x[:, at] = 2.0 ** power
            out = torch.zeros(m, n, dtype=dtype, device=gpu)
            plan.run(x, _packed(codes, scales), out)
            w = plain.values(codes, scales)[0, :, at].to(dtype).double()
            want = (w * 2.0 ** power).to(dtype).expand(m, n)
            assert bool(((out == want) | (out.isnan() & want.isnan())).all()), (power, at)
