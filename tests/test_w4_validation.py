"""What the plans and C entries of the products with 4-bit weights refuse, before any launch (no GPU)."""
import pytest
import torch

from baracuda_amd import ffi, w4
from baracuda_amd.plans import ElementKind, InvalidProblem, Misaligned, Unsupported
from tests import w4_plain as plain

BF = torch.bfloat16
U8 = torch.uint8


def _weights(**kw):
    return w4.W4WeightsDescriptor(**{**dict(n=40, k=64, matrices=2), **kw})


@pytest.mark.parametrize("error,kw", [
    (InvalidProblem, dict(n=0)), (InvalidProblem, dict(k=0)), (InvalidProblem, dict(matrices=-1)), (InvalidProblem, dict(n=-5)),
    (Unsupported, dict(k=48)), (Unsupported, dict(k=1)), (Unsupported, dict(element=ElementKind.F64)), (Unsupported, dict(n=2 ** 31)),
    (Unsupported, dict(n=2 ** 31 - 1)), (Unsupported, dict(k=2 ** 31 - 32)), (Unsupported, dict(matrices=2 ** 31 - 1))], ids=str)
def test_weights_descriptors(error, kw):
    with pytest.raises(error):
        w4.W4WeightsPlan.select(_weights(**kw))


def _linear(**kw):
    return w4.W4LinearDescriptor(**{**dict(m=3, n=64, k=64), **kw})


@pytest.mark.parametrize("error,kw", [
    (InvalidProblem, dict(m=-1)), (InvalidProblem, dict(n=0)), (InvalidProblem, dict(k=0)), (Unsupported, dict(k=40)),
    (Unsupported, dict(element=ElementKind.F32)), (Unsupported, dict(element=ElementKind.S8)), (Unsupported, dict(gated=True, n=96)),
    (Unsupported, dict(m=2 ** 31)), (Unsupported, dict(m=2 ** 21)), (Unsupported, dict(n=2 ** 30)), (Unsupported, dict(k=2 ** 30))],
    ids=str)
def test_linear_descriptors(error, kw):
    with pytest.raises(error):
        w4.W4LinearPlan.select(_linear(**kw))


def _moe(**kw):
    return w4.MoeW4GroupedDescriptor(**{**dict(num_experts=4, topk=2, size_m=6, n=64, k=64), **kw})


@pytest.mark.parametrize("error,kw", [
    (InvalidProblem, dict(num_experts=0)), (InvalidProblem, dict(topk=0)), (InvalidProblem, dict(topk=5)),
    (InvalidProblem, dict(size_m=-1)), (InvalidProblem, dict(n=0)), (Unsupported, dict(num_experts=1025)),
    (Unsupported, dict(size_m=2 ** 21)), (Unsupported, dict(k=33)), (Unsupported, dict(gated=True, n=32)),
    (Unsupported, dict(element=ElementKind.F32))], ids=str)
def test_moe_descriptors(error, kw):
    with pytest.raises(error):
        w4.MoeW4GroupedPlan.select(_moe(**kw))


def _refused(run, good, bad):
    for name, values in bad.items():
        for v in values:
            with pytest.raises(InvalidProblem):
                run(**{**good, name: v})
    with pytest.raises(InvalidProblem, match="GPU"):
        run(**good)


def test_weights_operands():
    plan = w4.W4WeightsPlan.select(_weights())
    size = w4.packed_bytes(40, 64)
    packed = [None, torch.zeros(2, size + 1, dtype=U8), torch.zeros(size, dtype=U8), torch.zeros(2, size), torch.zeros(2, 2 * size, dtype=U8)[:, ::2]]
    weights = [None, torch.zeros(2, 40, 64), torch.zeros(1, 40, 64, dtype=BF), torch.zeros(40, 64, dtype=BF), torch.zeros(64, dtype=BF),
               torch.zeros(2, 40, 128, dtype=BF)[..., ::2], "weights"]
    good = dict(weights=torch.zeros(2, 40, 64, dtype=BF), packed=torch.zeros(2, size, dtype=U8), stream=0)
    _refused(plan.quantize, good, dict(weights=weights, packed=packed))
    _refused(plan.read, good, dict(weights=weights, packed=packed))
    good = dict(codes=torch.zeros(2, 40, 32, dtype=U8), scales=torch.zeros(2, 40, 2, dtype=U8), packed=torch.zeros(2, size, dtype=U8), stream=0)
    _refused(plan.pack, good, dict(codes=[None, torch.zeros(2, 40, 33, dtype=U8), torch.zeros(2, 40, 32, dtype=torch.int8), torch.zeros(0, dtype=U8)],
                                   scales=[None, torch.zeros(2, 40, 3, dtype=U8), torch.zeros(2, 40, 4, dtype=U8)[..., ::2]], packed=packed))


def test_linear_operands():
    plan = w4.W4LinearPlan.select(_linear())
    good = dict(x=torch.zeros(3, 64, dtype=BF), packed=torch.zeros(w4.packed_bytes(64, 64), dtype=U8), out=torch.zeros(3, 64, dtype=BF),
                bias=torch.zeros(64), stream=0)
    _refused(plan.run, good, dict(
        x=[None, torch.zeros(3, 64), torch.zeros(2, 64, dtype=BF), torch.zeros(3, 96, dtype=BF), torch.zeros(3, 128, dtype=BF)[:, ::2],
           torch.zeros(64, dtype=BF)],
        packed=[None, torch.zeros(64, 64, dtype=U8)], bias=[torch.zeros(63), torch.zeros(64, dtype=BF), torch.zeros(1, 64)],
        out=[None, torch.zeros(3, 32, dtype=BF), torch.zeros(3, 64), torch.zeros(64, 3, dtype=BF).t()],
        workspace=[torch.zeros(8, 2, dtype=U8)[:, 0], 5]))
    gated = w4.W4LinearPlan.select(_linear(gated=True))
    with pytest.raises(InvalidProblem, match="out"):
        gated.run(**good)


def test_moe_operands():
    plan = w4.MoeW4GroupedPlan.select(_moe())
    i32 = dict(dtype=torch.int32)
    good = dict(x=torch.zeros(3, 64, dtype=BF), packed=torch.zeros(4, w4.packed_bytes(64, 64), dtype=U8), sorted_token_ids=torch.zeros(6, **i32),
                expert_ids=torch.zeros(6, **i32), out=torch.zeros(6, 64, dtype=BF), expert_counts=torch.zeros(4, **i32),
                expert_offsets=torch.zeros(5, **i32), stream=0)
    _refused(plan.run, good, dict(
        x=[None, torch.zeros(6, 64, dtype=BF), torch.zeros(3, 128, dtype=BF)[:, :64]], packed=[torch.zeros(w4.packed_bytes(64, 64), dtype=U8)],
        sorted_token_ids=[None, torch.zeros(6, dtype=torch.int64), torch.zeros(5, **i32)], expert_ids=[None, torch.zeros(12, **i32)[::2]],
        out=[torch.zeros(3, 64, dtype=BF), torch.zeros(6, 128, dtype=BF)[:, :64]], expert_counts=[None, torch.zeros(5, **i32)],
        expert_offsets=[None, torch.zeros(4, **i32)], bias=[torch.zeros(64), torch.zeros(4, 32)],
        topk_weights=[torch.zeros(6), torch.zeros(3)]))      # with weights x has a row for each pair


def test_c_entries_refuse():
    L = ffi.lib()
    p = 1 << 20     # an aligned address; nothing is launched with what follows
    run = L.w4_linear_gfx950_run
    good = dict(m=2, n=64, k=64, element=2, gated=0, x=p, ldx=64, packed=p, bias=None, out=p, ldo=64, ws=None, nb=0, stream=None)

    def linear(**kw):
        return run(*{**good, **kw}.values())

    for kw, status in ((dict(x=None), 2), (dict(packed=None), 2), (dict(out=None), 2), (dict(x=p + 2), 1), (dict(packed=p + 8), 1),
                       (dict(ldx=68), 1), (dict(out=p + 1), 1), (dict(bias=p + 2), 1), (dict(ldo=63), 2), (dict(ldx=-64), 2), (dict(element=0), 3),
                       (dict(m=-1), 2), (dict(k=63), 3), (dict(gated=1, n=32), 3)):
        assert linear(**kw) == status, kw
    assert linear(m=0) == 0
    assert linear(ldx=2 ** 23) == 3 and linear(ldx=2 ** 40) == 3                # a tile of x past 31 bits
    assert L.w4_pack_gfx950_run(1, 32, 32, p, p, p + 4, None) == 1
    assert L.w4_pack_gfx950_run(1, 32, 32, None, p, p, None) == 2
    assert L.w4_pack_gfx950_run(0, 32, 32, None, None, None, None) == 0
    assert L.w4_read_gfx950_run(2, 32, 32, 2, p, p, 100, 32, None) == 2          # matrices that overlap
    assert L.w4_read_gfx950_run(1, 32, 32, 2, p, p, 0, 31, None) == 2
    assert L.w4_quantize_gfx950_run(1, 32, 32, 0, p + 2, 0, 32, p, None) == 1
    moe = L.moe_w4_grouped_gfx950_run
    assert moe(4, 2, 0, 64, 64, 2, 0, *(None,) * 9, None, 0, None) == 2          # nowhere to put the counts
    assert moe(4, 2, 4, 64, 64, 2, 0, p, p, p, None, None, None, p, p, p, None, 0, None) == 2
    assert moe(4, 2, 4, 64, 64, 2, 0, p + 2, p, p, p, None, None, p, p, p, None, 0, None) == 1
    assert moe(4, 1, 2 ** 20, 64, 4096, 2, 0, p, p, p, p, None, None, p, p, p, None, 0, None) == 3      # x past 31 bits


@pytest.mark.parametrize("n,k", [(1, 32), (32, 128), (33, 96), (64, 256), (100, 288), (4096, 4096)])
def test_packed_bytes(n, k):
    codes, scales = torch.zeros(1, n, k // 2, dtype=U8), torch.zeros(1, n, k // 32, dtype=U8)
    assert w4.packed_bytes(n, k) == plain.packed(codes, scales).shape[1]


def test_plain_quantizer():
    """The plain quantizer's codes stand for the nearest values."""
    g = torch.Generator().manual_seed(1)
    w = torch.randn(7, 96, generator=g)
    codes, scales = plain.quantized(w)
    v, s = plain.values(codes, scales), torch.exp2(scales.double() - 127).repeat_interleave(32, -1)
    assert float((w.abs() / s).max()) < 7 and bool(((w.unflatten(-1, (-1, 32)).abs().amax(-1) / torch.exp2(scales.double() - 127)) >= 3.5).all())
    levels = torch.tensor(plain.LEVELS, dtype=torch.float64)
    best = ((w.abs() / s)[..., None] - levels).abs().amin(-1)
    assert torch.equal((w.double() - v).abs(), best * s)
