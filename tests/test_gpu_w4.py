"""Products with 4-bit weights against plain forms in 64 bits."""
import pytest
import torch

from baracuda_amd import w4
from baracuda_amd.plans import ElementKind
from tests import w4_plain as plain

pytestmark = pytest.mark.gpu

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
KIND = {BF: ElementKind.Bf16, F16: ElementKind.F16, F32: ElementKind.F32}


def _gen(seed):
    return torch.Generator(device="cuda:0").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda:0")


def _packed(codes, scales):
    """By the plan, from codes [matrices, N, K / 2]."""
    e, n, half = codes.shape
    plan = w4.W4WeightsPlan.select(w4.W4WeightsDescriptor(n, 2 * half, e))
    out = torch.full((e, w4.packed_bytes(n, 2 * half)), 0xA5, dtype=torch.uint8, device=codes.device)
    plan.pack(codes, scales, out)
    return out


# ---- weights --------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, F16, F32], ids=str)
@pytest.mark.parametrize("matrices,n,k", [(1, 1, 32), (1, 33, 96), (3, 64, 128), (2, 31, 320), (1, 100, 1024), (2, 70, 4128)])
def test_quantize_and_read(gpu, dtype, matrices, n, k):
    g = _gen(n + k)
    w = (_randn(g, matrices, n, k) * torch.exp2(4 * _randn(g, matrices, n, 1))).to(dtype)
    flat = w.view(-1, 32)
    flat[0] = 0                                                     # an empty group
    steps = torch.tensor([0, .25, .5, .75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 6.5], device=gpu)
    flat[-1] = torch.cat((steps, -steps)).to(dtype)                 # ties, both signs
    if len(flat) > 8:
        flat[1] = torch.inf
        flat[2, 5] = torch.nan
        flat[3] = (steps.repeat(2) * 2.0 ** -24).to(dtype)          # the smallest halves
        flat[4] = torch.finfo(dtype).max
        flat[5, 0], flat[5, 1:] = 7, 0.874                          # the border between two scales
        flat[6, 0] = 6.996 if dtype == F32 else 6.97
        flat[7] = -0.0
    most = 13 if dtype == F16 else 125
    codes, scales = plain.quantized(w, most)
    desc = w4.W4WeightsDescriptor(n, k, matrices, element=KIND[dtype])
    plan = w4.W4WeightsPlan.select(desc)
    packed = torch.full((matrices, w4.packed_bytes(n, k)), 0x5A, dtype=torch.uint8, device=gpu)
    plan.quantize(w, packed)
    assert torch.equal(packed, plain.packed(codes, scales))
    out = torch.full((matrices, n + 2, k + 3), 7.0, dtype=dtype, device=gpu)
    plan.read(packed, out[:, 1:-1, 2:-1])                           # rows that are not dense, an odd start
    want = plain.values(codes, scales).to(dtype)
    assert torch.equal(out[:, 1:-1, 2:-1].nan_to_num(9e3), want.nan_to_num(9e3))
    out[:, 1:-1, 2:-1] = 7
    assert bool((out == 7).all())                                   # nothing around it was written
    # from rows that are not dense, matrices inside rows
    wide = torch.zeros(n, matrices, k + 5, dtype=dtype, device=gpu)
    wide[:, :, 3:-2] = w.transpose(0, 1)
    again = torch.zeros_like(packed)
    plan.quantize(wide[:, :, 3:-2].transpose(0, 1), again)
    assert torch.equal(again, packed)


@pytest.mark.parametrize("dtype", [BF, F16, F32], ids=str)
def test_pack_every_code_and_scale(gpu, dtype):
    n, k = 256, 512
    codes = torch.arange(256, dtype=torch.uint8, device=gpu).repeat(n, 1).view(1, n, k // 2).contiguous()
    scales = torch.arange(256, dtype=torch.uint8, device=gpu).view(1, n, 1).repeat(1, 1, k // 32).contiguous()
    packed = _packed(codes, scales)
    assert torch.equal(packed, plain.packed(codes, scales))
    out = torch.empty(1, n, k, dtype=dtype, device=gpu)
    w4.W4WeightsPlan.select(w4.W4WeightsDescriptor(n, k, element=KIND[dtype])).read(packed, out)
    want = plain.values(codes, scales)
    lo, hi = (2, 252) if dtype != F16 else (0, 254)                  # outside 2^-125 .. 2^125 nothing is promised
    assert torch.equal(out[:, lo:hi + 1], want[:, lo:hi + 1].to(dtype))
    assert bool(out[:, 255].isnan().all())


# ---- linear ----------------------------------------------------------------------
def _linear(m, n, k, dtype, gated, bias, seed, x=None, codes=None, scales=None):
    g = _gen(seed)
    if x is None:
        x = _randn(g, m, k).to(dtype)
    if codes is None:
        codes, scales = plain.checkpoint(g, 1, n, k)
    b = _randn(g, n) if bias else None
    plan = w4.W4LinearPlan.select(w4.W4LinearDescriptor(m, n, k, element=KIND[dtype], gated=gated))
    cols = n // 2 if gated else n
    out = torch.full((m, cols), 5.0, dtype=dtype, device="cuda:0")
    ws = torch.full((plan.workspace_size(),), 0xA5, dtype=torch.uint8, device="cuda:0")
    plan.run(x, _packed(codes, scales), out, bias=b, workspace=ws)
    want, error = plain.product(x, plain.values(codes, scales)[0], b, gated)
    return out, want, error


SIZES = [
    (1, 1, 32), (1, 17, 64), (1, 64, 96), (1, 4096, 4096), (1, 130, 14336), (1, 4097, 288), (2, 48, 160), (3, 1000, 352),
    (5, 96, 2880), (8, 515, 1024), (15, 33, 224), (16, 256, 256), (17, 64, 512), (31, 257, 1056), (32, 320, 2048), (33, 96, 416),
    (48, 1024, 1024), (63, 130, 96), (64, 512, 4096), (65, 192, 640), (100, 1027, 768), (128, 384, 128), (129, 160, 1184),
    (200, 448, 2048), (256, 512, 1024), (257, 300, 544), (300, 1500, 96), (511, 520, 1056), (777, 1031, 512), (1030, 640, 2080),
]


@pytest.mark.parametrize("dtype", [BF, F16], ids=str)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_linear(gpu, dtype, m, n, k):
    ok, why = plain.close(*_linear(m, n, k, dtype, False, (m + n) % 2 == 0, seed=m + n + k))
    assert ok, why


@pytest.mark.parametrize("dtype", [BF, F16], ids=str)
@pytest.mark.parametrize("m,n,k", [(1, 64, 32), (1, 8192, 4096), (2, 128, 96), (6, 320, 2880), (16, 192, 1024), (17, 576, 544),
                                   (40, 64, 4096), (64, 1024, 256), (65, 448, 320), (130, 512, 1024), (200, 192, 160),
                                   (256, 1024, 512), (300, 640, 2080), (520, 1088, 352)])
def test_linear_gated(gpu, dtype, m, n, k):
    ok, why = plain.close(*_linear(m, n, k, dtype, True, (m + n) % 3 == 0, seed=m + n + k))
    assert ok, why


@pytest.mark.parametrize("m", [1, 5, 40, 300])
def test_linear_strides(gpu, m):
    """Rows of x and of the output inside wider ones, an output of any alignment."""
    n, k, g = 99, 224, _gen(m)
    codes, scales = plain.checkpoint(g, 1, n, k)
    x = _randn(g, m, k + 24).to(BF)[:, 8:-16]
    out = torch.full((m + 2, n + 6), 3.0, dtype=BF, device=gpu)
    plan = w4.W4LinearPlan.select(w4.W4LinearDescriptor(m, n, k))
    plan.run(x, _packed(codes, scales)[0], out[1:-1, 5:-1])
    ok, why = plain.close(out[1:-1, 5:-1], *plain.product(x, plain.values(codes, scales)[0]))
    assert ok, why
    out[1:-1, 5:-1] = 3
    assert bool((out == 3).all())


@pytest.mark.parametrize("dtype,low,high", [(BF, 2 - 127, 100), (F16, -23, 13)], ids=["bf16", "f16"])
@pytest.mark.parametrize("m", [1, 20, 90, 300])
def test_linear_scales_of_any_size(gpu, dtype, low, high, m):
    """Every scale with which the weights are elements, one a row."""
    n, k, g = high - low + 1, 96, _gen(m)
    codes, _ = plain.checkpoint(g, 1, n, k)
    scales = (torch.arange(low, high + 1, device=gpu) + 127).to(torch.uint8).view(1, n, 1).repeat(1, 1, k // 32).contiguous()
    x = torch.randint(-8, 9, (m, k), generator=g, device=gpu).to(dtype) / (1024 if dtype == F16 else 1)
    out, want, error = _linear(m, n, k, dtype, False, False, m, x, codes, scales)
    ok, why = plain.close(out, want, error)
    assert ok, why


@pytest.mark.parametrize("m", [2, 33, 260])
@pytest.mark.parametrize("k", [96, 544])
def test_linear_infinities(gpu, m, k):
    """A NaN or an infinity in one row of x, or in a group of one row of the weights,
    reaches that row alone, whatever lies behind the last value of a row."""
    n, g = 70, _gen(m)
    codes, scales = plain.checkpoint(g, 1, n, k)
    codes[codes & 7 == 0] |= 1                                     # no zero times infinity
    codes[codes & 0x70 == 0] |= 0x10
    wide = torch.full((m, k + 64), torch.nan, device=gpu, dtype=BF)
    wide[:, :k] = _randn(g, m, k).to(BF)
    wide[0, 3], wide[m - 1, k - 1] = torch.nan, torch.inf
    scales[0, 5, -1] = 255
    out, want, error = _linear(m, n, k, BF, False, False, 0, wide[:, :k], codes, scales)
    assert bool(out[0].isnan().all()) and bool(out[:, 5].isnan().all())
    keep = torch.arange(n, device=gpu) != 5
    assert bool(torch.equal(out[m - 1, keep].double(), want[m - 1, keep]))
    ok, why = plain.close(out[1:-1, keep], want[1:-1, keep], error[1:-1, keep])
    assert ok, why


# ---- by expert ---------------------------------------------------------------------
def _pairs(counts, g, none=0, topk=1):
    """Positions sorted by expert with these counts, and `none` pairs of no expert."""
    ids = torch.repeat_interleave(torch.arange(len(counts), device="cuda:0"), torch.tensor(counts, device="cuda:0"))
    ids = torch.cat((ids, torch.full((none,), len(counts), device="cuda:0")))
    return torch.randperm(len(ids), generator=g, device="cuda:0").int(), ids.int()


def _grouped(counts, n, k, dtype, gated, topk, mix, bias, seed, none=0):
    g = _gen(seed)
    order, ids = _pairs(counts, g, none)
    e, p = len(counts), len(ids)
    codes, scales = plain.checkpoint(g, e, n, k)
    x = _randn(g, p if mix else -(-p // topk), k).to(dtype)
    b = _randn(g, e, n) if bias else None
    t = torch.rand(p, generator=g, device="cuda:0") if mix else None
    plan = w4.MoeW4GroupedPlan.select(w4.MoeW4GroupedDescriptor(e, topk, p, n, k, element=KIND[dtype], gated=gated))
    cols = n // 2 if gated else n
    out = torch.full((p, cols), 5.0, dtype=dtype, device="cuda:0")
    held, first = (torch.full((c,), -1, dtype=torch.int32, device="cuda:0") for c in (e, e + 1))
    ws = torch.full((plan.workspace_size(),), 0xA5, dtype=torch.uint8, device="cuda:0")
    plan.run(x, _packed(codes, scales), order, ids, out, held, first, bias=b, topk_weights=t, workspace=ws)
    want, error = torch.full(out.shape, 5.0, dtype=torch.float64, device="cuda:0"), torch.zeros(out.shape, device="cuda:0").double()
    at = 0
    for i, c in enumerate(counts):
        pair = order[at:at + c].long()
        y, s = plain.product(x[pair if mix else pair // topk], plain.values(codes[i], scales[i]), None if b is None else b[i], gated)
        if mix:       # one more rounding, in 32 bits
            y, s = y * t[pair, None].double(), s * t[pair, None].double()
            s = s + 2.0 ** -23 * y.abs()
        want[pair], error[pair] = y, s
        at += c
    assert held.tolist() == list(counts)
    assert first.tolist() == [sum(counts[:i]) for i in range(e + 1)]
    return out, want, error


COUNTS = {
    "one": [1], "two of eight": [0, 0, 1, 0, 0, 0, 1, 0], "few": [0, 3, 0, 1, 2], "sixteen": [16, 0, 17, 15], "uneven": [5, 70, 0, 33],
    "many": [i % 4 for i in range(130)], "large": [100, 0, 260, 31, 129], "all in one": [0, 0, 513],
}


@pytest.mark.parametrize("dtype", [BF, F16], ids=str)
@pytest.mark.parametrize("name", list(COUNTS))
@pytest.mark.parametrize("n,k", [(130, 96), (64, 544), (320, 1024)])
def test_grouped(gpu, dtype, name, n, k):
    counts = COUNTS[name]
    gated, mix = n % 64 == 0 and k != 1024, k == 1024
    ok, why = plain.close(*_grouped(counts, n, k, dtype, gated, min(2, len(counts)), mix, n == 64, seed=n + k))
    assert ok, why


@pytest.mark.parametrize("counts,none", [([0, 0], 3), ([4, 0, 40], 9), ([200, 100], 1)])
def test_grouped_pairs_of_no_expert(gpu, counts, none):
    """... leave their rows as they were."""
    ok, why = plain.close(*_grouped(counts, 130, 160, BF, False, 2, False, False, seed=7, none=none))
    assert ok, why


def test_grouped_ids_outside(gpu):
    """A pair that does not exist is left out."""
    n, k, g = 64, 96, _gen(3)
    codes, scales = plain.checkpoint(g, 2, n, k)
    x = _randn(g, 6, k).to(BF)
    order = torch.tensor([2, -1, 0, 6, 2 ** 31 - 1, 4], dtype=torch.int32, device=gpu)
    ids = torch.tensor([0, 0, 0, 1, 1, 1], dtype=torch.int32, device=gpu)
    plan = w4.MoeW4GroupedPlan.select(w4.MoeW4GroupedDescriptor(2, 1, 6, n, k))
    out = torch.full((6, n), 5.0, dtype=BF, device=gpu)
    plan.run(x, _packed(codes, scales), order, ids, out, torch.empty(2, dtype=torch.int32, device=gpu),
             torch.empty(3, dtype=torch.int32, device=gpu))
    for row, e in ((2, 0), (0, 0), (4, 1)):
        ok, why = plain.close(out[row:row + 1], *plain.product(x[row:row + 1], plain.values(codes[e], scales[e])))
        assert ok, why
    assert bool((out[[1, 3, 5]] == 5).all())


# ---- as they are used ------------------------------------------------------------------
def _mlp(gpu, tokens, e, topk, hidden, inner, seed):
    """A mixture's layer: quantized weights, gate and up, down weighted by the router."""
    g = _gen(seed)
    up, down = _randn(g, e, 2 * inner, hidden) * hidden ** -0.5, _randn(g, e, hidden, inner) * inner ** -0.5
    packs, vals = [], []
    for w in (up, down):
        plan = w4.W4WeightsPlan.select(w4.W4WeightsDescriptor(w.shape[1], w.shape[2], e, element=ElementKind.F32))
        p = torch.empty(e, w4.packed_bytes(w.shape[1], w.shape[2]), dtype=torch.uint8, device=gpu)
        plan.quantize(w, p)
        v = torch.empty_like(w)
        plan.read(p, v)
        packs.append(p)
        vals.append(v.double())
    pairs = tokens * topk
    s = dict(x=torch.empty(tokens, hidden, dtype=BF, device=gpu), order=torch.empty(pairs, dtype=torch.int32, device=gpu),
             ids=torch.empty(pairs, dtype=torch.int32, device=gpu), mix=torch.empty(pairs, device=gpu),
             h=torch.empty(pairs, inner, dtype=BF, device=gpu), y=torch.empty(pairs, hidden, dtype=BF, device=gpu),
             counts=torch.empty(e, dtype=torch.int32, device=gpu), offsets=torch.empty(e + 1, dtype=torch.int32, device=gpu))
    first = w4.MoeW4GroupedPlan.select(w4.MoeW4GroupedDescriptor(e, topk, pairs, 2 * inner, hidden, gated=True))
    second = w4.MoeW4GroupedPlan.select(w4.MoeW4GroupedDescriptor(e, topk, pairs, hidden, inner))
    ws = [torch.empty(p.workspace_size(), dtype=torch.uint8, device=gpu) for p in (first, second)]

    def fill(seed):
        r = _gen(seed)
        s["x"].copy_(_randn(r, tokens, hidden))
        top = torch.topk(_randn(r, tokens, e), topk, dim=1)
        ids, order = torch.sort(top.indices.flatten(), stable=True)
        s["ids"].copy_(ids)
        s["order"].copy_(order)
        s["mix"].copy_(torch.softmax(top.values, 1).flatten())

    def step():
        first.run(s["x"], packs[0], s["order"], s["ids"], s["h"], s["counts"], s["offsets"], workspace=ws[0])
        second.run(s["h"], packs[1], s["order"], s["ids"], s["y"], s["counts"], s["offsets"], topk_weights=s["mix"], workspace=ws[1])

    def want():
        order, ids = s["order"].long(), s["ids"].long()
        h, y = torch.empty_like(s["h"]), torch.empty_like(s["y"])
        hw, yw = torch.empty(pairs, inner, device=gpu).double(), torch.empty(pairs, hidden, device=gpu).double()
        eh, ey = torch.empty_like(hw), torch.empty_like(yw)
        for i in range(e):
            p = order[ids == i]
            hw[p], eh[p] = plain.product(s["x"][p // topk], vals[0][i], None, True)
            # the second product is that of the first one's rounded results
            w, err = plain.product(s["h"][p], vals[1][i])
            m = s["mix"][p, None].double()
            yw[p], ey[p] = w * m, err * m + 2.0 ** -23 * (w * m).abs()
        return (hw, eh), (yw, ey)

    return s, fill, step, want


@pytest.mark.parametrize("tokens", [1, 30, 300])
def test_layer(gpu, tokens):
    s, fill, step, want = _mlp(gpu, tokens, 8, 2, 256, 352, seed=5)
    fill(1)
    step()
    for got, (w, err) in zip((s["h"], s["y"]), want()):
        ok, why = plain.close(got, w, err)
        assert ok, why


@pytest.mark.parametrize("tokens", [2, 150])
def test_layer_captured(gpu, tokens):
    """Captured on a stream of its own and replayed with other tokens and routes."""
    s, fill, step, want = _mlp(gpu, tokens, 8, 2, 256, 352, seed=6)
    fill(0)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        fill(10 + i)
        s["h"].fill_(9)
        s["y"].fill_(9)
        graph.replay()
        torch.cuda.synchronize()
        for got, (w, err) in zip((s["h"], s["y"]), want()):
            ok, why = plain.close(got, w, err)
            assert ok, why
        first = s["y"].clone()
        step()
        torch.cuda.synchronize()
        assert torch.equal(first, s["y"])


@pytest.mark.parametrize("m", [1, 24, 600])
def test_linear_on_another_stream(gpu, m):
    n, k, g = 256, 512, _gen(m)
    codes, scales = plain.checkpoint(g, 1, n, k)
    packed, x = _packed(codes, scales), _randn(g, m, k).to(BF)
    plan = w4.W4LinearPlan.select(w4.W4LinearDescriptor(m, n, k))
    ws = torch.empty(plan.workspace_size(), dtype=torch.uint8, device=gpu)
    out = torch.zeros(m, n, dtype=BF, device=gpu)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    plan.run(x, packed, out, workspace=ws, stream=stream)
    stream.synchronize()
    ok, why = plain.close(out, *plain.product(x, plain.values(codes, scales)[0]))
    assert ok, why
    again = torch.zeros_like(out)
    plan.run(x, packed, again, workspace=ws)
    assert torch.equal(out, again)             # sums in a fixed order
