"""The operators around a 4-bit key-value cache against plain 64-bit arithmetic
(tests/kv4_plain.py): codes and whole numbers exactly, values within bounds that
count the roundings."""
import math
import random

import pytest
import torch

from baracuda_amd import kv4
from baracuda_amd.plans import ElementKind
from tests import kv4_plain as plain
from tests.gpu_util import sync

pytestmark = pytest.mark.gpu

KIND = {torch.float32: ElementKind.F32, torch.float16: ElementKind.F16, torch.bfloat16: ElementKind.Bf16}
BF, HF, FL = torch.bfloat16, torch.float16, torch.float32


def _dev(t):
    return t.to("cuda:0")


def _same(got, want, what=""):
    assert torch.equal(got.cpu(), want), f"{what}: {(got.cpu() != want).sum()} of {want.numel()} differ"


# ---- norm and rotation -------------------------------------------------------
def _rows(g, t, heads, d, dt):
    x = torch.randn(t, heads, d, generator=g) * (1 + 5 * (torch.rand(heads, d, generator=g) < 0.05))
    return x.to(dt)


def _rotation(g, t, rope, axes, rows=97):
    if not rope:
        return dict(positions=None, cos=None, sin=None, pair_axis=None)
    half = rope // 2
    angle = torch.rand(rows, half, generator=g) * 6.3
    axis = torch.randint(0, axes, (half,), generator=g, dtype=torch.int32) if axes > 1 else None
    return dict(positions=torch.randint(0, rows, (axes, t), generator=g, dtype=torch.int32), cos=angle.cos(), sin=angle.sin(),
                pair_axis=axis)


def _on_gpu(rot):
    return {k: None if v is None else _dev(v) for k, v in rot.items()}


def _plain_rows(x, w, eps, rope, rot, interleaved):
    axis = [0] * (rope // 2) if rot["pair_axis"] is None else rot["pair_axis"].tolist()
    return plain.norm_rope(x, w, eps, rope, rot["positions"], rot["cos"], rot["sin"], axis, interleaved)


def _near(got, want, size, dt):
    # one rounding to the type, and the statistics and products in 32 bits:
    # a sum of D squares in lanes of 8 and a tree, a root, a division, three products
    bound = plain.half_step(dt) * want.abs() + 32 * 2.0 ** -24 * size + torch.finfo(dt).tiny
    off = (got.cpu().double() - want).abs()
    assert bool((off <= bound).all()), f"worst {float((off / bound).max()):.2f} of the bound"


QK = [  # tokens, hq, hk, D, rope, axes, interleaved, dtype
    (1, 32, 8, 128, 128, 1, False, BF), (3, 5, 1, 64, 64, 1, True, HF), (7, 1, 1, 16, 16, 1, False, FL),
    (5, 7, 3, 80, 32, 3, False, BF), (2, 9, 2, 256, 64, 1, True, BF), (33, 4, 4, 256, 256, 3, False, FL),
    (4, 3, 1, 112, 112, 2, False, HF), (6, 2, 2, 48, 0, 1, False, BF), (129, 40, 8, 128, 64, 3, True, BF),
    (600, 28, 4, 128, 128, 1, False, BF), (2100, 8, 1, 64, 32, 1, False, HF)]


@pytest.mark.parametrize("case", QK, ids=str)
def test_qk_norm_rope(gpu, case):
    t, hq, hk, d, rope, axes, inter, dt = case
    print(f"qk {case}", flush=True)
    g = torch.Generator().manual_seed(t * 131 + d)
    row = _rows(g, t, hq + 2 * hk, d, dt)
    wq, wk = ((1 + 0.2 * torch.randn(d, generator=g)).to(dt) for _ in range(2))
    rot = _rotation(g, t, rope, axes)
    x = _dev(row)
    q_out = torch.empty(t, hq, d, dtype=dt, device=gpu)
    k_out = torch.empty(t, hk, d, dtype=dt, device=gpu)
    plan = kv4.QkNormRopePlan.select(kv4.QkNormRopeDescriptor(t, hq, hk, d, rope, KIND[dt], axes, inter, 1e-5))
    assert plan.workspace_size() == 0
    plan.run(x[:, :hq], x[:, hq:hq + hk], q_out, k_out, q_weight=_dev(wq), k_weight=_dev(wk), **_on_gpu(rot))
    for got, part, w in ((q_out, row[:, :hq], wq), (k_out, row[:, hq:hq + hk], wk)):
        want, size = _plain_rows(part, w, 1e-5, rope, rot, inter)
        _near(got, want, size, dt)
    _same(x, row, "input")
    # the same in place, and with heads before tokens
    plan.run(x[:, :hq], x[:, hq:hq + hk], x[:, :hq], x[:, hq:hq + hk], q_weight=_dev(wq), k_weight=_dev(wk), **_on_gpu(rot))
    _same(x[:, :hq], q_out.cpu(), "in place")
    _same(x[:, hq:hq + hk], k_out.cpu(), "in place")
    _same(x[:, hq + hk:], row[:, hq + hk:], "V")
    turned = torch.empty(hq, t, d, dtype=dt, device=gpu).transpose(0, 1)
    plan.run(_dev(row)[:, :hq], _dev(row)[:, hq:hq + hk], turned, k_out, q_weight=_dev(wq), k_weight=_dev(wk), **_on_gpu(rot))
    _same(turned, q_out.cpu(), "heads first")


def test_qk_without_norm_and_odd_addresses(gpu):
    t, hq, hk, d = 5, 3, 2, 64
    g = torch.Generator().manual_seed(4)
    buf = torch.randn(t * (hq + hk) * (d + 3) + 1, generator=g).to(BF)
    rot = _rotation(g, t, d, 1)
    x = _dev(buf)[1:].view(t, hq + hk, d + 3)[..., 1:d + 1]     # rows start at any even address
    q_out = torch.empty(t * hq * d + 1, dtype=BF, device=gpu)[1:].view(t, hq, d)
    k_out = torch.empty(t, hk, d, dtype=BF, device=gpu)
    plan = kv4.QkNormRopePlan.select(kv4.QkNormRopeDescriptor(t, hq, hk, d, d, norm=False))
    plan.run(x[:, :hq], x[:, hq:], q_out, k_out, **_on_gpu(rot))
    host = x.cpu()
    for got, part in ((q_out, host[:, :hq]), (k_out, host[:, hq:])):
        want, size = _plain_rows(part, None, 0, d, rot, False)
        _near(got, want, size, BF)


def test_qk_positions_out_of_range_give_nan(gpu):
    t, d = 4, 64
    g = torch.Generator().manual_seed(5)
    x = _rows(g, t, 2, d, BF)
    rot = _rotation(g, t, 32, 1, rows=9)
    rot["positions"] = torch.tensor([[0, -1, 9, 8]], dtype=torch.int32)
    w = torch.ones(d, dtype=BF)
    out = [torch.empty(t, 1, d, dtype=BF, device=gpu) for _ in range(2)]
    kv4.QkNormRopePlan.select(kv4.QkNormRopeDescriptor(t, 1, 1, d, 32)).run(
        _dev(x[:, :1]), _dev(x[:, 1:]), *out, q_weight=_dev(w), k_weight=_dev(w), **_on_gpu(rot))
    for o in out:
        bad = torch.isnan(o.cpu())
        assert bad[1:3, :, :32].all() and not bad[1:3, :, 32:].any() and not bad[0].any() and not bad[3].any()


@pytest.mark.parametrize("dt", [BF, FL], ids=str)
@pytest.mark.parametrize("t", [5, 520])
def test_qk_squares_out_of_range(gpu, dt, t):
    # next to heads of ordinary size, heads whose squares 32 bits do not hold
    d, eps = 128, 0.0
    g = torch.Generator().manual_seed(6)
    x = _rows(g, t, 4, d, FL)
    x[:, 0] *= 1e25
    x[:, 2] *= 1e-25
    x[::2, 3] *= 2e35
    x = x.to(dt)
    w = (1 + 0.2 * torch.randn(d, generator=g)).to(dt)
    rot = _rotation(g, t, 64, 1)
    out = [torch.empty(t, 2, d, dtype=dt, device=gpu) for _ in range(2)]
    kv4.QkNormRopePlan.select(kv4.QkNormRopeDescriptor(t, 2, 2, d, 64, KIND[dt], eps=eps)).run(
        _dev(x[:, :2]), _dev(x[:, 2:]), *out, q_weight=_dev(w), k_weight=_dev(w), **_on_gpu(rot))
    for got, part in ((out[0], x[:, :2]), (out[1], x[:, 2:])):
        want, size = _plain_rows(part, w, eps, 64, rot, False)
        _near(got, want, size, dt)


@pytest.mark.parametrize("t", [5, 520])
def test_append_squares_out_of_range(gpu, t):
    hq, hk, d, ps = 1, 3, 64, 16
    g = torch.Generator().manual_seed(7)
    x = _rows(g, t, hq + 2 * hk, d, FL)
    x[:, 0] *= 1e30
    x[:, 1] *= 1e25
    x[:, 2] *= 1e-25
    x = x.to(BF)
    w = (1 + 0.2 * torch.randn(d, generator=g)).to(BF)
    rot = _rotation(g, t, d, 1)
    pages = -(-t // ps)
    cache = torch.zeros(pages, hk, kv4.head_bytes(ps, d), dtype=torch.uint8)
    got, q_out = _dev(cache), torch.empty(t, hq, d, dtype=BF, device=gpu)
    kv4.Kv4AppendPlan.select(kv4.Kv4AppendDescriptor(t, hq, hk, d, ps, pages, d, eps=0.0)).run(
        _dev(x[:, hq:hq + hk]), _dev(x[:, hq + hk:]), got, _dev(torch.arange(t)), q=_dev(x[:, :hq]), q_out=q_out,
        q_weight=_dev(w), k_weight=_dev(w), **_on_gpu(rot))
    want, size = _plain_rows(x[:, :hq], w, 0.0, d, rot, False)
    _near(q_out, want, size, BF)
    k = _plain_rows(x[:, hq:hq + hk], w, 0.0, d, rot, False)[0].float().to(BF)
    for i in range(t):
        for h in range(hk):
            plain.put(cache, i, h, k[i, h], x[i, hq + hk + h], plain.most(BF))
    _same(got, cache, "cache")


def test_qk_rows_of_zeros_and_infinities(gpu):
    t, d = 3, 128
    x = torch.zeros(t, 2, d, dtype=BF)
    x[1, :, 5], x[2, :, 7] = math.inf, math.nan
    w = torch.ones(d, dtype=BF)
    out = [torch.empty(t, 1, d, dtype=BF, device=gpu) for _ in range(2)]
    kv4.QkNormRopePlan.select(kv4.QkNormRopeDescriptor(t, 1, 1, d, 0)).run(
        _dev(x[:, :1]), _dev(x[:, 1:]), *out, q_weight=_dev(w), k_weight=_dev(w))
    for o in out:
        o = o.cpu()
        assert (o[0] == 0).all() and torch.isnan(o[1, 0, 5]) and torch.isnan(o[2]).all()


# ---- into the cache and back -------------------------------------------------
def _read(cache, slots, d, ps, dt):
    t, hk = slots.numel(), cache.shape[1]
    k = torch.empty(t, hk, d, dtype=dt, device=cache.device)
    v = torch.empty_like(k)
    kv4.Kv4ReadPlan.select(kv4.Kv4ReadDescriptor(t, hk, d, ps, cache.shape[0], KIND[dt])).run(cache, slots, k, v)
    return k, v


@pytest.mark.parametrize("dt", [BF, HF], ids=str)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_codes_of_every_value(gpu, dt, d):
    """Every bit pattern of the type among 31 others of every size (infinities and
    NaN among them) and among others near its own."""
    g = torch.Generator().manual_seed(d)
    bits = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16)
    wild = bits[torch.randperm(65536, generator=g)]
    step = 10 if dt == HF else 7                      # mantissa bits: neighbours within a few powers of two
    near = (bits.int() & 0x7fff).sort()[0]
    near = (near.view(-1, 32)[:, torch.randperm(32, generator=g)] - torch.randint(0, 4 << step, (2048, 32), generator=g)).clamp(0, 0x7fff)
    near = (near | (torch.randint(0, 2, near.shape, generator=g) << 15)).to(torch.int16).flatten()
    vals = torch.cat((wild, near)).view(dt).view(-1, 1, d)
    t = vals.shape[0]
    ps, pages = 64, -(-t // 64)
    cache = torch.zeros(pages, 1, kv4.head_bytes(ps, d), dtype=torch.uint8, device=gpu)
    slots = torch.arange(t, device=gpu)
    x = _dev(vals)
    kv4.Kv4AppendPlan.select(kv4.Kv4AppendDescriptor(t, 0, 1, d, ps, pages, element=KIND[dt], norm=False)).run(
        x, x, cache, slots)
    sync()
    code, byte = plain.encode(vals[:, 0].double(), plain.most(dt))
    k, v, ks, vs = plain.places(ps, d)
    host = cache.cpu()[:, 0]
    for codes, scales in ((k, ks), (v, vs)):
        got = host[:, codes].flatten(0, 1)[:t]
        got = torch.stack((got & 15, got >> 4), -1).flatten(-2)
        _same(host[:, scales].flatten(0, 1)[:t], byte, "scales")
        _same(got, code, "codes")
    want = plain.decode(code, byte).to(torch.float32)
    for got in _read(cache, slots, d, ps, FL):
        got = got.cpu()[:, 0]
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(), want.nan_to_num())


APPEND = [  # tokens, hq, hk, D, rope, axes, interleaved, dtype, page size
    (1, 32, 8, 128, 128, 1, False, BF, 64), (48, 32, 8, 128, 128, 1, False, BF, 16), (37, 16, 2, 256, 64, 1, True, HF, 16),
    (5, 10, 5, 64, 64, 3, False, BF, 32), (131, 7, 1, 64, 32, 1, False, HF, 128), (3, 2, 1, 256, 256, 1, False, BF, 1024),
    (19, 0, 4, 128, 64, 1, False, BF, 16), (260, 4, 4, 128, 0, 1, False, HF, 64)]


@pytest.mark.parametrize("case", APPEND, ids=str)
def test_append(gpu, case):
    t, hq, hk, d, rope, axes, inter, dt, ps = case
    print(f"append {case}", flush=True)
    g = torch.Generator().manual_seed(t * 17 + d)
    row = _rows(g, t, hq + 2 * hk, d, dt)
    wq, wk = ((1 + 0.2 * torch.randn(d, generator=g)).to(dt) for _ in range(2))
    rot = _rotation(g, t, rope, axes)
    pages = -(-t // ps) + 2
    slots = torch.randperm(pages * ps, generator=g)[:t]
    if t > 4:
        slots[1], slots[3] = -1, pages * ps           # neither is written
    start = torch.randint(0, 256, (pages, hk, kv4.head_bytes(ps, d)), generator=g, dtype=torch.uint8)
    cache, x = _dev(start), _dev(row)
    q_out = torch.empty(t, hq, d, dtype=dt, device=gpu) if hq else None
    kv4.Kv4AppendPlan.select(kv4.Kv4AppendDescriptor(t, hq, hk, d, ps, pages, rope, KIND[dt], axes, inter)).run(
        x[:, hq:hq + hk], x[:, hq + hk:], cache, _dev(slots), q=x[:, :hq] if hq else None, q_out=q_out, q_weight=_dev(wq),
        k_weight=_dev(wk), **_on_gpu(rot))
    sync()
    if hq:
        want, size = _plain_rows(row[:, :hq], wq, 1e-6, rope, rot, inter)
        _near(q_out, want, size, dt)
    k = _plain_rows(row[:, hq:hq + hk], wk, 1e-6, rope, rot, inter)[0].float().to(dt)
    want = start.clone()
    for i in range(t):
        if 0 <= slots[i] < pages * ps:
            for h in range(hk):
                plain.put(want, slots[i], h, k[i, h], row[i, hq + hk + h], plain.most(dt))
    _same(cache, want, "cache")


@pytest.mark.parametrize("dt", [BF, HF, FL], ids=str)
def test_read(gpu, dt):
    t, hk, d, ps, pages = 50, 3, 128, 32, 3
    g = torch.Generator().manual_seed(9)
    host = torch.randint(0, 256, (pages, hk, kv4.head_bytes(ps, d)), generator=g, dtype=torch.uint8)
    host[:, :, ps * d:] = torch.randint(110, 140, host[:, :, ps * d:].shape, generator=g, dtype=torch.uint8)
    slots = torch.randint(0, pages * ps, (t,), generator=g)
    slots[7], slots[8], slots[9] = -1, pages * ps, 2 ** 40
    wide = torch.full((hk, t, 2 * d), 7.0, dtype=dt, device=gpu)
    k_out, v_out = wide[..., :d].transpose(0, 1), wide[..., d:].transpose(0, 1)
    kv4.Kv4ReadPlan.select(kv4.Kv4ReadDescriptor(t, hk, d, ps, pages, KIND[dt])).run(_dev(host), _dev(slots), k_out, v_out)
    k, v = plain.get(host, torch.arange(pages), d)     # [heads, tokens, D]
    ok = (slots >= 0) & (slots < pages * ps)
    for got, want in ((k_out, k), (v_out, v)):
        want = torch.where(ok[:, None, None], want[:, slots.clamp(0, pages * ps - 1)].transpose(0, 1), 0.0)
        _same(got, want.float().to(dt))


# ---- attention -----------------------------------------------------------------
def _scene(g, lens, qs, hq, hk, d, ps, dt, extra=3, garbage=True):
    """A cache with sequences in pages of any order; what no sequence holds is garbage, NaN scales among it."""
    need = [-(-max(n, 0) // ps) for n in lens]
    pages = sum(need) + extra
    cache = torch.zeros(pages, hk, kv4.head_bytes(ps, d), dtype=torch.uint8)
    cache[:, :, :ps * d] = torch.randint(0, 256, cache[:, :, :ps * d].shape, generator=g, dtype=torch.uint8)
    cache[:, :, ps * d:] = torch.randint(125, 128, cache[:, :, ps * d:].shape, generator=g, dtype=torch.uint8)
    order = torch.randperm(pages, generator=g)
    tables = torch.full((len(lens), max(need + [1]) + 1), -1, dtype=torch.int32)
    at, places = 0, plain.places(ps, d)
    for b, n in enumerate(need):
        tables[b, :n] = order[at:at + n]
        if garbage and n and lens[b] % ps:
            last = int(order[at + n - 1])
            for p in places[2:]:
                cache[last][:, p[lens[b] % ps:].flatten()] = 255
        at += n
    if garbage:
        cache[order[at:]] = 255
    cu = torch.cumsum(torch.tensor([0] + qs), 0).to(torch.int32)
    q = (torch.randn(int(cu[-1]), hq, d, generator=g) * 1.5).to(dt)
    return cache, tables, torch.tensor(lens, dtype=torch.int32), cu, q


def _check_attention(got, q, cache, tables, lens, cu, causal, window, scale):
    want, size, score = plain.attention(q, cache, tables, lens, cu, causal, window, scale)
    dt, d = q.dtype, q.shape[2]
    u = plain.half_step(dt)
    # one rounding of the result; P rounded to the type; scores as sums of D
    # products in 32 bits, and their exponentials; f16 has no weights below 2^-24
    score_error = (d + 8) * 2.0 ** -24 * score[..., None] + 2.0 ** -20
    top = float(size.max()) if size.numel() else 0.0
    tiny = 2.0 ** -25 * float(lens.max()) * 6 * top if dt == torch.float16 else 0.0
    bound = u * want.abs() + (1.02 * u + 2 * score_error) * size + tiny + 1e-30
    off = (got.cpu().double() - want).abs()
    assert not torch.isnan(got).any()
    assert bool((off <= bound).all()), f"worst {float((off / bound).max()):.2f} of the bound"


def _attend(scene, hk, causal=True, window=0, scale=None, max_kv=None, out=None, workspace_fill=0x7f):
    cache, tables, lens, cu, q = scene
    total, hq, d = q.shape
    ps = cache.shape[2] // (d + d // 16)
    qs = (cu[1:] - cu[:-1]).tolist()
    plan = kv4.Kv4AttentionPlan.select(kv4.Kv4AttentionDescriptor(
        len(lens), total, max(qs + [0]), int(lens.max()) if max_kv is None else max_kv, hq, hk, d, ps, cache.shape[0],
        tables.shape[1], KIND[q.dtype], causal, window, scale))
    ws = torch.full((plan.workspace_size(),), workspace_fill, dtype=torch.uint8, device="cuda:0")
    out = torch.full((total, hq, d), 3.0, dtype=q.dtype, device="cuda:0") if out is None else out
    plan.run(_dev(q), _dev(cache), _dev(tables), _dev(lens), out, cu_q=_dev(cu), workspace=ws)
    sync()
    return out


ATTN = [  # lens, new tokens, hq, hk, D, page size, dtype, causal, window
    ([1], [1], 8, 8, 128, 16, BF, True, 0),
    ([777], [1], 32, 8, 128, 16, BF, True, 0),
    ([5, 0, 17, 64, 65, 1], [1] * 6, 8, 2, 64, 16, HF, True, 0),
    ([300, 31], [1, 1], 7, 1, 256, 32, BF, True, 0),
    ([1500, 3, 2049], [1, 1, 1], 16, 2, 128, 64, BF, True, 0),
    ([2600, 1200], [5, 5], 10, 2, 64, 32, HF, True, 1024),
    ([130, 9], [9, 9], 8, 1, 128, 128, BF, True, 0),
    ([1300], [9], 8, 1, 256, 16, HF, True, 100),
    ([200, 90, 33], [70, 90, 1], 4, 2, 128, 64, BF, True, 0),
    ([1100, 150], [300, 20], 2, 1, 64, 16, BF, True, 33),
    ([140, 70], [40, 3], 5, 5, 128, 16, HF, False, 0),
    ([1400, 90], [3, 2], 8, 4, 256, 64, BF, False, 0),
    ([20, 3], [4, 0], 14, 2, 128, 16, BF, True, 1),
    ([40], [64], 4, 2, 64, 16, BF, True, 0),               # more new tokens than the cache holds: rows that see nothing
    ([1025] * 3, [17, 1, 33], 16, 2, 128, 32, BF, True, 7),
    ([600, 130], [257, 129], 8, 2, 256, 64, HF, True, 0),
]


@pytest.mark.parametrize("case", ATTN, ids=str)
def test_attention(gpu, case):
    lens, qs, hq, hk, d, ps, dt, causal, window = case
    print(f"attention {case}", flush=True)
    scene = _scene(torch.Generator().manual_seed(sum(lens) + d), lens, qs, hq, hk, d, ps, dt)
    got = _attend(scene, hk, causal, window)
    cache, tables, lens_t, cu, q = scene
    _check_attention(got, q, cache, tables, lens_t, cu, causal, window, d ** -0.5)


def test_attention_drawn_cases(gpu):
    rng = random.Random(20)
    for i in range(24):
        hk = rng.choice((1, 2, 3))
        hq, d, ps = hk * rng.choice((1, 2, 4, 5, 7, 8)), rng.choice((64, 128, 256)), rng.choice((16, 32, 64, 128))
        most_q = rng.choice((1, 1, 4, 9, 40, 150))
        qs = [rng.randint(0, most_q) for _ in range(rng.randint(1, 4))]
        qs[0] = most_q
        lens = [q + rng.choice((0, 1, rng.randint(0, 40), rng.randint(0, 1500))) for q in qs]
        dt, causal, window = rng.choice((BF, HF)), rng.random() < 0.8, rng.choice((0, 0, rng.randint(1, 200)))
        case = (lens, qs, hq, hk, d, ps, dt, causal, window)
        print(f"attention {i} {case}", flush=True)
        scene = _scene(torch.Generator().manual_seed(i), lens, qs, hq, hk, d, ps, dt)
        got = _attend(scene, hk, causal, window, max_kv=rng.choice((None, 6000)))
        cache, tables, lens_t, cu, q = scene
        _check_attention(got, q, cache, tables, lens_t, cu, causal, window, d ** -0.5)


@pytest.mark.parametrize("qs", [[1, 1, 1], [40, 33, 90]], ids=str)
def test_attention_pages_that_are_missing(gpu, qs):
    """An entry outside the cache, in a sequence's middle or everywhere, stands for tokens that no row sees."""
    lens = [200, 150, 90]
    cache, tables, lens_t, cu, q = _scene(torch.Generator().manual_seed(3), lens, qs, 4, 2, 128, 16, BF)
    tables[0, 4], tables[0, 5], tables[2, :] = -1, cache.shape[0], -7
    scene = cache, tables, lens_t, cu, q
    got = _attend(scene, 2)
    _check_attention(got, q, cache, tables, lens_t, cu, True, 0, 128 ** -0.5)
    assert (got.cpu()[int(cu[2]):] == 0).all()


@pytest.mark.parametrize("q1", [1, 70])
def test_attention_strides_and_streams(gpu, q1):
    lens, qs, hq, hk, d = [130, 1400], [q1, 2], 4, 2, 128
    cache, tables, lens_t, cu, q = _scene(torch.Generator().manual_seed(6), lens, qs, hq, hk, d, 32, BF)
    plan = kv4.Kv4AttentionPlan.select(kv4.Kv4AttentionDescriptor(2, q1 + 2, q1 + 1, 1400, hq, hk, d, 32, cache.shape[0],
                                                                 tables.shape[1]))
    wide = torch.zeros(2, tables.shape[1] + 5, dtype=torch.int32, device=gpu)
    wide[:, :tables.shape[1]] = _dev(tables)
    fused = torch.zeros(q1 + 2, hq + 3, d + 5, dtype=BF, device=gpu)[:, 1:hq + 1, 3:d + 3]
    out = torch.zeros(hq, q1 + 2, d + 1, dtype=BF, device=gpu)[..., 1:].transpose(0, 1)
    args = [_dev(x) for x in (cache, lens_t, cu, q)]
    ws = torch.empty(plan.workspace_size(), dtype=torch.uint8, device=gpu)
    sync()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        fused.copy_(args[3])
        plan.run(fused, args[0], wide[:, :tables.shape[1]], args[1], out, cu_q=args[2], workspace=ws)
    side.synchronize()
    _check_attention(out, q, cache, tables, lens_t, cu, True, 0, d ** -0.5)


def test_attention_one_row_each_needs_no_cu(gpu):
    lens = [100, 7, 1100]
    cache, tables, lens_t, cu, q = _scene(torch.Generator().manual_seed(8), lens, [1] * 3, 8, 4, 64, 16, BF)
    plan = kv4.Kv4AttentionPlan.select(kv4.Kv4AttentionDescriptor(3, 3, 1, 1100, 8, 4, 64, 16, cache.shape[0], tables.shape[1]))
    ws = torch.empty(plan.workspace_size(), dtype=torch.uint8, device=gpu)
    out = torch.empty(3, 8, 64, dtype=BF, device=gpu)
    plan.run(_dev(q), _dev(cache), _dev(tables), _dev(lens_t), out, workspace=ws)
    _check_attention(out, q, cache, tables, lens_t, cu, True, 0, 64 ** -0.5)


@pytest.mark.parametrize("n", [1, 60])
def test_attention_past_32_bits(gpu, n):
    """A cache of more than 4 GiB, the sequence's pages at its end."""
    hk, d, ps = 8, 128, 128
    cache, tables, lens, cu, q = _scene(torch.Generator().manual_seed(2), [1200], [n], 16, hk, d, ps, BF, extra=0)
    have = cache.shape[0]
    pages = 6 * 2 ** 30 // (hk * kv4.head_bytes(ps, d))
    big = torch.empty(pages, hk, kv4.head_bytes(ps, d), dtype=torch.uint8, device=gpu)
    big[pages - have:] = _dev(cache)
    plan = kv4.Kv4AttentionPlan.select(kv4.Kv4AttentionDescriptor(1, n, n, 1200, 16, hk, d, ps, pages, tables.shape[1]))
    ws = torch.empty(plan.workspace_size(), dtype=torch.uint8, device=gpu)
    out = torch.empty(n, 16, d, dtype=BF, device=gpu)
    moved = torch.where(tables >= 0, tables + pages - have, -1)
    plan.run(_dev(q), big, _dev(moved), _dev(lens), out, cu_q=_dev(cu), workspace=ws)
    _check_attention(out, q, cache, tables, lens, cu, True, 0, d ** -0.5)
    # and the slots that append and read take
    slots = torch.tensor([(pages - 1) * ps + 5], device=gpu)
    x = torch.randn(1, hk, d, device=gpu).to(BF)
    kv4.Kv4AppendPlan.select(kv4.Kv4AppendDescriptor(1, 0, hk, d, ps, pages, norm=False)).run(x, x, big, slots)
    k, v = _read(big, slots, d, ps, BF)
    want = plain.decode(*plain.encode(x.cpu()[0], 125)).to(BF)
    _same(k[0], want)
    _same(v[0], want)


BIG = 2_000_000    # tokens that the host is told of where the large blocks of rows are meant to be taken


@pytest.mark.parametrize("part", ["K", "V"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("ratio,max_kv", [(1, None), (4, None), (8, None), (8, BIG)], ids=["16 rows", "32 rows", "48 rows", "large"])
def test_attention_of_values_that_are_not_finite(gpu, part, d, ratio, max_kv):
    """A NaN that a row sees makes it NaN, in V the values of its group; the rows
    before it, which do not see it, stay as they are."""
    lens, qs = [64], [6]
    cache, tables, lens_t, cu, q = _scene(torch.Generator().manual_seed(12), lens, qs, ratio, 1, d, 16, BF)
    if part == "V":
        cache[int(tables[0, 3]), 0, plain.places(16, d)[3][13, 1]] = 127     # so that its place is one of the two before
    clean = _attend((cache, tables, lens_t, cu, q), 1, max_kv=max_kv).cpu()
    _check_attention(clean, q, cache, tables, lens_t, cu, True, 0, d ** -0.5)
    if part == "K":
        cache[int(tables[0, 3]), 0, plain.places(16, d)[2][13]] = 255        # token 61, seen by the last three of six
        got = _attend((cache, tables, lens_t, cu, q), 1, max_kv=max_kv).cpu()
        assert torch.equal(got[:3], clean[:3]) and torch.isnan(got[3:]).all()
    else:
        cache[int(tables[0, 3]), 0, plain.places(16, d)[3][13, 1]] = 255     # values 32 to 63
        got = _attend((cache, tables, lens_t, cu, q), 1, max_kv=max_kv).cpu()
        assert torch.equal(got[:3], clean[:3]) and torch.isnan(got[3:, :, 32:64]).all()
        assert torch.equal(got[3:, :, :32], clean[3:, :, :32]) and torch.equal(got[3:, :, 64:], clean[3:, :, 64:])


LARGE = [  # as ATTN, cut into parts by what the host is told
    ([200, 90, 33], [70, 90, 1], 4, 2, 128, 64, BF, True, 0), ([1100, 150], [300, 20], 2, 1, 64, 16, BF, True, 33),
    ([140, 70], [40, 3], 5, 5, 128, 16, HF, False, 0), ([40], [64], 4, 2, 64, 16, BF, True, 0),
    ([600, 130], [257, 129], 8, 2, 256, 64, HF, True, 0), ([1400, 700], [37, 260], 4, 1, 128, 32, BF, True, 500),
    ([1025] * 3, [17, 1, 33], 16, 2, 128, 32, BF, True, 7), ([129, 128], [128, 127], 2, 2, 256, 128, BF, True, 0)]


@pytest.mark.parametrize("case", LARGE, ids=str)
def test_attention_in_large_blocks(gpu, case):
    lens, qs, hq, hk, d, ps, dt, causal, window = case
    print(f"attention {case}", flush=True)
    scene = _scene(torch.Generator().manual_seed(sum(lens) + d), lens, qs, hq, hk, d, ps, dt)
    got = _attend(scene, hk, causal, window, max_kv=BIG)
    cache, tables, lens_t, cu, q = scene
    _check_attention(got, q, cache, tables, lens_t, cu, causal, window, d ** -0.5)
    missing = tables.clone()
    missing[0, 1] = -1
    got = _attend((cache, missing, lens_t, cu, q), hk, causal, window, max_kv=BIG)
    _check_attention(got, q, cache, missing, lens_t, cu, causal, window, d ** -0.5)


@pytest.mark.parametrize("d,ratio,dt", [(128, 8, BF), (64, 16, HF)], ids=str)
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 90), (False, 0)])
def test_attention_in_blocks_from_both_ends(gpu, d, ratio, dt, causal, window):
    """Prompts of several large blocks of rows that are not cut: a workgroup has rows from
    the sequence's start and from its end, and an odd number of blocks a middle one."""
    qs = [70, 33, 1, 0, 64, 2, 17, 1, 40, 3, 1]
    lens = [70, 40, 300, 9, 64, 2, 200, 30, 41, 20, 1]
    scene = _scene(torch.Generator().manual_seed(d), lens, qs, 8 * ratio, 8, d, 16, dt)
    got = _attend(scene, 8, causal, window, max_kv=512)
    cache, tables, lens_t, cu, q = scene
    _check_attention(got, q, cache, tables, lens_t, cu, causal, window, d ** -0.5)


@pytest.mark.parametrize("seqs", [40, 70])
@pytest.mark.parametrize("most_q", [1, 41])
@pytest.mark.parametrize("d,told", [(64, 900), (128, 3000), (256, 3000)])
def test_attention_many_sequences(gpu, seqs, most_q, d, told):
    """More sequences than a wave has lanes, and more than a round of workgroups; with
    41 rows blocks of 32, or whole large ones, as the host's bound has it."""
    rng = random.Random(seqs + most_q)
    qs = [rng.randint(0, most_q) for _ in range(seqs)]
    qs[3] = most_q
    lens = [q + rng.randint(0, 60) for q in qs]
    lens[5] += 500
    hk = 8 if most_q > 1 else 2
    scene = _scene(torch.Generator().manual_seed(seqs), lens, qs, hk, hk, d, 16, BF)
    got = _attend(scene, hk, max_kv=told)
    cache, tables, lens_t, cu, q = scene
    _check_attention(got, q, cache, tables, lens_t, cu, True, 0, d ** -0.5)


@pytest.mark.parametrize("causal,window", [(True, 0), (True, 90), (False, 0)])
def test_attention_in_blocks_from_both_ends_told_of_1024_tokens(gpu, causal, window):
    qs = [70, 33, 1, 0, 64, 2, 17, 1, 40, 3, 1]
    lens = [70, 40, 300, 9, 64, 2, 200, 30, 41, 20, 1]
    scene = _scene(torch.Generator().manual_seed(3), lens, qs, 64, 8, 128, 16, BF)
    got = _attend(scene, 8, causal, window, max_kv=1024)
    cache, tables, lens_t, cu, q = scene
    _check_attention(got, q, cache, tables, lens_t, cu, causal, window, 128 ** -0.5)


@pytest.mark.parametrize("d,dt", [(64, HF), (128, BF), (256, BF)], ids=str)
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 90), (False, 0)])
def test_attention_in_blocks_of_32(gpu, d, dt, causal, window):
    """Blocks of 32 rows, one and two a sequence, enough of them to fill the card, some cut."""
    rng = random.Random(d)
    qs = [rng.randint(0, 12) for _ in range(35)]
    lens = [q + rng.randint(0, 40) for q in qs]
    qs[0], lens[0], qs[9], lens[9], qs[20], lens[20] = 11, 64, 12, 1400, 1, 333
    scene = _scene(torch.Generator().manual_seed(d), lens, qs, 24, 8, d, 16, dt)
    cache, tables, lens_t, cu, q = scene
    got = _attend(scene, 8, causal, window, max_kv=1500).cpu()
    _check_attention(got, q, cache, tables, lens_t, cu, causal, window, d ** -0.5)
    if causal:      # a NaN in V of token 61 of 64: rows 8 to 10 of the first sequence see it
        cache[int(tables[0, 3]), :, plain.places(16, d)[3][13, 1]] = 255
        odd = _attend((cache, tables, lens_t, cu, q), 8, causal, window, max_kv=1500).cpu()
        assert torch.isnan(odd[8:11, :, 32:64]).all()
        rest = torch.ones_like(odd, dtype=torch.bool)
        rest[8:11, :, 32:64] = False
        assert not torch.isnan(odd[rest]).any() and torch.equal(odd[11:], got[11:])


# ---- pages -----------------------------------------------------------------------
def _pages_plan(layers, pages, size, ps, rows, width):
    return kv4.KvPagesPlan.select(kv4.KvPagesDescriptor(layers, pages, size, ps, rows, width))


@pytest.mark.parametrize("size", [16, 17408, 1000, 33, 40000])
def test_pages_copy(gpu, size):
    g = torch.Generator().manual_seed(size)
    layers, pages = 3, 40
    host = torch.randint(0, 256, (layers, pages, size), generator=g, dtype=torch.uint8)
    order = torch.randperm(pages, generator=g).to(torch.int32)
    src, dst = order[:9].clone(), order[9:18].clone()
    want = host.clone()
    want[:, dst[:7].long()] = host[:, src[:7].long()]
    src[7], dst[8] = -1, pages
    cache = _dev(host)
    _pages_plan(layers, pages, size, 16, 1, 1).copy(cache, _dev(src), _dev(dst))
    _same(cache, want)


def _plain_fork(cache, tables, lens, refs, parents, children, ps):
    fresh = []
    for p, c in zip(parents, children):
        n = int(lens[p])
        full, part = n // ps, n % ps > 0
        free = (refs == 0).nonzero()
        page = -1
        if part:
            if not len(free):
                fresh.append(-2)
                tables[c], lens[c] = -1, 0
                continue
            page = int(free[0])
        tables[c] = -1
        tables[c, :full] = tables[p, :full]
        refs[tables[p, :full].long()] += 1
        if part:
            tables[c, full], refs[page] = page, 1
            cache[:, page] = cache[:, tables[p, full].long()]
        lens[c] = n
        fresh.append(page)
    return torch.tensor(fresh, dtype=torch.int32)


@pytest.mark.parametrize("case", [(3, 5, 4, False), (16, 37, 16, False), (1, 1, 16, True), (9, 50, 32, True)], ids=str)
def test_pages_fork_and_release(gpu, case):
    n, first, ps, scarce = case
    g = torch.Generator().manual_seed(n)
    layers, rows, width, size = 2, 24, 20, 48
    held = [-(-first // ps), 2, 3]
    pages = sum(held) + (n // 2 if scarce else 2 * n + 5)
    order = torch.randperm(pages, generator=g).to(torch.int32)
    tables = torch.full((rows, width), -1, dtype=torch.int32)
    lens, refs = torch.zeros(rows, dtype=torch.int32), torch.zeros(pages, dtype=torch.int32)
    at = 0
    for r, k in enumerate(held):
        tables[r, :k] = order[at:at + k]
        refs[order[at:at + k].long()] = 1
        at += k
    lens[0], lens[1], lens[2] = first, 2 * ps, 2 * ps + 1
    parents = torch.arange(n, dtype=torch.int32) % 3
    children = torch.randperm(rows - 4, generator=g)[:n].to(torch.int32) + 4
    cache = torch.randint(0, 256, (layers, pages, size), generator=g, dtype=torch.uint8)
    dev = [_dev(x) for x in (cache, tables, lens, refs)]
    fresh = torch.empty(n, dtype=torch.int32, device=gpu)
    plan = _pages_plan(layers, pages, size, ps, rows, width)
    plan.fork(*dev, _dev(parents), _dev(children), fresh)
    want = [x.clone() for x in (cache, tables, lens, refs)]
    want_fresh = _plain_fork(*want, parents.tolist(), children.tolist(), ps)
    _same(fresh, want_fresh, "fresh")
    for got, w in zip(dev, want):
        _same(got, w)
    gone = torch.cat((children[:2], children[:1], torch.tensor([-1, rows], dtype=torch.int32)))   # one twice, two that are none
    plan.release(*dev[1:], _dev(gone))
    for c in set(children[:2].tolist()):
        for e in want[1][c][want[1][c] >= 0].tolist():
            want[3][e] -= 1
        want[1][c], want[2][c] = -1, 0
    for got, w in zip(dev[1:], want[1:]):
        _same(got, w)


def test_pages_fork_of_rows_that_are_none(gpu):
    tables = torch.tensor([[0, 1], [-1, -1], [-1, -1], [-1, -1]], dtype=torch.int32)
    dev = [_dev(x) for x in (torch.zeros(1, 6, 32, dtype=torch.uint8), tables, torch.tensor([6, 0, 0, 0], dtype=torch.int32),
                             torch.tensor([1, 1, 0, 0, 0, 0], dtype=torch.int32))]
    fresh = torch.empty(4, dtype=torch.int32, device=gpu)
    parents, children = torch.tensor([9, 0, 0, 1]), torch.tensor([1, 7, 2, 3])
    _pages_plan(1, 6, 32, 4, 4, 2).fork(*dev, _dev(parents.int()), _dev(children.int()), fresh)
    _same(fresh, torch.tensor([-2, -2, 2, -1], dtype=torch.int32))
    _same(dev[1], torch.tensor([[0, 1], [-1, -1], [0, 2], [-1, -1]], dtype=torch.int32))
    _same(dev[2], torch.tensor([6, 0, 6, 0], dtype=torch.int32))
    _same(dev[3], torch.tensor([2, 1, 1, 0, 0, 0], dtype=torch.int32))


@pytest.mark.parametrize("case", [(1, 1, 16), (50, 0, 16), (50, 50, 33), (300, 100, 1008), (2500, 900, 16), (2500, 2000, 17)], ids=str)
def test_pages_compact(gpu, case):
    pages, used, size = case
    g = torch.Generator().manual_seed(pages + used)
    layers, rows, width = 2, 7, -(-max(used, 1) // 7) + 2
    order = torch.randperm(pages, generator=g).to(torch.int32)
    tables = torch.full((rows, width), -1, dtype=torch.int32)
    refs = torch.zeros(pages, dtype=torch.int32)
    for i in range(used):
        tables[i % rows, 1 + i // rows] = order[i]
        refs[int(order[i])] += 1
    if used:
        tables[:, 0] = order[0]
        refs[int(order[0])] += rows
    cache = torch.randint(0, 256, (layers, pages, size), generator=g, dtype=torch.uint8)
    live = refs > 0
    high = [p for p in range(used, pages) if live[p]]
    hole = [p for p in range(used) if not live[p]]
    remap = torch.where(live, torch.arange(pages, dtype=torch.int32), -1)
    want, moved = cache.clone(), torch.zeros_like(refs)
    for h, o in zip(high, hole):
        remap[h] = o
        want[:, o] = cache[:, h]
    for p in range(pages):
        if live[p]:
            moved[remap[p]] = refs[p]
    dev = [_dev(x) for x in (cache, tables, refs)]
    out = [torch.full_like(dev[1], 7), torch.full_like(dev[2], 7), torch.full_like(dev[2], 7)]
    count = torch.full((1,), 7, dtype=torch.int32, device=gpu)
    plan = _pages_plan(layers, pages, size, 16, rows, width)
    ws = torch.full((plan.workspace_size(),), 0x55, dtype=torch.uint8, device=gpu)
    plan.compact(*dev, *out, count, workspace=ws)
    _same(dev[0], want, "cache")
    _same(out[0], torch.where(tables >= 0, remap[tables.long().clamp(min=0)], -1), "tables")
    _same(out[1], moved, "refs")
    _same(out[2], remap, "remap")
    assert int(count) == used


# ---- captured ----------------------------------------------------------------------
def test_step_replayed_from_a_graph(gpu):
    """A step of a serving loop (append, attention, fork, release, compact) as a
    graph: every replay gives what eager calls give on the same state."""
    b, hq, hk, d, ps, rows, pages, width = 3, 8, 2, 128, 16, 8, 300, 96
    g = torch.Generator().manual_seed(1)
    cache = torch.zeros(pages, hk, kv4.head_bytes(ps, d), dtype=torch.uint8)
    cache[:, :, :ps * d] = torch.randint(0, 256, cache[:, :, :ps * d].shape, generator=g, dtype=torch.uint8)
    cache[:, :, ps * d:] = 126
    lens = torch.tensor([1100, 40, 333] + [0] * (rows - 3), dtype=torch.int32)
    tables = torch.full((rows, width), -1, dtype=torch.int32)
    refs = torch.zeros(pages, dtype=torch.int32)
    at = 0
    for r in range(b):
        n = -(-int(lens[r]) // ps)
        tables[r, :n] = torch.arange(at, at + n) * 2
        refs[torch.arange(at, at + n) * 2] = 1
        at += n
    rot = _on_gpu(_rotation(g, b, d, 1, rows=50))
    w = _dev(torch.ones(d, dtype=BF))
    append = kv4.Kv4AppendPlan.select(kv4.Kv4AppendDescriptor(b, hq, hk, d, ps, pages, d))
    attend = kv4.Kv4AttentionPlan.select(kv4.Kv4AttentionDescriptor(b, b, 1, width * ps, hq, hk, d, ps, pages, width))
    manage = _pages_plan(1, pages, cache[0].numel(), ps, rows, width)

    def state():
        return {"cache": _dev(cache), "tables": _dev(tables), "lens": _dev(lens), "refs": _dev(refs),
                "x": torch.zeros(b, hq + 2 * hk, d, dtype=BF, device=gpu), "slots": torch.zeros(b, dtype=torch.int64, device=gpu),
                "q": torch.empty(b, hq, d, dtype=BF, device=gpu), "out": torch.empty(b, hq, d, dtype=BF, device=gpu),
                "fresh": torch.empty(2, dtype=torch.int32, device=gpu), "tables2": torch.empty_like(_dev(tables)),
                "refs2": torch.empty_like(_dev(refs)), "remap": torch.empty_like(_dev(refs)),
                "live": torch.empty(1, dtype=torch.int32, device=gpu),
                "ws": torch.empty(attend.workspace_size(), dtype=torch.uint8, device=gpu),
                "ws2": torch.empty(manage.workspace_size(), dtype=torch.uint8, device=gpu)}

    parents, children = _dev(torch.tensor([0, 2], dtype=torch.int32)), _dev(torch.tensor([5, 6], dtype=torch.int32))

    def step(s):
        append.run(s["x"][:, hq:hq + hk], s["x"][:, hq + hk:], s["cache"], s["slots"], q=s["x"][:, :hq], q_out=s["q"],
                   q_weight=w, k_weight=w, **rot)
        attend.run(s["q"], s["cache"], s["tables"][:b], s["lens"][:b], s["out"], workspace=s["ws"])
        flat = s["cache"].view(1, pages, -1)
        manage.fork(flat, s["tables"], s["lens"], s["refs"], parents, children, s["fresh"])
        manage.release(s["tables"], s["lens"], s["refs"], children)
        manage.compact(flat, s["tables"], s["refs"], s["tables2"], s["refs2"], s["remap"], s["live"], workspace=s["ws2"])

    def feed(s, i):
        r = torch.Generator().manual_seed(100 + i)
        s["x"].copy_(torch.randn(b, hq + 2 * hk, d, generator=r).to(BF))
        new = lens[:b].clone() - i * torch.tensor([300, 3, 17])
        s["lens"][:b] = _dev(new.to(torch.int32))
        last = new.long() - 1
        s["slots"].copy_(_dev(tables[:b].gather(1, (last // ps)[:, None])[:, 0].long() * ps + last % ps))

    a, e = state(), state()
    feed(a, 0)
    step(a)
    sync()
    a = state()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(a)
    a2 = state()
    for k in a:
        a[k].copy_(a2[k])
    for i in range(4):
        feed(a, i)
        feed(e, i)
        step(e)
        sync()
        graph.replay()
        sync()
        print(f"replay {i}", flush=True)
        for k in ("cache", "tables", "lens", "refs", "q", "out", "fresh", "tables2", "refs2", "remap", "live"):
            assert torch.equal(a[k].view(torch.uint8) if a[k].dtype == BF else a[k],
                               e[k].view(torch.uint8) if e[k].dtype == BF else e[k]), k
        _ = torch.randn(512, 512, device=gpu) @ torch.randn(512, 512, device=gpu)
