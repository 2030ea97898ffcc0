"""Cases of products with weights held in 4 bits under group scales.

A case is a dict of plain values; `kind` names the operator and the other keys
its sizes and options:
  weights  matrices of float weights quantized to 4 bits and laid out for the
           products, and the values that they now stand for read back
  linear   x W^T for one token, a few, or a prompt, with a bias or with the gate
           of a gated MLP in the epilogue
  moe      the same by expert: token-expert pairs sorted by expert, an unequal
           number of them each
`listed()` holds the fixed cases, `draw()` more of the same ranges, `prepare()`
what a program holds before the call, `run()` one pass, `work()` the bytes and
operations that a pass cannot do without, and `exact()` the result in 64-bit
arithmetic.

A weight is a code times its group's scale: codes of sign, two exponent bits and
one mantissa bit (0, 0.5, 1, 1.5, 2, 3, 4, 6), and 2^(byte - 127) shared by 32
consecutive weights of a row.  In a checkpoint: codes uint8 [N, K / 2], two a
byte, the lower index in the lower four bits, and scales uint8 [N, K / 32].
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda:0"
_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_GROUP = 32      # weights that share a scale
_MAX_FLOPS = 2.0 * 4097 * 28672 * 4096      # of the largest linear case; the mixtures' is as large


def listed():
    return [
        # One token of one stream through a square projection: the smallest call.
        {"name": "linear_one", "kind": "linear", "m": 1, "n": 4096, "k": 4096, "dtype": "bf16", "gated": False,
         "bias": False},
        # The same token through the first half of a gated MLP, gate and up in one call.
        {"name": "linear_one_gated", "kind": "linear", "m": 1, "n": 28672, "k": 4096, "dtype": "bf16", "gated": True,
         "bias": False},
        # The token before and five drafted ones of one stream, a depth that is a
        # multiple of 64 only, with a bias.
        {"name": "linear_drafts", "kind": "linear", "m": 6, "n": 5120, "k": 2880, "dtype": "f16", "gated": False,
         "bias": True},
        # The second half of the MLP for a batch of streams.
        {"name": "linear_batch", "kind": "linear", "m": 48, "n": 4096, "k": 14336, "dtype": "bf16", "gated": False,
         "bias": False},
        # A chunk of a prompt, an odd number of tokens, into a vocabulary of odd size.
        {"name": "linear_chunk", "kind": "linear", "m": 777, "n": 11007, "k": 4096, "dtype": "bf16", "gated": False,
         "bias": False},
        # A long prompt through the gated MLP.
        {"name": "linear_prompt", "kind": "linear", "m": 4097, "n": 28672, "k": 4096, "dtype": "bf16", "gated": True,
         "bias": False},
        # One token, 2 of 8 experts, gate and up.
        {"name": "moe_one", "kind": "moe", "tokens": 1, "experts": 8, "topk": 2, "n": 28672, "k": 4096, "dtype": "bf16",
         "gated": True, "down": False, "bias": False},
        # A serving batch over many small experts, f16 with a bias.
        {"name": "moe_fine", "kind": "moe", "tokens": 512, "experts": 64, "topk": 6, "n": 2816, "k": 2048, "dtype": "f16",
         "gated": True, "down": False, "bias": True},
        # A serving batch on the way down, weighted by the router.
        {"name": "moe_down", "kind": "moe", "tokens": 61, "experts": 8, "topk": 2, "n": 4096, "k": 14336, "dtype": "bf16",
         "gated": False, "down": True, "bias": False},
        # A prompt over 2 of 8 experts, gate and up.
        {"name": "moe_prompt", "kind": "moe", "tokens": 2047, "experts": 8, "topk": 2, "n": 28672, "k": 4096,
         "dtype": "bf16", "gated": True, "down": False, "bias": False},
        # One projection's weights.
        {"name": "weights_one", "kind": "weights", "matrices": 1, "n": 4096, "k": 4096, "dtype": "bf16"},
        # The weights of a layer's experts, as they come out of training.
        {"name": "weights_experts", "kind": "weights", "matrices": 8, "n": 14336, "k": 4096, "dtype": "f32"},
    ]


def _spread(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], even over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return min(hi, max(lo, int(round(v / step)) * step))


def draw(rng):
    kind = rng.choice(("linear", "linear", "linear", "moe", "moe", "weights"))
    k = _spread(rng, 256, 14336, 32)
    if kind == "weights":
        return {"kind": kind, "matrices": rng.choice((1, 1, 2, 5, 8)), "n": _spread(rng, 100, 12000), "k": k,
                "dtype": rng.choice(("bf16", "bf16", "f16", "f32"))}
    gated = rng.random() < 0.4
    dtype, bias = rng.choice(("bf16", "bf16", "f16")), rng.random() < 0.3
    if kind == "linear":
        m = rng.choice((1, 1, rng.randint(2, 9), _spread(rng, 10, 250), _spread(rng, 100, 4097), _spread(rng, 1, 4097)))
        n = _spread(rng, 256, 28672, 64) if gated else _spread(rng, 200, 28672)
        m = max(1, min(m, int(_MAX_FLOPS / (2.0 * n * k))))
        return {"kind": kind, "m": m, "n": n, "k": k, "dtype": dtype, "gated": gated, "bias": bias}
    experts = rng.choice((4, 8, 16, 64, 128))
    topk = rng.choice((1, 2, 2, 4, 6, 8)[:4 if experts < 8 else 6])
    n = _spread(rng, 256, 28672 if experts <= 8 else 4096, 64) if gated else _spread(rng, 200, 14336 if experts <= 8 else 4096)
    k = _spread(rng, 256, 14336 if experts <= 8 and n <= 8192 else 4096, 32)
    tokens = rng.choice((1, rng.randint(1, 16), _spread(rng, 10, 300), _spread(rng, 1, 4096)))
    tokens = max(1, min(tokens, int(_MAX_FLOPS / (2.0 * topk * n * k))))
    return {"kind": kind, "tokens": tokens, "experts": experts, "topk": topk, "n": n, "k": k, "dtype": dtype,
            "gated": gated, "down": not gated and rng.random() < 0.5, "bias": bias}


# ---- what a pass cannot do without ----------------------------------------------
def work(case):
    n, k = case["n"], case["k"]
    held = n * k // 2 + n * k // _GROUP
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "weights":
        return {"bytes": case["matrices"] * (2 * n * k * size + 2 * held), "flops": 0}
    cols = n // 2 if case["gated"] else n
    if case["kind"] == "linear":
        m = case["m"]
        return {"bytes": held + 2 * m * (k + cols) + (4 * n if case["bias"] else 0), "flops": 2.0 * m * n * k}
    e, pairs = case["experts"], case["tokens"] * case["topk"]
    used = e * (1 - (1 - case["topk"] / e) ** case["tokens"])      # experts that have rows, were all alike
    rows = pairs if case["down"] else case["tokens"]
    return {"bytes": int(used * held) + 2 * rows * k + 2 * pairs * cols + 8 * pairs, "flops": 2.0 * pairs * n * k}


# ---- what a program has in hand ---------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _activations(g, rows, k, dt):
    """Rows with a few channels that are much larger than the others."""
    gain = 1 + 9 * (torch.rand(k, generator=g, device=DEV) < 0.01)
    return (_randn(g, rows, k) * gain).to(dt)


def _checkpoint(g, n, k):
    """Codes and scales as a quantizer leaves them: the largest of a group has
    code 6 or 7, and the scales lie within a few powers of two."""
    w = _randn(g, n, k // _GROUP, _GROUP) * (0.02 * torch.exp2(2 * _randn(g, n, 1, 1)).clamp(0.1, 10))
    top = torch.frexp(w.abs().amax(-1, keepdim=True))
    power = top.exponent - 3 + (top.mantissa >= 0.875)
    y = torch.ldexp(w.abs(), -power)
    step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0))
    y = (torch.round(y / step) * step).clamp_max(6)
    code = torch.where(y < 2, y * 2, torch.where(y < 4, y + 2, y / 2 + 4)).to(torch.uint8) | ((w < 0).to(torch.uint8) << 3)
    code = code.view(n, k)
    return code[:, ::2] | (code[:, 1::2] << 4), (power.view(n, -1) + 127).to(torch.uint8)


def prepare(case, seed):
    g = _gen(seed)
    state = {"case": case,
             "pairs": torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6], device=DEV)}
    {"weights": _prepare_weights, "linear": _prepare_linear, "moe": _prepare_moe}[case["kind"]](case, g, state)
    low, high = torch.arange(256, device=DEV) & 15, torch.arange(256, device=DEV) >> 4
    state["pairs"] = torch.stack((state["pairs"][low], state["pairs"][high]), 1)
    return state


def _element(case):
    from baracuda_amd import plans
    return {"bf16": plans.ElementKind.Bf16, "f16": plans.ElementKind.F16, "f32": plans.ElementKind.F32}[case["dtype"]]


def _laid_out(case, codes, scales, matrices):
    """The weights in the products' order, once when a program loads them."""
    from baracuda_amd import w4
    plan = w4.W4WeightsPlan.select(w4.W4WeightsDescriptor(case["n"], case["k"], matrices))
    packed = torch.empty(matrices, w4.packed_bytes(case["n"], case["k"]), dtype=torch.uint8, device=DEV)
    plan.pack(codes, scales, packed)
    return packed


def _prepare_weights(case, g, state):
    e, n, k = case["matrices"], case["n"], case["k"]
    w = torch.empty(e, n, k, dtype=_DT[case["dtype"]], device=DEV)
    for i in range(e):
        row = 0.02 * torch.exp2(_randn(g, n, 1)).clamp(0.1, 10)
        w[i] = (_randn(g, n, k) * row).to(w.dtype)
    state.update(w=w)
    if own:
        from baracuda_amd import w4
        state.update(plan=w4.W4WeightsPlan.select(w4.W4WeightsDescriptor(n, k, e, element=_element(case))),
                     packed=torch.empty(e, w4.packed_bytes(n, k), dtype=torch.uint8, device=DEV),
                     values=torch.empty_like(w))


def _workspace(plan):
    return torch.empty(plan.workspace_size(), dtype=torch.uint8, device=DEV)


def _prepare_linear(case, g, state):
    m, n, k, dt = case["m"], case["n"], case["k"], _DT[case["dtype"]]
    codes, scales = _checkpoint(g, n, k)
    state.update(x=_activations(g, m, k, dt), bias=_randn(g, n) if case["bias"] else None)
    if not own:
        state.update(codes=codes, scales=scales)
        return
    from baracuda_amd import w4
    plan = w4.W4LinearPlan.select(w4.W4LinearDescriptor(m, n, k, element=_element(case), gated=case["gated"]))
    state.update(packed=_laid_out(case, codes, scales, 1), plan=plan, workspace=_workspace(plan),
                 out=torch.empty(m, n // 2 if case["gated"] else n, dtype=dt, device=DEV))


def _prepare_moe(case, g, state):
    """Experts drawn for each token, some of them far more often than others."""
    t, e, topk, n, k, dt = case["tokens"], case["experts"], case["topk"], case["n"], case["k"], _DT[case["dtype"]]
    parts = [_checkpoint(g, n, k) for _ in range(e)]
    codes, scales = torch.stack([p[0] for p in parts]), torch.stack([p[1] for p in parts])
    score = torch.randn(t, e, generator=g, device=DEV) + torch.randn(e, generator=g, device=DEV)
    top = torch.topk(score, topk, dim=1)
    ids, order = torch.sort(top.indices.flatten(), stable=True)
    rows = t * topk if case["down"] else t
    state.update(x=_activations(g, rows, k, dt), bias=_randn(g, e, n) if case["bias"] else None,
                 order=order.to(torch.int32), ids=ids.to(torch.int32),
                 mix=torch.softmax(top.values, 1).flatten().contiguous() if case["down"] else None)
    if not own:
        state.update(codes=codes, scales=scales, counts=torch.bincount(ids, minlength=e).tolist())
        return
    from baracuda_amd import w4
    plan = w4.MoeW4GroupedPlan.select(w4.MoeW4GroupedDescriptor(e, topk, t * topk, n, k, element=_element(case),
                                                                gated=case["gated"]))
    state.update(packed=_laid_out(case, codes, scales, e), plan=plan, workspace=_workspace(plan),
                 counts=torch.empty(e, dtype=torch.int32, device=DEV),
                 offsets=torch.empty(e + 1, dtype=torch.int32, device=DEV),
                 out=torch.empty(t * topk, n // 2 if case["gated"] else n, dtype=dt, device=DEV))


# ---- one pass -------------------------------------------------------------------------
def run(state):
    return {"weights": _weights, "linear": _linear, "moe": _moe}[state["case"]["kind"]](state)


def _values(state, codes, scales):
    """float32 [N, K] of a matrix as a checkpoint holds it."""
    n, half = codes.shape
    w = state["pairs"][codes.int()].view(n, -1, _GROUP)
    return torch.ldexp(w, scales.int()[..., None] - 127).view(n, 2 * half)


def _finished(case, y, bias):
    """Bias and gate, in 32 bits."""
    if bias is not None:
        y = y + bias
    if case["gated"]:
        gate, up = y.chunk(2, dim=1)
        y = gate / (1 + torch.exp(-gate)) * up
    return y


def _weights(state):
    w, case = state["w"], state["case"]
    if own:
        state["plan"].quantize(w, state["packed"])
        state["plan"].read(state["packed"], state["values"])
        return state["values"]
    out = torch.empty_like(w)
    for i in range(case["matrices"]):
        x = w[i].float().view(-1, _GROUP)
        top = torch.frexp(x.abs().amax(-1, keepdim=True))
        power = top.exponent - 3 + (top.mantissa >= 0.875)
        y = torch.ldexp(x.abs(), -power)
        step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0))
        y = torch.ldexp((torch.round(y / step) * step).clamp_max(6), power)
        out[i] = torch.where(x < 0, -y, y).view(w.shape[1:]).to(w.dtype)
    return out


def _linear(state):
    x, case = state["x"], state["case"]
    if own:
        state["plan"].run(x, state["packed"], state["out"], bias=state["bias"], workspace=state["workspace"])
        return state["out"]
    y = x.float() @ _values(state, state["codes"], state["scales"]).t()
    return _finished(case, y, state["bias"]).to(x.dtype)


def _moe(state):
    x, case, bias, mix = state["x"], state["case"], state["bias"], state["mix"]
    if own:
        state["plan"].run(x, state["packed"], state["order"], state["ids"], state["out"], state["counts"],
                          state["offsets"], bias=bias, topk_weights=mix, workspace=state["workspace"])
        return state["out"]
    order = state["order"].long()
    source = order if case["down"] else order // case["topk"]
    out = torch.empty(len(order), case["n"] // 2 if case["gated"] else case["n"], dtype=x.dtype, device=DEV)
    at = 0
    for e, count in enumerate(state["counts"]):
        if count:
            pairs = order[at:at + count]
            y = x[source[at:at + count]].float() @ _values(state, state["codes"][e], state["scales"][e]).t()
            y = _finished(case, y, None if bias is None else bias[e])
            out[pairs] = (y if mix is None else y * mix[pairs, None]).to(x.dtype)
            at += count
    return out


# ---- 64-bit arithmetic -------------------------------------------------------------------
def exact(case, seed):
    """On the inputs of prepare(case, seed)."""
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["kind"] == "weights":
        return torch.stack([_exact_nearest(w) for w in s["w"].unbind()]).to(s["w"].dtype)
    if case["kind"] == "linear":
        return _exact_product(case, s["x"], s["codes"], s["scales"], s["bias"])
    out = torch.empty(len(s["ids"]), case["n"] // (2 if case["gated"] else 1), dtype=torch.float64, device=DEV)
    for e in s["ids"].unique().tolist():
        pairs = s["order"][s["ids"] == e].long()
        rows = pairs if case["down"] else torch.div(pairs, case["topk"], rounding_mode="floor")
        out[pairs] = _exact_product(case, s["x"][rows], s["codes"][e], s["scales"][e],
                                    None if s["bias"] is None else s["bias"][e])
    return out if s["mix"] is None else out * s["mix"].double()[:, None]


def _exact_product(case, x, codes, scales, bias):
    """The definition of a code: sign, then the value 2^(e - 1) (1 + m / 2) of two
    exponent bits and a mantissa bit, m / 2 where e is 0."""
    w = torch.empty(codes.shape[0], 2 * codes.shape[1], dtype=torch.float64, device=DEV)
    for i, c in enumerate((codes % 16, codes // 16)):
        e, m = ((c // 2) % 4).double(), (c % 2).double()
        size = torch.where(e == 0, m / 2, torch.exp2(e - 1) * (1 + m / 2))
        w[:, i::2] = torch.where(c >= 8, -size, size)
    w *= torch.exp2(scales.double() - 127).repeat_interleave(_GROUP, dim=1)
    y = torch.matmul(x.double(), w.t())
    if bias is not None:
        y += bias.double()
    if case["gated"]:
        half = y.shape[1] // 2
        y = y[:, :half] * torch.sigmoid(y[:, :half]) * y[:, half:]
    return y


def _exact_nearest(w):
    """The scale is the smallest power of two under which no weight of the group
    reaches 7; codes by the midpoints between them, ties to the even one."""
    x = w.double().view(-1, _GROUP)
    top = x.abs().amax(1, keepdim=True)
    power = torch.floor(torch.log2(top)) - 3
    for _ in range(2):      # the logarithm may be off by a rounding next to a power of two
        power = torch.where(top >= 7 * torch.exp2(power), power + 1, power)
    y = x.abs() / torch.exp2(power)
    low = torch.tensor([.25, 1.25, 2.5, 5], dtype=torch.float64, device=DEV)       # a tie stays below these
    high = torch.tensor([.75, 1.75, 3.5], dtype=torch.float64, device=DEV)         # and goes above these
    value = torch.zeros_like(y)
    for point, step in ((low[0], .5), (low[1], .5), (low[2], 1.), (low[3], 2.)):
        value += step * (y > point)
    for point, step in ((high[0], .5), (high[1], .5), (high[2], 1.)):
        value += step * (y >= point)
    return (torch.sign(x) * value * torch.exp2(power)).view(w.shape)
