"""Cases of the operators around a key-value cache held in 4 bits.

A case is a dict of plain values; `kind` names the operator and the other keys
its sizes and options:
  qk      RMS norm of each head of Q and K and the position rotation, one pass
  append  the same, then K and V quantized to 4 bits into pages of the cache,
          and the values that the pages now stand for read back
  attn    attention of a batch of ragged sequences over such pages
  pages   copying, forking, releasing and compacting pages
`listed()` holds the fixed cases, `draw()` more of the same ranges, `prepare()`
what a serving program holds before the call, `run()` one pass, `work()` the
bytes and operations that a pass cannot do without, and `exact()` the result in
64-bit arithmetic.

The cache: uint8 [pages, kv heads, head bytes], two codes a byte, the lower
index in the lower four bits.  A code is sign, two exponent bits and one
mantissa bit (0, 0.5, 1, 1.5, 2, 3, 4, 6); 32 consecutive values of a head
share a scale 2^(byte - 127).  The head bytes of a page of PS tokens and a head
of D values, in order:
  K codes   [PS][D / 2]
  V codes   [PS / 4][16][4][D / 32]  (four tokens together; 16 runs of D / 16 values)
  K scales  [PS][D / 32]
  V scales  [PS / 4][D / 32][4]
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda:0"
_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_GROUP = 32      # values that share a scale
_MAX_POS = 40960  # rows of the rotation table


def listed():
    return [
        # One new token of one stream: norms of 32 + 8 heads and the rotation.
        {"name": "qk_one", "kind": "qk", "t": 1, "hq": 32, "hk": 8, "d": 128, "rope": 128, "axes": 1,
         "interleaved": False, "dtype": "bf16"},
        # A prompt with images in it: an odd number of tokens, positions in
        # time, height and width.
        {"name": "qk_image", "kind": "qk", "t": 6145, "hq": 32, "hk": 8, "d": 128, "rope": 128, "axes": 3,
         "interleaved": False, "dtype": "bf16"},
        # The new tokens of 48 streams go into the cache.
        {"name": "append_step", "kind": "append", "t": 48, "hq": 32, "hk": 8, "d": 128, "rope": 128, "axes": 1,
         "interleaved": False, "dtype": "bf16", "ps": 64},
        # A long prompt goes into the cache: wide heads that are rotated in part,
        # neighbouring values in pairs.
        {"name": "append_prompt", "kind": "append", "t": 8191, "hq": 16, "hk": 2, "d": 256, "rope": 64, "axes": 1,
         "interleaved": True, "dtype": "f16", "ps": 16},
        # One stream's next token after a page and a half of text.
        {"name": "attn_one", "kind": "attn", "b": 1, "q": 1, "kv": 777, "hq": 32, "hk": 8, "d": 128, "ps": 16,
         "window": 0, "dtype": "bf16"},
        # The next tokens of a batch of chats of very different lengths.
        {"name": "attn_batch", "kind": "attn", "b": 48, "q": 1, "kv": 8192, "hq": 32, "hk": 8, "d": 128, "ps": 64,
         "window": 0, "dtype": "bf16"},
        # Two streams with whole books before them.
        {"name": "attn_long", "kind": "attn", "b": 2, "q": 1, "kv": 200001, "hq": 64, "hk": 8, "d": 128, "ps": 64,
         "window": 0, "dtype": "bf16"},
        # Drafted tokens checked, five a stream, by heads in groups of five that
        # look back over a window.
        {"name": "attn_draft", "kind": "attn", "b": 24, "q": 5, "kv": 5000, "hq": 40, "hk": 8, "d": 64, "ps": 32,
         "window": 1024, "dtype": "f16"},
        # Chunks of prompts after what earlier chunks left in the cache.
        {"name": "attn_prompt", "kind": "attn", "b": 3, "q": 2047, "kv": 6000, "hq": 32, "hk": 8, "d": 128, "ps": 64,
         "window": 0, "dtype": "bf16"},
        # Pages that two streams share are copied before one of them writes.
        {"name": "pages_copy", "kind": "pages", "op": "copy", "layers": 32, "pages": 2000, "page_bytes": 17408,
         "n": 7, "rows": 48, "ps": 16},
        # Sixteen samples of one prompt are begun, and given back.
        {"name": "pages_fork", "kind": "pages", "op": "fork", "layers": 32, "pages": 700, "page_bytes": 69632,
         "n": 16, "rows": 48, "ps": 64},
        # The pages in use are moved to the front, a third of the cache in use.
        {"name": "pages_compact", "kind": "pages", "op": "compact", "layers": 32, "pages": 1200,
         "page_bytes": 34816, "n": 400, "rows": 48, "ps": 32},
    ]


def _spread(rng, lo, hi):
    """A size between lo and hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("qk", "append", "attn", "attn", "attn", "pages"))
    if kind == "pages":
        op = rng.choice(("copy", "fork", "compact"))
        ps = rng.choice((16, 32, 64))
        pages = _spread(rng, 64, 1200)
        return {"kind": kind, "op": op, "layers": rng.randint(1, 32), "pages": pages,
                "page_bytes": ps * rng.choice((68, 136, 544, 1088)), "n": rng.randint(1, max(1, pages // 3)) if op != "fork"
                else rng.randint(1, 16), "rows": 48, "ps": ps}
    d = rng.choice((64, 128, 128, 256))
    hk = rng.choice((1, 2, 4, 5, 8))
    hq = hk * rng.choice((1, 2, 4, 5, 7, 8))
    if kind in ("qk", "append"):
        case = {"kind": kind, "t": _spread(rng, 1, 8000), "hq": hq, "hk": hk, "d": d,
                "rope": rng.choice((d, d, d // 2, 0)), "axes": rng.choice((1, 1, 3)), "interleaved": rng.random() < 0.3,
                "dtype": rng.choice(("bf16", "bf16", "f16", "f32") if kind == "qk" else ("bf16", "bf16", "f16"))}
        return dict(case, ps=rng.choice((16, 32, 64, 128))) if kind == "append" else case
    q = rng.choice((1, 1, rng.randint(2, 9), _spread(rng, 16, 1500)))
    b = _spread(rng, 1, 40) if q < 16 else rng.randint(1, 3)
    return {"kind": kind, "b": b, "q": q, "kv": _spread(rng, 1, 16000 if b <= 8 else 6000), "hq": hq, "hk": hk, "d": d,
            "ps": rng.choice((16, 32, 64, 128)), "window": rng.choice((0, 0, 0, rng.randint(1, 4096))),
            "dtype": rng.choice(("bf16", "bf16", "f16"))}


# ---- the sizes that go by the case alone ------------------------------------
def _lengths(case):
    """New tokens and tokens in the cache (the new ones among them) of each
    sequence; the first is the longest."""
    r = random.Random(case["b"] * 1000003 + case["kv"])
    q = [case["q"]] + [case["q"] if case["q"] < 16 else r.randint(1, case["q"]) for _ in range(case["b"] - 1)]
    return q, [max(case["kv"], q[0])] + [max(_spread(r, 1, case["kv"]), n) for n in q[1:]]


def _head_bytes(case):
    return case["ps"] * (case["d"] + case["d"] // 16)


def _fork_lengths(case):
    """Tokens in the rows that are forked: n forks of one prompt in two."""
    r = random.Random(case["pages"])
    most = max(1, (case["pages"] - case["n"]) // 4)
    return [r.randint(1, most * case["ps"]) for _ in range(2)]


def work(case):
    kind = case["kind"]
    if kind == "pages":
        if case["op"] == "fork":
            copies = case["n"] if all(x % case["ps"] for x in _fork_lengths(case)) else case["n"] // 2
        elif case["op"] == "copy":
            copies = case["n"]
        else:   # of n pages in use anywhere, this share lies past the first n
            copies = case["n"] * (case["pages"] - case["n"]) / case["pages"]
        return {"bytes": 2 * copies * case["layers"] * case["page_bytes"] + 8 * case["pages"], "flops": 0}
    d, hq, hk = case["d"], case["hq"], case["hk"]
    if kind == "attn":
        q, kv = _lengths(case)
        pairs = tokens = 0
        for n, m in zip(q, kv):
            w = case["window"] or m + n
            pairs += sum(min(x + 1, w) for x in range(m - n, m))
            tokens += min(m, w + n - 1)
        return {"bytes": tokens * hk * (d + d // 16) + 4 * sum(q) * hq * d, "flops": 4 * pairs * hq * d}
    size = 4 if case["dtype"] == "f32" else 2
    rot = case["t"] * case["rope"] * 4
    if kind == "qk":
        return {"bytes": case["t"] * (hq + hk) * d * 2 * size + rot, "flops": 8 * case["t"] * (hq + hk) * d}
    held = case["t"] * hk * (d + d // 16)
    return {"bytes": case["t"] * (2 * hq + 2 * hk) * d * size + rot + 2 * held + 2 * case["t"] * hk * d * size,
            "flops": 10 * case["t"] * (hq + 2 * hk) * d}


# ---- what a program has in hand ----------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _perm(g, n):
    return torch.randperm(n, generator=g, device=DEV)


def prepare(case, seed):
    g = _gen(seed)
    state = {"case": case, "levels": torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6],
                                                  device=DEV)}
    {"qk": _prepare_tokens, "append": _prepare_tokens, "attn": _prepare_attn, "pages": _prepare_pages}[case["kind"]](
        case, g, state)
    return state


def _prepare_tokens(case, g, state):
    """The rows of a fused projection (Q, K and V side by side), the norms'
    weights, the rotation table, positions and, for the cache, its pages and the
    tokens' places in them."""
    t, hq, hk, d, dt = case["t"], case["hq"], case["hk"], case["d"], _DT[case["dtype"]]
    # projections have channels that are much larger than the others
    gain = 1 + 6 * (torch.rand((hq + 2 * hk) * d, generator=g, device=DEV) < 0.02)
    row = (_randn(g, t, (hq + 2 * hk) * d) * gain).to(dt).view(t, hq + 2 * hk, d)
    state.update(q=row[:, :hq], k=row[:, hq:hq + hk], v=row[:, hq + hk:],
                 q_weight=(1 + 0.2 * _randn(g, d)).to(dt), k_weight=(1 + 0.2 * _randn(g, d)).to(dt),
                 q_out=torch.empty(t, hq, d, dtype=dt, device=DEV), k_out=torch.empty(t, hk, d, dtype=dt, device=DEV),
                 positions=None, cos=None, sin=None, pair_axis=None)
    if case["rope"]:
        half, axes = case["rope"] // 2, case["axes"]
        inv = 1e6 ** (-torch.arange(half, dtype=torch.float64, device=DEV) / half)
        angle = torch.arange(_MAX_POS, dtype=torch.float64, device=DEV)[:, None] * inv
        start = torch.randint(0, _MAX_POS - t, (axes, 1), generator=g, device=DEV)
        walk = torch.arange(t, device=DEV) if axes == 1 else torch.randint(0, t, (axes, t), generator=g, device=DEV)
        state.update(cos=angle.cos().float(), sin=angle.sin().float(), positions=(start + walk).view(axes, t).to(torch.int32))
        if axes > 1:   # time for the first quarter of the pairs, then height, then width
            share = torch.arange(half, device=DEV) * 8
            state["pair_axis"] = ((share >= 2 * half).int() + (share >= 5 * half).int())
    if case["kind"] == "append":
        ps = case["ps"]
        pages = -(-t // ps) + 3
        state["cache"] = torch.zeros(pages, hk, _head_bytes(case), dtype=torch.uint8, device=DEV)
        if t <= 256:   # a step: each stream's token in a page of its own stream
            state["slots"] = _perm(g, pages * ps)[:t].contiguous()
        else:          # a prompt: page after page, the pages in any order
            at = torch.arange(t, device=DEV)
            state["slots"] = _perm(g, pages)[at // ps] * ps + at % ps
        state.update(k_read=torch.empty(t, hk, d, dtype=dt, device=DEV), v_read=torch.empty(t, hk, d, dtype=dt, device=DEV))


def _prepare_attn(case, g, state):
    """A cache in use: pages of the sequences in any order, tables, lengths and
    the new tokens' queries."""
    b, hq, hk, d, ps, dt = case["b"], case["hq"], case["hk"], case["d"], case["ps"], _DT[case["dtype"]]
    q, kv = _lengths(case)
    need = [-(-n // ps) for n in kv]
    pages = sum(need) + 5
    state["cache"] = cache = torch.empty(pages, hk, _head_bytes(case), dtype=torch.uint8, device=DEV)
    gain = 1 + 3 * (torch.rand(hk, 1, d, generator=g, device=DEV) < 0.03)
    _store(cache, _randn(g, pages, hk, ps, d) * gain, _randn(g, pages, hk, ps, d), case)
    at = torch.cumsum(torch.tensor([0] + need), 0)
    j = torch.arange(max(need))[None, :]
    order = _perm(g, pages).cpu()
    tables = torch.where(j < torch.tensor(need)[:, None], order[(at[:-1, None] + j).clamp(max=pages - 1)], -1)
    state.update(tables=tables.to(torch.int32).to(DEV), kv_lens=torch.tensor(kv, dtype=torch.int32, device=DEV),
                 cu_q=torch.cumsum(torch.tensor([0] + q), 0).to(torch.int32).to(DEV),
                 q=(_randn(g, sum(q), hq, d) * 1.5).to(dt), out=torch.empty(sum(q), hq, d, dtype=dt, device=DEV),
                 max_q=max(q), max_kv=max(kv), scale=d ** -0.5)


def _prepare_pages(case, g, state):
    layers, pages, size, n, rows, ps = (case[x] for x in ("layers", "pages", "page_bytes", "n", "rows", "ps"))
    state["cache"] = torch.randint(0, 256, (layers, pages, size), generator=g, device=DEV, dtype=torch.uint8)
    order = _perm(g, pages).to(torch.int32)
    if case["op"] == "copy":
        state.update(src=order[:n].contiguous(), dst=order[n:2 * n].contiguous())
        return
    width = pages
    tables = torch.full((rows, width), -1, dtype=torch.int32, device=DEV)
    lens = torch.zeros(rows, dtype=torch.int32, device=DEV)
    refs = torch.zeros(pages, dtype=torch.int32, device=DEV)
    if case["op"] == "fork":
        first, second = _fork_lengths(case)
        k, m = -(-first // ps), -(-second // ps)
        tables[0, :k], tables[1, :m] = order[:k], order[k:k + m]
        lens[0], lens[1] = first, second
        refs[order[:k + m].long()] = 1
        i = torch.arange(n, device=DEV, dtype=torch.int32)
        state.update(parents=i % 2, children=2 + i, rows=2 + i, fresh=torch.empty(n, dtype=torch.int32, device=DEV))
    else:   # n pages in use: the first one is every row's, the others belong to the rows in turn
        i = torch.arange(n - 1, device=DEV)
        tables[:, 0] = order[0]
        tables[i % rows, 1 + i // rows] = order[1:n]
        flat = tables[tables >= 0].long()
        refs += torch.bincount(flat, minlength=pages).to(torch.int32)
        state.update(tables_out=torch.empty_like(tables), refs_out=torch.empty_like(refs), remap=torch.empty_like(refs),
                     live=torch.empty(1, dtype=torch.int32, device=DEV))
    state.update(tables=tables, lens=lens, refs=refs)


# ---- one pass ------------------------------------------------------------------
def run(state):
    return {"qk": _qk, "append": _append, "attn": _attn, "pages": _pages}[state["case"]["kind"]](state)


def _plan(state, name, cls, descriptor, **sizes):
    """The plan that a program keeps for its sizes."""
    if name not in state:
        state[name] = cls.select(descriptor(**sizes))
    return state[name]


def _element(case):
    from baracuda_amd.plans import ElementKind
    return {"bf16": ElementKind.Bf16, "f16": ElementKind.F16, "f32": ElementKind.F32}[case["dtype"]]


def _rotation(state):
    return {k: state[k] for k in ("q_weight", "k_weight", "positions", "cos", "sin", "pair_axis")}


def _qk(state):
    c = state["case"]
    if own:
        from baracuda_amd import kv4
        plan = _plan(state, "plan", kv4.QkNormRopePlan, kv4.QkNormRopeDescriptor, tokens=c["t"], num_heads=c["hq"],
                     num_kv_heads=c["hk"], head_dim=c["d"], rope_dim=c["rope"], element=_element(c),
                     axes=c["axes"], interleaved=c["interleaved"], eps=1e-6)
        plan.run(state["q"], state["k"], state["q_out"], state["k_out"], **_rotation(state))
        return state["q_out"], state["k_out"]
    return _norm_rope(state, state["q"], state["q_weight"]), _norm_rope(state, state["k"], state["k_weight"])


def _norm_rope(state, x, weight):
    """In 64 bits: K is quantized from this, and values next to a border between
    two codes have to fall on the same side."""
    c, y = state["case"], x.double()
    y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + 1e-6) * weight.double()
    rope = c["rope"]
    if rope:
        pos, half = state["positions"].long(), torch.arange(rope // 2, device=DEV)
        axis = torch.zeros_like(half) if state["pair_axis"] is None else state["pair_axis"].long()
        row = pos[axis].T                                       # [T, pairs]
        cos, sin = (state[n][row, half].double()[:, None] for n in ("cos", "sin"))
        if c["interleaved"]:
            a, b = y[..., 0:rope:2], y[..., 1:rope:2]
            turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        else:
            a, b = y[..., :rope // 2], y[..., rope // 2:rope]
            turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        y = torch.cat((turned, y[..., rope:]), -1)
    return y.to(x.dtype)


def _codes(x, most):
    """Codes (one a byte) and scale bytes of x [..., D]: the scale is the power of
    two that brings the group's largest value below 7 (to 6 with the rounding),
    2^most at most; a group with an infinity or a NaN gets the scale 255."""
    y = x.float().unflatten(-1, (-1, _GROUP))
    top = y.abs().amax(-1)
    byte = (((top.view(torch.int32) + 0x200000) >> 23) - 2).clamp(2, most + 127)
    a = y * ((254 - byte) << 23).view(torch.float32)[..., None]
    m = a.abs()
    code = ((m > 0.25).to(torch.uint8) + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5) + (m > 5))
    code += 8 * torch.signbit(a)
    good = torch.isfinite(top)
    return (code * good[..., None]).flatten(-2), torch.where(good, byte, 255).to(torch.uint8)


def _parts(cache, case):
    """Views of the pages' K codes, V codes, K scales and V scales."""
    ps, d = case["ps"], case["d"]
    lead, half, few = cache.shape[:-1], ps * d // 2, ps * d // 32
    cut = cache.split((half, half, few, few), -1)
    return (cut[0].view(*lead, ps, d // 2), cut[1].view(*lead, ps // 4, 16, 4, d // 32),
            cut[2].view(*lead, ps, d // 32), cut[3].view(*lead, ps // 4, d // 32, 4))


def _most(case):
    """The largest scale's exponent: six times it has to be a number of the type."""
    return 13 if case["dtype"] == "f16" else 125


def _packed(x, case):
    code, scale = _codes(x, _most(case))
    return code[..., 0::2] | code[..., 1::2] << 4, scale


def _store(cache, k, v, case):
    """Whole pages: k and v [pages, heads, PS, D]."""
    kc, vc, ks, vs = _parts(cache, case)
    code, scale = _packed(k, case)
    kc.copy_(code)
    ks.copy_(scale)
    code, scale = _packed(v, case)
    vc.copy_(code.view(*code.shape[:2], case["ps"] // 4, 4, 16, -1).transpose(3, 4))
    vs.copy_(scale.view(*scale.shape[:2], case["ps"] // 4, 4, -1).transpose(3, 4))


def _values(code, scale, levels):
    """What packed codes [..., D / 2] and scales [..., D / 32] stand for, in 32 bits."""
    c = torch.stack((code & 15, code >> 4), -1).flatten(-2)
    size = (scale.int() << 23).view(torch.float32)
    size = torch.where(scale == 255, math.nan, size)
    return (levels[c.int()].unflatten(-1, (-1, _GROUP)) * size[..., None]).flatten(-2)


def _append(state):
    c, cache, slots = state["case"], state["cache"], state["slots"]
    if own:
        from baracuda_amd import kv4
        plan = _plan(state, "plan", kv4.Kv4AppendPlan, kv4.Kv4AppendDescriptor, tokens=c["t"], num_heads=c["hq"],
                     num_kv_heads=c["hk"], head_dim=c["d"], page_size=c["ps"], num_pages=cache.shape[0],
                     rope_dim=c["rope"], element=_element(c), axes=c["axes"], interleaved=c["interleaved"], eps=1e-6)
        back = _plan(state, "back", kv4.Kv4ReadPlan, kv4.Kv4ReadDescriptor, tokens=c["t"], num_kv_heads=c["hk"],
                     head_dim=c["d"], page_size=c["ps"], num_pages=cache.shape[0], element=_element(c))
        plan.run(state["k"], state["v"], cache, slots, q=state["q"], q_out=state["q_out"], **_rotation(state))
        back.run(cache, slots, state["k_read"], state["v_read"])
        return state["q_out"], state["k_read"], state["v_read"]
    q, k = _norm_rope(state, state["q"], state["q_weight"]), _norm_rope(state, state["k"], state["k_weight"])
    kc, vc, ks, vs = _parts(cache, c)
    page, off = slots // c["ps"], slots % c["ps"]
    kc[page, :, off], ks[page, :, off] = _packed(k, c)
    code, scale = _packed(state["v"], c)
    vc[page, :, off // 4, :, off % 4] = code.unflatten(-1, (16, -1))
    vs[page, :, off // 4, :, off % 4] = scale
    return (q, _values(kc[page, :, off], ks[page, :, off], state["levels"]).to(q.dtype),
            _values(vc[page, :, off // 4, :, off % 4].flatten(-2), vs[page, :, off // 4, :, off % 4],
                    state["levels"]).to(q.dtype))


def _attn(state):
    c, cache, tables, lens, cu, q = (state[x] for x in ("case", "cache", "tables", "kv_lens", "cu_q", "q"))
    if own:
        from baracuda_amd import kv4
        plan = _plan(state, "plan", kv4.Kv4AttentionPlan, kv4.Kv4AttentionDescriptor, num_seqs=c["b"],
                     total_q=q.shape[0], max_q=state["max_q"], max_kv=state["max_kv"], num_heads=c["hq"],
                     num_kv_heads=c["hk"], head_dim=c["d"], page_size=c["ps"], num_pages=cache.shape[0],
                     max_pages=tables.shape[1], element=_element(c), causal=True, window=c["window"],
                     scale=state["scale"])
        if "workspace" not in state:
            state["workspace"] = torch.empty(plan.workspace_size(), dtype=torch.uint8, device=DEV)
        plan.run(q, cache, tables, lens, state["out"], cu_q=cu, workspace=state["workspace"])
        return state["out"]
    b, hq, hk, d, ps = c["b"], c["hq"], c["hk"], c["d"], c["ps"]
    n, top = state["max_q"], tables.shape[1] * ps
    kc, vc, ks, vs = _parts(cache[tables.long().clamp(min=0)], c)          # [B, pages, Hk, ...]
    k = _values(kc, ks, state["levels"]).transpose(1, 2).reshape(b * hk, top, d)
    vc = vc.transpose(-3, -2).reshape(*vc.shape[:3], ps, d // 2)
    vs = vs.transpose(-2, -1).reshape(*vs.shape[:3], ps, d // 32)
    v = _values(vc, vs, state["levels"]).transpose(1, 2).reshape(b * hk, top, d)
    i = torch.arange(n, device=DEV)
    cu = cu.long()
    rows = (cu[:-1, None] + i).clamp(max=q.shape[0] - 1)                   # [B, n]
    qs = q[rows].float().view(b, n, hk, hq // hk, d).permute(0, 2, 1, 3, 4).reshape(b * hk, n * (hq // hk), d)
    s = torch.matmul(qs, k.transpose(1, 2)).view(b, hk, n, hq // hk, top) * state["scale"]
    j = torch.arange(top, device=DEV)
    here = (lens.long() - (cu[1:] - cu[:-1]))[:, None] + i                  # positions of the new tokens
    seen = (j <= here[..., None]) & (j < lens[:, None, None])
    if c["window"]:
        seen &= j > here[..., None] - c["window"]
    seen = seen[:, None, :, None]                                          # [B, 1, n, 1, top]
    s = torch.where(seen, s, -math.inf)
    s = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e30))
    total = s.sum(-1, keepdim=True)
    s = s / torch.where(total > 0, total, 1.0)
    o = torch.matmul(s.view(b * hk, n * (hq // hk), top), v)
    o = o.view(b, hk, n, hq // hk, d).transpose(1, 2).reshape(b, n, hq, d)
    at = torch.arange(q.shape[0], device=DEV)
    seq = torch.searchsorted(cu, at, right=True) - 1
    return o[seq, at - cu[seq]].to(q.dtype)


def _pages(state):
    c, cache = state["case"], state["cache"]
    if own:
        return _pages_own(state)
    if c["op"] == "copy":
        cache[:, state["dst"].long()] = cache[:, state["src"].long()]
        return cache
    tables, lens, refs = (state[x] for x in ("tables", "lens", "refs"))
    if c["op"] == "fork":
        fresh = _fork(c, cache, tables, lens, refs, state["parents"].long(), state["children"].long())
        begun = tables.clone(), lens.clone(), refs.clone()
        mine = tables[state["rows"].long()].long().flatten()
        refs.index_add_(0, mine.clamp(min=0), -(mine >= 0).to(torch.int32))
        tables[state["rows"].long()] = -1
        lens[state["rows"].long()] = 0
        return cache, fresh, begun, tables, lens, refs
    live = refs > 0
    count = live.sum(dtype=torch.int32)
    at = torch.arange(c["pages"], device=DEV, dtype=torch.int32)
    high, hole = torch.nonzero(live & (at >= count))[:, 0], torch.nonzero(~live & (at < count))[:, 0]
    remap = torch.where(live, at, -1)
    remap[high] = hole.to(torch.int32)
    cache[:, hole] = cache[:, high]
    moved = torch.zeros_like(refs)
    moved[remap[live].long()] = refs[live]
    entries = torch.where(tables >= 0, remap[tables.long().clamp(min=0)], -1)
    return cache, entries, moved, remap, count[None]


def _fork(c, cache, tables, lens, refs, parents, children):
    """Each child shares its parent's full pages and gets a copy of the last,
    partly filled one in the lowest page that is free."""
    ps = c["ps"]
    n, full, part = lens[parents], lens[parents] // ps, lens[parents] % ps > 0
    free = torch.cumsum(refs == 0, 0)                                       # pages that are free up to here
    rank = torch.cumsum(part, 0)
    fresh = torch.where(part, torch.searchsorted(free, rank), -1).to(torch.int32)
    j = torch.arange(tables.shape[1], device=DEV)
    old = tables[parents]
    shared = j < full[:, None]
    tables[children] = torch.where(shared, old, torch.where((j == full[:, None]) & part[:, None], fresh[:, None], -1))
    lens[children] = n
    refs.index_add_(0, old.clamp(min=0).long().flatten(), shared.flatten().to(torch.int32))
    refs.index_add_(0, fresh.clamp(min=0).long(), part.to(torch.int32))
    last = old.gather(1, full[:, None].long())[:, 0]
    # a child that needs no page copies the page onto itself
    cache[:, torch.where(part, fresh, old[:, 0]).long()] = cache[:, torch.where(part, last, old[:, 0]).long()]
    return fresh


def _pages_own(state):
    from baracuda_amd import kv4
    c, cache = state["case"], state["cache"]
    plan = _plan(state, "plan", kv4.KvPagesPlan, kv4.KvPagesDescriptor, layers=c["layers"], num_pages=c["pages"],
                 page_bytes=c["page_bytes"], page_size=c["ps"], rows=c["rows"], max_pages=c["pages"])
    if c["op"] == "copy":
        plan.copy(cache, state["src"], state["dst"])
        return cache
    tables, lens, refs = (state[x] for x in ("tables", "lens", "refs"))
    if c["op"] == "fork":
        plan.fork(cache, tables, lens, refs, state["parents"], state["children"], state["fresh"])
        begun = tables.clone(), lens.clone(), refs.clone()
        plan.release(tables, lens, refs, state["rows"])
        return cache, state["fresh"], begun, tables, lens, refs
    if "workspace" not in state:
        state["workspace"] = torch.empty(plan.workspace_size(), dtype=torch.uint8, device=DEV)
    plan.compact(cache, tables, refs, state["tables_out"], state["refs_out"], state["remap"], state["live"],
                 workspace=state["workspace"])
    return cache, state["tables_out"], state["refs_out"], state["remap"], state["live"]


# ---- the same in 64 bits, from the definitions ----------------------------------
def exact(case, seed):
    if case["kind"] == "pages":
        return None        # whole numbers only
    s = prepare(case, seed)
    if case["kind"] == "attn":
        return _exact_attn(case, s)
    turned = [_exact_turn(case, s, s[x], s[x + "_weight"]) for x in ("q", "k")]
    if case["kind"] == "qk":
        return tuple(turned)
    dt = _DT[case["dtype"]]
    return turned[0], _exact_nearest(turned[1].to(dt), case), _exact_nearest(s["v"], case)


def _exact_turn(case, s, x, weight):
    """The norm, then each pair as a complex number times e^(i angle)."""
    x = x.to(torch.float64)
    y = x * weight.to(torch.float64) * torch.rsqrt((x * x).sum(-1, keepdim=True) / case["d"] + 1e-6)
    rope = case["rope"]
    if not rope:
        return y
    axes = [0] * (rope // 2) if s["pair_axis"] is None else s["pair_axis"].tolist()
    rows = [s["positions"][a].long() for a in axes]
    turn = torch.stack([torch.complex(s["cos"][r, p].double(), s["sin"][r, p].double()) for p, r in enumerate(rows)], -1)
    turn = turn[:, None]
    first, second = (slice(0, rope, 2), slice(1, rope, 2)) if case["interleaved"] else (
        slice(0, rope // 2), slice(rope // 2, rope))
    z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * turn
    y = y.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_nearest(x, case):
    """Each group's values as the nearest of the fifteen that its scale allows,
    of two as near the one with the even code."""
    y = x.to(torch.float64).unflatten(-1, (-1, _GROUP))
    top = y.abs().amax(-1, keepdim=True)
    mantissa, exponent = torch.frexp(top)           # top = mantissa 2^exponent, mantissa in [0.5, 1)
    power = exponent.double() - 3 + (mantissa >= 0.875)
    size = torch.exp2(torch.where(top > 0, power, -125.0).clamp(-125, _most(case)))
    levels = torch.tensor([0, 1, 2, 4, .5, 1.5, 3, 6], dtype=torch.float64, device=DEV)
    off = ((y / size).abs()[..., None] - levels).abs()
    off[..., 4:] += 1e-9          # the odd codes lose a tie
    best = levels[off.argmin(-1)]
    return (torch.copysign(best, y) * size).flatten(-2)


def _exact_side(code, scale):
    """Packed codes and scale bytes to 64-bit values by the format's formula."""
    c = torch.stack((code % 16, code // 16), -1).flatten(-2).double()
    sign, c = 1 - 2 * (c >= 8).double(), c % 8
    e, m = torch.div(c, 2, rounding_mode="floor"), c % 2
    value = sign * torch.where(e == 0, 0.5 * m, (1 + 0.5 * m) * torch.exp2(e - 1))
    return value * torch.exp2(scale.double() - 127).repeat_interleave(_GROUP, -1)


def _exact_attn(case, s):
    return torch.cat([_exact_rows(case, s, b) for b in range(case["b"])])


def _exact_rows(case, s, b):
    """One sequence, head after head."""
    hk, d, ps = case["hk"], case["d"], case["ps"]
    half, few = ps * d // 2, ps * d // 32
    n, m = int(s["cu_q"][b + 1] - s["cu_q"][b]), int(s["kv_lens"][b])
    need = -(-m // ps)
    q = s["q"][int(s["cu_q"][b]):int(s["cu_q"][b + 1])].double()
    pos = torch.arange(n, device=DEV) + m - n
    j = torch.arange(m, device=DEV)
    hidden = (j > pos[:, None]) | (j <= pos[:, None] - (case["window"] or m + n + 1))

    def group(h):
        x = s["cache"][s["tables"][b, :need].long(), h]
        k = _exact_side(x[:, :half].reshape(need * ps, d // 2), x[:, 2 * half:2 * half + few].reshape(need * ps, -1))
        v = _exact_side(x[:, half:2 * half].reshape(need, ps // 4, 16, 4, d // 32).transpose(2, 3).reshape(need * ps, -1),
                        x[:, 2 * half + few:].reshape(need, ps // 4, d // 32, 4).transpose(2, 3).reshape(need * ps, -1))
        return k[:m], v[:m]

    def head(r, k, v):
        return torch.softmax((q[:, r] @ k.T * s["scale"]).masked_fill(hidden, -math.inf), -1) @ v

    ratio = case["hq"] // hk
    return torch.stack([head(h * ratio + r, *kv) for h in range(hk) for kv in (group(h),) for r in range(ratio)], 1)
