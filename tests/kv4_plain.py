"""The operators around a 4-bit key-value cache in plain 64-bit arithmetic, on
the CPU, one token at a time where that is the simplest."""
import math

import torch

LEVELS = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def half_step(dtype) -> float:
    """The largest relative error of a rounding to `dtype`."""
    return torch.finfo(dtype).eps / 2


def most(dtype) -> int:
    return 13 if dtype == torch.float16 else 125


def norm_rope(x, w, eps, rope, positions, cos, sin, axis_of, interleaved):
    """x [T, H, D] -> (the rotated heads, the magnitudes |a cos| + |b sin| that bound their error)."""
    y = x.double()
    if w is not None:
        y = y * w.double() / torch.sqrt((y * y).mean(-1, keepdim=True) + eps)
    out, size = y.clone(), y.abs()
    for p in range(rope // 2):
        i, j = (2 * p, 2 * p + 1) if interleaved else (p, p + rope // 2)
        row = positions[axis_of[p]].long()
        c, s = cos[row, p].double()[:, None], sin[row, p].double()[:, None]
        out[..., i] = y[..., i] * c - y[..., j] * s
        out[..., j] = y[..., j] * c + y[..., i] * s
        size[..., i] = (y[..., i] * c).abs() + (y[..., j] * s).abs()
        size[..., j] = (y[..., j] * c).abs() + (y[..., i] * s).abs()
    return out, size


def encode(x, top_exponent):
    """x [..., D] -> codes [..., D], scale bytes [..., D / 32]."""
    g = x.double().unflatten(-1, (-1, 32))
    top = g.abs().amax(-1)
    good = torch.isfinite(g).all(-1)
    g = torch.where(good[..., None], g, 0.0)
    top = torch.where(good, top, 1.0)
    e = torch.full_like(top, -125.0)
    while True:                       # the least power that brings the group below 7
        small = (top >= 7 * torch.exp2(e)) & (e < top_exponent)
        if not small.any():
            break
        jump = torch.floor(torch.log2(torch.where(small, top / (7 * torch.exp2(e)), 1.0))).clamp(min=0)
        e = torch.where(small, torch.minimum(e + torch.where(jump > 1, jump - 1, 1.0), torch.tensor(float(top_exponent)).double()), e)
    a = (g / torch.exp2(e)[..., None]).abs().clamp(max=6.0)
    far = (a[..., None] - LEVELS).abs()
    far[..., 1::2] += 1e-12           # ties to the even code
    code = far.argmin(-1) + 8 * torch.signbit(g)
    code = torch.where(good[..., None], code, 0)
    byte = torch.where(good, e + 127, 255.0)
    return code.flatten(-2).to(torch.uint8), byte.to(torch.uint8)


def decode(code, byte):
    c = code.long()
    v = LEVELS[c % 8] * torch.where(c >= 8, -1.0, 1.0).double()
    s = torch.exp2(byte.double() - 127)
    s = torch.where(byte == 255, math.nan, s)
    return (v.unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)


def places(ps, d):
    """Byte offsets in a head of a page: K codes [PS, D/2], V codes [PS, D/2],
    K scales [PS, D/32], V scales [PS, D/32]."""
    t = torch.arange(ps)[:, None]
    b = torch.arange(d // 2)[None, :]
    run, within = b // (d // 32), b % (d // 32)
    k = t * (d // 2) + b
    v = ps * d // 2 + ((t // 4 * 16 + run) * 4 + t % 4) * (d // 32) + within
    g = torch.arange(d // 32)[None, :]
    ks = ps * d + t * (d // 32) + g
    vs = ps * d + ps * d // 32 + (t // 4 * (d // 32) + g) * 4 + t % 4
    return k, v, ks, vs


def put(cache, slot, head, k, v, top_exponent):
    """K and V [D] of one token into a CPU cache."""
    d = k.shape[-1]
    ps = cache.shape[2] // (d + d // 16)
    at = places(ps, d)
    page, t = divmod(int(slot), ps)
    for x, where, scale_where in ((k, at[0], at[2]), (v, at[1], at[3])):
        code, byte = encode(x, top_exponent)
        cache[page, head, where[t]] = code[0::2] | code[1::2] << 4
        cache[page, head, scale_where[t]] = byte


def get(cache, pages, d):
    """K and V [heads, len(pages) * PS, D] in 64 bits."""
    ps = cache.shape[2] // (d + d // 16)
    k, v, ks, vs = places(ps, d)
    out = []
    for codes, scales in ((k, ks), (v, vs)):
        x, s = cache[pages][:, :, codes], cache[pages][:, :, scales]
        code = torch.stack((x & 15, x >> 4), -1).flatten(-2)
        out.append(decode(code, s).transpose(0, 1).flatten(1, 2))
    return out


def attention(q, cache, tables, lens, cu, causal, window, scale):
    """Outputs in 64 bits and, for each, a size that its error is measured by:
    sum p |v| and the largest score's sum |q k|."""
    total, hq, d = q.shape
    hk, ps = cache.shape[1], cache.shape[2] // (d + d // 16)
    ratio = hq // hk
    out = torch.zeros(total, hq, d, dtype=torch.float64)
    size = torch.zeros_like(out)
    score = torch.zeros(total, hq, dtype=torch.float64)
    for b in range(len(lens)):
        lo, hi, m = int(cu[b]), int(cu[b + 1]), int(lens[b])
        if hi == lo:
            continue
        need = min(-(-max(m, 0) // ps), tables.shape[1])
        entry = tables[b, :need].long()
        held = ((entry >= 0) & (entry < cache.shape[0])).repeat_interleave(ps)
        k, v = get(cache, entry.clamp(0, cache.shape[0] - 1), d)
        j = torch.arange(need * ps)
        pos = torch.arange(hi - lo) + m - (hi - lo)
        seen = held[None, :] & (j < m)[None, :] & torch.ones(hi - lo, 1, dtype=torch.bool)
        if causal:
            seen = seen & (j[None, :] <= pos[:, None])
        if window:
            seen = seen & (j[None, :] > pos[:, None] - window)
        for h in range(hq):
            kk, vv, qq = k[h // ratio], v[h // ratio], q[lo:hi, h].double()
            for i in range(hi - lo):
                at = seen[i].nonzero()[:, 0]
                if not len(at):
                    continue
                s = (kk[at] * qq[i]).sum(-1) * scale
                p = torch.softmax(s, 0)
                out[lo + i, h] = p @ vv[at]
                size[lo + i, h] = p @ vv[at].abs()
                score[lo + i, h] = (kk[at] * qq[i]).abs().sum(-1).max() * scale
    return out, size, score
