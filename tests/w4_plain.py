"""Plain forms of the products with 4-bit weights, in 64 bits, on any device."""
import torch

LEVELS = [0, .5, 1, 1.5, 2, 3, 4, 6]


def values(codes, scales):
    """float64 [.., K] of codes uint8 [.., K / 2] and scales uint8 [.., K / 32]."""
    levels = torch.tensor(LEVELS + [-v for v in LEVELS], dtype=torch.float64, device=codes.device)
    w = torch.stack((levels[(codes & 15).long()], levels[(codes >> 4).long()]), -1).flatten(-2)
    s = torch.where(scales == 255, torch.nan, torch.exp2(scales.double() - 127))
    return w * s.repeat_interleave(32, -1)


def quantized(w, most=125):
    """Codes and scales of weights [.., K]: the smallest power of two (of 2^-125 to
    2^most) under which no magnitude of a group reaches 7, the nearest code, ties to
    the even one; a group with an infinity or a NaN: codes 0, byte 255."""
    g = w.double().unflatten(-1, (-1, 32))
    good = torch.isfinite(g).all(-1, keepdim=True)
    g = torch.where(good, g, 0.0)
    power = torch.full_like(g[..., :1], -125.0)
    top = g.abs().amax(-1, keepdim=True)
    for p in range(-125, most):
        power = torch.where(top >= 7 * 2.0 ** p, float(p + 1), power)
    levels = torch.tensor(LEVELS, dtype=torch.float64, device=w.device)
    y = (g.abs() / torch.exp2(power)).clamp_max(6)
    far = (y[..., None] - levels).abs()
    near = far.amin(-1, keepdim=True)
    code = torch.arange(8, device=w.device)
    # among the nearest (one, or two at a tie) the even code
    code = torch.where(far == near, code + 100 * (code % 2), 1000).amin(-1) % 100
    code = torch.where(good, code | (torch.signbit(g).long() << 3), 0).flatten(-2).to(torch.uint8)
    byte = torch.where(good, power + 127, 255.0).squeeze(-1).to(torch.uint8)
    return code[..., ::2] | (code[..., 1::2] << 4), byte


def packed(codes, scales):
    """uint8 [matrices, bytes] of codes [matrices, N, K / 2] and scales [matrices, N, K / 32]."""
    e, n, half = codes.shape
    k = 2 * half
    blocks, tiles, words = -(-n // 32), 2 * -(-k // 128), -(-k // 256)
    c = torch.zeros(e, blocks * 32, tiles * 2, 16, dtype=torch.uint8, device=codes.device)
    c[:, :n, :k // 32] = codes.view(e, n, k // 32, 16)
    c = c.view(e, blocks, 32, tiles, 2, 16).permute(0, 1, 3, 4, 2, 5)          # block, tile, half, row, byte
    s = torch.full((e, blocks * 32, words * 8), 2, dtype=torch.uint8, device=codes.device)
    s[:, :n, :k // 32] = scales
    s = s.view(e, blocks, 32, words, 4, 2).permute(0, 1, 3, 5, 2, 4)           # block, word, half, row, tile
    return torch.cat((c.reshape(e, -1), s.reshape(e, -1)), 1)


def checkpoint(g, *shape, spread=2, device="cuda:0"):
    """Random codes and scales of weights [.., K] of a size like those of a model."""
    *rows, k = shape
    codes = torch.randint(0, 256, (*rows, k // 2), generator=g, device=device, dtype=torch.uint8)
    scales = 127 - 7 + torch.randint(-spread, spread + 1, (*rows, k // 32), generator=g, device=device)
    return codes, scales.to(torch.uint8)


def product(x, w, bias=None, gated=False):
    """The result in 64 bits, and a bound on the error of sums held in 32.

    Each of the K products is exact in 32 bits (24 bits hold those of 8 or 11 by 2);
    each addition is off by at most a step, 2^-23, of a partial sum, and no partial sum
    passes S = sum |x w| + |bias|: (K + 2) 2^-23 S, one more each for bias and
    rounding."""
    x, k = x.double(), x.shape[-1]
    y, s = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        y, s = y + bias.double(), s + bias.double().abs()
    e = (k + 2) * 2.0 ** -23 * s
    if not gated:
        return y, e
    n = y.shape[-1] // 2
    gate, up, eg, eu = y[..., :n], y[..., n:], e[..., :n], e[..., n:]
    silu = gate * torch.sigmoid(gate)
    # |silu'| <= 1.1; the exponential is off by 2^-22 and 2^-23 |gate|, quotient and products by a step each
    own = silu.abs() * (2.0 ** -20 + 2.0 ** -22 * gate.abs())
    return silu * up, (1.1 * eg + own) * (up.abs() + eu) + silu.abs() * eu


def close(got, want, error):
    """Within the error of the sums and half a step of the type, of what is rounded."""
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * half * 2
    limit = error + half * (want.abs() + error) + tiny
    off = (got.double() - want).abs()
    bad = ~(off <= limit) & ~(torch.isnan(got) & torch.isnan(want))
    worst = float((off / limit).nan_to_num().max()) if bad.numel() else 0.0
    return not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, worst {worst:.3g} of the limit"
