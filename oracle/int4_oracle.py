"""Plain statements of the 4-bit operators, in 64 bits, for the tests.

Format: a block of ``block`` values of a row has the scale max|x| and the codes rint(7 x / scale), -7 to 7; a value is scale * code / 7.
"""
import math

import torch


def quantize(x, block):
    """Codes (float64, -7 to 7) ``[..., K]`` and scales (float64) ``[..., ceil(K/block)]``; a block with an infinity or a NaN: 0, NaN."""
    x = x.double()
    codes, scales = torch.zeros_like(x), []
    for lo in range(0, x.shape[-1], block):
        part = x[..., lo:lo + block]
        s = part.abs().amax(-1)
        ok = torch.isfinite(s)
        q = torch.round(7 * part / torch.where((s == 0) | ~ok, torch.ones_like(s), s)[..., None])
        codes[..., lo:lo + block] = torch.where(ok[..., None], q, torch.zeros_like(q))
        scales.append(torch.where(ok, s, torch.full_like(s, math.nan)))
    return codes, torch.stack(scales, -1) if scales else x.new_zeros(x.shape[:-1] + (0,))


def pack(codes):
    u = (codes + 8).to(torch.uint8)
    if u.shape[-1] % 2:
        u = torch.nn.functional.pad(u, (0, 1), value=8)
    return u[..., 0::2] | (u[..., 1::2] << 4)


def values(codes, scales, block):
    """``[..., K]`` in 64 bits."""
    return codes * scales.double().repeat_interleave(block, -1)[..., :codes.shape[-1]] / 7


def rotate(x, cis):
    """What the append leaves of ``x [..., D]`` for (cos, sin) pairs ``cis [..., D/2, 2]``: products and sums as fp32 rounds them, the result
    as x's type does (a product of a 16-bit value and an fp32 one is exact in 64 bits, and so is a sum of two fp32 numbers near enough)."""
    f = lambda t: t.float().double()
    a, b = x[..., 0::2].double(), x[..., 1::2].double()
    c, s = cis[..., 0].double(), cis[..., 1].double()
    return torch.stack((f(f(a * c) - f(b * s)), f(f(a * s) + f(b * c))), -1).flatten(-2).to(x.dtype)


def attention(q, k, v, lengths, starts=None, scale=None):
    """``q [B, Hq, T, D]``, ``k`` / ``v`` ``[B, Hkv, L, D]`` of any type: the result in 64 bits."""
    B, Hq, T, D = q.shape
    G, L = Hq // k.shape[1], k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for b in range(B):
        n, lo = int(lengths[b]), 0 if starts is None else max(0, int(starts[b]))
        for t in range(T):
            hi = max(0, min(L, n - T + t + 1))
            if hi <= lo:
                continue
            kk, vv = (x[b, :, lo:hi].double().repeat_interleave(G, 0) for x in (k, v))
            p = torch.softmax((kk @ q[b, :, t].double()[..., None])[..., 0] * scale, -1)
            out[b, :, t] = (p[:, None] @ vv)[:, 0]
    return out
