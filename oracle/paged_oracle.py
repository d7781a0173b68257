"""Plain statements, in 64 bits on the CPU, of the rotary positions and of the paged key/value cache's append and attention."""
import torch


def rope(x, cis, positions, layout, conj=False):
    """x [..., H, D], cis complex [rows, R/2], positions int64 of x's leading sizes; tokens outside the table are zeros."""
    pairs = cis.shape[1]
    inside = (positions >= 0) & (positions < cis.shape[0])
    z = cis.to(torch.complex128)[torch.where(inside, positions, 0)].unsqueeze(-2)
    z = z.conj() if conj else z
    y = x.double().clone()
    a, b = (slice(0, pairs), slice(pairs, 2 * pairs)) if layout == "half" else (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2))
    w = torch.complex(y[..., a], y[..., b]) * z
    y[..., a], y[..., b] = w.real, w.imag
    return y * inside[..., None, None]


def rope_float(x, cis, positions, layout, conj=False):
    """The same with fp32 products and sums that are each rounded on their own, and one rounding to x's type: what the kernels do, bit for bit."""
    pairs = cis.shape[1]
    inside = (positions >= 0) & (positions < cis.shape[0])
    z = cis[torch.where(inside, positions, 0)].unsqueeze(-2)
    c, s = z.real, -z.imag if conj else z.imag
    y = x.float().clone()
    a, b = (slice(0, pairs), slice(pairs, 2 * pairs)) if layout == "half" else (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2))
    u, v = y[..., a].clone(), y[..., b].clone()
    y[..., a], y[..., b] = u * c - v * s, u * s + v * c
    return torch.where(inside[..., None, None], y, 0.0).to(x.dtype)


def tokens_of(n, b, cu):
    """First token and number of tokens of every sequence."""
    if cu is None:
        return [(i * (n // b), n // b) for i in range(b)]
    return [(cu[i], cu[i + 1] - cu[i]) for i in range(b)]


def append(qkv, cis, k, v, pages, lengths, cu, layout):
    """Rotated q; k and v [pages, heads, rows, D] are written in place."""
    n, heads, _ = qkv.shape
    hkv, rows = k.shape[1], k.shape[2]
    hq = heads - 2 * hkv
    q = torch.zeros_like(qkv[:, :hq])
    for b, (first, count) in enumerate(tokens_of(n, len(lengths), cu)):
        for i in range(count):
            p = lengths[b] - count + i
            if not (0 <= p < cis.shape[0] and p < pages.shape[1] * rows and 0 <= pages[b, p // rows] < k.shape[0]):
                continue
            x = qkv[first + i]
            turned = rope_float(x[None, :hq + hkv], cis, torch.tensor([p]), layout)[0]
            q[first + i] = turned[:hq]
            k[pages[b, p // rows], :, p % rows], v[pages[b, p // rows], :, p % rows] = turned[hq:], x[hq + hkv:]
    return q


def attention(q, k, v, pages, lengths, cu, starts, scale):
    """Result, the sum of weights times |v|, and the largest sum of |q k| * |scale| of a query's rows: what tolerances are made of."""
    n, hq, d = q.shape
    hkv, rows = k.shape[1], k.shape[2]
    out, spread, size = torch.zeros(n, hq, d, dtype=torch.float64), torch.zeros(n, hq, d, dtype=torch.float64), torch.zeros(n, hq, 1, dtype=torch.float64)
    for b, (first, count) in enumerate(tokens_of(n, len(lengths), cu)):
        most = min(lengths[b], pages.shape[1] * rows)
        if most <= 0 or count == 0:
            continue
        at = torch.arange(most)
        number = pages[b, at // rows].long()
        there = (number >= 0) & (number < k.shape[0])
        for h in range(hq):
            kk, vv = (torch.where(there[:, None], t[torch.where(there, number, 0), h // (hq // hkv), at % rows].double(), 0.0) for t in (k, v))
            x = q[first:first + count, h].double()
            lo = max(0, starts[b]) if starts is not None else 0
            seen = (at >= lo) & (at <= lengths[b] - count + torch.arange(count)[:, None])
            score = (x @ kk.T * scale).masked_fill(~seen, -torch.inf)
            p = torch.softmax(score, -1).masked_fill(~seen.any(-1, keepdim=True), 0.0)
            rows_seen = seen.any(0)
            vv = torch.where(rows_seen[:, None], vv, 0.0)
            kk = torch.where(rows_seen[:, None], kk, 0.0)
            out[first:first + count, h], spread[first:first + count, h] = p @ vv, p @ vv.abs()
            size[first:first + count, h] = (x.abs() @ kk.abs().T).masked_fill(~seen, 0.0).amax(-1, keepdim=True) * abs(scale)
    return out, spread, size
