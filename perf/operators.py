"""Serving in 4 bits: the operators behind weights and key/value caches that are held in 4 bits, as cases that can be timed and
compared.

A case is a dict of plain values.  ``kind`` says which operator it takes, through the public functions:

  round_trip   ``quantize_block_int4`` and ``dequantize_block_int4``: a weight matrix into 4 bits and back, as for storing a layer
               and for looking at what it became
  matmul       ``int4_matmul``: the activations of a few tokens through a layer whose weights are held in 4 bits
  append       ``rope_cache_append_int4``: what a fused q/k/v projection leaves for new tokens; q and k are rotated, k and v are
               quantized into the cache.  The whole cache is read back by ``dequantize_block_int4``, as for handing it on
  attention    ``attention_int4_cache``: the queries of the newest tokens over everything their sequences have in the cache

The 4-bit format: a block of consecutive values of a row has the scale s = max|x|, in x's own type, and every value the code
rint(7 x / s), -7 to 7, which stands for s * code / 7.  Two codes share a byte, offset by 8, the even one in its low half.  Weights
have blocks of 32, 64 or 128, caches of 64.

Sizes are those of the Llama-7B and GPT-2 small models in the examples and generic ones.  ``T`` is the number of new tokens of a
sequence, ``Hq`` and ``Hkv`` the heads of queries and of the cache, ``D`` the head size, ``L`` the rows that the cache has room for.
``fill`` is the share of those rows that the longest sequence uses; with ``ragged`` the others use anything from one row to that.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
CACHE_BLOCK = 64


def _round_trip(name, N, K, block=64, dtype="bf16"):
    return {"name": name, "kind": "round_trip", "N": N, "K": K, "block": block, "dtype": dtype}


def _matmul(name, M, K, N, block=64, dtype="bf16", bias=False, residual=False):
    return {"name": name, "kind": "matmul", "M": M, "K": K, "N": N, "block": block, "dtype": dtype, "bias": bias, "residual": residual}


def _append(name, B, T, Hq, Hkv, D, L, dtype="bf16"):
    return {"name": name, "kind": "append", "B": B, "T": T, "Hq": Hq, "Hkv": Hkv, "D": D, "L": L, "dtype": dtype}


def _attention(name, B, T, Hq, Hkv, D, L, fill=1.0, ragged=False, dtype="bf16"):
    return {"name": name, "kind": "attention", "B": B, "T": T, "Hq": Hq, "Hkv": Hkv, "D": D, "L": L, "fill": fill, "ragged": ragged,
            "dtype": dtype}


def listed():
    return [
        # a checkpoint's up projection is put into 4 bits
        _round_trip("store_up_projection", 11008, 4096),
        # a layer whose sizes nobody rounded, in half precision and short blocks
        _round_trip("store_ragged_fp16", 777, 1001, block=32, dtype="fp16"),
        # generating text for one user: one token through an attention projection; latency is all
        _matmul("token_projection", 1, 4096, 4096),
        # a decode step of a small serving batch: the up projection, and the down projection with its residual sum
        _matmul("batch8_up", 8, 4096, 11008),
        _matmul("batch32_down", 32, 11008, 4096, block=128, residual=True),
        # the ragged layer at work
        _matmul("ragged_fp16", 13, 1001, 777, block=32, dtype="fp16", bias=True),
        # a decode step of a large batch with shared key/value heads; the caches are short, so that what is appended counts
        _append("batch128_append", 128, 1, 32, 8, 128, 24),
        # a prompt is read in: 8 sequences of 512 tokens
        _append("prompt_append", 8, 512, 32, 32, 128, 512),
        # a decode step of the example: 8 sequences somewhere behind their prompt of 512 tokens
        _attention("batch8_decode", 8, 1, 32, 32, 128, 640, fill=0.9),
        # a serving batch of sequences of every length, four query heads on each key/value head
        _attention("batch32_ragged", 32, 1, 32, 8, 128, 8192, ragged=True),
        # one user with a long document
        _attention("long_document", 1, 1, 32, 8, 128, 131072, fill=0.97),
        # a part of a prompt behind what was read before, small heads, half precision
        _attention("prompt_part_fp16", 2, 200, 12, 12, 64, 1500, dtype="fp16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    block = rng.choice([32, 64, 64, 128])

    def features(lo, hi):      # odd sizes among the even ones
        n = _log(rng, lo, hi)
        return n if rng.random() < 0.3 else max(64, n // 64 * 64)

    kind = rng.choice(["round_trip", "matmul", "matmul", "append", "attention", "attention"])
    if kind == "round_trip":
        return _round_trip("", features(64, 11008), features(64, 4096), block, dtype)
    if kind == "matmul":
        return _matmul("", _log(rng, 1, 64), features(256, 11008), features(256, 8192), block, dtype, rng.random() < 0.3, rng.random() < 0.3)
    D, (Hq, Hkv) = rng.choice([64, 128, 128, 256]), rng.choice([(32, 32), (32, 8), (12, 12), (16, 2), (8, 1), (20, 4)])
    if kind == "append":
        T = rng.choice([1, 1, _log(rng, 2, 256)])
        B = _log(rng, 1, max(1, min(128, 2048 // T)))
        return _append("", B, T, Hq, Hkv, D, T + rng.randrange(0, 24), dtype)
    T = rng.choice([1, 1, 1, _log(rng, 2, 128)])
    L = _log(rng, 16, 65536)
    # the cache's values, and for many new tokens the scores, bound the batch
    B = _log(rng, 1, max(1, min(64, (1 << 27) // (L * Hkv * D), (1 << 27) // (L * Hq * T))))
    return _attention("", B, T, Hq, Hkv, D, L, rng.uniform(0.3, 1.0), rng.random() < 0.6, dtype)


# ---- inputs -----------------------------------------------------------------------------------------------------------------
def _normal(gen, shape, dtype, std=1.0, outliers=0.0):
    x = torch.randn(shape, device="cuda", generator=gen) * std
    if outliers:               # the few large values of activations
        x = torch.where(torch.rand(shape, device="cuda", generator=gen) < outliers, x * 20.0, x)
    return x.to(dtype)


def _blocks(x, block):
    """x [..., K] as [..., ceil(K / block), block], the last block filled up with zeros."""
    pad = -x.shape[-1] % block
    return torch.nn.functional.pad(x, (0, pad)).unflatten(-1, (-1, block))


def _codes(x, block):
    """Codes -7 to 7 as floats [..., K] and scales in x's type.  7 x is exact in 32 bits, and so is which code its quotient is
    nearest to: for 16-bit values it is a tie or 2^-16 away from one."""
    b = _blocks(x, block).float()
    s = b.abs().amax(-1, keepdim=True)
    q = torch.where(s > 0, torch.round(7.0 * b / s), torch.zeros_like(b))
    return q.flatten(-2)[..., :x.shape[-1]], s[..., 0].to(x.dtype)


def _pack(q):
    u = (q + 8.0).to(torch.uint8)
    if u.shape[-1] % 2:
        u = torch.nn.functional.pad(u, (0, 1), value=8)
    return u[..., 0::2] + u[..., 1::2] * 16


def _unpack(packed, K):
    q = torch.stack((packed & 15, packed >> 4), dim=-1).flatten(-2)[..., :K]
    return q.float() - 8.0


def _values(packed, state, K, block):
    """What packed codes stand for, in 32 bits."""
    q = _unpack(packed, K)
    return (_blocks(q, block) * state.float()[..., None]).flatten(-2)[..., :K] / 7.0


def _rope_table(rows, D):
    inv = 1.0 / (10000.0 ** (torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D))
    ang = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * inv
    return torch.complex(ang.cos().float(), ang.sin().float())


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt, kind = DTYPES[case["dtype"]], case["kind"]
    st = dict(case)
    if kind == "round_trip":
        st["w"] = _normal(gen, (case["N"], case["K"]), dt, 0.02)
    elif kind == "matmul":
        M, K, N = case["M"], case["K"], case["N"]
        w = _normal(gen, (N, K), dt, 0.02)
        q, st["state"] = _codes(w, case["block"])
        st["codes"] = _pack(q)
        st["x"] = _normal(gen, (M, K), dt, 1.0, outliers=0.001)
        st["bias"] = _normal(gen, (N,), dt) if case["bias"] else None
        st["res"] = _normal(gen, (M, N), dt) if case["residual"] else None
    else:
        B, T, Hq, Hkv, D, L = (case[n] for n in ("B", "T", "Hq", "Hkv", "D", "L"))
        rows = (B, Hkv, L, D)
        cache = []
        # outstanding channels are what keys have and values lack
        channel = torch.where(torch.rand((Hkv, 1, D), device="cuda", generator=gen) < 0.03, 6.0, 1.0)
        for key in (True, False):
            x = torch.randn(rows, device="cuda", generator=gen)
            q, s = _codes((x * channel if key else x).to(dt), CACHE_BLOCK)
            cache += [_pack(q), s]
        st["cache"] = cache
        if kind == "append":
            st["qkv"] = _normal(gen, (B, T, Hq + 2 * Hkv, D), dt, 1.0, outliers=0.001)
            st["cis"] = _rope_table(L + 8, D)
            st["pos"] = torch.randint(0, L - T + 1, (B,), device="cuda", generator=gen)
        else:
            st["q"] = _normal(gen, (B, Hq, T, D), dt)
            longest = max(1, min(L, int(L * case["fill"])))
            lengths = torch.full((B,), longest, device="cuda", dtype=torch.int64)
            if case["ragged"] and B > 1:
                lengths[1:] = torch.randint(1, longest + 1, (B - 1,), device="cuda", generator=gen)
            st["lengths"] = lengths
    if own:
        from blockwise_int8_linear_b200.decode_ops import Int4KVCache
        if "cache" in st:
            st["cache"] = Int4KVCache(*st["cache"])
    return st


# ---- one pass ---------------------------------------------------------------------------------------------------------------
def run(st):
    return _run_own(st) if own else _PLAIN[st["kind"]](st)


def _run_own(st):
    from blockwise_int8_linear_b200 import decode_ops, int4_functions as f
    kind, dt = st["kind"], DTYPES[st["dtype"]]
    if kind == "round_trip":
        codes, state = f.quantize_block_int4(st["w"], st["block"])
        return f.dequantize_block_int4(codes, state, st["block"], features=st["K"], dtype=dt), state
    if kind == "matmul":
        return f.int4_matmul(st["x"], st["codes"], st["state"], st["bias"], residual=st["res"], fblock_size=st["block"], dtype=dt)
    cache = st["cache"]
    if kind == "append":
        q = decode_ops.rope_cache_append_int4(st["qkv"], st["cis"], st["pos"], cache)
        return (q, f.dequantize_block_int4(cache.k, cache.k_state, CACHE_BLOCK, dtype=dt),
                f.dequantize_block_int4(cache.v, cache.v_state, CACHE_BLOCK, dtype=dt))
    return decode_ops.attention_int4_cache(st["q"], cache, st["lengths"])


def _plain_round_trip(st):
    w, block = st["w"], st["block"]
    q, state = _codes(w, block)
    v = (_blocks(q, block) * state.float()[..., None]).flatten(-2)[..., :w.shape[1]] / 7.0
    return v.to(w.dtype), state


def _plain_matmul(st):
    y = st["x"].float() @ _values(st["codes"], st["state"], st["K"], st["block"]).t()
    for addend in (st["bias"], st["res"]):
        if addend is not None:
            y = y + addend.float()
    return y.to(st["x"].dtype)


def _rotate(x, c, s):
    """(x0 + i x1) * (c + i s) of neighbouring features; every product and sum is rounded on its own."""
    x0, x1 = x[..., 0::2], x[..., 1::2]
    return torch.stack((x0 * c - x1 * s, x0 * s + x1 * c), dim=-1).flatten(-2)


def _plain_append(st):
    qkv, (kc, ks, vc, vs) = st["qkv"], st["cache"]
    B, T, Hq, Hkv, D, L = (st[n] for n in ("B", "T", "Hq", "Hkv", "D", "L"))
    rows = st["pos"][:, None] + torch.arange(T, device=qkv.device)                                  # [B, T]
    cis = st["cis"][rows][:, :, None]                                                              # [B, T, 1, D/2]
    x = qkv.float()
    q = _rotate(x[:, :, :Hq], cis.real, cis.imag).to(qkv.dtype).transpose(1, 2).contiguous()
    k = _rotate(x[:, :, Hq:Hq + Hkv], cis.real, cis.imag).to(qkv.dtype)
    b, h, r = torch.arange(B, device=qkv.device)[:, None, None], torch.arange(Hkv, device=qkv.device), rows[..., None]
    for new, codes, state in ((k, kc, ks), (qkv[:, :, Hq + Hkv:], vc, vs)):
        n, s = _codes(new, CACHE_BLOCK)
        codes[b, h, r], state[b, h, r] = _pack(n), s
    return q, _values(kc, ks, D, CACHE_BLOCK).to(qkv.dtype), _values(vc, vs, D, CACHE_BLOCK).to(qkv.dtype)


def _plain_attention(st):
    q, (kc, ks, vc, vs) = st["q"], st["cache"]
    B, Hq, T, D = q.shape
    Hkv, L = kc.shape[1], kc.shape[2]
    k, v = _values(kc, ks, D, CACHE_BLOCK), _values(vc, vs, D, CACHE_BLOCK)
    qg = q.float().reshape(B, Hkv, Hq // Hkv * T, D)
    score = qg @ k.transpose(-1, -2) * (1.0 / math.sqrt(D))                                         # [B, Hkv, G * T, L]
    last = st["lengths"][:, None] - T + torch.arange(T, device=q.device)                            # [B, T]
    seen = torch.arange(L, device=q.device) <= last[..., None]                                      # [B, T, L]
    score = score.view(B, Hkv, Hq // Hkv, T, L).masked_fill(~seen[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    return (p.view(B, Hkv, -1, L) @ v).view(B, Hq, T, D).to(q.dtype)


_PLAIN = {"round_trip": _plain_round_trip, "matmul": _plain_matmul, "append": _plain_append, "attention": _plain_attention}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------------
def _exact_codes(x, block):
    """Codes and scales of x [..., K] (values of the 16-bit type, in 64 bits), block by block."""
    out, scales = torch.empty_like(x), []
    for lo in range(0, x.shape[-1], block):
        part = x[..., lo:lo + block]
        s = part.abs().max(-1).values
        code = torch.round(part * 7 / torch.where(s == 0, 1.0, s)[..., None])
        out[..., lo:lo + block] = s[..., None] * code / 7
        scales.append(s)
    return out, torch.stack(scales, -1)


def _exact_values(packed, state, K, block):
    out = torch.empty(packed.shape[:-1] + (packed.shape[-1] * 2,), dtype=torch.float64, device=packed.device)
    out[..., 0::2], out[..., 1::2] = packed % 16, packed // 16
    out = (out[..., :K] - 8) / 7
    return out * state.double().repeat_interleave(block, -1)[..., :K]


def exact(case, seed):
    global own
    mode, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = mode
    kind = case["kind"]
    if kind == "round_trip":
        return _exact_codes(st["w"].double(), case["block"])
    if kind == "matmul":
        w = _exact_values(st["codes"], st["state"], case["K"], case["block"])
        y = torch.einsum("mk,nk->mn", st["x"].double(), w)
        if st["bias"] is not None:
            y += st["bias"].double()
        return y if st["res"] is None else y + st["res"].double()
    kc, ks, vc, vs = st["cache"]
    D, T, Hq, Hkv = case["D"], case["T"], case["Hq"], case["Hkv"]
    k, v = _exact_values(kc, ks, D, CACHE_BLOCK), _exact_values(vc, vs, D, CACHE_BLOCK)
    if kind == "append":
        x, dt = st["qkv"].double(), st["qkv"].dtype
        turn = torch.stack([st["cis"][p:p + T] for p in st["pos"].tolist()])[:, :, None]            # [B, T, 1, D/2]
        c, s = turn.real.double(), turn.imag.double()
        even, odd = x[..., 0::2], x[..., 1::2]
        q = torch.empty_like(x[:, :, :Hq])
        q[..., 0::2], q[..., 1::2] = (even * c - odd * s)[:, :, :Hq], (even * s + odd * c)[:, :, :Hq]
        # what is quantized is the rotated key as its type holds it: products and sums as 32 bits round them
        f = lambda t: t.float().double()
        e, o = even[:, :, Hq:Hq + Hkv], odd[:, :, Hq:Hq + Hkv]
        key = torch.empty_like(x[:, :, Hq:Hq + Hkv])
        key[..., 0::2], key[..., 1::2] = f(f(e * c) - f(o * s)), f(f(e * s) + f(o * c))
        key = _exact_codes(key.to(dt).double(), CACHE_BLOCK)[0]
        val = _exact_codes(x[:, :, Hq + Hkv:], CACHE_BLOCK)[0]
        for i, p in enumerate(st["pos"].tolist()):
            k[i, :, p:p + T], v[i, :, p:p + T] = key[i].transpose(0, 1), val[i].transpose(0, 1)
        return q.transpose(1, 2).contiguous(), k, v
    # attention: sequence by sequence, over the rows that it has
    q = st["q"].double()
    out = torch.zeros_like(q)
    for i, n in enumerate(st["lengths"].tolist()):
        kk, vv = (t[i, :, :n].repeat_interleave(Hq // Hkv, 0) for t in (k, v))
        score = torch.einsum("htd,hld->htl", q[i], kk) / math.sqrt(D)
        ahead = torch.arange(n, device=q.device)[None] - (n - T + torch.arange(T, device=q.device))[:, None] > 0
        score = score.masked_fill(ahead, -math.inf)
        p = torch.nan_to_num(torch.softmax(score, -1), nan=0.0)
        out[i] = torch.einsum("htl,hld->htd", p, vv)
    return out


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind in ("round_trip", "matmul"):
        N, K = case["N"], case["K"]
        blocks = -(-K // case["block"])
        if kind == "round_trip":            # the matrix in, its values and scales out
            return {"bytes": 4 * N * K + 2 * N * blocks, "flops": 6 * N * K}
        M = case["M"]
        moved = N * (-(-K // 2)) + 2 * N * blocks + 2 * M * (K + N) + (2 * N if case["bias"] else 0) + (2 * M * N if case["residual"] else 0)
        return {"bytes": moved, "flops": 2 * M * N * K}
    B, T, Hq, Hkv, D, L = (case[n] for n in ("B", "T", "Hq", "Hkv", "D", "L"))
    row = D // 2 + 2 * D // CACHE_BLOCK       # codes and scales of a row
    if kind == "append":                      # q/k/v in, q out; the cache is read for its values, new rows come from q/k/v
        old = 2 * B * Hkv * (L - T) * row
        return {"bytes": 2 * B * T * (2 * Hq + 2 * Hkv) * D + old + 4 * B * Hkv * L * D + 8 * B * T * D // 2,
                "flops": 3 * B * T * (Hq + Hkv) * D + 12 * B * Hkv * L * D}
    longest = max(1, min(L, int(L * case["fill"])))
    used = longest + (B - 1) * ((longest + 1) / 2 if case["ragged"] else longest)      # rows of all sequences, on average
    seen = max(used * T - B * T * (T - 1) / 2, used)
    return {"bytes": int(2 * Hkv * row * used + 4 * B * Hq * T * D), "flops": int(4 * Hq * D * seen)}
