"""Serving from a paged key/value cache, and rotary positions: the operators as cases that can be timed and compared.

A case is a dict of plain values.  ``kind`` says which operator it takes, through the public functions of ``decode_ops``:

  rope         ``rope``: q and k of a layer are turned by the angles of their positions; with ``grad`` the gradient comes with it
  append       ``rope_cache_append_paged``: what a fused q/k/v projection leaves for the new tokens of some sequences; q and k are
               rotated, k and v go to their pages.  The cache's pages are the state: outputs are q and all of both
  attention    ``attention_paged_cache``: the new tokens' queries over everything that their sequences have in the pages

The cache: pages of ``page`` rows for each of ``Hkv`` heads, ``[pages, Hkv, page, D]`` for keys and for values, and a table
``[B, width]`` of the numbers of a sequence's pages.  New tokens of all sequences lie one behind the other, ``[N, heads, D]``; ``cu_tokens``
says where a sequence's begin (without it every sequence has N / B).  A sequence of ``lengths`` rows has its new tokens in the last ones.

Sizes are those of the Llama-7B and GPT-2 small models in the examples and generic ones.  ``B`` is the number of sequences, of which
``chunks`` have ``T`` new tokens and the others one; ``pad`` unused token rows lie behind the last sequence, as in a batch of a captured
graph.  ``Hq`` and ``Hkv`` are the heads of queries and of the cache, ``D`` the head size, ``R`` the features that are rotated.  ``L`` is how many
rows the longest sequence has; with ``ragged`` the others have anything from their new tokens to that.  With ``starts`` a sequence's first
rows, up to half of those that are not new, are not seen.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _rope(name, B, T, H, D, R, layout="half", dtype="bf16", grad=True, rows=0, factor=1.0):
    return {"name": name, "kind": "rope", "B": B, "T": T, "H": H, "D": D, "R": R, "layout": layout, "dtype": dtype, "grad": grad,
            "rows": rows or T, "factor": factor}


def _append(name, B, chunks, T, Hq, Hkv, D, page, L, R=0, layout="interleaved", pad=0, ragged=True, dtype="bf16"):
    return {"name": name, "kind": "append", "B": B, "chunks": chunks, "T": T, "Hq": Hq, "Hkv": Hkv, "D": D, "page": page, "L": L, "R": R or D,
            "layout": layout, "pad": pad, "ragged": ragged, "dtype": dtype}


def _attention(name, B, chunks, T, Hq, Hkv, D, page, L, pad=0, ragged=False, starts=False, dtype="bf16"):
    return {"name": name, "kind": "attention", "B": B, "chunks": chunks, "T": T, "Hq": Hq, "Hkv": Hkv, "D": D, "page": page, "L": L, "pad": pad,
            "ragged": ragged, "starts": starts, "dtype": dtype}


def listed():
    return [
        # a training step's q and k of one layer: 4 sequences of 4096 tokens, 32 query and 8 key heads
        _rope("train_q_and_k", 4, 4096, 40, 128, 128),
        # a small model in half precision that rotates half of each head; a batch whose length nobody rounded
        _rope("train_part_fp16", 3, 777, 24, 64, 32, "interleaved", "fp16"),
        # reading far into a document whose positions were stretched eightfold, in single precision
        _rope("far_positions_fp32", 2, 2048, 32, 128, 128, "half", "fp32", grad=False, rows=131072, factor=8.0),
        # a decode step of a large batch with shared key/value heads; latency counts
        _append("batch128_append", 128, 0, 1, 32, 8, 128, 16, 256),
        # four prompts are read in
        _append("prompt_append", 4, 4, 2048, 32, 32, 128, 64, 2048, layout="half", ragged=False),
        # a mixed batch of a small half-precision model: a part of a prompt among single tokens, odd pages, unused rows behind
        _append("mixed_append_fp16", 13, 1, 333, 12, 12, 64, 48, 1000, R=32, pad=7, dtype="fp16"),
        # generating text for one user with the example's heads: a short sequence, latency is all
        _attention("one_user", 1, 0, 1, 32, 32, 128, 16, 600),
        # a serving batch of sequences of every length, four query heads on each key/value head
        _attention("batch32_ragged", 32, 0, 1, 32, 8, 128, 16, 8192, ragged=True),
        # one user with a long document
        _attention("long_document", 1, 0, 1, 32, 8, 128, 64, 131072),
        # the next part of a long prompt
        _attention("prompt_part", 1, 1, 2048, 32, 8, 128, 64, 32768),
        # prompts' parts among the single tokens of other users, with unused rows behind
        _attention("mixed_batch", 16, 2, 512, 32, 8, 128, 16, 4096, pad=2, ragged=True),
        # prompts from their first token on, small heads in half precision, odd pages
        _attention("prompts_fp16", 8, 8, 500, 12, 12, 64, 48, 500, dtype="fp16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "append", "attention", "attention", "attention"])
    dtype, layout = rng.choice(["bf16", "bf16", "fp16"]), rng.choice(["interleaved", "half"])
    if kind == "rope":
        D = rng.choice([64, 96, 128, 128, 256])
        H = rng.choice([1, 8, 12, 24, 32, 40])
        T = _log(rng, 1, 4000)
        B = _log(rng, 1, max(1, min(64, (1 << 25) // (T * H * D))))
        R = rng.choice([D, D, D // 2, D // 4])
        return _rope("", B, T, H, D, R, layout, rng.choice(["bf16", "bf16", "fp16", "fp32"]), rng.random() < 0.6,
                     T + rng.choice([0, 100, 100000]), rng.choice([1.0, 1.0, 8.0]))
    D, (Hq, Hkv) = rng.choice([64, 128, 128, 256]), rng.choice([(32, 32), (32, 8), (12, 12), (16, 2), (8, 1), (20, 4), (15, 5)])
    page = rng.choice([16, 16, 32, 48, 64, 128, 256])
    T = _log(rng, 2, 2048)
    # single tokens only, prompts or their parts only, or both
    form = rng.choice(["single", "chunks", "mixed"])
    if kind == "append":
        B = _log(rng, 1, 128 if form == "single" else max(1, min(64, (1 << 26) // (T * (Hq + 2 * Hkv) * D))))
    else:
        L = _log(rng, 16, min(65536, (1 << 27) // (Hkv * D)))      # the cache's values are bounded
        room = (1 << 27) // (L * Hkv * D)                          # and so the batch
        if form != "single":                                       # as are the products, and the scores of a head group
            T = min(T, L, max(2, min((1 << 29) // (L * (Hq // Hkv)), (1 << 37) // (L * Hq * D))))
            room = min(room, (1 << 37) // (L * Hq * D * T), (1 << 25) // (Hq * D * T))
        B = _log(rng, 1, max(1, min(64, room)))
    if B == 1 and form == "mixed":
        form = "chunks"
    chunks = {"single": 0, "chunks": B, "mixed": rng.randrange(1, max(2, B // 2))}[form]
    T = T if chunks else 1
    pad = rng.choice([0, 0, rng.randrange(1, 20)])
    if kind == "append":
        return _append("", B, chunks, T, Hq, Hkv, D, page, T + rng.randrange(0, 500), rng.choice([D, D, D // 2]), layout, pad, rng.random() < 0.7, dtype)
    return _attention("", B, chunks, T, Hq, Hkv, D, page, max(L, T), pad, rng.random() < 0.6, rng.random() < 0.15, dtype)


# ---- inputs -----------------------------------------------------------------------------------------------------------------
def _table(rows, R, factor=1.0):
    """cos and sin of every position for R features: angles in 64 bits."""
    inv = 1.0 / (10000.0 ** (torch.arange(0, R, 2, device="cuda", dtype=torch.float64) / R)) / factor
    ang = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * inv
    return torch.complex(ang.cos().float(), ang.sin().float())


def _tokens(case):
    """New tokens of every sequence: the ones with a chunk lie in the middle."""
    n = [1] * case["B"]
    first = (case["B"] - case["chunks"]) // 2
    n[first:first + case["chunks"]] = [case["T"]] * case["chunks"]
    return n


def _packed(case):
    return case["pad"] > 0 or 0 < case["chunks"] < case["B"]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    normal = lambda *shape: torch.randn(shape, device="cuda", generator=gen)
    below = lambda hi, n: torch.randint(0, hi, (n,), device="cuda", generator=gen)
    st = dict(case)
    if case["kind"] == "rope":
        B, T, H, D = (case[n] for n in ("B", "T", "H", "D"))
        st["cis"] = _table(case["rows"], case["R"], case["factor"])
        # without spare rows every sequence begins at 0, as in training; otherwise anywhere
        st["positions"] = torch.arange(T, device="cuda")
        if case["rows"] > T:
            st["positions"] = below(case["rows"] - T + 1, B)[:, None] + st["positions"]
        st["x"] = normal(B, T, H, D).to(dt)
        if case["grad"]:
            st["g"] = normal(B, T, H, D).to(dt)
            st["x"].requires_grad_(own)
        return st
    B, Hq, Hkv, D, page, L = (case[n] for n in ("B", "Hq", "Hkv", "D", "page", "L"))
    n = _tokens(case)
    total = sum(n) + case["pad"]
    tokens = torch.tensor(n, device="cuda")
    lengths = torch.full((B,), L, device="cuda")
    if case["ragged"] and B > 1:
        lengths[1:] = tokens[1:] + (torch.rand(B - 1, device="cuda", generator=gen) * (L - tokens[1:] + 1)).long().clamp_(max=L)
        lengths = torch.minimum(lengths, torch.full_like(lengths, L))
    st["lengths"], st["tokens"], st["N"] = lengths, tokens, sum(n)
    st["cu_tokens"] = None
    if _packed(case):
        st["cu_tokens"] = torch.cat((tokens.new_zeros(1), tokens.cumsum(0)))
    # pages in the order in which a pool gave them out; entries behind a sequence's last page are no page's number
    width = -(-L // page)
    pages = torch.randperm(B * width + 3, device="cuda", generator=gen)[:B * width].view(B, width).to(torch.int32)
    st["pages"] = torch.where(torch.arange(width, device="cuda") * page < lengths[:, None], pages, -1)
    # outstanding channels are what keys have and values lack
    channel = torch.where(torch.rand((Hkv, 1, D), device="cuda", generator=gen) < 0.03, 4.0, 1.0)
    shape = (B * width + 3, Hkv, page, D)
    st["k"], st["v"] = (normal(*shape) * channel).to(dt), normal(*shape).to(dt)
    if case["kind"] == "append":
        st["qkv"] = normal(total, Hq + 2 * Hkv, D).to(dt)
        st["cis"] = _table(L, case["R"])
    else:
        st["q"] = normal(total, Hq, D).to(dt)
        st["starts"] = None
        if case["starts"]:
            st["starts"] = (torch.rand(B, device="cuda", generator=gen) * (lengths - tokens) / 2).long()
    if own:
        from blockwise_int8_linear_b200.decode_ops import PagedKVCache
        st["cache"] = PagedKVCache(st["k"], st["v"])
    return st


# ---- one pass ---------------------------------------------------------------------------------------------------------------
def run(st):
    return _run_own(st) if own else _PLAIN[st["kind"]](st)


def _run_own(st):
    from blockwise_int8_linear_b200 import decode_ops as f
    if st["kind"] == "rope":
        y = f.rope(st["x"], st["cis"], st["positions"], layout=st["layout"])
        return (y.detach(), *torch.autograd.grad(y, st["x"], st["g"])) if st["grad"] else y
    if st["kind"] == "append":
        q = f.rope_cache_append_paged(st["qkv"], st["cis"], st["cache"], st["pages"], st["lengths"], st["cu_tokens"], layout=st["layout"])
        return q, st["k"], st["v"]
    return f.attention_paged_cache(st["q"], st["cache"], st["pages"], st["lengths"], st["cu_tokens"], starts=st["starts"])


def _turn(x, c, s, layout):
    """The first features of x [..., heads, D] as pairs times c + i s [..., 1, pairs], in 32 bits; the others as they are."""
    R = 2 * c.shape[-1]
    head, rest = x[..., :R].float(), x[..., R:].float()
    if layout == "half":
        a, b = head[..., :R // 2], head[..., R // 2:]
        return torch.cat((a * c - b * s, a * s + b * c, rest), dim=-1)
    a, b = head[..., 0::2], head[..., 1::2]
    return torch.cat((torch.stack((a * c - b * s, a * s + b * c), dim=-1).flatten(-2), rest), dim=-1)


def _plain_rope(st):
    cis = st["cis"][st["positions"]][..., None, :]
    y = _turn(st["x"], cis.real, cis.imag, st["layout"]).to(st["x"].dtype)
    if not st["grad"]:
        return y
    return y, _turn(st["g"], cis.real, -cis.imag, st["layout"]).to(y.dtype)


def _places(st):
    """Sequence and position of every new token."""
    n = st["tokens"]
    seq = torch.repeat_interleave(torch.arange(st["B"], device=n.device), n, output_size=st["N"])
    return seq, torch.arange(st["N"], device=n.device) - (n.cumsum(0) - st["lengths"])[seq]


def _plain_append(st):
    qkv, Hq, Hkv, page, N = (st[s] for s in ("qkv", "Hq", "Hkv", "page", "N"))
    seq, row = _places(st)
    cis = st["cis"][row][:, None]
    qk = _turn(qkv[:N, :Hq + Hkv], cis.real, cis.imag, st["layout"]).to(qkv.dtype)
    at = st["pages"][seq, row // page].long(), slice(None), row % page
    st["k"][at], st["v"][at] = qk[:, Hq:], qkv[:N, Hq + Hkv:]
    q = torch.zeros((qkv.shape[0], Hq, st["D"]), device=qkv.device, dtype=qkv.dtype)
    q[:N] = qk[:, :Hq]
    return q, st["k"], st["v"]


def _plain_attention(st):
    q, B, T, Hq, Hkv, D, N, lengths = (st[s] for s in ("q", "B", "T", "Hq", "Hkv", "D", "N", "lengths"))
    seq, row = _places(st)
    t = row - (lengths - st["tokens"])[seq]                        # which of its sequence's new tokens
    x = torch.zeros((B, T, Hq, D), device=q.device)
    x[seq, t] = q[:N].float()
    x = x.view(B, T, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B * Hkv, -1, D)
    k, v = (st[s][st["pages"].clamp(min=0).long()].transpose(1, 2).reshape(B * Hkv, -1, D).float() for s in ("k", "v"))
    rows = torch.arange(k.shape[1], device=q.device)
    last = (lengths - st["tokens"])[:, None] + torch.arange(T, device=q.device)
    seen = (rows <= last[..., None]) & (rows < lengths[:, None, None])
    if st["starts"] is not None:
        seen &= rows >= st["starts"][:, None, None]
    score = (x @ k.transpose(1, 2) * (1.0 / math.sqrt(D))).view(B, Hkv, -1, T, len(rows)).masked_fill_(~seen[:, None, None], float("-inf"))
    p = torch.exp(score - score.amax(-1, keepdim=True))
    o = (p.view(B * Hkv, -1, len(rows)) @ v).view(B, Hkv, -1, T, D) / p.sum(-1, keepdim=True)
    out = torch.zeros_like(q)
    out[:N] = o.permute(0, 3, 1, 2, 4).reshape(B, T, Hq, D)[seq, t].to(q.dtype)
    return out


_PLAIN = {"rope": _plain_rope, "append": _plain_append, "attention": _plain_attention}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------------
def _exact_turn(x, cis, layout, conj=False):
    """x [..., D] in 64 bits, cis [..., R/2] of the same leading sizes."""
    half = cis.shape[-1]
    z = cis.to(torch.complex128)
    y = x.double().clone()
    first, second = (slice(0, half), slice(half, 2 * half)) if layout == "half" else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
    w = torch.complex(y[..., first], y[..., second]) * (z.conj() if conj else z)
    y[..., first], y[..., second] = w.real, w.imag
    return y


def exact(case, seed):
    global own
    mode, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = mode
    kind = case["kind"]
    if kind == "rope":
        x = st["x"]
        cis = st["cis"][st["positions"].expand(x.shape[:2])].unsqueeze(2).expand(*x.shape[:3], -1)
        y = _exact_turn(x, cis, case["layout"])
        return (y, _exact_turn(st["g"], cis, case["layout"], conj=True)) if case["grad"] else y
    Hq, Hkv, D, page = case["Hq"], case["Hkv"], case["D"], case["page"]
    pages, lengths = st["pages"].tolist(), st["lengths"].tolist()
    starts = [0] * case["B"] if st.get("starts") is None else st["starts"].tolist()
    sequences, begin = list(zip(_tokens(case), lengths, starts)), 0
    if kind == "append":
        q = torch.zeros((st["qkv"].shape[0], Hq, D), dtype=torch.float64, device="cuda")
        k, v = st["k"].double(), st["v"].double()
        for b, (n, length, _) in enumerate(sequences):
            x = st["qkv"][begin:begin + n]
            turned = _exact_turn(x[:, :Hq + Hkv], st["cis"][length - n:length, None].expand(-1, Hq + Hkv, -1), case["layout"])
            q[begin:begin + n] = turned[:, :Hq]
            r = length - n
            while r < length:                                      # page by page
                m = min(length, (r // page + 1) * page) - r
                part = slice(r - length + n, r - length + n + m)
                at = pages[b][r // page], slice(None), slice(r % page, r % page + m)
                k[at], v[at] = turned[part, Hq:].transpose(0, 1), x[part, Hq + Hkv:].double().transpose(0, 1)
                r += m
            begin += n
        return q, k, v
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    for b, (n, length, start) in enumerate(sequences):
        rows = torch.arange(start, length, device="cuda")
        number, place = st["pages"][b].long()[rows // page], rows % page
        hidden = rows[None] > (length - n + torch.arange(n, device="cuda"))[:, None]
        for h in range(Hq):
            k, v = (st[s][number, h // (Hq // Hkv), place].double() for s in ("k", "v"))
            score = torch.einsum("td,ld->tl", st["q"][begin:begin + n, h].double(), k) / math.sqrt(D)
            out[begin:begin + n, h] = torch.softmax(score.masked_fill_(hidden, -math.inf), -1) @ v
        begin += n
    return out


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------
def work(case):
    D = case["D"]
    if case["kind"] == "rope":
        B, T, H, R = (case[n] for n in ("B", "T", "H", "R"))
        size, passes = 4 if case["dtype"] == "fp32" else 2, 2 if case["grad"] else 1
        angles = T if case["rows"] == T else B * T
        return {"bytes": passes * 2 * size * B * T * H * D + 4 * angles * R, "flops": passes * 3 * B * T * H * R}
    B, Hq, Hkv, L = (case[n] for n in ("B", "Hq", "Hkv", "L"))
    n = _tokens(case)
    total = sum(n)
    if case["kind"] == "append":              # q/k/v in; q and the new rows of k and v out
        return {"bytes": 4 * total * (Hq + 2 * Hkv) * D + 4 * total * case["R"], "flops": 3 * total * (Hq + Hkv) * case["R"]}
    rows = [L if b == 0 or not case["ragged"] else (L + t) / 2 for b, t in enumerate(n)]              # on average
    if case["starts"]:
        rows = [r - (r - t) / 4 for r, t in zip(rows, n)]
    seen = sum(t * r - t * (t - 1) / 2 for t, r in zip(n, rows))
    return {"bytes": int(4 * Hkv * D * sum(rows) + 4 * total * Hq * D), "flops": int(4 * Hq * D * seen)}
