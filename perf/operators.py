"""The 8-bit cache's operators: calls of its public entry points over the range of sizes that the framework serves.

A case's ``op`` names what is called:

- ``write``: ``ops.qk_norm_rope_write8``, one step's norm, rotation and quantised write of keys and values (LFM3's attention layer between its
  projection and its attention). Outputs: the queries, and the cache's pages as the values that they stand for.
- ``decode`` / ``prompt``: ``ops.attention_kv8_decode`` / ``ops.attention_kv8_prefill``, one layer's attention over the cache for sequences that
  bring one token, or portions of their prompts.
- ``copy``: ``ops.copy_rows``, pages of every layer copied to others: a request forked for another reply.

Widths are those of the LFM3 1.2B-, 350M- and 2.6B-size configurations (32 or 16 heads over 8 of 64) and of the other decoders' heads of 128
(16 over 4).
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
EPS = 1e-5
THETA = 1000000.0
GREATEST = 448.0                  # e4m3's largest value
EXPONENTS = (-40, 40)             # of the blocks' scales
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed() -> list[dict]:
    return [
        # a decode step of a small batch: the smallest write, launch and latency
        dict(name="write decode b8", op="write", dtype="bf16", heads=32, kv_heads=8, dim=64, page=16, seqs=8, new=1, ctx=2048),
        # a whole prompt's keys and values
        dict(name="write prompt 2048", op="write", dtype="bf16", heads=32, kv_heads=8, dim=64, page=16, seqs=1, new=2048, ctx=0),
        # the 32-bit model, three prompts' portions that begin inside pages
        dict(name="write fp32 3x333", op="write", dtype="fp32", heads=16, kv_heads=8, dim=64, page=16, seqs=3, new=333, ctx=1000),
        # one user's decode step: latency
        dict(name="decode b1 2048", op="decode", dtype="bf16", heads=32, kv_heads=8, dim=64, page=16, seqs=1, ctx=2048, window=0),
        # a busy server's decode step, contexts of unequal length
        dict(name="decode b64 3000", op="decode", dtype="bf16", heads=32, kv_heads=8, dim=64, page=16, seqs=64, ctx=3000, window=0),
        # a few users far into long documents
        dict(name="decode b8 32000", op="decode", dtype="bf16", heads=16, kv_heads=8, dim=64, page=16, seqs=8, ctx=32000, window=0),
        # a layer with a window and heads of 128
        dict(name="decode b16 window", op="decode", dtype="bf16", heads=16, kv_heads=4, dim=128, page=16, seqs=16, ctx=5000, window=1024),
        # the time to the first token
        dict(name="prompt 2048", op="prompt", dtype="bf16", heads=32, kv_heads=8, dim=64, page=16, seqs=1, new=2048, ctx=0, window=0),
        # a portion far into a long prompt
        dict(name="prompt 512@8192", op="prompt", dtype="bf16", heads=32, kv_heads=8, dim=64, page=16, seqs=1, new=512, ctx=8192, window=0),
        # the 32-bit model reading two short prompts of odd length
        dict(name="prompt fp32 2x301", op="prompt", dtype="fp32", heads=16, kv_heads=8, dim=64, page=16, seqs=2, new=301, ctx=77, window=0),
        # one request forked: the page that it is filling, in the six attention layers of the 1.2B size
        dict(name="copy 1 page", op="copy", dtype="fp8", kv_heads=8, dim=64, page=16, layers=6, pages=1024, pairs=1),
        # sequences moved to other pages, in a 16-bit cache
        dict(name="copy 512 pages", op="copy", dtype="bf16", kv_heads=8, dim=64, page=16, layers=6, pages=2048, pairs=512),
    ]


def _log(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    op = rng.choice(("write", "decode", "decode", "prompt", "prompt", "copy"))
    page = rng.choice((8, 16, 16, 32, 64))
    if op == "copy":
        case = dict(op=op, dtype=rng.choice(("bf16", "fp32", "fp8")), kv_heads=rng.choice((2, 4, 8)), dim=rng.choice((64, 128)), page=page,
                    layers=rng.randint(1, 8), pages=512)
        most = work(case | {"pairs": 1})["bytes"]
        return case | {"pairs": _log(rng, 1, max(1, min(250, (200 << 20) // most)))}
    dtype, dim = rng.choice(("bf16", "bf16", "fp32")), rng.choice((64, 64, 128))
    kv_heads = rng.choice((1, 2, 4, 8))
    group = rng.choice([g for g in (1, 2, 3, 4, 8) if kv_heads * g * dim <= 2048])
    case = dict(op=op, dtype=dtype, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, page=page)
    if op == "write":
        new = _log(rng, 1, 1024)
        case |= dict(seqs=_log(rng, 1, max(1, min(64, 1024 // new))), new=new, ctx=_log(rng, 1, 20000) - 1)
    elif op == "decode":
        ctx = _log(rng, 1, 30000)
        case |= dict(seqs=_log(rng, 1, max(1, min(64, 100000 // ctx))), ctx=ctx, window=rng.choice((0, 0, _log(rng, 16, 2048))))
    else:
        new = _log(rng, 2, 900)
        ctx = _log(rng, 1, 4000) - 1
        case |= dict(seqs=rng.randint(1, max(1, min(4, 1000 // new))), new=new, ctx=ctx, window=rng.choice((0, 0, _log(rng, 16, 2048))))
    return case


def lengths(case: dict) -> list[tuple[int, int]]:
    """(positions cached, new tokens) of each sequence: unequal where there are several."""
    out = []
    for i in range(case["seqs"]):
        new = max(1, case.get("new", 1) - (i * 37) % max(1, case.get("new", 1) // 2))
        out.append((max(0, case["ctx"] - (i * 131) % max(1, case["ctx"] // 2)), new))
    return out


def seen(case: dict) -> tuple[int, int]:
    """(pairs of a query and a key that it sees, keys that at least one query sees)."""
    pairs = keys = 0
    window = case.get("window") or 1 << 30
    for ctx, new in lengths(case):
        pairs += sum(min(ctx + t + 1, window) for t in range(new))
        keys += ctx + new - max(0, ctx + 1 - window)
    return pairs, keys


def work(case: dict) -> dict:
    if case["op"] == "copy":
        size = {"bf16": 2, "fp32": 4, "fp8": 1}[case["dtype"]]
        row = 2 * case["kv_heads"] * case["page"] * case["dim"] * size + (8 * case["kv_heads"] if case["dtype"] == "fp8" else 0)
        return {"bytes": 2 * case["pairs"] * case["layers"] * row, "flops": 0}
    H, G, D, P = case["heads"], case["kv_heads"], case["dim"], case["page"]
    size = 2 if case["dtype"] == "bf16" else 4
    tokens = sum(n for _, n in lengths(case))
    if case["op"] == "write":
        blocks = sum((c + n - 1) // P - c // P + 1 for c, n in lengths(case))
        return {"bytes": tokens * ((2 * H + 2 * G) * D * size + 2 * G * D) + blocks * 2 * G * 4, "flops": tokens * (H + 2 * G) * D * 6}
    pairs, keys = seen(case)
    return {"bytes": keys * 2 * G * D + keys // P * 8 * G + tokens * 2 * H * D * size, "flops": 4 * D * H * pairs}


# ---- inputs ----

def _e4m3(shape, gen) -> torch.Tensor:
    """Bytes as blocks of unit-variance keys and values have them under scales around 2^-7."""
    return (torch.randn(shape, generator=gen, device=DEVICE) * 110).clamp_(-GREATEST, GREATEST).to(torch.float8_e4m3fn)


def _scales(shape, gen) -> torch.Tensor:
    return torch.exp2(torch.randint(-8, -5, shape, generator=gen, device=DEVICE).float())


def _ints(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    if case["op"] == "copy":
        # (a cache's pages in every layer; the pairs are the plan of the cache's books, on the host)
        order = torch.randperm(case["pages"] - 1, generator=torch.Generator().manual_seed(seed)) + 1
        src, dst = order[:case["pairs"]].tolist(), order[case["pairs"]:2 * case["pairs"]].tolist()
        shape = (case["pages"], 2, case["kv_heads"], case["page"], case["dim"])
        pools = []
        for _ in range(case["layers"]):
            if case["dtype"] == "fp8":
                pools += [_e4m3(shape, gen).view(torch.uint8), _scales(shape[:3], gen)]
            else:
                pools.append(torch.randn(shape, generator=gen, device=DEVICE).to(DTYPES[case["dtype"]]))
        return {"case": case, "pools": pools, "src": src, "dst": dst}
    H, G, D, P = case["heads"], case["kv_heads"], case["dim"], case["page"]
    dtype = DTYPES[case["dtype"]]
    lens = lengths(case)
    T = sum(n for _, n in lens)
    state = {"case": case, "window": case.get("window") or None, "scale": D ** -0.5, "longest": max(c + n for c, n in lens)}
    state["positions"] = _ints([c + t for c, n in lens for t in range(n)])
    state["tok_seq"] = _ints([s for s, (_, n) in enumerate(lens) for _ in range(n)])
    state["lens"], state["ctx"] = _ints([n for _, n in lens]), _ints([c for c, _ in lens])
    # the blocks that the call touches have a page each, in no order; a write follows only those of its new positions
    first = [c // P if case["op"] == "write" else 0 for c, _ in lens]
    blocks = [-(-(c + n) // P) for c, n in lens]
    pages = 1 + sum(b - f for f, b in zip(first, blocks))
    order = (torch.randperm(pages - 1, generator=torch.Generator().manual_seed(seed)) + 1).tolist()
    table = torch.zeros(len(lens), max(blocks), dtype=torch.int32)
    at = 0
    for s, (f, b) in enumerate(zip(first, blocks)):
        table[s, f:b] = torch.tensor(order[at:at + b - f], dtype=torch.int32)
        at += b - f
    state["table"] = table.to(DEVICE)
    state["pool"], state["scales"] = _e4m3((pages, 2, G, P, D), gen), _scales((pages, 2, G), gen)
    raw = state["pool"].view(torch.uint8)
    if case["op"] == "write":
        # behind the positions that are there the pages are empty
        raw[0] = 0
        for s, (c, _) in enumerate(lens):
            raw[table[s, c // P].item(), :, :, c % P:] = 0
            raw[table[s, c // P + 1:].long().tolist()] = 0
        state["scales"][0] = 1.0
        state["qkv"] = torch.randn(T, (H + 2 * G) * D, generator=gen, device=DEVICE).to(dtype)
        state["wq"], state["wk"] = (1 + 0.2 * torch.randn(2, D, generator=gen, device=DEVICE)).unbind(0)
        state["inv_freq"] = (1.0 / (THETA ** (torch.arange(0, D, 2, dtype=torch.float32) / D))).to(DEVICE)
        return state
    # behind a sequence's last position its page holds what nobody wrote: not a number
    for s, (c, n) in enumerate(lens):
        if (c + n) % P:
            raw[table[s, (c + n) // P].item(), :, :, (c + n) % P:] = 0x7F
    state["q"] = torch.randn(T, H, D, generator=gen, device=DEVICE).to(dtype)
    state["out"] = torch.empty_like(state["q"])
    if own and case["op"] == "prompt":
        # the step's layout: runs of so many tokens of one sequence, as the engine cuts them once for all layers
        from tokenomos_b200 import ops
        size = ops.attention_kv8_tokens(H, G, D, P, dtype)
        tiles, start = [], 0
        for _, n in lens:
            tiles += [(start + o, min(size, n - o)) for o in range(0, n, size)]
            start += n
        state["tile_tok0"], state["tile_ntok"] = _ints([t for t, _ in tiles]), _ints([n for _, n in tiles])
    return state


# ---- one pass ----

def run(state: dict):
    op = state["case"]["op"]
    return (_run_own if own else _run_plain)(state, op)


def _run_own(state: dict, op: str):
    from tokenomos_b200 import ops

    s, case = state, state["case"]
    if op == "copy":
        ops.copy_rows(s["pools"], s["src"], s["dst"])
        return s["pools"]
    if op == "write":
        q = ops.qk_norm_rope_write8(s["qkv"], s["pool"], s["scales"], s["wq"], s["wk"], EPS, s["inv_freq"], s["positions"], s["tok_seq"],
                                    s["table"], case["heads"], case["kv_heads"], case["dim"], case["page"])
        return {"q": q, "cache": _values(s["pool"], s["scales"])}
    if op == "decode":
        ops.attention_kv8_decode(s["q"], s["pool"], s["scales"], s["out"], s["positions"], s["tok_seq"], s["table"], None, s["window"],
                                 s["scale"], s["longest"])
    else:
        ops.attention_kv8_prefill(s["q"], s["pool"], s["scales"], s["out"], s["positions"], s["tok_seq"], s["table"], s["tile_tok0"],
                                  s["tile_ntok"], s["window"], s["scale"], s["longest"])
    return s["out"]


def _values(pool: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """What the bytes stand for (bfloat16 holds it exactly)."""
    return pool.to(torch.bfloat16).mul_(scales.to(torch.bfloat16)[..., None, None])


def _run_plain(state: dict, op: str):
    if op == "copy":
        src = torch.tensor(state["src"], device=DEVICE)
        dst = torch.tensor(state["dst"], device=DEVICE)
        for pool in state["pools"]:
            pool[dst] = pool[src]
        return state["pools"]
    return _write_plain(state) if op == "write" else _attend_plain(state)


def _norm_rope(x: torch.Tensor, w: torch.Tensor, angles: torch.Tensor) -> torch.Tensor:
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    c, s = angles.cos().float()[:, None], angles.sin().float()[:, None]
    return torch.cat((a * c - b * s, b * c + a * s), -1)


def _write_plain(state: dict):
    case = state["case"]
    H, G, D, P = case["heads"], case["kv_heads"], case["dim"], case["page"]
    pool, old = state["pool"].float(), state["scales"]
    x = state["qkv"].float().view(-1, H + 2 * G, D)
    pos, seq = state["positions"].long(), state["tok_seq"].long()
    angles = pos.double()[:, None] * state["inv_freq"].double()          # (in 64 bits: far positions)
    q = _norm_rope(x[:, :H], state["wq"], angles)
    kv = torch.stack((_norm_rope(x[:, H:H + G], state["wk"], angles), x[:, H + G:]), 1)         # [T, 2, G, D]
    page, at = state["table"].long()[seq, pos // P], pos % P
    reach = kv.abs().amax(-1)
    bad = ~(reach.amax(1) <= GREATEST * 2.0 ** EXPONENTS[1])                                       # [T, G]
    reach = torch.where(bad[:, None], 0.0, reach)
    most = torch.zeros_like(old).scatter_reduce_(0, page[:, None, None].expand_as(reach), reach, "amax")
    m, e = torch.frexp(most)
    e = torch.where(most > 0, torch.where(m <= 0.875, e - 9, e - 8), EXPONENTS[0]).clamp(*EXPONENTS)
    touched = torch.zeros(pool.shape[0], dtype=torch.bool, device=DEVICE)
    touched[page] = True
    fresh = torch.zeros_like(touched)
    fresh[torch.where(at == 0, page, 0)] = True          # (page 0 is nobody's)
    new = torch.exp2(e.float())
    new = torch.where(fresh[:, None, None], new, torch.maximum(new, old))
    new = torch.where(touched[:, None, None], new, old)
    pool = (pool * (old / new)[..., None, None]).to(torch.float8_e4m3fn).float()
    rows = kv / new[page][..., None]
    rows[:, 0] = torch.where(bad[..., None], float("nan"), rows[:, 0])
    rows[:, 1] = torch.where(bad[..., None], 0.0, rows[:, 1])
    pool[page, :, :, at] = rows.to(torch.float8_e4m3fn).float()
    return {"q": q.to(state["qkv"].dtype), "cache": (pool * new[..., None, None]).to(torch.bfloat16)}


def _attend_plain(state: dict) -> torch.Tensor:
    case = state["case"]
    H, G, D, P = case["heads"], case["kv_heads"], case["dim"], case["page"]
    table, S = state["table"].long(), case["seqs"]
    n, ctx = state["lens"].long(), state["ctx"].long()
    L, most = table.shape[1] * P, max(b for _, b in lengths(case))
    kv = state["pool"].view(torch.uint8)[table].view(torch.float8_e4m3fn).float()
    kv = kv * state["scales"][table][..., None, None]                       # [S, blocks, 2, G, P, D]
    kv = kv.permute(2, 0, 3, 1, 4, 5).reshape(2, S, G, L, D)
    j = torch.arange(L, device=DEVICE)
    there = j < (ctx + n)[:, None]                                          # [S, L]
    kv = torch.where(there[None, :, None, :, None], kv, 0.0)
    seq = state["tok_seq"].long()
    row = torch.arange(len(seq), device=DEVICE) - (n.cumsum(0) - n)[seq]
    q = torch.zeros(S, most, H, D, device=DEVICE)
    q[seq, row] = state["q"].float()
    q = q.view(S, most, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(S, G, (H // G) * most, D)
    s = (q @ kv[0].transpose(2, 3)).view(S, G, H // G, most, L) * state["scale"]
    i = ctx[:, None] + torch.arange(most, device=DEVICE)                    # [S, most]
    see = (j <= i[..., None]) & there[:, None]
    if state["window"]:
        see &= j > i[..., None] - state["window"]
    s = s.masked_fill(~see[:, None, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top.isfinite(), top, 0.0))
    total = p.sum(-1, keepdim=True)
    o = (p.view(S, G, -1, L) @ kv[1]).view(S, G, H // G, most, D) / torch.where(total > 0, total, 1.0)
    o = o.permute(0, 3, 1, 2, 4).reshape(S, most, H, D)
    return o[seq, row].to(state["q"].dtype)


# ---- 64 bits, from the definitions ----

def exact(case: dict, seed: int):
    state = prepare(case, seed)
    if case["op"] == "copy":
        return [_copied(p, state["src"], state["dst"]) for p in state["pools"]]
    if case["op"] == "write":
        return _write_exact(case, state)
    return _attend_exact(case, state)


def _copied(pool, src, dst):
    out = pool.clone()
    for a, b in zip(src, dst):
        out[b] = pool[a]
    return out


def _write_exact(case: dict, state: dict):
    """The queries. What the cache holds in 8 bits has no such value: next to the middle between two neighbours the last bit of 32 decides."""
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    x = state["qkv"].double().unflatten(1, (H + 2 * G, D))[:, :H]
    turn = torch.polar(torch.ones(1, dtype=torch.float64, device=DEVICE),
                       state["positions"].double()[:, None] * state["inv_freq"].double())[:, None]
    x = x / (x.square().sum(-1, keepdim=True) / D + EPS).sqrt() * state["wq"].double()
    z = torch.complex(x[..., :D // 2].contiguous(), x[..., D // 2:].contiguous()) * turn
    return {"q": torch.cat((z.real, z.imag), -1), "cache": None}


def _attend_exact(case: dict, state: dict) -> torch.Tensor:
    """Sequence by sequence, some query rows at a time."""
    H, G, D, P = case["heads"], case["kv_heads"], case["dim"], case["page"]
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device=DEVICE)
    start = 0
    for s, (ctx, new) in enumerate(lengths(case)):
        end = ctx + new
        pages = state["table"][s, :-(-end // P)].long()
        rows = state["pool"].view(torch.uint8)[pages].view(torch.float8_e4m3fn).double() * state["scales"][pages].double()[..., None, None]
        k, v = (rows[:, w].transpose(0, 1).reshape(G, -1, D)[:, :end].repeat_interleave(H // G, 0) for w in (0, 1))
        for a in range(0, new, 256):
            b = min(new, a + 256)
            at = torch.arange(ctx + a, ctx + b, device=DEVICE)[:, None]
            keys = torch.arange(end, device=DEVICE)
            hidden = (keys > at) | ((keys <= at - case["window"]) if case["window"] else (keys < 0))
            x = torch.einsum("thd,hkd->htk", state["q"][start + a:start + b].double(), k) * state["scale"]
            x = torch.softmax(x.masked_fill(hidden, -math.inf), -1)
            out[start + a:start + b] = torch.einsum("htk,hkd->thd", x, v)
        start += new
    return out
