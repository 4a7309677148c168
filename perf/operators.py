"""Performance cases of the paged key / value cache: what fills it and what reads it, over the ranges a server runs them in.

    append    a step's keys and values rotated and written to their pages, its queries rotated (q4_0 caches hand back what the
              tokens' rows hold: what a program that moves a sequence elsewhere reads)
    attend    the step's queries over the pages: causal, with a sliding window and first tokens that stay visible, over caches of 16
              bits and of 4 bits; one token a sequence (decoding), prompts, and prompts that continue a cached one

A sequence s of a step has token_start[s + 1] - token_start[s] new tokens, the last of the lengths[s] that it has with them.  Position
p of it lies in row p % P of page page_table[s][p // P].  Rows of a step behind its last sequence are padding and stay as they are."""
from __future__ import annotations

import math

import torch

own = False

IO = {"f32": torch.float32, "bf16": torch.bfloat16}
CACHE = {"f16": torch.float16, "bf16": torch.bfloat16, "q4_0": torch.uint8}


def _case(name, op, cache, io, seqs, new, longest, shortest=None, heads=32, kv_heads=8, dim=128, page=32, window=0, sinks=0, rot=None,
          pairs="adjacent", padding=0):
    """new: new tokens of the longest sequence's kind (1: every sequence decodes); longest, shortest: tokens with the new ones."""
    return {"name": name, "op": op, "cache": cache, "io": io, "seqs": seqs, "new": new, "longest": longest,
            "shortest": longest if shortest is None else shortest, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "window": window, "sinks": sinks, "rot": dim if rot is None else rot, "pairs": pairs, "padding": padding}


def listed():
    return [
        # one token of one conversation enters a cache: nothing but latency
        _case("append_one", "append", "f16", "f32", 1, 1, 715, page=16),
        # a serving step of a prompt budget of 8 k tokens: six prompts of unequal length, padded rows at the end
        _case("append_prompts", "append", "bf16", "bf16", 6, 2200, 2200, 310, page=64, pairs="halves", padding=13),
        # the same into a cache of 4 bits, half of the dimensions rotated
        _case("append_prompts_q4", "append", "q4_0", "f32", 4, 1900, 4100, 1900, page=32, rot=64, pairs="halves"),
        # sixteen conversations of very unequal length decode a token each
        _case("decode", "attend", "f16", "f32", 16, 1, 8192, 512, page=16),
        # one conversation far behind its window: latency
        _case("decode_window_one", "attend", "f16", "f32", 1, 1, 4100, page=16, window=1024, sinks=4),
        # many long conversations, each with a window of 4 k and its first tokens
        _case("decode_window", "attend", "bf16", "bf16", 48, 1, 32768, 2000, page=64, window=4096, sinks=16),
        # one long prompt
        _case("prompt", "attend", "bf16", "bf16", 1, 8192, 8192, page=64),
        # the next portion of a prompt that is cached up to here
        _case("prompt_next", "attend", "f16", "bf16", 1, 512, 16895, page=16),
        # prompts of unequal length under a window
        _case("prompts_window", "attend", "bf16", "bf16", 5, 3000, 3000, 129, page=32, window=1024, sinks=4, heads=16, kv_heads=4, dim=64, padding=7),
        # one conversation over a cache of 4 bits
        _case("decode_q4_one", "attend", "q4_0", "f32", 1, 1, 2049, page=32),
        # a full server over caches of 4 bits
        _case("decode_q4", "attend", "q4_0", "bf16", 64, 1, 16384, 1024, page=64),
        # portions of prompts over cached ones in 4 bits
        _case("prompt_next_q4", "attend", "q4_0", "bf16", 3, 700, 6000, 700, page=32, heads=28, kv_heads=4),
    ]


def draw(rng):
    def log(a, b):
        return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))

    op = rng.choice(["append", "attend", "attend", "attend"])
    cache, io = rng.choice(["f16", "bf16", "q4_0"]), rng.choice(["f32", "bf16"])
    kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 7, 8])
    dim, page = rng.choice([64, 128]), rng.choice([16, 32, 64, 128])
    kind = rng.choice(["decode", "decode", "prompt"]) if op == "attend" else rng.choice(["decode", "prompt"])
    if kind == "decode":
        seqs, new = log(1, 64), rng.choice([1, 1, 1, 2, 5])
        longest = log(max(8, new), 16384)
        shortest = rng.randint(max(1, new), longest)
    else:
        seqs = rng.randint(1, 6)
        new = log(9, 2048 // seqs + 9) if io == "bf16" or op == "append" else log(9, 300)
        longest = new + (log(1, 8192) if rng.random() < 0.5 else 0)
        shortest = rng.randint(min(9, longest), longest)
    window = log(16, 4096) if rng.random() < 0.4 else 0
    return {"op": op, "cache": cache, "io": io, "seqs": seqs, "new": new, "longest": longest, "shortest": shortest, "heads": kv_heads * group,
            "kv_heads": kv_heads, "dim": dim, "page": page, "window": window, "sinks": rng.choice([0, 1, 4, 64]) if window else 0,
            "rot": rng.choice([dim, dim // 2, 32]), "pairs": rng.choice(["adjacent", "halves"]), "padding": rng.choice([0, 0, 3])}


def _lengths(case):
    """(lengths, new tokens) of every sequence: evenly spread between the shortest and the longest, in an order that is neither"""
    n, a, b = case["seqs"], case["shortest"], case["longest"]
    lens = [b if n == 1 else a + (b - a) * ((i * 7 + 3) % n) // (n - 1) if n % 7 else a + (b - a) * i // (n - 1) for i in range(n)]
    news = [min(case["new"], x) if i % 2 == 0 else max(1, min(case["new"], x) - i % 5) if case["new"] > 8 else min(case["new"], x) for i, x in enumerate(lens)]
    return lens, news


def _seen(case, length, new):
    """(rows of the cache that some query sees, sum over queries of what each sees)"""
    w, s = case["window"], case["sinks"]
    if not w:
        return length, sum(range(length - new + 1, length + 1))
    lo = max(0, length - new - w + 1)
    rows = length - lo + min(s, lo)
    pairs = 0
    for p in range(length - new, length):
        a = max(0, p - w + 1)
        pairs += p - a + 1 + min(s, a)
    return rows, pairs


def _row_bytes(case):
    return case["dim"] // 2 + case["dim"] // 16 if case["cache"] == "q4_0" else 2 * case["dim"]


def work(case):
    lens, news = _lengths(case)
    n, e = sum(news), 4 if case["io"] == "f32" else 2
    row, kv = _row_bytes(case), case["kv_heads"]
    if case["op"] == "append":
        moved = n * case["dim"] * e * (2 * case["heads"] + 2 * kv) + 2 * n * kv * row
        if case["cache"] == "q4_0":        # read again, and handed back
            moved += 2 * n * kv * (row + 4 * case["dim"])
        return {"bytes": moved, "flops": 3 * n * case["rot"] * (case["heads"] + kv)}
    seen = [_seen(case, a, b) for a, b in zip(lens, news)]
    return {"bytes": 2 * kv * row * sum(r for r, _ in seen) + 2 * n * case["heads"] * case["dim"] * e,
            "flops": 4 * case["dim"] * case["heads"] * sum(p for _, p in seen)}


# ---- a page of one head in 4 bits: quants [dim / 32][page][16], then scales [page][dim / 32] of fp16 ------------------------------------
# Per 32 dimensions the value of largest size m gives d = m / -8, kept as fp16; byte j holds q[j] and, in its upper half, q[j + 16];
# q = x / d + 8 rounded, 0 .. 15, the quotient from the fp32 reciprocal of d and in 64 bits, since a value next to a border is one step off
# otherwise.


def _quantise(x):
    """x [..., dim] fp32 -> (bytes [..., dim / 32, 16], scales [..., dim / 32] fp16)"""
    b = x.unflatten(-1, (-1, 32))
    m = b.gather(-1, b.abs().argmax(-1, keepdim=True))
    d = m / -8
    inv = torch.where(d == 0, torch.zeros_like(d), 1 / d)
    q = (b.double() * inv.double() + 8.5).floor().clamp(0, 15).to(torch.uint8)
    return q[..., :16] | (q[..., 16:] << 4), d[..., 0].half()


def _pack(x):
    """x [pages, heads, page, dim] fp32 -> a pool of bytes"""
    q, d = _quantise(x)
    return torch.cat([q.transpose(2, 3).flatten(2), d.flatten(2).contiguous().view(torch.uint8)], -1).contiguous()


def _unpack(pool, page, dim):
    """a pool of bytes -> [pages, heads, page, dim] fp32"""
    nb = dim // 32
    q = pool[..., :page * dim // 2].unflatten(-1, (nb, page, 16)).transpose(2, 3)
    d = pool[..., page * dim // 2:].contiguous().view(torch.float16).unflatten(-1, (page, nb)).float()
    q = torch.cat([q & 15, q >> 4], -1).float() - 8
    return (q * d[..., None]).flatten(3)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev = torch.device("cuda")
    lens, news = _lengths(case)
    total, P, D, kv, H, io = sum(news), case["page"], case["dim"], case["kv_heads"], case["heads"], IO[case["io"]]
    per = [-(-x // P) for x in lens]
    cols = max(per)
    n_pages = sum(per) + 3
    order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).int()
    table = torch.full((len(lens), cols), -1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(per):
        table[s, :n] = order[at:at + n]
        at += n
        if case["op"] == "attend" and case["window"]:     # pages that no query sees any more have been given back
            first = max(0, lens[s] - news[s] - case["window"] + 1) // P
            table[s, -(-case["sinks"] // P):first] = -1
    starts = torch.zeros(len(lens) + 1, dtype=torch.int32)
    starts[1:] = torch.tensor(news, dtype=torch.int32).cumsum(0)
    n = total + case["padding"]

    def pool():
        x = torch.randn(n_pages, kv, P, D, device=dev, generator=g)
        return _pack(x) if case["cache"] == "q4_0" else x.to(CACHE[case["cache"]])

    st = {"case": case, "k_pool": pool(), "v_pool": pool(), "table": table.to(dev), "starts": starts.to(dev),
          "lens": torch.tensor(lens, dtype=torch.int32, device=dev), "total": total, "n": n, "max_new": max(news),
          "q": (1.5 * torch.randn(n, H, D, device=dev, generator=g)).to(io), "q_out": torch.zeros(n, H, D, device=dev, dtype=io)}
    if case["op"] == "append":
        st["k"] = torch.randn(n, kv, D, device=dev, generator=g).to(io)
        st["v"] = torch.randn(n, kv, D, device=dev, generator=g).to(io)
        if case["cache"] == "q4_0":
            st["k_rows"], st["v_rows"] = (torch.zeros(n, kv, D, device=dev) for _ in range(2))
    return st


# ---- the plain forms ----------------------------------------------------------------------------------------------------------


def _tokens(st):
    """sequence, position, page and row of every token"""
    i = torch.arange(st["total"], device="cuda")
    s = torch.searchsorted(st["starts"][1:].long(), i, right=True)
    pos = st["lens"][s].long() - st["starts"][s + 1].long() + i
    P = st["case"]["page"]
    return s, pos, st["table"][s, pos // P].long(), pos % P


def _rotate(x, pos, case):
    """x [n, heads, dim] -> the rotated heads in fp32; in 64 bits, for far positions' angles and for values next to a border of 4 bits"""
    R = case["rot"]
    angle = pos.double()[:, None, None] * 10000.0 ** (-torch.arange(0, R, 2, device=x.device, dtype=torch.float64) / R)
    c, s, x = torch.cos(angle), torch.sin(angle), x.double()
    if case["pairs"] == "adjacent":
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        turned = torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
    else:
        a, b = x[..., :R // 2], x[..., R // 2:R]
        turned = torch.cat([a * c - b * s, a * s + b * c], -1)
    return torch.cat([turned, x[..., R:]], -1).float()


def _put(pool, x, page, row, case):
    if case["cache"] != "q4_0":
        pool[page, :, row] = x.to(pool.dtype)
        return
    P, nb = case["page"], case["dim"] // 32
    q, d = _quantise(x)
    quants = pool[..., :P * nb * 16].unflatten(-1, (nb, P, 16))
    quants[page, :, :, row] = q
    pool.view(torch.float16)[..., P * nb * 8:].unflatten(-1, (P, nb))[page, :, row] = d


def _append(st):
    case, n = st["case"], st["total"]
    _, pos, page, row = _tokens(st)
    _put(st["k_pool"], _rotate(st["k"][:n], pos, case), page, row, case)
    _put(st["v_pool"], st["v"][:n].float(), page, row, case)
    st["q_out"][:n] = _rotate(st["q"][:n], pos, case).to(st["q_out"].dtype)
    if case["cache"] != "q4_0":
        return {"q": st["q_out"], "k": st["k_pool"], "v": st["v_pool"]}
    for x in ("k", "v"):
        st[x + "_rows"][:n] = _unpack(st[x + "_pool"][page], case["page"], case["dim"])[torch.arange(n, device="cuda"), :, row]
    return {"q": st["q_out"], "k": st["k_rows"], "v": st["v_rows"]}


def _dense(st, pool):
    """the sequences' rows, [seqs, kv heads, longest, dim] fp32"""
    case = st["case"]
    pool = pool[st["table"].clamp(min=0).long()]
    x = _unpack(pool.flatten(0, 1), case["page"], case["dim"]).unflatten(0, pool.shape[:2]) if case["cache"] == "q4_0" else pool.float()
    return x.transpose(1, 2).flatten(2, 3)


def _attend(st):
    case, T, D = st["case"], st["max_new"], st["case"]["dim"]
    k, v = _dense(st, st["k_pool"]), _dense(st, st["v_pool"])
    S, kv, L = k.shape[:3]
    new = (st["starts"][1:] - st["starts"][:-1]).long()
    t = torch.arange(T, device="cuda")
    i = (st["starts"][:-1].long()[:, None] + t).clamp(max=st["n"] - 1)                 # [S, T]
    pos = st["lens"].long()[:, None] - new[:, None] + t
    key = torch.arange(L, device="cuda")
    see = (key <= pos[..., None]) & (t < new[:, None])[..., None]
    if case["window"]:
        see &= (key > pos[..., None] - case["window"]) | (key < case["sinks"])
    q = st["q"][i].float().unflatten(2, (kv, -1)).permute(0, 2, 3, 1, 4)               # [S, kv, group, T, D]
    p = torch.matmul(q.flatten(2, 3) * (1 / math.sqrt(D)), k.transpose(2, 3)).unflatten(2, (-1, T))
    p = p.masked_fill_(~see[:, None, None], -math.inf)
    top = p.amax(-1, keepdim=True).clamp_(min=-1e30)
    p = p.sub_(top).exp_()
    out = torch.matmul(p.flatten(2, 3), v).unflatten(2, (-1, T)) / p.sum(-1, keepdim=True).clamp_(min=1e-30)
    out = out.permute(0, 3, 1, 2, 4).flatten(2, 3)                                      # [S, T, heads, D]
    real = t < new[:, None]
    st["q_out"][i[real]] = out[real].to(st["q_out"].dtype)
    return st["q_out"]


# ---- the library's ---------------------------------------------------------------------------------------------------------------

_context = None


def _handle(st):
    """(cache over the state's pools, the step's description), made once, as a server keeps them"""
    global _context
    if "handle" not in st:
        import skainet_b200 as skn
        _context = _context or skn.Context(0)
        case = st["case"]
        cache = skn.PagedKVCache(_context, st["k_pool"].shape[0], case["page"], case["kv_heads"], case["dim"], case["cache"], rot_dims=case["rot"],
                                 rot_base=10000.0, rot_pairs=case["pairs"], pools=(st["k_pool"], st["v_pool"]))
        st["handle"] = cache, skn.PagedBatch(st["table"], st["starts"], st["lens"], st["n"], st["max_new"])
    return st["handle"]


def _run_own(st):
    case = st["case"]
    cache, batch = _handle(st)
    if case["op"] == "attend":
        cache.attend_dev(batch, st["q"], st["q_out"], window=case["window"], sinks=case["sinks"])
        return st["q_out"]
    cache.append_dev(batch, st["k"], st["v"], st["q"], st["q_out"])
    if case["cache"] != "q4_0":
        return {"q": st["q_out"], "k": st["k_pool"], "v": st["v_pool"]}
    cache.gather_dev(batch, st["k_rows"], st["v_rows"])
    return {"q": st["q_out"], "k": st["k_rows"], "v": st["v_rows"]}


def run(st):
    if own:
        return _run_own(st)
    return _append(st) if st["case"]["op"] == "append" else _attend(st)


# ---- from the definition, in 64 bits -------------------------------------------------------------------------------------------------


def _exact_rows(x, cache):
    """what a cache holds of the fp32 rows x [..., dim], as fp64"""
    if cache != "q4_0":
        return x.to(CACHE[cache]).double()
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for b in range(0, x.shape[-1], 32):
        v = x[..., b:b + 32]
        top = torch.take_along_dim(v, v.abs().argmax(-1, keepdim=True), -1)
        d = top / -8.0
        inv = torch.nan_to_num(d.reciprocal(), posinf=0.0, neginf=0.0)
        q = torch.trunc(v.double() * inv.double() + 8.5).clamp(0, 15)
        out[..., b:b + 32] = (q - 8) * d.half().double()
    return out


def exact(case, seed):
    st = prepare(case, seed)
    lens, news = _lengths(case)
    P, D, kv = case["page"], case["dim"], case["kv_heads"]
    group = case["heads"] // kv
    if case["op"] == "append":
        R = case["rot"]
        pos = torch.cat([torch.arange(a - b, a, device="cuda", dtype=torch.float64) for a, b in zip(lens, news)])
        first = [2 * j if case["pairs"] == "adjacent" else j for j in range(R // 2)]
        other = [2 * j + 1 if case["pairs"] == "adjacent" else j + R // 2 for j in range(R // 2)]
        turn = torch.exp(1j * pos[:, None] * torch.tensor([10000.0 ** (-2 * j / R) for j in range(R // 2)], device="cuda", dtype=torch.float64))[:, None]

        def rotated(x):
            y = x[:st["total"]].double()
            z = torch.complex(y[..., first], y[..., other]) * turn
            y[..., first], y[..., other] = z.real, z.imag
            return y

        n, q = st["total"], st["q_out"].double()
        q[:n] = rotated(st["q"])
        rows = [_exact_rows(x.float(), case["cache"]) for x in (rotated(st["k"]), st["v"][:n].double())]
        if case["cache"] == "q4_0":
            return {"q": q} | {k: torch.cat([r, r.new_zeros(st["n"] - n, kv, D)]) for k, r in zip("kv", rows)}
        got = {"q": q}
        for name, r in zip("kv", rows):
            pool, at = st[name + "_pool"].double(), 0
            for s, (a, b) in enumerate(zip(lens, news)):
                p = torch.arange(a - b, a, device="cuda")
                pool[st["table"][s, p // P].long(), :, p % P] = r[at:at + b]
                at += b
            got[name] = pool
        return got
    out, at = st["q_out"].double(), 0
    for s, (a, b) in enumerate(zip(lens, news)):
        pages = st["table"][s, :-(-a // P)].long()
        kept = torch.arange(a, device="cuda")[pages.repeat_interleave(P)[:a] >= 0]
        for h in range(kv):
            k, v = ((_exact_held(x[pages.clamp(min=0), h], case)).reshape(-1, D)[kept] for x in (st["k_pool"], st["v_pool"]))
            for t in range(0, b, 1024):
                e = min(b, t + 1024)
                q = st["q"][at + t:at + e, h * group:(h + 1) * group].double()
                p = torch.arange(a - b + t, a - b + e, device="cuda")[:, None]
                hidden = kept > p
                if case["window"]:
                    hidden |= (kept <= p - case["window"]) & (kept >= case["sinks"])
                z = (torch.einsum("tgd,kd->tgk", q, k) / math.sqrt(D)).masked_fill(hidden[:, None], -math.inf)
                out[at + t:at + e, h * group:(h + 1) * group] = torch.softmax(z, -1) @ v
        at += b
    return out


def _exact_held(pages, case):
    """[pages, ...] of one head -> [pages, page, dim] fp64"""
    if case["cache"] != "q4_0":
        return pages.double()
    P, nb = case["page"], case["dim"] // 32
    out = torch.empty(pages.shape[0], P, case["dim"], dtype=torch.float64, device=pages.device)
    d = pages[:, P * nb * 16:].contiguous().view(torch.float16).reshape(-1, P, nb).double()
    for b in range(nb):
        raw = pages[:, b * P * 16:(b + 1) * P * 16].reshape(-1, P, 16)
        out[:, :, 32 * b:32 * b + 16] = (torch.bitwise_and(raw, 15).double() - 8) * d[:, :, b, None]
        out[:, :, 32 * b + 16:32 * b + 32] = (torch.div(raw, 16, rounding_mode="floor").double() - 8) * d[:, :, b, None]
    return out
