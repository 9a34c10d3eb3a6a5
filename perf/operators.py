"""The operators of a batched decode step over a paged 8-bit KV cache, as measured cases: block tables and slot maps built
on the GPU, the append into the cache, attention over it, and sampling with parameters of each row.

Each case is prepared as a serving loop would have it in hand (torch tensors on the GPU, in the layouts that include/gq.h
documents), runs in plain torch where ``own`` is false and through grilly2_b200's public calls where it is true.

The pool's layouts (one layer): k int8 [blocks][kv_heads][block_size / 8][dim / 16][8][16], v int8
[blocks][kv_heads][dim / 8][block_size / 16][8][16] (the value transposed), kscale / vscale float32 [blocks][kv_heads].
What is cached is code * scale."""
import math

import torch

own = False

_TINY = 1.0e-30  # smaller than any scale that the cases hold


def listed():
    return [
        # one step of eight running requests: the smallest call, all latency
        {"name": "plan decode 8", "op": "plan", "seqs": 8, "block": 64, "cached_lo": 40, "cached_hi": 1000, "count_lo": 1, "count_hi": 1, "pad": 0},
        # a thousand requests, some with long prompts, some finished (no token), a padded token budget
        {"name": "plan mixed 1000", "op": "plan", "seqs": 1000, "block": 32, "cached_lo": 0, "cached_hi": 3000, "count_lo": 0, "count_hi": 100, "pad": 777},
        # one token of each of 64 requests, the heads of the repository's own decoder configuration
        {"name": "append decode 64", "op": "append", "seqs": 64, "heads": 14, "kv_heads": 2, "dim": 64, "block": 64, "cached_lo": 1, "cached_hi": 1500,
         "count_lo": 1, "count_hi": 1, "pad": 0},
        # ragged prompts that continue cached prefixes, wide heads
        {"name": "append prompts 8", "op": "append", "seqs": 8, "heads": 32, "kv_heads": 8, "dim": 128, "block": 32, "cached_lo": 0, "cached_hi": 700,
         "count_lo": 300, "count_hi": 1700, "pad": 5},
        # a single request: few keys, latency
        {"name": "attend decode 1", "op": "attend", "seqs": 1, "heads": 14, "kv_heads": 2, "dim": 64, "block": 64, "cached_lo": 700, "cached_hi": 700,
         "count_lo": 1, "count_hi": 1, "pad": 0},
        # a batch with ragged lengths, a few just begun
        {"name": "attend decode 64", "op": "attend", "seqs": 64, "heads": 14, "kv_heads": 2, "dim": 64, "block": 64, "cached_lo": 0, "cached_hi": 4095,
         "count_lo": 1, "count_hi": 1, "pad": 0},
        # long contexts, wide heads, large blocks: bytes
        {"name": "attend decode long", "op": "attend", "seqs": 32, "heads": 32, "kv_heads": 8, "dim": 128, "block": 128, "cached_lo": 2000,
         "cached_hi": 15000, "count_lo": 1, "count_hi": 1, "pad": 0},
        # prompts from an empty cache, ragged
        {"name": "attend prompts 5", "op": "attend", "seqs": 5, "heads": 14, "kv_heads": 2, "dim": 64, "block": 64, "cached_lo": 0, "cached_hi": 0,
         "count_lo": 301, "count_hi": 1100, "pad": 3},
        # chunks of prompts over a cached prefix: arithmetic
        {"name": "attend chunk 2", "op": "attend", "seqs": 2, "heads": 32, "kv_heads": 8, "dim": 128, "block": 32, "cached_lo": 2500, "cached_hi": 3333,
         "count_lo": 1024, "count_hi": 1500, "pad": 0},
        # one row, the usual settings
        {"name": "sample 1", "op": "sample", "rows": 1, "vocab": 151936, "top_k": True, "top_p": True, "min_p": False},
        # a batch without top-k: every token is a candidate
        {"name": "sample 64", "op": "sample", "rows": 64, "vocab": 151936, "top_k": False, "top_p": True, "min_p": True},
        # many rows of a smaller, odd vocabulary, settings of all kinds
        {"name": "sample 200", "op": "sample", "rows": 200, "vocab": 32003, "top_k": True, "top_p": True, "min_p": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend", "sample"])
    if op == "sample":
        rows = _log_int(rng, 1, 200)
        return {"op": op, "rows": rows, "vocab": _log_int(rng, 1000, min(151936, 9000000 // rows)), "top_k": rng.random() < 0.5,
                "top_p": rng.random() < 0.7, "min_p": rng.random() < 0.5}
    block = rng.choice([16, 32, 64, 128])
    pad = rng.choice([0, 0, rng.randrange(1, 50)])
    if op == "plan":
        seqs, hi, most = _log_int(rng, 1, 1000), _log_int(rng, 1, 3000), _log_int(rng, 1, 100)
        return {"op": op, "seqs": seqs, "block": block, "cached_lo": rng.randrange(0, hi), "cached_hi": hi, "count_lo": rng.randrange(0, most + 1),
                "count_hi": most, "pad": pad}
    heads, kv_heads, dim = rng.choice([(14, 2, 64), (32, 8, 128), (8, 8, 32), (12, 4, 64), (16, 1, 128), (40, 8, 128), (6, 6, 64)])
    shape = {"op": op, "heads": heads, "kv_heads": kv_heads, "dim": dim, "block": block, "pad": pad}
    if op == "append":
        if rng.random() < 0.5:
            hi = _log_int(rng, 1, 1500)
            return {**shape, "seqs": _log_int(rng, 1, 128), "cached_lo": rng.randrange(0, hi), "cached_hi": hi, "count_lo": 1, "count_hi": 1}
        hi, most = _log_int(rng, 1, 700), _log_int(rng, 2, 1500)
        return {**shape, "seqs": rng.randrange(1, 6), "cached_lo": 0, "cached_hi": hi, "count_lo": rng.randrange(1, most + 1), "count_hi": most}
    if rng.random() < 0.6:  # single tokens: at most as many cached keys and heads as the longest listed case
        seqs = _log_int(rng, 1, 128)
        hi = _log_int(rng, 1, max(2, min(15000, 200000 // (seqs * max(1, kv_heads * dim // 512)))))
        return {**shape, "seqs": seqs, "cached_lo": rng.randrange(0, hi), "cached_hi": hi, "count_lo": 1, "count_hi": 1}
    seqs, most = rng.randrange(1, 5), _log_int(rng, 2, 700)
    hi = _log_int(rng, 1, 2500)
    return {**shape, "seqs": seqs, "cached_lo": rng.randrange(0, hi), "cached_hi": hi, "count_lo": rng.randrange(1, most + 1), "count_hi": most}


# ── what a case holds, the same for every seed ─────────────────────────────


def _spread(lo, hi, n, step):
    """n whole numbers over [lo, hi], the last one hi, in no order."""
    f = [((i + 1) * step) % 1.0 for i in range(n)]
    v = [lo + int((hi - lo) * x * x + 0.5) for x in f]
    v[n // 2] = hi
    return v


def _lengths(case):
    n = case["seqs"]
    cached = _spread(case["cached_lo"], case["cached_hi"], n, 0.6180339887)
    counts = _spread(case["count_lo"], case["count_hi"], n, 0.7548776662)
    return cached, counts


def _geometry(case):
    cached, counts = _lengths(case)
    bs = case["block"]
    total = sum(counts)
    held = [-(-(c + k) // bs) for c, k in zip(cached, counts)]
    return {"cached": cached, "counts": counts, "total": total, "tokens": max(total + case["pad"], 1), "held": held,
            "max_blocks": max(max(held), 1) + 1, "blocks": sum(held) + 7, "runs": _runs_cap(max(total + case["pad"], 1), bs, case["seqs"])}


def _runs_cap(tokens, bs, seqs):
    return min(tokens, tokens // bs + 2 * seqs)


def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + 28 * case["rows"], "flops": 4 * n}
    g = _geometry(case)
    seqs, bs = case["seqs"], case["block"]
    if g["total"] == 0:
        g["total"] = 1
    if case["op"] == "plan":
        touched = sum(-(-(c + k) // bs) - c // bs for c, k in zip(g["cached"], g["counts"]) if k)
        return {"bytes": 4 * (4 * seqs + 3 * touched + 2 * g["tokens"] + g["runs"]), "flops": 4 * g["tokens"]}
    hd, kd = case["heads"] * case["dim"], case["kv_heads"] * case["dim"]
    if case["op"] == "append":
        return {"bytes": g["total"] * (4 * (hd + 2 * kd) + 8 * case["dim"] + 4 * hd + 2 * kd), "flops": g["total"] * (3 * hd + 8 * kd)}
    keys = sum(c + k for c, k in zip(g["cached"], g["counts"]) if k)
    pairs = sum(k * c + k * (k + 1) // 2 for c, k in zip(g["cached"], g["counts"]))
    return {"bytes": keys * 2 * kd + 2 * 4 * case["kv_heads"] * (keys // bs + 1) + 8 * g["total"] * hd, "flops": 4 * pairs * hd}


# ── inputs ─────────────────────────────────────────────────────────────────


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(1000003 * seed + 17)
    if case["op"] == "sample":
        return _prepare_sample(case, gen, dev)
    g = _geometry(case)
    seqs, bs, mb, blocks = case["seqs"], case["block"], g["max_blocks"], g["blocks"]
    st = {"case": dict(case), "g": g}
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    st["lens"], st["counts"] = i32(g["cached"]), i32(g["counts"])
    order = torch.randperm(blocks, generator=gen, device=dev).to(torch.int32)
    j = torch.arange(mb, device=dev)[None]
    if case["op"] == "plan":  # the blocks of what is cached are held, the others are free
        held = i32([-(-c // bs) for c in g["cached"]])[:, None]
    else:
        held = i32(g["held"])[:, None]
    taken = j < held
    at = torch.cumsum(taken.reshape(-1).to(torch.int64), 0).reshape(seqs, mb) - 1
    st["table"] = torch.where(taken, order[at.clamp(min=0)], torch.full_like(at, -1).to(torch.int32)).to(torch.int32).contiguous()
    n_held = int(taken.sum())
    st["free"] = torch.cat([order[n_held:], torch.full((n_held,), -1, dtype=torch.int32, device=dev)]).contiguous()
    st["free_count"] = i32([blocks - n_held])
    for name, n in (("starts", seqs + 1), ("slots", g["tokens"]), ("positions", g["tokens"]), ("runs", g["runs"] + 1), ("last", seqs), ("info", 2)):
        st[name] = torch.zeros(n, dtype=torch.int32, device=dev)
    if case["op"] == "plan":
        return st
    _maps(st)  # the step's maps are in hand before its layers run
    heads, kvh, dim = case["heads"], case["kv_heads"], case["dim"]
    st["k"] = torch.randint(-127, 128, (blocks, kvh, bs // 8, dim // 16, 8, 16), dtype=torch.int8, device=dev, generator=gen)
    st["v"] = torch.randint(-127, 128, (blocks, kvh, dim // 8, bs // 16, 8, 16), dtype=torch.int8, device=dev, generator=gen)
    for name in ("kscale", "vscale"):  # values of about unit size
        st[name] = (torch.rand((blocks, kvh), device=dev, generator=gen) + 0.5) / 73.0
    if case["op"] == "append":
        st["qkv"] = torch.randn((g["tokens"], (heads + 2 * kvh) * dim), device=dev, generator=gen) * 1.5
        longest = mb * bs
        inv = 10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=dev) / dim)
        ang = torch.arange(longest, dtype=torch.float64, device=dev)[:, None] * inv[None]
        ang = torch.cat([ang, ang], 1)
        st["cos"], st["sin"] = ang.cos().float().contiguous(), ang.sin().float().contiguous()
    st["q"] = torch.randn((g["tokens"], heads * dim), device=dev, generator=gen) * 1.5 if case["op"] == "attend" else torch.zeros(
        (g["tokens"], heads * dim), device=dev)
    st["out"] = torch.zeros((g["tokens"], heads * dim), device=dev)
    return st


def _prepare_sample(case, gen, dev):
    rows, vocab = case["rows"], case["vocab"]
    x = torch.randn((rows, vocab), device=dev, generator=gen) * 2.5
    peaks = torch.randint(0, vocab, (rows, 8), device=dev, generator=gen)
    x.scatter_add_(1, peaks, 4.0 + 6.0 * torch.rand((rows, 8), device=dev, generator=gen))
    kept = torch.randint(0, vocab, (rows, 3), device=dev, generator=gen)
    x.scatter_(1, kept, float("-inf"))  # tokens that a grammar forbids
    u = lambda: torch.rand(rows, device=dev, generator=gen)  # noqa: E731
    st = {"case": dict(case), "logits": x.contiguous(), "uniforms": u(), "temperature": 0.6 + 0.7 * u()}
    st["top_k"] = torch.where(u() < 0.8, (1 + 99 * u()).to(torch.int32), torch.zeros(rows, dtype=torch.int32, device=dev)) if case["top_k"] else \
        torch.zeros(rows, dtype=torch.int32, device=dev)
    if case["top_k"] and rows == 1:
        st["top_k"].fill_(50)
    st["top_p"] = 0.8 + 0.19 * u() if case["top_p"] else torch.ones(rows, device=dev)
    st["min_p"] = 0.002 + 0.05 * u() if case["min_p"] else torch.zeros(rows, device=dev)
    st["tokens"] = torch.zeros(rows, dtype=torch.int32, device=dev)
    st["probs"] = torch.zeros(rows, device=dev)
    return st


# ── one pass ───────────────────────────────────────────────────────────────


def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_plain(state):
    return {"plan": _plan, "append": _append, "attend": _attend, "sample": _sample}[state["case"]["op"]](state)


def _outputs(s):
    """What an operator returns: the step's maps and the tables, the updated pool (its codes are whole numbers of the scales
    beside them), the attention's rows, or the tokens."""
    names = {"plan": ("starts", "slots", "positions", "runs", "last", "info", "table", "free_count"), "append": ("q", "k", "v", "kscale", "vscale"),
             "attend": ("out",), "sample": ("tokens", "probs")}[s["case"]["op"]]
    return {n: s[n] for n in names}


def _plan(s):
    _maps(s)
    return _outputs(s)


def _maps(s):
    """Block tables and slot maps: every request's new tokens get positions behind what is cached, a new block where one
    begins (the free list is a stack), and the slot block * block_size + offset."""
    bs, seqs, tokens = s["case"]["block"], s["case"]["seqs"], s["g"]["tokens"]
    table, mb, runs_cap = s["table"], s["g"]["max_blocks"], s["g"]["runs"]
    lens = s["lens"].long().clamp(min=0, max=mb * bs)
    ends = torch.cumsum(s["counts"].long().clamp(min=0), 0).clamp(max=tokens)
    starts = torch.cat([ends.new_zeros(1), ends])
    c = starts[1:] - starts[:-1]
    first, behind = lens // bs, (lens + c + bs - 1) // bs
    j = torch.arange(mb, device=table.device)[None]
    need = (j >= first[:, None]) & (j < behind[:, None]) & (c > 0)[:, None] & (table < 0)
    rank = (torch.cumsum(need.reshape(-1).long(), 0) - 1).reshape(seqs, mb)
    have = s["free_count"].long()
    given = need & (rank < have)
    fresh = s["free"][(have - 1 - rank).clamp(min=0)]
    table.copy_(torch.where(given, fresh, table))
    t = torch.arange(tokens, device=table.device)
    b = torch.searchsorted(ends, t, right=True).clamp(max=seqs - 1)
    valid = t < ends[-1]
    i = t - starts[b]
    p = lens[b] + i
    block = table[b, (p // bs).clamp(max=mb - 1)].long()
    slot = torch.where(valid & (p < mb * bs) & (block >= 0), block * bs + p % bs, -1)
    begins = valid & ((i == 0) | (p % bs == 0))
    where = torch.where(begins, torch.cumsum(begins.long(), 0) - 1, runs_cap + 1)
    runs = torch.full((runs_cap + 2,), 0, dtype=torch.int64, device=table.device) + ends[-1]
    runs.scatter_(0, where, torch.where(begins, t, ends[-1]))
    s["starts"].copy_(starts)
    s["slots"].copy_(slot)
    s["positions"].copy_(torch.where(valid, p, -1))
    s["runs"].copy_(runs[:-1])
    s["last"].copy_(torch.where(c > 0, ends - 1, -1))
    s["info"].copy_(torch.stack([ends[-1], (need & ~given).sum()]))
    s["free_count"].copy_((have - given.sum()).reshape(1))


def _rotate(x, cos, sin):
    """x cos + rot(x) sin, each operation rounded to 32 bits: codes that lie next to a border need the same rounding everywhere."""
    half = x.shape[-1] // 2
    return x * cos + torch.cat([-x[..., half:], x[..., :half]], -1) * sin


def _append(s):
    """Rotary on q and k, then k and v into their blocks: scale = max |value| / 127 over the block's tokens so far; where a
    new token raises it, the codes that are there already are rounded again to the new scale."""
    c, g = s["case"], s["g"]
    n, bs, kvh, dim, heads = g["total"], c["block"], c["kv_heads"], c["dim"], c["heads"]
    qkv = s["qkv"][:n].view(n, heads + 2 * kvh, dim)
    pos = s["positions"][:n].long()
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    s["q"][:n] = _rotate(qkv[:, :heads], cos, sin).reshape(n, -1)
    slot = s["slots"][:n].long()
    block, off = slot // bs, slot % bs
    # each token's run, and its block
    begins = torch.cat([torch.ones_like(off[:1], dtype=torch.bool), (off[1:] == 0) | (block[1:] != block[:-1])])
    run = torch.cumsum(begins.long(), 0) - 1
    runs = g["runs"]
    run_block = torch.full((runs,), g["blocks"], dtype=torch.int64, device=off.device).scatter_(0, run, block)  # behind the last run: no block
    run_first = torch.full((runs,), bs, dtype=torch.int64, device=off.device).scatter_reduce_(0, run, off, "amin")
    lanes = torch.full((), 127.0, device=off.device)  # a tensor: dividing by a number multiplies by its reciprocal
    for name, x in (("k", _rotate(qkv[:, heads:heads + kvh], cos, sin)), ("v", qkv[:, heads + kvh:].contiguous())):
        most = torch.zeros((runs, kvh), device=off.device).scatter_reduce_(0, run[:, None].expand(n, kvh), x.abs().amax(-1), "amax")
        scales = torch.cat([s[name + "scale"], s[name + "scale"].new_zeros(1, kvh)])
        old = torch.where((run_first > 0)[:, None], scales[run_block], torch.zeros_like(most))
        new = torch.maximum(old, most / lanes)
        ratio = torch.where(new > old, old / new, torch.ones_like(new))
        codes = torch.cat([s[name], torch.zeros_like(s[name][:1])])
        codes[run_block] = torch.round(codes[run_block].float() * ratio[:, :, None, None, None, None]).to(torch.int8)
        t = torch.round(x / new[run][:, :, None].clamp(min=_TINY)).clamp(-127, 127).to(torch.int8)
        h, d = torch.arange(kvh, device=off.device)[None, :, None], torch.arange(dim, device=off.device)[None, None]
        bl, of = block[:, None, None], off[:, None, None]
        if name == "k":
            codes[bl, h, of // 8, d // 16, of % 8, d % 16] = t
        else:
            codes[bl, h, d // 8, of // 16, d % 8, of % 16] = t
        s[name].copy_(codes[:-1])
        scales[run_block] = new
        s[name + "scale"].copy_(scales[:-1])
    return _outputs(s)


def _attend(s):
    """softmax(scale q k^T) v over the keys at positions 0 .. the query's own, of the pool's codes times their scales, with
    the requests side by side in a padded batch."""
    c, g = s["case"], s["g"]
    seqs, bs, kvh, dim, heads = c["seqs"], c["block"], c["kv_heads"], c["dim"], c["heads"]
    group, most = heads // kvh, max(max(g["counts"]), 1)
    table = s["table"].long().clamp(min=0)
    nb = max(max(g["held"]), 1)
    table = table[:, :nb]
    k = s["k"][table].permute(0, 2, 1, 3, 5, 4, 6).reshape(seqs, kvh, nb * bs, dim).float()  # [b][h][block][t8][8][d16][16]
    k *= s["kscale"][table].permute(0, 2, 1).repeat_interleave(bs, 2)[..., None]
    i = torch.arange(most, device=table.device)[None]
    rows = s["starts"][:-1].long()[:, None] + i
    alive = i < s["counts"].long()[:, None]
    at = rows.clamp(max=g["tokens"] - 1)
    q = s["q"][at].view(seqs, most, kvh, group, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kvh, group * most, dim)
    a = (q @ k.transpose(-1, -2)).view(seqs, kvh, group, most, nb * bs) * dim ** -0.5
    del k
    pos = s["lens"].long()[:, None] + i
    seen = torch.arange(nb * bs, device=table.device)[None, None] <= pos[..., None]
    a = a.masked_fill(~seen[:, None, None], float("-inf"))
    a = torch.exp(a - a.amax(-1, keepdim=True))
    a = a / a.sum(-1, keepdim=True)
    v = s["v"][table].permute(0, 2, 1, 4, 6, 3, 5).reshape(seqs, kvh, nb * bs, dim).float()  # [b][h][block][t16][16][d8][8]
    v *= s["vscale"][table].permute(0, 2, 1).repeat_interleave(bs, 2)[..., None]
    o = (a.view(seqs, kvh, group * most, nb * bs) @ v).view(seqs, kvh, group, most, dim).permute(0, 3, 1, 2, 4).reshape(seqs, most, heads * dim)
    put = torch.where(alive, at, g["tokens"])
    out = torch.cat([s["out"], s["out"][:1]])
    out[put.reshape(-1)] = o.reshape(seqs * most, -1)
    s["out"].copy_(out[:-1])
    return _outputs(s)


def _sample(s):
    """Temperature, top-k, top-p and min-p, then the draw by the inverse distribution in token order. In 64 bits: a token
    next to a border is kept or dropped by less than 32 bits hold."""
    x = s["logits"].double()
    rows, vocab = x.shape
    top = x.amax(1, keepdim=True)
    w = torch.exp((x - top) / s["temperature"].double()[:, None])
    down, at = torch.sort(x, dim=1, descending=True, stable=True)
    k = s["top_k"].long()
    k = torch.where((k <= 0) | (k > vocab), vocab, k)
    border = down.gather(1, (k - 1)[:, None])
    w = torch.where(x >= border, w, 0.0)
    mass = torch.cumsum(w.gather(1, at), 1)
    before = torch.cat([mass.new_zeros(rows, 1), mass[:, :-1]], 1)
    equal = torch.cat([torch.zeros_like(down[:, :1], dtype=torch.bool), down[:, 1:] == down[:, :-1]], 1)
    before = torch.cummax(torch.where(equal, -1.0, before), 1).values  # the mass above a value: that of the first of its ties
    p = s["top_p"].double()[:, None]
    in_p = (before < p * mass[:, -1:]) | (p >= 1.0)
    in_p[:, 0] = True
    low = torch.where(in_p, down, float("inf")).amin(1, keepdim=True)
    w = torch.where((x >= low) & (w >= s["min_p"].double()[:, None]), w, 0.0)
    up_to = torch.cumsum(w, 1)
    total = up_to[:, -1:]
    chosen = torch.where((up_to > s["uniforms"].double()[:, None] * total) & (w > 0), torch.arange(vocab, device=x.device)[None], vocab).amin(1)
    last = torch.where(w > 0, torch.arange(vocab, device=x.device)[None], -1).amax(1)
    chosen = torch.where(chosen == vocab, last, chosen)
    s["tokens"].copy_(chosen)
    s["probs"].copy_((w.gather(1, chosen.clamp(min=0)[:, None]) / total)[:, 0])
    return _outputs(s)


# ── the framework's calls ──────────────────────────────────────────────────


def _run_own(s):
    api = s.get("api") or _open(s)
    op = s["case"]["op"]
    if op == "plan":
        api["cache"].plan(api["counts"], api["step"])
    elif op == "append":
        api["cache"].append(0, api["qkv"], s["case"]["heads"], api["cos"], api["sin"], api["step"], q_out=api["q"])
    elif op == "attend":
        api["cache"].attend(0, api["q"], s["case"]["heads"], api["step"], max_count=max(s["g"]["counts"]), out=api["out"])
    else:
        api["sample_rows"](api["logits"], api["uniforms"], temperature=api["temperature"], top_k=api["top_k"], top_p=api["top_p"],
                           min_p=api["min_p"], tokens=api["tokens"], probs=api["probs"])
    return _outputs(s)


def _open(s):
    """The handles that a program keeps on its tensors."""
    from grilly2_b200 import _C
    from grilly2_b200.infer.paged import PagedKvCache, PagedStep
    from grilly2_b200.infer.sampling import sample_rows

    def held(name):
        t = s[name]
        if t.dtype is torch.int8:
            t = t.view(torch.int32)
        return _C.Tensor.from_pointer(t.data_ptr(), tuple(t.shape), "int32" if t.dtype is torch.int32 else "float32")

    c, api = s["case"], {"sample_rows": sample_rows}
    if c["op"] == "sample":
        api.update({n: held(n) for n in ("logits", "uniforms", "temperature", "top_k", "top_p", "min_p", "tokens", "probs")})
    else:
        g, names = s["g"], ("table", "lens", "free", "free_count")
        shape = {"kv_heads": c.get("kv_heads", 1), "head_dim": c.get("dim", 32)}
        names += ("k", "v", "kscale", "vscale") if c["op"] != "plan" else ()
        api["cache"] = PagedKvCache(layers=1, blocks=g["blocks"], block_size=c["block"], seqs=c["seqs"], max_blocks=g["max_blocks"],
                                    buffers={n: held(n) for n in names}, **shape)
        api["step"] = PagedStep(api["cache"], g["tokens"], buffers={n: held(n) for n in ("starts", "slots", "positions", "runs", "last", "info")})
        api.update({n: held(n) for n in ("counts", "qkv", "cos", "sin", "q", "out") if n in s})
    s["api"] = api
    return api


# ── the definitions in 64 bits, request by request ─────────────────────────


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "plan":
        return None  # whole numbers
    if op == "append":
        return _exact_append(s)
    return {"out": _exact_attend(s)} if op == "attend" else {"tokens": None, "probs": _exact_probs(s)}


def _exact_append(s):
    c, g = s["case"], s["g"]
    heads, kvh, dim, bs = c["heads"], c["kv_heads"], c["dim"], c["block"]
    q, at = s["q"].double(), 0
    scales = {n: s[n + "scale"].double() for n in "kv"}
    for b, (cached, count) in enumerate(zip(g["cached"], g["counts"])):
        x = s["qkv"][at:at + count].double().view(count, -1, dim)
        swap = torch.cat([-x[..., dim // 2:], x[..., :dim // 2]], 2)
        turned = x * s["cos"][cached:cached + count].double()[:, None] + swap * s["sin"][cached:cached + count].double()[:, None]
        q[at:at + count] = turned[:, :heads].reshape(count, -1)
        parts = {"k": turned[:, heads:heads + kvh], "v": x[:, heads + kvh:]}
        for j in range(cached // bs, -(-(cached + count) // bs)):
            lo, hi = max(j * bs - cached, 0), min((j + 1) * bs - cached, count)
            block = int(s["table"][b, j])
            for n, values in parts.items():
                peak = values[lo:hi].abs().amax((0, 2)) / 127
                scales[n][block] = peak if cached <= j * bs else torch.maximum(scales[n][block], peak)
        at += count
    return {"q": q, "k": None, "v": None, "kscale": scales["k"], "vscale": scales["v"]}


def _exact_attend(s):
    c, g = s["case"], s["g"]
    heads, kvh, dim, bs = c["heads"], c["kv_heads"], c["dim"], c["block"]
    out, at = s["out"].double(), 0
    for b, (cached, count) in enumerate(zip(g["cached"], g["counts"])):
        if not count:
            continue
        n = cached + count
        blocks = s["table"][b, :-(-n // bs)].long()
        for h in range(kvh):
            keys = s["k"][blocks, h].double().transpose(2, 3).reshape(-1, dim)[:n] * s["kscale"][blocks, h].double().repeat_interleave(bs)[:n, None]
            values = s["v"][blocks, h].double().permute(0, 2, 4, 1, 3).reshape(-1, dim)[:n]
            values = values * s["vscale"][blocks, h].double().repeat_interleave(bs)[:n, None]
            for r in range(heads // kvh):
                lo = (h * (heads // kvh) + r) * dim
                logits = s["q"][at:at + count, lo:lo + dim].double() @ keys.T / math.sqrt(dim)
                logits.masked_fill_(torch.ones(count, n, dtype=torch.bool, device=logits.device).triu(cached + 1), -math.inf)
                out[at:at + count, lo:lo + dim] = torch.softmax(logits, 1) @ values
        at += count
    return out


def _exact_probs(s):
    """Row by row on the sorted candidates: each drawn token's share of what is left."""
    probs = []
    for r in range(s["logits"].shape[0]):
        x = s["logits"][r].double()
        keep = torch.isfinite(x)
        k = int(s["top_k"][r])
        if 0 < k < x.numel():
            keep &= x >= torch.topk(x, k).values[-1]
        share = torch.where(keep, torch.softmax((x / float(s["temperature"][r])).masked_fill(~keep, -math.inf), 0), 0.0)
        p = float(s["top_p"][r])
        if p < 1.0:
            values, at = torch.sort(share, descending=True)
            above = torch.cumsum(values, 0) - values
            keep &= share >= values[(above < p).sum().clamp(min=1) - 1]
        keep &= share >= float(s["min_p"][r]) * share.max()
        share = torch.where(keep, share, 0.0)
        share = share / share.sum()
        chosen = int(torch.searchsorted(torch.cumsum(share, 0), float(s["uniforms"][r]), right=True).clamp(max=x.numel() - 1))
        probs.append(share[chosen])
    return torch.stack(probs)
