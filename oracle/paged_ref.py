"""Oracle of the paged int8 KV cache and of sampling by rows: numpy, request by request, attention and sampling in
float64, the stored codes in the float32 steps that include/gq.h states."""
import numpy as np


def pack_k(codes):
    """[..., block, dim] -> the pool's key layout [..., block / 8, dim / 16, 8, 16]."""
    *lead, bs, dim = codes.shape
    return np.ascontiguousarray(np.moveaxis(codes.reshape(*lead, bs // 8, 8, dim // 16, 16), -3, -2))


def pack_v(codes):
    """[..., block, dim] -> the value layout [..., dim / 8, block / 16, 8, 16]."""
    return pack_k(np.swapaxes(codes, -1, -2))


def unpack_k(pool, bs, dim):
    lead = pool.shape[:-4]
    return np.moveaxis(pool, -2, -3).reshape(*lead, bs, dim)


def unpack_v(pool, bs, dim):
    return np.swapaxes(unpack_k(pool, dim, bs), -1, -2)


def runs_cap(tokens, bs, seqs):
    return min(tokens, tokens // bs + 2 * seqs)


def plan(lens, counts, table, free, free_count, bs, blocks, tokens):
    """The step's maps; table (updated in place), free_count after."""
    seqs, mb = table.shape
    refused = 0
    starts, slots, positions, runs, last = [0], np.full(tokens, -1, np.int32), np.full(tokens, -1, np.int32), [], np.full(seqs, -1, np.int32)
    have = min(max(int(free_count), 0), blocks)
    wanted = 0
    for b in range(seqs):
        n, c = min(max(int(lens[b]), 0), mb * bs), min(max(int(counts[b]), 0), tokens - starts[-1])
        row = starts[-1]
        for p in range(n, n + c):
            j = p // bs
            if p == n or p % bs == 0:
                runs.append(row)
                if j < mb and table[b, j] < 0:
                    if p % bs:  # its earlier tokens found no room: a block given now would be read as theirs
                        refused += 1
                    else:
                        if wanted < have:
                            table[b, j] = free[have - 1 - wanted]
                        wanted += 1
            if j < mb and 0 <= table[b, j] < blocks:
                slots[row] = table[b, j] * bs + p % bs
            positions[row] = p
            row += 1
        if c:
            last[b] = row - 1
        starts.append(row)
    cap = runs_cap(tokens, bs, seqs)
    return {"starts": np.array(starts, np.int32), "slots": slots, "positions": positions, "last": last,
            "runs": np.array(runs + [starts[-1]] * (cap + 1 - len(runs)), np.int32),
            "info": np.array([starts[-1], wanted - min(wanted, have) + refused], np.int32)}, have - min(wanted, have)


def rotate(x, cos, sin):
    half = x.shape[-1] // 2
    swap = np.concatenate([-x[..., half:], x[..., :half]], -1)
    with np.errstate(invalid="ignore"):
        return (x * cos).astype(np.float32) + (swap * sin).astype(np.float32)


def append(codes, scales, values, steps, bs):
    """One layer's keys or values: codes int8 [blocks][heads][bs][dim] and scales [blocks][heads] updated in place with the rows
    ``values`` float32 [rows][heads][dim]."""
    slots, runs, total = steps["slots"], steps["runs"], steps["starts"][-1]
    f = np.float32
    with np.errstate(all="ignore"):
        for r in range(len(runs) - 1):
            t0, t1 = int(runs[r]), int(runs[r + 1])
            if t0 >= t1 or t1 > total or slots[t0] < 0:
                continue
            block, off = slots[t0] // bs, slots[t0] % bs
            x = values[t0:t1]
            most = np.abs(x).max((0, 2)).astype(f)
            most[~np.isfinite(x).all((0, 2)) & np.isnan(x).any((0, 2))] = np.nan
            fresh = (most / f(127)).astype(f)
            old = scales[block].copy() if off else np.zeros_like(fresh)
            grows = fresh.view(np.uint32) & 0x7FFFFFFF > old.view(np.uint32) & 0x7FFFFFFF
            new = np.where(grows, fresh, old).astype(f)
            ratio = np.where(grows, (old / new).astype(f), f(1))
            kept = codes[block].astype(f) * ratio[:, None, None]  # the whole block: a new one starts as zeros
            codes[block] = np.nan_to_num(np.rint(kept)).astype(np.int8)
            c = np.where(new[None, :, None] == 0, f(0), (x / new[None, :, None]).astype(f))
            c = np.clip(np.rint(np.nan_to_num(c, nan=0.0, posinf=127, neginf=-127)), -127, 127).astype(np.int8)
            codes[block, :, off:off + t1 - t0] = np.moveaxis(c, 0, 1)
            scales[block] = new


def attend(q, kcodes, vcodes, kscale, vscale, table, lens, steps, scale):
    """float64 attention of every row, and how far a float32 kernel may be from it: [rows][heads][dim] and [rows][heads]. q float32
    [rows][heads][dim]; codes [blocks][kv][bs][dim].

    The allowance, per row and head. A score is off by half a step of q's 23-bit fixed point on every component (2^-22 of
    max|q| times the sum of |k|), by six float32 roundings of its own size and by one of the exponent it becomes, which holds
    log2 of a value scale too; its weight by as much, by 2^-21 for the exponential and by a rounding for each tile of 128 keys that a sum
    runs over. That bears on the weighted values and, through the denominator, on the row itself.
    Beside it the weights are whole numbers of a step: a contribution c = w vscale is off by half of one at most, and by no more
    than itself. The step is 2^-31 of a power of two that lies at most 2^15 above the largest c of the tile and 2^6 above that of the row;
    where a tile's towers over all others' (by more than 2^8) the power has just been set: at most 2^6 above it, or 2 where it
    towers over a quarter of its own tile too. It never lies more than 2^60 below the row's largest (less where value scales are
    so small that the weights' sum needs the room): what the step is then is the bound for all tiles."""
    rows, heads, dim = q.shape
    blocks, kvh, bs, _ = kcodes.shape
    out, tol = np.zeros(q.shape), np.zeros((rows, heads))
    for b in range(len(lens)):
        for t in range(int(steps["starts"][b]), int(steps["starts"][b + 1])):
            n = min(int(lens[b]) + t - int(steps["starts"][b]) + 1, table.shape[1] * bs)
            pos = np.arange(n)
            e = table[b, pos // bs]
            ok = (e >= 0) & (e < blocks)
            e, o = e[ok], pos[ok] % bs
            if not len(e):
                continue
            for h in range(heads):
                g = h // (heads // kvh)
                k = kcodes[e, g, o].astype(np.float64) * kscale[e, g, None].astype(np.float64)
                v = vcodes[e, g, o].astype(np.float64) * vscale[e, g, None].astype(np.float64)
                qd = q[t, h].astype(np.float64)
                s = (k @ qd) * scale
                w = np.exp(s - s.max())
                out[t, h] = (w @ v) / w.sum()
                logs = np.abs(np.log2(np.maximum(vscale[e, g].astype(np.float64), 2.0 ** -100))).max()
                ds = scale * 2.0 ** -22 * np.abs(qd).max() * np.abs(k).sum(1).max() + 2.0 ** -24 * (6 * 1.45 * np.abs(s).max() + logs)
                c, tile = w * vscale[e, g], pos[ok] // 128
                top, quarters = np.zeros(n // 128 + 1), np.zeros((n // 128 + 1, 4))
                np.maximum.at(top, tile, c)
                np.maximum.at(quarters, (tile, pos[ok] % 128 // 32), c)
                most = np.argmax(top)
                step = np.minimum(2.0 ** 15 * top, 2.0 ** 6 * top[most])
                if top[most] > 2.0 ** 8 * np.delete(top, most).max(initial=0.0):
                    step[most] = top[most] * (2.0 if quarters[most].min() < 2.0 ** -10.1 * top[most] else 2.0 ** 6)
                step = np.maximum(step, top[most] * 2.0 ** (6 - min(max(94 - logs, 0), 60)))
                codes = np.abs(vcodes[e, g, o].astype(np.float64)).max(1)
                lost = (np.minimum(c, 2.0 ** -32 * step[tile]) * codes).sum()
                off = ds + 2.0 ** -21 + (n // 128 + 1) * 2.0 ** -24
                tol[t, h] = ((w * np.abs(v).max(1)).sum() / w.sum() + np.abs(out[t, h]).max()) * off + lost / w.sum()
    return out, tol


def sample(x, temperature, top_k, top_p, min_p, u):
    """One row's token and its share of what was kept."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    top = x.max()
    if top == -np.inf:
        return -1, 0.0
    if not temperature > 0:
        i = int(np.argmax(x))
        return i, 1.0 / float((x == top).sum())
    with np.errstate(invalid="ignore"):
        w = np.where(x == top, 1.0, np.exp((x - top) / np.float64(temperature)))
    keep = x > -np.inf
    if 0 < top_k < len(x):
        keep &= x >= np.sort(x)[-top_k]
    if top_p < 1:
        total = w[keep].sum()
        values = np.unique(x[keep])[::-1]
        above = 0.0
        low = values[0]
        for val in values:
            if not above < np.float64(top_p) * total:
                break
            low = val
            above += w[keep & (x == val)].sum()
        keep &= (x >= low)
    keep &= (w >= np.float64(min_p)) | (x == top)
    w = np.where(keep, w, 0.0)
    c = np.cumsum(w)
    hit = np.nonzero((c > np.float64(u) * c[-1]) & (w > 0))[0]
    i = int(hit[0]) if len(hit) else int(np.nonzero(w > 0)[0][-1])
    return i, w[i] / c[-1]


class PagedDecoderRef:
    """float64 model of a decoder whose requests share a paged int8 cache: oracle.llama_ref's arithmetic with the cached rows as
    the codes and block scales that ``append`` leaves. ``step`` takes the new tokens of every request and returns the logits
    of each one's last token (None where it has none)."""

    def __init__(self, cfg, weights, cos, sin, seqs, block):
        from .llama_ref import DecoderRef
        self.m, self.cfg, self.block, self.seqs = DecoderRef(cfg, weights, cos, sin), cfg, block, seqs
        per = -(-cfg.max_cache_len // block)
        shape = (cfg.num_hidden_layers, seqs * per, cfg.num_key_value_heads)
        self.codes = {n: np.zeros(shape + (block, cfg.head_dim), np.int8) for n in "kv"}
        self.scales = {n: np.zeros(shape, np.float32) for n in "kv"}
        self.table = np.arange(seqs * per, dtype=np.int32).reshape(seqs, per)  # which block holds what does not matter here
        self.lens = np.zeros(seqs, np.int64)

    def step(self, new):
        c, m, D = self.cfg, self.m, self.cfg.head_dim
        counts = [len(t) for t in new]
        steps, _ = plan(self.lens, counts, self.table, [], 0, self.block, self.table.size, max(sum(counts), 1))
        pos = steps["positions"][:sum(counts)]
        h = m.embed[[t for r in new for t in r]].copy()
        norm = lambda x, w: x / np.sqrt((x * x).mean(-1, keepdims=True) + c.rms_norm_eps) * w  # noqa: E731

        def turn(x):
            x = x.reshape(len(pos), -1, D)
            return x * m.cos[pos][:, None] + np.concatenate([-x[..., D // 2:], x[..., :D // 2]], -1) * m.sin[pos][:, None]

        for li, lw in enumerate(m.layers):
            x = norm(h, lw["input_norm"])
            q = turn(x @ lw["q"].T + lw["q_bias"])
            k, v = turn(x @ lw["k"].T + lw["k_bias"]), (x @ lw["v"].T + lw["v_bias"]).reshape(len(pos), -1, D)
            append(self.codes["k"][li], self.scales["k"][li], k.astype(np.float32), steps, self.block)
            append(self.codes["v"][li], self.scales["v"][li], v.astype(np.float32), steps, self.block)
            out, _ = attend(q, self.codes["k"][li], self.codes["v"][li], self.scales["k"][li], self.scales["v"][li], self.table, self.lens, steps,
                            D ** -0.5)
            h = h + out.reshape(len(pos), -1) @ lw["o"].T
            x = norm(h, lw["post_norm"])
            g, u = x @ lw["gate"].T, x @ lw["up"].T
            h = h + (g / (1.0 + np.exp(-g)) * u) @ lw["down"].T
        self.lens = self.lens + counts
        return [m.head @ norm(h[r], m.norm) if r >= 0 else None for r in steps["last"]]
