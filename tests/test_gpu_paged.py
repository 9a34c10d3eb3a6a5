"""The paged int8 KV cache: maps, append and attention against the numpy checker (oracle/paged_ref.py), through the Python
calls. Codes, scales and maps must be equal; attention is held to the allowance that the checker derives row by row."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _env():
    from grilly2_b200 import _C
    from grilly2_b200.infer.paged import PagedKvCache, PagedStep
    from oracle import paged_ref
    return _C, PagedKvCache, PagedStep, paged_ref


def dev(a):
    from grilly2_b200 import _C
    return _C.Tensor.from_numpy(np.ascontiguousarray(a))


def words(codes):
    return dev(codes.reshape(-1).view(np.int32))


def maps(step):
    return {n: getattr(step, n).numpy() for n in ("starts", "slots", "positions", "runs", "last", "info")}


def tables_for(rng, held, mb, blocks):
    """A table in which request b holds held[b] blocks in shuffled order, and the free list of the others."""
    order = rng.permutation(blocks).astype(np.int32)
    table, at = np.full((len(held), mb), -1, np.int32), 0
    for b, h in enumerate(held):
        table[b, :h] = order[at:at + h]
        at += h
    free = np.full(blocks, -1, np.int32)
    free[:blocks - at] = order[at:]
    return table, free, blocks - at


# ── block tables and slot maps ─────────────────────────────────────────────

PLANS = {
    "one token": dict(bs=16, lens=[0], counts=[1], mb=2, blocks=4, tokens=1),
    "decode": dict(bs=64, lens=[63, 64, 65, 0, 127], counts=[1] * 5, mb=3, blocks=40, tokens=5),
    "ragged prompts": dict(bs=16, lens=[5, 0, 33, 16], counts=[40, 17, 0, 16], mb=9, blocks=64, tokens=90),
    "nothing": dict(bs=32, lens=[3, 9], counts=[0, -4], mb=2, blocks=4, tokens=8),
    "cut rows": dict(bs=16, lens=[1, 2, 3], counts=[10, 30, 5], mb=4, blocks=30, tokens=23),
    "beyond the table": dict(bs=16, lens=[30, 31, 90], counts=[5, 1, 3], mb=2, blocks=30, tokens=12),
    "empty free list": dict(bs=16, lens=[0, 0, 0], counts=[33, 20, 1], mb=4, blocks=4, tokens=60),
    "many requests": dict(bs=32, lens=list(range(1500)), counts=[i % 4 for i in range(1500)], mb=50, blocks=60000, tokens=2500),
    "a long prompt": dict(bs=16, lens=[7, 3], counts=[1, 40000], mb=2600, blocks=3000, tokens=40100),
    "4096 requests": dict(bs=128, lens=[i * 37 % 300 for i in range(4096)], counts=[1 + i % 3 for i in range(4096)], mb=4, blocks=17000, tokens=9000),
}


@pytest.mark.parametrize("name", PLANS)
def test_plan_equals_the_checker_and_repeats(name):
    _C, PagedKvCache, PagedStep, ref = _env()
    p = PLANS[name]
    rng = np.random.default_rng(len(name))
    held = [min(-(-max(n, 0) // p["bs"]), p["mb"]) for n in p["lens"]]
    table, free, count = tables_for(rng, held, p["mb"], p["blocks"])
    cache = PagedKvCache(layers=1, kv_heads=1, head_dim=32, blocks=p["blocks"], seqs=len(p["lens"]), max_blocks=p["mb"], block_size=p["bs"],
                         buffers={"table": dev(table), "free": dev(free), "free_count": dev(np.array([count], np.int32)),
                                  "lens": dev(np.array(p["lens"], np.int32))})
    step = PagedStep(cache, p["tokens"])
    want, left = ref.plan(p["lens"], p["counts"], table, free, count, p["bs"], p["blocks"], p["tokens"])
    for again in range(2):  # the second call finds every block in place
        cache.plan(dev(np.array(p["counts"], np.int32)), step)
        got = maps(step)
        if again:
            want["info"][1] = max(0, want["info"][1] - left)
        for n in want:
            np.testing.assert_array_equal(got[n], want[n], err_msg=f"{n} ({name}, call {again})")
        np.testing.assert_array_equal(cache.table.numpy(), table)
        assert cache.free_blocks() == left
    cap = p["mb"] * p["bs"]
    cache.advance(step)
    rows = np.diff(want["starts"])
    clipped = np.clip(np.array(p["lens"]), 0, cap)
    np.testing.assert_array_equal(cache.lengths(), np.where(rows > 0, np.minimum(clipped + rows, cap), p["lens"]))


def test_entries_outside_the_pool_count_as_no_block():
    _C, PagedKvCache, PagedStep, ref = _env()
    table = np.array([[7, -1], [1, -1], [-9, 2]], np.int32)
    cache = PagedKvCache(layers=1, kv_heads=1, head_dim=32, blocks=5, seqs=3, max_blocks=2, block_size=16,
                         buffers={"table": dev(table), "lens": dev(np.array([3, 3, 20], np.int32)),
                                  "free_count": dev(np.array([1 << 30], np.int32)), "free": dev(np.array([4, 3, 2, 1, 99], np.int32))})
    step = PagedStep(cache, 8)
    cache.plan(dev(np.array([1, 14, 2], np.int32)), step)
    got = maps(step)
    want, _ = ref.plan([3, 3, 20], [1, 14, 2], table, [4, 3, 2, 1, 99], 1 << 30, 16, 5, 8)
    np.testing.assert_array_equal(got["slots"], want["slots"])
    assert got["slots"][0] == -1


def test_release_gives_the_blocks_back_and_they_are_taken_again():
    _C, PagedKvCache, PagedStep, ref = _env()
    cache = PagedKvCache(layers=1, kv_heads=1, head_dim=32, blocks=9, seqs=4, max_blocks=3, block_size=16)
    step = PagedStep(cache, 128)
    cache.plan(dev(np.array([40, 1, 17, 16], np.int32)), step)
    cache.advance(step)
    assert cache.free_blocks() == 9 - 3 - 1 - 2 - 1
    before = cache.table.numpy()
    cache.release(dev(np.array([1, 0, 5, 0], np.int32)))
    assert cache.free_blocks() == 7
    table = cache.table.numpy()
    assert (table[[0, 2]] == -1).all() and (table[[1, 3]] == before[[1, 3]]).all()
    np.testing.assert_array_equal(cache.lengths(), [0, 1, 0, 16])
    np.testing.assert_array_equal(cache.free.numpy()[2:7], list(before[0]) + list(before[2][:2]))
    cache.plan(dev(np.array([48, 0, 48, 17], np.int32)), step)
    assert step.shortfall() == 1 and cache.free_blocks() == 0
    held = cache.table.numpy()
    assert len(set(held[held >= 0])) == 9


# ── append ─────────────────────────────────────────────────────────────────


def rotary(mp, dim, rng):
    ang = rng.standard_normal((mp, dim)).astype(np.float32)
    return np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)


class Twin:
    """A cache on the device and the checker's copy of it, stepping together."""

    def __init__(self, rng, *, seqs, heads, kvh, dim, bs, mb, blocks, layers=2, layer=1):
        _C, PagedKvCache, PagedStep, self.ref = _env()
        self.rng, self.heads, self.kvh, self.dim, self.bs, self.layer, self.blocks = rng, heads, kvh, dim, bs, layer, blocks
        self.cache = PagedKvCache(layers=layers, kv_heads=kvh, head_dim=dim, blocks=blocks, seqs=seqs, max_blocks=mb, block_size=bs)
        self.Step = PagedStep
        self.codes = {n: np.zeros((blocks, kvh, bs, dim), np.int8) for n in "kv"}
        self.scales = {n: np.zeros((blocks, kvh), np.float32) for n in "kv"}
        self.lens = np.zeros(seqs, np.int64)
        self.table = np.full((seqs, mb), -1, np.int32)
        self.free, self.count = self.cache.free.numpy(), blocks
        self.cos, self.sin = rotary(mb * bs, dim, rng)

    def step(self, counts, sigma=1.0, pad=0, qkv=None):
        tokens = max(int(np.maximum(counts, 0).sum()) + pad, 1)
        st = self.Step(self.cache, tokens)
        self.cache.plan(dev(np.array(counts, np.int32)), st)
        want, self.count = self.ref.plan(self.lens, counts, self.table, self.free, self.count, self.bs, self.blocks, tokens)
        if qkv is None:
            qkv = (self.rng.standard_normal((tokens, self.heads + 2 * self.kvh, self.dim)) * sigma).astype(np.float32)
        q = _C_filled((tokens, self.heads * self.dim), 7.0)
        self.cache.append(self.layer, dev(qkv.reshape(tokens, -1)), self.heads, dev(self.cos), dev(self.sin), st, q_out=q)
        p = np.minimum(np.maximum(want["positions"], 0), len(self.cos) - 1)
        turned = self.ref.rotate(qkv, self.cos[p][:, None], self.sin[p][:, None])
        n = int(want["starts"][-1])
        self.ref.append(self.codes["k"], self.scales["k"], turned[:, self.heads:self.heads + self.kvh], want, self.bs)
        self.ref.append(self.codes["v"], self.scales["v"], qkv[:, self.heads + self.kvh:], want, self.bs)
        got_q = q.numpy().reshape(tokens, self.heads, self.dim)
        np.testing.assert_array_equal(got_q[:n], turned[:n, :self.heads])
        assert (got_q[n:] == 7.0).all(), "a padded row was written"
        return st, want, turned[:, :self.heads]

    def check_pool(self):
        c = self.cache
        shape = (c.layers, self.blocks, self.kvh)
        k = c.k.numpy().view(np.int8).reshape(*shape, self.bs // 8, self.dim // 16, 8, 16)
        v = c.v.numpy().view(np.int8).reshape(*shape, self.dim // 8, self.bs // 16, 8, 16)
        np.testing.assert_array_equal(self.ref.unpack_k(k[self.layer], self.bs, self.dim), self.codes["k"])
        np.testing.assert_array_equal(self.ref.unpack_v(v[self.layer], self.bs, self.dim), self.codes["v"])
        for n, t in (("k", c.kscale), ("v", c.vscale)):
            np.testing.assert_array_equal(t.numpy().reshape(shape)[self.layer], self.scales[n])
        others = [i for i in range(c.layers) if i != self.layer]
        assert not k[others].any() and not v[others].any() and not c.kscale.numpy().reshape(shape)[others].any(), "another layer was written"

    def advance(self, st, want):
        self.cache.advance(st)
        self.lens = np.minimum(self.lens + np.diff(want["starts"]), self.table.shape[1] * self.bs)
        np.testing.assert_array_equal(self.cache.lengths(), self.lens)

    def check_attention(self, st, want, turned, scale=None, max_count=None):
        c = self.cache
        scale = self.dim ** -0.5 if scale is None else scale
        tokens = st.max_tokens
        out = _C_filled((tokens, self.heads * self.dim), 3.0)
        c.attend(self.layer, dev(turned.reshape(tokens, -1)), self.heads, st, scale=scale, max_count=max_count, out=out)
        got = out.numpy().reshape(tokens, self.heads, self.dim)
        exact, tol = self.ref.attend(turned, self.codes["k"], self.codes["v"], self.scales["k"], self.scales["v"], self.table, self.lens, want, scale)
        n = int(want["starts"][-1])
        assert (got[n:] == 3.0).all(), "a padded row was written"
        off = np.abs(got[:n] - exact[:n]).max(-1) if n else np.zeros((0, self.heads))
        worst = float((off / np.maximum(tol[:n], 1e-30)).max(initial=0.0))
        print(f"[paged attention] worst error / allowance {worst:.3f}")
        assert (off <= tol[:n]).all(), worst


def _C_filled(shape, value):
    return dev(np.full(shape, value, np.float32))


SHAPES = [(14, 2, 64, 64), (4, 4, 32, 16), (8, 1, 128, 32), (6, 2, 128, 128), (5, 1, 64, 16), (3, 3, 32, 128), (16, 1, 128, 64), (40, 1, 64, 32)]


@pytest.mark.parametrize("heads,kvh,dim,bs", SHAPES)
def test_append_and_attention_step_by_step(heads, kvh, dim, bs):
    """Prompts, single tokens of growing size (so that scales grow inside a block), requests without a token, padded rows."""
    t = Twin(np.random.default_rng(heads * dim + bs), seqs=4, heads=heads, kvh=kvh, dim=dim, bs=bs, mb=6, blocks=23)
    for i, counts in enumerate([[bs + 3, 1, 0, 2 * bs], [1, 1, 1, 1], [1, 0, 5, 1], [2, bs, 1, 0], [1, 1, 1, 1]]):
        st, want, turned = t.step(counts, sigma=0.5 * 1.7 ** i, pad=i % 3)
        t.check_pool()
        t.check_attention(st, want, turned, max_count=max(counts))
        t.check_attention(st, want, turned)  # the hint changes nothing that is computed
        t.advance(st, want)


def test_append_zeros_and_values_that_are_no_numbers():
    rng = np.random.default_rng(5)
    t = Twin(rng, seqs=3, heads=2, kvh=2, dim=32, bs=16, mb=2, blocks=6)
    t.cos[:], t.sin[:] = 1.0, 0.0
    qkv = rng.standard_normal((6, 6, 32)).astype(np.float32)
    qkv[0:2, 2:] = 0.0               # a block of zeros: scale 0
    qkv[3, 2, 4] = np.inf            # a key of request 1, head 0
    qkv[5, 5, 9] = np.nan            # a value of request 2, head 1
    st, want, turned = t.step([2, 2, 2], qkv=qkv)
    t.check_pool()
    assert t.scales["k"][want["slots"][0] // 16].max() == 0.0
    t.advance(st, want)
    st, want, turned = t.step([1, 1, 1], sigma=1.0)
    t.check_pool()
    out = t.cache.attend(1, dev(turned.reshape(3, -1)), 2, st, max_count=1).numpy().reshape(3, 2, 32)
    bad = ~np.isfinite(out).all(-1)
    np.testing.assert_array_equal(bad, [[False, False], [True, False], [False, True]])


@pytest.mark.parametrize("size", [1e-43, 3e-39, 1e-30, 0.37, 1e31, 2.5e38])
def test_append_next_to_halves_and_at_the_ends_of_the_range(size):
    """Values on and beside every border between two codes, for scales from the subnormal ones to the largest: the codes are the
    rounded quotients, bit for bit."""
    t = Twin(np.random.default_rng(8), seqs=1, heads=1, kvh=1, dim=128, bs=16, mb=1, blocks=1)
    t.cos[:], t.sin[:] = 1.0, 0.0
    with np.errstate(all="ignore"):
        step = np.float32(size) / np.float32(127)
        border = ((np.arange(-127, 128) + 0.5)[:, None] * step).astype(np.float32)
        x = np.concatenate([np.nextafter(border, np.float32(-np.inf)), border, np.nextafter(border, np.float32(np.inf))], 1).reshape(-1)
    x = np.clip(x, -np.float32(size), np.float32(size))[:6 * 128].reshape(-1)
    rows = -(-x.size // 128)
    x = np.concatenate([x, np.full(rows * 128 - x.size, size, np.float32)]).reshape(rows, 1, 128)
    assert rows <= 16 and np.abs(x).max() == np.float32(size)
    t.step([rows], qkv=np.concatenate([x, x, x], 1))
    t.check_pool()


def test_append_skips_rows_without_room():
    t = Twin(np.random.default_rng(6), seqs=3, heads=2, kvh=1, dim=32, bs=16, mb=2, blocks=3)
    st, want, turned = t.step([40, 3, 20])  # 32 tokens fit the table, three blocks the pool
    assert (want["slots"][:43] == -1).any() and want["info"][1] == 2
    t.check_pool()
    t.check_attention(st, want, turned)  # rows that see no cached key give zeros


# ── attention ──────────────────────────────────────────────────────────────


def filled(rng, heads, kvh, dim, bs, lens, counts, spread=1.0, blocks_more=3):
    """A twin whose pool holds random codes and scales behind tables for lens + counts tokens."""
    need = [-(-(a + c) // bs) for a, c in zip(lens, counts)]
    mb = max(max(need), 1)
    t = Twin(rng, seqs=len(lens), heads=heads, kvh=kvh, dim=dim, bs=bs, mb=mb, blocks=sum(need) + blocks_more, layers=1, layer=0)
    t.table, t.free, t.count = tables_for(rng, need, mb, t.blocks)
    for n in "kv":
        t.codes[n] = rng.integers(-127, 128, t.codes[n].shape).astype(np.int8)
        t.scales[n] = (np.exp(spread * rng.standard_normal(t.scales[n].shape)) / 73).astype(np.float32)
    t.lens = np.array(lens)
    from grilly2_b200.infer.paged import PagedKvCache
    t.cache = PagedKvCache(layers=1, kv_heads=kvh, head_dim=dim, blocks=t.blocks, seqs=len(lens), max_blocks=mb, block_size=bs,
                           buffers={"k": words(t.ref.pack_k(t.codes["k"])), "v": words(t.ref.pack_v(t.codes["v"])), "kscale": dev(t.scales["k"]),
                                    "vscale": dev(t.scales["v"]), "table": dev(t.table), "lens": dev(np.array(lens, np.int32)),
                                    "free": dev(t.free), "free_count": dev(np.array([t.count], np.int32))})
    return t


def attend(t, counts, pad=0, **kw):
    tokens = int(sum(counts)) + pad
    st = t.Step(t.cache, tokens)
    t.cache.plan(dev(np.array(counts, np.int32)), st)
    want, t.count = t.ref.plan(t.lens, counts, t.table, t.free, t.count, t.bs, t.blocks, tokens)
    q = (t.rng.standard_normal((tokens, t.heads, t.dim)) * 1.5).astype(np.float32)
    t.check_attention(st, want, q, **kw)
    return st, want, q


@pytest.mark.parametrize("heads,kvh,dim,bs", SHAPES + [(14, 2, 64, 128), (32, 8, 128, 16)])
@pytest.mark.parametrize("lens", [[0], [1, 126, 127, 128, 129, 255, 0, 3], [1000, 17, 2047]], ids=["first", "edges", "ragged"])
def test_single_tokens_against_float64(heads, kvh, dim, bs, lens):
    rng = np.random.default_rng(heads + dim + len(lens))
    t = filled(rng, heads, kvh, dim, bs, lens, [1] * len(lens))
    attend(t, [1] * len(lens), max_count=1)


@pytest.mark.parametrize("heads,kvh,dim,bs", [(14, 2, 64, 64), (8, 8, 32, 16), (32, 8, 128, 32), (40, 1, 64, 128), (4, 2, 128, 64)])
@pytest.mark.parametrize("lens,counts", [([0, 0], [1, 2]), ([5, 0, 130], [33, 129, 70]), ([300], [150]), ([0, 77], [257, 0])],
                         ids=["tiny", "ragged", "chunk", "one empty"])
def test_prompts_against_float64(heads, kvh, dim, bs, lens, counts):
    rng = np.random.default_rng(heads + dim + sum(counts))
    t = filled(rng, heads, kvh, dim, bs, lens, counts)
    attend(t, counts, pad=3, max_count=max(counts))


@pytest.mark.parametrize("counts", [[1, 1], [40, 90]], ids=["tokens", "prompts"])
def test_scales_far_apart_and_a_block_of_zeros(counts):
    """Block scales over many powers of two: what a small-scaled block contributes may not drown in a large one's steps
    where the large one has no weight."""
    rng = np.random.default_rng(9)
    t = filled(rng, 7, 1, 64, 16, [70, 200], counts, spread=3.0)
    zero = t.table[1, 2]
    t.scales["k"][zero] = t.scales["v"][zero] = 0.0
    t.cache.kscale.copy_(dev(t.scales["k"]).reshape(t.cache.kscale.shape))
    t.cache.vscale.copy_(dev(t.scales["v"]).reshape(t.cache.vscale.shape))
    attend(t, counts)


@pytest.mark.parametrize("counts", [[1, 1, 1], [3, 140, 20]], ids=["tokens", "prompts"])
def test_missing_and_bad_blocks_are_skipped(counts):
    rng = np.random.default_rng(10)
    lens = [100, 60, 31]
    t = filled(rng, 4, 2, 64, 32, lens, counts)
    t.table[0, 1], t.table[1, 0], t.table[2, :] = -1, t.blocks + 5, -1
    t.count = 0  # nothing is free: the missing blocks stay missing
    t.cache.table.copy_(dev(t.table).reshape(t.cache.table.shape))
    t.cache.free_count.copy_(dev(np.array([0], np.int32)))
    attend(t, counts)


def test_a_key_of_a_masked_position_does_not_poison_a_row():
    """A later block with a scale that is no number: rows before it are untouched, rows that see it are NaN."""
    rng = np.random.default_rng(11)
    t = filled(rng, 2, 1, 32, 16, [0], [40])
    bad = t.table[0, 2]
    t.scales["v"][bad] = np.nan
    t.cache.vscale.copy_(dev(t.scales["v"]).reshape(t.cache.vscale.shape))
    st = t.Step(t.cache, 40)
    t.cache.plan(dev(np.array([40], np.int32)), st)
    q = rng.standard_normal((40, 2 * 32)).astype(np.float32)
    q[5, 3] = np.inf
    out = t.cache.attend(0, dev(q), 2, st).numpy().reshape(40, 2, 32)
    finite = np.isfinite(out).all(-1)
    want = np.ones((40, 2), bool)
    want[32:] = False
    want[5, 0] = False
    np.testing.assert_array_equal(finite, want)


def test_peaked_and_flat_scores():
    """Scores hundreds apart (one key takes everything, early or late) and all equal."""
    rng = np.random.default_rng(12)
    for scale in (40.0, 0.0, 1e-8):
        t = filled(rng, 14, 2, 64, 64, [500, 3], [1, 30], spread=0.1)
        attend(t, [1, 30], scale=scale)


@pytest.mark.parametrize("value", [1e-25, 1e-6, 1e6, 1e20])
def test_value_scales_of_any_size(value):
    rng = np.random.default_rng(16)
    t = filled(rng, 4, 2, 64, 32, [200, 40], [1, 33], spread=0.3)
    t.scales["v"] *= np.float32(value)
    t.cache.vscale.copy_(dev(t.scales["v"]).reshape(t.cache.vscale.shape))
    attend(t, [1, 33])


def test_scales_that_are_none_make_their_rows_nan():
    rng = np.random.default_rng(17)
    for name, bad in [("k", -1.0), ("k", np.inf), ("v", -1.0), ("v", np.inf), ("v", 2.0 ** 91), ("k", np.nan)]:
        t = filled(rng, 2, 1, 32, 32, [70, 70], [1, 1])
        scales, on_device = t.scales[name], t.cache.kscale if name == "k" else t.cache.vscale
        scales[t.table[1, 0]] = bad
        on_device.copy_(dev(scales).reshape(on_device.shape))
        st = t.Step(t.cache, 2)
        t.cache.plan(dev(np.ones(2, np.int32)), st)
        out = t.cache.attend(0, dev(rng.standard_normal((2, 64)).astype(np.float32)), 2, st, max_count=1).numpy()
        assert np.isfinite(out[0]).all() and np.isnan(out[1]).all(), (name, bad)


def test_two_requests_may_read_the_same_blocks():
    rng = np.random.default_rng(13)
    t = filled(rng, 8, 2, 64, 32, [64, 70, 64], [1, 1, 1])
    t.table[1, :2] = t.table[0, :2]
    t.cache.table.copy_(dev(t.table).reshape(t.cache.table.shape))
    attend(t, [1, 1, 1], max_count=1)


def test_a_captured_step_follows_the_device_state():
    """plan, append, attend and advance in one graph: replays equal eager steps on a second cache."""
    _C, PagedKvCache, PagedStep, ref = _env()
    rng = np.random.default_rng(14)
    heads, kvh, dim, bs, seqs = 4, 2, 64, 16, 5
    make = lambda: PagedKvCache(layers=1, kv_heads=kvh, head_dim=dim, blocks=30, seqs=seqs, max_blocks=5, block_size=bs)  # noqa: E731
    a, b = make(), make()
    sa, sb = PagedStep(a, seqs), PagedStep(b, seqs)
    cos, sin = (dev(x) for x in rotary(80, dim, rng))
    counts, qkv = dev(np.zeros(seqs, np.int32)), dev(np.zeros((seqs, (heads + 2 * kvh) * dim), np.float32))
    out = [_C.Tensor.empty((seqs, heads * dim), "float32") for _ in range(2)]
    q = [_C.Tensor.empty((seqs, heads * dim), "float32") for _ in range(2)]

    def one(cache, step, i):
        cache.plan(counts, step)
        cache.append(0, qkv, heads, cos, sin, step, q_out=q[i])
        cache.attend(0, q[i], heads, step, max_count=1, out=out[i])
        cache.advance(step)

    one(a, sa, 0)  # nobody has a token: an eager run before the capture
    one(b, sb, 1)
    _C.begin_capture()
    one(a, sa, 0)
    graph = _C.end_capture()
    for i in range(40):
        c = (rng.random(seqs) < 0.8).astype(np.int32)
        counts.copy_(dev(c))
        qkv.copy_(dev(rng.standard_normal(qkv.shape).astype(np.float32)))
        graph.replay()
        one(b, sb, 1)
        n = int(c.sum())
        np.testing.assert_array_equal(out[0].numpy()[:n], out[1].numpy()[:n])
        np.testing.assert_array_equal(a.lengths(), b.lengths())
    np.testing.assert_array_equal(a.k.numpy(), b.k.numpy())


def test_two_graphs_and_eager_calls_share_the_scratch():
    """Captured steps of both kinds, replayed in turn with an eager step between, give what each gives alone."""
    from grilly2_b200 import _C
    rng = np.random.default_rng(31)
    kinds = []
    for lens, counts in (([900, 40, 2000], [1, 1, 1]), ([300, 0, 777], [60, 200, 31])):
        t = filled(rng, 14, 2, 64, 64, lens, counts)
        tokens = sum(counts)
        st = t.Step(t.cache, tokens)
        t.cache.plan(dev(np.array(counts, np.int32)), st)
        q, out = dev((rng.standard_normal((tokens, 14 * 64))).astype(np.float32)), _C_filled((tokens, 14 * 64), 0.0)
        kinds.append((lambda t=t, q=q, st=st, out=out, m=max(counts): t.cache.attend(0, q, 14, st, max_count=m, out=out), out))
    alone = []
    for call, out in kinds:
        call()
        alone.append(out.numpy())
    graphs = []
    for call, _ in kinds:
        _C.begin_capture()
        call()
        graphs.append(_C.end_capture())
    for turn in ((0, 1), (1, 0), (1, 1), (0, 0)):
        for _, out in kinds:
            out.copy_(_C_filled(out.shape, 9.0))
        graphs[turn[0]].replay()
        kinds[turn[1]][0]()
        graphs[1 - turn[0]].replay()
        for (_, out), want in zip(kinds, alone):
            np.testing.assert_array_equal(out.numpy(), want)


def test_the_same_call_twice_gives_the_same_bits():
    rng = np.random.default_rng(15)
    t = filled(rng, 14, 2, 64, 64, [3000, 10, 777], [1, 1, 1])
    st = t.Step(t.cache, 3)
    t.cache.plan(dev(np.ones(3, np.int32)), st)
    q = dev(rng.standard_normal((3, 14 * 64)).astype(np.float32))
    first = t.cache.attend(0, q, 14, st, max_count=1).numpy()
    for _ in range(5):
        np.testing.assert_array_equal(t.cache.attend(0, q, 14, st, max_count=1).numpy(), first)


# ── refusals ───────────────────────────────────────────────────────────────


def test_refusals():
    import ctypes
    import re
    from grilly2_b200 import _lib
    _C, PagedKvCache, PagedStep, _ = _env()
    cache = PagedKvCache(layers=2, kv_heads=2, head_dim=32, blocks=4, seqs=2, max_blocks=2, block_size=16)
    step = PagedStep(cache, 4)
    f = lambda *s: _C.Tensor.empty(s, "float32")  # noqa: E731
    q = f(4, 4 * 32)
    with pytest.raises(RuntimeError, match="do not group"):
        cache.attend(0, f(4, 3 * 32), 3, step)
    with pytest.raises(RuntimeError, match="layer 2 of 2"):
        cache.attend(2, q, 4, step)
    with pytest.raises(RuntimeError, match="must not overlap q"):
        cache.attend(0, q, 4, step, out=q)
    with pytest.raises(RuntimeError, match="max_count"):
        cache.attend(0, q, 4, step, max_count=0)
    with pytest.raises(RuntimeError, match="must hold 512 values"):
        cache.attend(0, f(3, 4 * 32), 4, step)
    with pytest.raises(NotImplementedError, match="int32"):
        cache.attend(0, _C.Tensor.empty((4, 128), "int32"), 4, step)
    with pytest.raises(RuntimeError, match="counts must hold 2"):
        cache.plan(_C.Tensor.empty((3,), "int32"), step)
    qkv = f(4, 8 * 32)
    with pytest.raises(RuntimeError, match="cos and sin"):
        cache.append(0, qkv, 4, f(8, 32), f(9, 32), step)
    with pytest.raises(RuntimeError, match="positions"):
        cache.append(0, qkv, 4, f(0, 32), f(0, 32), step)
    with pytest.raises(RuntimeError, match="must not overlap qkv"):
        cache.append(0, qkv, 4, f(8, 32), f(8, 32), step, q_out=_C.Tensor(qkv.storage, (4, 128), "float32"))
    room, y = f(4 * 128 + 4), f(4, 128)
    odd = _C.Tensor.from_pointer(_pointer(room) + 4, (4, 128), "float32")
    with pytest.raises(RuntimeError, match="16-byte"):
        cache.attend(0, odd, 4, step)
    lib, ctx = _lib.load(), _C.context()
    for change, match in [({"block_size": 24}, "block_size"), ({"seqs": 5000}, "requests"), ({"dim": 48}, "head_dim"), ({"blocks": 1 << 27}, "2\\^31"),
                          ({"blocks": 9}, "pool"), ({"kv_heads": 0}, "KV heads"), ({"max_blocks": 3}, "table")]:
        d = _lib.PagedCache(**{n: getattr(cache._desc, n) for n, _ in _lib.PagedCache._fields_})
        for n, v in change.items():
            setattr(d, n, v)
        status = lib.gq_paged_attn(ctx, ctypes.byref(d), 0, q.storage.handle, 4, 1.0, step._ref, 1, y.storage.handle)
        assert status == _lib.GQ_ERR and re.search(match, _lib.last_error()), (change, _lib.last_error())
    assert lib.gq_paged_attn(ctx, None, 0, q.storage.handle, 4, 1.0, step._ref, 1, q.storage.handle) == _lib.GQ_ERR
    assert lib.gq_paged_plan(ctx, cache._ref, q.storage.handle, q.storage.handle, q.storage.handle, None) == _lib.GQ_ERR


def _pointer(t):
    import ctypes
    from grilly2_b200 import _C, _lib
    out = ctypes.c_void_p()
    _lib.check(_lib.load().gq_buffer_ptr(_C.context(), t.storage.handle, ctypes.byref(out)))
    return out.value
