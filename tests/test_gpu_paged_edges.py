"""The paged int8 cache where it could go wrong beside the cases of test_gpu_paged.py, whose twin of device and oracle this uses:
pools that run out and are filled again, contributions far apart, batches of many requests, sums near the ends of their range."""
import numpy as np
import pytest

from test_gpu_paged import Twin, _C_filled, attend, dev, filled, words

pytestmark = pytest.mark.gpu


def test_a_request_never_reads_what_another_left_in_its_block():
    """A pool that is full drops tokens of a request; the block it gets later, in the middle of that block's positions, held
    another request's keys. Outputs and maps are those of a pool in which the other request never was."""
    outs = []
    for other in (9.0, 0.0):
        t = Twin(np.random.default_rng(41), seqs=2, heads=2, kvh=1, dim=32, bs=16, mb=3, blocks=2, layers=1, layer=0)
        st, want, _ = t.step([16, 16], qkv=_rows(1, 32, 4, 32, [1.0] * 16 + [other] * 16))
        t.advance(st, want)
        st, want, turned = t.step([1, 0], qkv=_rows(2, 1, 4, 32, [1.0]))  # position 16: no block is free
        assert want["info"][1] == 1 and step_info(st) == 1 and want["slots"][0] == -1
        t.advance(st, want)
        t.cache.release(dev(np.array([0, 1], np.int32)))
        t.free, t.count = t.cache.free.numpy(), t.cache.free_blocks()
        t.lens[1], t.table[1] = 0, -1
        got = []
        for i in range(16):  # positions 17 .. 32; from 32 on there is a block again
            st, want, turned = t.step([1, 0], qkv=_rows(3 + i, 1, 4, 32, [1.0]))
            np.testing.assert_array_equal(st.slots.numpy(), want["slots"])
            np.testing.assert_array_equal(st.info.numpy(), want["info"])
            np.testing.assert_array_equal(t.cache.table.numpy(), t.table)
            assert (want["slots"][0] < 0) == (i < 15) and want["info"][1] == (i < 15)
            t.check_pool()
            t.check_attention(st, want, turned, max_count=1)
            got.append(t.cache.attend(0, dev(turned.reshape(1, -1)), 2, st, max_count=1).numpy())
            t.advance(st, want)
        outs.append(got)
    np.testing.assert_array_equal(outs[0], outs[1])


def _rows(seed, n, heads, dim, sizes):
    x = np.random.default_rng(seed).standard_normal((n, heads, dim)) * np.array(sizes)[:, None, None]
    return x.astype(np.float32)


def step_info(st):
    return int(st.info.numpy()[1])


def test_every_row_without_room_is_counted():
    """A step says how many of its rows found no place: beyond the table, where no block is wanted, as well as without a block."""
    from grilly2_b200.infer.paged import PagedKvCache, PagedStep
    cache = PagedKvCache(layers=1, kv_heads=1, head_dim=32, blocks=3, seqs=2, max_blocks=2, block_size=16)
    step = PagedStep(cache, 50)
    for counts, dropped, shortfall in (([16, 16], 0, 0), ([16, 16], 16, 1), ([1, 1], 2, 0), ([0, 0], 0, 0)):
        cache.plan(dev(np.array(counts, np.int32)), step)
        assert (step.dropped(), step.shortfall()) == (dropped, shortfall)
        cache.advance(step)


def test_a_new_cache_is_made_on_the_device(monkeypatch):
    """Nothing of the size of the pool or the tables passes through the host's memory; the pool is zeros, the table empty."""
    from grilly2_b200 import _C
    from grilly2_b200.infer.paged import PagedKvCache, PagedStep
    sent, upload = [], _C.Tensor.from_numpy
    monkeypatch.setattr(_C.Tensor, "from_numpy", staticmethod(lambda a, persistent=False: (sent.append(np.asarray(a).size), upload(a, persistent))[1]))
    rubbish = [_C.Tensor.from_numpy(np.full(n, 77, np.int32)) for n in (1 << 18, 1 << 12, 1 << 12)]
    del rubbish, sent[:]
    cache = PagedKvCache(layers=4, kv_heads=2, head_dim=64, blocks=128, seqs=8, max_blocks=200, block_size=16)
    step = PagedStep(cache, 500)
    assert max(sent) <= 128
    for t in (cache.k, cache.v, cache.kscale, cache.vscale, cache.lens, step.slots, step.runs):
        assert not t.numpy().any()
    assert (cache.table.numpy() == -1).all() and cache.table.shape == (8, 200) and cache.free_blocks() == 128
    np.testing.assert_array_equal(np.sort(cache.free.numpy()), np.arange(128))


# ── contributions far apart ────────────────────────────────────────────────


def put(t):
    """The twin's codes and scales on the device."""
    for name, a in (("k", words(t.ref.pack_k(t.codes["k"]))), ("v", words(t.ref.pack_v(t.codes["v"]))), ("kscale", dev(t.scales["k"])), ("vscale", dev(t.scales["v"]))):
        on = getattr(t.cache, name)
        on.copy_(a.reshape(on.shape))


def with_sink(keys, gap, at, value, dim=64, bs=64):
    """One request of `keys` cached tokens, one of which scores `gap` nats above the others' mean (0.3 nats apart), with
    values of one sign so that nothing cancels, the lone key's of size `value` of theirs."""
    rng = np.random.default_rng(keys + int(gap))
    t = filled(rng, 2, 1, dim, bs, [keys - 1], [1], spread=0.0)
    t.codes["k"] = rng.integers(-30, 31, t.codes["k"].shape).astype(np.int8)
    t.codes["v"] = rng.integers(40, 127, t.codes["v"].shape).astype(np.int8)
    block, off = t.table[0, at // bs], at % bs
    t.codes["k"][block, :, off] = 127
    t.codes["v"][block, :, off] = (t.codes["v"][block, :, off] * value).astype(np.int8)
    put(t)
    st = t.Step(t.cache, 1)
    t.cache.plan(dev(np.ones(1, np.int32)), st)
    want, _ = t.ref.plan(t.lens, [1], t.table, t.free, t.count, bs, t.blocks, 1)
    q = np.ones((1, 2, dim), np.float32)
    scale = gap / (dim * 127 * float(t.scales["k"][block, 0]))
    return t, st, want, q, scale


@pytest.mark.parametrize("value", [0.0, 1.0], ids=["null", "full"])
@pytest.mark.parametrize("gap", [10.0, 14.0, 17.0, 40.0])
@pytest.mark.parametrize("keys,at", [(200, 5), (4096, 0), (4096, 3000), (15000, 0), (15000, 14990)])
def test_one_key_far_above_the_others(keys, at, gap, value):
    """The allowance is the oracle's: what a weight's whole steps lose is bounded tile by tile, so the row's other keys
    keep their digits outside the lone key's own tile, and inside it down to 2^-31 of it."""
    t, st, want, q, scale = with_sink(keys, gap, at, value)
    exact, tol = t.ref.attend(q, t.codes["k"], t.codes["v"], t.scales["k"], t.scales["v"], t.table, t.lens, want, scale)
    got = t.cache.attend(0, dev(q.reshape(1, -1)), 2, st, scale=scale, max_count=1).numpy().reshape(1, 2, -1)
    off = np.abs(got - exact).max(-1)
    size = np.abs(exact).max(-1)
    print(f"[sink] {keys} keys, {gap} nats, value {value}: {float((off / size).max()):.2e} of the row, {float((off / tol).max()):.2f} of the allowance "
          f"({float((tol / size).max()):.1e})")
    assert (off <= tol).all()


@pytest.mark.parametrize("every", [1, 3])
def test_references_that_move_up_and_down(every):
    """Tiles whose largest scores lie some 15 nats apart in turn, rows of a prompt with different scores: the reference follows the
    tiles down and up again, nothing is lost on the way."""
    rng = np.random.default_rng(52)
    for heads, counts in ((2, [1, 1]), (14, [70, 5])):
        t = filled(rng, heads, 1, 64, 32, [3000, 900], counts, spread=0.2)
        t.codes["v"] = rng.integers(1, 127, t.codes["v"].shape).astype(np.int8)
        for b in range(2):
            for j, block in enumerate(t.table[b]):
                if block >= 0 and (j // 4) % (2 * every) >= every:
                    t.codes["k"][block] = t.codes["k"][block] // 8
        put(t)
        attend(t, counts, scale=0.55, max_count=max(counts))


@pytest.mark.parametrize("counts", [[1], [33]], ids=["token", "prompt"])
def test_value_scales_at_the_lower_end(counts):
    """Thousands of keys of about equal weight, value scales of 2^-100: the sums' quotients stay normal numbers."""
    rng = np.random.default_rng(53)
    t = filled(rng, 2, 1, 64, 64, [5000], counts, spread=0.0)
    t.codes["v"] = np.abs(t.codes["v"])
    t.scales["v"][:] = np.float32(2.0 ** -100)
    put(t)
    attend(t, counts, scale=1e-3)


# ── many requests, long ranges ─────────────────────────────────────────────


@pytest.mark.parametrize("kind", ["tokens", "prompts", "holes"])
@pytest.mark.parametrize("seqs", [33, 65, 1025, 4096])
def test_batches_of_many_requests(seqs, kind):
    """More requests than the lanes that look for a range's start: stretches of several requests a lane, whole stretches
    without a token, more requests in a stretch than lanes."""
    rng = np.random.default_rng(seqs)
    lens = rng.integers(0, 40, seqs)
    if kind == "tokens":
        counts = np.ones(seqs, np.int64)
    elif kind == "prompts":
        counts = rng.integers(0, 6, seqs)
    else:
        counts = (rng.random(seqs) < 0.05).astype(np.int64) * rng.integers(1, 4, seqs)
        counts[: seqs // 3] = 0
        counts[seqs - 1] = 2
        lens[seqs // 2] = 900
        counts[seqs // 2] = 1
    t = filled(rng, 2, 1, 32, 16, [int(n) for n in lens], [int(c) for c in counts])
    attend(t, [int(c) for c in counts], pad=1, max_count=int(counts.max()))


@pytest.mark.parametrize("dim", [32, 64, 128])
def test_attention_right_behind_an_int4_linear(dim):
    """Both hold tensor memory, and the linear lets the next launch start before it has its own: eager and captured runs of
    the two one behind the other end and give what each gives alone."""
    from grilly2_b200 import _C, _lib
    rng = np.random.default_rng(61)
    w = _C.Int4Weight.quantize(_C.Tensor.from_numpy((rng.standard_normal((148 * 128, 512)) * 0.02).astype(np.float32)), 128)
    x = _C.Tensor.from_numpy(rng.standard_normal((8, 512)).astype(np.float32))
    t = filled(rng, 8, 2, dim, 32, [500, 40, 1000], [1, 1, 1])
    st = t.Step(t.cache, 3)
    t.cache.plan(dev(np.ones(3, np.int32)), st)
    q, out = dev(rng.standard_normal((3, 8 * dim)).astype(np.float32)), _C_filled((3, 8 * dim), 0.0)
    for kernel in (_lib.KERNEL_UMMA_LANES, _lib.KERNEL_UMMA):
        y_alone = w.linear(x, None, kernel).numpy()
        alone = t.cache.attend(0, q, 8, st, max_count=1, out=out).numpy()
        for _ in range(20):
            y = w.linear(x, None, kernel)
            t.cache.attend(0, q, 8, st, max_count=1, out=out)
            again = w.linear(x, None, kernel)
        for got in (y, again):
            np.testing.assert_array_equal(got.numpy(), y_alone)
        np.testing.assert_array_equal(out.numpy(), alone)
        _C.begin_capture()
        for _ in range(4):
            y = w.linear(x, None, kernel)
            t.cache.attend(0, q, 8, st, max_count=1, out=out)
        graph = _C.end_capture()
        for _ in range(10):
            graph.replay()
        np.testing.assert_array_equal(out.numpy(), alone)
        np.testing.assert_array_equal(y.numpy(), y_alone)
        del graph


@pytest.mark.parametrize("dim,block", [(32, 128), (64, 128)])
def test_a_range_of_more_tiles_than_the_integer_sums_may_hold(dim, block):
    """Tables that name a few blocks over and over: every CTA has some 700 tiles of one request, all of equal scores, codes of
    127. Value scales of 0.99 and of just under 64 times that: a reference that a tile of small ones laid is not moved by the large ones,
    whose weights then fill their 32 bits, and the sums are read out only because they would leave 32 bits. The mean of the
    values is known exactly."""
    from grilly2_b200.infer.paged import PagedKvCache, PagedStep
    rng = np.random.default_rng(54)
    seqs, entries, blocks = 4, 100000, 16
    table = rng.integers(0, blocks, (seqs, entries)).astype(np.int32)
    last = entries * block - 1  # the last position of the table
    codes = np.full((blocks, 1, block, dim), 127, np.int8)
    vscale = np.where(np.arange(blocks) % 8, 62.5, 0.99).astype(np.float32)[:, None]
    cache = PagedKvCache(layers=1, kv_heads=1, head_dim=dim, blocks=blocks, seqs=seqs, max_blocks=entries, block_size=block,
                         buffers={"k": words(codes), "v": words(codes), "kscale": dev(np.ones((blocks, 1), np.float32)), "vscale": dev(vscale),
                                  "table": dev(table), "lens": dev(np.full(seqs, last, np.int32)), "free_count": dev(np.zeros(1, np.int32))})
    st = PagedStep(cache, seqs)
    cache.plan(dev(np.ones(seqs, np.int32)), st)
    got = cache.attend(0, _C_filled((seqs, dim), 0.0), 1, st, max_count=1).numpy()
    want = 127 * vscale[table, 0].astype(np.float64).mean(1)
    tiles = seqs * entries * block // 128
    # the sums of a CTA's range, one rounding a tile each for numerator and denominator at most, and their joining
    allowed = (2 * (tiles / 148 + 1) + 16) * 2.0 ** -24
    off = np.abs(got - want[:, None]).max(1) / want
    print(f"[long range] {tiles} tiles: {off.max():.2e} ({allowed:.1e})")
    assert (off <= allowed).all()


# ── refusals ───────────────────────────────────────────────────────────────


def test_buffers_that_a_call_writes_lie_apart():
    from grilly2_b200 import _C
    from grilly2_b200.infer.paged import PagedKvCache, PagedStep
    ints = lambda n: dev(np.zeros(n, np.int32))  # noqa: E731
    geometry = dict(layers=1, kv_heads=2, head_dim=32, blocks=4, seqs=2, max_blocks=2, block_size=16)
    cache, counts = PagedKvCache(**geometry), ints(2)
    step = PagedStep(cache, 4)
    over = lambda t, *shape: _C.Tensor(t.storage, shape, t.dtype)  # noqa: E731
    shared = ints(16)
    for names in (("slots", "positions"), ("starts", "last"), ("runs", "info")):
        with pytest.raises(RuntimeError, match="must not overlap"):
            cache.plan(counts, PagedStep(cache, 4, buffers={n: shared for n in names}))
    with pytest.raises(RuntimeError, match="the step's last rows must not overlap the counts"):
        cache.plan(step.last, step)
    with pytest.raises(RuntimeError, match="the block table must not overlap the cached lengths"):
        PagedKvCache(**geometry, buffers={"table": shared, "lens": shared}).plan(counts, step)
    with pytest.raises(RuntimeError, match="the free count must not overlap the free list"):
        PagedKvCache(**geometry, buffers={"free": shared, "free_count": shared}).plan(counts, step)
    with pytest.raises(RuntimeError, match="the cached lengths must not overlap the step's starts"):
        PagedKvCache(**geometry, buffers={"lens": step.starts}).advance(step)
    with pytest.raises(RuntimeError, match="the cached lengths must not overlap the requests"):
        cache.release(cache.lens)
    with pytest.raises(RuntimeError, match="the block table must not overlap the free list"):
        PagedKvCache(**geometry, buffers={"table": shared, "free": shared}).release(counts)
    f = lambda *s: dev(np.zeros(s, np.float32))  # noqa: E731
    qkv, cos, sin, room = f(4, 8 * 32), f(64, 32), f(64, 32), f(4096)
    with pytest.raises(RuntimeError, match="the output must not overlap cos"):
        cache.append(0, qkv, 4, cos, sin, step, q_out=over(cos, 4, 128))
    with pytest.raises(RuntimeError, match="the output must not overlap the key pool"):
        cache.append(0, qkv, 4, cos, sin, step, q_out=_C.Tensor(cache.k.storage, (4, 128), "float32"))
    one = PagedKvCache(**geometry, buffers={"k": cache.k, "v": cache.k})
    with pytest.raises(RuntimeError, match="the key pool must not overlap the value pool"):
        one.append(0, qkv, 4, cos, sin, step)
    with pytest.raises(RuntimeError, match="the key scales must not overlap the value scales"):
        PagedKvCache(**geometry, buffers={"kscale": room, "vscale": room}).append(0, qkv, 4, cos, sin, step)
    q = f(4, 128)
    with pytest.raises(RuntimeError, match="the output must not overlap the value scales"):
        PagedKvCache(**geometry, buffers={"vscale": room}).attend(0, q, 4, step, out=over(room, 4, 128))
    with pytest.raises(RuntimeError, match="the output must not overlap the key pool"):
        cache.attend(0, q, 4, step, out=_C.Tensor(cache.k.storage, (4, 128), "float32"))
    one.attend(0, q, 4, step)  # what is only read may be named twice
    cache.plan(counts, step)


def test_more_tiles_than_their_numbers_hold_are_refused():
    from grilly2_b200.infer.paged import PagedKvCache, PagedStep
    for entries, refused in ((1 << 20, True), ((1 << 20) - 4, False)):
        cache = PagedKvCache(layers=1, kv_heads=4096, head_dim=32, blocks=1, seqs=1, max_blocks=entries, block_size=128)
        step = PagedStep(cache, 1)
        cache.plan(dev(np.ones(1, np.int32)), step)
        q = dev(np.zeros((1, 4096 * 32), np.float32))
        if refused:
            with pytest.raises(RuntimeError, match="2\\^32 tiles"):
                cache.attend(0, q, 4096, step)
        else:
            cache.attend(0, q, 4096, step)
