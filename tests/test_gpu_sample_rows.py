"""Sampling with settings of each row (gq_sample_rows) against the float64 checker: tokens equal, shares to a float32
rounding (2^-24 relative; the sums are 64-bit, allowed 1e-12 more)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def run(x, t, k, p, m, u, draws=None):
    from grilly2_b200 import _C
    from grilly2_b200.infer.sampling import sample_rows
    T = lambda a, d: _C.Tensor.from_numpy(np.ascontiguousarray(a, dtype=d))  # noqa: E731
    probs = _C.Tensor.empty((len(x),), "float32")
    tok = sample_rows(T(x, np.float32), T(u, np.float32), temperature=T(t, np.float32), top_k=T(k, np.int32), top_p=T(p, np.float32),
                      min_p=T(m, np.float32), draws=draws, probs=probs)
    return tok.numpy(), probs.numpy()


def check(x, t, k, p, m, u):
    from oracle import paged_ref
    rows = len(x)
    t, p, m, u = (np.broadcast_to(np.asarray(a, np.float32), (rows,)) for a in (t, p, m, u))
    k = np.broadcast_to(np.asarray(k, np.int32), (rows,))
    tok, prob = run(x, t, k, p, m, u)
    for r in range(rows):
        want, share = paged_ref.sample(x[r], t[r], int(k[r]), p[r], m[r], u[r])
        assert tok[r] == want, (r, tok[r], want)
        assert abs(prob[r] - share) <= (2.0 ** -24 + 1e-12) * share, (r, prob[r], share)


@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (2, 31), (5, 1000), (1, 151936), (7, 32003), (40, 4097), (2, 500000)])
def test_settings_of_all_kinds(rows, vocab):
    rng = np.random.default_rng(rows + vocab)
    x = (rng.standard_normal((rows, vocab)) * 2.5).astype(np.float32)
    x[:, rng.integers(0, vocab, 3)] += 6.0
    u = rng.random(rows).astype(np.float32)
    each = lambda *v: np.array([v[i % len(v)] for i in range(rows)])  # noqa: E731
    check(x, 1.0, 0, 1.0, 0.0, u)
    check(x, each(0.7, 1.3, 0.2), each(50, 1, 7, 0, vocab, vocab - 1, -3), 1.0, 0.0, u)
    check(x, each(0.9, 1.1), 0, each(0.9, 0.5, 0.999, 1.0), 0.0, u)
    check(x, each(0.9, 1.1), 0, 1.0, each(0.01, 0.3, 1.0), u)
    check(x, each(0.8, 1.5, 0.05), each(40, 0, 300), each(0.95, 0.2, 0.99999), each(0.02, 0.0, 0.001), u)


def test_borders_of_the_draw():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((6, 5000)).astype(np.float32)
    check(x, 1.0, 0, 1.0, 0.0, [0.0, 1.0 - 2.0 ** -24, 1.0, 0.5, 2.0, 1e-30])
    check(x, 1.0, 3, 0.0, 0.0, 0.7)   # top_p 0: the largest alone
    check(x, 1.0, 0, 1.0, 2.0, 0.7)   # min_p above one: the largest alone
    check(x, 0.0, 5, 0.3, 0.5, 0.7)   # greedy
    check(x, 1e-6, 0, 0.9, 0.0, 0.7)
    check(x, 1e6, 0, 0.9, 0.0, 0.7)


def test_ties_infinities_and_values_that_are_no_numbers():
    rng = np.random.default_rng(2)
    x = rng.integers(-4, 3, (8, 3000)).astype(np.float32)  # every value many times: ties with each border stay
    u = rng.random(8).astype(np.float32)
    check(x, 1.0, 100, 1.0, 0.0, u)
    check(x, 1.0, 0, 0.6, 0.0, u)
    check(x, 0.0, 0, 1.0, 0.0, u)
    x = rng.standard_normal((7, 2500)).astype(np.float32)
    x[0, 1::2] = -np.inf
    x[1, ::3] = np.nan
    x[2, [7, 900]] = np.inf
    x[3, :] = -np.inf
    x[4, :] = np.nan
    x[5, :] = -np.inf
    x[5, 2499] = -3.0e38
    x[6, :] = np.finfo(np.float32).min
    for k, p, m in [(0, 1.0, 0.0), (2000, 1.0, 0.0), (0, 0.9, 0.0), (30, 0.9, 0.1)]:
        check(x, 0.9, k, p, m, u[:7])
    x = np.zeros((2, 70000), np.float32)
    x[1] = -0.0
    check(x, 1.0, 10, 0.5, 0.5, [0.3, 0.99])  # all equal


def test_the_draws_follow_the_distribution():
    """20000 draws of one distribution: every token's frequency within 5 standard deviations of its probability."""
    rng = np.random.default_rng(3)
    n, v = 20000, 12
    x = np.repeat(rng.standard_normal((1, v)).astype(np.float32), n, 0)
    tok, _ = run(x, np.ones(n), np.zeros(n), np.ones(n), np.zeros(n), rng.random(n).astype(np.float32))
    p = np.exp(x[0].astype(np.float64))
    p /= p.sum()
    seen = np.bincount(tok, minlength=v) / n
    assert (np.abs(seen - p) <= 5 * np.sqrt(p * (1 - p) / n)).all()


def test_a_captured_draw_takes_the_next_numbers_at_each_replay():
    from grilly2_b200 import _C
    from grilly2_b200.infer.sampling import sample_rows
    from oracle import paged_ref
    rng = np.random.default_rng(4)
    rows, vocab, n = 3, 4000, 5
    x = rng.standard_normal((rows, vocab)).astype(np.float32)
    u = rng.random((n, rows)).astype(np.float32)
    T = _C.Tensor.from_numpy
    full = lambda v, d=np.float32: T(np.full(rows, v, d))  # noqa: E731
    args = dict(temperature=full(1.0), top_k=full(0, np.int32), top_p=full(0.95), min_p=full(0.0), draws=T(np.zeros(1, np.int32)),
                tokens=_C.Tensor.empty((rows,), "int32"))
    logits, uniforms = T(x), T(u)
    want = lambda i: [paged_ref.sample(x[r], 1.0, 0, np.float32(0.95), 0.0, u[i % n, r])[0] for r in range(rows)]  # noqa: E731
    assert list(sample_rows(logits, uniforms, **args).numpy()) == want(0)
    _C.begin_capture()
    sample_rows(logits, uniforms, **args)
    graph = _C.end_capture()  # runs what was recorded once
    for i in range(1, 8):
        if i > 1:
            graph.replay()
        assert list(args["tokens"].numpy()) == want(i)
    assert int(args["draws"].numpy()[0]) == 8


def test_logits_at_an_offset_and_refusals():
    from grilly2_b200 import _C
    from grilly2_b200.infer.sampling import sample_rows
    from oracle import paged_ref
    rng = np.random.default_rng(5)
    x = rng.standard_normal((5, 777)).astype(np.float32)
    T = _C.Tensor.from_numpy
    full = lambda v, n=2, d=np.float32: T(np.full(n, v, d))  # noqa: E731
    args = dict(temperature=full(1.0), top_k=full(0, 2, np.int32), top_p=full(1.0), min_p=full(0.0))
    got = sample_rows(T(x).narrow_rows(3, 2), full(0.4), **args).numpy()
    assert [int(g) for g in got] == [paged_ref.sample(x[r], 1.0, 0, 1.0, 0.0, np.float32(0.4))[0] for r in (3, 4)]
    with pytest.raises(RuntimeError, match="one value per row"):
        sample_rows(T(x), full(0.4, 5), **args)
    with pytest.raises(RuntimeError, match="uniforms"):
        sample_rows(T(x).narrow_rows(0, 2), full(0.4, 4), **args)
    with pytest.raises(NotImplementedError, match="top_k"):
        sample_rows(T(x).narrow_rows(0, 2), full(0.4), **{**args, "top_k": full(0.0)})
    with pytest.raises(RuntimeError, match="batch, vocab"):
        sample_rows(full(1.0), full(0.4), **args)
    with pytest.raises(RuntimeError, match="vocab > 0"):
        sample_rows(_C.Tensor.empty((2, 0), "float32"), full(0.4), **args)
    with pytest.raises(RuntimeError, match="must not overlap the inputs"):
        sample_rows(T(x).narrow_rows(0, 2), full(0.4), probs=args["temperature"], **args)
    with pytest.raises(RuntimeError, match="must not overlap the inputs"):
        sample_rows(T(x).narrow_rows(0, 2), full(0.4), tokens=args["top_k"], **args)
    empty = sample_rows(_C.Tensor.empty((0, 9), "float32"), _C.Tensor.empty((0,), "float32"), **{n: _C.Tensor.empty((0,), t.dtype) for n, t in args.items()})
    assert empty.numel() == 0
