"""The paged cache's host side and its checker, without a device: layouts, refusals that come before any allocation, the run
count the header and the Python call share, and the checker against its own definitions."""
import os
import re

import numpy as np
import pytest

from oracle import paged_ref as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_layouts_round_trip_and_place_bytes_as_documented():
    codes = np.random.default_rng(0).integers(-127, 128, (2, 3, 32, 64)).astype(np.int8)
    k, v = ref.pack_k(codes), ref.pack_v(codes)
    assert k.shape == (2, 3, 4, 4, 8, 16) and v.shape == (2, 3, 8, 2, 8, 16)
    np.testing.assert_array_equal(ref.unpack_k(k, 32, 64), codes)
    np.testing.assert_array_equal(ref.unpack_v(v, 32, 64), codes)
    for t, d in [(0, 0), (13, 37), (31, 63), (8, 16)]:
        assert k[1, 2, t // 8, d // 16, t % 8, d % 16] == codes[1, 2, t, d] == v[1, 2, d // 8, t // 16, d % 8, t % 16]


def test_refusals_before_anything_is_allocated():
    from grilly2_b200.infer.paged import PagedKvCache
    ok = dict(layers=1, kv_heads=1, head_dim=64, blocks=4, seqs=1, max_blocks=2)
    for change, match in [({"block_size": 48}, "block_size"), ({"head_dim": 96}, "head_dim"), ({"blocks": 0}, "at least one"), ({"seqs": 0}, "at least one")]:
        with pytest.raises(RuntimeError, match=match):
            PagedKvCache(**{**ok, **change})
    with pytest.raises(TypeError, match="must be a tensor"):
        PagedKvCache(**ok, buffers={"k": np.zeros(4)})


def test_run_count_matches_the_header():
    text = open(os.path.join(ROOT, "include", "gq.h")).read()
    body = re.search(r"#define GQ_PAGED_RUNS\(max_tokens, block_size, seqs\)(.*?)\n(?:/\*|int32)", text, re.S).group(1).replace("\\\n", " ")
    expr = re.sub(r"\(uint64_t\)", "", body).replace("/", "//")
    cond, yes, no = re.match(r"\s*\((.*)\?(.*):(.*)\)\s*$", expr, re.S).groups()
    for tokens, bs, seqs in [(1, 16, 1), (5, 64, 5), (100, 16, 3), (9000, 128, 4096), (40, 16, 2)]:
        env = {"max_tokens": tokens, "block_size": bs, "seqs": seqs}
        one = lambda e: eval(e.strip(), {}, env)  # noqa: E731
        assert (one(yes) if one(cond) else one(no)) == ref.runs_cap(tokens, bs, seqs)


def test_runs_never_exceed_their_room():
    rng = np.random.default_rng(1)
    for _ in range(200):
        seqs, bs = int(rng.integers(1, 9)), int(rng.choice([16, 32]))
        lens, counts = rng.integers(0, 70, seqs), rng.integers(0, 50, seqs)
        tokens = max(int(counts.sum()) - int(rng.integers(0, 5)), 1)
        out, left = ref.plan(lens, counts, np.full((seqs, 9), -1, np.int32), np.arange(40), 40, bs, 40, tokens)
        assert len(out["runs"]) == ref.runs_cap(tokens, bs, seqs) + 1 and out["runs"][-1] == out["starts"][-1]


def test_the_checkers_append_is_one_rounding_per_growth():
    """A block filled token by token: every cached value is within half a step of each scale it was rounded at."""
    rng = np.random.default_rng(2)
    codes, scales = np.zeros((1, 1, 16, 32), np.int8), np.zeros((1, 1), np.float32)
    x = (rng.standard_normal((16, 1, 32)) * np.linspace(0.2, 3.0, 16)[:, None, None]).astype(np.float32)
    allowed = np.zeros(16)
    for t in range(16):
        before = scales[0, 0]
        ref.append(codes, scales, x[t:t + 1], {"slots": np.array([t]), "runs": np.array([0, 1]), "starts": np.array([0, 1])}, 16)
        if scales[0, 0] != before:
            allowed[:t + 1] += scales[0, 0] / 2
        else:
            allowed[t] += scales[0, 0] / 2
        got = codes[0, 0, :t + 1].astype(np.float64) * scales[0, 0]
        assert (np.abs(got - x[:t + 1, 0]) <= allowed[:t + 1, None] * (1 + 1e-5)).all()


def test_the_checkers_sampling_against_a_direct_count():
    """Top-k, top-p and min-p on a row small enough to enumerate."""
    x = np.log(np.array([0.4, 0.3, 0.15, 0.1, 0.05]))
    pick = lambda u, **kw: ref.sample(x.astype(np.float32), 1.0, kw.get("k", 0), kw.get("p", 1.0), kw.get("m", 0.0), u)[0]  # noqa: E731
    assert [pick(u) for u in (0.0, 0.39, 0.41, 0.69, 0.71, 0.86, 0.96)] == [0, 0, 1, 1, 2, 3, 4]
    assert [pick(u, k=2) for u in (0.56, 0.58, 0.99)] == [0, 1, 1]
    assert [pick(u, p=0.75) for u in (0.46, 0.48, 0.81, 0.83)] == [0, 1, 1, 2]  # 0.4 + 0.3 < 0.75: the third is still kept
    assert [pick(u, m=0.3) for u in (0.0, 0.99)] == [0, 2]                       # 0.15 / 0.4 passes, 0.1 / 0.4 does not
