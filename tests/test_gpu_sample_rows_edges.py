"""Sampling with settings of each row where the kept tokens' weights lie far apart, against the float64 oracle."""
import numpy as np
import pytest

from test_gpu_sample_rows import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("top_k", [2, 3, 40, 1000], ids=lambda k: f"k{k}")
def test_light_tokens_of_a_short_list_are_drawn(top_k):
    """Kept tokens 30 to 60 nats below the largest, with numbers that choose them: the draw's sums are 64-bit, with top-k or without."""
    rng = np.random.default_rng(6)
    vocab, u = 1500, [0.0, 1e-30, 1e-26, 3e-14, 1e-9, 0.5, 1.0 - 2.0 ** -24, 1.0]
    x = np.full((len(u), vocab), -100.0, np.float32) - rng.random((len(u), vocab)).astype(np.float32)
    x[:, 0], x[:, 1], x[:, 2] = -29.0, 0.0, -50.0
    x[:, 700], x[:, 1400] = -60.0, -30.0
    for k in (top_k, 0):
        check(x, 1.0, k, 1.0, 0.0, u[:-1] + [0.25])
    check(x, 1.0, min(top_k, 5), 1.0, 0.0, u)
    x[:, 5:905:3] = -20.0 - rng.random((len(u), 300)).astype(np.float32) * 40
    check(x, 1.0, top_k, 1.0, 0.0, u[:-1] + [0.25])


def test_many_light_tokens_before_the_heavy_one():
    """A list of hundreds of tokens of 2^-42 of the largest each: they weigh together, and each is drawn where it lies."""
    x = np.full((9, 4000), -200.0, np.float32)
    x[:, 10:410] = np.float32(-29.2)
    x[:, 2000] = 0.0
    w = np.exp(np.float64(np.float32(-29.2)))
    u = [w * (i + 0.5) for i in (0, 1, 2, 3, 200, 398, 399, 1500)] + [0.9]
    check(x, 1.0, 401, 1.0, 0.0, np.array(u, np.float32))
