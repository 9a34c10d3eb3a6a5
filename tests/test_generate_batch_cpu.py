"""What generate_batch() refuses before it touches a device."""
import numpy as np
import pytest


@pytest.mark.parametrize("bad", [2 ** 32 + 5, 2 ** 31, -2 ** 31 - 1])
def test_token_ids_beyond_32_bits_are_refused(bad):
    """They would be cut to other tokens' ids."""
    from grilly2_b200.infer.generation import generate_batch
    for prompt in ([3, bad], np.array([bad, 1], np.int64)):
        with pytest.raises(ValueError, match="32 bits"):
            generate_batch(None, [[1], prompt], max_new_tokens=1)
    if bad > 0:
        with pytest.raises(ValueError, match="32 bits"):
            generate_batch(None, [np.array([bad], np.uint64)], max_new_tokens=1)
