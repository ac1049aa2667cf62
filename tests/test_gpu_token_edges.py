"""GPU tests of the new tokens' calls at their edges: rows of equal scores, sums next to and beyond 32 bits.  The
helpers are those of test_gpu_tokens.py; every result is a whole number and is compared exactly with the numpy oracle."""
import numpy as np
import pytest
import torch
from oracle import witness_oracle as wo
from test_gpu_tokens import dev, exp_table, filled, gauss, ops, paged, run_attention  # noqa: F401  (two of them are fixtures)

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ one launch: a row's scores and exponentials in one place
@pytest.mark.parametrize("each", [1, 2, 4])
@pytest.mark.parametrize("score", [0, 3 << 20, -(3 << 20)])
def test_equal_scores_set_no_bit(ops, exp_table, each, score):
    """Every score of a row is the same, so that none of its exponentials - 2^16 each - would pass for a score: read in a score's
    place, the exponential's index is above the table with scores of 0 or less and below it with scores of 3 * 2^20.  One, two and four query
    heads a cache head give a row's positions to eight, four and two waves."""
    rng = np.random.default_rng(each)
    HK, D, page = 2, 64, 16
    q = np.zeros((3, each * HK, D), dtype=np.int32)
    q[:, :, 5] = score
    for n in (100, 129, 200, 255, 256):
        lens = [n, n - 1, 100]
        table, kc, vc = paged(rng, lens, page, HK, D)
        kc[..., 5] = 1
        got = run_attention(ops, q, kc, vc, table, lens, None, exp_table, n, qk_scale=1)
        assert ops.wit_status() == 0
        assert bool((got["scores"][0] == score).all()) and bool((got["exp_output"][0] == 1 << 16).all())
        assert ops.wit_status() == 0
