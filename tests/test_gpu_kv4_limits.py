"""The 4-bit key/value cache on the GPU where its precision, ranges and sizes end, against plain 64-bit forms."""
import pytest
import torch

from test_gpu_kv4 import BF16, FP16, HALF_STEP, attend64, both_ways, make_cache, queries, score_error

pytestmark = pytest.mark.gpu


def close_to_the_rounding(got, want, spread, size, D, n):
    """As close as P in two terms is, whatever the queries' type: P times the value's scale is off by 2^-16 (two bf16
    terms, half a step of 2^-8 each), by twice the score error and by 2^-22 per step of 16 in sums over n keys, the
    output by its own rounding."""
    p_off = 2 * score_error(size, D) + 2.0 ** -16 + (n / 16 + 8) * 2.0 ** -22
    tol = p_off * spread + HALF_STEP[got.dtype] * want.abs() * (1 + 2.0 ** -6) + (2.0 ** -25 if got.dtype is FP16 else 0)
    worst = ((got.double() - want).abs() / tol.clamp(min=1e-300)).max().item()
    assert worst <= 1, f"off by {worst:.3g} times the tolerance"


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rep, N, lens", [(4, 1, [3000, 700]), (2, 1, [150, 60]), (3, 5, [2500, 2000]), (4, 40, [2000, 1777])])
def test_outputs_as_exact_as_their_type(rep, N, lens, D, dtype):
    """Values that cancel out show what a rounding of the probabilities costs: with one bf16 term each they are off by
    2^-8 of what was added up, several times the output's own rounding."""
    cache = make_cache(2, 2, max(lens) + 5, D, lens, seed=rep)
    q = queries(2, 2 * rep, N, D, dtype, seed=N)
    want, spread, _, size = attend64(cache, q, [N, N], True)
    close_to_the_rounding(cache.attend(q), want, spread, size, D, max(lens))
    if rep * N > 48:  # the kernel for many rows
        close_to_the_rounding(both_ways(cache, q)[0], want, spread, size, D, max(lens))
