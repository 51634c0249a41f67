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


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("Z, H, C, L, rep, N", [(5, 1, 1 << 23, 1500, 4, 4), (3, 2, 1 << 22, 1500, 8, 6), (1, 3, 1 << 23, 1500, 24, 2),
                                           (5000, 2, 2000, 200, 4, 4)])
def test_weights_of_large_caches(Z, H, C, L, rep, N, dtype):
    """Caches whose scores are kept for some sequences, or some heads, at a time."""
    from qflash_b200 import KV4Cache
    D = 64
    lens = [(397 * z + 700) % L for z in range(Z)]
    lens[Z // 2] = 0
    small = make_cache(Z, H, L, D, lens, seed=N, garbage=False)
    cache = KV4Cache.empty(Z, H, C, D)
    for name in ("k_codes", "v_codes", "k_param", "v_param", "weight"):
        getattr(cache, name)[:, :, :L] = getattr(small, name)
    cache.lens.copy_(small.lens)
    new = [min(n, N - z % 2) for z, n in enumerate(lens)]
    counts = torch.tensor(new, dtype=torch.int32, device="cuda")
    q = queries(Z, H * rep, N, D, dtype, seed=Z)
    start = cache.weight.clone()
    out = cache.attend(q, new_lens=counts, accumulate=True)
    want, spread, cols, size = attend64(small, q, new, True)
    close_to_the_rounding(out, want, spread, size, D, L)
    assert torch.equal(cache.weight[:, :, L:], start[:, :, L:])
    # p by twice its score error, fp32 sums over the rows by half a step each
    first = start[:, :, :L].double()
    tol = (2 * score_error(size.max(), D) + (rep * N + 2) * 2.0 ** -24) * cols + 2.0 ** -23 * (first + cols)
    assert ((cache.weight[:, :, :L].double() - first - cols).abs() <= tol).all()
