"""The 4-bit key/value cache on the GPU where its precision, ranges and sizes end, against plain 64-bit forms."""
import numpy as np
import pytest
import torch

from test_gpu_kv4 import (BF16, FP16, FP32, HALF_STEP, attend64, both_ways, gen, make_cache, pack, quantise, queries,
                          same, score_error)

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


def kept64(cache, budget, recent):
    """Positions that stay, for weights without NaN."""
    w, kept = cache.weight.cpu().numpy(), np.full((*cache.shape[:2], budget), -1, np.int32)
    for z, n in enumerate(cache.lens.tolist()):
        for h in range(cache.shape[1]):
            keep = np.arange(n)
            if n > budget:
                heavy = np.argsort(-w[z, h, :n - recent], kind="stable")[:budget - recent]
                keep = np.concatenate((np.sort(heavy), np.arange(n - recent, n)))
            kept[z, h, :len(keep)] = keep
    return torch.from_numpy(kept).cuda()


def check_evict(cache, budget, recent):
    from qflash_b200 import KV4Cache
    Z, H, _, D = cache.shape
    to = KV4Cache.empty(Z, H, budget, D)
    kept, want = cache.evict(budget, recent, out=to), kept64(cache, budget, recent)
    assert torch.equal(kept, want) and torch.equal(to.lens, cache.lens.clamp(max=budget))
    there, at = want >= 0, want.clamp(min=0).long()
    for name in ("k_codes", "v_codes", "k_param", "v_param"):
        src = getattr(cache, name)
        rows = torch.gather(src, 2, at[..., None].expand(*at.shape, src.shape[-1]))
        assert torch.equal(getattr(to, name)[there], rows[there])
    assert torch.equal(to.weight[there], torch.gather(cache.weight, 2, at)[there])


@pytest.mark.parametrize("Z, H, lens, budget, recent", [
    (10, 8, None, 5001, 77),  # a CTA per head, two or three tiles of positions each
    (1, 2, [300001], 7000, 1000),  # eight CTAs per head, three tiles each; two in the next
    (1, 1, [140000], 69999, 0), (2, 1, [262144, 131073], 4096, 4095)])
@pytest.mark.parametrize("kind", ["random", "equal", "few", "sparse"])
def test_evict_over_several_tiles(Z, H, lens, budget, recent, kind):
    """Counts of heavier and equal positions are carried from tile to tile and from CTA to CTA."""
    lens = lens or [40000 - 1234 * z for z in range(Z)]
    cache = make_cache(Z, H, max(lens), 64, lens, seed=budget, garbage=False)
    g = gen(budget)
    if kind == "equal":
        cache.weight.fill_(0.5)
    elif kind == "few":
        cache.weight.copy_(torch.randint(0, 3, cache.weight.shape, generator=g, device="cuda"))
    elif kind == "sparse":  # some hundred heavy positions, and ties among the others
        cache.weight.mul_((torch.rand(cache.weight.shape, generator=g, device="cuda") < 0.004) * 2.0)
    check_evict(cache, budget, recent)


def test_evict_of_more_heads_than_a_grid_has_rows():
    """Heads from 65536 on are moved by a launch of their own."""
    Z, H, C = 1025, 64, 12
    cache = make_cache(Z, H, C, 64, [(5 * z) % (C + 1) for z in range(Z)], seed=1, garbage=False)
    check_evict(cache, 7, 2)


def test_append_fp32_prompts():
    """fp32 keys and values at a prompt's length, of which one in some ten thousand lies at a border between codes."""
    from qflash_b200 import KV4Cache
    N, D = 3001, 128
    x = torch.randn(2, 3, N, 2 * D, generator=gen(4), device="cuda") * torch.exp(3 * torch.randn(2, 3, N, 1, generator=gen(5), device="cuda"))
    x[:, :, ::2] = (x[:, :, ::2] * 8).round() / 8  # many of them do
    cache = KV4Cache.empty(2, 3, N + 2, D)
    cache.append(x[..., :D], x[..., D:], new_lens=torch.tensor([N, 1234], dtype=torch.int32, device="cuda"))
    assert cache.lens.tolist() == [N, 1234]
    for t, codes, param in ((x[..., :D], cache.k_codes, cache.k_param), (x[..., D:], cache.v_codes, cache.v_param)):
        code, p = quantise(t)
        for z, n in enumerate(cache.lens.tolist()):
            assert torch.equal(codes[z, :, :n], pack(code)[z, :, :n]) and same(param[z, :, :n], p[z, :, :n])
            assert not codes[z, :, n:].any() and not param[z, :, n:].any()
    assert cache.read(5, dtype=FP32)[0].any()
    cache.check()


def test_append_and_evict_read_lengths_outside_the_cache_as_its_ends():
    from qflash_b200 import KV4Cache
    C, D, N = 20, 64, 8
    k = torch.randn(4, 2, N, D, generator=gen(6), device="cuda").to(BF16)
    cache, want = KV4Cache.empty(4, 2, C, D), KV4Cache.empty(4, 2, C, D)
    cache.lens.copy_(torch.tensor([-5, 3, -2 ** 31, 0], dtype=torch.int32))
    want.lens.copy_(torch.tensor([0, 3, 0, 0], dtype=torch.int32))
    for c in (cache, want):
        c.append(k, k.flip(2))
        c.check()  # nothing was dropped
    assert cache.lens.tolist() == [8, 11, 8, 8]
    for name in ("k_codes", "v_codes", "k_param", "v_param", "weight", "lens"):
        assert torch.equal(getattr(cache, name), getattr(want, name)), name
    full = KV4Cache.empty(2, 2, C, D)
    full.lens.copy_(torch.tensor([C + 7, 2 ** 31 - 1], dtype=torch.int32))
    full.append(k[:2], k[:2], new_lens=torch.tensor([0, 0], dtype=torch.int32, device="cuda"))
    full.check()
    assert full.lens.tolist() == [C, C]
    full.lens.fill_(C + 1)
    full.append(k[:2], k[:2])
    assert full.lens.tolist() == [C, C] and not full.k_codes.any()
    with pytest.raises(OverflowError):
        full.check()
    cache.lens.copy_(torch.tensor([-5, C + 3, 2 ** 31 - 1, 4], dtype=torch.int32))
    to = KV4Cache.empty(4, 2, 6, D)
    kept = cache.evict(6, 2, out=to)
    assert to.lens.tolist() == [0, 6, 6, 4]
    assert (kept[0] == -1).all() and kept[1, 0, -2:].tolist() == [C - 2, C - 1] and kept[3, 0].tolist() == [0, 1, 2, 3, -1, -1]


def test_attend_of_no_rows_still_sets_the_weights():
    """Weights of stored positions become those given plus nothing, as with rows that all see nothing."""
    for lens in ([300, 0, 17], [5000, 4999, 1]):
        cache = make_cache(3, 2, max(lens), 64, lens)
        before, start = cache.weight.clone(), torch.rand(cache.weight.shape, generator=gen(3), device="cuda")
        q = torch.empty(3, 4, 0, 64, dtype=BF16, device="cuda")
        assert cache.attend(q, accumulate=True, weights=start).shape == q.shape
        live = (torch.arange(max(lens), device="cuda") < cache.lens[:, None])[:, None, :].expand(cache.weight.shape)
        assert torch.equal(cache.weight, torch.where(live, start, before))
        cache.attend(q, accumulate=True)
        cache.attend(q)
        assert torch.equal(cache.weight, torch.where(live, start, before))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("N", [2, 60])
@pytest.mark.parametrize("rising", [0, 30, 150, 300, 700])
@pytest.mark.parametrize("power", [0, 40, 88, -88])
def test_values_of_any_scale_under_rising_scores(power, rising, N, dtype):
    """Probabilities are formed against a reference that lags behind where a CTA walks from tile to tile (so there are
    more heads than CTAs); with the values' scale they must neither overflow nor vanish, in the kernels for few and for
    many rows alike."""
    D, H, n = 64, 160, 700
    cache = make_cache(1, H, n, D, [n], garbage=False)
    cache.v_param[..., 0] = (cache.v_param[..., 0].double() * 2.0 ** power).to(BF16)  # powers of two: exact
    q = torch.zeros(1, H, N, D, dtype=dtype, device="cuda")
    q[..., 0] = 1.0
    cache.k_codes.fill_(0)
    cache.k_codes[..., 0] = 1  # element 0 is the key's scale, the others 0
    ramp = torch.arange(n, device="cuda") / n * rising * np.log(2)  # scores rise by 2^rising in all
    jump = torch.where(torch.arange(n, device="cuda") % 64 == 37, 5.0 * (rising > 0), 0.0)
    cache.k_param[..., 0], cache.k_param[..., 1] = (ramp + jump).bfloat16(), 0.0
    want, spread, cols, size = attend64(cache, q, [N], True, 1.0)
    # errors of scores stay below 1/8, where exp(x) - 1 < 1.07 x
    assert 2 * score_error(size.max().item(), D) < 0.125
    many, weight = both_ways(cache, q, scale=1.0)
    outs = [cache.attend(q, scale=1.0), many]
    cache.check()
    for x in outs:
        if dtype is FP16 and power > 0:  # beyond the type: infinity wherever the value surely is
            sure = want.abs() > 2.0 ** 17 + 2.0 ** -8 * spread
            assert sure.any() and not torch.isnan(x).any()
            assert torch.equal(x[sure].double(), torch.sign(want[sure]) * torch.inf)
        else:
            close_to_the_rounding(x, want, spread * 1.1, size, D, n)
    # p by twice its score error, fp32 sums over the rows by half a step each; what is below fp32's range counts as 0
    tol = (1.1 * 2 * score_error(size.max(), D) + (N + 2) * 2.0 ** -24) * cols + N * 2.0 ** -126
    assert ((weight.double() - cols).abs() <= tol).all()
