"""The 4-bit key/value cache on the GPU against plain 64-bit forms of its operators."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
HALF_STEP = {BF16: 2.0 ** -8, FP16: 2.0 ** -11, FP32: 2.0 ** -24}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def quantise(x):
    """Codes [..., D] and (scale, zero) of the header's formula; every rounding written out."""
    x64 = x.double()
    lo, hi = x64.amin(-1).clamp(max=0), x64.amax(-1).clamp(min=0)
    scale = ((hi - lo) / 15).float().bfloat16()
    s = scale.float()
    zero = torch.where(s > 0, ((-lo).float() / s).round().clamp(0, 15), 0)
    code = torch.where(s[..., None] > 0, ((x.float() / s[..., None]).round() + zero[..., None]).clamp(0, 15), 0)
    bad = ~torch.isfinite(x64).all(-1)
    scale = torch.where(bad, torch.full_like(scale, math.nan), scale)
    zero, code = torch.where(bad, 0, zero), torch.where(bad[..., None], 0, code)
    return code.to(torch.uint8), torch.stack((scale, zero.bfloat16()), -1)


def same(a, b):
    """Equal, NaN to NaN."""
    return a.shape == b.shape and bool(((a == b) | (torch.isnan(a) & torch.isnan(b))).all())


def unpack(codes):
    return torch.stack((codes & 15, codes >> 4), -1).flatten(-2)


def pack(code):
    return code[..., 0::2] | code[..., 1::2] << 4


def values(codes, param):
    p = param.double()
    return p[..., :1] * (unpack(codes).double() - p[..., 1:])


def make_cache(Z, H, C, D, lens, seed=0, strength=1.0, garbage=True):
    """A cache of random vectors; behind each sequence's length there is garbage that must not leak."""
    from qflash_b200 import KV4Cache
    g = gen(seed)
    bufs = []
    for _ in range(2):
        code, param = quantise((torch.randn(Z, H, C, D, generator=g, device="cuda") * strength).to(BF16))
        bufs.append((pack(code), param))
    lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    if garbage:
        behind = (torch.arange(C, device="cuda") >= lens[:, None])[:, None, :].expand(Z, H, C)
        for codes, param in bufs:
            codes[behind] = 255
            param[behind] = math.nan
    weight = torch.rand(Z, H, C, generator=g, device="cuda")
    return KV4Cache(bufs[0][0], bufs[1][0], bufs[0][1], bufs[1][1], weight, lens)


def attend64(cache, q, new, causal, scale=None):
    """(out, sum of p |v|, column sums of p, score error per row) in 64 bits."""
    Z, H, C, D = cache.shape
    _, Hq, N, _ = q.shape
    rep = Hq // H
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    spread, cols = torch.zeros_like(out), torch.zeros(Z, H, C, dtype=torch.float64, device="cuda")
    size = torch.zeros(Z, Hq, N, 1, dtype=torch.float64, device="cuda")
    for z, (n, m) in enumerate(zip(cache.lens.tolist(), new)):
        n = min(max(n, 0), C)
        K, V = values(cache.k_codes[z, :, :n], cache.k_param[z, :, :n]), values(cache.v_codes[z, :, :n], cache.v_param[z, :, :n])
        for i in range(m):
            seen = max(0, n - m + i + 1) if causal else n
            if not seen:
                continue
            x = q[z, :, i].double().view(H, rep, D)
            s = torch.einsum("hrd,hjd->hrj", x, K[:, :seen]) * scale
            p = torch.softmax(s, -1)
            out[z, :, i] = torch.einsum("hrj,hjd->hrd", p, V[:, :seen]).reshape(Hq, D)
            spread[z, :, i] = torch.einsum("hrj,hjd->hrd", p, V[:, :seen].abs()).reshape(Hq, D)
            cols[z, :, :seen] += p.sum(1)
            size[z, :, i, 0] = (torch.einsum("hrd,hjd->hrj", x.abs(), K[:, :seen].abs()).amax(-1) * abs(scale)).reshape(Hq)
    return out, spread, cols, size


def score_error(size, D):
    # fp32 sums of exact products in D / 16 steps, each off by at most 2^-22 of the terms' size, then a product
    # with the fp32 scale (2^-23 with its own rounding), a difference to the maximum and an exp2 of 2^-22
    return (D / 16 + 2) * 2.0 ** -22 * size + 2.0 ** -21


def close_out(got, want, spread, size, D, n):
    dt = got.dtype
    # each p is off by twice the score error (its own and the sum's), P v by the rounding of P (bf16: one term;
    # fp16: two terms), the sums over n keys by 2^-22 per step of 16; the output by its rounding
    p_off = 2 * score_error(size, D) + (2.0 ** -8 if dt is BF16 else 2.0 ** -16) + (n / 16 + 8) * 2.0 ** -22
    tol = p_off * spread + HALF_STEP[dt] * want.abs() * (1 + 2.0 ** -6) + (2.0 ** -25 if dt is FP16 else 0)
    off = (got.double() - want).abs()
    assert not torch.isnan(got).any()
    worst = (off / tol.clamp(min=1e-300)).max().item() if off.numel() else 0.0
    assert worst <= 1, f"off by {worst:.3g} times the tolerance"


def queries(Z, Hq, N, D, dtype, seed, layout="znhd"):
    g = gen(seed + 100)
    x = torch.randn(Z, N, Hq, D, generator=g, device="cuda").to(dtype)
    return x.transpose(1, 2) if layout == "znhd" else x.transpose(1, 2).contiguous()


# ------------------------------------------------------------------ append, read
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("Z, H, N, C", [(1, 1, 1, 1), (3, 2, 7, 20), (2, 5, 33, 61)])
def test_append_codes(D, dtype, Z, H, N, C):
    from qflash_b200 import KV4Cache
    g = gen(N + D)
    x = (torch.randn(Z, H, N, 2 * D, generator=g, device="cuda") * torch.exp(4 * torch.randn(Z, H, N, 1, generator=g, device="cuda"))).to(dtype)
    k, v = x[..., :D], x[..., D:].abs()
    cache = KV4Cache.empty(Z, H, C, D)
    cache.weight.fill_(3)
    cache.append(k, v)
    assert cache.lens.tolist() == [N] * Z
    for t, codes, param in ((k, cache.k_codes, cache.k_param), (v, cache.v_codes, cache.v_param)):
        code, p = quantise(t)
        assert torch.equal(unpack(codes[:, :, :N]), code)
        assert same(param[:, :, :N], p)
        assert not codes[:, :, N:].any() and not param[:, :, N:].any()
    assert (cache.weight[:, :, :N] == 0).all() and (cache.weight[:, :, N:] == 3).all()
    for out in (BF16, FP16, FP32):
        rk, rv = cache.read(C, dtype=out)
        for got, codes, param in ((rk, cache.k_codes, cache.k_param), (rv, cache.v_codes, cache.v_param)):
            want = values(codes, param).float().to(out)  # 13 bits: exact in fp32
            assert same(got[:, :, :N], want[:, :, :N]) and not got[:, :, N:].any()
    cache.check()


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_append_hard_vectors(dtype):
    from qflash_b200 import KV4Cache
    D, top, tiny = 64, torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    rows = []
    for head in ([0.0], [-0.0], [1.0], [-1.0], [top, -top], [top], [-top], [tiny, -tiny / 4], [tiny / 8], [math.inf],
                 [-math.inf, 1.0], [math.nan], [5.0, math.nan, math.inf], list(np.linspace(-1, 1, D)),
                 list(np.linspace(3, 4, D)), list(np.linspace(-4, -3, D)), [i - 7.5 for i in range(16)],
                 [15.0] + [i + 0.5 for i in range(15)]):
        rows.append(head + [0.0] * (D - len(head)))
    x = torch.tensor(rows, dtype=torch.float64, device="cuda").to(dtype)[None, None]
    cache = KV4Cache.empty(1, 1, x.shape[2], D)
    cache.append(x, x.flip(-1))
    for t, codes, param in ((x, cache.k_codes, cache.k_param), (x.flip(-1), cache.v_codes, cache.v_param)):
        code, p = quantise(t)
        assert torch.equal(unpack(codes), code)
        assert same(param, p)
    bad = ~torch.isfinite(x[0, 0]).all(-1)
    k, _ = cache.read(dtype=FP32)
    assert torch.equal(torch.isnan(k[0, 0]).all(-1), bad) and torch.equal(torch.isnan(k[0, 0]).any(-1), bad)


def test_append_every_16_bit_quotient_at_a_border():
    """Vectors whose elements sit at and next to the borders between codes: fp32 quotients must round as exact ones."""
    from qflash_b200 import KV4Cache
    g = gen(3)
    n, D = 4096, 128
    top = torch.rand(n, 1, generator=g, device="cuda") * 15 + 1
    scale = ((top.to(BF16).double()) / 15).float().bfloat16().double()
    border = torch.randint(0, 15, (n, D), generator=g, device="cuda") + 0.5
    x = (scale * border).to(BF16)
    x[:, 0] = top[:, 0].to(BF16)
    cache = KV4Cache.empty(1, 1, n, D)
    cache.append(x[None, None], -x[None, None])
    for t, codes, param in ((x, cache.k_codes, cache.k_param), (-x, cache.v_codes, cache.v_param)):
        code, p = quantise(t)
        assert torch.equal(param[0, 0], p)
        s = p[..., :1].double()
        exact = ((t.double() / s).round() + p[..., 1:].double()).clamp(0, 15).to(torch.uint8)
        assert torch.equal(exact, code)  # the fp32 quotient of 16-bit numbers never crosses a border
        assert torch.equal(unpack(codes[0, 0]), exact)


@pytest.mark.parametrize("shift", [0, 1])
def test_append_strides_and_alignment(shift):
    """Head-interleaved projections, and views that start on no 16-byte boundary."""
    from qflash_b200 import KV4Cache
    Z, N, H, D = 2, 9, 3, 64
    buf = torch.randn(Z * N * 2 * H * D + 8, generator=gen(1), device="cuda").to(BF16)
    qkv = buf[shift:shift + Z * N * 2 * H * D].view(Z, N, 2, H, D).permute(2, 0, 3, 1, 4)
    cache, plain = KV4Cache.empty(Z, H, 12, D), KV4Cache.empty(Z, H, 12, D)
    cache.append(qkv[0], qkv[1])
    plain.append(qkv[0].clone(memory_format=torch.contiguous_format), qkv[1].clone(memory_format=torch.contiguous_format))
    for n in ("k_codes", "v_codes", "k_param", "v_param", "lens"):
        assert torch.equal(getattr(cache, n), getattr(plain, n))
    inner = qkv[0].transpose(-1, -2).contiguous().transpose(-1, -2)  # head dim not innermost
    cache.append(inner, qkv[1], at=torch.zeros(Z, dtype=torch.int32, device="cuda"))
    assert torch.equal(cache.k_codes, plain.k_codes)


def test_append_positions_and_overflow():
    from qflash_b200 import KV4Cache
    Z, H, C, D, N = 5, 2, 10, 64, 4
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    k = torch.randn(Z, H, N, D, generator=gen(5), device="cuda")
    cache = KV4Cache.empty(Z, H, C, D)
    for t in (cache.k_codes, cache.v_codes):
        t.fill_(0x77)
    cache.weight.fill_(1)
    cache.append(k, k, new_lens=i32(0, 1, 4, 9, -3))
    assert cache.lens.tolist() == [0, 1, 4, 4, 0]
    cache.check()
    cache.append(k, k, new_lens=i32(2, 2, 2, 2, 2), at=i32(0, 0, 8, 3, 5))
    assert cache.lens.tolist() == [2, 2, 10, 5, 7]
    cache.check()
    code = pack(quantise(k)[0])
    written = torch.zeros(Z, C, dtype=torch.bool, device="cuda")
    for z, (first, m) in enumerate(((0, 2), (0, 2), (8, 2), (3, 2), (5, 2))):
        assert torch.equal(cache.k_codes[z, :, first:first + m], code[z, :, :m])
        written[z, first:first + m] = True
    written[1, 0], written[2, :4], written[3, :4] = True, True, True
    assert (cache.k_codes.transpose(1, 2)[~written] == 0x77).all() and (cache.weight.transpose(1, 2)[~written] == 1).all()
    cache.append(k, k, at=i32(8, 10, 0, -1, 2 ** 31 - 2))  # past the end, before the beginning
    assert cache.lens.tolist() == [10, 10, 4, 3, 10]
    with pytest.raises(OverflowError):
        cache.check()
    cache.check()  # reported once
    assert torch.equal(cache.k_codes[0, :, 8:], code[0, :, :2]) and torch.equal(cache.k_codes[3, :, :3], code[3, :, 1:])


def test_read_positions():
    cache = make_cache(4, 2, 50, 64, [50, 0, 13, 60])
    start = torch.tensor([45, 0, -2, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    k, v = cache.read(20, start=start, dtype=FP32)
    for got, codes, param in ((k, cache.k_codes, cache.k_param), (v, cache.v_codes, cache.v_param)):
        want = values(codes, param).float()
        assert torch.equal(got[0, :, :5], want[0, :, 45:]) and not got[0, :, 5:].any()
        assert not got[1].any() and not got[3].any()
        assert torch.equal(got[2, :, 2:15], want[2, :, :13]) and not got[2, :, :2].any() and not got[2, :, 15:].any()
    assert cache.read(0)[0].shape == (4, 2, 0, 64)
    full, _ = cache.read()
    assert full.shape == (4, 2, 50, 64) and full.dtype is BF16


# ------------------------------------------------------------------ attend
CASES = [  # Z, H, rep, N, C, lens, new, causal
    (1, 1, 1, 1, 1, [1], None, True),
    (1, 2, 1, 1, 130, [129], None, True),
    (4, 3, 4, 1, 300, [300, 1, 0, 128], [1, 1, 0, 1], True),
    (3, 2, 7, 1, 700, [31, 33, 700], None, True),
    (2, 2, 8, 1, 515, [515, 256], None, False),
    (2, 1, 16, 1, 257, [255, 257], None, True),
    (2, 2, 5, 3, 400, [399, 2], None, True),
    (2, 2, 1, 17, 99, [99, 20], [17, 5], True),
    (3, 1, 3, 40, 300, [300, 40, 7], [40, 40, 7], True),
    (2, 2, 4, 70, 150, [150, 64], [70, 1], False),
    (2, 1, 2, 150, 290, [290, 130], [150, 130], True),
    (1, 1, 64, 2, 140, [139], None, True),
]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("Z, H, rep, N, C, lens, new, causal", CASES)
def test_attend(D, dtype, Z, H, rep, N, C, lens, new, causal):
    cache = make_cache(Z, H, C, D, lens, seed=N + C)
    q = queries(Z, H * rep, N, D, dtype, seed=C)
    counts = new or [N] * Z
    nl = None if new is None else torch.tensor(new, dtype=torch.int32, device="cuda")
    want, spread, cols, size = attend64(cache, q, [min(c, N) for c in counts], causal)
    out = cache.attend(q, causal=causal, new_lens=nl)
    close_out(out, want, spread, size, D, C)
    # the same with weights: outputs as before, every stored position's weight, nothing behind them touched
    before = cache.weight.clone()
    start = torch.rand(Z, H, C, generator=gen(9), device="cuda")
    both = torch.empty_like(q)
    cache.attend(q, causal=causal, new_lens=nl, accumulate=True, weights=start, out=both)
    close_out(both, want, spread, size, D, C)
    live = (torch.arange(C, device="cuda") < cache.lens[:, None])[:, None, :].expand(Z, H, C)
    # p is off by twice its score error, fp32 sums over the rows by half a step each
    tol = (2 * score_error(size.max(), D) + (rep * N + 2) * 2.0 ** -24) * cols + 2.0 ** -23 * (start.double() + cols) + 1e-30
    off = (cache.weight.double() - start.double() - cols).abs()
    assert ((off / tol)[live] <= 1).all(), (off / tol)[live].max()
    assert torch.equal(cache.weight[~live], before[~live])


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("Z, H, rep, D, lens", [(1, 2, 4, 128, [20000]), (5, 1, 8, 64, [9000, 1, 0, 130, 4097]), (40, 2, 2, 64, None)])
def test_attend_long_and_many(dtype, Z, H, rep, D, lens):
    """Units cut over many CTAs, many units in one, and both in one batch."""
    lens = lens or [(37 * z) % 260 for z in range(Z)]
    C = max(lens) + 3
    cache = make_cache(Z, H, C, D, lens, seed=Z)
    q = queries(Z, H * rep, 1, D, dtype, seed=1, layout="zhnd")
    new = [min(1, n) for n in lens]
    want, spread, cols, size = attend64(cache, q, new, True)
    cache.weight.zero_()
    out = cache.attend(q, accumulate=True)
    close_out(out, want, spread, size, D, C)
    close_out(cache.attend(q, causal=False), want, spread, size, D, C)
    tol = (2 * score_error(size.max(), D) + (rep + 4) * 2.0 ** -24) * cols + 1e-30
    live = (torch.arange(C, device="cuda") < cache.lens[:, None])[:, None, :].expand(Z, H, C)
    assert (((cache.weight.double() - cols).abs() / tol)[live] <= 1).all()


@pytest.mark.parametrize("N", [1, 200])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_attend_values_of_any_size(N, dtype):
    """Scales far from 1: the values' scale may be far outside fp16."""
    cache = make_cache(2, 1, 300, 64, [300, 250], strength=1.0)
    for f in (1e-6, 1e-3, 300.0):
        c2 = make_cache(2, 1, 300, 64, [300, 250], strength=1.0)
        c2.v_param[..., 0] = (cache.v_param[..., 0].float() * f).bfloat16()
        q = queries(2, 4, N, 64, dtype, seed=2)
        want, spread, _, size = attend64(c2, q, [N, N], True)
        close_out(c2.attend(q), want, spread, size, 64, 300)


@pytest.mark.parametrize("N", [1, 5, 200])
def test_attend_scale_and_sharp_rows(N):
    """Scores far apart: a softmax of one or few positions, and moving maxima."""
    cache = make_cache(2, 2, 400, 128, [400, 211], strength=3.0)
    for scale in (0.7, 3.0, -0.5, 0.0):
        q = queries(2, 8, N, 128, FP16, seed=4)
        want, spread, _, size = attend64(cache, q, [N, N], True, scale)
        # errors of scores are larger here; they stay below 1/8, where exp(x) - 1 < 1.07 x
        assert 2 * score_error(size.max().item(), 128) < 0.125
        close_out(cache.attend(q, scale=scale), want, spread * 1.1, size, 128, 400)


@pytest.mark.parametrize("N", [1, 130])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_attend_poisoned_token_reaches_only_rows_that_see_it(N, dtype):
    cache = make_cache(1, 2, 260, 64, [260])
    cache.k_param[0, 0, 255, 0] = math.nan  # head 0's key
    cache.v_param[0, 1, 256, 0] = math.nan  # head 1's value
    q = queries(1, 4, N, 64, dtype, seed=8)
    out = cache.attend(q)
    first = 260 - N
    for i in range(N):
        assert torch.isnan(out[0, :2, i]).all() == (first + i >= 255), i
        assert torch.isnan(out[0, 2:, i]).all() == (first + i >= 256), i
        if first + i < 255:
            assert torch.isfinite(out[0, :, i]).all()


@pytest.mark.parametrize("N", [1, 130])
def test_attend_infinite_queries(N):
    """As a softmax in 64 bits has it: a score of +inf gives NaN, one of -inf weight 0."""
    D = 64
    cache = make_cache(1, 1, 140, D, [140])
    cache.k_codes.fill_(0x88)
    cache.k_param[..., 0], cache.k_param[..., 1] = 1.0, 7.0  # every key is all ones ...
    cache.k_codes[0, 0, 5] = 0x66  # ... but one of minus ones
    q = torch.zeros(1, 2, N, D, dtype=BF16, device="cuda")
    q[:, 0] = -math.inf
    q[:, 1] = math.inf
    out = cache.attend(q, causal=False)
    assert torch.isnan(out).all()
    q[:, 0] = 0
    q[:, 0, :, 3] = 1.0
    want, spread, _, size = attend64(cache, q[:, :1], [N], False)
    close_out(cache.attend(q[:, :1].contiguous(), causal=False), want, spread, size, D, 140)


@pytest.mark.parametrize("N", [1, 3, 160])
def test_attend_strided_output_and_rows_behind(N):
    """Outputs as a [Z, N, Hq, D] buffer inside a larger one: nothing else is written."""
    Z, H, rep, D = 2, 2, 3, 64
    cache = make_cache(Z, H, 333, D, [333, 170])
    q = queries(Z, H * rep, N, D, BF16, seed=3)
    buf = torch.full((Z, N + 2, H * rep, D + 16), 7.0, dtype=BF16, device="cuda")
    view = buf[:, 1:1 + N, :, 8:8 + D].transpose(1, 2)
    got = cache.attend(q, out=view)
    assert got.data_ptr() == view.data_ptr() and torch.equal(view, cache.attend(q))
    buf[:, 1:1 + N, :, 8:8 + D] = 7.0
    assert (buf == 7).all()
    odd = torch.empty(Z * N * H * rep * D + 1, dtype=BF16, device="cuda")[1:].view(Z, N, H * rep, D).transpose(1, 2)
    odd.copy_(q)
    assert torch.equal(cache.attend(odd), cache.attend(q))


def test_attend_same_result_every_time():
    cache = make_cache(3, 2, 900, 128, [900, 411, 5])
    q = queries(3, 8, 1, 128, BF16, seed=6)
    first = cache.attend(q, accumulate=True, weights=torch.zeros_like(cache.weight))
    w = cache.weight.clone()
    for _ in range(5):
        again = cache.attend(q, accumulate=True, weights=torch.zeros_like(cache.weight))
        assert torch.equal(first, again) and torch.equal(w, cache.weight)


def test_attend_refusals():
    from qflash_b200 import _lib
    cache = make_cache(2, 2, 30, 64, [30, 3])
    q = queries(2, 4, 1, 64, BF16, seed=1)
    for bad in (q.float(), q[:1], q[:, :3], queries(2, 4, 1, 128, BF16, 1), q[0]):
        with pytest.raises(ValueError):
            cache.attend(bad)
    with pytest.raises(ValueError):
        cache.attend(q.cpu())
    with pytest.raises(ValueError, match="without accumulate"):
        cache.attend(q, weights=cache.weight)
    with pytest.raises(ValueError, match="weights"):
        cache.attend(q, accumulate=True, weights=cache.weight.double())
    with pytest.raises(ValueError, match="new_lens"):
        cache.attend(q, new_lens=torch.ones(2, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError, match="out"):
        cache.attend(q, out=q.half())
    with pytest.raises(_lib.QFlashError, match="above 64"):
        cache.attend(queries(2, 130, 1, 64, BF16, 1))
    with pytest.raises(_lib.QFlashError, match="finite"):
        cache.attend(q, scale=math.inf)
    with pytest.raises(ValueError):
        cache.append(q, q)
    with pytest.raises(ValueError):
        cache.append(q[:, :2], q[:, :2].half())
    with pytest.raises(ValueError):
        cache.read(-1)
    with pytest.raises(ValueError):
        cache.read(dtype=torch.int8)
    assert cache.attend(q[:, :, :0]).shape == (2, 4, 0, 64)


# ------------------------------------------------------------------ evict
def evict64(cache, budget, recent):
    kept = torch.full((*cache.shape[:2], budget), -1, dtype=torch.int32)
    w = cache.weight.cpu().numpy()
    for z, n in enumerate(cache.lens.tolist()):
        for h in range(cache.shape[1]):
            if n <= budget:
                keep = list(range(n))
            else:
                old, x = n - recent, w[z, h]
                heavy = sorted(range(old), key=lambda j: (0 if math.isnan(x[j]) else 1, 0.0 if math.isnan(x[j]) else -float(x[j]), j))
                keep = sorted(heavy[:budget - recent]) + list(range(old, n))
            kept[z, h, :len(keep)] = torch.tensor(keep, dtype=torch.int32)
    return kept.cuda()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("C, lens, budget, recent", [
    (1, [1, 0], 1, 0), (40, [40, 17], 16, 4), (40, [40, 16], 16, 16), (40, [40, 15], 16, 0), (300, [300, 299], 299, 1),
    (5000, [5000, 3001], 1000, 100), (5000, [4097, 1025], 1024, 1023), (3000, [3000, 2048], 1, 0)])
@pytest.mark.parametrize("kind", ["random", "equal", "few", "odd"])
def test_evict(D, C, lens, budget, recent, kind):
    from qflash_b200 import KV4Cache
    cache = make_cache(2, 3, C, D, lens, seed=C)
    g = gen(C + budget)
    if kind == "equal":
        cache.weight.fill_(0.25)
    elif kind == "few":
        cache.weight.copy_(torch.randint(0, 3, cache.weight.shape, generator=g, device="cuda"))
    elif kind == "odd":
        w = torch.randn(cache.weight.shape, generator=g, device="cuda") * 1e-3
        w[..., ::5], w[..., 1::7], w[..., 2::11], w[..., 3::13], w[..., 4::17] = 0.0, -0.0, math.nan, math.inf, 1e-42
        cache.weight.copy_(w)
    behind = torch.arange(C, device="cuda") >= cache.lens[:, None]
    cache.weight.transpose(1, 2)[behind] = math.inf  # not stored: never kept
    to = KV4Cache.empty(2, 3, budget + 5, D)
    to.weight.fill_(-1)
    want = evict64(cache, budget, recent)
    kept = cache.evict(budget, recent, out=to)
    assert torch.equal(kept, want)
    assert to.lens.tolist() == [min(n, budget) for n in lens]
    there = want >= 0
    at = want.clamp(min=0).long()
    for name in ("k_codes", "v_codes", "k_param", "v_param"):
        src = getattr(cache, name)
        rows = torch.gather(src, 2, at[..., None].expand(*at.shape, src.shape[-1]))
        got = getattr(to, name)
        assert torch.equal(got[:, :, :budget][there], rows[there])
        assert not got[:, :, :budget][~there].any() and not got[:, :, budget:].any()
    wt = torch.gather(cache.weight, 2, at)
    assert torch.equal(to.weight[:, :, :budget][there].view(torch.int32), wt[there].view(torch.int32))
    assert (to.weight[:, :, :budget][~there] == -1).all() and (to.weight[:, :, budget:] == -1).all()


def test_evict_long():
    from qflash_b200 import KV4Cache
    C = 70001
    cache = make_cache(1, 2, C, 64, [C], garbage=False)
    to = KV4Cache.empty(1, 2, 4000, 64)
    assert torch.equal(cache.evict(4000, 333, out=to), evict64(cache, 4000, 333))


def test_evict_refusals():
    from qflash_b200 import KV4Cache, _lib
    cache, to = make_cache(2, 2, 30, 64, [30, 3]), KV4Cache.empty(2, 2, 8, 64)
    for budget, recent in ((0, 0), (9, 0), (4, 5), (4, -1)):
        with pytest.raises(ValueError):
            cache.evict(budget, recent, out=to)
    for other in (KV4Cache.empty(1, 2, 8, 64), KV4Cache.empty(2, 1, 8, 64), KV4Cache.empty(2, 2, 8, 128)):
        with pytest.raises(ValueError):
            cache.evict(4, 1, out=other)
    with pytest.raises(_lib.QFlashError, match="share memory"):
        cache.evict(4, 1, out=cache)


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_prompt_decode_evict_decode(dtype):
    """As a serving loop uses them: two prompts, decoding with weights, eviction, decoding on; each step against the
    64-bit form of what the cache holds."""
    from qflash_b200 import KV4Cache
    Z, H, rep, D, N = 2, 2, 2, 64, 150
    g = gen(11)
    new = torch.tensor([150, 90], dtype=torch.int32, device="cuda")
    cache = KV4Cache.empty(Z, H, 200, D)
    draw = lambda heads, n: torch.randn(Z, n, heads, D, generator=g, device="cuda").to(dtype).transpose(1, 2)  # noqa: E731
    total = torch.zeros(Z, H, 200, dtype=torch.float64, device="cuda")

    def step(c, n, counts):
        nonlocal total
        c.append(draw(H, n), draw(H, n), new_lens=counts)
        q = draw(H * rep, n)
        want, spread, cols, size = attend64(c, q, counts.tolist() if counts is not None else [n] * Z, True)
        close_out(c.attend(q, new_lens=counts, accumulate=True), want, spread, size, D, 200)
        total = total + cols
        live = (torch.arange(c.shape[2], device="cuda") < c.lens[:, None])[:, None, :].expand(total.shape)
        torch.testing.assert_close(c.weight[live].double(), total[live], rtol=2e-5, atol=0)

    step(cache, N, new)
    for _ in range(3):
        step(cache, 1, None)
    small = KV4Cache.empty(Z, H, 80, D)
    kept = cache.evict(64, 16, out=small)
    assert torch.equal(kept, evict64(cache, 64, 16)) and small.lens.tolist() == [64, 64]
    total = torch.zeros(Z, H, 80, dtype=torch.float64, device="cuda").scatter_(2, torch.arange(64, device="cuda").expand(Z, H, 64), torch.gather(total, 2, kept.long()))
    step(small, 2, torch.tensor([2, 1], dtype=torch.int32, device="cuda"))
    for _ in range(2):
        step(small, 1, None)
    small.check()
    # what is stored also goes to the framework's attention over floats
    from qflash_b200 import qflash
    k, v = small.read(67, dtype=dtype)
    assert qflash.forward(draw(H, 67), k, v).shape == (Z, H, 67, D)


def test_take_back_drafted_tokens():
    """`at` and `weights` put the cache back to where a draft began."""
    from qflash_b200 import KV4Cache
    Z, H, D = 2, 1, 64
    a, b = KV4Cache.empty(Z, H, 64, D), KV4Cache.empty(Z, H, 64, D)
    x = lambda n, s: torch.randn(Z, H, n, D, generator=gen(s), device="cuda").to(BF16)  # noqa: E731
    for c in (a, b):
        c.append(x(20, 1), x(20, 2))
        c.attend(x(20, 3), accumulate=True)
    at, weights = a.lens.clone(), a.weight.clone()
    a.append(x(5, 4), x(5, 5))
    a.attend(x(5, 6), accumulate=True)
    a.append(x(3, 7), x(3, 8), at=at)
    weights[:, :, 20:] = 0
    got = a.attend(x(3, 9), accumulate=True, weights=weights)
    b.append(x(3, 7), x(3, 8))
    want = b.attend(x(3, 9), accumulate=True)
    assert torch.equal(got, want) and torch.equal(a.weight[:, :, :23], b.weight[:, :, :23]) and torch.equal(a.lens, b.lens)


def test_captured_decoding_step():
    """append and attend in a CUDA graph: lengths move on the device, so a replay is the next step."""
    from qflash_b200 import KV4Cache
    Z, H, rep, D = 2, 2, 4, 128
    g = gen(21)
    a, b = KV4Cache.empty(Z, H, 300, D), KV4Cache.empty(Z, H, 300, D)
    k0 = torch.randn(Z, H, 140, D, generator=g, device="cuda").to(FP16)
    for c in (a, b):
        c.append(k0, k0.flip(2))
    kn, vn = (torch.empty(Z, H, 1, D, dtype=FP16, device="cuda") for _ in range(2))
    qn = torch.empty(Z, H * rep, 1, D, dtype=FP16, device="cuda")
    for t in (kn, vn, qn):
        t.zero_()
    small = [KV4Cache.empty(Z, H, 100, D) for _ in range(2)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        a.append(kn, vn)
        out = a.attend(qn, accumulate=True)
        kept = a.evict(64, 8, out=small[0])
    for i in range(4):
        for t in (kn, vn, qn):
            t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
        graph.replay()
        b.append(kn, vn)
        want = b.attend(qn, accumulate=True)
        assert torch.equal(out, want) and torch.equal(a.weight, b.weight) and a.lens.tolist() == [141 + i] * Z
        assert torch.equal(kept, b.evict(64, 8, out=small[1])) and torch.equal(small[0].k_codes, small[1].k_codes)


def test_two_streams_read_one_cache():
    cache = make_cache(4, 2, 2000, 128, [2000, 1500, 3, 700])
    qs = [queries(4, 8, 1, 128, BF16, seed=s) for s in range(2)] + [queries(4, 8, 180, 128, BF16, seed=5)]
    want = [cache.attend(q) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    got = [[], [], []]
    for _ in range(10):
        for s, q, g in zip(streams, qs, got):
            with torch.cuda.stream(s):
                g.append(cache.attend(q))
    torch.cuda.synchronize()
    assert all(torch.equal(x, w) for g, w in zip(got, want) for x in g)


# ------------------------------------------------------------------ the kernel for many rows
# (accumulate, or a large cache, leads there; the tests above reach it with accumulate only)
def both_ways(cache, q, scale=None, causal=True, new_lens=None):
    """attend with weights, from zeros; the weight buffer behind the stored tokens stays as it was."""
    w = torch.zeros_like(cache.weight)
    out = cache.attend(q, scale=scale, causal=causal, new_lens=new_lens, accumulate=True, weights=w)
    return out, cache.weight


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("Z, H, rep, N, lens, causal", [
    (2, 8, 4, 70, [4000, 1], True), (3, 8, 3, 129, [2500, 129, 0], True), (1, 16, 16, 33, [3001], False),
    (5, 4, 1, 300, [4099, 300, 0, 7, 2048], True)])
def test_many_rows_over_a_large_cache(D, dtype, Z, H, rep, N, lens, causal):
    C = max(lens) + 1
    cache = make_cache(Z, H, C, D, lens, seed=N)
    q = queries(Z, H * rep, N, D, dtype, seed=N)
    new = [min(N, n) for n in lens]
    nl = torch.tensor(new, dtype=torch.int32, device="cuda")
    want, spread, cols, size = attend64(cache, q, new, causal)
    close_out(cache.attend(q, causal=causal, new_lens=nl), want, spread, size, D, C)
    out, weight = both_ways(cache, q, causal=causal, new_lens=nl)
    close_out(out, want, spread, size, D, C)
    live = (torch.arange(C, device="cuda") < cache.lens[:, None])[:, None, :].expand(Z, H, C)
    tol = (2 * score_error(size.max(), D) + (rep * N + 4) * 2.0 ** -24) * cols + 1e-30
    assert (((weight.double() - cols).abs() / tol)[live] <= 1).all()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("rep, N, lens", [(64, 3, [500, 2]), (7, 37, [260, 259]), (5, 101, [101, 50]), (1, 257, [257, 1000])])
def test_many_rows_odd_groups(dtype, rep, N, lens):
    """Row tiles that end inside a token's heads, and sequences shorter than the query tensor."""
    C = max(lens)
    cache = make_cache(2, 2, C, 64, lens, seed=rep)
    q = queries(2, 2 * rep, N, 64, dtype, seed=rep)
    want, spread, _, size = attend64(cache, q, [N, N], True)
    out, _ = both_ways(cache, q)
    close_out(out, want, spread, size, 64, C)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_many_rows_values_of_any_size(dtype):
    for f in (1e-6, 1e-3, 300.0):
        cache = make_cache(2, 1, 300, 64, [300, 250])
        cache.v_param[..., 0] = (cache.v_param[..., 0].float() * f).bfloat16()
        q = queries(2, 4, 200, 64, dtype, seed=2)
        want, spread, _, size = attend64(cache, q, [200, 200], True)
        close_out(both_ways(cache, q)[0], want, spread, size, 64, 300)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("rising", [0, 30, 90, 300])
def test_many_rows_moving_reference(dtype, rising):
    """Scores that grow along the keys, by up to some hundred (log2) within a tile: the reference has to follow, before
    and after P was stored, and what was summed up against the old one must not be lost or overflow."""
    D, n, N = 64, 700, 120
    cache = make_cache(1, 1, n, D, [n], garbage=False)
    q = torch.zeros(1, 2, N, D, dtype=dtype, device="cuda")
    q[..., 0] = 1.0
    cache.k_codes.fill_(0)
    cache.k_codes[0, 0, :, 0] = 1  # element 0 is the key's scale, the others 0
    ramp = torch.arange(n, device="cuda") / n * rising * math.log(2)
    jump = torch.where(torch.arange(n, device="cuda") % 64 == 37, 5.0 * (rising > 0), 0.0)
    cache.k_param[0, 0, :, 0], cache.k_param[0, 0, :, 1] = (ramp + jump).bfloat16(), 0.0
    want, spread, _, size = attend64(cache, q, [N], True, 1.0)
    assert 2 * score_error(size.max().item(), D) < 0.125
    close_out(both_ways(cache, q, scale=1.0)[0], want, spread * 1.1, size, D, n)
    q[:, 1] = -q[:, 1]  # falling scores: nothing behind the first tile counts
    want, spread, _, size = attend64(cache, q, [N], True, 1.0)
    close_out(both_ways(cache, q, scale=1.0)[0], want, spread * 1.1, size, D, n)


def test_many_rows_scale_and_sharp_rows():
    cache = make_cache(2, 2, 400, 128, [400, 211], strength=3.0)
    for scale in (0.7, 3.0, -0.5, 0.0):
        q = queries(2, 8, 100, 128, FP16, seed=4)
        want, spread, _, size = attend64(cache, q, [100, 100], True, scale)
        assert 2 * score_error(size.max().item(), 128) < 0.125
        close_out(both_ways(cache, q, scale=scale)[0], want, spread * 1.1, size, 128, 400)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_many_rows_poisoned_token(dtype):
    cache = make_cache(1, 2, 260, 64, [260])
    cache.k_param[0, 0, 255, 0] = math.nan
    cache.v_param[0, 1, 256, 0] = math.nan
    q = queries(1, 4, 130, 64, dtype, seed=8)
    out, weight = both_ways(cache, q)
    seen = torch.arange(130, 260, device="cuda")
    assert torch.equal(torch.isnan(out[0, 0]).all(-1), seen >= 255) and torch.equal(torch.isnan(out[0, 2]).all(-1), seen >= 256)
    assert torch.isfinite(out[0, :2, :125]).all() and torch.isfinite(out[0, 2:, :126]).all()
    # rows that see the poisoned key have no weights to give, so no position that they see has one
    assert torch.isnan(weight[0, 0]).all() and torch.isfinite(weight[0, 1]).all()


def test_many_rows_infinite_queries():
    D = 64
    cache = make_cache(1, 1, 140, D, [140])
    cache.k_codes.fill_(0x88)
    cache.k_param[..., 0], cache.k_param[..., 1] = 1.0, 7.0
    cache.k_codes[0, 0, 5] = 0x66
    q = torch.zeros(1, 2, 100, D, dtype=BF16, device="cuda")
    q[:, 0] = -math.inf
    q[:, 1] = math.inf
    assert torch.isnan(both_ways(cache, q, causal=False)[0]).all()


@pytest.mark.parametrize("N", [40, 160])
def test_many_rows_strides(N):
    Z, H, rep, D = 2, 2, 3, 64
    cache = make_cache(Z, H, 333, D, [333, 170])
    q = queries(Z, H * rep, N, D, BF16, seed=3)
    want, _ = both_ways(cache, q)
    buf = torch.full((Z, N + 2, H * rep, D + 16), 7.0, dtype=BF16, device="cuda")
    view = buf[:, 1:1 + N, :, 8:8 + D].transpose(1, 2)
    assert torch.equal(cache.attend(q, accumulate=True, out=view), want)
    buf[:, 1:1 + N, :, 8:8 + D] = 7.0
    assert (buf == 7).all()
    odd = torch.empty(Z * N * H * rep * D + 1, dtype=BF16, device="cuda")[1:].view(Z, N, H * rep, D).transpose(1, 2)
    odd.copy_(q)
    assert torch.equal(both_ways(cache, odd)[0], want)
    out = torch.empty(Z * N * H * rep * D + 1, dtype=BF16, device="cuda")[1:].view(Z, N, H * rep, D).transpose(1, 2)
    assert torch.equal(cache.attend(odd, accumulate=True, out=out), want)


def test_many_rows_same_result_every_time_and_side_by_side():
    cache = make_cache(3, 4, 1500, 128, [1500, 411, 5])
    qs = [queries(3, 16, n, 128, BF16, seed=n) for n in (150, 90)]
    want = [cache.attend(q) for q in qs]
    again = [both_ways(cache, q) for q in qs][1][1].clone()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    got = [[], []]
    for _ in range(8):
        for s, q, g in zip(streams, qs, got):
            with torch.cuda.stream(s):
                g.append(cache.attend(q))
    torch.cuda.synchronize()
    assert all(torch.equal(x, w) for g, w in zip(got, want) for x in g)
    for _ in range(3):
        assert torch.equal(both_ways(cache, qs[1])[1], again)
    cache.check()


def test_captured_prompt_then_decoding():
    """A padded prompt with weights, then an eviction, in a graph whose lengths change between replays."""
    from qflash_b200 import KV4Cache
    Z, H, rep, D, N = 2, 2, 4, 64, 90
    g = gen(31)
    caches = [KV4Cache.empty(Z, H, 500, D) for _ in range(2)]
    small = [KV4Cache.empty(Z, H, 60, D) for _ in range(2)]
    k, v = (torch.zeros(Z, H, N, D, dtype=BF16, device="cuda") for _ in range(2))
    q = torch.zeros(Z, H * rep, N, D, dtype=BF16, device="cuda")
    new = torch.zeros(Z, dtype=torch.int32, device="cuda")

    def step(i):
        caches[i].append(k, v, new_lens=new)
        out = caches[i].attend(q, new_lens=new, accumulate=True)
        return out, caches[i].evict(50, 10, out=small[i])

    graph, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=s):
        out, kept = step(0)
    for counts in ([90, 13], [0, 90], [77, 1], [1, 0]):
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
        new.copy_(torch.tensor(counts, dtype=torch.int32))
        graph.replay()
        want, want_kept = step(1)
        assert torch.equal(out, want) and torch.equal(kept, want_kept)
        assert torch.equal(caches[0].weight, caches[1].weight) and torch.equal(caches[0].lens, caches[1].lens)
        assert torch.equal(small[0].v_codes, small[1].v_codes)


def test_another_current_device_and_thread():
    """The calls go by the cache's device and restore the caller's; two threads may share the library."""
    import threading
    from qflash_b200 import KV4Cache
    results = {}

    def work(i):
        c = KV4Cache.empty(1, 1, 200, 64, device="cuda:0")
        x = torch.randn(1, 1, 150, 64, generator=gen(i), device="cuda").half()
        c.append(x, x)
        results[i] = c.attend(x), c.weight

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(4):
        x = torch.randn(1, 1, 150, 64, generator=gen(i), device="cuda").half()
        c = KV4Cache.empty(1, 1, 200, 64)
        c.append(x, x)
        assert torch.equal(c.attend(x), results[i][0])
    assert torch.cuda.current_device() == 0


def test_lengths_outside_the_cache_read_as_its_ends():
    cache = make_cache(2, 1, 100, 64, [100, 0], garbage=False)
    q = queries(2, 2, 1, 64, FP16, seed=1)
    want = cache.attend(q)
    cache.lens.copy_(torch.tensor([2 ** 31 - 1, -5], dtype=torch.int32))
    assert torch.equal(cache.attend(q), want)
    k, _ = cache.read(100)
    assert k[0].any() and not k[1].any()


def test_positions_behind_2_to_the_31_bytes():
    """Codes, parameters and weights of the last head lie behind 2^32 bytes of the buffers."""
    from qflash_b200 import KV4Cache
    H, C, D = 3, 1 << 24, 128  # 2^30 bytes of codes per head
    cache = KV4Cache.empty(1, H, C, D)
    at = torch.tensor([C - 3], dtype=torch.int32, device="cuda")
    x = torch.randn(1, H, 3, D, generator=gen(1), device="cuda").half()
    cache.append(x, x.flip(2), at=at)
    assert cache.lens.item() == C
    k, v = cache.read(3, start=at, dtype=FP32)
    for t, got in ((x, k), (x.flip(2), v)):
        code, p = quantise(t)
        assert torch.equal(got.double(), p[..., :1].double() * (code.double() - p[..., 1:].double()))
    # all other positions are zeros with scale 0: scores 0, values 0
    q = queries(1, H, 1, D, FP16, seed=2) * 40
    out = cache.attend(q, accumulate=True)
    s = torch.einsum("hd,hjd->hj", q[0, :, 0].double(), k[0].double()) / D ** 0.5
    z = torch.exp(s).sum(-1) + (C - 3)
    want = torch.einsum("hj,hjd->hd", torch.exp(s) / z[:, None], v[0].double())
    spread = torch.einsum("hj,hjd->hd", torch.exp(s) / z[:, None], v[0].double().abs())
    # the sums of 2^24 exponentials are added up in 512 parts of 2^15, each by 8 threads: 2^12 steps of 2^-24
    assert ((out[0, :, 0].double() - want).abs() <= (2.0 ** -11) * spread + 2.0 ** -25).all()
    assert ((cache.weight[0, :, -3:].double() - torch.exp(s) / z[:, None]).abs() <= 2.0 ** -11 * torch.exp(s) / z[:, None]).all()
    small = KV4Cache.empty(1, H, 8, D)
    cache.weight[0, :, 77] = 5.0
    kept = cache.evict(4, 3, out=small)
    assert kept.tolist() == [[[77, C - 3, C - 2, C - 1]] * H]
    assert torch.equal(small.read(4, dtype=FP32)[0][:, :, 1:], k)


def test_append_of_no_rows_takes_tokens_back():
    cache = make_cache(3, 1, 20, 64, [20, 7, 0], garbage=False)
    none = torch.empty(3, 1, 0, 64, dtype=BF16, device="cuda")
    codes = cache.k_codes.clone()
    cache.append(none, none)
    assert cache.lens.tolist() == [20, 7, 0]
    cache.append(none, none, at=torch.tensor([5, 7, 25], dtype=torch.int32, device="cuda"))
    assert cache.lens.tolist() == [5, 7, 20] and torch.equal(cache.k_codes, codes)
    with pytest.raises(OverflowError):
        cache.check()


def test_buffers_cannot_be_replaced_or_shared():
    from qflash_b200 import KV4Cache
    cache = make_cache(1, 1, 20, 64, [20])
    with pytest.raises(AttributeError):
        cache.weight = torch.zeros_like(cache.weight)
    with pytest.raises(ValueError, match="different"):
        KV4Cache(cache.k_codes, cache.k_codes, cache.k_param, cache.v_param, cache.weight, cache.lens)


def test_out_must_not_be_the_query_or_expanded():
    cache = make_cache(1, 2, 20, 64, [20])
    q = torch.randn(1, 2, 3, 64, device="cuda").half()
    with pytest.raises(ValueError, match="its own"):
        cache.attend(q, out=q)
    with pytest.raises(ValueError, match="its own"):
        cache.attend(q, out=torch.empty(1, 2, 1, 64, dtype=q.dtype, device="cuda").expand_as(q))
    both = torch.stack((q, q), dim=2)  # the query's rows between the output's
    assert torch.equal(cache.attend(both[:, :, 0], out=both[:, :, 1]), cache.attend(q))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("C", [150, 1400])
@pytest.mark.parametrize("rep, N", [(1, 1), (2, 1), (3, 1), (1, 5), (7, 1), (3, 3), (1, 11), (6, 3), (5, 6), (9, 4), (47, 1), (4, 12), (7, 7)])
def test_weights_of_any_number_of_rows(rep, N, C, dtype):
    """Scores are stored in twos or fours of rows, and read back as such; above 48 rows they are computed again."""
    lens, new = [C - 1, 3, C // 2, 0], [N, min(N, 3), (N + 1) // 2, 0]
    cache = make_cache(4, 2, C, 64, lens, seed=rep)
    q = queries(4, 2 * rep, N, 64, dtype, seed=N)
    want, spread, cols, size = attend64(cache, q, new, True)
    start, before = torch.rand(4, 2, C, generator=gen(3), device="cuda"), cache.weight.clone()
    out = cache.attend(q, new_lens=torch.tensor(new, dtype=torch.int32, device="cuda"), accumulate=True, weights=start)
    close_out(out, want, spread, size, 64, C)
    live = (torch.arange(C, device="cuda") < cache.lens[:, None])[:, None, :].expand(4, 2, C)
    # as in test_attend: p by twice its score error, fp32 sums over the rows by half a step each
    tol = (2 * score_error(size.max(), 64) + (rep * N + 2) * 2.0 ** -24) * cols + 2.0 ** -23 * (start.double() + cols) + 1e-30
    off = (cache.weight.double() - start.double() - cols).abs()
    assert ((off / tol)[live] <= 1).all(), (off / tol)[live].max()
    assert same(cache.weight[~live], before[~live])


@pytest.mark.parametrize("Z, N, accumulate", [(3, 1, False), (3, 1, True), (3, 700, False), (40, 60, True), (70, 3, True), (1, 5000, False)])
@pytest.mark.parametrize("empty", ["cache", "rows"])
def test_attend_where_nothing_is_seen(Z, N, accumulate, empty):
    lens = [0] * Z if empty == "cache" else [(31 * z) % 400 for z in range(Z)]
    cache = make_cache(Z, 2, 400, 64, lens, seed=Z)
    before = cache.weight.clone()
    new = torch.zeros(Z, dtype=torch.int32, device="cuda") if empty == "rows" else None
    q = queries(Z, 4, N, 64, BF16, seed=N)
    out = torch.full_like(q, float("nan"))
    cache.attend(q, new_lens=new, accumulate=accumulate, out=out)
    assert not out.any() and same(cache.weight, before)
    cache.check()


def test_attend_prompts_of_many_sequences():
    Z, N = 70, 40
    lens = [(37 * z) % 300 for z in range(Z)]
    cache = make_cache(Z, 1, 300, 64, lens, seed=2)
    q, new = queries(Z, 2, N, 64, FP16, seed=5), [min(n, N - z % 20) for z, n in enumerate(lens)]
    want, spread, cols, size = attend64(cache, q, new, True)
    cache.weight.zero_()
    out = cache.attend(q, new_lens=torch.tensor(new, dtype=torch.int32, device="cuda"), accumulate=True)
    close_out(out, want, spread, size, 64, 300)
    live = (torch.arange(300, device="cuda") < cache.lens[:, None])[:, None, :].expand(Z, 1, 300)
    tol = (2 * score_error(size.max(), 64) + (2 * N + 4) * 2.0 ** -24) * cols + 1e-30
    assert (((cache.weight.double() - cols).abs() / tol)[live] <= 1).all()


def test_first_calls_of_a_process_inside_a_capture():
    """Devices, attributes and occupancies are asked for on a first call, which may be a captured one."""
    import subprocess
    import sys
    from pathlib import Path
    code = """
import torch
from qflash_b200 import KV4Cache
torch.manual_seed(1)
make = lambda h, n: torch.randn(2, h, n, 64, device="cuda").bfloat16()
cache, small = KV4Cache.empty(2, 2, 3000, 64), KV4Cache.empty(2, 2, 200, 64)
k, v, q, piece = make(2, 2500), make(2, 2500), make(4, 1), make(4, 900)
def step():
    cache.lens.zero_()
    cache.append(k, v)
    outs = [cache.attend(q), cache.attend(q, accumulate=True), cache.attend(piece, accumulate=True)]
    kept = cache.evict(100, 10, out=small)
    return [*outs, kept, *small.read(150), small.attend(q)]
side = torch.cuda.Stream()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=side):
    got = step()
graph.replay()
torch.cuda.synchronize()
got = [x.clone() for x in got]
cache.weight.fill_(7.0)
assert all(torch.equal(x, y) for x, y in zip(got, step()))
cache.check()
small.check()
print("same")
"""
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                         cwd=Path(__file__).resolve().parents[1])
    assert run.returncode == 0 and "same" in run.stdout, run.stderr[-2000:]
