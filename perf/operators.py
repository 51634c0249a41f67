"""What is measured of the 4-bit key/value cache: its operators' plain forms and the framework's calls, over the same inputs.

A cache holds, for every sequence, key/value head and position, the key and the value in 4 bits: an affine code
0..15 per element, two to a byte (the even element in the low half), and per vector a scale (bfloat16) and a
zero point (a whole number 0..15, held beside it as bfloat16): x ~ scale * (code - zero).  The operators are

- append: quantise new tokens behind the stored ones (or at given positions),
- attend: softmax attention of the last tokens' queries over the cache, with grouped heads, a causal limit per row,
  and on request the attention weight that every stored position received, added up (what eviction goes by),
- evict: keep the last tokens and the heaviest of the others, packed in order into another cache,
- read: the values that stored codes stand for.
"""
import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one new token of 32 running sequences goes into the cache and is read back: latency
        dict(name="append-one", op="append", Z=32, H=8, D=128, cap=4096, length=4000, N=1, ragged=True, dtype="bf16"),
        # two prompts of unlike length, padded to one tensor
        dict(name="append-prompt", op="append", Z=2, H=8, D=128, cap=9000, length=8200, N=8191, ragged=True, dtype="fp16"),
        # one token of one short sequence: the smallest call of a decoding loop
        dict(name="decode-short", op="attend", Z=1, H=8, rep=4, D=64, cap=1024, length=333, N=1, ragged=False,
             causal=True, weights=False, dtype="fp16"),
        # a serving batch of unlike lengths, an idle slot among them
        dict(name="decode-batch", op="attend", Z=32, H=8, rep=4, D=128, cap=8192, length=8100, N=1, ragged=True,
             causal=True, weights=False, dtype="bf16"),
        # one very long sequence
        dict(name="decode-long", op="attend", Z=1, H=8, rep=8, D=128, cap=131072, length=131071, N=1, ragged=False,
             causal=True, weights=False, dtype="bf16"),
        # decoding with a bounded cache: the weights that eviction goes by are kept up
        dict(name="decode-weights", op="attend", Z=16, H=8, rep=4, D=128, cap=4352, length=4321, N=1, ragged=True,
             causal=True, weights=True, dtype="fp16"),
        # a few tokens at once, as when drafted tokens are checked; as many key/value heads as query heads
        dict(name="decode-few", op="attend", Z=8, H=12, rep=1, D=64, cap=6000, length=5999, N=5, ragged=True,
             causal=True, weights=False, dtype="bf16"),
        # a long prompt's next piece against everything before it
        dict(name="prompt-piece", op="attend", Z=1, H=8, rep=4, D=128, cap=8192, length=8000, N=2048, ragged=False,
             causal=True, weights=False, dtype="bf16"),
        # prompts of unlike length, padded, with the weights for the eviction after them
        dict(name="prompt-weights", op="attend", Z=4, H=6, rep=2, D=64, cap=2100, length=2085, N=2049, ragged=True,
             causal=True, weights=True, dtype="fp16"),
        # a decoding batch that reached its bound
        dict(name="evict-batch", op="evict", Z=16, H=8, D=128, cap=4352, length=4300, budget=2048, recent=256, ragged=True,
             dtype="bf16"),
        # a long prompt cut down to what decoding keeps
        dict(name="evict-long", op="evict", Z=1, H=8, D=128, cap=131072, length=131071, budget=8192, recent=1001,
             ragged=False, dtype="fp16"),
        # a cache handed on in 16 bits
        dict(name="read-all", op="read", Z=4, H=8, D=64, cap=8192, length=8191, N=8192, ragged=True, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)) - 0.5 / hi))) or lo)


def draw(rng):
    op = rng.choice(["append", "attend-one", "attend-one", "attend-few", "attend-prompt", "attend-prompt", "evict", "read"])
    D, dtype, ragged = rng.choice([64, 128]), rng.choice(["bf16", "fp16"]), rng.random() < 0.6
    Z, H = _log(rng, 1, 48), rng.choice([1, 2, 3, 4, 6, 8, 12, 16])
    if op in ("append", "read"):
        tokens = 2 ** 27 // (H * D * 2)
        N = _log(rng, 1, max(1, min(8191, tokens // Z)))
        length = N + _log(rng, 1, 4000)
        return dict(op=op, Z=Z, H=H, D=D, cap=length + rng.randrange(0, 300), length=length, N=N, ragged=ragged, dtype=dtype)
    if op == "evict":
        length = _log(rng, 64, min(131071, 2 ** 21 // (Z * H) + 64))
        budget = max(2, int(length * rng.uniform(0.05, 0.9)))
        return dict(op=op, Z=Z, H=H, D=D, cap=length + rng.randrange(0, 200), length=length, budget=budget,
                    recent=rng.randrange(0, budget + 1), ragged=ragged, dtype=dtype)
    rep = rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
    if op == "attend-prompt":
        N = _log(rng, 24, 2048)
        # score entries of all heads: at most those of the largest listed case
        length = N + _log(rng, 1, max(1, min(12000, 2 ** 28 // (Z * H * rep * N))))
        while Z * H * rep * N * length > 2 ** 28 and Z > 1:
            Z = Z // 2
        while H * rep * N * length > 2 ** 28 and H > 1:
            H = H // 2
    else:
        N = 1 if op == "attend-one" else rng.randrange(2, 17)
        length = N + _log(rng, 1, max(1, min(131000, 2 ** 21 // (Z * H))))
    return dict(op="attend", Z=Z, H=H, rep=rep, D=D, cap=length + rng.randrange(0, 300), length=length, N=N, ragged=ragged,
                causal=rng.random() < 0.85, weights=rng.random() < 0.4, dtype=dtype)


def _lens(case):
    """Stored tokens per sequence after the step, and how many of its N rows each sequence brings."""
    Z, L, N = case["Z"], case["length"], case.get("N", 1)
    if not case["ragged"]:
        return [L] * Z, [min(N, L)] * Z
    lens = [max(1, L - (z * 7919) % (L // 2 + 1)) for z in range(Z)]
    new = [min(n, N - (z * 31) % (N // 2 + 1)) for z, n in enumerate(lens)]
    if Z > 2:
        lens[1] = new[1]  # a sequence that begins with this step
        lens[2] = new[2] = 0  # an idle slot
    return lens, new


def _quantised(x):
    """Codes, scales and zero points of vectors x [..., D]: the range from min(x, 0) to max(x, 0) in 15 steps."""
    lo, hi = x.amin(-1).clamp(max=0).double(), x.amax(-1).clamp(min=0).double()
    scale = ((hi - lo) / 15).float().bfloat16()
    s = scale.float().unsqueeze(-1)
    zero = torch.where(s > 0, torch.round(-lo.float().unsqueeze(-1) / s).clamp(0, 15), 0)
    code = torch.where(s > 0, (torch.round(x.float() / s) + zero).clamp(0, 15), 0).to(torch.uint8)
    return code, torch.stack((scale, zero.squeeze(-1).bfloat16()), -1)


def _packed(code):
    return code[..., 0::2] | (code[..., 1::2] << 4)


def _values(codes, param):
    """float32 values of packed codes [..., D / 2]."""
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float()
    return param[..., :1].float() * (code - param[..., 1:].float())


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    Z, H, D, C, dt = c["Z"], c["H"], c["D"], c["cap"], DT[c["dtype"]]
    lens, new = _lens(c)
    N = c.get("N", 1)
    channel = 1 + 3 * (torch.rand(H, 1, D, generator=g, device="cuda") > 0.95)  # a few strong channels, as keys have
    st = {"case": c, "lens": torch.tensor(lens, dtype=torch.int32, device="cuda")}
    if c["op"] == "append":
        rows = torch.tensor(new, dtype=torch.int32, device="cuda")
        st["new"], st["at"] = rows, st["lens"] - rows
        st["key"] = (_normal(g, Z, N, H, D).transpose(1, 2) * channel).to(dt)
        st["value"] = _normal(g, Z, N, H, D).to(dt).transpose(1, 2)  # a projection's [Z, N, H, D] output, seen by heads
        st["cache"] = [torch.zeros(Z, H, C, D // 2, dtype=torch.uint8, device="cuda") for _ in "kv"] + [
            torch.zeros(Z, H, C, 2, dtype=torch.bfloat16, device="cuda") for _ in "kv"] + [
            torch.zeros(Z, H, C, device="cuda"), st["lens"].clone()]
        return st
    st["cache"] = []
    for scale in (channel, 1.0):
        code, param = _quantised((_normal(g, Z, H, C, D) * scale).to(dt))
        st["cache"] += [_packed(code), param]
    k, kp, v, vp = st["cache"]
    # weights as attention leaves them: a few heavy positions, most of them light; none behind the stored tokens
    live = torch.arange(C, device="cuda") < st["lens"].view(Z, 1, 1)
    weight = torch.exp(2 * _normal(g, Z, H, C)) * live
    st["cache"] = [k, v, kp, vp, weight, st["lens"]]
    if c["op"] == "attend":
        st["new"] = torch.tensor(new, dtype=torch.int32, device="cuda")
        st["query"] = _normal(g, Z, N, H * c["rep"], D).to(dt).transpose(1, 2)
        st["weights"] = weight.clone()
    if c["op"] == "evict":
        room = c["budget"] + 64
        st["kept"] = [torch.zeros(Z, H, room, D // 2, dtype=torch.uint8, device="cuda") for _ in "kv"] + [
            torch.zeros(Z, H, room, 2, dtype=torch.bfloat16, device="cuda") for _ in "kv"] + [
            torch.zeros(Z, H, room, device="cuda"), torch.zeros(Z, dtype=torch.int32, device="cuda")]
    return st


def run(st):
    c = st["case"]
    if own:
        return _run_own(st, c)
    return {"append": _plain_append, "attend": _plain_attend, "evict": _plain_evict, "read": _plain_read}[c["op"]](st, c)


def _run_own(st, c):
    from qflash_b200 import KV4Cache

    cache = st.get("handle")
    if cache is None:  # a program makes the handle of its buffers once
        cache = st["handle"] = KV4Cache(*st["cache"])
    if c["op"] == "append":
        cache.append(st["key"], st["value"], new_lens=st["new"], at=st["at"])
        return (*cache.read(c["N"], start=st["at"], dtype=DT[c["dtype"]]), cache.weight, cache.lens)
    if c["op"] == "attend":
        out = cache.attend(st["query"], causal=c["causal"], new_lens=st["new"], accumulate=c["weights"],
                           weights=st["weights"] if c["weights"] else None)
        return (out, cache.weight) if c["weights"] else (out,)
    if c["op"] == "evict":
        to = st.get("to")
        if to is None:
            to = st["to"] = KV4Cache(*st["kept"])
        kept = cache.evict(c["budget"], c["recent"], out=to)
        return (*to.read(c["budget"], dtype=DT[c["dtype"]]), to.weight, to.lens, kept)
    return cache.read(c["N"], dtype=DT[c["dtype"]])


def _plain_append(st, c):
    k, v, kp, vp, weight, lens = st["cache"]
    Z, H, N, D = st["key"].shape
    z, h, n = (torch.arange(m, device="cuda").view(s) for m, s in ((Z, (-1, 1, 1)), (H, (1, -1, 1)), (N, (1, 1, -1))))
    keep = (n < st["new"].view(Z, 1, 1)).expand(Z, H, N)
    at = st["at"].view(Z, 1, 1) + n
    index = [i.expand(Z, H, N)[keep] for i in (z, h, at)]
    out = []
    for x, codes, param in ((st["key"], k, kp), (st["value"], v, vp)):
        code, p = _quantised(x)
        codes[index[0], index[1], index[2]] = _packed(code)[keep]
        param[index[0], index[1], index[2]] = p[keep]
        out.append((p[..., :1].float() * (code.float() - p[..., 1:].float()) * keep.unsqueeze(-1)).to(x.dtype))
    weight[index[0], index[1], index[2]] = 0
    lens.copy_(st["at"] + st["new"])
    return out[0], out[1], weight, lens


def _plain_attend(st, c):
    k, v, kp, vp, weight, lens = st["cache"]
    Z, Hq, N, D = st["query"].shape
    H, C = k.shape[1], k.shape[2]
    q = st["query"].float().reshape(Z, H, Hq // H * N, D)
    s = torch.matmul(q, _values(k, kp).transpose(-1, -2)).view(Z, H, -1, N, C).mul_(1 / math.sqrt(D))
    row = torch.arange(N, device="cuda").view(1, N, 1)
    new, length = st["new"].view(Z, 1, 1), lens.view(Z, 1, 1)
    limit = length - new + row + 1 if c["causal"] else length.expand(Z, N, 1)
    limit = torch.where(row < new, limit, 0)
    live = (torch.arange(C, device="cuda") < limit).view(Z, 1, 1, N, C)
    s = torch.where(live, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s.sub_(torch.where(top > -math.inf, top, 0.0)))
    total = p.sum(-1, keepdim=True)
    p = p.mul_(torch.where(total > 0, 1 / total, 0.0))
    # a stored position that no row sees has weight 0 whatever its buffer holds
    value = torch.where((torch.arange(C, device="cuda") < lens.view(Z, 1)).view(Z, 1, C, 1), _values(v, vp), 0.0)
    out = torch.matmul(p.view(Z, H, -1, C), value).view(Z, Hq, N, D).to(st["query"].dtype)
    if not c["weights"]:
        return (out,)
    weight.copy_(st["weights"] + p.double().sum((2, 3)).float() if N > 64 else st["weights"] + p.sum((2, 3)))
    return out, weight


def _plain_evict(st, c):
    k, v, kp, vp, weight, lens = st["cache"]
    Z, H, C = weight.shape
    position, length = torch.arange(C, device="cuda"), lens.view(Z, 1, 1)
    rank = torch.where(position >= length - c["recent"], math.inf, weight)
    rank = torch.where(position < length, rank, -math.inf)
    first = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., : c["budget"]]
    first = torch.sort(torch.where(first < length, first, C), dim=-1).values
    there = first < C
    at = torch.where(there, first, 0)
    tk, tv, tkp, tvp, tw, tl = st["kept"]
    n, out = first.shape[-1], []
    for codes, param, to, to_param in ((k, kp, tk, tkp), (v, vp, tv, tvp)):
        code = torch.gather(codes, 2, at.unsqueeze(-1).expand(-1, -1, -1, codes.shape[-1]))
        par = torch.gather(param, 2, at.unsqueeze(-1).expand(-1, -1, -1, 2))
        to[:, :, :n], to_param[:, :, :n] = code, par
        out.append((_values(code, par) * there.unsqueeze(-1)).to(DT[c["dtype"]]))
    tw[:, :, :n] = torch.where(there, torch.gather(weight, 2, at), tw[:, :, :n])
    tl.copy_(lens.clamp(max=c["budget"]))
    return out[0], out[1], tw, tl, torch.where(there, first, -1).int()


def _plain_read(st, c):
    k, v, kp, vp, _, lens = st["cache"]
    live = (torch.arange(c["N"], device="cuda") < lens.view(-1, 1)).view(c["Z"], 1, -1, 1)
    return tuple(torch.where(live, _values(x[:, :, : c["N"]], p[:, :, : c["N"]]), 0.0).to(DT[c["dtype"]]) for x, p in ((k, kp), (v, vp)))


def work(case):
    lens, new = _lens(case)
    Z, H, D, N, e = case["Z"], case["H"], case["D"], case.get("N", 1), DT[case["dtype"]].itemsize
    stored = D + 8  # bytes of a key and a value: D / 2 of codes and 4 of scale and zero point, each
    if case["op"] == "append":
        t = sum(new)
        return {"bytes": H * (t * (2 * D * e + 2 * stored + 4) + Z * N * 2 * D * e), "flops": H * t * D * 8}
    if case["op"] == "read":
        return {"bytes": H * (sum(lens) * stored + Z * N * 2 * D * e), "flops": H * sum(lens) * D * 4}
    if case["op"] == "evict":
        kept = sum(min(n, case["budget"]) for n in lens)
        # the weights of all, what is kept copied and read back, the list of what was kept
        return {"bytes": H * (sum(lens) * 4 + kept * (3 * stored + 4) + Z * case["budget"] * (4 + 2 * D * e)), "flops": H * kept * D * 4}
    pairs = sum(sum(max(0, n - m + i + 1) for i in range(m)) if case["causal"] else n * m for n, m in zip(lens, new))
    seen = sum(lens) * (stored + (8 if case["weights"] else 0))
    return {"bytes": H * (seen + 2 * Z * N * case["rep"] * D * e), "flops": 4 * D * H * case["rep"] * pairs}


def exact(case, seed):
    c, st = case, prepare(case, seed)
    k, v, kp, vp, weight, lens = st["cache"]
    n = lens.tolist()

    def decoded(code, par):
        w = code.to(torch.int64)
        full = torch.empty(*w.shape[:-1], 2 * w.shape[-1], dtype=torch.float64, device=w.device)
        full[..., ::2], full[..., 1::2] = (w % 16).double(), (w // 16).double()
        return (full - par[..., 1].double()[..., None]) * par[..., 0].double()[..., None]

    if c["op"] == "append":
        new, out = st["new"].tolist(), []
        for x in (st["key"].double(), st["value"].double()):
            low, high = torch.minimum(x.min(-1).values, x.new_zeros(())), torch.maximum(x.max(-1).values, x.new_zeros(()))
            # the scale is held in bfloat16, reached over float32; a vector of zeros has scale 0 and stands for zeros
            s = ((high - low) / 15).to(torch.float32).to(torch.bfloat16).double().unsqueeze(-1)
            safe = torch.where(s > 0, s, 1.0)
            z = torch.clamp(torch.round(-low.unsqueeze(-1) / safe), 0, 15)
            y = s * (torch.clamp(torch.round(x / safe) + z, 0, 15) - z)
            for i, m in enumerate(new):
                y[i, :, m:] = 0
            out.append(y)
        return out[0], out[1], torch.zeros_like(weight, dtype=torch.float64), None
    if c["op"] == "read":
        out = []
        for codes, par in ((k, kp), (v, vp)):
            y = torch.zeros(c["Z"], c["H"], c["N"], c["D"], dtype=torch.float64, device="cuda")
            for z in range(c["Z"]):
                y[z, :, : n[z]] = decoded(codes[z, :, : n[z]], par[z, :, : n[z]])
            out.append(y)
        return tuple(out)
    if c["op"] == "evict":
        keys = torch.zeros(c["Z"], c["H"], c["budget"], c["D"], dtype=torch.float64, device="cuda")
        values, left = torch.zeros_like(keys), torch.zeros(c["Z"], c["H"], c["budget"] + 64, dtype=torch.float64, device="cuda")
        for z in range(c["Z"]):
            for h in range(c["H"]):
                if n[z] <= c["budget"]:
                    keep = torch.arange(n[z], device="cuda")
                else:
                    old = n[z] - c["recent"]
                    heavy = torch.argsort(-weight[z, h, :old].double(), stable=True)[: c["budget"] - c["recent"]]
                    keep = torch.cat((heavy.sort().values, torch.arange(old, n[z], device="cuda")))
                m = keep.numel()
                keys[z, h, :m], values[z, h, :m] = decoded(k[z, h, keep], kp[z, h, keep]), decoded(v[z, h, keep], vp[z, h, keep])
                left[z, h, :m] = weight[z, h, keep].double()
        return keys, values, left, None, None
    new, rep, N = st["new"].tolist(), c["rep"], c["N"]
    out = torch.zeros(st["query"].shape, dtype=torch.float64, device="cuda")
    total = st["weights"].double()
    for z in range(c["Z"]):
        for h in range(c["H"]):
            if new[z] == 0 or n[z] == 0:
                continue
            K, V = decoded(k[z, h, : n[z]], kp[z, h, : n[z]]), decoded(v[z, h, : n[z]], vp[z, h, : n[z]])
            for a in range(h * rep, (h + 1) * rep):
                s = st["query"][z, a, : new[z]].double() @ K.T / math.sqrt(c["D"])
                if c["causal"]:
                    s = s + torch.full_like(s, -math.inf).triu(n[z] - new[z] + 1)
                p = torch.softmax(s, -1)
                out[z, a, : new[z]] = p @ V
                total[z, h, : n[z]] += p.sum(0)
    return (out, total) if c["weights"] else (out,)
