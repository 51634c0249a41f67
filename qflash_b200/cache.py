"""A key/value cache in 4 bits and attention over it (serving; no counterpart in
the reference, whose ``qflash.forward`` attends over floats in one call).

    cache = KV4Cache.empty(batch, kv_heads, capacity, head_dim)
    cache.append(k, v)                      # [Z, H, N, D]: a prompt, then single tokens
    out = cache.attend(q)                   # [Z, Hq, N, D]: the queries of the last N tokens
    cache.attend(q, accumulate=True)        # and adds up the weight that every position receives
    kept = cache.evict(budget, recent, out=smaller)   # packs the heaviest and the last tokens
    k, v = cache.read(count)                # the stored values, e.g. for ``qflash.forward``

Every vector is held as codes 0..15, a bfloat16 scale and a zero point
(``scale * (code - zero)``); include/qflash_b200.h states the layout and the
rounding.  Sequences of a batch have lengths of their own (``lens``, on the
device); no call but ``check`` synchronises with the host, and all others can be
captured into CUDA graphs.  Calls that write a cache (``append``, ``attend`` with
``accumulate``, ``evict`` into it) must be ordered with all others on it, by one
stream or by events; others may run side by side.  Gradients are not computed.
"""
from __future__ import annotations

import ctypes

import torch
from torch import Tensor

from . import _lib

HEAD_DIMS = (64, 128)
MAX_CAPACITY, MAX_HEADS = 1 << 24, 1 << 20


class KV4Cache:
    """Handle of a cache's buffers, which it neither copies nor lays out anew:
    ``k_codes``, ``v_codes`` uint8 [Z, H, C, D / 2], ``k_param``, ``v_param``
    bfloat16 [Z, H, C, 2] (scale, zero point), ``weight`` float32 [Z, H, C] and
    ``lens`` int32 [Z], all contiguous CUDA tensors on one device."""

    __slots__ = ("_buffers", "_ctl", "_c", "_ref", "_index", "_workspace", "_scale", "shape", "device")
    # the calls go by the buffers' addresses, so the tensors can be written but not replaced
    k_codes, v_codes, k_param, v_param, weight, lens = (property(lambda self, i=i: self._buffers[i]) for i in range(6))

    def __init__(self, k_codes: Tensor, v_codes: Tensor, k_param: Tensor, v_param: Tensor, weight: Tensor,
                 lens: Tensor):
        if k_codes.dim() != 4:
            raise ValueError(f"k_codes must be [Z, H, C, D / 2], got {tuple(k_codes.shape)}")
        Z, H, C, half = k_codes.shape
        if not (H >= 1 and 1 <= C <= MAX_CAPACITY and Z * H <= MAX_HEADS):
            raise ValueError(f"at least one head and position, at most {MAX_CAPACITY} positions and {MAX_HEADS} heads "
                             f"in all: got Z, H, C = {Z}, {H}, {C}")
        if 2 * half not in HEAD_DIMS:
            raise ValueError(f"head dim {2 * half} not in {HEAD_DIMS}")
        buffers = (("k_codes", k_codes, (Z, H, C, half), torch.uint8), ("v_codes", v_codes, (Z, H, C, half), torch.uint8),
                   ("k_param", k_param, (Z, H, C, 2), torch.bfloat16), ("v_param", v_param, (Z, H, C, 2), torch.bfloat16),
                   ("weight", weight, (Z, H, C), torch.float32), ("lens", lens, (Z,), torch.int32))
        for name, t, shape, dtype in buffers:
            if tuple(t.shape) != shape or t.dtype != dtype or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {shape}, got {t.dtype} "
                                 f"{tuple(t.shape)} with strides {t.stride()}")
        for name, t, _, _ in buffers:
            if not t.is_cuda or t.device != k_codes.device:
                raise ValueError(f"{name} must be on the CUDA device of k_codes, got {t.device}")
        self._buffers = (k_codes, v_codes, k_param, v_param, weight, lens)
        if Z and len({t.data_ptr() for t in self._buffers}) < 6:
            raise ValueError("the buffers must be six different ones")
        self._ctl = torch.zeros(2, dtype=torch.int32, device=k_codes.device)
        self.shape, self.device = (Z, H, C, 2 * half), k_codes.device
        self._c = _lib.KV4CacheStruct(*(t.data_ptr() for t in (k_codes, v_codes, k_param, v_param, weight, lens,
                                                               self._ctl)), Z, H, C, 2 * half, self.device.index)
        self._ref = ctypes.byref(self._c)
        self._index, self._workspace, self._scale = self.device.index, {}, 1.0 / (2 * half) ** 0.5

    @classmethod
    def empty(cls, batch: int, kv_heads: int, capacity: int, head_dim: int, device="cuda") -> "KV4Cache":
        """A cache that holds no tokens."""
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head dim {head_dim} not in {HEAD_DIMS}")
        shape = (batch, kv_heads, capacity)
        codes = [torch.zeros(*shape, head_dim // 2, dtype=torch.uint8, device=device) for _ in range(2)]
        param = [torch.zeros(*shape, 2, dtype=torch.bfloat16, device=device) for _ in range(2)]
        return cls(*codes, *param, torch.zeros(shape, dtype=torch.float32, device=device),
                   torch.zeros(batch, dtype=torch.int32, device=device))

    def append(self, key: Tensor, value: Tensor, new_lens: Tensor | None = None, at: Tensor | None = None) -> None:
        """Quantise ``key`` and ``value`` [Z, H, N, D] (float32, float16 or
        bfloat16, any strides over a contiguous head dim) behind the stored
        tokens.  ``new_lens`` int32 [Z]: how many of the N rows each sequence
        brings (default all).  ``at`` int32 [Z]: where its first one goes
        (default ``lens``); ``lens`` becomes ``at + new_lens``, so an ``at``
        below ``lens`` takes tokens back (with N = 0 nothing else).  Tokens
        past the capacity are dropped, which ``check`` reports."""
        Z, H, _, D = self.shape
        if key.dim() != 4 or key.shape != value.shape or key.shape[:2] != (Z, H) or key.shape[3] != D:
            raise ValueError(f"key and value must be [{Z}, {H}, N, {D}], got {tuple(key.shape)}, {tuple(value.shape)}")
        if key.shape[2] >= 1 << 31:
            raise ValueError(f"{key.shape[2]} rows, 2^31 or more")
        if key.dtype not in _FLOATS or value.dtype != key.dtype:
            raise ValueError(f"key and value must be float32, float16 or bfloat16 of one dtype, got {key.dtype}, "
                             f"{value.dtype}")
        self._here("key", key)
        self._here("value", value)
        _lib.kv4_append(self._ref, _inner(key), _inner(value), self._counts("new_lens", new_lens),
                        self._counts("at", at), _stream(self._index))

    def attend(self, query: Tensor, scale: float | None = None, causal: bool = True, new_lens: Tensor | None = None,
               accumulate: bool = False, weights: Tensor | None = None, out: Tensor | None = None) -> Tensor:
        """Attention of ``query`` [Z, Hq, N, D] (float16 or bfloat16) over the
        stored tokens; Hq is a multiple of the cache's H, and head h reads
        key/value head h // (Hq // H).  Rows i < ``new_lens`` (default N) are
        each sequence's last tokens; with ``causal`` row i sees the tokens up
        to its own, else every one.  Rows that see nothing and padded rows are
        zeros.  ``scale`` defaults to 1 / sqrt(D).

        ``accumulate`` sets ``weight`` of every stored position to
        ``weights`` (float32 [Z, H, C], default ``weight`` itself) plus the
        probabilities that the position received, over rows and the heads of
        its group.  ``out``: the output tensor (any strides over a contiguous
        head dim, each element once, none of them the query's)."""
        Z, H, C, D = self.shape
        if query.dim() != 4 or query.shape[0] != Z or query.shape[3] != D or query.shape[1] % H or not query.shape[1]:
            raise ValueError(f"query must be [{Z}, a multiple of {H}, N, {D}], got {tuple(query.shape)}")
        if query.dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"query must be float16 or bfloat16, got {query.dtype}")
        self._here("query", query)
        if weights is None:
            weights = self.weight
        elif not accumulate:
            raise ValueError("weights without accumulate")
        elif tuple(weights.shape) != (Z, H, C) or weights.dtype != torch.float32 or not weights.is_contiguous() \
                or weights.device != self.device:
            raise ValueError(f"weights must be a contiguous float32 [{Z}, {H}, {C}] tensor on {self.device}")
        query = _inner(query)
        if out is None:
            out = torch.empty(query.shape, dtype=query.dtype, device=self.device)
        elif out.shape != query.shape or out.dtype != query.dtype or out.stride(-1) != 1 or out.device != self.device:
            raise ValueError(f"out must be a {tuple(query.shape)} {query.dtype} tensor on {self.device} with a "
                             "contiguous last dim")
        elif out.data_ptr() == query.data_ptr() and out.numel() or any(n > 1 and not s for n, s in zip(out.shape, out.stride())):
            raise ValueError("out must have elements of its own")
        shape = (query.dtype, query.shape[1], query.shape[2], accumulate)
        need = self._workspace.get(shape)
        if need is None:
            if len(self._workspace) > 4096:
                self._workspace.clear()
            need = self._workspace[shape] = _lib.kv4_attend_workspace(self._ref, *shape)
        # of this call alone: two calls on one cache may run side by side, on streams or in graphs
        ws = torch.empty(need, dtype=torch.uint8, device=self.device)
        _lib.kv4_attend(self._ref, query, out, self._counts("new_lens", new_lens),
                        self._scale if scale is None else scale, causal, weights if accumulate else None, ws, need,
                        _stream(self._index))
        return out

    def evict(self, budget: int, recent: int, out: "KV4Cache") -> Tensor:
        """Pack what stays into the cache ``out`` (same Z, H and D; it shares no
        memory with this one): of sequences longer than ``budget`` the last
        ``recent`` tokens and, per head, the heaviest others by ``weight`` (of
        equal ones the first), in order and with their weights; shorter
        sequences whole.  Returns the kept positions, int32 [Z, H, budget], -1
        behind the last."""
        Z, H, _, D = self.shape
        if out.shape[:2] != (Z, H) or out.shape[3] != D or out.device != self.device:
            raise ValueError(f"out must be a cache of {Z} x {H} heads of {D} on {self.device}, got {out.shape} on "
                             f"{out.device}")
        if not 1 <= budget <= out.shape[2]:
            raise ValueError(f"budget {budget} not in [1, {out.shape[2]}]")
        if not 0 <= recent <= budget:
            raise ValueError(f"recent {recent} not in [0, {budget}]")
        kept = torch.empty((Z, H, budget), dtype=torch.int32, device=self.device)
        _lib.kv4_evict(self._ref, out._ref, budget, recent, kept, _stream(self._index))
        return kept

    def read(self, count: int | None = None, start: Tensor | None = None,
             dtype: torch.dtype = torch.bfloat16) -> tuple[Tensor, Tensor]:
        """Keys and values of ``count`` positions (default: the capacity) from
        ``start`` int32 [Z] (default 0) on, as [Z, H, count, D] tensors of
        ``dtype``; zeros where nothing is stored."""
        Z, H, C, D = self.shape
        count = C if count is None else count
        if count < 0:
            raise ValueError(f"count {count} is negative")
        if dtype not in _FLOATS:
            raise ValueError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
        k, v = (torch.empty((Z, H, count, D), dtype=dtype, device=self.device) for _ in range(2))
        _lib.kv4_read(self._ref, k, v, count, self._counts("start", start),
                      _stream(self._index))
        return k, v

    def check(self) -> None:
        """Raise OverflowError if an append since the last check dropped tokens
        outside [0, capacity), QFlashError if a wait inside a kernel gave up
        (its output is then not valid; where both happened it says so).
        Synchronises."""
        status = int(self._ctl[1].item())
        if status:
            self._ctl[1] = 0
        dropped = f"tokens outside the cache's {self.shape[2]} positions were dropped"
        if status & 2:
            raise _lib.QFlashError("a bounded wait inside an attention kernel gave up" + (f"; {dropped}" if status & 1 else ""))
        if status & 1:
            raise OverflowError(dropped)

    def _counts(self, name, t):
        if t is not None and (t.shape != self.shape[:1] or t.dtype != torch.int32 or t.device != self.device
                              or not t.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous int32 [{self.shape[0]}] tensor on {self.device}, got "
                             f"{t.dtype} {tuple(t.shape)} on {t.device}")
        return t

    def _here(self, name, t):
        if t.device != self.device:
            raise ValueError(f"{name} is on {t.device}, the cache on {self.device}")


_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


def _stream(index: int) -> int:
    # torch.cuda.current_stream(device).cuda_stream without the object; looked up here, as builds of torch without CUDA lack it
    return torch._C._cuda_getCurrentRawStream(index)


def _inner(t: Tensor) -> Tensor:
    return t if t.stride(-1) == 1 else t.contiguous()
