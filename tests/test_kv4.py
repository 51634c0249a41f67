"""The 4-bit key/value cache on the CPU: refusals of the C entry points and of KV4Cache, before any CUDA call."""
import ctypes

import pytest
import torch

from qflash_b200 import KV4Cache, _lib


def cache(**over):
    f = dict(k_codes=256, v_codes=512, k_param=768, v_param=1024, weight=1280, lens=1536, ctl=1792, Z=1, H=2,
             capacity=16, D=64)
    return _lib.KV4CacheStruct(**{**f, **over})


ST = (ctypes.c_int64 * 4)(0, 0, 0, 1)
BAD_ST = (ctypes.c_int64 * 4)(0, 0, 0, 2)


def refused(rc, text, code=-1):
    assert rc == code and text in _lib.load().qflash_last_error(), (rc, _lib.load().qflash_last_error())


@pytest.mark.parametrize("over, text, code", [
    (dict(D=96), b"head dim", -1), (dict(D=0), b"head dim", -1), (dict(capacity=0), b"shape", -1),
    (dict(H=0), b"shape", -1), (dict(Z=-1), b"shape", -1), (dict(capacity=(1 << 24) + 1), b"capacity", -1),
    (dict(Z=1 << 16, H=32), b"heads", -1), (dict(lens=None), b"null", -1), (dict(k_codes=264), b"16-byte", -2),
    (dict(weight=1282), b"4-byte", -2)])
def test_every_call_refuses_a_bad_cache(over, text, code):
    lib, c, good = _lib.load(), cache(**over), cache()
    refused(lib.qflash_kv4_append(c, 16, 16, 1, ST, ST, 1, None, None, None), text, code)
    refused(lib.qflash_kv4_read(c, 16, 16, 1, 1, None, None), text, code)
    refused(lib.qflash_kv4_attend(c, 16, 1, ST, 16, ST, max(c.H, 1), 1, None, 1.0, 1, None, 16, 1 << 40, None), text, code)
    refused(lib.qflash_kv4_evict(c, good, 1, 0, 16, None), text, code)
    refused(lib.qflash_kv4_evict(good, c, 1, 0, 16, None), text, code)
    assert lib.qflash_kv4_attend_workspace(c, 1, max(c.H, 1), 1, 0) == 0


def test_null_cache():
    refused(_lib.load().qflash_kv4_read(None, 16, 16, 1, 1, None, None), b"null")


def test_append_and_read_refusals():
    lib, c = _lib.load(), cache()
    refused(lib.qflash_kv4_append(c, 16, 16, 3, ST, ST, 1, None, None, None), b"dtype")
    refused(lib.qflash_kv4_append(c, 16, 16, 1, ST, ST, -1, None, None, None), b"negative")
    refused(lib.qflash_kv4_append(c, 16, 16, 1, ST, BAD_ST, 1, None, None, None), b"stride")
    refused(lib.qflash_kv4_append(c, None, 16, 1, ST, ST, 1, None, None, None), b"null")
    refused(lib.qflash_kv4_append(cache(Z=1 << 10, H=1 << 10), 16, 16, 1, ST, ST, 1024, None, None, None), b"2^31", -6)
    assert lib.qflash_kv4_append(c, None, None, 1, ST, ST, 0, None, None, None) == 0  # nothing to do
    refused(lib.qflash_kv4_read(c, 16, 16, 5, 1, None, None), b"dtype")
    refused(lib.qflash_kv4_read(c, 16, 24, 1, 1, None, None), b"16-byte", -2)
    refused(lib.qflash_kv4_read(c, 16, None, 1, 1, None, None), b"null")
    refused(lib.qflash_kv4_read(c, 16, 16, 1, -1, None, None), b"negative")


def test_attend_refusals():
    lib, c = _lib.load(), cache()

    def attend(q=16, dtype=1, qs=ST, out=16, os=ST, Hq=2, N=1, scale=1.0, ws=256, n=1 << 40, c=c):
        return lib.qflash_kv4_attend(c, q, dtype, qs, out, os, Hq, N, None, scale, 1, None, ws, n, None)

    refused(attend(dtype=0), b"fp16 or bf16")
    refused(attend(Hq=3), b"heads")
    refused(attend(Hq=0), b"heads")
    refused(attend(Hq=130), b"above 64", -6)
    refused(attend(N=-1), b"negative")
    refused(attend(N=1 << 24), b"rows", -6)
    refused(attend(scale=float("nan")), b"finite")
    refused(attend(qs=BAD_ST), b"stride")
    refused(attend(os=BAD_ST), b"stride")
    refused(attend(q=None), b"null")
    refused(attend(ws=None), b"workspace")
    refused(attend(n=16), b"workspace")
    refused(attend(ws=264), b"16-byte", -2)
    assert attend(q=None, N=0) == 0
    assert attend(q=None, c=cache(Z=0)) == 0


def test_evict_refusals():
    lib, c = _lib.load(), cache()
    big = 1 << 20
    other = cache(k_codes=big, v_codes=2 * big, k_param=3 * big, v_param=4 * big, weight=5 * big, lens=6 * big)
    refused(lib.qflash_kv4_evict(c, other, 0, 0, 16, None), b"budget")
    refused(lib.qflash_kv4_evict(c, other, 17, 0, 16, None), b"budget")
    refused(lib.qflash_kv4_evict(c, other, 4, 5, 16, None), b"recent")
    refused(lib.qflash_kv4_evict(c, other, 4, -1, 16, None), b"recent")
    refused(lib.qflash_kv4_evict(c, other, 4, 1, None, None), b"null")
    refused(lib.qflash_kv4_evict(c, c, 4, 1, 16, None), b"share memory")
    shared = cache(k_codes=big, v_codes=2 * big, k_param=3 * big, v_param=4 * big, weight=5 * big)
    refused(lib.qflash_kv4_evict(c, shared, 4, 1, 16, None), b"share memory")
    other.H = 1
    refused(lib.qflash_kv4_evict(c, other, 4, 1, 16, None), b"heads")


def test_workspace_grows_with_the_weights():
    lib, c = _lib.load(), cache(Z=2, capacity=1000)
    plain = lib.qflash_kv4_attend_workspace(c, 1, 8, 3, 0)
    assert 0 < plain < lib.qflash_kv4_attend_workspace(c, 1, 8, 3, 1)


def buffers(Z=1, H=2, C=16, D=64):
    return [torch.zeros(Z, H, C, D // 2, dtype=torch.uint8), torch.zeros(Z, H, C, D // 2, dtype=torch.uint8),
            torch.zeros(Z, H, C, 2, dtype=torch.bfloat16), torch.zeros(Z, H, C, 2, dtype=torch.bfloat16),
            torch.zeros(Z, H, C), torch.zeros(Z, dtype=torch.int32)]


def test_handle_refuses_bad_buffers():
    with pytest.raises(ValueError, match="CUDA"):  # no CPU path
        KV4Cache(*buffers())
    with pytest.raises(ValueError, match="head dim"):
        KV4Cache(*buffers(D=32))
    with pytest.raises(ValueError, match="head dim"):
        KV4Cache.empty(1, 1, 16, 48)
    for i, bad in ((1, torch.zeros(1, 2, 15, 32, dtype=torch.uint8)), (2, torch.zeros(1, 2, 16, 2)),
                   (4, torch.zeros(1, 16, 2).transpose(1, 2)), (5, torch.zeros(1, dtype=torch.int64))):
        b = buffers()
        b[i] = bad
        with pytest.raises(ValueError, match="contiguous"):
            KV4Cache(*b)
    with pytest.raises(ValueError, match="k_codes"):
        KV4Cache(torch.zeros(2, 16, 32, dtype=torch.uint8), *buffers()[1:])


def test_handle_refuses_sizes_and_shared_buffers():
    for shape in ((1, 0, 16), (1, 1, 0)):
        with pytest.raises(ValueError, match="at least one"):
            KV4Cache(torch.zeros(*shape, 32, dtype=torch.uint8), *buffers()[1:])
    with pytest.raises(ValueError, match="at least one"):
        KV4Cache(torch.zeros(1, dtype=torch.uint8).expand(1, 1, (1 << 24) + 1, 32), *buffers()[1:])
    with pytest.raises(AttributeError):  # the calls go by the buffers' addresses
        KV4Cache.weight.__set__(object.__new__(KV4Cache), None)


def test_caches_on_two_devices_and_overlapping_weights():
    lib, c = _lib.load(), cache()
    big = 1 << 20
    other = cache(k_codes=big, v_codes=2 * big, k_param=3 * big, v_param=4 * big, weight=5 * big, lens=6 * big, device=1)
    refused(lib.qflash_kv4_evict(c, other, 4, 1, 16, None), b"devices")
    refused(lib.qflash_kv4_attend(c, 16, 1, ST, 16, ST, 2, 1, None, 1.0, 1, c.weight + 4, 256, 1 << 40, None), b"overlaps")
