"""The 4-bit key/value cache on the CPU: what its sources and host code have to hold to."""
import re
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from qflash_b200 import KV4Cache, _lib
from test_kv4 import BAD_ST, ST, cache, refused

CSRC = Path(__file__).resolve().parents[1] / "qflash_b200" / "csrc"
SOURCES = {p.name: re.sub(r"//[^\n]*", "", p.read_text()) for p in sorted(CSRC.glob("kv4_*"))}


def body_of(source, name):
    """A kernel's body, by its braces."""
    at = source.index("{", re.search(rf"__global__[^{{;]*\b{name}\(", source).end())
    depth, end = 0, at
    while True:
        depth += {"{": 1, "}": -1}.get(source[end], 0)
        end += 1
        if not depth:
            return source[at:end]


def arguments(text, at):
    """The text between the parenthesis at `at` and its partner."""
    depth, end = 0, at
    while True:
        depth += {"(": 1, ")": -1}.get(text[end], 0)
        end += 1
        if not depth:
            return text[at:end]


def test_kernels_that_begin_early_read_what_is_being_written_by_plain_loads():
    """A kernel launched to begin under the one before it must not read that one's results through the read-only path:
    that is for memory which nothing writes while the reading kernel runs."""
    found = 0
    for source in SOURCES.values():
        for name in {n for call in re.findall(r"\blaunch_behind\(([^;]*);", source) for n in re.findall(r"\w+_kernel", call)}:
            body = body_of(source, name)
            assert "wait_for_previous()" in body, name
            found += 1
            for load in re.finditer(r"\b(?:__ldg|load8)(?=\()", body):
                what = arguments(body, load.end())
                assert not re.search(r"\b(?:parts?|stats|scores|kept)\b", what), f"{name}: {load.group()}{what}"
    assert found == 3


@pytest.mark.parametrize("Z, H, C, D, rep, N", [
    (32, 8, 131072, 128, 8, 6), (32, 8, 131072, 128, 8, 1), (1, 8, 1 << 24, 128, 4, 12), (1 << 14, 64, 2048, 64, 1, 16),
    (1, 1, 1 << 24, 64, 48, 1)])
def test_scores_kept_for_the_weights_are_bounded(Z, H, C, D, rep, N):
    """They are kept for some sequences and heads at a time: 1 GB, or one head's where that is more."""
    need = _lib.load().qflash_kv4_attend_workspace(cache(Z=Z, H=H, capacity=C, D=D), 1, H * rep, N, 1)
    rows = (rep * N + 3) // 4 * 4
    pieces, stats = 2 * 148 * 5 * 16 * (D + 2) * 4, 8 * Z * H * (rep * N + 15)
    assert 0 < need <= max(1 << 30, 4 * C * rows) + pieces + stats


def handle(**fields):
    """A KV4Cache with CPU tensors in its fields, past the constructor's refusal of them."""
    c = object.__new__(KV4Cache)
    for name, value in fields.items():
        setattr(c, name, value)
    return c


@pytest.mark.parametrize("status, error, words", [
    (1, OverflowError, ["dropped"]), (2, _lib.QFlashError, ["gave up"]), (3, _lib.QFlashError, ["gave up", "dropped"])])
def test_check_reports_all_that_happened(status, error, words):
    c = handle(shape=(1, 1, 16, 64), _ctl=torch.tensor([0, status], dtype=torch.int32))
    with pytest.raises(error) as e:
        c.check()
    assert all(w in str(e.value) for w in words)
    c.check()  # reported once


def test_attend_refuses_a_scale_beyond_fp32():
    """It is held in fp32, as a factor of log2(e): one that is finite in fp64 alone would make every output NaN."""
    lib = _lib.load()
    for scale in (1e39, -1e39, 3e38, 1.7e308):
        refused(lib.qflash_kv4_attend(cache(), 16, 1, ST, 16, ST, 2, 1, None, scale, 1, None, 256, 1 << 40, None), b"finite")
    refused(lib.qflash_kv4_attend(cache(), 16, 1, BAD_ST, 16, ST, 2, 1, None, 2e38, 1, None, 256, 1 << 40, None), b"stride")


def test_append_refuses_rows_that_the_library_cannot_count():
    """2^32 + 1 rows, as an expanded tensor has them without memory, must not be taken for one."""
    c = handle(shape=(1, 1, 16, 64), device=torch.device("cpu"), _ref=None, _index=0)
    x = torch.zeros(1, 1, 1, 64)
    for rows in ((1 << 32) + 1, 1 << 31):
        with pytest.raises(ValueError, match="rows"):
            c.append(x.expand(1, 1, rows, 64), x.expand(1, 1, rows, 64))


def test_package_imports_without_a_cuda_build_of_torch():
    code = """
import torch
for name in [n for n in dir(torch._C) if n.startswith("_cuda")]:
    delattr(torch._C, name)
import qflash_b200, qflash
assert qflash.qflash and qflash.KV4Cache
"""
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=CSRC.parents[1])
    assert run.returncode == 0, run.stderr[-2000:]


def names_of(source):
    """Functions, constants and structs that a source defines in its namespaces (indented lines are inside of something)."""
    for line in source.split("\n"):
        line = re.sub(r"^template <[^>]*>\s*", "", line)
        if line.startswith(("static ", "namespace ", "extern ", "using ")):
            continue
        if m := re.match(r"struct (\w+) \{", line):
            yield m.group(1)
        elif line.startswith("constexpr ") and "(" not in line.split("=")[0]:
            yield from re.findall(r"(\w+) =", line)
        elif m := re.match(r"(?:__global__ void (?:__\w+__\([^()]*\) )*|[^\s#}][^;()]*\b)(\w+)\((?!\()", line):
            yield m.group(1)


def test_no_name_is_defined_in_two_sources():
    """Two bodies of one inline function in a namespace make no valid program, whatever the build makes of them. (A
    declaration in the header and its one definition are none.)"""
    where = {}
    for file, source in SOURCES.items():
        for name in names_of(source):
            where.setdefault(name, set()).add(file)
    assert {"kTile", "kDigits", "Waiter", "to_float", "length_of", "append_kernel"} <= set(where)
    declared = set(re.findall(r"^(?:int|size_t) (\w+)\([^;{]*;", SOURCES["kv4_common.cuh"], re.M))
    twice = {n: sorted(files) for n, files in where.items() if len(files) > 1 and n not in declared}
    assert not twice, twice
