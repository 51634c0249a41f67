"""The 4-bit key/value cache on the CPU: what its sources and host code have to hold to."""
import re
from pathlib import Path

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
