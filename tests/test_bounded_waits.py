"""Kernels whose waits are bounded leave their loops when one has run out.  A barrier of the hardware inside such a loop would then keep the
threads that are still in it for good, so there is none: what warps hand one another inside a loop goes over mbarriers."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "npa_b200" / "csrc"
BARRIER = re.compile(r"__syncthreads|bar\.sync|barrier\.sync|barrier\.cta|\w+_barrier\s*\(\s*\)")
WAIT = re.compile(r"umma_wait(_slow)?\s*\(")


def _without_comments(text):
    text = re.sub(r"//[^\n]*", "", text)
    return re.sub(r"/\*.*?\*/", "", text, flags=re.S)


def _block(text, start):
    """From the first brace behind `start` to its match."""
    at = text.index("{", start)
    depth = 0
    for k in range(at, len(text)):
        depth += {"{": 1, "}": -1}.get(text[k], 0)
        if depth == 0:
            return text[at:k + 1]
    raise AssertionError("braces do not match")


def _loops_that_waits_leave(text):
    for head in re.finditer(r"\b(for|while)\s*\(", text):
        depth, k = 0, head.end() - 1
        while True:  # behind the loop's head
            depth += {"(": 1, ")": -1}.get(text[k], 0)
            k += 1
            if depth == 0:
                break
        if not text[k:].lstrip().startswith("{"):
            continue
        body = _block(text, k)
        if WAIT.search(body) and re.search(r"\bbreak\b", body):
            yield body


FILES = sorted(p.name for p in CSRC.glob("*.cu") if WAIT.search(p.read_text()))


def test_there_are_such_kernels():
    assert "int8_tcgen05.cu" in FILES and len(FILES) >= 4


@pytest.mark.parametrize("name", FILES)
def test_no_unbounded_barrier_where_a_wait_may_leave(name):
    for body in _loops_that_waits_leave(_without_comments((CSRC / name).read_text())):
        assert not BARRIER.search(body), body[max(0, BARRIER.search(body).start() - 200):BARRIER.search(body).end() + 100]
