"""Wide buffer stores name no scalar offset register (no GPU needed).

A store of 12 or 16 bytes reads its last data registers up to two wait states after it is issued. The compiler keeps
instructions that write them away from stores with a constant offset only: behind one with an offset in a scalar
register the next conversion's result was stored instead."""

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "late-interaction-kernels_amd" / "csrc"
SOURCES = sorted([*CSRC.glob("*.hip"), *CSRC.glob("*.h")])


def _arguments(text, at):
    """The arguments of the call whose parenthesis opens at ``at``."""
    depth, start, out = 0, at + 1, []
    for i in range(at, len(text)):
        c = text[i]
        depth += (c in "([{") - (c in ")]}")
        if (c == "," and depth == 1) or depth == 0:
            out.append(text[start:i].strip())
            start = i + 1
            if depth == 0:
                return out
    raise AssertionError("unbalanced parentheses")


@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.name)
def test_wide_buffer_stores_have_constant_offsets(path):
    text = re.sub(r"//[^\n]*", "", path.read_text())
    for m in re.finditer(r"raw_(?:ptr_)?buffer_store_b(?:96|128)\s*\(", text):
        args = _arguments(text, m.end() - 1)
        assert args[3] == "0", f"{path.name}: offset {args[3]!r}"
    # (nor in assembly of our own, where the compiler counts nothing)
    assert not re.search(r"(buffer|global|flat)_store_dwordx[34]", text)


def test_the_walking_kernel_stores_by_buffer():
    assert "raw_buffer_store_b128(" in (CSRC / "lik_linear8.hip").read_text()
