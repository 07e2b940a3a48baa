"""Waits of the kernels that only their source can show: no GPU. A named barrier has no time limit, so
every thread that it counts has to come to it as often as the others."""

from __future__ import annotations

import os
import re

import mlx_diffuser_b200

CSRC = os.path.join(os.path.dirname(mlx_diffuser_b200.__file__), "csrc")


def _block(text: str, start: int) -> str:
    """The braces that open at or behind ``start``, without comments."""
    text = re.sub(r"//[^\n]*", "", text[start:])
    depth, first = 0, text.index("{")
    for i in range(first, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth == 0:
            return text[first : i + 1]
    raise AssertionError("unbalanced braces")


def test_epilogue_warps_meet_their_barrier_equally_often():
    """The projection's epilogue warps meet at epi_sync() once a tile. A warp whose wait has run out must not
    leave the loop over the tiles before the others, nor skip to the next tile ahead of the barrier."""
    with open(os.path.join(CSRC, "linear_tc.cu")) as f:
        text = f.read()
    text = text[text.index("__global__") :]
    assert text.count("epi_sync();") == 1
    at = text.rindex("for (int32_t t = unit", 0, text.index("epi_sync();"))
    loop = _block(text, at)
    head, tail = loop.split("epi_sync();")
    assert "break" not in loop and "return" not in loop and "goto" not in loop
    assert "continue" not in head
    # the waits behind the barrier are bounded, and a warp that has given up waits no more
    assert tail.index("if (!ok) continue;") < tail.index("mbar_wait_bounded")
    assert "mbar_try_wait" not in loop
