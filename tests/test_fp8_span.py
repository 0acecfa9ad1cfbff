"""CPU check of what the block-scaled tiles' loads may touch (fp8_span.h, compiled
for the host): every byte lies in its operand, whichever way a buffer's range
check takes the scalar offset."""

from __future__ import annotations

import ctypes
import os
import subprocess

import numpy as np
import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "livglm_amd", "csrc")
SOURCE = """
#include "fp8_span.h"
extern "C" void span(int first, int there, int *out) {
  const glm::Fp8Span s = glm::fp8_span(first, there);
  out[0] = s.first;
  out[1] = s.rows;
}
extern "C" int scale_group(int g, int j, int groups) { return glm::fp8_scale_group(g, j, groups); }
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    at = tmp_path_factory.mktemp("span")
    (at / "span.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}", str(at / "span.cpp"),
                    "-o", str(at / "span.so")], check=True)
    return ctypes.CDLL(str(at / "span.so"))


def touched(offsets, scalar, size, width):
    """The bytes [first, end) that a load's lanes touch, by each reading of the
    range check: offsets below the size, or below size - scalar in 32 bits."""
    for limit in (size, (size - scalar) % 2 ** 32):
        yield from (o + scalar for o in offsets if o < limit)
        yield from (o + scalar + width - 1 for o in offsets if o < limit)


@pytest.mark.parametrize("K", [16, 144, 400, 1024])
@pytest.mark.parametrize("step, tile", [(32, 64), (64, 128), (64, 256)])
def test_rows_of_a_tile(lib, K, step, tile):
    out = (ctypes.c_int * 2)()
    lanes = np.arange(step * 8)
    for there in [*range(1, tile, 7), step, step + 1, tile - 1, tile]:
        for first in range(0, tile, step):
            lib.span(first, there, out)
            begin, rows = out[0] * K, out[1]
            assert 0 <= out[0] < there and rows >= 1
            if first < there:  # what there is comes in its place
                assert (out[0], rows) == (first, there - first)
            for group in range(-(-K // 128)):
                piece = 16 * (lanes % 8)
                offsets = (lanes // 8 * K + piece)[piece < K - 128 * group].tolist()
                for byte in touched(offsets, 128 * group, rows * K, 16):
                    assert 0 <= begin + byte < there * K, (there, first, group)


@pytest.mark.parametrize("groups", [1, 2, 3, 5, 6, 7, 9])
@pytest.mark.parametrize("tokens", [1, 2, 63, 64])
def test_scales_of_a_tile(lib, groups, tokens):
    size = 4 * tokens * groups
    for g in range(0, groups, 4):
        for j in range(4):
            group = lib.scale_group(g, j, groups)
            if g + j < groups:
                assert group == g + j
            for byte in touched([4 * t * groups for t in range(64)], 4 * group, size, 4):
                assert 0 <= byte < size, (g, j)
