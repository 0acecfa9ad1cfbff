"""CPU checks of the block-scaled operators' limits: sizes at which their own
arithmetic would wrap are refused by the host."""

from __future__ import annotations

import ctypes

import pytest

from livglm_amd import native

FAKE = ctypes.c_void_p(0x1000)  # never dereferenced: validation fails first


@pytest.mark.parametrize("T", [0, 1, 1 << 20])
@pytest.mark.parametrize("K", [(1 << 31) - 8, (1 << 31) - 120])
@pytest.mark.parametrize("kind", [native.GLM_ROWS_BF16, native.GLM_ROWS_F32])
def test_rows_whose_groups_pass_32_bits(T, K, kind):
    # K + 127 is past 2^31 there: the number of groups, and with it the grid, would be negative
    lib = native.load()
    assert lib.glm_fp8_quantize_rows(None, FAKE, kind, T, K, FAKE, FAKE) == native.GLM_ERR_UNSUPPORTED_SHAPE
    assert lib.glm_fp8_quantize_rows(None, FAKE, kind, 0, (1 << 31) - 128, FAKE, FAKE) == native.GLM_OK
