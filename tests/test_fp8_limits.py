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


def test_gated_pairs_are_split_along_k_where_cus_are_idle_alone():
    # the workspace holds the f32 sums [split][2][T][N]: a pair of more than half a round of
    # 256 workgroups of 16 x 16 has one split, a smaller one as many as fill a round, at most
    # eight, each with a group of 128 for every of its eight waves
    need = native.load().glm_fp8_workspace_bytes
    split = 0
    for K in (16, 128, 1024, 2048, 4096, 16384, 1 << 20):
        for N in [*range(16, 8193, 208), 16384]:
            for T in [*range(1, 100), 128, 200, 333, 600, 1000]:
                one = -(-2 * T * N * 4 // 256) * 256
                have = need(native.GLM_ROWS_FP8, T, K, N, 1)
                if have == 0:  # tiles that gate by themselves
                    continue
                tiles = -(-N // 16) * -(-T // 16)
                want = min(256 // tiles, -(-K // 128) // 8, 8) if tiles <= 128 else 1
                split += want > 1
                assert abs(have - max(want, 1) * one) < 256 * max(want, 1), (T, K, N)
    assert split > 1000
