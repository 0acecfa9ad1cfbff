"""CPU checks of the block-scaled 8-bit format: the oracle's codes against
torch's conversion, and what the entry points refuse before they launch."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from glm53flash import fp8_block as F
from glm53flash.contract import ContractError
from glm53flash.layers import DeferredLinear, DenseMLP, RMSNorm
from livglm_amd import native
from oracle import fp8_oracle as P


def test_oracle_codes_are_e4m3():
    every = np.arange(256, dtype=np.uint8)
    ours, theirs = P.decode(every), torch.from_numpy(every).view(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(ours, theirs)
    rng = np.random.default_rng(1)
    values = np.unique(ours[np.isfinite(ours)])
    x = np.concatenate([values, (values[1:] + values[:-1]) / 2, rng.uniform(-448, 448, 5000),
                        rng.normal(0, 1e-2, 5000), [1e-30, -1e-40, 0.0]]).astype(np.float32)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    np.testing.assert_array_equal(P.encode(x), want)
    assert P.encode(np.array([np.nan], np.float32))[0] & 127 == 127


def test_oracle_quantiser_bounds():
    rng = np.random.default_rng(2)
    x = (rng.normal(0, 1, (5, 300)) * 10.0 ** rng.integers(-30, 30, (5, 300))).astype(np.float32)
    x[1] = 0
    x[2, :128] = 1e-44
    codes, scales = P.quantize_rows(x)
    assert codes.shape == (5, 300) and scales.shape == (5, 3)
    assert (scales >= np.float32(2.0 ** -126)).all() and not codes[1].any()
    err = np.abs(P.row_values(codes, scales) - x)
    step = np.repeat(scales, 128, 1)[:, :300].astype(np.float64)
    # half a step of the value, or of the subnormals
    assert (err <= np.maximum(np.abs(x) * (2.0 ** -4 + 2.0 ** -22), step * 2.0 ** -10 * 1.001)).all()


FAKE = ctypes.c_void_p(0x1000)  # never dereferenced: validation fails first


def refused(code, name, *args):
    assert getattr(native.load(), name)(*args) == code, native.load().glm_last_error()
    return native.load().glm_last_error().decode()


def linear_args(x_type=0, x=FAKE, xs=FAKE, T=1, K=128, w=FAKE, s=FAKE, n=16, ws=FAKE, need=1 << 40, out=FAKE):
    return None, x, x_type, xs, T, K, w, s, n, ws, need, out


def gate_args(x_type=0, x=FAKE, xs=FAKE, T=1, K=128, w=FAKE, s=FAKE, n=16, ws=FAKE, need=1 << 40, out=FAKE):
    return None, x, x_type, xs, T, K, w, s, w, s, n, 10.0, ws, need, out, FAKE


@pytest.mark.parametrize("name, args", [("glm_fp8_linear", linear_args), ("glm_fp8_gate_up", gate_args)])
def test_products_refuse(name, args):
    bad, shape = native.GLM_ERR_INVALID_ARGUMENT, native.GLM_ERR_UNSUPPORTED_SHAPE
    off = ctypes.c_void_p(0x1008)
    for kw in ({"x_type": 3}, {"x_type": -1}, {"T": -1}, {"K": 0}, {"n": 0}, {"x": None}, {"w": None},
               {"s": None}, {"out": None}, {"x_type": 2, "xs": None}, {"x": off}, {"w": off}, {"s": off},
               {"out": off}, {"ws": off}):
        refused(bad, name, *args(**kw))
    for kw in ({"K": 8}, {"K": 136}, {"K": (1 << 20) + 16}, {"n": (1 << 20) + 16}, {"T": (1 << 21) + 1}):
        refused(shape, name, *args(**kw))
    if name == "glm_fp8_gate_up":
        refused(shape, name, *args(n=24))
    lib = native.load()
    need = lib.glm_fp8_workspace_bytes(0, 500, 128, 16, int(name == "glm_fp8_gate_up"))
    assert need >= 500 * 132
    assert "workspace" in refused(native.GLM_ERR_WORKSPACE, name, *args(T=500, need=need - 1))
    refused(native.GLM_ERR_WORKSPACE, name, *args(T=500, ws=None, need=0))
    assert getattr(lib, name)(*args(T=0)) == native.GLM_OK  # no row: nothing to do


def test_quantisers_refuse():
    bad, shape = native.GLM_ERR_INVALID_ARGUMENT, native.GLM_ERR_UNSUPPORTED_SHAPE
    off = ctypes.c_void_p(0x1004)
    refused(shape, "glm_fp8_quantize_rows", None, FAKE, 0, 1, 12, FAKE, FAKE)
    for args in ((FAKE, 2, 1, 8, FAKE, FAKE), (FAKE, 0, -1, 8, FAKE, FAKE), (None, 0, 1, 8, FAKE, FAKE),
                 (FAKE, 0, 1, 8, None, FAKE), (FAKE, 0, 1, 8, FAKE, None), (off, 0, 1, 8, FAKE, FAKE)):
        refused(bad, "glm_fp8_quantize_rows", None, *args)
    refused(shape, "glm_fp8_quantize_weight", None, FAKE, 4, 12, FAKE, FAKE)
    refused(shape, "glm_fp8_quantize_weight", None, FAKE, 65535 * 128 + 1, 8, FAKE, FAKE)
    # grids of 2^32 threads and more
    refused(shape, "glm_fp8_quantize_weight", None, FAKE, 1, (1 << 31) - 8, FAKE, FAKE)
    refused(bad, "glm_fp8_quantize_weight", None, FAKE, 0, 8, FAKE, FAKE)
    refused(bad, "glm_fp8_quantize_weight", None, FAKE, 4, 8, None, FAKE)

    def norm(x=FAKE, xt=0, r=FAKE, rt=0, T=1, d=64, w=FAKE, eps=1e-6, ro=FAKE, c=FAKE, s=FAKE):
        return None, x, xt, r, rt, T, d, w, eps, ro, c, s

    for kw in ({"x": None}, {"xt": 2}, {"rt": 2}, {"T": -1}, {"d": 0}, {"eps": -1.0}, {"ro": None}, {"r": None},
               {"c": None}, {"s": None}, {"w": off}, {"eps": float("nan")}):
        refused(bad, "glm_add_rms_norm_fp8", *norm(**kw))
    for d in (12, 32776):
        refused(shape, "glm_add_rms_norm_fp8", *norm(d=d))
    refused(shape, "glm_add_rms_norm_fp8", *norm(T=1 << 24, d=8))
    refused(shape, "glm_add_rms_norm_fp8", *norm(T=1 << 22, d=8))
    assert native.load().glm_add_rms_norm_fp8(*norm(T=0)) == native.GLM_OK


def test_python_side_refuses_what_is_no_gpu_tensor():
    x = torch.zeros((2, 128), dtype=torch.bfloat16)
    w, s = torch.zeros((16, 128), dtype=torch.uint8), torch.zeros((1, 1))
    for call in (lambda: F.quantize_rows(x), lambda: F.quantize_weight(x), lambda: F.linear(x, w, s),
                 lambda: F.gate_up(x, w, s, w, s, 0.0), lambda: F.add_rms_norm(x, None, 1e-6),
                 lambda: F.linear((w, s), w, s), lambda: F.linear((w,), w, s), lambda: F.quantize_rows(None),
                 lambda: F.linear("rows", w, s)):
        with pytest.raises(ContractError):
            call()


def test_outputs_lie_apart():
    raw = torch.zeros(64, dtype=torch.uint8)
    for a, b in ((0, 0), (0, 8), (8, 0), (15, 0), (0, 15)):  # 16 bytes each
        with pytest.raises(ContractError, match="overlaps"):
            F._apart(raw[a:a + 16], "out", None, raw[40:], raw[b:b + 16])
    F._apart(raw[:16], "out", None, raw[16:32], raw[:0])


def test_layers_keep_their_rules():
    lin = DeferredLinear(128, 32, quantize_resident=False)
    with pytest.raises(ContractError, match="excluded"):
        lin.quantize_to_fp8_block()
    lin = DeferredLinear(24, 32)
    lin.weight = kept = torch.zeros((32, 24), dtype=torch.bfloat16)
    with pytest.raises(ContractError, match="multiple of 16"):
        lin.quantize_to_fp8_block()
    assert lin.weight is kept and lin.quantization_mode is None
    lin = DeferredLinear(128, 32)
    with pytest.raises(ContractError, match="not loaded"):
        lin.quantize_to_fp8_block()
    lin.quantization_mode = "mxfp8"
    with pytest.raises(ContractError, match="already"):
        lin.quantize_to_fp8_block()
    lin.quantization_mode = "fp8_block"
    with pytest.raises(ContractError, match="already"):
        lin.quantize_to_mxfp8()
    with pytest.raises(ContractError):
        lin.fmt
    mlp = DenseMLP(128, 32, 10.0)
    assert not mlp.block_scaled
    mlp.gate_proj.quantization_mode = "fp8_block"
    assert not mlp.block_scaled and mlp.fused_format() is None
    for p in (mlp.up_proj, mlp.down_proj):
        p.quantization_mode = "fp8_block"
    assert mlp.block_scaled and mlp.fused_format() is None
    with pytest.raises(ContractError, match="not loaded"):
        mlp(None)
    norm = RMSNorm(128, 1e-6)
    with pytest.raises(ContractError, match="not loaded"):
        norm.quantized(torch.zeros(2, 128))
    with pytest.raises(ContractError, match="features"):
        norm.quantized(torch.zeros(2, 64))
