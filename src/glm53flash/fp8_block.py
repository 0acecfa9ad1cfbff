"""Products of 8-bit rows and 8-bit weights with f32 scales.

The reference's resident weights are group-32 MXFP8 and its rows bf16
(``layers.py:38-99``).  Checkpoints also hold weights in E4M3 with an f32 scale
for each 128 x 128 block, to be multiplied with E4M3 rows that have a scale for
each 128 channels; here are the operators of that format:

* ``quantize_rows`` and ``quantize_weight`` make codes and scales;
* ``add_rms_norm`` adds the residual, norms and quantises the result;
* ``linear`` multiplies, and ``gate_up`` is the first half of a SwiGLU MLP.

They work on the current stream of the tensors' device, without host
synchronisation, and may be captured in a HIP graph.  ``DeferredLinear``,
``DenseMLP`` (``quantize_to_fp8_block``) and ``RMSNorm.quantized`` in
``layers`` are these operators behind the reference's interface.

Codes are u8 (a ``torch.float8_e4m3fn`` tensor is taken as its bytes): rows
``[..., K]`` with scales ``[..., ceil(K / 128)]``, weights ``[N, K]`` with
scales ``[ceil(N / 128), ceil(K / 128)]``.
"""

from __future__ import annotations

from functools import lru_cache
from typing import NamedTuple

import torch

from . import _native as N
from .contract import ContractError

GROUP = 128

_BF16, _F32, _U8, _F8 = torch.bfloat16, torch.float32, torch.uint8, torch.float8_e4m3fn
_ROWS = {_BF16: N.native.GLM_ROWS_BF16, _F32: N.native.GLM_ROWS_F32}
_getDevice = torch._C._cuda_getDevice
_getStream = torch._C._cuda_getCurrentRawStream
_empty = torch.empty


class Fp8Rows(NamedTuple):
    """Quantised rows: ``codes`` u8 ``[..., K]``, ``scales`` f32 ``[...,
    ceil(K / 128)]``; a code times its group's scale is the value."""

    codes: torch.Tensor
    scales: torch.Tensor


def _groups(n: int) -> int:
    return -(-n // GROUP)


def _run(device: int, name: str, *args) -> None:
    """A native call on the current stream of the tensors' device, which is the
    current one meanwhile, as a launch needs it."""
    function = getattr(N.native.load(), name)
    if device == _getDevice():
        code = function(_getStream(device), *args)
    else:
        with torch.cuda.device(device):
            code = function(_getStream(device), *args)
    if code:
        N.check(name, code)


def _check(t, name: str, dtypes: tuple, device: int) -> None:
    """A contiguous tensor of the call's device and one of the dtypes."""
    N.require_device(t, name, dtypes)
    if t.get_device() != device:
        raise ContractError(f"{name} is on {t.device}, the call's rows on device {device}")


def _out(out, name: str, shape: tuple, dtype: torch.dtype, like: torch.Tensor) -> torch.Tensor:
    if out is None:
        return _empty(shape, dtype=dtype, device=like.device)
    _check(out, name, (dtype,), like.get_device())
    if tuple(out.shape) != tuple(shape):
        raise ContractError(f"{name} {tuple(out.shape)}, expected {tuple(shape)}")
    return out


def _plain_rows(x, name: str) -> tuple[int, int, int]:
    """Device, rows and channels of bf16 or f32 rows ``[..., K]``."""
    N.require_device(x, name, (_BF16, _F32))
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ContractError(f"{name} must be [..., K] rows, got {tuple(x.shape)}")
    K = x.shape[-1]
    return x.get_device(), x.numel() // K, K


def _rows(x) -> tuple:
    """Device, rows, channels, leading shape and the native (pointer, type,
    scales) of a product's rows: bf16, f32 or ``Fp8Rows``."""
    if isinstance(x, tuple):
        if len(x) != 2:
            raise ContractError("quantised rows are (codes, scales)")
        codes, scales = x
        N.require_device(codes, "codes", (_U8, _F8))
        dev = codes.get_device()
        _check(scales, "scales", (_F32,), dev)
        if codes.dim() < 1 or codes.shape[-1] < 1 or \
                tuple(scales.shape) != (*codes.shape[:-1], _groups(codes.shape[-1])):
            raise ContractError(f"scales {tuple(scales.shape)} do not fit codes "
                                f"{tuple(codes.shape)}")
        K = codes.shape[-1]
        return dev, codes.numel() // K, K, codes.shape[:-1], codes.device, \
            (codes.data_ptr(), N.native.GLM_ROWS_FP8, scales.data_ptr())
    dev, T, K = _plain_rows(x, "x")
    return dev, T, K, x.shape[:-1], x.device, (x.data_ptr(), _ROWS[x.dtype], None)


def _weight(w, scales, name: str, K: int, dev: int) -> int:
    """The output features of a weight that fits rows of K channels."""
    _check(w, name, (_U8, _F8), dev)
    _check(scales, f"{name} scales", (_F32,), dev)
    if w.dim() != 2 or w.shape[1] != K or w.shape[0] < 1 or \
            tuple(scales.shape) != (_groups(w.shape[0]), _groups(K)):
        raise ContractError(f"{name} {tuple(w.shape)} with scales {tuple(scales.shape)} does not "
                            f"fit rows of {K} channels")
    return w.shape[0]


@lru_cache(maxsize=256)  # a function of the sizes alone
def _workspace_bytes(name: str, *sizes: int) -> int:
    if any(s >> 31 for s in sizes):
        raise ContractError(f"sizes {sizes} pass 32 bits")
    return int(getattr(N.native.load(), name)(*sizes))


def _workspace(device, name: str, *sizes: int) -> tuple:
    need = _workspace_bytes(name, *sizes)
    ws = _empty(need, dtype=_U8, device=device) if need else None
    return ws, need


def _sizes(name: str, *sizes: int) -> None:
    if any(s >> 31 for s in sizes):  # (the library's sizes are 32-bit: none may wrap)
        raise ContractError(f"{name}: sizes {sizes} pass 32 bits")


def quantize_rows(x: torch.Tensor, *, out: Fp8Rows | None = None) -> Fp8Rows:
    """Codes and scales of bf16 or f32 rows ``[..., K]``, K a multiple of 8:
    per 128 channels ``scale = amax / 448``, ``code = e4m3(x * (448 / amax))``
    with amax the largest finite magnitude; an infinity or a NaN becomes NaN."""
    dev, T, K = _plain_rows(x, "x")
    _sizes("quantize_rows", T, K)
    codes = _out(out and out[0], "codes", x.shape, _U8, x)
    scales = _out(out and out[1], "scales", (*x.shape[:-1], _groups(K)), _F32, x)
    if T:
        _run(dev, "glm_fp8_quantize_rows", x.data_ptr(), _ROWS[x.dtype], T, K, codes.data_ptr(),
             scales.data_ptr())
    return Fp8Rows(codes, scales)


def quantize_weight(weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes and block scales of a bf16 weight ``[N, K]``."""
    N.require_device(weight, "weight", (_BF16,))
    if weight.dim() != 2 or not weight.numel():
        raise ContractError(f"weight must be [N, K], got {tuple(weight.shape)}")
    n, K = weight.shape
    _sizes("quantize_weight", n, K)
    codes = _empty((n, K), dtype=_U8, device=weight.device)
    scales = _empty((_groups(n), _groups(K)), dtype=_F32, device=weight.device)
    _run(weight.get_device(), "glm_fp8_quantize_weight", weight.data_ptr(), n, K, codes.data_ptr(),
         scales.data_ptr())
    return codes, scales


def add_rms_norm(x: torch.Tensor, weight: torch.Tensor | None, eps: float, *,
                 residual: torch.Tensor | None = None, residual_out: torch.Tensor | None = None,
                 out: Fp8Rows | None = None) -> tuple[Fp8Rows, torch.Tensor | None]:
    """``(rows, h)``: ``h = x + residual`` in the residual's type, and the
    quantised ``h / sqrt(mean(h^2) + eps) * weight`` of the unrounded sum.
    ``x`` and ``residual`` bf16 or f32 ``[..., d]``, ``weight`` f32 ``[d]`` or
    None; ``residual_out`` may be ``residual`` itself.  Without a residual h is
    x, and None is returned for it."""
    dev, T, d = _plain_rows(x, "x")
    _sizes("add_rms_norm", T, d)
    if weight is not None:
        _check(weight, "weight", (_F32,), dev)
        if weight.numel() != d:
            raise ContractError(f"a weight of {weight.numel()} for rows of {d} channels")
    kind = N.native.GLM_ROWS_BF16
    if residual is not None:
        _check(residual, "residual", (_BF16, _F32), dev)
        if residual.shape != x.shape:
            raise ContractError(f"residual {tuple(residual.shape)}, rows {tuple(x.shape)}")
        kind = _ROWS[residual.dtype]
        residual_out = _out(residual_out, "residual_out", x.shape, residual.dtype, x)
    elif residual_out is not None:
        raise ContractError("residual_out comes with a residual")
    codes = _out(out and out[0], "codes", x.shape, _U8, x)
    scales = _out(out and out[1], "scales", (*x.shape[:-1], _groups(d)), _F32, x)
    if T:
        _run(dev, "glm_add_rms_norm_fp8", x.data_ptr(), _ROWS[x.dtype], N.ptr(residual), kind, T,
             d, N.ptr(weight), float(eps), N.ptr(residual_out), codes.data_ptr(),
             scales.data_ptr())
    return Fp8Rows(codes, scales), residual_out


def linear(x: torch.Tensor | Fp8Rows, weight: torch.Tensor, scales: torch.Tensor, *,
           out: torch.Tensor | None = None) -> torch.Tensor:
    """bf16 ``[..., N]`` of ``x @ weight.T``; bf16 and f32 rows are quantised as
    ``quantize_rows`` does.  K is a multiple of 16."""
    dev, T, K, lead, device, rows = _rows(x)
    n = _weight(weight, scales, "weight", K, dev)
    _sizes("linear", T, K, n)
    out = _out(out, "out", (*lead, n), _BF16, weight)
    if T:
        ws, need = _workspace(device, "glm_fp8_workspace_bytes", rows[1], T, K, n, 0)
        _run(dev, "glm_fp8_linear", *rows, T, K, weight.data_ptr(), scales.data_ptr(), n,
             N.ptr(ws), need, out.data_ptr())
    return out


def gate_up(x: torch.Tensor | Fp8Rows, gate: torch.Tensor, gate_scales: torch.Tensor,
            up: torch.Tensor, up_scales: torch.Tensor, limit: float, *,
            out: Fp8Rows | None = None) -> Fp8Rows:
    """Quantised ``silu(g) * u`` of ``g = x @ gate.T`` and ``u = x @ up.T``,
    both weights ``[I, K]``, I a multiple of 16; with ``limit > 0`` g is cut at
    ``limit`` and u at both ends.  f32 until the codes."""
    dev, T, K, lead, device, rows = _rows(x)
    n = _weight(gate, gate_scales, "gate", K, dev)
    if _weight(up, up_scales, "up", K, dev) != n:
        raise ContractError(f"gate {tuple(gate.shape)} and up {tuple(up.shape)} differ")
    _sizes("gate_up", T, K, n)
    codes = _out(out and out[0], "codes", (*lead, n), _U8, gate)
    codes_scales = _out(out and out[1], "scales", (*lead, _groups(n)), _F32, gate)
    if T:
        ws, need = _workspace(device, "glm_fp8_workspace_bytes", rows[1], T, K, n, 1)
        _run(dev, "glm_fp8_gate_up", *rows, T, K, gate.data_ptr(), gate_scales.data_ptr(),
             up.data_ptr(), up_scales.data_ptr(), n, float(limit), N.ptr(ws), need,
             codes.data_ptr(), codes_scales.data_ptr())
    return Fp8Rows(codes, codes_scales)


__all__ = ["Fp8Rows", "GROUP", "add_rms_norm", "gate_up", "linear", "quantize_rows",
           "quantize_weight"]
