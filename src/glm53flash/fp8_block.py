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
scales ``[ceil(N / 128), ceil(K / 128)]``.  A row's scale times a block's is
formed first, in f32: where that product is not finite, the row gets infinities
or NaN, and below 2^-126 it loses bits.  Every tensor's data begins on 16
bytes.  Outputs that the caller brings share no memory with a call's other
tensors, except where said.
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
_CODED = N.native.GLM_ROWS_FP8
_CODES, _SCALES = (_U8, _F8), (_F32,)
_getDevice = torch._C._cuda_getDevice
_getStream = torch._C._cuda_getCurrentRawStream
_empty, _empty_like = torch.empty, torch.empty_like


class Fp8Rows(NamedTuple):
    """Quantised rows: ``codes`` u8 ``[..., K]``, ``scales`` f32 ``[...,
    ceil(K / 128)]``; a code times its group's scale is the value."""

    codes: torch.Tensor
    scales: torch.Tensor


# The calls of a decode step are a few microseconds of GPU work each, so what
# the host does before them counts: what is right is recognised with a few
# attributes, and only what is not is looked at again for the message.


def _run(device: int, name: str, function, *args) -> None:
    """A native call on the current stream of the tensors' device, which is the
    current one meanwhile, as a launch needs it."""
    if device == _getDevice():
        code = function(_getStream(device), *args)
    else:
        with torch.cuda.device(device):
            code = function(_getStream(device), *args)
    if code:
        N.check(name, code)


def _check(t, name: str, dtypes: tuple, device: int) -> None:
    """A contiguous tensor of the call's device and one of the dtypes."""
    try:
        fine = t.dtype in dtypes and t.get_device() == device and t.is_contiguous()
    except AttributeError:  # no tensor
        fine = False
    if not fine:
        N.require_device(t, name, dtypes)
        raise ContractError(f"{name} is on {t.device}, the call's rows on device {device}")


def _given(out, name: str, shape, dtype: torch.dtype, device: int) -> torch.Tensor:
    """An output that the caller brings."""
    _check(out, name, (dtype,), device)
    if out.shape != shape:
        raise ContractError(f"{name} {tuple(out.shape)}, expected {tuple(shape)}")
    return out


def _apart(out: torch.Tensor, name: str, *inputs) -> None:
    """An output that the caller brings shares no memory with what is read for
    it: workgroups write while others still read."""
    first = out.data_ptr()
    end = first + out.nbytes
    for t in inputs:
        if t is not None and first < t.data_ptr() + t.nbytes and t.data_ptr() < end:
            raise ContractError(f"{name} overlaps another tensor of the call")


def _plain_rows(x, name: str = "x") -> tuple[int, int, int, int]:
    """Device, native type, rows and channels of bf16 or f32 rows ``[..., K]``."""
    try:
        kind, dev, shape = _ROWS.get(x.dtype), x.get_device(), x.shape
        K = shape[-1] if len(shape) else 0
        fine = kind is not None and dev >= 0 and K > 0 and x.is_contiguous()
    except AttributeError:  # no tensor
        fine = False
    if not fine:
        N.require_device(x, name, (_BF16, _F32))
        raise ContractError(f"{name} must be [..., K] rows, got {tuple(x.shape)}")
    T = shape[0] if len(shape) == 2 else x.numel() // K
    if (T | K) >> 31:  # (the library's sizes are 32-bit: none may wrap)
        raise ContractError(f"{name}: {T} rows of {K} channels pass 32 bits")
    return dev, kind, T, K


def _rows(x) -> tuple:
    """Device, native type, rows, channels, pointers of the rows and their
    scales, and the tensor whose leading shape they have, of a product's rows:
    bf16, f32 or ``Fp8Rows``."""
    if not isinstance(x, tuple):
        return *_plain_rows(x), x.data_ptr(), None, x
    if len(x) != 2:
        raise ContractError("quantised rows are (codes, scales)")
    codes, scales = x
    try:
        dev, shape = codes.get_device(), codes.shape
        K = shape[-1] if len(shape) else 0
        fine = codes.dtype in _CODES and dev >= 0 and K > 0 and codes.is_contiguous()
    except AttributeError:  # no tensor
        fine = False
    if not fine:
        N.require_device(codes, "codes", _CODES)
        raise ContractError(f"codes must be [..., K] rows, got {tuple(codes.shape)}")
    _check(scales, "scales", _SCALES, dev)
    if scales.shape != (*shape[:-1], (K + 127) >> 7):
        raise ContractError(f"scales {tuple(scales.shape)} do not fit codes {tuple(shape)}")
    T = shape[0] if len(shape) == 2 else codes.numel() // K
    if (T | K) >> 31:
        raise ContractError(f"codes: {T} rows of {K} channels pass 32 bits")
    return dev, _CODED, T, K, codes.data_ptr(), scales.data_ptr(), codes


def _weight(w, scales, name: str, K: int, dev: int) -> int:
    """The output features of a weight that fits rows of K channels."""
    _check(w, name, _CODES, dev)
    _check(scales, f"{name} scales", _SCALES, dev)
    shape = w.shape
    n = shape[0] if len(shape) == 2 else 0
    if n < 1 or n >> 31 or shape[1] != K or scales.shape != ((n + 127) >> 7, (K + 127) >> 7):
        raise ContractError(f"{name} {tuple(shape)} with scales {tuple(scales.shape)} does not "
                            f"fit rows of {K} channels")
    return n


@lru_cache(maxsize=256)  # a function of the sizes alone
def _workspace_bytes(*sizes: int) -> int:
    return int(N.native.load().glm_fp8_workspace_bytes(*sizes))


def _coded_out(out, like: torch.Tensor, T: int, n: int, dev: int, *inputs) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes ``[..., n]`` of a tensor's leading shape and their scales, apart
    from the inputs."""
    groups = (n + 127) >> 7
    shape = like.shape
    if out is None:
        device = like.device
        if len(shape) == 2:  # (sizes one by one: a tuple of them takes a third longer)
            return (_empty(T, n, dtype=_U8, device=device),
                    _empty(T, groups, dtype=_F32, device=device))
        return (_empty((*shape[:-1], n), dtype=_U8, device=device),
                _empty((*shape[:-1], groups), dtype=_F32, device=device))
    if not isinstance(out, tuple) or len(out) != 2:
        raise ContractError("quantised rows are (codes, scales)")
    codes = _given(out[0], "codes", (*shape[:-1], n), _U8, dev)
    scales = _given(out[1], "scales", (*shape[:-1], groups), _F32, dev)
    _apart(codes, "codes", scales, *inputs)
    _apart(scales, "scales", *inputs)
    return codes, scales


def quantize_rows(x: torch.Tensor, *, out: Fp8Rows | None = None) -> Fp8Rows:
    """Codes and scales of bf16 or f32 rows ``[..., K]``, K a multiple of 8:
    per 128 channels ``scale = amax / 448``, ``code = e4m3(x * (448 / amax))``
    with amax the largest finite magnitude; an infinity or a NaN becomes NaN."""
    dev, kind, T, K = _plain_rows(x)
    codes, scales = _coded_out(out, x, T, K, dev, x)
    if T:
        _run(dev, "glm_fp8_quantize_rows", N.native.load().glm_fp8_quantize_rows, x.data_ptr(),
             kind, T, K, codes.data_ptr(), scales.data_ptr())
    return Fp8Rows(codes, scales)


def quantize_weight(weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes and block scales of a bf16 weight ``[N, K]``."""
    N.require_device(weight, "weight", (_BF16,))
    if weight.dim() != 2 or not weight.numel():
        raise ContractError(f"weight must be [N, K], got {tuple(weight.shape)}")
    n, K = weight.shape
    if (n | K) >> 31:
        raise ContractError(f"a weight {tuple(weight.shape)} passes 32 bits")
    codes = _empty((n, K), dtype=_U8, device=weight.device)
    scales = _empty(((n + 127) >> 7, (K + 127) >> 7), dtype=_F32, device=weight.device)
    _run(weight.get_device(), "glm_fp8_quantize_weight", N.native.load().glm_fp8_quantize_weight,
         weight.data_ptr(), n, K, codes.data_ptr(), scales.data_ptr())
    return codes, scales


def add_rms_norm(x: torch.Tensor, weight: torch.Tensor | None, eps: float, *,
                 residual: torch.Tensor | None = None, residual_out: torch.Tensor | None = None,
                 out: Fp8Rows | None = None) -> tuple[Fp8Rows, torch.Tensor | None]:
    """``(rows, h)``: ``h = x + residual`` in the residual's type, and the
    quantised ``h / sqrt(mean(h^2) + eps) * weight`` of the unrounded sum.
    ``x`` and ``residual`` bf16 or f32 ``[..., d]``, ``weight`` f32 ``[d]`` or
    None; ``residual_out`` may be ``residual`` itself, or ``x`` where it has the
    residual's type.  Without a residual h is
    x, and None is returned for it."""
    dev, kind, T, d = _plain_rows(x)
    shape = x.shape
    if weight is not None:
        _check(weight, "weight", _SCALES, dev)
        if weight.numel() != d:
            raise ContractError(f"a weight of {weight.numel()} for rows of {d} channels")
    rkind = kind
    if residual is not None:
        _check(residual, "residual", (_BF16, _F32), dev)
        if residual.shape != shape:
            raise ContractError(f"residual {tuple(residual.shape)}, rows {tuple(shape)}")
        rkind = _ROWS[residual.dtype]
        if residual_out is None:
            residual_out = _empty_like(residual)
        else:
            _given(residual_out, "residual_out", shape, residual.dtype, dev)
            # (in the place of either, its own rows are read before they are written)
            _apart(residual_out, "residual_out", weight,
                   *(t for t in (x, residual) if t.dtype != residual.dtype
                     or t.data_ptr() != residual_out.data_ptr()))
    elif residual_out is not None:
        raise ContractError("residual_out comes with a residual")
    codes, scales = _coded_out(out, x, T, d, dev, x, weight, residual, residual_out)
    if T:
        _run(dev, "glm_add_rms_norm_fp8", N.native.load().glm_add_rms_norm_fp8, x.data_ptr(), kind,
             None if residual is None else residual.data_ptr(), rkind, T, d,
             None if weight is None else weight.data_ptr(), eps,
             None if residual is None else residual_out.data_ptr(), codes.data_ptr(),
             scales.data_ptr())
    return Fp8Rows(codes, scales), residual_out


def linear(x: torch.Tensor | Fp8Rows, weight: torch.Tensor, scales: torch.Tensor, *,
           out: torch.Tensor | None = None) -> torch.Tensor:
    """bf16 ``[..., N]`` of ``x @ weight.T``; bf16 and f32 rows are quantised as
    ``quantize_rows`` does.  K is a multiple of 16.  Up to 64 rows the products
    within a group are summed in f32; more rows go through the 8-bit matrix
    instruction, which drops what lies 2^-13 below the largest of eight products
    (1.5e-5 of the sum, where bf16 rounds by up to 2^-8)."""
    dev, kind, T, K, rows, row_scales, lead = _rows(x)
    n = _weight(weight, scales, "weight", K, dev)
    if out is not None:
        _given(out, "out", (*lead.shape[:-1], n), _BF16, dev)
        _apart(out, "out", weight, scales, *(x if kind == _CODED else (x,)))
    elif len(lead.shape) == 2:
        out = _empty(T, n, dtype=_BF16, device=lead.device)
    else:
        out = _empty((*lead.shape[:-1], n), dtype=_BF16, device=lead.device)
    if T:
        need = _workspace_bytes(kind, T, K, n, 0)
        ws = _empty(need, dtype=_U8, device=lead.device) if need else None
        _run(dev, "glm_fp8_linear", N.native.load().glm_fp8_linear, rows, kind, row_scales, T, K,
             weight.data_ptr(), scales.data_ptr(), n, ws.data_ptr() if need else None, need,
             out.data_ptr())
    return out


def gate_up(x: torch.Tensor | Fp8Rows, gate: torch.Tensor, gate_scales: torch.Tensor,
            up: torch.Tensor, up_scales: torch.Tensor, limit: float, *,
            out: Fp8Rows | None = None) -> Fp8Rows:
    """Quantised ``silu(g) * u`` of ``g = x @ gate.T`` and ``u = x @ up.T``,
    both weights ``[I, K]``, I a multiple of 16; with ``limit > 0`` g is cut at
    ``limit`` and u at both ends.  f32 until the codes."""
    dev, kind, T, K, rows, row_scales, lead = _rows(x)
    n = _weight(gate, gate_scales, "gate", K, dev)
    if _weight(up, up_scales, "up", K, dev) != n:
        raise ContractError(f"gate {tuple(gate.shape)} and up {tuple(up.shape)} differ")
    codes, scales = _coded_out(out, lead, T, n, dev, gate, gate_scales, up, up_scales,
                               *(x if kind == _CODED else (x,)))
    if T:
        need = _workspace_bytes(kind, T, K, n, 1)
        ws = _empty(need, dtype=_U8, device=lead.device) if need else None
        _run(dev, "glm_fp8_gate_up", N.native.load().glm_fp8_gate_up, rows, kind, row_scales, T, K,
             gate.data_ptr(), gate_scales.data_ptr(), up.data_ptr(), up_scales.data_ptr(), n,
             limit, ws.data_ptr() if need else None, need, codes.data_ptr(), scales.data_ptr())
    return Fp8Rows(codes, scales)


__all__ = ["Fp8Rows", "GROUP", "add_rms_norm", "gate_up", "linear", "quantize_rows",
           "quantize_weight"]
