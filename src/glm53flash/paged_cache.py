"""The attention's cache for a batch of requests, in pages.

The reference serves one request and keeps its history in arrays that grow
(``cache.py:53-103``).  Here a pool of pages serves many:

* ``cache_step`` takes and gives back pages from the requests' lengths, on the
  GPU, and says where each new token goes;
* ``cache_write`` puts the new tokens' keys and values (or latent rows) there,
  as bf16 or as group-32 MXFP8;
* ``paged_attention`` is the attention of the newest token of each request, or
  of the few of a verify step, over its history.

They work on the caller's tensors, on the current stream of those tensors'
device, without host synchronisation, and may be captured in a HIP graph.
``PageTable`` and ``PagedKVCache`` keep the tensors: one table for a model, one
cache for each of its layers.

Cache tensors are ``[pages, kv_heads, page_size, dim]``; a slot is ``page *
page_size + offset``.
"""

from __future__ import annotations

from functools import lru_cache
from numbers import Integral
from typing import NamedTuple

import torch

from . import _native as N
from .contract import ContractError
from .model_config import GLMTextConfig

OUT_OF_PAGES = N.native.GLM_CACHE_OUT_OF_PAGES
TABLE_FULL = N.native.GLM_CACHE_TABLE_FULL
TOO_MANY_TOKENS = N.native.GLM_CACHE_TOO_MANY_TOKENS
BAD_STATE = N.native.GLM_CACHE_BAD_STATE

_BF16, _U8, _I32 = torch.bfloat16, torch.uint8, torch.int32


# The calls here are a few microseconds of GPU work each, so what the host does
# before them counts: devices are compared as numbers, and the library's
# functions are called without a wrapper in between.
_getDevice = torch._C._cuda_getDevice
_getStream = torch._C._cuda_getCurrentRawStream
_empty = torch.empty


def _check(t: torch.Tensor, name: str, dtype: torch.dtype, device: int) -> None:
    """A contiguous tensor of the call's device and the dtype it has to have."""
    try:  # (no call beside those that a tensor needs)
        fine = t.dtype is dtype and t.get_device() == device and t.is_contiguous()
    except AttributeError:  # no tensor
        fine = False
    if not fine:
        N.require_device(t, name, (dtype,))
        raise ContractError(f"{name} is on {t.device}, the call's tensors on device {device}")


def _token_rows(t: torch.Tensor, name: str) -> int:
    """The elements from token to token of ``[..., heads, dim]`` rows whose heads
    lie together (a slice of a fused projection, or a contiguous tensor)."""
    if not isinstance(t, torch.Tensor):
        raise ContractError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ContractError(f"{name} must live on the GPU (got {t.device})")
    if t.dtype is not _BF16:
        raise ContractError(f"{name} has dtype {t.dtype}, expected {_BF16}")
    shape = t.shape
    dims = len(shape)
    if dims != 3 and dims != 4:
        raise ContractError(f"{name} must be [tokens, heads, dim] rows, got {tuple(shape)}")
    row = shape[-1] * shape[-2]
    if t.is_contiguous():
        return row
    stride = t.stride()
    if stride[-1] != 1 and shape[-1] != 1 or stride[-2] != shape[-1] and shape[-2] != 1:
        raise ContractError(f"{name}: a token's heads must lie together, strides {stride}")
    if len(shape) == 4 and stride[0] != shape[1] * stride[1] and shape[0] != 1 and shape[1] != 1:
        raise ContractError(f"{name}: the tokens must lie at one stride, strides {stride}")
    if len(shape) == 4 and shape[1] > 1:  # (the stride of an axis of one says nothing)
        return stride[1]
    return stride[0] if shape[0] > 1 else row


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


def _cache_format(cache: torch.Tensor, scales: torch.Tensor | None, name: str, device: int) -> int:
    if scales is None:
        _check(cache, name, _BF16, device)
        if cache.dim() != 4:
            raise ContractError(f"{name} must be [pages, kv_heads, page_size, dim], got "
                                f"{tuple(cache.shape)}")
        return N.FMT_BF16
    _check(cache, name, _U8, device)
    _check(scales, f"{name} scales", _U8, device)
    shape = cache.shape
    if len(shape) != 4 or shape[3] % 32 or scales.shape != (*shape[:3], shape[3] // 32):
        raise ContractError(f"{name} scales {tuple(scales.shape)} do not fit codes {tuple(shape)}")
    return N.FMT_MXFP8


class CacheStep(NamedTuple):
    """What a step gives: lengths after it, sums of the new tokens, each token
    row's slot (-1 past the last, and where its table entry is no page of the
    cache) and position, and the status (0, or the ``OUT_OF_PAGES`` ... bits,
    with which nothing has changed)."""

    kv_lens: torch.Tensor
    cu_new: torch.Tensor
    slots: torch.Tensor
    positions: torch.Tensor
    status: torch.Tensor


def cache_step(new_lens: torch.Tensor, lens: torch.Tensor, blocks: torch.Tensor,
               tables: torch.Tensor, free_pages: torch.Tensor, num_free: torch.Tensor, *,
               page_size: int, max_tokens: int, kv_lens: torch.Tensor | None = None) -> CacheStep:
    """Pages for ``new_lens`` i32 ``[B]`` more tokens of the first ``B`` requests.

    ``n >= 0`` appends ``n`` tokens; ``-1 - n`` gives the request's pages back
    and starts a new request of ``n`` tokens.  ``lens`` i32 ``[B]`` is read;
    ``blocks`` ``[B]``, ``tables`` ``[B, max_blocks]``, ``free_pages``
    ``[pages]`` and ``num_free`` ``[1]`` (all i32) are the state, updated in
    place.  ``kv_lens`` (allocated when not given; may be ``lens``) receives the
    lengths after the step.  Slots and positions have ``max_tokens`` rows.
    """
    dev = new_lens.get_device() if isinstance(new_lens, torch.Tensor) else -1
    if dev < 0:
        N.require_device(new_lens, "new_lens", (_I32,))
    _check(new_lens, "new_lens", _I32, dev)
    _check(lens, "lens", _I32, dev)
    _check(blocks, "blocks", _I32, dev)
    _check(tables, "tables", _I32, dev)
    _check(free_pages, "free_pages", _I32, dev)
    _check(num_free, "num_free", _I32, dev)
    B = new_lens.numel()
    shape = tables.shape
    if len(shape) != 2 or shape[0] < B or lens.numel() < B or blocks.numel() < B:
        raise ContractError(f"cache_step: {B} requests, tables {tuple(tables.shape)}, "
                            f"{lens.numel()} lens and {blocks.numel()} blocks")
    if num_free.numel() != 1:
        raise ContractError("cache_step: num_free must have one element")
    if not 0 <= max_tokens <= 1 << 30 or not 1 <= page_size < 1 << 31:
        raise ContractError(f"cache_step: max_tokens {max_tokens} or page_size {page_size}")
    if kv_lens is not None:
        _check(kv_lens, "kv_lens", _I32, dev)
        if kv_lens.numel() < B:
            raise ContractError(f"cache_step: kv_lens for {kv_lens.numel()} of {B} requests")
    if (B | shape[1] | free_pages.numel()) >> 31:  # (the library's sizes are 32-bit: none may wrap)
        raise ContractError(f"cache_step: {free_pages.numel()} pages or {shape[1]} blocks a request "
                            "pass 32 bits")
    # one allocation: cu_new | status | slots | positions | kv_lens
    if kv_lens is None:
        buf = _empty(2 * B + 2 + 2 * max_tokens, dtype=_I32, device=new_lens.device)
        cu, status, slots, positions, kv_lens = buf.split_with_sizes(
            (B + 1, 1, max_tokens, max_tokens, B))
    else:
        buf = _empty(B + 2 + 2 * max_tokens, dtype=_I32, device=new_lens.device)
        cu, status, slots, positions = buf.split_with_sizes((B + 1, 1, max_tokens, max_tokens))
    if B == 0:  # no request: no token either, and the state stays as it is
        buf.zero_()
        slots.fill_(-1)
        return CacheStep(kv_lens, cu, slots, positions, status)
    base = buf.data_ptr()
    _run(dev, "glm_cache_step", N.native.load().glm_cache_step, new_lens.data_ptr(), B,
         free_pages.numel(), page_size, shape[1], max_tokens, lens.data_ptr(),
         blocks.data_ptr(), tables.data_ptr(), free_pages.data_ptr(), num_free.data_ptr(),
         kv_lens.data_ptr(), base, base + 4 * (B + 2), base + 4 * (B + 2 + max_tokens),
         base + 4 * (B + 1))
    return CacheStep(kv_lens, cu, slots, positions, status)


def cache_write(keys: torch.Tensor, values: torch.Tensor | None, slots: torch.Tensor,
                key_cache: torch.Tensor, value_cache: torch.Tensor | None, *,
                key_scales: torch.Tensor | None = None,
                value_scales: torch.Tensor | None = None) -> None:
    """Writes rows ``keys`` ``[N, kv_heads, key_dim]`` and ``values`` ``[N,
    kv_heads, value_dim]`` (bf16; slices of a fused projection are taken as they
    are) to ``slots`` i32 ``[N]``; a slot outside the cache is skipped.  Two
    tokens with one slot leave a mixture of both rows there.
    ``values`` and ``value_cache`` are None for a latent cache.  With scales the
    caches are MXFP8."""
    key_stride = _token_rows(keys, "keys")
    dev = keys.get_device()
    fmt = _cache_format(key_cache, key_scales, "key_cache", dev)
    _check(slots, "slots", _I32, dev)
    pages, heads, page, key_dim = key_cache.shape
    n = slots.numel()
    if keys.shape != (n, heads, key_dim):
        raise ContractError(f"keys {tuple(keys.shape)} do not fit {n} slots of a cache "
                            f"{tuple(key_cache.shape)}")
    if (values is None) != (value_cache is None) or values is None and value_scales is not None:
        raise ContractError("values and value_cache come together")
    value_stride = value_dim = 0
    if values is not None:
        value_stride = _token_rows(values, "values")
        if _cache_format(value_cache, value_scales, "value_cache", dev) != fmt:
            raise ContractError("key_cache and value_cache must share one format")
        value_dim = value_cache.shape[3]
        if value_cache.shape[:3] != key_cache.shape[:3] or \
                values.shape != (n, heads, value_dim) or values.get_device() != dev:
            raise ContractError(f"values {tuple(values.shape)} and value_cache "
                                f"{tuple(value_cache.shape)} do not fit the keys")
    if n == 0:
        return
    if (n | pages | heads | page | key_dim | value_dim) >> 31:
        raise ContractError(f"cache_write: {n} slots or a cache {tuple(key_cache.shape)} pass 32 bits")
    _run(dev, "glm_cache_write", N.native.load().glm_cache_write, keys.data_ptr(), key_stride,
         N.ptr(values), value_stride, slots.data_ptr(), n, pages, page, heads, key_dim, value_dim,
         fmt, key_cache.data_ptr(), N.ptr(key_scales), N.ptr(value_cache), N.ptr(value_scales))


@lru_cache(maxsize=256)  # a function of the sizes alone
def _attention_workspace(B: int, q_len: int, heads: int, kv_heads: int, key_dim: int,
                         value_dim: int, latent: int, page: int, max_blocks: int,
                         pages: int) -> int:
    if (B | q_len | heads | kv_heads | key_dim | value_dim | page | max_blocks | pages) >> 31:
        raise ContractError(f"paged_attention: {B} requests, {pages} pages of {page}, {max_blocks} "
                            "blocks a request or their widths pass 32 bits")
    return int(N.native.load().glm_paged_attention_workspace_bytes(
        B, q_len, heads, kv_heads, key_dim, value_dim, latent, page, max_blocks))


def paged_attention(query: torch.Tensor, key_cache: torch.Tensor,
                    value_cache: torch.Tensor | None, tables: torch.Tensor, lens: torch.Tensor, *,
                    scale: float, value_dim: int | None = None,
                    key_scales: torch.Tensor | None = None,
                    value_scales: torch.Tensor | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of ``query`` ``[B, heads, key_dim]`` (one new token a request)
    or ``[B, q_len, heads, key_dim]`` (its ``q_len`` newest) over the first
    ``lens`` i32 ``[B]`` positions that ``tables`` i32 ``[>= B, max_blocks]``
    names (all of them: no selection of positions is made); the newest tokens'
    own rows are in the cache and counted in ``lens``, and token ``t`` sees the
    positions below ``lens - (q_len - 1 - t)``.
    ``value_cache`` None: the values are the first ``value_dim`` channels of the
    key rows.  Returns bf16 of the query's shape with ``value_dim`` channels; a
    row that sees nothing gives zeros."""
    q_stride = _token_rows(query, "query")
    dev = query.get_device()
    shape = query.shape
    B, heads = shape[0], shape[-2]
    q_len = shape[1] if len(shape) == 4 else 1
    fmt = _cache_format(key_cache, key_scales, "key_cache", dev)
    _check(tables, "tables", _I32, dev)
    _check(lens, "lens", _I32, dev)
    pages, kv_heads, page, key_dim = key_cache.shape
    if shape[-1] != key_dim:
        raise ContractError(f"query rows of {shape[-1]} channels, keys of {key_dim}")
    rows = tables.shape
    if len(rows) != 2 or rows[0] < B or lens.numel() < B:
        raise ContractError(f"{B} requests, tables {tuple(tables.shape)} and {lens.numel()} lens")
    if value_cache is not None:
        if _cache_format(value_cache, value_scales, "value_cache", dev) != fmt:
            raise ContractError("key_cache and value_cache must share one format")
        if value_cache.shape[:3] != key_cache.shape[:3] or \
                value_dim not in (None, value_cache.shape[3]):
            raise ContractError(f"value_cache {tuple(value_cache.shape)} does not fit key_cache "
                                f"{tuple(key_cache.shape)}, value_dim {value_dim}")
        value_dim = value_cache.shape[3]
    elif value_dim is None or value_scales is not None:
        raise ContractError("a latent cache needs value_dim and has no value scales")
    if out is None:
        out = _empty((*shape[:-1], value_dim), dtype=_BF16, device=query.device)
    else:
        _check(out, "out", _BF16, dev)
        if out.shape != (*shape[:-1], value_dim):
            raise ContractError(f"out {tuple(out.shape)}, expected {(*shape[:-1], value_dim)}")
    if B == 0 or q_len == 0:
        return out
    max_blocks = rows[1]
    need = _attention_workspace(B, q_len, heads, kv_heads, key_dim, value_dim,
                                int(value_cache is None), page, max_blocks, pages)
    ws = _empty(need, dtype=_U8, device=query.device)
    _run(dev, "glm_paged_attention", N.native.load().glm_paged_attention, query.data_ptr(),
         q_stride, B, q_len, heads, kv_heads, key_dim, value_dim, key_cache.data_ptr(),
         N.ptr(key_scales), N.ptr(value_cache), N.ptr(value_scales), fmt, pages, page,
         tables.data_ptr(), lens.data_ptr(), max_blocks, scale, ws.data_ptr(), need,
         out.data_ptr())
    return out


class PageTable:
    """The pages of up to ``max_requests`` requests: one for a model, shared by
    the caches of its layers.  ``lens`` are the tokens that each request holds;
    a program that rejects new tokens (a verify step) lowers them in place."""

    def __init__(self, num_pages: int, page_size: int, max_requests: int, max_blocks: int,
                 device="cuda"):
        if min(num_pages, page_size, max_requests, max_blocks) < 1:
            raise ContractError("page table sizes must be positive")
        self.num_pages = num_pages
        self.page_size = page_size
        self.lens = torch.zeros(max_requests, dtype=_I32, device=device)
        self.blocks = torch.zeros(max_requests, dtype=_I32, device=device)
        self.tables = torch.full((max_requests, max_blocks), -1, dtype=_I32, device=device)
        # page 0 on top, so that a fresh table hands the pages out in order
        self.free_pages = torch.arange(num_pages - 1, -1, -1, dtype=_I32, device=device)
        self.num_free = torch.full((1,), num_pages, dtype=_I32, device=device)

    def step(self, new_lens: torch.Tensor, max_tokens: int) -> CacheStep:
        """``cache_step`` on this table; ``lens`` become the lengths after it."""
        return cache_step(new_lens, self.lens, self.blocks, self.tables, self.free_pages,
                          self.num_free, page_size=self.page_size, max_tokens=max_tokens,
                          kv_lens=self.lens)


class PagedKVCache:
    """One layer's cache in the pages of a ``PageTable``: bf16, or MXFP8 with
    ``quantization_mode="mxfp8"``.  ``value_dim`` channels of values beside the
    keys, or, with ``latent``, the first ``value_dim`` channels of the keys."""

    def __init__(self, table: PageTable, kv_heads: int, key_dim: int, value_dim: int, *,
                 latent: bool = False, quantization_mode: str | None = None):
        if quantization_mode not in (None, "mxfp8"):
            raise ContractError(f"unsupported cache quantization: {quantization_mode}")
        if latent and value_dim > key_dim:
            raise ContractError(f"{value_dim} value channels of {key_dim} key channels")
        self.table = table
        self.kv_heads = kv_heads
        self.key_dim = key_dim
        self.value_dim = value_dim
        self.latent = latent
        self.quantization_mode = quantization_mode
        self.keys, self.key_scales = self._empty(key_dim)
        self.values, self.value_scales = (None, None) if latent else self._empty(value_dim)

    def _empty(self, dim: int):
        shape = (self.table.num_pages, self.kv_heads, self.table.page_size)
        dev = self.table.lens.device
        if self.quantization_mode is None:
            return torch.empty((*shape, dim), dtype=_BF16, device=dev), None
        if dim % 32:
            raise ContractError(f"an MXFP8 cache needs widths in groups of 32, got {dim}")
        return (torch.empty((*shape, dim), dtype=_U8, device=dev),
                torch.empty((*shape, dim // 32), dtype=_U8, device=dev))

    @classmethod
    def from_config(cls, config: GLMTextConfig, table: PageTable, *,
                    quantization_mode: str | None = None) -> "PagedKVCache":
        """The cache of the configuration's attention: latent rows of
        ``kv_lora_rank + qk_rope_head_dim`` channels where it compresses keys
        and values, else ``num_key_value_heads`` heads.  Where the model selects
        ``index_topk`` positions (more than 1), the dense attention here is its
        own up to that many (``dsa.py:41-56``), and a table whose requests may
        grow longer is refused; the constructor takes any."""
        for name in ("kv_lora_rank", "num_key_value_heads", "qk_nope_head_dim", "qk_rope_head_dim",
                     "v_head_dim", "index_topk"):
            value = getattr(config, name)
            if isinstance(value, bool) or not isinstance(value, Integral) or value < 0:
                raise ContractError(f"configuration field must be a size: {name}")
        longest = table.tables.shape[1] * table.page_size
        if 1 < config.index_topk < longest:
            raise ContractError(f"requests of up to {longest} positions: beyond index_topk "
                                f"{config.index_topk} the model's attention is not dense")
        if config.kv_lora_rank > 0:
            return cls(table, 1, config.kv_lora_rank + config.qk_rope_head_dim,
                       config.kv_lora_rank, latent=True, quantization_mode=quantization_mode)
        key_dim = config.qk_nope_head_dim + config.qk_rope_head_dim
        if key_dim < 1 or config.v_head_dim < 1 or config.num_key_value_heads < 1:
            raise ContractError("the configuration has no attention head sizes")
        return cls(table, config.num_key_value_heads, key_dim, config.v_head_dim,
                   quantization_mode=quantization_mode)

    def write(self, keys: torch.Tensor, values: torch.Tensor | None, slots: torch.Tensor) -> None:
        cache_write(keys, values, slots, self.keys, self.values, key_scales=self.key_scales,
                    value_scales=self.value_scales)

    def attend(self, query: torch.Tensor, scale: float, lens: torch.Tensor | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """``paged_attention`` of the table's first requests; ``lens`` defaults
        to the table's."""
        return paged_attention(query, self.keys, self.values, self.table.tables,
                               self.table.lens if lens is None else lens, scale=scale,
                               value_dim=self.value_dim, key_scales=self.key_scales,
                               value_scales=self.value_scales, out=out)


__all__ = ["CacheStep", "PageTable", "PagedKVCache", "cache_step", "cache_write",
           "paged_attention", "OUT_OF_PAGES", "TABLE_FULL", "TOO_MANY_TOKENS", "BAD_STATE"]
