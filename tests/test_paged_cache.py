"""The paged attention cache on the host: the oracle against plain statements,
and every refusal of the C ABI and of the Python entry points (nothing here
reaches a GPU)."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from livglm_amd import native
from oracle import paged_oracle as P

FAKE = ctypes.c_void_p(0x10000)  # never dereferenced: validation fails first
ODD = ctypes.c_void_p(0x10004)


# ---------------------------------------------------------------- the oracle

def test_oracle_step_keeps_every_page_once():
    rng = np.random.default_rng(5)
    B, page, width, pool = 7, 4, 12, 60
    lens, blocks = np.zeros(B, int), np.zeros(B, int)
    tables, free, top = np.full((B, width), -1, np.int32), np.arange(pool)[::-1].astype(np.int32), pool
    for _ in range(60):
        new = rng.integers(-9, 9, B)
        r = P.step(new, lens, blocks, tables, free, top, page, 80)
        if r["status"]:
            new = np.full(B, -1)  # all over
            r = P.step(new, lens, blocks, tables, free, top, page, 80)
        assert r["status"] == 0
        lens, blocks, tables, free, top = (r[k] for k in ("kv_lens", "blocks", "tables", "free_pages", "num_free"))
        held = [tables[b, j] for b in range(B) for j in range(blocks[b])]
        assert sorted(held + list(free[:top])) == list(range(pool))
        assert (blocks * page >= lens).all()
        used = r["slots"][: r["cu_new"][-1]]
        assert len(set(used)) == len(used) and (used >= 0).all()
        assert (r["slots"][r["cu_new"][-1]:] == -1).all()


def test_oracle_mx_rows_are_the_nearest_codes():
    rng = np.random.default_rng(6)
    x = (rng.standard_normal((9, 64)) * np.exp2(rng.integers(-140, 120, (9, 1)))).astype(np.float32)
    x = P.bf16_bits_to_f32((x.view(np.uint32) >> 16).astype(np.uint16)).astype(np.float64)
    x[0], x[1, 3], x[1, 40], x[2, :32] = 0, np.nan, -np.inf, 448.0
    codes, scales = P.mx_rows(x)
    assert (scales >= 3).all()
    v = P.mx_values(codes, scales)
    fine = np.isfinite(x)
    assert np.isnan(v[~fine]).all()
    step = np.maximum(np.exp2(scales.astype(float) - 127 - 9).repeat(32, -1), np.abs(x) / 8)
    assert (np.abs(v - x)[fine] <= 0.5 * step[fine] * (1 + 1e-12)).all()
    assert (scales[2, 0] - 127, codes[2, 0]) == (0, 0x7e)


# ---------------------------------------------------------------- the C ABI's refusals

def _step_args(**kw):
    a = dict(stream=None, new=FAKE, B=2, num_pages=8, page=16, max_blocks=4, max_tokens=8, lens=FAKE, blocks=FAKE,
             tables=FAKE, free=FAKE, num_free=FAKE, kv=FAKE, cu=FAKE, slots=FAKE, positions=FAKE, status=FAKE)
    a.update(kw)
    return list(a.values())


def _write_args(**kw):
    a = dict(stream=None, keys=FAKE, ks=256, values=FAKE, vs=256, slots=FAKE, N=2, num_pages=8, page=16, heads=2,
             dk=128, dv=128, fmt=native.GLM_FMT_BF16, kc=FAKE, ksc=None, vc=FAKE, vsc=None)
    a.update(kw)
    return list(a.values())


def _attend_args(**kw):
    a = dict(stream=None, q=FAKE, qs=1024, B=2, q_len=1, heads=8, kv_heads=2, dk=128, dv=128, kc=FAKE, ksc=None,
             vc=FAKE, vsc=None, fmt=native.GLM_FMT_BF16, num_pages=8, page=16, tables=FAKE, lens=FAKE, max_blocks=4,
             scale=0.1, ws=FAKE, nbytes=1 << 30, out=FAKE)
    a.update(kw)
    return list(a.values())


INVALID, SHAPE, WORKSPACE = (native.GLM_ERR_INVALID_ARGUMENT, native.GLM_ERR_UNSUPPORTED_SHAPE,
                             native.GLM_ERR_WORKSPACE)


@pytest.mark.parametrize("code, change", [
    *[(INVALID, {k: None}) for k in ("new", "lens", "blocks", "tables", "free", "num_free", "kv", "cu", "slots",
                                     "positions", "status")],
    (INVALID, {"B": 0}), (INVALID, {"B": -1}), (SHAPE, {"B": 4097}), (INVALID, {"num_pages": 0}),
    (INVALID, {"page": 0}), (INVALID, {"max_blocks": 0}), (INVALID, {"max_tokens": -1}),
    (SHAPE, {"max_tokens": (1 << 30) + 1}),
    (SHAPE, {"num_pages": 1 << 27}), (SHAPE, {"max_blocks": 1 << 27}),
])
def test_step_refusals(code, change):
    assert native.load().glm_cache_step(*_step_args(**change)) == code
    assert native.load().glm_last_error()


@pytest.mark.parametrize("code, change", [
    *[(INVALID, {k: None}) for k in ("keys", "slots", "kc", "values", "vc")],
    (INVALID, {"fmt": native.GLM_FMT_MXFP4}), (INVALID, {"fmt": native.GLM_FMT_MXFP8}),
    (INVALID, {"fmt": native.GLM_FMT_MXFP8, "ksc": FAKE}), (INVALID, {"N": -1}), (INVALID, {"page": 0}),
    (SHAPE, {"dk": 100}), (SHAPE, {"dv": 4}), (SHAPE, {"dk": 2048, "ks": 4096}), (INVALID, {"ks": 255}),
    (INVALID, {"ks": 260}), (INVALID, {"vs": 248}), (INVALID, {"keys": ODD}), (INVALID, {"vc": ODD}),
    (SHAPE, {"N": (1 << 30) + 1}), (SHAPE, {"heads": 65537, "ks": 1 << 24, "vs": 1 << 24}),
    (SHAPE, {"dk": 40, "fmt": native.GLM_FMT_MXFP8, "ksc": FAKE, "vsc": FAKE}),
    (SHAPE, {"num_pages": 1 << 27}),
])
def test_write_refusals(code, change):
    assert native.load().glm_cache_write(*_write_args(**change)) == code
    assert native.load().glm_last_error()


@pytest.mark.parametrize("code, change", [
    *[(INVALID, {k: None}) for k in ("q", "kc", "tables", "lens", "ws", "out")],
    (INVALID, {"fmt": native.GLM_FMT_MXFP4}), (INVALID, {"fmt": native.GLM_FMT_MXFP8}),
    (INVALID, {"fmt": native.GLM_FMT_MXFP8, "ksc": FAKE}), (INVALID, {"B": -1}), (INVALID, {"q_len": 0}),
    (SHAPE, {"q_len": 17}), (SHAPE, {"heads": 7}), (SHAPE, {"heads": 2048, "qs": 1 << 18}), (SHAPE, {"B": 65536}),
    (SHAPE, {"dk": 100}), (SHAPE, {"dv": 1032}), (SHAPE, {"vc": None, "dv": 136}), (INVALID, {"qs": 1016}),
    (INVALID, {"qs": 1028}), (INVALID, {"scale": float("nan")}), (INVALID, {"scale": float("inf")}),
    (INVALID, {"q": ODD}), (INVALID, {"out": ODD}), (INVALID, {"ws": ODD}), (WORKSPACE, {"nbytes": 16}),
    (SHAPE, {"num_pages": 1 << 27}), (SHAPE, {"max_blocks": 1 << 27}), (INVALID, {"max_blocks": 0}),
    (SHAPE, {"max_blocks": (1 << 27) - 64}),
])
def test_attend_refusals(code, change):
    assert native.load().glm_paged_attention(*_attend_args(**change)) == code
    assert native.load().glm_last_error()


REASONS = [({"q_len": 17}, "16 new tokens"), ({"heads": 7}, "multiple of the kv heads"),
           ({"heads": 2048, "qs": 1 << 18}, "1024 heads"), ({"B": 65536}, "65535 requests"), ({"dk": 100}, "multiples of 8"),
           ({"dv": 1032}, "up to 1024"), ({"vc": None, "dv": 136}, "value channels"),
           ({"max_blocks": 1 << 27}, "pass 32 bits"), ({"B": 4096, "heads": 128, "kv_heads": 128, "qs": 1 << 14,
                                                        "max_blocks": 8192}, "tiles of all requests")]


@pytest.mark.parametrize("change, why", REASONS)
def test_attend_says_why(change, why):
    """A refused size has no workspace, and its reason comes before the workspace's null pointer."""
    a = _attend_args(**change)
    size = native.load().glm_paged_attention_workspace_bytes
    latent = int(change.get("vc", FAKE) is None)
    assert size(*a[3:9], latent, a[15], a[18]) == 0
    for ws in (FAKE, None):
        assert native.load().glm_paged_attention(*_attend_args(**{**change, "ws": ws, "nbytes": 0})) == SHAPE
        assert why in native.load().glm_last_error().decode()


def test_step_says_why():
    for change, why in (({"num_pages": 0, "free": None}, "sizes"), ({"max_blocks": 0, "tables": None}, "sizes"),
                        ({"B": 4097, "new": None}, "4096")):
        assert native.load().glm_cache_step(*_step_args(**change)) in (INVALID, SHAPE)
        assert why in native.load().glm_last_error().decode()


def test_attend_table_limit():
    """Requests x kv heads x tiles of the tables' width: the documented bound is taken, just beyond it is not."""
    size = native.load().glm_paged_attention_workspace_bytes
    for heads, dk, dv, latent in ((128, 128, 128, 0), (128, 96, 96, 0), (1, 576, 512, 1)):
        kv = 1 if latent else heads
        B = 65535 if latent else 4096
        tiles = (1 << 30) // (B * kv)
        assert size(B, 1, heads, kv, dk, dv, latent, 64, tiles - 4) > 0  # B kv (tiles - 4 + 3) < 2^30
        assert size(B, 1, heads, kv, dk, dv, latent, 64, tiles + 1) == 0


def test_attend_workspace():
    size = native.load().glm_paged_attention_workspace_bytes
    need = size(2, 1, 8, 2, 128, 128, 0, 16, 4)
    assert need > 0
    assert native.load().glm_paged_attention(*_attend_args(nbytes=need - 1 - 256)) == WORKSPACE
    assert size(2, 1, 7, 2, 128, 128, 0, 16, 4) == 0 and size(-1, 1, 8, 2, 128, 128, 0, 16, 4) == 0
    assert size(1, 1, 8, 2, 128, 128, 0, 16, (1 << 27) - 64) == 0 < size(1, 1, 8, 2, 128, 128, 0, 16, (1 << 27) - 65)
    # bounded by the work that the chip takes at once, not by the batch
    assert 0 < size(4096, 1, 128, 8, 128, 128, 0, 16, 8192) < 512 << 20
    assert 0 < size(4096, 2, 128, 1, 576, 512, 1, 64, 2048) < 512 << 20


def test_empty_batches_are_no_ops():
    assert native.load().glm_cache_write(*_write_args(N=0)) == native.GLM_OK
    assert native.load().glm_paged_attention(*_attend_args(B=0)) == native.GLM_OK


# ---------------------------------------------------------------- the Python refusals

def test_python_refuses_host_tensors():
    from glm53flash import paged_cache as C
    from glm53flash.contract import ContractError
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ContractError):
        C.cache_step(i, i, i, i.view(1, 4), i, i[:1], page_size=4, max_tokens=4)
    x, cache = torch.zeros(4, 2, 64, dtype=torch.bfloat16), torch.zeros(4, 2, 8, 64, dtype=torch.bfloat16)
    with pytest.raises(ContractError):
        C.cache_write(x, x, i, cache, cache)
    with pytest.raises(ContractError):
        C.paged_attention(x, cache, cache, i.view(4, 1), i, scale=1.0)


def test_python_objects():
    from glm53flash import paged_cache as C
    from glm53flash.contract import ContractError
    from glm53flash.model_config import GLMTextConfig
    table = C.PageTable(8, 16, 4, 6, device="cpu")
    assert table.free_pages.tolist() == list(range(7, -1, -1)) and table.num_free.item() == 8
    cfg = GLMTextConfig(kv_lora_rank=512, qk_rope_head_dim=64)
    cache = C.PagedKVCache.from_config(cfg, table, quantization_mode="mxfp8")
    assert cache.keys.shape == (8, 1, 16, 576) and cache.key_scales.shape == (8, 1, 16, 18)
    assert cache.latent and cache.values is None and cache.value_dim == 512
    cfg = GLMTextConfig(num_key_value_heads=2, qk_nope_head_dim=64, qk_rope_head_dim=64, v_head_dim=96)
    cache = C.PagedKVCache.from_config(cfg, table)
    assert cache.keys.shape == (8, 2, 16, 128) and cache.values.shape == (8, 2, 16, 96)
    with pytest.raises(ContractError):
        C.PagedKVCache.from_config(GLMTextConfig(), table)
    moe = {"hidden_size": 64, "moe_intermediate_size": 64, "n_routed_experts": 8, "num_experts_per_tok": 2,
           "n_shared_experts": 1, "n_group": 1, "topk_group": 1, "routed_scaling_factor": 1.0}
    read = GLMTextConfig.from_model_dict
    cache = C.PagedKVCache.from_config(read({**moe, "kv_lora_rank": 256, "qk_rope_head_dim": 64}), table)
    assert cache.latent and cache.keys.shape == (8, 1, 16, 320) and cache.value_dim == 256
    cache = C.PagedKVCache.from_config(read({**moe, "kv_lora_rank": None, "num_key_value_heads": 4,
                                             "qk_nope_head_dim": 96, "qk_rope_head_dim": 32, "v_head_dim": 64}), table)
    assert cache.keys.shape == (8, 4, 16, 128) and cache.values.shape == (8, 4, 16, 64)
    with pytest.raises(ContractError):
        C.PagedKVCache.from_config(read(moe), table)
    with pytest.raises(ContractError):
        C.PagedKVCache(table, 1, 64, 128, latent=True)
    with pytest.raises(ContractError):
        C.PagedKVCache(table, 1, 72, 72, quantization_mode="mxfp8")
    with pytest.raises(ContractError):
        C.PagedKVCache(table, 1, 64, 64, quantization_mode="int8")
    with pytest.raises(ContractError):
        C.PageTable(0, 16, 4, 6, device="cpu")


def test_token_rows_strides():
    from glm53flash.contract import ContractError
    from glm53flash import paged_cache as C
    qkv = torch.zeros(6, 10, 64, dtype=torch.bfloat16, device="meta")

    class OnGpu:  # the check reads shapes and strides alone
        def __init__(self, t):
            self.shape, self.dtype, self.is_cuda, self.device = t.shape, t.dtype, True, "cuda"
            self.stride, self.is_contiguous = t.stride, t.is_contiguous

    def rows(t):
        real, torch.Tensor_ = torch.Tensor, None
        try:
            C.torch = type("T", (), {"Tensor": (OnGpu, real), "bfloat16": torch.bfloat16})
            return C._token_rows(OnGpu(t), "t")
        finally:
            C.torch = torch
            del torch.Tensor_

    assert rows(qkv[:, 2:6]) == 640
    assert rows(qkv[:1, 2:6]) == 256
    assert rows(qkv.view(3, 2, 10, 64)[:, :, :4]) == 640
    assert rows(qkv.view(3, 2, 10, 64)[:, :1, :4]) == 1280
    assert rows(qkv.view(3, 2, 10, 64)[:1, :, :4]) == 640
    for bad in (qkv.transpose(1, 2), qkv[:, ::2], qkv.view(2, 3, 10, 64)[:, :2], qkv[0]):
        with pytest.raises(ContractError):
            rows(bad)


MOE = {"hidden_size": 64, "moe_intermediate_size": 64, "n_routed_experts": 8, "num_experts_per_tok": 2,
       "n_shared_experts": 1, "n_group": 1, "topk_group": 1, "routed_scaling_factor": 1.0}
HEADS = {"num_attention_heads": 8, "num_key_value_heads": 2, "qk_nope_head_dim": 64, "qk_rope_head_dim": 64,
         "v_head_dim": 96}


@pytest.mark.parametrize("value", ["4", "auto", [4, 8], True, 4.0, 1.5, -4, {}, float("nan")])
@pytest.mark.parametrize("key", ["num_key_value_heads", "qk_nope_head_dim", "qk_rope_head_dim", "v_head_dim",
                                 "kv_lora_rank"])
def test_mistyped_head_sizes(key, value):
    """The FFN site's configuration does not depend on the attention's sizes; the cache refuses what is no size."""
    from glm53flash import paged_cache as C
    from glm53flash.contract import ContractError
    from glm53flash.model_config import GLMTextConfig
    cfg = GLMTextConfig.from_model_dict({**MOE, **HEADS, key: value})
    assert cfg.hidden_size == 64 and hash(cfg) == hash(cfg)
    table = C.PageTable(8, 16, 4, 6, device="cpu")
    with pytest.raises(ContractError, match=key):
        C.PagedKVCache.from_config(cfg, table)
    with pytest.raises(ContractError):
        C.PagedKVCache.from_config(GLMTextConfig(**{**HEADS, key: value}), table)


def test_head_counts_of_none():
    from glm53flash import paged_cache as C
    from glm53flash.contract import ContractError
    from glm53flash.model_config import GLMTextConfig
    with pytest.raises(ContractError):
        C.PagedKVCache.from_config(GLMTextConfig.from_model_dict({**MOE, **HEADS, "num_key_value_heads": 0}),
                                   C.PageTable(8, 16, 4, 6, device="cpu"))


@pytest.mark.parametrize("change, heads", [({}, 2), ({"num_key_value_heads": None}, 8), ({"num_key_value_heads": 8}, 8),
                                           ({"num_key_value_heads": None, "num_attention_heads": 12}, 12)])
def test_unstated_kv_heads(change, heads):
    """A configuration without a kv head count has one kv head for each head."""
    from glm53flash import paged_cache as C
    from glm53flash.model_config import GLMTextConfig
    table = C.PageTable(8, 16, 4, 6, device="cpu")
    text = {**MOE, **HEADS, **change}
    cache = C.PagedKVCache.from_config(GLMTextConfig.from_model_dict(text), table)
    assert cache.keys.shape == (8, heads, 16, 128) and cache.values.shape == (8, heads, 16, 96)
    if text["num_key_value_heads"] is None:
        del text["num_key_value_heads"]
        assert C.PagedKVCache.from_config(GLMTextConfig.from_model_dict(text), table).kv_heads == heads


@pytest.mark.parametrize("heads", ["8", None])
def test_no_head_count_for_kv_heads(heads):
    from glm53flash import paged_cache as C
    from glm53flash.contract import ContractError
    from glm53flash.model_config import GLMTextConfig
    text = {**MOE, **HEADS, "num_key_value_heads": None, "num_attention_heads": heads}
    with pytest.raises(ContractError):
        C.PagedKVCache.from_config(GLMTextConfig.from_model_dict(text), C.PageTable(8, 16, 4, 6, device="cpu"))


@pytest.mark.parametrize("topk, taken", [(None, True), (1, True), (96, True), (2048, True), (95, False), (64, False),
                                         ("96", False), (-1, False)])
@pytest.mark.parametrize("latent", [False, True])
def test_dense_up_to_index_topk(topk, taken, latent):
    """A table of 96 positions a request, and models that select as many, more or fewer."""
    from glm53flash import paged_cache as C
    from glm53flash.contract import ContractError
    from glm53flash.model_config import GLMTextConfig
    table = C.PageTable(8, 16, 4, 6, device="cpu")
    text = {**MOE, **HEADS, "kv_lora_rank": 256 if latent else None, "index_topk": topk}
    cfg = GLMTextConfig.from_model_dict(text)
    if taken:
        assert C.PagedKVCache.from_config(cfg, table).latent == latent
    else:
        with pytest.raises(ContractError, match="index_topk"):
            C.PagedKVCache.from_config(cfg, table)


@pytest.mark.parametrize("thing", [None, [1, 2], np.zeros(4, np.int32), 5, torch.int32, torch.zeros(4, dtype=torch.int32)])
def test_python_refuses_what_is_no_tensor(thing):
    from glm53flash import paged_cache as C
    from glm53flash.contract import ContractError
    with pytest.raises(ContractError, match="lens"):
        C._check(thing, "lens", torch.int32, 0)
    with pytest.raises(ContractError, match="key_cache"):
        C._cache_format(thing, None, "key_cache", 0)


def test_head_sizes_of_other_integer_types():
    from glm53flash import paged_cache as C
    from glm53flash.model_config import GLMTextConfig
    table = C.PageTable(8, 16, 4, 6, device="cpu")
    cfg = GLMTextConfig(num_key_value_heads=np.int64(2), qk_nope_head_dim=np.int32(64), v_head_dim=np.int64(32))
    assert C.PagedKVCache.from_config(cfg, table).values.shape == (8, 2, 16, 32)
