"""GPU tests of what the block-scaled products promise beyond a tolerance.

Exact sums within a group (up to 64 rows of ``linear``, every ``gate_up``): in
every eight channels two products are 448 x 448 and its negative and six are 1, 2
or 4.  All partial sums are whole numbers below 2^24, so that any order in f32
gives the whole sum; the 8-bit matrix instruction, which drops what lies 2^-13
below the largest of eight products (2^17 and more here, so below 2^3), gives
none of the six.  Scales are 1, 2 or 4.  Results are compared bit for bit: a
product's is rounded to bf16 once; a gate of 30 or more is its own silu in f32
(exp(-30) is below 2^-24), the product with the other half is rounded once, and
the quantiser is the oracle's.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import fp8_oracle as P

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def F():
    from glm53flash import fp8_block
    return fp8_block


def gpu(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def scales(rng, rows, K):
    return (2.0 ** rng.integers(0, 3, (rows, P.groups(K)))).astype(np.float32)


def values(rng, rows, K, big, small):
    """[rows, K]: of every eight channels, in an order that rng gives (the same
    for all rows), two with the values that big gives and six with small's."""
    v = np.empty((rows, K // 8, 8), np.float32)
    order = np.argsort(rng.random((K // 8, 8)), 1)
    full = np.concatenate([big((rows, K // 8)), small((rows, K // 8, 6))], 2)
    np.put_along_axis(v, np.broadcast_to(order, v.shape), full.astype(np.float32), 2)
    return v.reshape(rows, K)


def cancelling(seed, T, K, N, positive=False):
    """x [T, K] and a weight [N, K] whose large products cancel within eight channels."""
    small = lambda shape: np.random.default_rng(seed + 1).integers(1, 3, shape)
    x = values(np.random.default_rng(seed), T, K, lambda s: np.full((*s, 2), 448), small)

    def signed(shape):
        rng = np.random.default_rng(seed + 2)
        return rng.integers(1, 3, shape) * (1 if positive else rng.choice([-1, 1], shape))

    def pair(shape):
        sign = np.random.default_rng(seed + 3).choice([-448, 448], shape)
        return np.stack([sign, -sign], -1)

    return x, values(np.random.default_rng(seed), N, K, pair, signed)  # (the same order of channels)


def sums(x, xs, w, ws):
    a = x.astype(np.float64) * np.repeat(xs, P.GROUP, 1)[:, :x.shape[1]]
    b = w.astype(np.float64) * np.repeat(np.repeat(ws, P.GROUP, 0)[:w.shape[0]], P.GROUP, 1)[:, :x.shape[1]]
    return a @ b.T


def given(F, kind, x, xs):
    """The rows as the kernel gets them; bf16 and f32 ones, whose groups' largest
    magnitude is 448, with scales of 1."""
    if kind == "fp8":
        return F.Fp8Rows(gpu(P.encode(x)), gpu(xs)), xs
    return gpu(x, torch.bfloat16 if kind == "bf16" else None), np.ones_like(xs)


# by kernel: few rows; 16 x 16, 16 x 32, 32 x 32 and 16 x 64 features and rows
@pytest.mark.parametrize("kind, T, K, N", [
    ("fp8", 1, 272, 33), ("fp8", 8, 1040, 48), ("bf16", 1, 4096, 40), ("bf16", 16, 400, 40), ("f32", 3, 272, 40),
    ("f32", 16, 2048, 33), ("fp8", 13, 1040, 48), ("bf16", 40, 1024, 48), ("fp8", 49, 2064, 1040), ("f32", 64, 2064, 1040),
    ("fp8", 20, 144, 80), ("bf16", 64, 400, 4096), ("fp8", 49, 16400, 2064)])
def test_up_to_64_rows_are_summed_exactly(F, kind, T, K, N):
    x, w = cancelling(T + K, T, K, N)
    rng = np.random.default_rng(N)
    rows, xs = given(F, kind, x, scales(rng, T, K))
    ws = scales(rng, N, K)[::128]
    want = sums(x, xs, w, ws)
    assert np.abs(want).max() < 2 ** 24 and (np.abs(want) >= 8).mean() > 0.5
    got = F.linear(rows, gpu(P.encode(w)), gpu(ws))
    assert torch.equal(got, torch.from_numpy(want.astype(np.float32)).bfloat16().cuda())


# few rows; streamed 16 x 16 (split along K and whole), 16 x 32, 16 x 48, 32 x 32, 32 x 48, 32 x 64; tiles of
# 128 features and 64, 128 and 256 rows
@pytest.mark.parametrize("kind, T, K, N", [
    ("fp8", 1, 272, 48), ("fp8", 8, 2064, 96), ("bf16", 2, 2048, 272), ("bf16", 16, 400, 1040), ("f32", 5, 272, 144),
    ("fp8", 30, 4112, 80), ("fp8", 9, 272, 272), ("bf16", 64, 272, 1040), ("fp8", 100, 272, 1040), ("fp8", 150, 1040, 1040),
    ("f32", 256, 1040, 1040), ("fp8", 200, 1040, 2032), ("fp8", 100, 272, 2032), ("bf16", 600, 272, 4096),
    ("fp8", 1500, 272, 4096)])
def test_gated_pairs_are_summed_exactly(F, kind, T, K, N):
    x, g = cancelling(T + K, T, K, N, positive=True)
    u = cancelling(T + K, T, K, N)[1]
    rng = np.random.default_rng(N)
    rows, xs = given(F, kind, x, scales(rng, T, K))
    gs, us = (scales(rng, N, K)[::128] for _ in range(2))
    a, b = sums(x, xs, g, gs), sums(x, xs, u, us)
    assert a.min() >= 30 and max(a.max(), np.abs(b).max()) < 2 ** 24
    codes, want = P.quantize_rows(a.astype(np.float32) * b.astype(np.float32))
    got = F.gate_up(rows, gpu(P.encode(g)), gpu(gs), gpu(P.encode(u)), gpu(us), 0.0)
    assert torch.equal(got.scales, gpu(want))
    # (zeros of either sign are the same)
    assert torch.equal(got.codes.view(torch.float8_e4m3fn).float(), gpu(codes).view(torch.float8_e4m3fn).float())


@pytest.mark.parametrize("T", [1, 16, 64])
def test_the_exact_cases_tell_the_sums_apart(F, T):
    # the same rows among more than 64, by the 8-bit instruction: all six products of an eight are gone
    K, N = 1040, 48
    x, w = cancelling(T, 65, K, N)
    rows, ws = F.Fp8Rows(gpu(P.encode(x)), torch.ones((65, 9), device="cuda")), torch.ones((1, 9), device="cuda")
    many = F.linear(rows, gpu(P.encode(w)), ws)
    few = F.linear(F.Fp8Rows(rows.codes[:T].contiguous(), rows.scales[:T].contiguous()), gpu(P.encode(w)), ws)
    assert (many[:T] != few).float().mean() > 0.5


@pytest.mark.parametrize("T", [3, 40, 300])
def test_scales_of_products_near_the_ends_of_f32(F, T):
    # a row's scale times a block's is formed in f32, before it meets the group's sum: within its range
    # a zero group stays zero and a sum is right; a row whose product is infinite is no number, and alone so
    K, N = 400, 48
    rng = np.random.default_rng(T)
    codes, w = P.encode(rng.integers(-8, 9, (T, K)).astype(np.float32)), P.encode(rng.integers(-8, 9, (N, K)).astype(np.float32))
    codes[:, 128:256] = 0
    xs = np.ones((T, 4), np.float32)
    ws = np.ones((1, 4), np.float32)
    ws[0, 1:3] = 2.0 ** 60, 2.0 ** -60
    xs[:, 1:3] = 2.0 ** 67, 2.0 ** 62  # products of 2^127 and 4
    xs[1, 1] = 2.0 ** 68               # 2^128
    got = F.linear(F.Fp8Rows(gpu(codes), gpu(xs)), gpu(w), gpu(ws)).float().cpu().numpy()
    assert np.isnan(got[1]).all()
    x, one = P.decode(codes), P.decode(w)
    want = x[:, :128] @ one[:, :128].T + 4 * (x[:, 256:384] @ one[:, 256:384].T) + x[:, 384:] @ one[:, 384:].T
    rest = np.arange(T) != 1
    assert np.array_equal(got[rest], torch.from_numpy(want[rest].astype(np.float32)).bfloat16().float().numpy())


@pytest.fixture(scope="module")
def layer():
    # the MoE layer with a block-scaled shared expert
    import gpu_util as gu
    from livglm_amd.workloads import SHAPES, make_layer
    from test_gpu_mirror import _moe
    shape = SHAPES["verify_t2"]
    moe, _ = _moe(gu, shape, make_layer(shape, 7500))
    s = moe.shared_experts
    for p in (s.gate_proj, s.up_proj, s.down_proj):
        p.quantize_to_fp8_block()
    return moe, shape.d


@pytest.mark.parametrize("T", [1, 5, 64, 300, 1100])
def test_a_block_scaled_shared_expert_at_every_number_of_tokens(F, layer, T):
    # few tokens, decode, the grouped products streamed and wide: each adds the ready output, the last of the f32 sum
    moe, d = layer
    x = gpu(np.random.default_rng(T).normal(0, 1, (T, d)).astype(np.float32), torch.bfloat16)
    shared = moe.shared_experts(x)
    out = moe(x)
    scales = moe.shared_experts.down_proj.scales
    moe.shared_experts.down_proj.scales = torch.zeros_like(scales)
    rest = moe(x)
    moe.shared_experts.down_proj.scales = scales
    assert float(shared.float().abs().max()) > 0
    assert bool(((out - (rest + shared.float())).abs() <= 2.0 ** -22 * (rest.abs() + shared.float().abs())).all())


@pytest.mark.parametrize("T", [2, 64])
def test_a_layer_with_a_block_scaled_shared_expert_in_a_graph(F, layer, T):
    moe, d = layer
    rng = np.random.default_rng(T)
    x = gpu(rng.normal(0, 1, (T, d)).astype(np.float32), torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        moe(x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = moe(x)
    for _ in range(3):
        x.copy_(gpu(rng.normal(0, 1, (T, d)).astype(np.float32), torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        again = got.clone()
        assert torch.equal(moe(x), again)
