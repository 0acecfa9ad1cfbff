"""GPU tests of the block-scaled 8-bit operators against the oracle in 64 bits.

Codes and scales of given rows are compared bit for bit.  Tolerances elsewhere:

* a product rounds its output once (2^-8 of its value); its f32 sums run over K
  products and at most 64 partial sums, each scaled with two roundings, in any
  order, and the matrix core may cut where it adds (2^-23 a step): together at
  most (K + K / 128 + 72) 2^-23 of the sum of the terms' magnitudes S;
* the bf16 product of many rows (more than 64) runs on the 8-bit matrix
  instruction, which aligns eight products at a time to the largest sum e of two
  exponents among them and drops what lies below 2^(e - 13) (seen with 448 x 448
  less itself beside single powers of two: 2^3 stays, 2^2 goes).  The largest is at
  least 2^e and the one that sets e is whole, so eight products lose at most 7 x
  2^-13 of the largest, itself at most the product of the largest codes of either
  side.  The bound is far from what is lost (each product a part, in either
  direction), so the whole is held to 2^-8 in the 2-norm too, which the output's
  rounding alone may take;
* the gated product: g and u as above (dg, du, no rounding to bf16), silu's slope
  is at most 1.1, exp and the quotient cost at most 2^-20 of h: dh = 1.1 |u| dg +
  |silu(g)| du + 2^-20 |h| + 1.1 dg du;
* codes of a computed value y known to dy: half a step of e4m3 (2^-4 of the value,
  2^-10 scales for its subnormals) beside dy; scales amax / 448 to dy's maximum in
  the group / 448 and three roundings;
* the norm: a sum of squares over d terms in any order is off by at most (d / 32 +
  48) 2^-24 (a thread adds 32 terms or fewer of it in turn and the rest is a tree),
  half of that on the root, four roundings beside it."""

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


def host(t):
    return t.float().cpu().numpy() if t.dtype == torch.bfloat16 else t.cpu().numpy()


def gpu(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def fenced(a, fill):
    """A copy on the GPU between bytes that are `fill`."""
    a = np.ascontiguousarray(a)
    raw = torch.full((a.nbytes + 8192,), fill, dtype=torch.uint8, device="cuda")
    view = raw[4096:4096 + a.nbytes].view(torch.from_numpy(a[:0]).dtype).view(a.shape)
    view.copy_(torch.from_numpy(a))
    return view, raw


def bf16(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.float32)).bfloat16().float().numpy()


def rows(rng, T, K):
    x = rng.normal(0, 1, (T, K)) * 2.0 ** rng.normal(0, 2, (T, 1))
    x[:, rng.random(K) < 0.01] *= 30
    return x.astype(np.float32)


def weight(rng, N, K):
    codes = rng.integers(0, 256, (N, K)).astype(np.uint8)
    codes[(codes & 127) == 127] = 0  # no NaN
    return codes, (2.0 ** rng.normal(-9, 1, (P.groups(N), P.groups(K)))).astype(np.float32)


def product_error(K, S):
    return (K + K / 128 + 72) * 2.0 ** -23 * S


def dropped(q, w):
    """What the 8-bit matrix instruction may drop of q w^T."""
    def peaks(v):
        pad = np.zeros((v.shape[0], -(-v.shape[1] // 8) * 8))
        pad[:, :v.shape[1]] = np.abs(v)
        return pad.reshape(v.shape[0], -1, 8).max(-1)
    return 7 * 2.0 ** -13 * (peaks(P.row_values(*q)) @ peaks(P.weight_values(*w)).T)


def check_bf16(got, want, err):
    off = np.abs(host(got).astype(np.float64) - want)
    tol = np.abs(want) * 2.0 ** -8 + err * (1 + 2.0 ** -8) + 1e-38
    assert np.all(off <= tol), (off / tol).max()


def check_codes(got, y, dy):
    codes, scales = host(got.codes), host(got.scales).astype(np.float64)
    T, K = y.shape
    pad = np.zeros((T, P.groups(K) * 128))
    pad[:, :K] = np.abs(y)
    amax = np.maximum(pad.reshape(T, -1, 128).max(-1), float(P.TINY))
    pad[:, :K] = dy
    most = pad.reshape(T, -1, 128).max(-1)
    off = np.abs(scales - amax / 448)
    tol = most / 448 + amax / 448 * 3 * 2.0 ** -24
    assert np.all(off <= tol), (off / tol).max()
    step = np.repeat(scales, 128, 1)[:, :K]
    off = np.abs(P.row_values(codes, scales) - y)
    tol = np.maximum((np.abs(y) + dy) * 2.0 ** -4, step * 2.0 ** -10) * (1 + 2.0 ** -20) + dy
    assert np.all(off <= tol), (off / tol).max()


# ---------------------------------------------------------------- quantisers

@pytest.mark.parametrize("T, K", [(1, 8), (1, 128), (3, 136), (2, 576), (17, 2048), (5, 1000), (1500, 144),
                                  (9000, 2056)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_rows(F, T, K, dtype):
    rng = np.random.default_rng(T + K)
    x = rows(rng, T, K)
    x[0, :min(K, 128)] = 0
    x[-1, -8:] *= 2.0 ** -60
    x = bf16(x) if dtype is torch.bfloat16 else x
    got = F.quantize_rows(gpu(x, dtype))
    codes, scales = P.quantize_rows(x)
    np.testing.assert_array_equal(host(got.scales), scales)
    np.testing.assert_array_equal(host(got.codes), codes)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_rows_edges(F, dtype):
    rng = np.random.default_rng(3)
    x = rows(rng, 8, 384)
    x[0, 5], x[1, 200], x[2, 300] = np.inf, -np.inf, np.nan
    x[3, :] = 0
    x[4, :128] = np.inf
    x[5, :] = np.float32(3e38) * np.sign(x[5])
    x[6, :] = 1e-40
    x[7, :128] = np.nan
    x = bf16(x) if dtype is torch.bfloat16 else x
    got = F.quantize_rows(gpu(x, dtype))
    codes, scales = P.quantize_rows(x)
    np.testing.assert_array_equal(host(got.scales), scales)
    nan = (codes & 127) == 127
    assert nan.sum() == 3 + 128 + 128
    np.testing.assert_array_equal((host(got.codes) & 127) == 127, nan)
    np.testing.assert_array_equal(host(got.codes)[~nan], codes[~nan])


def test_quantize_rows_writes_no_further(F):
    x = rows(np.random.default_rng(4), 3, 200)
    codes, raw = fenced(np.zeros((3, 200), np.uint8), 0xA5)
    scales, raw_s = fenced(np.zeros((3, 2), np.float32), 0xA5)
    got = F.quantize_rows(gpu(x), out=F.Fp8Rows(codes, scales))
    assert got.codes is codes and got.scales is scales
    np.testing.assert_array_equal(host(codes), P.quantize_rows(x)[0])
    for r, n in ((raw, 600), (raw_s, 24)):
        assert (r[:4096] == 0xA5).all() and (r[4096 + n:] == 0xA5).all()


@pytest.mark.parametrize("N, K", [(1, 8), (128, 128), (129, 136), (576, 2048), (100, 1000)])
def test_quantize_weight(F, N, K):
    rng = np.random.default_rng(N)
    w = bf16(rows(rng, N, K))
    if N > 100:
        w[3, 4], w[100, 7] = np.inf, np.nan
    codes, scales = F.quantize_weight(gpu(w, torch.bfloat16))
    want, want_s = P.quantize_weight(w)
    np.testing.assert_array_equal(host(scales), want_s)
    nan = (want & 127) == 127
    np.testing.assert_array_equal((host(codes) & 127) == 127, nan)
    np.testing.assert_array_equal(host(codes)[~nan], want[~nan])


# ---------------------------------------------------------------- the norm

@pytest.mark.parametrize("T, d", [(1, 8), (1, 4096), (3, 200), (65, 2048), (7, 2056), (2, 4104), (5, 8192),
                                  (3, 8200), (2, 20000), (1, 32768), (3000, 136)])
@pytest.mark.parametrize("xt, rt, weighted", [(torch.bfloat16, torch.bfloat16, True), (torch.float32, torch.bfloat16, True),
                                              (torch.bfloat16, torch.float32, False), (torch.float32, torch.float32, True),
                                              (torch.float32, None, True), (torch.bfloat16, None, False)])
def test_add_rms_norm(F, T, d, xt, rt, weighted):
    rng = np.random.default_rng(T * d)
    x, r = rows(rng, T, d), 3 * rows(rng, T, d)
    x = bf16(x) if xt is torch.bfloat16 else x
    r = None if rt is None else bf16(r) if rt is torch.bfloat16 else r
    w = (1 + 0.3 * rng.normal(0, 1, d)).astype(np.float32) if weighted else None
    got, h = F.add_rms_norm(gpu(x, xt), None if w is None else gpu(w), 1e-6, residual=None if r is None else gpu(r, rt))
    y, exact = P.add_rms_norm(x, r, w, 1e-6)
    if r is None:
        assert h is None
    else:
        assert h.dtype is rt
        want = x + r  # in f32, as the sum is
        np.testing.assert_array_equal(host(h), bf16(want) if rt is torch.bfloat16 else want)
    rel = ((d / 32 + 48) / 2 + 5) * 2.0 ** -24
    add = 0 if r is None else 2.0 ** -24  # the sum x + residual, rounded once; it moves every norm alike by less
    check_codes(got, y, np.abs(y) * (rel + 2 * add))


def test_add_rms_norm_in_place_and_nan(F):
    rng = np.random.default_rng(11)
    x, r = gpu(rows(rng, 4, 512)), gpu(rows(rng, 4, 512))
    x[1, 7] = float("nan")
    x[2, 9] = float("inf")
    x[3] = 0
    r[3] = 0
    want, h = F.add_rms_norm(x, None, 1e-6, residual=r)
    into = r.clone()
    got, same = F.add_rms_norm(x, None, 1e-6, residual=into, residual_out=into)
    assert same is into and torch.equal(into.view(torch.int32), h.view(torch.int32))
    assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales)
    into = x.clone()  # in the rows' own place
    got2, same = F.add_rms_norm(into, None, 1e-6, residual=r, residual_out=into)
    assert same is into and torch.equal(into.view(torch.int32), h.view(torch.int32))
    assert torch.equal(got2.codes, want.codes) and torch.equal(got2.scales, want.scales)
    codes = host(got.codes)
    assert ((codes[1] & 127) == 127).all()  # a NaN spreads over its row
    assert (codes[2, 9] & 127) == 127 and not (np.delete(codes[2], 9) & 127).any()
    assert not codes[3].any() and (host(got.scales)[3] == np.float32(2.0 ** -126)).all()


# ---------------------------------------------------------------- the products

SHAPES = [
    # T, K, N: around each kernel's tiles, K off its groups, N off its blocks
    (1, 16, 1), (1, 128, 16), (2, 2048, 768), (1, 4096, 4096), (3, 144, 17), (15, 576, 130), (16, 1408, 256),
    (17, 1408, 255), (31, 112, 129), (32, 4112, 96), (33, 272, 100), (48, 2048, 576), (64, 1024, 384), (65, 1040, 513),
    (100, 256, 1000), (128, 384, 128), (129, 400, 144), (200, 4096, 300), (256, 2048, 2048), (257, 528, 515),
    (333, 1536, 640), (700, 656, 1100), (1025, 896, 2047), (2000, 512, 4096),
    # each way to cut a product, beside the above
    (24, 272, 4096), (30, 144, 8000), (56, 400, 4100), (24, 2064, 4096), (50, 16400, 2064),
    (140, 272, 4100), (250, 272, 4090), (370, 272, 4095), (230, 272, 6000),
    (450, 272, 4096), (620, 272, 4095), (850, 144, 4096), (900, 1040, 4090), (1600, 144, 4096),
    (3000, 144, 4096), (2900, 528, 4090),
    (70, 9008, 40), (4, 9008, 40), (40, 16400, 24),
    # the longest rows that a workgroup quantises, longer ones, the longest
    (2, 16384, 40), (8, 4096, 40), (7, 4112, 33), (1, 32784, 24), (6, 1040, 4100), (16, 2048, 70), (13, 2064, 40),
    (11, 400, 4100), (5, 272, 8192), (5, 272, 8200), (2, 1 << 20, 20), (66, 1 << 17, 33),
]


@pytest.mark.parametrize("T, K, N", SHAPES)
@pytest.mark.parametrize("kind", ["fp8", "bf16", "f32"])
def test_linear(F, T, K, N, kind):
    rng = np.random.default_rng(T + K + N)
    x, w = rows(rng, T, K), weight(rng, N, K)
    if kind == "fp8":
        q = weight(rng, T, K)[0], (2.0 ** rng.normal(-9, 2, (T, P.groups(K)))).astype(np.float32)
        given = F.Fp8Rows(fenced(q[0], 0x7F)[0], fenced(q[1], 0xFF)[0])
    else:
        x = bf16(x) if kind == "bf16" else x
        q = P.quantize_rows(x)
        if kind == "bf16":
            given = fenced(torch.from_numpy(x).bfloat16().view(torch.int16).numpy(), 0xFF)[0].view(torch.bfloat16)
        else:
            given = fenced(x, 0xFF)[0]
    out, raw = fenced(np.zeros((T, N), np.int16), 0xA5)
    # NaN codes and scales around the operands: nothing behind them may enter
    got = F.linear(given, fenced(w[0], 0x7F)[0], fenced(w[1], 0xFF)[0], out=out.view(torch.bfloat16))
    want, S = P.product(q, w)
    check_bf16(got, want, product_error(K, S) + (dropped(q, w) if T > 64 else 0))
    assert np.linalg.norm(host(got) - want) <= 2.0 ** -8 * np.linalg.norm(want)
    assert (raw[:4096] == 0xA5).all() and (raw[4096 + 2 * T * N:] == 0xA5).all()


GATED = [(1, 128, 16), (2, 2048, 768), (5, 144, 144), (16, 1408, 240), (17, 272, 128), (48, 2048, 512), (64, 4096, 2048),
         (65, 528, 400), (129, 512, 256), (256, 1024, 1408), (333, 656, 272), (1030, 384, 768), (2000, 512, 2048), (100, 272, 1024),
         (333, 272, 1408), (150, 1040, 2048), (96, 272, 2048), (120, 528, 2032),
         (700, 528, 2032), (250, 272, 7168),
         (500, 4112, 2048), (3000, 400, 2048), (2950, 272, 2032), (70, 9008, 48), (3, 9008, 48),
         (2, 16384, 48), (8, 4096, 1040), (16, 2048, 272), (11, 400, 1040), (5, 144, 8208), (3, 16400, 32), (7, 4112, 48)]


@pytest.mark.parametrize("T, K, N", GATED)
@pytest.mark.parametrize("kind, limit", [("fp8", 10.0), ("bf16", 0.0), ("f32", 1.5)])
def test_gate_up(F, T, K, N, kind, limit):
    rng = np.random.default_rng(T + K + N)
    x = rows(rng, T, K)
    x = bf16(x) if kind == "bf16" else x
    q = P.quantize_rows(x)
    given = {"fp8": lambda: F.Fp8Rows(gpu(q[0]), gpu(q[1])), "bf16": lambda: gpu(x, torch.bfloat16),
             "f32": lambda: gpu(x)}[kind]()
    g, u = weight(rng, N, K), weight(rng, N, K)
    for one in (g, u):  # of a size that meets the limits
        one[1][:] *= 8 / np.sqrt(K)
    codes, raw = fenced(np.zeros((T, N), np.uint8), 0xA5)
    scales, raw_s = fenced(np.zeros((T, P.groups(N)), np.float32), 0xA5)
    got = F.gate_up(given, fenced(g[0], 0x7F)[0], fenced(g[1], 0xFF)[0], fenced(u[0], 0x7F)[0], fenced(u[1], 0xFF)[0],
                    limit, out=F.Fp8Rows(codes, scales))
    (yg, sg), (yu, su) = P.product(q, g), P.product(q, u)
    dg, du = product_error(K, sg), product_error(K, su)
    h = P.gated(yg, yu, limit)
    if limit > 0:
        yu = np.clip(yu, -limit, limit)
        yg = np.minimum(yg, limit)
    silu = P.gated(yg, np.ones_like(yg), 0.0)
    check_codes(got, h, 1.1 * np.abs(yu) * dg + np.abs(silu) * du + 2.0 ** -20 * np.abs(h) + 1.1 * dg * du)
    for r, n in ((raw, T * N), (raw_s, 4 * T * P.groups(N))):
        assert (r[:4096] == 0xA5).all() and (r[4096 + n:] == 0xA5).all()


@pytest.mark.parametrize("T", [1, 5, 40, 300])
def test_products_pass_nan_and_infinity_on(F, T):
    # a NaN in one row, an infinite scale of another: their rows alone are no numbers
    rng = np.random.default_rng(T)
    K, N = 400, 272
    codes, scales = P.quantize_rows(rows(rng, T, K))
    w = weight(rng, N, K)
    codes[0, K - 1] = 0x7F
    if T > 3:
        scales[3, 1] = np.inf
    rows8 = F.Fp8Rows(gpu(codes), gpu(scales))
    y = host(F.linear(rows8, gpu(w[0]), gpu(w[1])))
    h = F.gate_up(rows8, gpu(w[0]), gpu(w[1]), gpu(w[0]), gpu(w[1]), 10.0)
    bad = np.zeros(T, bool)
    bad[0] = True
    if T > 3:
        bad[3] = True
    assert np.isnan(y[0]).all() and not np.isfinite(y[bad]).any() and np.isfinite(y[~bad]).all()
    hv = host(h.codes) & 127
    assert (hv[0] == 127).all() and not (hv[~bad] == 127).any() and np.isfinite(host(h.scales)).all()
    # and a NaN weight: its column alone
    wn = w[0].copy()
    wn[5, 0] = 0xFF
    y = host(F.linear(F.Fp8Rows(gpu(P.quantize_rows(rows(rng, T, K))[0]), gpu(np.ones((T, 4), np.float32))), gpu(wn),
                      gpu(w[1])))
    assert np.isnan(y[:, 5]).all() and np.isfinite(np.delete(y, 5, 1)).all()


@pytest.mark.parametrize("T", [1, 3, 8, 16])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_quantised_by_the_product_are_the_quantisers(F, T, dtype):
    # zeros of either sign, infinities and NaN, tiny and huge groups
    rng = np.random.default_rng(T)
    x = rows(rng, T, 656)
    x[0, :128] = np.where(rng.random(128) < 0.5, -0.0, 0.0)
    x[0, 128:256] *= 1e-38
    x[0, 256:384] *= 1e30
    x[-1, 5], x[-1, 300], x[T // 2, 655] = np.inf, -np.inf, np.nan
    x, w, u = gpu(x, dtype), [gpu(a) for a in weight(rng, 272, 656)], [gpu(a) for a in weight(rng, 272, 656)]
    q = F.quantize_rows(x)
    a, b = F.linear(x, *w).float(), F.linear(q, *w).float()
    assert bool((a.isnan() == b.isnan()).all()) and bool(a[-1].isnan().all())
    # the same f32 products, added up in the same order
    assert torch.equal(a.nan_to_num(0.0), b.nan_to_num(0.0))
    a, b = F.gate_up(x, *w, *u, 7.0), F.gate_up(q, *w, *u, 7.0)
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)


def test_shapes_of_rows(F):
    rng = np.random.default_rng(6)
    x, w = gpu(rows(rng, 6, 256), torch.bfloat16), [gpu(a) for a in weight(rng, 48, 256)]
    flat = F.linear(x, *w)
    assert torch.equal(F.linear(x.view(2, 3, 256), *w), flat.view(2, 3, 48))
    assert torch.equal(F.linear(x[0], *w), flat[0])
    q = F.quantize_rows(x.view(3, 2, 256))
    assert tuple(q.scales.shape) == (3, 2, 2)
    assert torch.equal(F.linear(q, *w), flat.view(3, 2, 48))
    assert torch.equal(F.linear(q, w[0].view(torch.float8_e4m3fn), w[1]), flat.view(3, 2, 48))
    for empty in (x[:0], F.quantize_rows(x[:0])):
        assert tuple(F.linear(empty, *w).shape) == (0, 48)
        assert tuple(F.gate_up(empty, *w, *w, 0.0).codes.shape) == (0, 48)
    assert F.add_rms_norm(x[:0], None, 0.0)[0].scales.shape == (0, 2)


def test_refusals(F):
    from glm53flash.contract import ContractError
    rng = np.random.default_rng(7)
    x, (w, s) = gpu(rows(rng, 4, 256)), [gpu(a) for a in weight(rng, 48, 256)]
    q = F.quantize_rows(x)
    big = torch.zeros(2048, device="cuda")
    square, wide = big[:512].view(torch.bfloat16).view(4, 256), [gpu(a) for a in weight(rng, 256, 256)]
    cases = [
        lambda: F.linear(x[:, :128], w, s),                       # not contiguous
        lambda: F.linear(x.double(), w, s), lambda: F.linear(x.half(), w, s),
        lambda: F.linear(x[:, :128].contiguous(), w, s),          # another width
        lambda: F.linear(x, w, s[:, :1].contiguous()), lambda: F.linear(x, w, s.double()),
        lambda: F.linear(x, w.float(), s), lambda: F.linear(x, w.t(), s), lambda: F.linear(x, w.cpu(), s),
        lambda: F.linear((q.codes, q.scales[:2]), w, s), lambda: F.linear((q.codes.float(), q.scales), w, s),
        lambda: F.linear(x, w, s, out=torch.empty(4, 48, device="cuda")),
        lambda: F.linear(x, w, s, out=torch.empty(4, 40, dtype=torch.bfloat16, device="cuda")),
        lambda: F.linear(torch.zeros(4, 8, device="cuda"), w[:, :8].contiguous(), s[:, :1].contiguous()),  # K % 16
        lambda: F.linear(x.view(-1)[1:1 + 256], w, s),            # off its alignment
        lambda: F.gate_up(x, w, s, w[:32].contiguous(), s, 0.0),
        lambda: F.gate_up(x, w[:40].contiguous(), s, w[:40].contiguous(), s, 0.0),  # features % 16
        lambda: F.quantize_rows(torch.zeros(2, 12, device="cuda")),
        lambda: F.quantize_rows(x, out=F.Fp8Rows(q.codes[:2], q.scales)),
        lambda: F.quantize_weight(x), lambda: F.quantize_weight(x[0].bfloat16()),
        lambda: F.add_rms_norm(x, w, 1e-6), lambda: F.add_rms_norm(x, x[0, :128].contiguous(), 1e-6),
        lambda: F.add_rms_norm(x, None, -1.0), lambda: F.add_rms_norm(x, None, 1e-6, residual=x[:2]),
        lambda: F.add_rms_norm(x, None, 1e-6, residual_out=x.clone()),
        lambda: F.add_rms_norm(x, None, 1e-6, residual=x, residual_out=x.bfloat16()),
        lambda: F.linear(torch.zeros((), device="cuda"), w, s),
        # outputs over what is read
        lambda: F.linear(square, *wide, out=square),
        lambda: F.linear((big[:256].view(torch.uint8).view(4, 256), q.scales), *wide, out=square),
        lambda: F.gate_up(q, *wide, *wide, 0.0, out=q),
        lambda: F.quantize_rows(x, out=F.Fp8Rows(x.view(-1)[:256].view(torch.uint8).view(4, 256), q.scales)),
        lambda: F.add_rms_norm(square, None, 1e-6, residual=x, residual_out=big[:1024].view(4, 256)),
        lambda: F.add_rms_norm(big[:1024].view(4, 256), None, 1e-6, residual=x, residual_out=big[8:1032].view(4, 256)),
        lambda: F.add_rms_norm(x, None, 1e-6, residual=x.clone(), residual_out=big[:1024].view(4, 256),
                               out=F.Fp8Rows(big[:256].view(torch.uint8).view(4, 256), q.scales)),
    ]
    for i, case in enumerate(cases):
        with pytest.raises(ContractError):
            case()
            pytest.fail(f"case {i} was taken")


def test_offsets_past_32_bits(F):
    # 2^20 rows of 2064 channels: codes, bf16 rows and outputs beyond 2^31 and 2^32 bytes
    T, K = 1 << 20, 2064
    gen = torch.Generator(device="cuda").manual_seed(13)
    some = torch.tensor([0, 1, 777_777, *range(T - 70, T)], device="cuda")
    x = torch.empty((T, K), dtype=torch.bfloat16, device="cuda").normal_(generator=gen)
    r = torch.empty((T, K), dtype=torch.bfloat16, device="cuda").normal_(generator=gen)
    q = F.quantize_rows(x)
    want = P.quantize_rows(host(x[some]))
    assert np.array_equal(host(q.codes[some]), want[0]) and np.array_equal(host(q.scales[some]), want[1])
    n, h = F.add_rms_norm(x, None, 1e-6, residual=r)
    few, few_h = F.add_rms_norm(x[some], None, 1e-6, residual=r[some])
    assert torch.equal(n.codes[some], few.codes) and torch.equal(n.scales[some], few.scales)
    assert torch.equal(h[some], few_h)
    del n, h, r, x
    w = weight(np.random.default_rng(14), K, K)
    y = F.linear(q, gpu(w[0]), gpu(w[1]))
    dot, S = P.product(want, w)
    check_bf16(y[some], dot, product_error(K, S) + dropped(want, w))
    del y
    short = F.Fp8Rows(q.codes[:, :144].contiguous(), q.scales[:, :2].contiguous())
    ws = [gpu(w[0][:, :144]), gpu(w[1][:, :2])]
    got = F.gate_up(short, *ws, *ws, 5.0)
    few = F.gate_up(F.Fp8Rows(short.codes[some], short.scales[some]), *ws, *ws, 5.0)
    # exact products of two groups either way: the same f32 sums but for their order, a code apart at most
    a, b = (P.row_values(host(v.codes), host(v.scales)) for v in (F.Fp8Rows(got.codes[some], got.scales[some]), few))
    step = np.repeat(host(few.scales).astype(np.float64), 128, 1)[:, :K]
    assert np.all(np.abs(a - b) <= np.maximum(np.abs(b) * 2.0 ** -3, step * 2.0 ** -9) * (1 + 2.0 ** -10))


# ---------------------------------------------------------------- as they are used

def mlp_of(rng, d, I):
    from glm53flash.layers import DenseMLP
    mlp = DenseMLP(d, I, 10.0)
    for p, shape in ((mlp.gate_proj, (I, d)), (mlp.up_proj, (I, d)), (mlp.down_proj, (d, I))):
        p.weight = gpu(rng.normal(0, 0.03, shape).astype(np.float32), torch.bfloat16)
        p.quantize_to_fp8_block()
    return mlp


@pytest.mark.parametrize("T, d, I", [(1, 2048, 768), (7, 1024, 512), (40, 512, 272), (300, 512, 768)])
def test_a_layer_of_them(F, T, d, I):
    # norm with the residual -> MLP, through the layers, against the same steps by the operators and against 64 bits
    from glm53flash.layers import RMSNorm
    rng = np.random.default_rng(T)
    norm, mlp = RMSNorm(d, 1e-6), mlp_of(rng, d, I)
    norm.weight = gpu(1 + 0.1 * rng.normal(0, 1, d).astype(np.float32), torch.bfloat16)
    x, r = gpu(rows(rng, T, d), torch.bfloat16), gpu(rows(rng, T, d))
    q, h = norm.quantized(x, r)
    out = mlp(q)
    assert torch.equal(h, x.float() + r) and out.dtype == torch.bfloat16 and out.shape == x.shape
    g, u, dn = mlp.gate_proj, mlp.up_proj, mlp.down_proj
    hidden = F.gate_up(q, g.weight, g.scales, u.weight, u.scales, 10.0)
    assert torch.equal(out, F.linear(hidden, dn.weight, dn.scales)) and torch.equal(out, dn(hidden))
    hq, dq = (host(hidden.codes), host(hidden.scales)), (host(dn.weight), host(dn.scales))
    want, S = P.product(hq, dq)
    check_bf16(out, want, product_error(I, S) + (dropped(hq, dq) if T > 64 else 0))
    # bf16 rows are quantised by the product
    y = norm(x)
    assert torch.equal(mlp(y), mlp(F.quantize_rows(y)))
    assert torch.equal(g(y), g(F.quantize_rows(y)))


def test_linear_of_a_quantised_weight_is_near_the_bf16_one(F):
    # the format's own error: products of two e4m3 roundings, each at most 2^-4 of its value (subnormals aside)
    from glm53flash.layers import DeferredLinear
    rng = np.random.default_rng(8)
    lin = DeferredLinear(2048, 576)
    w = bf16(rng.normal(0, 0.02, (576, 2048)))
    lin.weight = gpu(w, torch.bfloat16)
    source, size = lin.quantize_to_fp8_block()
    assert source == 2 * 576 * 2048 and size == 576 * 2048 + 4 * 5 * 16
    x = bf16(rng.normal(0, 1, (33, 2048)))
    got = host(lin(gpu(x, torch.bfloat16))).astype(np.float64)
    want = x.astype(np.float64) @ w.T.astype(np.float64)
    S = np.abs(x).astype(np.float64) @ np.abs(w).T.astype(np.float64)
    assert np.all(np.abs(got - want) <= S * 2.2 * 2.0 ** -4)
    assert np.linalg.norm(got - want) / np.linalg.norm(want) < 2.0 ** -4


def test_a_side_stream_and_a_graph(F):
    rng = np.random.default_rng(9)
    d, I = 512, 384
    mlp = mlp_of(rng, d, I)
    norm_w = gpu(np.ones(d, np.float32))
    for T in (2, 20, 200):
        x, r = gpu(rows(rng, T, d), torch.bfloat16), gpu(rows(rng, T, d), torch.bfloat16)

        def step():
            q, h = F.add_rms_norm(x, norm_w, 1e-6, residual=r)
            return mlp(q), mlp(x), h

        want = [t.clone() for t in step()]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert torch.equal(a, b)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        for i in range(3):  # new inputs each time, eager work in between
            x.copy_(gpu(rows(rng, T, d), torch.bfloat16))
            graph.replay()
            torch.cuda.synchronize()
            again = [t.clone() for t in got]
            for a, b in zip(step(), again):
                assert torch.equal(a, b), (T, i)


def test_two_calls_at_once(F):
    rng = np.random.default_rng(10)
    mlp = mlp_of(rng, 1024, 512)
    xs = [gpu(rows(rng, T, 1024), torch.bfloat16) for T in (20, 70)]
    want = [mlp(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append(mlp(x))
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert torch.equal(a, b)


@pytest.mark.parametrize("T", [2, 24])
def test_a_block_scaled_shared_expert(F, T):
    # the MoE layer with it is the layer without a shared expert's part plus the MLP's own output
    import gpu_util as gu
    from livglm_amd.workloads import SHAPES as LAYERS, make_layer
    from test_gpu_mirror import _moe
    shape = LAYERS["verify_t2"]
    moe, dl = _moe(gu, shape, make_layer(shape, 7400))
    rng = np.random.default_rng(12)
    x = gpu(rng.normal(0, 1, (T, shape.d)).astype(np.float32), torch.bfloat16)
    for p in (moe.shared_experts.gate_proj, moe.shared_experts.up_proj, moe.shared_experts.down_proj):
        p.quantize_to_fp8_block()
    out = moe(x)
    shared = moe.shared_experts(x)
    assert moe(x[:0]).shape == (0, shape.d)
    # with the FFN site's residual streams: the same layer, then post y + comb residual
    from glm53flash.mhc import hyper_residual
    streams, post, comb = (torch.from_numpy(rng.normal(0, 1, n).astype(np.float32)).cuda()
                           for n in ((T, 4, shape.d), (T, 4), (T, 4, 4)))
    whole = moe.with_hyper_residual(x, streams, post, comb)
    apart = hyper_residual(streams, out, post, comb)
    moe.shared_experts = mlp_of(rng, shape.d, shape.I_shared)
    moe.shared_experts.down_proj.scales.zero_()
    rest = moe(x)
    # f32 sums of at most nine terms, the shared one last
    err = (out - (rest + shared.float())).abs()
    assert bool((err <= 2.0 ** -22 * (rest.abs() + shared.float().abs())).all())
    # at most nine terms of y in another order, and ten roundings of the five terms
    most = hyper_residual(streams.abs(), rest.abs() + shared.float().abs(), post.abs(), comb.abs())
    assert bool(((whole - apart).abs() <= 2.0 ** -20 * most).all())
    assert float(shared.float().abs().max()) > 0 and out.dtype == torch.float32
