"""GPU tests of the paged attention cache against the oracle in 64 bits.

Tolerance of the attention, element by element: the output is rounded once
(2^-8 of its value) and each probability once for its product with the values
(2^-8 of sum p |v|); a score's error is at most (key_dim + 4) 2^-24 of
scale sum |q k| (f32 products and sums, the scale and log2 e rounded) plus
2^-22 of the score, which a hardware exp2 of 2 ulp adds to, and moves numerator
and denominator alike, 2 delta each way; the sums over n positions add at most
(n + 64) 2^-24."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import paged_oracle as P

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def C():
    from glm53flash import paged_cache
    return paged_cache


def dev(a, dtype=torch.int32):
    return torch.as_tensor(np.ascontiguousarray(a)).to(dtype).cuda()


def f64(t):
    return t.float().cpu().numpy().astype(np.float64)


# ---------------------------------------------------------------- the step

def run_step(C, new, lens, blocks, tables, free, top, page, max_tokens, alias=False):
    t = {k: dev(v) for k, v in (("new", new), ("lens", lens), ("blocks", blocks), ("tables", tables), ("free", free))}
    nf = dev([top])
    r = C.cache_step(t["new"], t["lens"], t["blocks"], t["tables"], t["free"], nf, page_size=page,
                     max_tokens=max_tokens, kv_lens=t["lens"] if alias else None)
    torch.cuda.synchronize()
    got = {k: getattr(r, k).cpu().numpy() for k in ("kv_lens", "cu_new", "slots", "positions")}
    got |= {"status": int(r.status), "blocks": t["blocks"].cpu().numpy(), "tables": t["tables"].cpu().numpy(),
            "free_pages": t["free"].cpu().numpy(), "num_free": int(nf)}
    return got


def same_step(got, want, B):
    for k, v in want.items():
        np.testing.assert_array_equal(got[k][:B] if k == "kv_lens" else got[k], v, err_msg=k)


def random_state(rng, B, page, width, pool):
    blocks = rng.integers(0, width + 1, B)
    while blocks.sum() > pool:
        blocks //= 2
    lens = np.array([rng.integers(0, n * page + 1) for n in blocks])
    order = rng.permutation(pool).astype(np.int32)
    tables = np.full((B, width), -1, np.int32)
    at = 0
    for b in range(B):
        tables[b, :blocks[b]] = order[at:at + blocks[b]]
        at += blocks[b]
    return lens, blocks, tables, np.concatenate([order[at:], order[:at]]), pool - at


@pytest.mark.parametrize("B, page, width, tokens", [
    (1, 16, 4, 10), (1, 1, 1, 0), (3, 5, 9, 40), (64, 16, 64, 70), (65, 7, 30, 4096), (300, 16, 20, 4097),
    (1000, 1, 8, 2000), (1025, 64, 3, 9000), (4096, 16, 6, 20001), (70, 16, 20, 8192), (70, 16, 20, 8193),
])
@pytest.mark.parametrize("alias", [False, True])
def test_step(C, B, page, width, tokens, alias):
    rng = np.random.default_rng(B + page)
    pool = B * width + 3
    lens, blocks, tables, free, top = random_state(rng, B, page, width, pool)
    room = width * page - lens
    share = max(1, tokens // B)
    new = np.minimum(rng.integers(0, share + 1, B), room)
    gone = rng.random(B) < 0.3
    new = np.where(gone, -1 - np.minimum(rng.integers(0, share + 1, B), width * page), new)
    if tokens == 0:
        new[:] = 0
    want = P.step(new, lens, blocks, tables, free, top, page, tokens)
    same_step(run_step(C, new, lens, blocks, tables, free, top, page, tokens, alias), want, B)
    assert want["status"] == 0


@pytest.mark.parametrize("what, bits", [("pages", 1), ("table", 2), ("tokens", 4), ("len", 8), ("blocks", 8),
                                        ("short", 8), ("free", 8), ("all", 7)])
@pytest.mark.parametrize("tokens", [33, 5000])
def test_step_refuses_and_changes_nothing(C, what, bits, tokens):
    B, page, width, pool = 5, 4, 1500, 40
    rng = np.random.default_rng(9)
    blocks = np.array([2, 0, 3, 1, 4])
    lens = np.array([7, 0, 12, 4, 13])
    order = rng.permutation(pool).astype(np.int32)
    tables = np.full((B, width), -1, np.int32)
    at = 0
    for b in range(B):
        tables[b, :blocks[b]] = order[at:at + blocks[b]]
        at += blocks[b]
    free, top = np.concatenate([order[at:], order[:at]]), pool - at
    new = np.array([1, 2, -4, 0, 3])
    if what == "pages":
        new[1], tokens = 4 * (top + 4), max(tokens, 200)
    elif what == "table":
        new[1], tokens, top, free = width * page + 1, 20000, 2900, np.arange(3000, dtype=np.int32)
    elif what == "tokens":
        new[1], tokens = 30, 20
    elif what == "len":
        lens[0] = -1
    elif what == "blocks":
        blocks[3] = width + 1
        lens[3] = 3
    elif what == "short":
        lens[4] = 17
    elif what == "free":
        top = pool
    elif what == "all":
        new[1] = 2 ** 31 - 1
    want = P.step(new, lens, blocks, tables, free, top, page, tokens)
    assert want["status"] == bits
    same_step(run_step(C, new, lens, blocks, tables, free, top, page, tokens), want, B)
    assert (want["tables"] == tables).all() and want["num_free"] == top


@pytest.mark.parametrize("B", [2, 1025])  # (1025: two requests a thread)
@pytest.mark.parametrize("page, width", [(2 ** 31 - 1, 1), (2 ** 30 - 1, 2)])
def test_step_lengths_within_a_page_of_32_bits(C, B, page, width):
    """A length and a page together pass 32 bits: the last page goes to the request that needs it."""
    for who in (0, B - 2, B - 1):
        lens, blocks = np.zeros(B, int), np.zeros(B, int)
        tables, free = np.full((B, width), -1, np.int32), np.arange(width, dtype=np.int32)
        blocks[who] = width - 1
        lens[who] = (width - 1) * page
        tables[who, :width - 1] = width - 1
        new = np.zeros(B, int)
        new[who] = 5
        want = P.step(new, lens, blocks, tables, free, 1, page, 8)
        assert want["status"] == 0 and want["blocks"][who] == width and want["num_free"] == 0
        same_step(run_step(C, new, lens, blocks, tables, free, 1, page, 8), want, B)


@pytest.mark.parametrize("tokens", [8, 9000])
def test_step_of_pages_outside_the_cache(C, tokens):
    """A token whose table entry is no page of the cache has no slot, also where entry times page passes 32 bits."""
    page, pool = 16, 12
    wild = [pool, -1, 2 ** 28, 2 ** 28 + 3, -2 ** 31, 2 ** 31 - 1, -2 ** 28]
    B = len(wild) + 1
    tables = np.array([[w, -1] for w in wild] + [[5, -1]], np.int32)
    lens, blocks = np.full(B, 10), np.ones(B, int)
    got = run_step(C, np.ones(B, int), lens, blocks, tables, np.arange(pool, dtype=np.int32), 4, page, tokens)
    assert got["status"] == 0
    np.testing.assert_array_equal(got["slots"], [-1] * len(wild) + [5 * page + 10] + [-1] * (tokens - B))
    np.testing.assert_array_equal(got["positions"], [10] * B + [0] * (tokens - B))
    np.testing.assert_array_equal(got["tables"], tables)


@pytest.mark.parametrize("tokens", [0, 5])
def test_step_of_no_requests(C, tokens):
    """An empty batch goes through step, write and attention, and leaves the table as it was."""
    table = C.PageTable(6, 4, 3, 2)
    cache = C.PagedKVCache(table, 2, 64, 64)
    table.step(dev([3, 0, 5]), 8)
    before = [t.clone() for t in (table.lens, table.blocks, table.tables, table.free_pages, table.num_free, cache.keys)]
    step = table.step(dev(np.zeros(0)), tokens)
    assert step.cu_new.tolist() == [0] and int(step.status) == 0
    assert step.slots.tolist() == [-1] * tokens and step.positions.tolist() == [0] * tokens
    rows = torch.ones((tokens, 2, 64), device="cuda", dtype=torch.bfloat16)
    cache.write(rows, rows, step.slots)
    assert cache.attend(torch.ones((0, 4, 64), device="cuda", dtype=torch.bfloat16), 1.0).shape == (0, 4, 64)
    after = (table.lens, table.blocks, table.tables, table.free_pages, table.num_free, cache.keys)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(after, before))
    empty = C.cache_step(dev(np.zeros(0)), table.lens, table.blocks, table.tables, table.free_pages, table.num_free,
                         page_size=4, max_tokens=tokens)
    assert empty.kv_lens.numel() == 0 and empty.cu_new.tolist() == [0] and empty.slots.tolist() == [-1] * tokens


def test_step_captured_and_replayed(C):
    """A graph of steps over the table's own state, replayed with new inputs in between."""
    table = C.PageTable(40, 4, 3, 12)
    new = torch.zeros(3, dtype=torch.int32, device="cuda")
    table.step(new, 16)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step = table.step(new, 16)
    lens, blocks, tables = np.zeros(3, int), np.zeros(3, int), np.full((3, 12), -1, np.int32)
    free, top = np.arange(39, -1, -1).astype(np.int32), 40
    for values in ([5, 0, 3], [1, 1, 1], [-1, 7, -6], [4, -1, 0], [0, 16, 0]):
        new.copy_(dev(values))
        g.replay()
        torch.cuda.synchronize()
        want = P.step(values, lens, blocks, tables, free, top, 4, 16)
        lens, blocks, tables, free, top = (want[k] for k in ("kv_lens", "blocks", "tables", "free_pages", "num_free"))
        np.testing.assert_array_equal(step.slots.cpu(), want["slots"])
        np.testing.assert_array_equal(table.tables.cpu(), tables)
        np.testing.assert_array_equal(table.lens.cpu(), lens)
        assert int(table.num_free) == top and int(step.status) == 0


# ---------------------------------------------------------------- the write

def make_cache(rng, pages, heads, page, dim, fmt):
    """Random cache tensors and their values in 64 bits."""
    x = torch.from_numpy(rng.standard_normal((pages, heads, page, dim), np.float32)).to(torch.bfloat16)
    if fmt == "bf16":
        return x.cuda(), None, f64(x)
    codes, scales = P.mx_rows(f64(x))
    return dev(codes, torch.uint8), dev(scales, torch.uint8), P.mx_values(codes, scales)


WRITES = [(1, 1, 1, 8, 8, "bf16", 0), (5, 2, 3, 64, 40, "bf16", 0), (64, 8, 16, 128, 128, "bf16", 24),
          (333, 1, 64, 576, 0, "bf16", 0), (1, 1, 1, 32, 0, "mxfp8", 0), (7, 3, 5, 96, 32, "mxfp8", 8),
          (64, 8, 16, 128, 128, "mxfp8", 0), (201, 1, 64, 576, 0, "mxfp8", 64)]


@pytest.mark.parametrize("N, heads, page, dk, dv, fmt, pad", WRITES)
def test_write(C, N, heads, page, dk, dv, fmt, pad):
    rng = np.random.default_rng(N + dk)
    pages = N // page + 3
    kc, ks, kv = make_cache(rng, pages, heads, page, dk, fmt)
    vc, vs, vv = make_cache(rng, pages, heads, page, dv, fmt) if dv else (None, None, None)
    # keys and values are slices of one projection
    rows = torch.from_numpy(rng.standard_normal((N, heads * (dk + dv) + pad), np.float32)).to(torch.bfloat16)
    rows *= torch.from_numpy(np.exp2(rng.integers(-30, 30, (N, 1))).astype(np.float32)).to(torch.bfloat16)
    rows[0, 0], rows[-1, dk - 1], rows[N // 2, :dk // 2] = float("nan"), float("inf"), 0.0
    rows = rows.cuda()
    keys, values = rows[:, :heads * dk].unflatten(1, (heads, dk)), None
    if dv:
        values = rows[:, heads * dk:heads * (dk + dv)].unflatten(1, (heads, dv))
    slots = rng.permutation(pages * page)[:N].astype(np.int32)
    if N > 4:
        slots[1], slots[3], slots[4] = -1, pages * page, -2 ** 31
    C.cache_write(keys, values, dev(slots), kc, vc, key_scales=ks, value_scales=vs)
    torch.cuda.synchronize()
    for cache, scales, old, x, d in ((kc, ks, kv, keys, dk), (vc, vs, vv, values, dv)):
        if cache is None:
            continue
        want = f64(x)
        codes = want_scales = None
        if fmt == "mxfp8":
            codes, want_scales = P.mx_rows(want)
            want = P.mx_values(codes, want_scales)
        full = old.copy()
        for t in range(N):
            if 0 <= slots[t] < pages * page:
                full[slots[t] // page, :, slots[t] % page] = want[t]
        got = f64(cache) if fmt == "bf16" else P.mx_values(cache.cpu().numpy(), scales.cpu().numpy())
        np.testing.assert_array_equal(got, full)
        if fmt == "mxfp8":
            for t in range(N):
                if 0 <= slots[t] < pages * page:
                    np.testing.assert_array_equal(scales.cpu().numpy()[slots[t] // page, :, slots[t] % page], want_scales[t])


def test_write_every_magnitude(C):
    """Every finite bf16 value, in groups of one exponent and in mixed ones, to MXFP8 and back."""
    bits = np.arange(1 << 16, dtype=np.uint16)
    rng = np.random.default_rng(3)
    bits = np.concatenate([bits, rng.permutation(bits)])
    with np.errstate(invalid="ignore"):  # (signalling NaNs)
        x = P.bf16_bits_to_f32(bits).astype(np.float64).reshape(-1, 1, 64)
    t = torch.from_numpy(bits.view(np.int16)).view(torch.bfloat16).view(-1, 1, 64).cuda()
    n = len(x)
    codes = torch.zeros((n, 1, 1, 64), dtype=torch.uint8, device="cuda")
    scales = torch.zeros((n, 1, 1, 2), dtype=torch.uint8, device="cuda")
    C.cache_write(t, None, dev(np.arange(n)), codes, None, key_scales=scales)
    want, want_scales = P.mx_rows(x[:, :, None])
    np.testing.assert_array_equal(scales.cpu().numpy(), want_scales)
    np.testing.assert_array_equal(P.mx_values(codes.cpu().numpy(), want_scales), P.mx_values(want, want_scales))


# ---------------------------------------------------------------- the attention

def attend_case(C, rng, B, q_len, heads, kv_heads, dk, dv, lens, page, fmt="bf16", latent=False, spread=1.0, pad=0,
                bad=0, poison=True, more_blocks=0, scale=None):
    """Runs one call and checks it element by element; returns its output."""
    scale = dk ** -0.5 if scale is None else scale
    lens = np.asarray(lens)
    counts = -(-np.maximum(lens, 0) // page)
    pool, width = int(counts.sum()) + 2, max(1, int(counts.max()) + more_blocks)
    order = rng.permutation(pool)
    tables = np.full((B, width), -1, np.int32)
    at = 0
    for b in range(B):
        tables[b, :counts[b]] = order[at:at + counts[b]]
        at += counts[b]
    kc, ks, kv = make_cache(rng, pool, kv_heads, page, dk, fmt)
    vc, vs, vv = (None, None, kv[..., :dv]) if latent else make_cache(rng, pool, kv_heads, page, dv, fmt)
    if poison:  # what no request holds must not be used: NaN there
        held = np.zeros((pool, page), bool)
        for b in range(B):
            for j in range(max(0, lens[b])):
                held[tables[b, j // page], j % page] = True
        gone = torch.from_numpy(~held).cuda()[:, None, :, None]
        nan = 0x7f if fmt == "mxfp8" else float("nan")
        kc = kc.masked_fill(gone, nan)
        vc = None if vc is None else vc.masked_fill(gone, nan)
    for _ in range(bad):  # pages that the cache does not have
        b = int(rng.integers(B))
        if counts[b]:
            tables[b, rng.integers(counts[b])] = rng.choice([-1, -2 ** 31, pool, 2 ** 31 - 1])
    q = torch.from_numpy(rng.standard_normal((B, q_len, heads * dk + pad), np.float32) * np.float32(spread))
    q = q.to(torch.bfloat16).cuda()
    query = q[:, :, pad:].unflatten(2, (heads, dk)) if pad else q.unflatten(2, (heads, dk))
    out = C.paged_attention(query, kc, vc, dev(tables), dev(lens), scale=scale, value_dim=dv, key_scales=ks,
                            value_scales=vs)
    torch.cuda.synchronize()
    want, size, reach = P.attend(f64(query), kv, vv, tables, lens, scale)
    delta = (dk + 4) * 2.0 ** -24 * reach + 2.0 ** -22 * (1 + reach)
    n = max(1, lens.max())
    tol = 2.0 ** -8 * np.abs(want) + (2.0 ** -8 + 2 * delta[..., None] + (n + 64) * 2.0 ** -24) * 1.01 * size + 1e-30
    got = f64(out)
    assert got.shape == want.shape
    off = np.abs(got - want) / tol
    assert np.isfinite(got).all() and off.max() <= 1, (off.max(), np.unravel_index(off.argmax(), off.shape))
    return out


@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
@pytest.mark.parametrize("lens", [[1], [0], [2], [15, 16, 17, 0, 31, 32, 33], [63, 64, 65, 127, 128, 129, 1, 300],
                                  [517], [1000, 3, 1500]])
@pytest.mark.parametrize("heads, kv_heads, dk, dv, q_len", [(8, 2, 128, 128, 1), (4, 4, 64, 64, 2), (2, 1, 96, 32, 3)])
def test_attend_lengths(C, fmt, lens, heads, kv_heads, dk, dv, q_len):
    rng = np.random.default_rng(sum(lens) + dk)
    attend_case(C, rng, len(lens), q_len, heads, kv_heads, dk, dv, lens, 16, fmt)


@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 64, 100, 1000])
def test_attend_pages(C, fmt, page):
    rng = np.random.default_rng(page)
    attend_case(C, rng, 3, 1, 8, 2, 128, 128, [333, 100, 64], page, fmt, more_blocks=3)
    attend_case(C, rng, 2, 2, 16, 1, 576, 512, [200, 77], page, fmt, latent=True)


@pytest.mark.parametrize("heads, kv_heads", [(1, 1), (3, 1), (16, 16), (16, 1), (24, 2), (40, 8), (71, 1), (64, 2)])
@pytest.mark.parametrize("q_len", [1, 2, 5])
def test_attend_head_layouts(C, heads, kv_heads, q_len):
    rng = np.random.default_rng(heads * 10 + q_len)
    attend_case(C, rng, 3, q_len, heads, kv_heads, 128, 128, [130, 4, 259], 16, pad=64)


@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
@pytest.mark.parametrize("dk, dv", [(64, 64), (128, 128), (256, 256), (32, 32), (96, 96), (192, 128), (64, 256), (576, 512),
                                    (1024, 1024)])
def test_attend_widths(C, fmt, dk, dv):
    rng = np.random.default_rng(dk + dv)
    attend_case(C, rng, 2, 1, 8, 2, dk, dv, [200, 65], 16, fmt)


@pytest.mark.parametrize("dk, dv", [(8, 8), (24, 40), (136, 72)])
def test_attend_odd_widths(C, dk, dv):
    attend_case(C, np.random.default_rng(dk), 2, 2, 6, 2, dk, dv, [77, 130], 16)


@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
@pytest.mark.parametrize("heads", [1, 16, 40, 64, 128])
@pytest.mark.parametrize("q_len", [1, 2])
def test_attend_latent(C, fmt, heads, q_len):
    rng = np.random.default_rng(heads + q_len)
    attend_case(C, rng, 4, q_len, heads, 1, 576, 512, [1, 333, 0, 130], 64, fmt, latent=True)


def test_attend_other_latents(C):
    rng = np.random.default_rng(8)
    attend_case(C, rng, 2, 1, 8, 1, 128, 64, [70, 200], 16, latent=True)
    attend_case(C, rng, 2, 1, 8, 2, 128, 128, [70, 200], 16, latent=True)
    attend_case(C, rng, 2, 1, 8, 2, 576, 512, [70, 200], 16, "mxfp8", latent=True)


@pytest.mark.parametrize("latent", [False, True])
@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
def test_attend_bad_pages(C, latent, fmt):
    """Table entries outside the cache: their positions are not seen, in a whole request too."""
    rng = np.random.default_rng(12)
    shape = (16, 1, 576, 512) if latent else (8, 2, 128, 128)
    attend_case(C, rng, 3, 2, *shape, [333, 100, 640], 16, fmt, latent, bad=9, poison=False)
    attend_case(C, rng, 2, 1, *shape, [16, 300], 16, fmt, latent, bad=12, poison=False)


@pytest.mark.parametrize("latent", [False, True])
@pytest.mark.parametrize("spread, scale", [(20.0, None), (1.0, -0.3), (1.0, 0.0), (1e-30, None), (300.0, 1.0)])
def test_attend_scores(C, latent, spread, scale):
    """One position taking all, negative and zero scales, vanishing and huge scores."""
    rng = np.random.default_rng(13)
    shape = (16, 1, 576, 512) if latent else (8, 2, 128, 128)
    attend_case(C, rng, 2, 1, *shape, [700, 33], 16, "bf16", latent, spread=spread, scale=scale)


@pytest.mark.parametrize("latent", [False, True])
@pytest.mark.parametrize("step", [0.02, 0.3, 5.0, -0.3])
def test_attend_rising_scores(C, latent, step):
    """Scores that rise by `step` powers of two from position to position, in small steps and in large ones, beside
    rows whose scores fall: a running maximum lags behind, leaps, or stays, row by row."""
    rng = np.random.default_rng(15)
    n, page, heads = 1000, 16, 16
    dk, dv = (576, 512) if latent else (128, 128)
    kc, _, kv = make_cache(rng, 63, 1, page, dk, "bf16")
    vc, vv = (None, kv[..., :dv]) if latent else make_cache(rng, 63, 1, page, dv, "bf16")[::2]
    tables = np.arange(63, dtype=np.int32).reshape(1, -1)
    at = torch.arange(63 * page, device="cuda").view(63, 1, page)
    kc[..., dk - 1] = (at % 256).to(torch.bfloat16)  # (integers to 256 are exact)
    kc[..., dk - 2] = (at // 256).to(torch.bfloat16)
    q = torch.from_numpy(rng.standard_normal((1, 1, heads, dk), np.float32)).to(torch.bfloat16).cuda()
    for h in range(heads):
        sign = 1.0 if h % 2 else -1.0
        q[0, 0, h, dk - 1] = sign * step * 0.6931 * dk ** 0.5
        q[0, 0, h, dk - 2] = sign * step * 0.6931 * dk ** 0.5 * 256
    lens = np.array([n])
    got = f64(C.paged_attention(q, kc, vc, dev(tables), dev(lens), scale=dk ** -0.5, value_dim=dv))
    kv = f64(kc)
    want, size, reach = P.attend(f64(q), kv, kv[..., :dv] if latent else vv, tables, lens, dk ** -0.5)
    delta = (dk + 4) * 2.0 ** -24 * reach + 2.0 ** -22 * (1 + reach)
    tol = 2.0 ** -8 * np.abs(want) + (2.0 ** -8 + 2 * delta[..., None] + (n + 64) * 2.0 ** -24) * 1.01 * size + 1e-30
    assert (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("dk, dv, latent", [(128, 128, False), (96, 96, False), (576, 512, True)])
@pytest.mark.parametrize("step, leap, n", [(0.02, 0, 300), (0.0, 7, 300), (0.0, 7, 5000)])
def test_attend_largest_values(C, dk, dv, latent, step, leap, n):
    """Values near the largest of the type, whose weighted mean is finite: weights are held at 1 at most, also where a
    running maximum lags behind scores that rise by `step` powers of two a position, or by `leap` at the last one."""
    rng = np.random.default_rng(n + leap)
    page, heads = 16, 16
    pages = -(-n // page)
    kc, _, _ = make_cache(rng, pages, 1, page, dk, "bf16")
    vc = None if latent else make_cache(rng, pages, 1, page, dv, "bf16")[0]
    at = torch.arange(pages * page, device="cuda").view(pages, 1, page)
    kc[..., dk - 1] = (at % 256).to(torch.bfloat16)  # (integers to 256 are exact)
    kc[..., dk - 2] = (at // 256).to(torch.bfloat16)
    kc[..., dk - 3] = (at == n - 1).to(torch.bfloat16)
    values = kc[..., :dv] if latent else vc
    values *= 2.0 ** 116 if leap else 2.0 ** 120
    if leap:
        values[(n - 1) // page, 0, (n - 1) % page] = 2.0 ** 126
    q = torch.zeros((1, 1, heads, dk), dtype=torch.bfloat16, device="cuda")  # (nothing of the values' channels)
    share = (torch.arange(heads, device="cuda") + 1) / heads * 0.6931 * dk ** 0.5
    q[0, 0, :, dk - 1], q[0, 0, :, dk - 2], q[0, 0, :, dk - 3] = share * step, share * step * 256, share * leap
    tables, lens = np.arange(pages, dtype=np.int32).reshape(1, -1), np.array([n])
    got = f64(C.paged_attention(q, kc, vc, dev(tables), dev(lens), scale=dk ** -0.5, value_dim=dv))
    want, size, reach = P.attend(f64(q), f64(kc), f64(values), tables, lens, dk ** -0.5)
    delta = (dk + 4) * 2.0 ** -24 * reach + 2.0 ** -22 * (1 + reach)
    tol = 2.0 ** -8 * np.abs(want) + (2.0 ** -8 + 2 * delta[..., None] + (n + 64) * 2.0 ** -24) * 1.01 * size
    assert np.isfinite(got).all() and (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("latent", [False, True])
def test_attend_rows_do_not_depend_on_others(C, latent):
    """A head's result is the same bits whatever the other heads of its kv head ask."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    dk, dv = (576, 512) if latent else (128, 128)
    kc = torch.randn((60, 1, 16, dk), generator=gen, device="cuda", dtype=torch.bfloat16)
    vc = None if latent else torch.randn((60, 1, 16, dv), generator=gen, device="cuda", dtype=torch.bfloat16)
    table = torch.randperm(60, generator=gen, device="cuda").int().view(2, 30)
    q = torch.randn((2, 16, dk), generator=gen, device="cuda", dtype=torch.bfloat16)
    lens = dev([471, 333])
    want = C.paged_attention(q, kc, vc, table, lens, scale=0.5, value_dim=dv)
    q[:, 3:] *= -7
    got = C.paged_attention(q, kc, vc, table, lens, scale=0.5, value_dim=dv)
    assert torch.equal(got[:, :3], want[:, :3])


@pytest.mark.parametrize("latent", [False, True])
def test_attend_on_two_streams_at_once(C, latent):
    """Calls that run beside each other share no workspace."""
    gen = torch.Generator(device="cuda").manual_seed(7)
    dk, dv = (576, 512) if latent else (128, 128)
    kc = torch.randn((600, 1, 64, dk), generator=gen, device="cuda", dtype=torch.bfloat16)
    vc = None if latent else torch.randn((600, 1, 64, dv), generator=gen, device="cuda", dtype=torch.bfloat16)
    calls = []
    for i in range(2):
        table = torch.randperm(600, generator=gen, device="cuda").int().view(4, 150)
        q = torch.randn((4, 32, dk), generator=gen, device="cuda", dtype=torch.bfloat16)
        lens = dev([9600, 5000 + i, 1, 7777])
        calls.append((q, kc, vc, table, lens))
    want = [C.paged_attention(*c, scale=0.05, value_dim=dv) for c in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for s, c, g in zip(streams, calls, got):
            with torch.cuda.stream(s):
                g.append(C.paged_attention(*c, scale=0.05, value_dim=dv))
    torch.cuda.synchronize()
    for w, gs in zip(want, got):
        assert all(torch.equal(w, g) for g in gs)


def test_attend_many_requests(C):
    """More requests than a wave, lengths from none on, and far more than the chip takes at once."""
    rng = np.random.default_rng(14)
    lens = rng.integers(0, 90, 261)
    lens[5], lens[200] = 3000, 1500
    attend_case(C, rng, 261, 1, 4, 2, 64, 64, lens, 16)
    attend_case(C, rng, 70, 2, 16, 1, 576, 512, rng.integers(0, 150, 70), 32, latent=True)
    attend_case(C, rng, 1500, 1, 2, 2, 64, 64, rng.integers(0, 20, 1500), 4)


@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
@pytest.mark.parametrize("heads, kv_heads, dk, dv, latent", [
    (8, 1, 128, 128, False), (3, 3, 64, 64, False), (4, 2, 256, 256, False), (6, 2, 192, 128, False), (2, 1, 32, 64, False),
    (4, 1, 576, 512, True), (20, 1, 576, 512, True)])
@pytest.mark.parametrize("q_len", [7, 16])
def test_attend_many_new_tokens(C, fmt, heads, kv_heads, dk, dv, latent, q_len):
    """More new tokens than a request has, as many, and tiles that end among them."""
    rng = np.random.default_rng(heads + q_len)
    attend_case(C, rng, 7, q_len, heads, kv_heads, dk, dv, [1, 16, 17, 40, 0, 70, 200], 16, fmt, latent)


def long_case(C, kv_heads, group, dk, dv, n, latent, fmt, q_len=1, page=64):
    """A long history against 64-bit torch on the GPU (the oracle's formula, one request)."""
    gen = torch.Generator(device="cuda").manual_seed(n)
    pages = -(-n // page)
    x = torch.randn((pages, kv_heads, page, dk), generator=gen, device="cuda", dtype=torch.bfloat16)
    ks = vs = None
    v = x[..., :dv] if latent else torch.randn((pages, kv_heads, page, dv), generator=gen, device="cuda",
                                               dtype=torch.bfloat16)
    q = torch.randn((1, q_len, kv_heads * group, dk), generator=gen, device="cuda", dtype=torch.bfloat16)
    kc, vc = x, None if latent else v
    if fmt == "mxfp8":
        slots = torch.arange(pages * page, device="cuda", dtype=torch.int32)
        rows = x.transpose(1, 2).reshape(pages * page, kv_heads, dk)
        kc, ks = torch.empty(x.shape, dtype=torch.uint8, device="cuda"), torch.empty((*x.shape[:3], dk // 32), dtype=torch.uint8, device="cuda")
        C.cache_write(rows, None, slots, kc, None, key_scales=ks)
        x = (kc.view(torch.float8_e4m3fn).double().unflatten(-1, (-1, 32)) * torch.exp2(ks.double() - 127)[..., None]).flatten(-2)
        if not latent:
            raise ValueError
        v = x[..., :dv]
    table = torch.randperm(pages, generator=gen, device="cuda").int().view(1, -1)
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    got = C.paged_attention(q, kc, vc, table, lens, scale=dk ** -0.5, value_dim=dv, key_scales=ks, value_scales=vs)
    k64 = x[table[0].long()].double().transpose(0, 1).flatten(1, 2)[:, :n]
    v64 = v[table[0].long()].double().transpose(0, 1).flatten(1, 2)[:, :n]
    for t in range(q_len):
        m = n - (q_len - 1 - t)
        qt = q[0, t].double().view(kv_heads, group, dk)
        p = torch.softmax(qt @ k64[:, :m].transpose(1, 2) * dk ** -0.5, -1)
        want, size = (p @ v64[:, :m]).view(-1, dv), (p @ v64[:, :m].abs()).view(-1, dv)
        # here the roundings of many probabilities average: the 2-norm over the row set is a fraction of the worst case
        err = (got[0, t].double() - want).abs()
        assert (err <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + n * 2.0 ** -24 + 2.0 ** -12) * size).all()
        assert (err.norm() / want.norm()).item() < 2.0 ** -7


@pytest.mark.parametrize("kv_heads, group, dk, dv, n, latent, fmt, q_len", [
    (1, 8, 128, 128, 65537, False, "bf16", 1), (2, 4, 64, 64, 30001, False, "bf16", 2),
    (1, 32, 576, 512, 33333, True, "bf16", 2), (1, 64, 576, 512, 20000, True, "mxfp8", 1)])
def test_attend_long(C, kv_heads, group, dk, dv, n, latent, fmt, q_len):
    long_case(C, kv_heads, group, dk, dv, n, latent, fmt, q_len)


def test_attend_beyond_32_bits(C):
    """A cache of more than 2^32 elements; the pages used lie at its end."""
    page, dk = 256, 256
    pages = 70000  # 4.6e9 elements of keys, 9.2 GB
    kc = torch.zeros((pages, 1, page, dk), dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(1)
    last = torch.randn((2, 1, page, dk), generator=gen, device="cuda", dtype=torch.bfloat16)
    rows = last.view(2 * page, 1, dk)
    slots = torch.arange((pages - 2) * page, pages * page, dtype=torch.int32, device="cuda")
    C.cache_write(rows, None, slots, kc, None)
    assert torch.equal(kc[-2:], last) and not kc[:-2].any()
    table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device="cuda")
    q = torch.randn((1, 4, dk), generator=gen, device="cuda", dtype=torch.bfloat16)
    got = C.paged_attention(q, kc, None, table, torch.tensor([500], dtype=torch.int32, device="cuda"), scale=0.1,
                            value_dim=dk)
    k = torch.cat([last[1, 0], last[0, 0]])[:500].double()
    want = torch.softmax(q[0].double() @ k.T * 0.1, -1) @ k
    assert ((got[0].double() - want).norm() / want.norm()).item() < 2.0 ** -7


def test_attend_values_that_are_not_finite(C):
    """An infinity or NaN in a position that is seen comes through; another request's does not."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    kc = torch.randn((8, 2, 16, 128), generator=gen, device="cuda", dtype=torch.bfloat16)
    vc = torch.randn((8, 2, 16, 128), generator=gen, device="cuda", dtype=torch.bfloat16)
    vc[1, 0, 3, 7], vc[2, 1, 0, 0] = float("inf"), float("nan")
    table = torch.tensor([[0, 1], [2, 3], [4, 5]], dtype=torch.int32, device="cuda")
    q = torch.randn((3, 8, 128), generator=gen, device="cuda", dtype=torch.bfloat16)
    out = C.paged_attention(q, kc, vc, table, torch.tensor([32, 20, 32], dtype=torch.int32, device="cuda"), scale=0.1)
    bad = ~out.isfinite()
    want = torch.zeros_like(bad)
    want[0, :4, 7] = True
    want[1, 4:, 0] = True
    assert torch.equal(bad, want) and out[0, :4, 7].isposinf().all() and out[1, 4:, 0].isnan().all()


@pytest.mark.parametrize("latent", [False, True])
@pytest.mark.parametrize("n", [33, 64, 700])
def test_attend_earlier_tokens_do_not_see_later_ones(C, latent, n):
    """NaN in the newest token's row reaches that token alone; the tokens before it stay as they were."""
    gen = torch.Generator(device="cuda").manual_seed(n)
    dk, dv = (576, 512) if latent else (128, 128)
    kc = torch.randn((50, 1, 16, dk), generator=gen, device="cuda", dtype=torch.bfloat16)
    vc = None if latent else torch.randn((50, 1, 16, dv), generator=gen, device="cuda", dtype=torch.bfloat16)
    table = torch.arange(50, dtype=torch.int32, device="cuda").view(1, -1)
    q = torch.randn((1, 3, 8, dk), generator=gen, device="cuda", dtype=torch.bfloat16)
    lens = dev([n])
    want = C.paged_attention(q, kc, vc, table, lens, scale=0.05, value_dim=dv)
    for t, pos in ((2, n - 1), (1, n - 2)):
        (kc if latent else vc)[pos // 16, 0, pos % 16, 5] = float("nan")
        got = C.paged_attention(q, kc, vc, table, lens, scale=0.05, value_dim=dv)
        assert torch.equal(got[:, :t], want[:, :t])
        assert got[:, t:, :, 5].isnan().all()


def test_attend_leaves_what_is_behind(C):
    """Nothing is written past the batch's rows, and the same call gives the same bits."""
    rng = np.random.default_rng(21)
    kc, _, _ = make_cache(rng, 200, 2, 16, 128, "bf16")
    vc, _, _ = make_cache(rng, 200, 2, 16, 128, "bf16")
    table = dev(rng.permutation(200)[:150].reshape(3, 50))
    lens = dev([800, 1, 555])
    q = torch.randn((3, 16, 128), device="cuda", dtype=torch.bfloat16)
    room = torch.full((5, 16, 128), 7.0, device="cuda", dtype=torch.bfloat16)
    first = C.paged_attention(q, kc, vc, table, lens, scale=0.1)
    for _ in range(3):
        C.paged_attention(q, kc, vc, table, lens, scale=0.1, out=room[1:4])
        assert torch.equal(room[1:4], first)
    assert (room[0] == 7).all() and (room[4] == 7).all()


# ---------------------------------------------------------------- used together

@pytest.mark.parametrize("mode", [None, "mxfp8"])
@pytest.mark.parametrize("latent", [False, True])
def test_serving_run(C, mode, latent):
    """Requests come, are prefilled, decoded, verified with tokens rejected, end and are replaced; the cache's
    contents and every attention are checked against histories kept on the host."""
    rng = np.random.default_rng(31)
    B, page = 4, 8
    heads, kv_heads, dk, dv = (16, 1, 576, 512) if latent else (8, 2, 64, 64)
    table = C.PageTable(40, page, B, 16)
    caches = [C.PagedKVCache(table, kv_heads, dk, dv, latent=latent, quantization_mode=mode) for _ in range(2)]
    past = [[([], []) for _ in caches] for _ in range(B)]

    def draw(n, d):
        return torch.from_numpy(rng.standard_normal((n, kv_heads, d), np.float32)).to(torch.bfloat16).cuda()

    script = [[20, 7, 0, 33], [1, 1, 0, 1], [2, 2, -10, 2], [1, -1, 1, -13], [2, 2, 2, 2], [1, 1, 1, 1]]
    rejected = [0, 0, 1, 0, 1, 0]
    for new, drop in zip(script, rejected):
        total = sum(n if n >= 0 else -1 - n for n in new)
        step = table.step(dev(new), total + 3)
        assert int(step.status) == 0
        cu = step.cu_new.tolist()
        for layer, cache in enumerate(caches):
            keys, values = draw(total + 3, dk), None if latent else draw(total + 3, dv)
            cache.write(keys, values, step.slots)
            for b, n in enumerate(new):
                if n < 0:
                    past[b][layer] = ([], [])
                k, v = past[b][layer]
                for t in range(cu[b], cu[b + 1]):
                    k.append(f64(keys[t]))
                    v.append(f64(keys[t])[..., :dv] if latent else f64(values[t]))
            q_len = 2 if all(n == 2 for n in new) else 1
            q = torch.from_numpy(rng.standard_normal((B, q_len, heads, dk), np.float32)).to(torch.bfloat16).cuda()
            got = f64(cache.attend(q, dk ** -0.5))
            for b in range(B):
                k, v = past[b][layer]
                assert int(step.kv_lens[b]) == len(k)
                if not k:
                    assert (got[b] == 0).all()
                    continue
                kk, vv = np.stack(k), np.stack(v)  # [n, kv_heads, d]
                if mode == "mxfp8":
                    kk = P.mx_values(*P.mx_rows(kk))
                    vv = kk[..., :dv] if latent else P.mx_values(*P.mx_rows(vv))
                n = len(k)
                want, size, reach = P.attend(f64(q[b:b + 1]), kk.transpose(1, 0, 2)[None], vv.transpose(1, 0, 2)[None],
                                             np.zeros((1, 1), int), [n], dk ** -0.5)
                delta = (dk + 4) * 2.0 ** -24 * reach + 2.0 ** -22 * (1 + reach)
                tol = 2.0 ** -8 * np.abs(want) + (2.0 ** -8 + 2 * delta[..., None] + (n + 64) * 2.0 ** -24) * 1.01 * size + 1e-30
                assert (np.abs(got[b] - want[0]) <= tol[0]).all()
        if drop:  # the verify step's last token is rejected where there is one
            table.lens.sub_((table.lens > 0).int() * drop)
            for b in range(B):
                for layer in range(2):
                    for side in past[b][layer]:
                        if side:
                            side.pop()


def test_decode_step_captured(C):
    """Step, write and attention of two layers in one graph, replayed with other inputs and eager calls between;
    a second graph on another stream with a state of its own."""
    B, page, heads, kv_heads, d = 5, 16, 8, 2, 128

    def build(seed):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        table = C.PageTable(200, page, B, 32)
        caches = [C.PagedKVCache(table, kv_heads, d, d) for _ in range(2)]
        first = table.step(dev([40, 3, 100, 16, 1]), 160)
        for c in caches:
            c.write(torch.randn((160, kv_heads, d), generator=gen, device="cuda", dtype=torch.bfloat16),
                    torch.randn((160, kv_heads, d), generator=gen, device="cuda", dtype=torch.bfloat16), first.slots)
        x = torch.randn((B, heads + 2 * kv_heads, d), generator=gen, device="cuda", dtype=torch.bfloat16)
        new = dev([1] * B)

        def once():
            step = table.step(new, B)
            return [(c.write(x[:, heads:heads + kv_heads], x[:, heads + kv_heads:], step.slots),
                     c.attend(x[:, :heads], d ** -0.5))[1] for c in caches]
        return gen, table, caches, x, once

    runs = []
    for seed in (1, 2):
        gen, table, caches, x, once = build(seed)
        egen, etable, ecaches, ex, eonce = build(seed)  # the same, eagerly
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            outs = once()
        runs.append((stream, graph, outs, x, gen, ex, eonce, table, etable, once))  # (once: the graph's tensors live)
    for turn in range(20):
        for stream, graph, outs, x, gen, *_ in runs:
            x.copy_(torch.randn(x.shape, generator=gen, device="cuda", dtype=torch.bfloat16))
        torch.cuda.synchronize()
        for stream, graph, *_ in runs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for stream, graph, outs, x, gen, ex, eonce, table, etable, _ in runs:
            ex.copy_(x)
            for got, want in zip(outs, eonce()):
                assert torch.equal(got, want)
            assert torch.equal(table.tables, etable.tables) and torch.equal(table.lens, etable.lens)


def test_other_stream(C):
    rng = np.random.default_rng(41)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        attend_case(C, rng, 3, 1, 8, 2, 128, 128, [130, 4, 900], 16)


@pytest.mark.parametrize("change", ["dtype", "cache dtype", "heads", "width", "table", "lens", "format", "values",
                                    "latent", "out", "query", "stride", "slots", "scales"])
def test_python_refusals(C, change):
    from glm53flash.contract import ContractError
    kc, vc = (torch.zeros((4, 2, 16, 64), device="cuda", dtype=torch.bfloat16) for _ in range(2))
    q = torch.zeros((2, 8, 64), device="cuda", dtype=torch.bfloat16)
    table, lens = dev([[0, 1], [2, 3]]), dev([3, 4])
    kw = {"scale": 1.0}
    codes = torch.zeros((4, 2, 16, 64), device="cuda", dtype=torch.uint8)
    if change == "dtype":
        q = q.float()
    elif change == "cache dtype":
        kc = kc.half()
    elif change == "heads":
        q = q[:, :7].contiguous()
    elif change == "width":
        q = torch.zeros((2, 8, 128), device="cuda", dtype=torch.bfloat16)
    elif change == "table":
        table = table[:1]
    elif change == "lens":
        lens = lens.long()
    elif change == "format":
        kc, kw["key_scales"] = codes, torch.zeros((4, 2, 16, 2), device="cuda", dtype=torch.uint8)
    elif change == "values":
        vc = vc[:, :1].contiguous()
    elif change == "latent":
        vc = None
    elif change == "out":
        kw["out"] = torch.zeros((2, 8, 32), device="cuda", dtype=torch.bfloat16)
    elif change == "query":
        q = q[0]
    elif change == "stride":
        q = q.transpose(1, 2)
    elif change == "slots":
        with pytest.raises(ContractError):
            C.cache_write(q[:, :2], q[:, :2], lens[:1], kc, vc)
        return
    elif change == "scales":
        kc, kw["key_scales"] = codes, torch.zeros((4, 2, 16, 1), device="cuda", dtype=torch.uint8)
    with pytest.raises(ContractError):
        C.paged_attention(q, kc, vc, table, lens, **kw)


@pytest.mark.parametrize("q_len, heads, kv_heads, dim, width, why", [
    (17, 8, 2, 64, 2, "16 new tokens"), (1, 7, 2, 64, 2, "multiple of the kv heads"), (1, 8, 2, 60, 2, "multiples of 8"),
    (1, 2, 1, 64, 1 << 27, "pass 32 bits")])
def test_python_refusals_say_why(C, q_len, heads, kv_heads, dim, width, why):
    from glm53flash.contract import ContractError
    kc = torch.zeros((4, kv_heads, 16, dim), device="cuda", dtype=torch.bfloat16)
    q = torch.zeros((1, q_len, heads, dim), device="cuda", dtype=torch.bfloat16)
    table = torch.zeros((1, width), device="cuda", dtype=torch.int32)
    with pytest.raises(ContractError, match=why):
        C.paged_attention(q, kc, kc, table, dev([3]), scale=1.0)


# ---------------------------------------------------------------- edges of the attention, in all forms

FORMS = [(8, 2, 128, 128, False), (16, 1, 576, 512, True), (6, 2, 96, 96, False)]  # grouped, latent, any widths


def score_tolerance(want, size, reach, n):
    """For scores that are exact integers times a power of two: log2 e and one product are rounded (2^-24 of a
    score each, at the position and at the maximum), beside exp2, the probabilities, the sums and the output."""
    delta = 2 * 1.45 * 2.0 ** -24 * reach + 2.0 ** -22
    tol = 2.0 ** -8 * np.abs(want) + (2.0 ** -8 + 2 * delta[..., None] + (n + 64) * 2.0 ** -24) * 1.01 * size
    assert (tol <= 0.1 * size).all(), "the bound says nothing"
    return tol + 1e-30  # (weights below 2^-126 are none in 32 bits)


@pytest.mark.parametrize("heads, kv_heads, dk, dv, latent", FORMS)
@pytest.mark.parametrize("q_len", [1, 3])
@pytest.mark.parametrize("scale", [1.0, 0.25, -1.0])
def test_attend_huge_scores(C, heads, kv_heads, dk, dv, latent, q_len, scale):
    """Scores of thousands, exact in 32 bits, with ties for the largest: small whole numbers as keys and queries."""
    rng = np.random.default_rng(heads + q_len)
    page, lens = 16, np.array([700, 33, 130])
    width = 44
    tables = rng.permutation(3 * width).reshape(3, width).astype(np.int32)

    def whole(*shape):
        return torch.from_numpy(rng.integers(-8, 9, shape).astype(np.float32)).to(torch.bfloat16)
    kc = whole(3 * width, kv_heads, page, dk)
    for b in range(3):  # every row's largest score has a twin, further on or behind
        for _ in range(lens[b] // 3):
            i, j = rng.integers(0, lens[b], 2)
            tail = slice(dv, None) if latent else slice(None)
            kc[tables[b, i // page], :, i % page, tail] = kc[tables[b, j // page], :, j % page, tail]
            if latent:  # (values of its own)
                kc[tables[b, i // page], :, i % page, :dv] = kc[tables[b, j // page], :, j % page, :dv]
    vc = None if latent else torch.from_numpy(rng.standard_normal((3 * width, kv_heads, page, dv), np.float32)).to(torch.bfloat16)
    q = whole(3, q_len, heads, dk)
    values = kc[..., :dv] if latent else vc
    want, size, reach = P.attend(f64(q), f64(kc), f64(values), tables, lens, scale)
    got = f64(C.paged_attention(q.cuda(), kc.cuda(), None if latent else vc.cuda(), dev(tables), dev(lens), scale=scale,
                                value_dim=dv))
    assert reach.max() > 2000 * abs(scale)
    assert (np.abs(got - want) <= score_tolerance(want, size, reach, 700)).all()


@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
@pytest.mark.parametrize("heads, kv_heads, dk, dv, latent", FORMS)
def test_attend_lengths_beyond_the_table(C, fmt, heads, kv_heads, dk, dv, latent):
    """Lengths below none and past the table are those of none and of the whole table; rows of the table and of
    the lengths behind the batch are not read."""
    rng = np.random.default_rng(dk)
    page, width = 16, 5
    kc, ks, kv = make_cache(rng, 8 * width, kv_heads, page, dk, fmt)
    vc, vs, vv = (None, None, kv[..., :dv]) if latent else make_cache(rng, 8 * width, kv_heads, page, dv, fmt)
    tables = rng.permutation(8 * width).reshape(8, width).astype(np.int32)
    tables[6:] = 2 ** 31 - 1
    lens = np.array([-1, -2 ** 31, 81, 2 ** 31 - 1, 80, 3, 2 ** 31 - 1, -7])
    q = torch.from_numpy(rng.standard_normal((6, 2, heads, dk), np.float32)).to(torch.bfloat16).cuda()
    got = f64(C.paged_attention(q, kc, vc, dev(tables), dev(lens), scale=dk ** -0.5, value_dim=dv, key_scales=ks,
                                value_scales=vs))
    want, size, reach = P.attend(f64(q), kv, vv, tables[:6], lens, dk ** -0.5)
    delta = (dk + 4) * 2.0 ** -24 * reach + 2.0 ** -22 * (1 + reach)
    tol = 2.0 ** -8 * np.abs(want) + (2.0 ** -8 + 2 * delta[..., None] + 144 * 2.0 ** -24) * 1.01 * size
    assert (np.abs(got - want) <= tol).all() and (got[:2] == 0).all()


@pytest.mark.parametrize("heads, kv_heads, dk, dv, latent", FORMS)
def test_attend_not_finite_queries_and_keys(C, heads, kv_heads, dk, dv, latent):
    """A NaN in a query row reaches that row alone.  An infinite key channel of a seen position: a score of -infinity
    takes nothing from the row, one of +infinity makes it NaN, as in the formula."""
    gen = torch.Generator(device="cuda").manual_seed(dk)
    pages, n = 40, 600
    kc = torch.randn((pages, kv_heads, 16, dk), generator=gen, device="cuda", dtype=torch.bfloat16)
    vc = None if latent else torch.randn((pages, kv_heads, 16, dv), generator=gen, device="cuda", dtype=torch.bfloat16)
    table = torch.randperm(pages, generator=gen, device="cuda").int().view(1, -1)
    q = torch.randn((1, 2, heads, dk), generator=gen, device="cuda", dtype=torch.bfloat16)
    q[..., dk - 1] = 1.0
    q[:, :, 1::2, dk - 1] = -1.0
    lens = dev([n])

    def attend(query):
        return C.paged_attention(query, kc, vc, table, lens, scale=0.05, value_dim=dv)
    want = attend(q)
    bad = q.clone()
    bad[0, 0, 2, 3] = float("nan")
    got = attend(bad)
    assert got[0, 0, 2].isnan().all()
    got[0, 0, 2] = want[0, 0, 2]
    assert torch.equal(got, want)
    # channel dk - 1 is none of the latent form's values
    kc[table[0, 17].long(), :, 4, dk - 1] = float("inf")
    got = attend(q)
    assert got[:, :, ::2].isnan().all() and got[:, :, 1::2].isfinite().all()
    shorter = [x for x in range(n) if x != 17 * 16 + 4]
    flat = (lambda t: t[table[0].long()].double().transpose(0, 1).flatten(1, 2)[:, shorter])
    k = flat(kc)
    v = k[..., :dv] if latent else flat(vc)
    group = heads // kv_heads
    for h in range(1, heads, 2):  # (the last token sees all n positions)
        kh, vh, qh = k[h // group], v[h // group], q[0, 1, h].double()
        p = torch.softmax(kh @ qh * 0.05, 0)
        reach = 0.05 * (kh.abs() @ qh.abs()).max()
        delta = (dk + 4) * 2.0 ** -24 * reach + 2.0 ** -22 * (1 + reach)
        tol = 2.0 ** -8 * (p @ vh).abs() + (2.0 ** -8 + 2 * delta + (n + 64) * 2.0 ** -24) * 1.01 * (p @ vh.abs())
        assert ((got[0, 1, h].double() - p @ vh).abs() <= tol).all()


@pytest.mark.parametrize("heads, kv_heads, dk, dv, latent", FORMS)
def test_attend_scale_bytes_of_unowned_rows(C, heads, kv_heads, dk, dv, latent):
    """MXFP8 rows that no request holds: NaN codes and scales of any byte there change nothing."""
    rng = np.random.default_rng(dv)
    page, lens = 16, np.array([70, 0, 129, 16])
    kc, ks, kv = make_cache(rng, 20, kv_heads, page, dk, "mxfp8")
    vc, vs, vv = (None, None, kv[..., :dv]) if latent else make_cache(rng, 20, kv_heads, page, dv, "mxfp8")
    tables = np.full((4, 9), -1, np.int32)
    order, held = rng.permutation(20), np.zeros((20, page), bool)
    for b, n in enumerate(lens):
        for j in range(-(-n // page)):
            tables[b, j], order = order[0], order[1:]
            held[tables[b, j], :min(page, n - j * page)] = True
    q = torch.from_numpy(rng.standard_normal((4, 2, heads, dk), np.float32)).to(torch.bfloat16).cuda()

    def attend(k, ks, v, vs):
        return C.paged_attention(q, k, v, dev(tables), dev(lens), scale=0.1, value_dim=dv, key_scales=ks, value_scales=vs)
    want = attend(kc, ks, vc, vs)
    gone = torch.from_numpy(~held).cuda()[:, None, :, None]
    for code, byte in ((0x7f, 255), (0xff, 0), (0x7e, 255), (0x7e, 254)):
        k, s = kc.masked_fill(gone, code), ks.masked_fill(gone, byte)
        v, t = (None, None) if latent else (vc.masked_fill(gone, code), vs.masked_fill(gone, byte))
        assert torch.equal(attend(k, s, v, t), want)


@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
@pytest.mark.parametrize("heads, kv_heads, dk, dv, latent", FORMS)
def test_attend_captured(C, fmt, heads, kv_heads, dk, dv, latent):
    """Every form in a graph, replayed with other lengths, tables and queries, eager calls between."""
    rng = np.random.default_rng(heads)
    page, width, B = 16, 40, 5
    kc, ks, _ = make_cache(rng, B * width, kv_heads, page, dk, fmt)
    vc, vs, _ = (None, None, None) if latent else make_cache(rng, B * width, kv_heads, page, dv, fmt)
    q = torch.zeros((B, 2, heads, dk), device="cuda", dtype=torch.bfloat16)
    tables, lens = dev(np.zeros((B, width))), dev(np.zeros(B))

    def attend():
        return C.paged_attention(q, kc, vc, tables, lens, scale=0.1, value_dim=dv, key_scales=ks, value_scales=vs)
    attend()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attend()
    for turn in range(6):
        q.copy_(torch.from_numpy(rng.standard_normal(q.shape, np.float32)))
        tables.copy_(dev(rng.permutation(B * width).reshape(B, width)))
        lens.copy_(dev(rng.integers(0, [1, 20, width * page + 1, 300, 2][turn % 5], B)))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, attend())


@pytest.mark.parametrize("kv_heads, group, dk, dv, n", [(1, 8, 128, 128, 30001), (2, 4, 64, 64, 20000), (1, 4, 192, 128, 9000),
                                                        (1, 4, 256, 256, 9000), (1, 2, 96, 96, 5000)])
def test_attend_long_mxfp8(C, kv_heads, group, dk, dv, n):
    """Long histories of keys and values apart in MXFP8, against 64-bit torch on the GPU."""
    gen = torch.Generator(device="cuda").manual_seed(n)
    page = 64
    pages = -(-n // page)
    slots = torch.arange(pages * page, device="cuda", dtype=torch.int32)
    caches, values = [], []
    for d in (dk, dv):
        rows = torch.randn((pages * page, kv_heads, d), generator=gen, device="cuda", dtype=torch.bfloat16)
        codes = torch.empty((pages, kv_heads, page, d), dtype=torch.uint8, device="cuda")
        scales = torch.empty((pages, kv_heads, page, d // 32), dtype=torch.uint8, device="cuda")
        C.cache_write(rows, None, slots, codes, None, key_scales=scales)
        caches.append((codes, scales))
        values.append((codes.view(torch.float8_e4m3fn).double().unflatten(-1, (-1, 32))
                       * torch.exp2(scales.double() - 127)[..., None]).flatten(-2))
    q = torch.randn((1, kv_heads * group, dk), generator=gen, device="cuda", dtype=torch.bfloat16)
    table = torch.randperm(pages, generator=gen, device="cuda").int().view(1, -1)
    got = C.paged_attention(q, caches[0][0], caches[1][0], table, dev([n]), scale=dk ** -0.5, key_scales=caches[0][1],
                            value_scales=caches[1][1])
    k, v = (x[table[0].long()].transpose(0, 1).flatten(1, 2)[:, :n].contiguous() for x in values)
    scores = torch.bmm(k, q[0].double().view(kv_heads, group, dk).transpose(1, 2).contiguous()) * dk ** -0.5
    p = torch.softmax(scores, 1).transpose(1, 2).contiguous()
    want, size = torch.bmm(p, v).view(-1, dv), torch.bmm(p, v.abs()).view(-1, dv)
    reach = (k.abs().amax(1) * 1.0) @ torch.ones(dk, device="cuda", dtype=torch.float64)  # sum of largest |k| ..
    reach = (reach.max() * q.double().abs().max() * dk ** -0.5).item()  # .. times the largest |q|: above every sum |q k|
    delta = (dk + 4) * 2.0 ** -24 * reach + 2.0 ** -22 * (1 + reach)
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2 * delta + (n + 64) * 2.0 ** -24) * 1.01 * size
    assert ((got[0].double() - want).abs() <= tol).all() and (tol < 0.1 * size).all()


@pytest.mark.parametrize("heads, kv_heads, dk, dv, latent, fmt", [
    (8, 1, 576, 512, True, "bf16"), (8, 1, 576, 512, True, "mxfp8"), (8, 2, 128, 128, False, "mxfp8"),
    (4, 2, 96, 96, False, "bf16"), (4, 2, 96, 96, False, "mxfp8")])
def test_every_form_beyond_32_bits(C, heads, kv_heads, dk, dv, latent, fmt):
    """Caches of more than 2^32 elements (and bytes), in all forms and both formats; the pages used lie at their end."""
    page, n = 64, 150
    pages = (1 << 32) // (kv_heads * page * dk) + 40
    kind = torch.bfloat16 if fmt == "bf16" else torch.uint8

    def empty(d):
        shape = (pages, kv_heads, page, d)
        return (torch.zeros(shape, dtype=kind, device="cuda"),
                None if fmt == "bf16" else torch.zeros((*shape[:3], d // 32), dtype=torch.uint8, device="cuda"))
    kc, ks = empty(dk)
    vc, vs = (None, None) if latent else empty(dv)
    gen = torch.Generator(device="cuda").manual_seed(dk)
    keys = torch.randn((3 * page, kv_heads, dk), generator=gen, device="cuda", dtype=torch.bfloat16)
    values = None if latent else torch.randn((3 * page, kv_heads, dv), generator=gen, device="cuda", dtype=torch.bfloat16)
    slots = torch.arange((pages - 3) * page, pages * page, dtype=torch.int32, device="cuda")
    C.cache_write(keys, values, slots, kc, vc, key_scales=ks, value_scales=vs)

    def small(t):
        return None if t is None else t[-3:].clone()
    q = torch.randn((1, 2, heads, dk), generator=gen, device="cuda", dtype=torch.bfloat16)
    order = [2, 0, 1]
    got = C.paged_attention(q, kc, vc, dev([[pages - 3 + i for i in order]]), dev([n]), scale=0.1, value_dim=dv,
                            key_scales=ks, value_scales=vs)
    # the same rows in a cache of three pages: the same bits
    k3, v3, ks3, vs3 = small(kc), small(vc), small(ks), small(vs)
    want = C.paged_attention(q, k3, v3, dev([order]), dev([n]), scale=0.1, value_dim=dv, key_scales=ks3, value_scales=vs3)
    assert torch.equal(got, want) and got.isfinite().all()
    rows = f64(keys) if fmt == "bf16" else P.mx_values(*P.mx_rows(f64(keys)))
    k64 = f64(k3) if fmt == "bf16" else P.mx_values(k3.cpu().numpy(), ks3.cpu().numpy())
    np.testing.assert_array_equal(k64.transpose(0, 2, 1, 3).reshape(3 * page, kv_heads, dk), rows)
    assert not kc[:-3].any() and (vc is None or not vc[:-3].any())


@pytest.mark.parametrize("what", ["pages", "page", "blocks", "free"])
def test_sizes_that_pass_32_bits(C, what):
    """Tensors with an axis beyond 2^32, whose low bits alone would be a size that fits: refused by all."""
    from glm53flash.contract import ContractError
    long = (1 << 32) + 8
    lens = dev([3])
    q = torch.zeros((1, 2, 8), device="cuda", dtype=torch.bfloat16)
    try:
        if what in ("pages", "page"):
            shape = (long, 1, 1, 8) if what == "pages" else (1, 1, long, 8)
            kc = torch.empty(shape, device="cuda", dtype=torch.bfloat16)  # 69 GB, never touched
            with pytest.raises(ContractError, match="32 bits"):
                C.paged_attention(q, kc, None, dev([[0]]), lens, scale=1.0, value_dim=8)
            with pytest.raises(ContractError, match="32 bits"):
                C.cache_write(q[:, :1], None, dev([-1]), kc, None)
        else:
            wide = torch.zeros((1, long), device="cuda", dtype=torch.int32)  # 17 GB
            if what == "blocks":
                kc = torch.zeros((1, 1, 1, 8), device="cuda", dtype=torch.bfloat16)
                with pytest.raises(ContractError, match="32 bits"):
                    C.paged_attention(q, kc, None, wide, lens, scale=1.0, value_dim=8)
            tables, free = (wide, dev([0])) if what == "blocks" else (dev([[0]]), wide.view(-1))
            with pytest.raises(ContractError, match="32 bits"):
                C.cache_step(dev([0]), dev([0]), dev([0]), tables, free, dev([1]), page_size=1, max_tokens=1)
    finally:
        kc = wide = tables = free = None
        torch.cuda.empty_cache()


@pytest.mark.parametrize("N, heads, page, dk, dv, fmt, pad", [
    (5, 33, 4, 96, 64, "bf16", 8), (5, 33, 4, 96, 64, "mxfp8", 0), (70, 64, 16, 128, 128, "mxfp8", 8),
    (2, 65536, 1, 8, 0, "bf16", 0), (3, 1, 1, 1024, 1024, "mxfp8", 0), (2500, 1, 16, 8, 8, "bf16", 8)])
def test_write_wide_and_narrow_tokens(C, N, heads, page, dk, dv, fmt, pad):
    """Tokens of more pieces than a workgroup has threads, of as few as two, and the widest rows."""
    test_write(C, N, heads, page, dk, dv, fmt, pad)


@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
@pytest.mark.parametrize("dk, dv", [(64, 64), (192, 128), (256, 256), (320, 256), (576, 64)])
def test_attend_latents_of_other_forms(C, fmt, dk, dv):
    """Values that are the keys' first channels, at the grouped form's widths and at others."""
    attend_case(C, np.random.default_rng(dk), 3, 2, 8, 2, dk, dv, [70, 200, 1], 16, fmt, latent=True)


@pytest.mark.parametrize("dk, dv, latent", [(64, 64, False), (576, 512, True), (32, 32, False)])
def test_attend_most_rows(C, dk, dv, latent):
    """1024 heads of one kv head and 16 new tokens: 16384 rows share every position."""
    attend_case(C, np.random.default_rng(dk), 1, 16, 1024, 1, dk, dv, [70], 16, latent=latent)


@pytest.mark.parametrize("heads, dk, dv, latent", [(2, 64, 64, False), (1, 576, 512, True), (1, 32, 32, False)])
def test_attend_most_requests(C, heads, dk, dv, latent):
    """65535 short requests: the same bits as in batches of 5000, since no request here is cut."""
    gen = torch.Generator(device="cuda").manual_seed(dk)
    B, page, pages = 65535, 4, 3000
    kc = torch.randn((pages, 1, page, dk), generator=gen, device="cuda", dtype=torch.bfloat16)
    vc = None if latent else torch.randn((pages, 1, page, dv), generator=gen, device="cuda", dtype=torch.bfloat16)
    table = torch.randint(0, pages, (B, 2), generator=gen, device="cuda", dtype=torch.int32)
    lens = torch.randint(0, 9, (B,), generator=gen, device="cuda", dtype=torch.int32)
    q = torch.randn((B, heads, dk), generator=gen, device="cuda", dtype=torch.bfloat16)
    got = C.paged_attention(q, kc, vc, table, lens, scale=0.1, value_dim=dv)
    for b in range(0, B, 5000):
        some = slice(b, b + 5000)
        want = C.paged_attention(q[some], kc, vc, table[some], lens[some], scale=0.1, value_dim=dv)
        assert torch.equal(got[some], want)
    assert (got[lens == 0] == 0).all() and not (got[lens > 0] == 0).all(-1).any()
