"""Oracle of the paged attention cache: the step's bookkeeping in plain integers,
the MXFP8 rows and the attention in 64 bits (numpy)."""

from __future__ import annotations

import numpy as np

from .moe_oracle import bf16_bits_to_f32  # noqa: F401  (re-exported for the tests)

OUT_OF_PAGES, TABLE_FULL, TOO_MANY_TOKENS, BAD_STATE = 1, 2, 4, 8


def step(new, lens, blocks, tables, free, num_free, page, max_tokens):
    """One step on copies of the state; returns a dict of what it leaves."""
    new, lens, blocks = (np.array(x, np.int64) for x in (new, lens, blocks))
    tables, free, top = tables.copy(), free.copy(), int(num_free)
    B, width = len(new), tables.shape[1]
    gone = new < 0
    n = np.where(gone, -1 - new, new)
    base, have = np.where(gone, 0, lens[:B]), np.where(gone, 0, blocks[:B])
    need = np.maximum(0, -(-(base + n) // page) - have)
    given = int(blocks[:B][gone].sum())
    status = 0
    if top + given < need.sum():
        status |= OUT_OF_PAGES
    if (base + n > width * page).any():
        status |= TABLE_FULL
    if n.sum() > max_tokens:
        status |= TOO_MANY_TOKENS
    if (lens[:B] < 0).any() or (blocks[:B] < 0).any() or (blocks[:B] > width).any() or \
            (base > have * page).any() or top < 0 or top + given > len(free):
        status |= BAD_STATE
    slots, positions = np.full(max_tokens, -1, np.int32), np.zeros(max_tokens, np.int32)
    kv, cu = lens[:B].copy(), np.zeros(B + 1, np.int64)
    if status == 0:
        for b in range(B):
            if gone[b]:
                for j in range(blocks[b]):
                    free[top] = tables[b, j]
                    tables[b, j] = -1
                    top += 1
                blocks[b] = 0
        t = 0
        for b in range(B):
            for _ in range(need[b]):
                top -= 1
                tables[b, blocks[b]] = free[top]
                blocks[b] += 1
            for pos in range(base[b], base[b] + n[b]):
                slots[t], positions[t] = tables[b, pos // page] * page + pos % page, pos
                t += 1
            kv[b], cu[b + 1] = base[b] + n[b], t
    return {"kv_lens": kv, "cu_new": cu, "slots": slots, "positions": positions, "status": status,
            "blocks": blocks, "tables": tables, "free_pages": free, "num_free": top}


E4M3 = np.array([np.nan if c & 0x7f == 0x7f else (-1.0 if c & 0x80 else 1.0) *
                 ((c & 7) * 2.0 ** -9 if c & 0x78 == 0 else (1 + (c & 7) / 8) * 2.0 ** (((c >> 3) & 15) - 7))
                 for c in range(256)])


def mx_rows(x):
    """f64 rows [..., dim] (bf16 values) -> (E4M3 codes, E8M0 bytes): per 32 channels the smallest
    exponent >= -124 with amax <= 448 2^e, nearest even; what is not finite becomes NaN."""
    g = x.reshape(*x.shape[:-1], -1, 32)
    fine = np.isfinite(g)
    amax = np.where(fine, np.abs(g), 0).max(-1)
    m, e = np.frexp(amax / 448.0)  # amax / 448 = m 2^e, m in [0.5, 1)
    e = np.where(amax == 0, -124, np.maximum(np.where(m == 0.5, e - 1, e), -124))
    v = np.where(fine, g, 0) * 2.0 ** -e[..., None].astype(np.float64)
    values = E4M3[:0x7f]
    hi = np.clip(np.searchsorted(values, np.abs(v)), 0, 126)
    lo = np.maximum(hi - 1, 0)
    up, down = values[hi] - np.abs(v), np.abs(v) - values[lo]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo).astype(np.uint8)
    code = np.where(fine, code | np.where(np.signbit(v), 0x80, 0), 0x7f).astype(np.uint8)
    return code.reshape(x.shape), (e + 127).astype(np.uint8)


def mx_values(codes, scales):
    """What codes and scale bytes stand for, f64."""
    v = E4M3[codes].reshape(*codes.shape[:-1], -1, 32)
    return (v * 2.0 ** (scales.astype(np.float64) - 127)[..., None]).reshape(codes.shape)


def attend(q, keys, values, tables, lens, scale):
    """q f64 [B, q_len, heads, dk]; keys, values f64 [pages, kv_heads, page, d].  Returns (out, spread, reach):
    out [B, q_len, heads, dv]; spread the same with |v| in v's place; reach [B, q_len, heads] the largest
    scale sum_c |q_c k_c| of a row's positions, which the error of its scores goes by."""
    B, q_len, heads, _ = q.shape
    pages, kv_heads, page, dv = values.shape
    out = np.zeros((B, q_len, heads, dv))
    spread, reach = np.zeros_like(out), np.zeros((B, q_len, heads))
    for b in range(B):
        n = max(0, min(int(lens[b]), tables.shape[1] * page))
        pos = np.arange(n)
        ids = tables[b, pos // page]
        fine = (ids >= 0) & (ids < pages)
        pos, ids = pos[fine], ids[fine]
        for t in range(q_len):
            seen = pos < n - (q_len - 1 - t)
            if not seen.any():
                continue
            at, off = ids[seen], pos[seen] % page
            for h in range(heads):
                g = h // (heads // kv_heads)
                k, v = keys[at, g, off], values[at, g, off]
                s = scale * (k @ q[b, t, h])
                p = np.exp(s - s.max())
                p /= p.sum()
                out[b, t, h] = p @ v
                spread[b, t, h] = p @ np.abs(v)
                reach[b, t, h] = abs(scale) * (np.abs(k) @ np.abs(q[b, t, h])).max()
    return out, spread, reach
