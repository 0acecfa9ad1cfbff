"""The paged attention cache's operators as cases that can be timed and compared.

Three kinds of case:

* ``step``    ``cache_step``: request lengths -> pages taken and given back, block tables, slots and positions
* ``write``   ``cache_write``: new keys and values (or latent rows) into the pages, as bf16 or as MXFP8
* ``attend``  ``paged_attention``: the new tokens of a batch over their cached history, keys and values apart
              or a latent cache whose rows' first channels are the values

With ``own`` false, ``run`` computes them in elementary torch operations (32 bits, rounded once at the end); with ``own``
true it calls the package.  Lengths follow from the case alone, values and the order of requests and pages from the seed.
"""

import functools
import math
import os
import random
import sys

import numpy as np
import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@functools.lru_cache(maxsize=1)
def _package():
    src = os.path.join(_ROOT, "src")
    if src not in sys.path:
        sys.path.insert(0, src)
    from glm53flash import paged_cache
    return paged_cache


# ---------------------------------------------------------------- cases

def _step(name, B, page, blocks, **more):
    return {"kind": "step", "name": name, "B": B, "page": page, "blocks": blocks, **more}


def _write(name, N, heads, key_dim, value_dim, fmt, page=16):
    return {"kind": "write", "name": name, "N": N, "kv_heads": heads, "key_dim": key_dim,
            "value_dim": value_dim, "fmt": fmt, "page": page}


def _attend(name, B, shortest, longest, heads, kv_heads, key_dim, value_dim, fmt="bf16", q_len=1, page=16,
            latent=False, spread=1):
    return {"kind": "attend", "name": name, "B": B, "shortest": shortest, "longest": longest, "heads": heads,
            "kv_heads": kv_heads, "key_dim": key_dim, "value_dim": value_dim, "fmt": fmt, "q_len": q_len,
            "page": page, "latent": latent, "spread": spread}


def listed():
    return [
        # the smallest: one decode step of a batch, one token each
        _step("step_decode_b64", 64, 16, 1024, mode="decode", longest=9000),
        # admission: finished requests give their pages back, prompts of ragged lengths take them
        _step("step_prefill_b48", 48, 16, 256, mode="replace", longest=2500),
        # a decode step's new keys and values
        _write("write_b64", 64, 8, 128, 128, "bf16"),
        # a prefill chunk into an MXFP8 cache
        _write("write_t7777_mxfp8", 7777, 8, 128, 128, "mxfp8"),
        # a prefill chunk of latent rows
        _write("write_latent_t4001", 4001, 1, 576, 0, "bf16", 64),
        # one user, a short history: latency
        _attend("attend_b1_l517", 1, 517, 517, 32, 8, 128, 128),
        # a serving batch with ragged histories
        _attend("attend_b32_ragged", 32, 61, 16000, 32, 8, 128, 128, spread=3),
        # two very long histories: the length has to be split
        _attend("attend_b2_l131000", 2, 130900, 131000, 64, 8, 128, 128),
        # the two-token verify step of a large batch on an MXFP8 cache
        _attend("attend_verify_b96_mxfp8", 96, 33, 8000, 32, 4, 128, 128, "mxfp8", 2, 64),
        # every query head with keys of its own, narrow heads, odd lengths
        _attend("attend_heads_b45", 45, 1, 3001, 16, 16, 64, 64, page=32),
        # a serving batch on a latent cache
        _attend("attend_latent_b64", 64, 100, 8100, 64, 1, 576, 512, page=64, latent=True, spread=2),
        # few long histories on a latent MXFP8 cache, the verify step
        _attend("attend_latent_b5_mxfp8", 5, 20000, 50001, 64, 1, 576, 512, "mxfp8", 2, 64, True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["step", "write", "attend", "attend", "latent"])
    page = rng.choice([8, 16, 32, 64])
    if kind == "step":
        B = _log_int(rng, 1, 1000)
        if rng.random() < 0.5:
            return {"kind": "step", "mode": "decode", "B": B, "page": page, "longest": _log_int(rng, 100, 9000),
                    "blocks": 9000 // page + 64}
        longest = _log_int(rng, 40, 3000 if B < 50 else 400)
        return {"kind": "step", "mode": "replace", "B": B, "page": page, "longest": longest,
                "blocks": longest // page + 2}
    fmt = rng.choice(["bf16", "mxfp8"])
    if kind == "write":
        heads, kd, vd = rng.choice([(1, 576, 0), (2, 128, 128), (4, 64, 64), (8, 128, 128), (16, 64, 64), (4, 256, 256)])
        return {"kind": "write", "N": _log_int(rng, 1, 9000), "kv_heads": heads, "key_dim": kd, "value_dim": vd,
                "fmt": fmt, "page": page}
    q_len = rng.choice([1, 1, 2, 4])
    latent = kind == "latent"
    if latent:
        heads, kv_heads, kd, vd = rng.choice([16, 32, 64, 128]), 1, 576, 512
    else:
        kv_heads = rng.choice([1, 2, 4, 8, 16])
        heads = kv_heads * rng.choice([1, 2, 4, 8])
        kd = vd = rng.choice([64, 128, 128, 256])
    B = _log_int(rng, 1, 200)
    # no more than 400 M cached values and 40 GFLOP, whatever the lengths that come out
    most = max(2, min(100000, int(4e8 / (B * kv_heads * (kd + vd))), int(2e10 / (B * heads * q_len * (kd + vd)))))
    longest = _log_int(rng, min(40, most), most)
    return {"kind": "attend", "B": B, "shortest": max(1, int(longest * rng.choice([0.02, 0.3, 1.0]))), "longest": longest,
            "heads": heads, "kv_heads": kv_heads, "key_dim": kd, "value_dim": vd, "fmt": fmt, "q_len": q_len,
            "page": page, "latent": latent, "spread": rng.choice([1, 3])}


def _lengths(case):
    """The requests' lengths: spread over their logarithm, a function of the case alone."""
    lo, hi = case.get("shortest", 1), case["longest"]
    rng = random.Random(7 * case["B"] + hi)
    return [hi if b == 0 else _log_int(rng, lo, hi) for b in range(case["B"])]


# ---------------------------------------------------------------- inputs

def _quantise(x):
    """MXFP8 of [..., 32 g] values: e the smallest exponent from -124 on with amax <= 448 2^e over 32 channels."""
    g = x.float().unflatten(-1, (-1, 32))
    m, e = torch.frexp(g.abs().amax(-1, keepdim=True))  # amax = m 2^e, m in [0.5, 1)
    e = torch.where(m == 0, torch.full_like(e, -124), e - 9 + (m > 0.875).int()).clamp_min(-124)
    codes = (g * ((127 - e.int()) << 23).view(torch.float32)).to(torch.float8_e4m3fn)  # times 2^-e, exact
    return codes.flatten(-2).view(torch.uint8), (e + 127).squeeze(-1).to(torch.uint8)


def _values(cache, scales):
    """What a cache's rows stand for, in 32 bits."""
    if scales is None:
        return cache.float()
    x = cache.view(torch.float8_e4m3fn).float().unflatten(-1, (-1, 32))
    return (x * (scales.int().unsqueeze(-1) << 23).view(torch.float32)).flatten(-2)  # byte b is 2^(b - 127)


def _cache(pages, case, dim, gen):
    """A filled cache [pages, kv_heads, page, dim], as a program finds it after its earlier steps."""
    x = torch.randn((pages, case["kv_heads"], case["page"], dim), generator=gen, device="cuda", dtype=torch.bfloat16)
    return _quantise(x) if case["fmt"] == "mxfp8" else (x, None)


def _pages(counts, pool, width, gen):
    """A block table of the requests' pages, dealt out of a shuffled pool, and the pages left."""
    order = torch.randperm(pool, generator=gen, device="cuda").int()
    counts = torch.tensor(counts, device="cuda")
    first = counts.cumsum(0) - counts
    col = torch.arange(width, device="cuda")
    taken = order[(first[:, None] + col).clamp_max(pool - 1)]
    return torch.where(col < counts[:, None], taken, -1), order, int(counts.sum())


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    page = case["page"]
    if case["kind"] == "write":
        N, H = case["N"], case["kv_heads"]
        pages = -(-N * 5 // (4 * page)) + 1
        s = {"slots": torch.randperm(pages * page, generator=gen, device="cuda")[:N].int()}
        s["keys"] = torch.randn((N, H, case["key_dim"]), generator=gen, device="cuda", dtype=torch.bfloat16)
        s["key_cache"], s["key_scales"] = _cache(pages, case, case["key_dim"], gen)
        s["values"] = s["value_cache"] = s["value_scales"] = None
        if case["value_dim"]:
            s["values"] = torch.randn((N, H, case["value_dim"]), generator=gen, device="cuda", dtype=torch.bfloat16)
            s["value_cache"], s["value_scales"] = _cache(pages, case, case["value_dim"], gen)
        return {**s, "kind": "write"}
    lens = _lengths(case)
    random.Random(seed).shuffle(lens)
    if case["kind"] == "step":
        counts = [-(-n // page) for n in lens]
        pool = sum(counts) + case["B"] * 2 + 7
        new = [1] * case["B"]
        if case["mode"] == "replace":
            new = list(lens)
            random.Random(seed + 1).shuffle(new)
            new = [-1 - n for n in new]
        tables, order, used = _pages(counts, pool, case["blocks"], gen)
        return {"kind": "step", "page": page, "max_tokens": sum(n if n >= 0 else -1 - n for n in new) + 5,
                "new_lens": torch.tensor(new, dtype=torch.int32, device="cuda"),
                "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"),
                "blocks": torch.tensor(counts, dtype=torch.int32, device="cuda"), "tables": tables.contiguous(),
                "free_pages": torch.cat([order[used:], order[:used]]).contiguous(),
                "num_free": torch.tensor([pool - used], dtype=torch.int32, device="cuda")}
    counts = [-(-n // page) for n in lens]
    pool = sum(counts) + 3
    tables, _, _ = _pages(counts, pool, max(counts), gen)
    s = {"kind": "attend", "tables": tables.contiguous(), "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"),
         "value_dim": case["value_dim"], "scale": 1.0 / math.sqrt(case["key_dim"])}
    s["query"] = case["spread"] * torch.randn((case["B"], case["q_len"], case["heads"], case["key_dim"]), generator=gen,
                                              device="cuda", dtype=torch.bfloat16)
    s["key_cache"], s["key_scales"] = _cache(pool, case, case["key_dim"], gen)
    s["value_cache"] = s["value_scales"] = None
    if not case["latent"]:
        s["value_cache"], s["value_scales"] = _cache(pool, case, case["value_dim"], gen)
    return s


# ---------------------------------------------------------------- the plain forms

def _plain_step(s):
    new, lens, blocks, tables, free = s["new_lens"], s["lens"], s["blocks"], s["tables"], s["free_pages"]
    page, B, width, pool = s["page"], new.numel(), s["tables"].shape[1], s["free_pages"].numel()
    dev = new.device
    nf = s["num_free"].long()
    gone = new < 0
    n = torch.where(gone, -1 - new, new).long()
    base = torch.where(gone, 0, lens).long()
    have = torch.where(gone, 0, blocks).long()
    given = torch.where(gone, blocks, 0).long()
    total = base + n
    need = ((total + page - 1) // page - have).clamp_min(0)
    left = nf + given.sum() - need.sum()
    sound = ((lens >= 0) & (blocks >= 0) & (blocks <= width) & (base <= have * page)).all()
    sound = sound & (nf >= 0) & (nf + given.sum() <= pool)
    status = ((left < 0).int() + 2 * (total > width * page).any().int() + 4 * (n.sum() > s["max_tokens"]).int()
              + 8 * (~sound).int())
    ok = status == 0
    col = torch.arange(width, device=dev)
    # pages given back go on top of the free ones, in the requests' order
    to = nf + (given.cumsum(0) - given)[:, None] + col
    to = torch.where(ok & (col < given[:, None]), to, pool)
    stack = torch.cat([free, free.new_zeros(1)]).scatter_(0, to.flatten(), tables.flatten())
    # new pages come from the top, requests in order
    is_new = (col >= have[:, None]) & (col < (have + need)[:, None])
    at = nf + given.sum() - 1 - ((need.cumsum(0) - need)[:, None] + col - have[:, None])
    taken = stack[at.clamp(0, pool - 1)]
    after = torch.where(is_new, taken, torch.where(gone[:, None], -1, tables))
    tables.copy_(torch.where(ok, after, tables))
    free.copy_(stack[:pool])
    kv_lens = torch.where(ok, total, lens).int()
    blocks.copy_(torch.where(ok, have + need, blocks))
    s["num_free"].copy_(torch.where(ok, left, nf))
    cu = torch.cat([n.new_zeros(1), n.cumsum(0)]) * ok
    t = torch.arange(s["max_tokens"], device=dev)
    r = torch.searchsorted(cu[1:].contiguous(), t, right=True).clamp_max(B - 1)
    there = t < cu[-1]
    pos = torch.where(there, base[r] + t - cu[r], 0)
    slots = torch.where(there, tables[r, pos // page].long() * page + pos % page, -1)
    return {"kv_lens": kv_lens, "cu_new": cu.int(), "slots": slots.int(), "positions": pos.int(), "status": status.int(),
            "blocks": blocks, "tables": tables, "free_pages": free, "num_free": s["num_free"]}


def _put(cache, scales, rows, slots):
    page = cache.shape[2]
    at, off = (slots // page).long(), (slots % page).long()
    if scales is None:
        cache[at, :, off] = rows
    else:
        codes, e = _quantise(rows)
        cache[at, :, off] = codes
        scales[at, :, off] = e


def _written(s):
    out = [s["key_cache"], s["value_cache"]]
    if s["key_scales"] is not None:  # 8-bit codes as the values they stand for
        out = [None if x is None else x.view(torch.float8_e4m3fn) for x in out]
    return {"keys": out[0], "values": out[1], "key_scales": s["key_scales"], "value_scales": s["value_scales"]}


def _history(cache, scales, tables):
    """[B, kv_heads, width, dim] of the pages that the tables name."""
    x = _values(cache[tables], None if scales is None else scales[tables])  # [B, blocks, H, page, dim]
    return x.transpose(1, 2).flatten(2, 3)


def _plain_attend(s):
    q = s["query"].float()
    B, q_len, heads, _ = q.shape
    tables = s["tables"].clamp_min(0).long()
    k = _history(s["key_cache"], s["key_scales"], tables)
    H, width = k.shape[1], k.shape[2]
    if s["value_cache"] is None:
        v = k[..., :s["value_dim"]]
    else:
        v = _history(s["value_cache"], s["value_scales"], tables)
    # rows (token, head of the group) of one kv head together
    q = q.view(B, q_len, H, heads // H, -1).transpose(1, 2).reshape(B, H, q_len * (heads // H), -1)
    last = s["lens"][:, None] - (q_len - 1) + torch.arange(q_len, device=q.device)  # positions below it are seen
    seen = torch.arange(width, device=q.device) < last.repeat_interleave(heads // H, 1)[:, None, :, None]
    scores = torch.matmul(q, k.transpose(-1, -2)) * s["scale"]
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    w = torch.where(seen, torch.exp(scores - top), 0.0)
    total = w.sum(-1, keepdim=True)
    out = torch.matmul(w, v) / torch.where(total == 0, 1.0, total)
    out = out.view(B, H, q_len, heads // H, -1).transpose(1, 2).reshape(B, q_len, heads, -1)
    return out.to(torch.bfloat16)


def run(state):
    s = state
    if s["kind"] == "step":
        if not own:
            return _plain_step(s)
        step = _package().cache_step(s["new_lens"], s["lens"], s["blocks"], s["tables"], s["free_pages"], s["num_free"],
                                     page_size=s["page"], max_tokens=s["max_tokens"])
        return {"kv_lens": step.kv_lens, "cu_new": step.cu_new, "slots": step.slots, "positions": step.positions,
                "status": step.status, "blocks": s["blocks"], "tables": s["tables"], "free_pages": s["free_pages"],
                "num_free": s["num_free"]}
    if s["kind"] == "write":
        if not own:
            _put(s["key_cache"], s["key_scales"], s["keys"], s["slots"])
            if s["values"] is not None:
                _put(s["value_cache"], s["value_scales"], s["values"], s["slots"])
            return _written(s)
        _package().cache_write(s["keys"], s["values"], s["slots"], s["key_cache"], s["value_cache"],
                               key_scales=s["key_scales"], value_scales=s["value_scales"])
        return _written(s)
    if not own:
        return _plain_attend(s)
    return _package().paged_attention(s["query"], s["key_cache"], s["value_cache"], s["tables"], s["lens"],
                                      scale=s["scale"], value_dim=s["value_dim"], key_scales=s["key_scales"],
                                      value_scales=s["value_scales"])


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    if case["kind"] == "step":
        lens, page, B = _lengths(case), case["page"], case["B"]
        if case["mode"] == "decode":
            tokens, pages = B, sum(n % page == 0 for n in lens)
        else:  # every request's pages given back and as many taken
            tokens, pages = sum(lens), 2 * sum(-(-n // page) for n in lens)
        return {"bytes": 4 * (6 * B + 2 * pages + 2 * tokens), "flops": 0}
    row = case["kv_heads"] * (case["key_dim"] + (case["value_dim"] if not case.get("latent") else 0))
    held = row * 2 if case["fmt"] == "bf16" else row + row // 32
    if case["kind"] == "write":
        return {"bytes": case["N"] * (2 * row + held + 4), "flops": 0}
    lens, rows = _lengths(case), case["q_len"] * case["heads"]
    dims = case["key_dim"] + case["value_dim"]
    return {"bytes": sum(lens) * held + case["B"] * rows * dims * 2 + 4 * sum(-(-n // case["page"]) for n in lens),
            "flops": 2 * rows * dims * sum(lens)}


# ---------------------------------------------------------------- from the definitions, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "step":
        page, width = s["page"], s["tables"].shape[1]
        new, lens, blocks = s["new_lens"].tolist(), s["lens"].tolist(), s["blocks"].tolist()
        tables, free, top = s["tables"].cpu().numpy().copy(), s["free_pages"].tolist(), int(s["num_free"])
        kv, cu, slots, positions = [], [0], [], []
        for b, n in enumerate(new):
            if n < 0:
                for j in range(blocks[b]):
                    free[top] = int(tables[b, j])
                    top += 1
                tables[b], lens[b], blocks[b] = -1, 0, 0
        for b, n in enumerate(new):
            n = n if n >= 0 else -1 - n
            while blocks[b] * page < lens[b] + n:
                top -= 1
                tables[b, blocks[b]] = free[top]
                blocks[b] += 1
            for p in range(lens[b], lens[b] + n):
                slots.append(int(tables[b, p // page]) * page + p % page)
                positions.append(p)
            kv.append(lens[b] + n)
            cu.append(cu[-1] + n)
        rest = s["max_tokens"] - len(slots)
        return {"kv_lens": np.array(kv, np.int32), "cu_new": np.array(cu, np.int32),
                "slots": np.array(slots + [-1] * rest, np.int32), "positions": np.array(positions + [0] * rest, np.int32),
                "status": np.zeros(1, np.int32), "blocks": np.array(blocks, np.int32), "tables": tables,
                "free_pages": np.array(free, np.int32), "num_free": np.array([top], np.int32)}
    if case["kind"] == "write":
        out = {"keys": None, "values": None, "key_scales": None, "value_scales": None}
        for name, one in (("keys", "key"), ("values", "value")):
            if s[name] is None:
                continue
            cache = s[one + "_cache"]
            mx = case["fmt"] == "mxfp8"
            held = (cache.view(torch.float8_e4m3fn) if mx else cache).double()
            pages, H, page, dim = held.shape
            flat = held.transpose(1, 2).reshape(pages * page, H, dim).clone()
            rows = s[name].double()
            if mx:
                scales = s[one + "_scales"].transpose(1, 2).reshape(pages * page, H, dim // 32).clone()
                peak = rows.view(-1, H, dim // 32, 32).abs().amax(-1)
                e = torch.full_like(peak, -124).long()
                for up in range(-123, 121):  # the smallest exponent that keeps the group within 448
                    e = torch.where(peak > 448 * 2.0 ** (up - 1), up, e)
                rows = rows * torch.pow(torch.full_like(peak, 0.5), e.double()).repeat_interleave(32, -1)
                scales[s["slots"].long()] = (e + 127).to(torch.uint8)
                out[one + "_scales"] = scales.view(pages, page, H, -1).transpose(1, 2).contiguous()
            flat[s["slots"].long()] = rows
            out[name] = flat.view(pages, page, H, dim).transpose(1, 2).contiguous()
        return out
    q = s["query"].double()
    B, q_len, heads, _ = q.shape
    out = torch.zeros((B, q_len, heads, case["value_dim"]), dtype=torch.float64, device=q.device)

    def rows_of(cache, scales, pages, n):
        x = cache[pages]
        if scales is not None:
            x = (x.view(torch.float8_e4m3fn).double().unflatten(-1, (-1, 32))
                 * torch.exp2(scales[pages].double() - 127).unsqueeze(-1)).flatten(-2)
        return x.double().transpose(0, 1).flatten(1, 2)[:, :n]

    for b, n in enumerate(s["lens"].tolist()):
        pages = s["tables"][b, :-(-n // case["page"])].long()
        k = rows_of(s["key_cache"], s["key_scales"], pages, n)
        v = k[..., :case["value_dim"]] if case["latent"] else rows_of(s["value_cache"], s["value_scales"], pages, n)
        group = heads // case["kv_heads"]
        for t in range(q_len):
            m = n - (q_len - 1 - t)
            if m <= 0:
                continue
            a = torch.softmax(torch.matmul(q[b, t].view(-1, group, case["key_dim"]), k[:, :m].transpose(1, 2)) * s["scale"], -1)
            out[b, t] = torch.matmul(a, v[:, :m]).view(heads, -1)
    return out
