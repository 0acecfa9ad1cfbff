"""The block-scaled 8-bit operators as cases that can be timed and compared.

Four kinds of case:

* ``quantise``  ``quantize_rows``: rows -> E4M3 codes with an f32 scale for each 128 channels
* ``norm``      ``add_rms_norm``: the residual's addition, the RMS norm and its quantisation
* ``linear``    ``linear``: rows (quantised already, or bf16) x a weight with a scale for each 128 x 128 block
* ``gate_up``   ``gate_up``: two such products, the limited SwiGLU of them and its quantisation

With ``own`` false, ``run`` computes them in elementary torch operations (32 bits, rounded once at the end); with ``own``
true it calls the package.
"""

import functools
import math
import os
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_TINY = 448.0 * 2.0 ** -126  # a group's scale is 2^-126 at least
_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_EPS = 1e-6


@functools.lru_cache(maxsize=1)
def _package():
    src = os.path.join(_ROOT, "src")
    if src not in sys.path:
        sys.path.insert(0, src)
    from glm53flash import fp8_block
    return fp8_block


# ---------------------------------------------------------------- cases

def _quantise_case(name, T, K, dtype="bf16"):
    return {"kind": "quantise", "name": name, "T": T, "K": K, "dtype": dtype}


def _norm(name, T, K, dtype="bf16", residual="bf16"):
    return {"kind": "norm", "name": name, "T": T, "K": K, "dtype": dtype, "residual": residual}


def _linear(name, T, K, N, rows="fp8"):
    return {"kind": "linear", "name": name, "T": T, "K": K, "N": N, "rows": rows}


def _gate_up(name, T, K, N, rows="fp8"):
    return {"kind": "gate_up", "name": name, "T": T, "K": K, "N": N, "rows": rows, "limit": 10.0}


def listed():
    return [
        # the smallest: one token's norm in front of its projections
        _norm("norm_t1", 1, 4096),
        # a prompt chunk of odd length, the residual kept in 32 bits
        _norm("norm_t1500_f32", 1500, 2048, "f32", "f32"),
        # a long prompt's norm
        _norm("norm_t8191", 8191, 4096),
        # a decode batch whose rows come from elsewhere (the attention's output)
        _quantise_case("quantise_t64", 64, 4096),
        # the same of a long prompt
        _quantise_case("quantise_t7777", 7777, 4096),
        # one token's output projection, from bf16 rows: latency and the weights' bytes
        _linear("linear_t1", 1, 4096, 4096, "bf16"),
        # a decode batch through a latent projection: widths off the 128 blocks
        _linear("linear_t48_ragged", 48, 2048, 576),
        # a prompt chunk of a few hundred tokens
        _linear("linear_t333", 333, 4096, 4096),
        # a long prompt
        _linear("linear_t4096", 4096, 4096, 4096),
        # the verify step of two tokens through a shared expert's first half
        _gate_up("gate_up_t2", 2, 2048, 768, "bf16"),
        # a decode batch
        _gate_up("gate_up_t64", 64, 4096, 2048),
        # a long prompt of odd length
        _gate_up("gate_up_t4001", 4001, 4096, 2048),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quantise", "norm", "linear", "linear", "gate_up"])
    T = _log_int(rng, 1, 8000)
    K = 16 * _log_int(rng, 8, 512)
    if kind in ("quantise", "norm"):
        K = min(K, 16 * (33 * 10 ** 6 // (16 * T)))  # no more than 33 M values
        case = {"kind": kind, "T": T, "K": K, "dtype": rng.choice(["bf16", "f32"])}
        if kind == "norm":
            case["residual"] = rng.choice(["bf16", "f32"])
        return case
    N = 16 * _log_int(rng, 8, 512)
    if kind == "linear":
        N -= rng.choice([0, 0, 1, 5])
    products = 1 if kind == "linear" else 2
    while products * T * K * N > 2 ** 36:  # no more than 137 GFLOP
        T = T // 2
    case = {"kind": kind, "T": T, "K": K, "N": N, "rows": rng.choice(["bf16", "fp8"])}
    if kind == "gate_up":
        case["limit"] = rng.choice([0.0, 2.0, 10.0])
    return case


# ---------------------------------------------------------------- inputs

def _rows(T, K, gen, dtype=torch.bfloat16):
    """Activations: normal values whose rows differ in size, a few channels of which are far larger than the others."""
    x = torch.randn((T, K), generator=gen, device="cuda")
    x *= torch.exp2(torch.randn((T, 1), generator=gen, device="cuda"))
    loud = torch.rand(K, generator=gen, device="cuda") < 0.004
    return (x * torch.where(loud, 12.0, 1.0)).to(dtype)


def _weight(N, K, gen):
    """A weight as a checkpoint holds it: E4M3 codes [N, K] and f32 scales for each 128 x 128 block."""
    n, k = -(-N // 128), -(-K // 128)
    w = torch.randn((N, K), generator=gen, device="cuda") * 112.0
    codes = w.clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    size = torch.exp2(0.5 * torch.randn((n, k), generator=gen, device="cuda"))
    return codes, size / (112.0 * math.sqrt(K))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    T, K = case["T"], case["K"]
    s = {"kind": case["kind"]}
    if case["kind"] in ("quantise", "norm"):
        s["x"] = _rows(T, K, gen, _TYPES[case["dtype"]])
        if case["kind"] == "norm":
            s["residual"] = 2 * _rows(T, K, gen, _TYPES[case["residual"]])
            s["weight"] = 1 + 0.1 * torch.randn(K, generator=gen, device="cuda")
        return s
    x = _rows(T, K, gen)
    s["x"] = x if case["rows"] == "bf16" else _quantise(x.float())
    if case["kind"] == "linear":
        s["w"], s["w_scales"] = _weight(case["N"], K, gen)
        return s
    s["gate"], s["gate_scales"] = _weight(case["N"], K, gen)
    s["up"], s["up_scales"] = _weight(case["N"], K, gen)
    s["limit"] = case["limit"]
    return s


# ---------------------------------------------------------------- the plain forms

def _groups(y):
    """[T, K] -> [T, groups, 128], zeros behind the last channel."""
    return torch.nn.functional.pad(y, (0, -y.shape[-1] % 128)).unflatten(-1, (-1, 128))


def _quantise(y):
    """Codes u8 [T, K] and scales f32 [T, groups] of f32 rows: scale = amax / 448, code = e4m3(y * (448 / amax))."""
    g = _groups(y)
    amax = torch.where(torch.isfinite(g), g.abs(), 0.0).amax(-1).clamp_min(_TINY)
    most = torch.full_like(amax, 448.0)  # (a tensor: a quotient with a Python number is a product with its reciprocal)
    codes = (g * (most / amax).unsqueeze(-1)).to(torch.float8_e4m3fn)
    return codes.view(torch.uint8).flatten(1)[:, :y.shape[1]].contiguous(), amax / most


def _values(codes, scales):
    """What quantised rows stand for, in 32 bits."""
    return codes.view(torch.float8_e4m3fn).float() * scales.repeat_interleave(128, 1)[:, :codes.shape[1]]


def _weight_values(codes, scales):
    return _values(codes, scales.repeat_interleave(128, 0)[:codes.shape[0]])


def _coded(codes, scales):
    return {"codes": codes.view(torch.float8_e4m3fn), "scales": scales}


def _plain(s):
    if s["kind"] == "quantise":
        return _coded(*_quantise(s["x"].float()))
    if s["kind"] == "norm":
        h = s["x"].float() + s["residual"].float()
        y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + _EPS) * s["weight"]
        return {**_coded(*_quantise(y)), "residual": h.to(s["residual"].dtype)}
    x = s["x"]
    x = _values(*(_quantise(x.float()) if isinstance(x, torch.Tensor) else x))
    if s["kind"] == "linear":
        return torch.matmul(x, _weight_values(s["w"], s["w_scales"]).t()).to(torch.bfloat16)
    g = torch.matmul(x, _weight_values(s["gate"], s["gate_scales"]).t())
    u = torch.matmul(x, _weight_values(s["up"], s["up_scales"]).t())
    if s["limit"] > 0:
        g, u = g.clamp_max(s["limit"]), u.clamp(-s["limit"], s["limit"])
    return _coded(*_quantise(g / (1 + torch.exp(-g)) * u))


def run(state):
    s = state
    if not own:
        return _plain(s)
    f = _package()
    if s["kind"] == "quantise":
        return _coded(*f.quantize_rows(s["x"]))
    if s["kind"] == "norm":
        rows, residual = f.add_rms_norm(s["x"], s["weight"], _EPS, residual=s["residual"])
        return {**_coded(*rows), "residual": residual}
    x = s["x"] if isinstance(s["x"], torch.Tensor) else f.Fp8Rows(*s["x"])
    if s["kind"] == "linear":
        return f.linear(x, s["w"], s["w_scales"])
    return _coded(*f.gate_up(x, s["gate"], s["gate_scales"], s["up"], s["up_scales"], s["limit"]))


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    T, K = case["T"], case["K"]
    size = {"bf16": 2, "f32": 4}
    coded = K + 4 * -(-K // 128)
    if case["kind"] == "quantise":
        return {"bytes": T * (size[case["dtype"]] * K + coded), "flops": 0}
    if case["kind"] == "norm":
        return {"bytes": T * (size[case["dtype"]] * K + 2 * size[case["residual"]] * K + coded) + 4 * K, "flops": 0}
    N = case["N"]
    rows = T * (2 * K if case["rows"] == "bf16" else coded)
    weight = N * K + 4 * -(-N // 128) * -(-K // 128)
    if case["kind"] == "linear":
        return {"bytes": rows + weight + 2 * T * N, "flops": 2 * T * K * N}
    return {"bytes": rows + 2 * weight + T * (N + 4 * -(-N // 128)), "flops": 4 * T * K * N}


# ---------------------------------------------------------------- from the definitions, in 64 bits

def _exact_codes(y):
    """Unrounded codes and scales of f64 rows, a group at a time."""
    T, K = y.shape
    codes, scales = torch.empty_like(y), y.new_empty((T, -(-K // 128)))
    for g, k in enumerate(range(0, K, 128)):
        one = y[:, k:k + 128]
        scales[:, g] = torch.clamp(one.abs().max(1).values / 448, min=2.0 ** -126)
        codes[:, k:k + 128] = one / scales[:, g:g + 1]
    return {"codes": codes, "scales": scales}


def _exact_product(x, w, w_scales):
    """sum over the blocks of K of (codes x codes) sx sw; bf16 rows are quantised as the operator's definition has it."""
    T, N = (x if isinstance(x, torch.Tensor) else x[0]).shape[0], w.shape[0]
    out = torch.zeros((T, N), dtype=torch.float64, device=w.device)
    block = torch.arange(N, device=w.device) // 128
    for g, k in enumerate(range(0, w.shape[1], 128)):
        if isinstance(x, torch.Tensor):
            one = x[:, k:k + 128].double()
            amax = torch.clamp(one.abs().max(1, keepdim=True).values, min=_TINY)
            most = torch.full_like(amax, 448)
            up = (most / amax).float().double()  # (the factor is the quotient in 32 bits by definition)
            a = (one * up).float().to(torch.float8_e4m3fn).double()
            sx = (amax / most).float().double()
        else:
            a = x[0][:, k:k + 128].contiguous().view(torch.float8_e4m3fn).double()
            sx = x[1][:, g:g + 1].double()
        b = w[:, k:k + 128].contiguous().view(torch.float8_e4m3fn).double()
        out += torch.matmul(a * sx, (b * w_scales[block, g].double().unsqueeze(1)).t().contiguous())
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "quantise":
        return _exact_codes(s["x"].double())
    if case["kind"] == "norm":
        h = s["x"].double() + s["residual"].double()
        root = torch.sqrt(torch.sum(h ** 2, 1, keepdim=True) / case["K"] + _EPS)
        return {**_exact_codes(h / root * s["weight"].double()), "residual": h}
    if case["kind"] == "linear":
        return _exact_product(s["x"], s["w"], s["w_scales"])
    g = _exact_product(s["x"], s["gate"], s["gate_scales"])
    u = _exact_product(s["x"], s["up"], s["up_scales"])
    if case["limit"] > 0:
        g = torch.where(g > case["limit"], case["limit"], g)
        u = torch.where(u.abs() > case["limit"], torch.sign(u) * case["limit"], u)
    return _exact_codes(g * torch.sigmoid(g) * u)
