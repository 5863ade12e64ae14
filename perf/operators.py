"""Cases of the 8-bit linear layer's operators: rows put into 8 bits with scales and taken out again, the RMS norm that puts them there in
one pass, the scaled 8-bit matrix product, and the two backward passes that read an 8-bit checkpoint.

quantize  Q, s <- rows of X: s = max(max|x| / qmax, 2^-126) and q = round(x * qmax / max|x|); where the case says
          pow2, s is rounded up to a power of two and q = round(x / s).  V = q * s, read back
norm      h = x + r, rstd = 1 / sqrt(mean(h^2) + eps), y = h * rstd * w; Q, s <- rows of y; H = h in x's type
gemm      C[m, n] = (sum_k A[m, k] B[n, k]) * sa[m] * sb[n] + bias[n]
wgrad     dW[n, k] = sum_m dY[m, n] * s[m] * Q[m, k]
bwd       xh = s * Q * rstd, g = dy * w: dx = rstd * (g - xh * mean(g * xh)) + dr, dw = sum_m dy * xh

The 8-bit rows of a quantize or norm case are read back within the pass, as q * s in the type of the operator's input (bf16 where that is
32 bits wide: what an 8-bit row holds needs no more).
"""
import importlib.util
import math
import os
import sys

import torch

own = False

_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32, "i8": torch.int8,
          "e4m3": torch.float8_e4m3fn}
_QMAX = {"i8": 127.0, "e4m3": 448.0}
_SIZE = {"f16": 2, "bf16": 2, "f32": 4, "i8": 1, "e4m3": 1}
_EPS = 1e-6
_lib = None


def _b2g():
    """The package's binding (its folder's name is no Python name, so it is loaded by path)."""
    global _lib
    if _lib is None:
        if "b2g" not in sys.modules:
            path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rdna4-gemm-wmma_b200", "b2g.py")
            spec = importlib.util.spec_from_file_location("b2g", path)
            mod = importlib.util.module_from_spec(spec)
            sys.modules["b2g"] = mod
            spec.loader.exec_module(mod)
        _lib = sys.modules["b2g"]
    return _lib


def listed():
    return [
        # one token of a decoding step through a square projection: the weights' bytes and the launch
        {"name": "gemm 1x8192x8192 i8", "op": "gemm", "M": 1, "N": 8192, "K": 8192, "q": "i8", "c": "bf16", "bias": False, "pad": 0},
        # a small decoding batch with an odd number of tokens
        {"name": "gemm 43x10240x8192 i8", "op": "gemm", "M": 43, "N": 10240, "K": 8192, "q": "i8", "c": "f16", "bias": True, "pad": 0},
        # a long prompt through the widest layer that the library's own benchmark has
        {"name": "gemm 8192x28672x8192 i8", "op": "gemm", "M": 8192, "N": 28672, "K": 8192, "q": "i8", "c": "bf16", "bias": False, "pad": 0},
        # fp8, every extent ragged, an output pitch that no 16-byte store can take
        {"name": "gemm 1000x4099x2064 e4m3", "op": "gemm", "M": 1000, "N": 4099, "K": 2064, "q": "e4m3", "c": "f32", "bias": True, "pad": 0},
        # the input of a projection that follows no norm, one token
        {"name": "quantize 1x8192 f16 i8", "op": "quantize", "M": 1, "N": 8192, "x": "f16", "q": "i8", "pow2": False, "pad": 0},
        # a training step's activations put aside for the backward pass
        {"name": "quantize 16384x8192 bf16 i8", "op": "quantize", "M": 16384, "N": 8192, "x": "bf16", "q": "i8", "pow2": True, "pad": 0},
        # a prompt's residual stream into an int8 projection
        {"name": "norm 8192x8192 bf16 i8", "op": "norm", "M": 8192, "N": 8192, "x": "bf16", "q": "i8", "res": True, "pow2": False, "pad": 0},
        # a decoding batch, odd row length (no 16-byte loads), fp8 output
        {"name": "norm 37x5001 f16 e4m3", "op": "norm", "M": 37, "N": 5001, "x": "f16", "q": "e4m3", "res": True, "pow2": False, "pad": 3},
        # the weight gradient of a square projection over one training batch
        {"name": "wgrad 4096x8192x8192 bf16", "op": "wgrad", "M": 4096, "N": 8192, "K": 8192, "x": "bf16", "q": "i8", "c": "f32", "pad": 0},
        # a small layer, an odd number of tokens, the gradient kept in 16 bits
        {"name": "wgrad 1001x1032x2000 f16", "op": "wgrad", "M": 1001, "N": 1032, "K": 2000, "x": "f16", "q": "e4m3", "c": "f16", "pad": 8},
        # the norm's backward pass over a training batch, from the checkpoint
        {"name": "bwd 8192x8192 bf16 i8", "op": "bwd", "M": 8192, "N": 8192, "x": "bf16", "q": "i8", "res": True, "pad": 0},
        # a short batch of a narrow model
        {"name": "bwd 333x1000 f32 e4m3", "op": "bwd", "M": 333, "N": 1000, "x": "f32", "q": "e4m3", "res": False, "pad": 0},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _round(rng, v, to):
    """Most extents of real models are round; one in four stays as drawn."""
    return v if rng.random() < 0.25 else max(to, v // to * to)


def draw(rng):
    op = rng.choice(["gemm", "gemm", "quantize", "norm", "wgrad", "bwd"])
    q = rng.choice(["i8", "i8", "e4m3"])
    pad = rng.choice([0, 0, 16, 5])
    if op == "gemm":
        return {"op": op, "M": _log(rng, 1, 8192), "N": _round(rng, _log(rng, 256, 28672), 128), "K": _round(rng, _log(rng, 256, 8192), 128),
                "q": q, "c": rng.choice(["bf16", "f16", "f32"]), "bias": rng.random() < 0.5, "pad": pad}
    if op == "wgrad":
        return {"op": op, "M": _log(rng, 64, 4096), "N": _round(rng, _log(rng, 256, 8192), 128), "K": _round(rng, _log(rng, 256, 8192), 128),
                "x": rng.choice(["bf16", "bf16", "f16"]), "q": q, "c": rng.choice(["f32", "f32", "16"]), "pad": pad}
    case = {"op": op, "M": _log(rng, 1, 16384), "N": _round(rng, _log(rng, 128, 16384), 64), "x": rng.choice(["bf16", "bf16", "f16", "f32"]), "q": q, "pad": pad}
    if op != "quantize":
        case["res"] = rng.random() < 0.7
    if op != "bwd":
        case["pow2"] = rng.random() < 0.3
    return case


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(g, M, N, dtype, pad):
    """Activations: normal rows whose channels differ in size, a few of them by much, as a residual stream's do.  Row pitch N + pad."""
    buf = torch.zeros((M, N + pad), dtype=dtype, device="cuda")
    size = torch.exp(0.5 * torch.randn(N, generator=g, device="cuda"))
    size[torch.randint(0, N, (max(1, N // 512),), generator=g, device="cuda")] *= 8
    v = buf[:, :N]
    v.copy_(torch.randn((M, N), generator=g, device="cuda").mul_(size))
    return v


def _empty(M, N, dtype, pad):
    return torch.empty((M, N + pad), dtype=dtype, device="cuda")[:, :N]


def _eight_bits(g, M, K, q, pad, pow2):
    """An 8-bit matrix and its row scales, as a program has them from an earlier step."""
    x = torch.randn((M, K), generator=g, device="cuda").mul_(torch.exp(0.5 * torch.randn(M, 1, generator=g, device="cuda")))
    s = x.abs().amax(1, keepdim=True).clamp_(min=1e-20) / _QMAX[q]
    if pow2:
        s = torch.exp2(torch.ceil(torch.log2(s)))
    x /= s
    buf = torch.zeros((M, K + pad), dtype=torch.int8 if q == "i8" else torch.float8_e4m3fn, device="cuda")
    v = buf[:, :K]
    v.copy_(x.round_() if q == "i8" else x)
    return v, s.reshape(-1).contiguous()


def _values_type(x):
    return torch.bfloat16 if x == "f32" else _TYPES[x]


def prepare(case, seed):
    g, op, M, N, pad = _gen(seed), case["op"], case["M"], case["N"], case["pad"]
    s = {"case": case}
    if op == "gemm":
        K = case["K"]
        s["A"], s["sa"] = _eight_bits(g, M, K, case["q"], pad, False)
        s["B"], s["sb"] = _eight_bits(g, N, K, case["q"], pad, False)
        s["bias"] = torch.randn(N, generator=g, device="cuda") if case["bias"] else None
        s["C"] = _empty(M, N, _TYPES[case["c"]], pad)
        return s
    x = _TYPES[case["x"]]
    if op == "wgrad":
        s["Q"], s["s"] = _eight_bits(g, M, case["K"], case["q"], pad, True)
        s["dY"] = _rows(g, M, N, x, pad).mul_(2.0 ** -7)
        s["dW"] = _empty(N, case["K"], torch.float32 if case["c"] == "f32" else x, pad)
        return s
    if op in ("quantize", "norm"):
        s["X"] = _rows(g, M, N, x, pad)
        s["Q"] = _empty(M, N, _TYPES[case["q"]], pad)
        s["s"] = torch.empty(M, device="cuda")
        s["V"] = _empty(M, N, _values_type(case["x"]), pad)
        if op == "norm":
            s["w"] = (1 + 0.1 * torch.randn(N, generator=g, device="cuda")).to(x)
            s["R"] = _rows(g, M, N, x, pad) if case["res"] else None
            s["H"] = _empty(M, N, x, pad) if case["res"] else None
            s["rstd"] = torch.empty(M, device="cuda")
        return s
    s["Q"], s["s"] = _eight_bits(g, M, N, case["q"], pad, False)
    s["rstd"] = 1 / torch.sqrt((s["Q"].float() * s["s"][:, None]).square().mean(1) + _EPS)
    s["dY"] = _rows(g, M, N, x, pad).mul_(2.0 ** -7)
    s["dR"] = _rows(g, M, N, x, pad).mul_(2.0 ** -7) if case["res"] else None
    s["w"] = (1 + 0.1 * torch.randn(N, generator=g, device="cuda")).to(x)
    s["dX"] = _empty(M, N, x, pad)
    s["dw"] = torch.empty(N, device="cuda")
    return s


# ---------------------------------------------------------------- one pass
def _plain_rows_to_8(y, q, pow2):
    """(the rounded values as floats, s) of fp32 rows.  The quotient is taken in 64 bits: those of 16-bit inputs often lie on a border
    between two 8-bit values, and a quotient by the rounded scale would fall to either side."""
    amax = y.abs().amax(1)
    s = (amax / torch.full_like(amax, _QMAX[q])).clamp(min=2.0 ** -126)
    if pow2:
        m, e = torch.frexp(s)
        s = torch.ldexp(torch.ones_like(s), e - (m == 0.5).to(e.dtype))
        v = y.double() / s.double()[:, None]
    else:
        v = y.double() * _QMAX[q] / amax.double().clamp(min=_QMAX[q] * 2.0 ** -126)[:, None]
    return (v.round().float() if q == "i8" else v.to(torch.float8_e4m3fn).float()), s


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "gemm":
        C = (s["A"].float() @ s["B"].float().t()) * s["sa"][:, None] * s["sb"]
        if s["bias"] is not None:
            C = C + s["bias"]
        return {"C": C.to(_TYPES[case["c"]])}
    x = _TYPES[case["x"]]
    if op == "wgrad":
        dW = s["dY"].float().t() @ (s["Q"].float() * s["s"][:, None])
        return {"dW": dW.to(s["dW"].dtype)}
    if op == "quantize":
        q, sc = _plain_rows_to_8(s["X"].float(), case["q"], case["pow2"])
        return {"Q": (q * sc[:, None]).to(s["V"].dtype), "s": sc}
    if op == "norm":
        h = s["X"].float()
        if s["R"] is not None:
            h = h + s["R"].float()
        rstd = 1 / torch.sqrt(h.square().mean(1) + _EPS)
        q, sc = _plain_rows_to_8(h * rstd[:, None] * s["w"].float(), case["q"], case["pow2"])
        return {"Q": (q * sc[:, None]).to(s["V"].dtype), "s": sc, "rstd": rstd, "H": h.to(x) if s["R"] is not None else None}
    dy, rstd = s["dY"].float(), s["rstd"][:, None]
    xh = s["Q"].float() * s["s"][:, None] * rstd
    g = dy * s["w"].float()
    dx = rstd * (g - xh * (g * xh).mean(1, keepdim=True))
    if s["dR"] is not None:
        dx = dx + s["dR"].float()
    return {"dX": dx.to(x), "dw": (dy * xh).sum(0)}


def _code(b, name):
    return {"f16": b.DTYPE_F16, "bf16": b.DTYPE_BF16, "f32": b.DTYPE_F32, "i8": b.DTYPE_I8, "e4m3": b.DTYPE_E4M3}[name]


def run(state):
    if not own:
        return _plain(state)
    b, s = _b2g(), state
    case = s["case"]
    op, M, N = case["op"], case["M"], case["N"]
    q = _code(b, case["q"])
    if op == "gemm":
        b.gemm_q8(s["A"], s["B"], s["C"], M, N, case["K"], dtype=q, a_scale=s["sa"], b_scale=s["sb"], bias=s["bias"], c_dtype=_code(b, case["c"]))
        return {"C": s["C"]}
    x = _code(b, case["x"])
    if op == "wgrad":
        b.wgrad_q8(s["dY"], s["Q"], s["s"], s["dW"], M, N, case["K"], dtype=x, q_dtype=q, c_dtype=b.DTYPE_F32 if case["c"] == "f32" else x)
        return {"dW": s["dW"]}
    if op == "quantize":
        b.quantize_q8(s["X"], s["Q"], s["s"], M, N, dtype=x, q_dtype=q, pow2=case["pow2"])
        b.dequantize_q8(s["Q"], s["s"], s["V"], M, N, dtype=b.DTYPE_BF16 if case["x"] == "f32" else x, q_dtype=q)
        return {"Q": s["V"], "s": s["s"]}
    if op == "norm":
        b.rmsnorm_q8(s["X"], s["w"], s["Q"], s["s"], M, N, dtype=x, q_dtype=q, R=s["R"], H=s["H"], rstd=s["rstd"], eps=_EPS, pow2=case["pow2"])
        b.dequantize_q8(s["Q"], s["s"], s["V"], M, N, dtype=b.DTYPE_BF16 if case["x"] == "f32" else x, q_dtype=q)
        return {"Q": s["V"], "s": s["s"], "rstd": s["rstd"], "H": s["H"]}
    b.rmsnorm_bwd_q8(s["dY"], s["Q"], s["s"], s["w"], s["rstd"], s["dX"], s["dw"], M, N, dtype=x, x_dtype=q, dres=s["dR"])
    return {"dX": s["dX"], "dw": s["dw"]}


def work(case):
    op, M, N = case["op"], case["M"], case["N"]
    if op == "gemm":
        K = case["K"]
        return {"bytes": M * K + N * K + 4 * (M + N) + (4 * N if case["bias"] else 0) + M * N * _SIZE[case["c"]], "flops": 2 * M * N * K}
    x = _SIZE[case["x"]]
    if op == "wgrad":
        K = case["K"]
        return {"bytes": M * N * x + M * K + 4 * M + N * K * (4 if case["c"] == "f32" else x), "flops": 2 * M * N * K}
    if op == "quantize":  # X in; Q, its scales and the values read back out
        return {"bytes": M * N * (x + 1 + 2) + 4 * M, "flops": 5 * M * N}
    if op == "norm":  # X, R and w in; H, Q, scales, rstd and the values read back out
        return {"bytes": M * N * ((3 if case["res"] else 1) * x + 1 + 2) + N * x + 8 * M, "flops": 9 * M * N}
    return {"bytes": M * N * ((3 if case["res"] else 2) * x + 1) + N * x + 8 * M + 4 * N, "flops": 12 * M * N}


# ---------------------------------------------------------------- the definition in 64 bits
def _binade(v, up):
    """The power of two at (or, with `up`, at or next above) each positive normal number, from the bits."""
    bits = v.view(torch.int64)
    low = bits & ~((1 << 52) - 1)
    return torch.where((bits != low) & up, low + (1 << 52), low).view(torch.float64)


def _grid_e4m3(v):
    """The nearest number of 4 exponent and 3 fraction bits (largest 448, least step 2^-9), ties to the even one."""
    a = v.abs()
    step = _binade(a.clamp(min=2.0 ** -6), False) / 8
    return torch.sign(v) * torch.minimum(torch.round(a / step) * step, torch.full_like(a, 448.0))


def _values_64(y, q, pow2):
    top = y.abs().max(dim=1).values.clamp(min=_QMAX[q] * 2.0 ** -126)
    s = top / torch.full_like(top, _QMAX[q])  # a quotient of two tensors is rounded once, and 127 / 127 is 1
    if pow2:
        s = _binade(s, True)
        v = y / s.unsqueeze(1)
    else:
        v = y * _QMAX[q] / top.unsqueeze(1)
    return (torch.round(v) if q == "i8" else _grid_e4m3(v)) * s.unsqueeze(1), s


def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.to(torch.float64) for k, v in s.items() if isinstance(v, torch.Tensor) and k not in ("C", "dW", "dX", "dw", "V", "H")}
    op = case["op"]
    if op == "gemm":
        out = torch.einsum("mk,nk->mn", d["A"] * d["sa"].unsqueeze(1), d["B"] * d["sb"].unsqueeze(1))
        return {"C": out + d["bias"] if case["bias"] else out}
    if op == "wgrad":
        return {"dW": torch.einsum("mn,mk->nk", d["dY"] * d["s"].unsqueeze(1), d["Q"])}
    if op == "quantize":
        v, sc = _values_64(d["X"], case["q"], case["pow2"])
        return {"Q": v, "s": sc}
    if op == "norm":
        h = d["X"] + d["R"] if case["res"] else d["X"]
        rstd = torch.rsqrt((h * h).sum(1) / case["N"] + _EPS)
        v, sc = _values_64(torch.einsum("mn,m,n->mn", h, rstd, d["w"]), case["q"], case["pow2"])
        return {"Q": v, "s": sc, "rstd": rstd, "H": h if case["res"] else None}
    xh = torch.einsum("mn,m->mn", d["Q"], d["s"] * d["rstd"])
    g = d["dY"] * d["w"]
    c = (g * xh).sum(1) / case["N"]
    dx = (g - xh * c.unsqueeze(1)) * d["rstd"].unsqueeze(1)
    return {"dX": dx + d["dR"] if case["res"] else dx, "dw": torch.einsum("mn,mn->n", d["dY"], xh)}
