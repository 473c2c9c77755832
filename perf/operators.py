"""Operators of 8-bit floating-point layers: their plain forms and the library's calls, on the same inputs.

Three operators that follow one another in a layer whose products run on 8-bit floats with a scale for every block of
128 values:

  quantize   och_quantize_blocks   a matrix to 8-bit codes and one float scale per block
  norm       och_rms_norm          residual addition, root-mean-square norm, output in the input's type or in 8 bits
             och_rms_norm_grad     its gradients
  gemm       och_gemm_scaled       the product of two such matrices

All matrices are column-major (element (i, j) at i + j * ld); a torch tensor [tokens, features] with contiguous features
is the column-major matrix features x tokens. The 8-bit codes come back as torch.float8 tensors, which stand for the
codes' values; scales are float32.

A block's scale is max|x| / max_code (max_code 448 for e4m3, 57344 for e5m2; a maximum below 2^-100 counts as 2^-100, and
a block with a NaN or an infinity has scale NaN and NaN codes), its codes are x * (max_code / max|x|) rounded to nearest.
"""
import math
import os
import sys

import torch

own = False                     # False: the plain forms below; True: the library's kernels

BLOCK = 128
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CODES = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
MAX_CODE = {"e4m3": 448.0, "e5m2": 57344.0}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
SMALLEST = 2.0 ** -100


# ---- cases ------------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one token's activations on their way into a product: a call that is all latency
        {"name": "quantize_token", "op": "quantize", "m": 4096, "n": 1, "bm": 128, "bn": 1, "type": "bf16", "code": "e4m3", "pad": 0},
        # the activations of a long batch, blocks along the features
        {"name": "quantize_batch", "op": "quantize", "m": 8192, "n": 8192, "bm": 128, "bn": 1, "type": "bf16", "code": "e4m3", "pad": 0},
        # gradients of an odd batch, blocks along the tokens, as the weights' gradient product reads them
        {"name": "quantize_tokens_axis", "op": "quantize", "m": 5003, "n": 4001, "bm": 1, "bn": 128, "type": "fp16", "code": "e5m2", "pad": 5},
        # a layer's master weights to 128 x 128 tiles
        {"name": "quantize_weights", "op": "quantize", "m": 8192, "n": 4096, "bm": 128, "bn": 128, "type": "fp32", "code": "e4m3", "pad": 0},
        # sixteen tokens being decoded: residual stream in and out, 8-bit output for the next product
        {"name": "norm_decode", "op": "norm", "n": 4096, "rows": 16, "type": "fp16", "weight": "fp16", "out": "e4m3", "residual": True, "pad": 0},
        # a long prompt
        {"name": "norm_prompt", "op": "norm", "n": 8192, "rows": 8192, "type": "bf16", "weight": "bf16", "out": "e4m3", "residual": True, "pad": 0},
        # training in float32, a width that no vector length divides
        {"name": "norm_odd", "op": "norm", "n": 5003, "rows": 2047, "type": "fp32", "weight": "fp32", "out": "same", "residual": False, "pad": 0},
        # the backward pass of a training batch
        {"name": "norm_grad", "op": "norm_grad", "n": 4096, "rows": 8192, "type": "bf16", "weight": "fp32", "residual": True, "pad": 0},
        # one token through a wide layer: the weights are read once
        {"name": "gemm_token", "op": "gemm", "m": 14336, "n": 1, "k": 4096, "ta": "T", "tb": "N", "ba": 128, "bb": 1, "ca": "e4m3", "cb": "e4m3", "out": "fp16"},
        # a decode batch
        {"name": "gemm_decode", "op": "gemm", "m": 8192, "n": 48, "k": 8192, "ta": "T", "tb": "N", "ba": 128, "bb": 1, "ca": "e4m3", "cb": "e4m3", "out": "bf16"},
        # a long prompt through a square layer
        {"name": "gemm_prompt", "op": "gemm", "m": 8192, "n": 8192, "k": 8192, "ta": "T", "tb": "N", "ba": 128, "bb": 1, "ca": "e4m3", "cb": "e4m3", "out": "bf16"},
        # the weights' gradient of an odd batch: both operands contiguous along their rows, blocks along the tokens
        {"name": "gemm_weights_grad", "op": "gemm", "m": 4096, "n": 5000, "k": 4001, "ta": "N", "tb": "T", "ba": 1, "bb": 1, "ca": "e4m3", "cb": "e5m2", "out": "fp32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A feature count: usually a multiple of 128 or 16, now and then odd."""
    x = _log(rng, lo, hi)
    step = rng.choice([128, 128, 16, 1])
    return max(step, x // step * step)


def draw(rng):
    op = rng.choice(["quantize", "norm", "norm_grad", "gemm", "gemm"])
    kind = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "quantize":
        m = _width(rng, 64, 16384)
        n = min(_log(rng, 1, 16384), 2 ** 26 // m)
        bm, bn = rng.choice([(128, 1), (128, 1), (1, 128), (128, 128)])
        return {"op": op, "m": m, "n": n, "bm": bm, "bn": bn, "type": kind, "code": rng.choice(["e4m3", "e5m2"]), "pad": rng.choice([0, 0, 8, 3])}
    if op in ("norm", "norm_grad"):
        n = _width(rng, 64, 16384)
        case = {"op": op, "n": n, "rows": min(_log(rng, 1, 32768), 2 ** (26 if op == "norm" else 25) // n), "type": kind,
                "weight": rng.choice([kind, "fp32"]), "residual": rng.random() < 0.6, "pad": rng.choice([0, 0, 8, 3])}
        if op == "norm":
            case["out"] = rng.choice(["e4m3", "e4m3", "same"])
        return case
    m, k = _width(rng, 128, 16384), _width(rng, 128, 16384)
    n = _log(rng, 1, 128) if rng.random() < 0.4 else _width(rng, 64, 8192)
    n = max(1, min(n, 2 ** 38 // (m * k)))
    use = rng.choice(["forward", "forward", "input_grad", "weights_grad"])
    case = {"op": op, "m": m, "n": n, "k": k, "out": rng.choice(["bf16", "fp16", "fp32"])}
    if use == "forward":
        case.update(ta="T", tb="N", ba=rng.choice([128, 128, 1]), bb=1, ca="e4m3", cb="e4m3")
    elif use == "input_grad":
        case.update(ta="N", tb="N", ba=128, bb=1, ca="e4m3", cb=rng.choice(["e4m3", "e5m2"]))
    else:
        case.update(ta="N", tb="T", ba=1, bb=1, ca="e4m3", cb=rng.choice(["e4m3", "e5m2"]))
    return case


# ---- inputs -----------------------------------------------------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _rows(g, rows, cols, pad, kind, scale=1.0):
    """rows x cols values as a layer sees them (features of different size, a few large ones), in rows that lie `pad`
    elements further apart than they are long."""
    feature = torch.exp(0.5 * torch.randn(cols, generator=g, device="cuda"))
    feature = torch.where(torch.rand(cols, generator=g, device="cuda") < 0.002, feature * 20, feature)
    x = torch.empty(rows, cols + pad, dtype=TYPES[kind], device="cuda")
    x[:, :cols] = torch.randn(rows, cols, generator=g, device="cuda") * feature * scale
    x[:, cols:] = 0
    return x[:, :cols]


def _coded(g, rows, cols, along_rows, block, code, scale):
    """Codes [rows, cols] and scales of a matrix quantized with blocks of `block` x 128 (along_rows: 128 along the columns'
    index, else along the rows' index)."""
    x = _rows(g, rows, cols, 0, "bf16", scale)
    bm, bn = (128, block) if along_rows else (block, 128)
    return _quantize(x.float(), bm, bn, code)


def prepare(case, seed):
    g = _generator(seed)
    c = case
    if c["op"] == "quantize":
        return {"case": c, "x": _rows(g, c["n"], c["m"], c["pad"], c["type"], 0.02 if c["bn"] == 128 else 1.0)}
    if c["op"] in ("norm", "norm_grad"):
        n, rows, pad = c["n"], c["rows"], c["pad"]
        s = {"case": c, "x": _rows(g, rows, n, pad, c["type"])}
        s["w"] = (1 + 0.1 * torch.randn(n, generator=g, device="cuda")).to(TYPES[c["weight"]])
        s["r"] = _rows(g, rows, n, pad, c["type"], 3.0) if c["residual"] else None
        if c["op"] == "norm_grad":      # x is the normalised sum of the forward pass here, r the residual stream's gradient
            s["dy"] = _rows(g, rows, n, pad, c["type"], 0.01)
            s["r"] = None if s["r"] is None else (s["r"].float() * 0.01).to(TYPES[c["type"]])
            s["rstd"] = torch.rsqrt(s["x"].float().square().mean(1) + EPS)
        return s
    # op(A) is m x k and op(B) k x n; as rows of a torch tensor: 'T' / 'N' of A is [m, k] / [k, m], 'N' / 'T' of B [n, k] / [k, n]
    a, sa = _coded(g, c["m"], c["k"], True, c["ba"], c["ca"], 0.02) if c["ta"] == "T" else _coded(g, c["k"], c["m"], False, c["ba"], c["ca"], 0.02)
    b, sb = _coded(g, c["n"], c["k"], True, c["bb"], c["cb"], 1.0) if c["tb"] == "N" else _coded(g, c["k"], c["n"], False, c["bb"], c["cb"], 1.0)
    return {"case": c, "a": a, "sa": sa, "b": b, "sb": sb}


EPS = 1e-6


# ---- plain forms ------------------------------------------------------------------------------------------------------

def _blocks(x, bm, bn):
    """x [n, m] with zeros behind its ends, as [n / bn, bn, m / bm, bm]."""
    n, m = x.shape
    p = torch.zeros(-(-n // bn) * bn, -(-m // bm) * bm, dtype=x.dtype, device=x.device)
    p[:n, :m] = x
    return p.view(p.shape[0] // bn, bn, p.shape[1] // bm, bm)


def _quantize(x, bm, bn, code):
    """Codes [n, m] and scales [n / bn, m / bm] of x [n, m] (float32)."""
    n, m = x.shape
    most = MAX_CODE[code]
    p = _blocks(x, bm, bn)
    amax = p.abs().amax(3).amax(1)
    amax = torch.where(torch.isfinite(amax), amax.clamp(min=SMALLEST), torch.full_like(amax, math.nan))
    factor = torch.full_like(amax, most) / amax
    q = (p * factor[:, None, :, None]).clamp(-most, most).to(CODES[code])
    q = q.view(p.shape[0] * bn, p.shape[2] * bm)[:n, :m].contiguous()
    return q, amax / torch.full_like(amax, most)


def _values(q, s, bm, bn):
    """The float32 values that codes q [n, m] with scales s stand for."""
    n, m = q.shape
    wide = s.repeat_interleave(bn, 0)[:n] if bn > 1 else s
    wide = wide.repeat_interleave(bm, 1)[:, :m] if bm > 1 else wide
    return q.float() * wide


def _plain_norm(s):
    c = s["case"]
    h = s["x"].float()
    if s["r"] is not None:
        h = (h + s["r"].float()).to(TYPES[c["type"]])
    out = {"h": h} if s["r"] is not None else {}
    h = h.float()
    rstd = torch.rsqrt(h.square().mean(1) + EPS)
    y = h * rstd[:, None] * s["w"].float()
    out["rstd"] = rstd
    if c["out"] == "same":
        out["y"] = y.to(TYPES[c["type"]])
    else:
        out["q"], out["s"] = _quantize(y, 128, 1, c["out"])
    return out


def _plain_norm_grad(s):
    c = s["case"]
    h, dy, rstd = s["x"].float(), s["dy"].float(), s["rstd"][:, None]
    hat = h * rstd
    g = dy * s["w"].float()
    dx = rstd * (g - hat * (g * hat).mean(1, keepdim=True))
    if s["r"] is not None:
        dx = dx + s["r"].float()
    return {"dx": dx.to(TYPES[c["type"]]), "dw": (dy * hat).sum(0)}


def _plain_gemm(s):
    c = s["case"]
    a = _values(s["a"], s["sa"], *((128, c["ba"]) if c["ta"] == "T" else (c["ba"], 128)))
    b = _values(s["b"], s["sb"], *((128, c["bb"]) if c["tb"] == "N" else (c["bb"], 128)))
    a = a if c["ta"] == "T" else a.t()
    b = b if c["tb"] == "N" else b.t()
    return (b @ a.t()).to(TYPES[c["out"]])


# ---- the library's calls ----------------------------------------------------------------------------------------------

_LIB = []


def _library():
    if not _LIB:
        path = os.path.join(os.getcwd(), "ocean-tensor-package_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        import ocean_hip
        types = {"bf16": ocean_hip.BFLOAT16, "fp16": ocean_hip.HALF, "fp32": ocean_hip.FLOAT, "e4m3": ocean_hip.FLOAT8_E4M3, "e5m2": ocean_hip.FLOAT8_E5M2}
        _LIB.append((ocean_hip.lib, ocean_hip.check, types))
    return _LIB[0]


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _ptr(t):
    return None if t is None else t.data_ptr()


def _ld(t):
    return 0 if t is None else t.stride(0)


def _own_quantize(s):
    lib, check, types = _library()
    c, x = s["case"], s["x"]
    n, m = x.shape
    q = torch.empty(n, m, dtype=CODES[c["code"]], device=x.device)
    scale = torch.empty(-(-n // c["bn"]), -(-m // c["bm"]), dtype=torch.float32, device=x.device)
    check(lib.och_quantize_blocks(types[c["type"]], types[c["code"]], m, n, x.data_ptr(), x.stride(0), c["bm"], c["bn"],
                                  q.data_ptr(), m, scale.data_ptr(), scale.shape[1], _stream()))
    return {"q": q, "s": scale}


def _own_norm(s):
    lib, check, types = _library()
    c, x, r, w = s["case"], s["x"], s["r"], s["w"]
    rows, n = x.shape
    same = c["out"] == "same"
    h = None if r is None else torch.empty(rows, n, dtype=x.dtype, device=x.device)
    y = torch.empty(rows, n, dtype=x.dtype if same else CODES[c["out"]], device=x.device)
    scale = None if same else torch.empty(rows, -(-n // BLOCK), dtype=torch.float32, device=x.device)
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
    check(lib.och_rms_norm(types[c["type"]], n, rows, x.data_ptr(), x.stride(0), _ptr(r), _ld(r), _ptr(h), _ld(h), types[c["weight"]], w.data_ptr(), EPS,
                           types[c["type"] if same else c["out"]], y.data_ptr(), n, _ptr(scale), _ld(scale), rstd.data_ptr(), _stream()))
    out = {"rstd": rstd, "y": y} if same else {"rstd": rstd, "q": y, "s": scale}
    if r is not None:
        out["h"] = h
    return out


def _own_norm_grad(s):
    lib, check, types = _library()
    c, x, r, w, dy = s["case"], s["x"], s["r"], s["w"], s["dy"]
    rows, n = x.shape
    dx = torch.empty(rows, n, dtype=x.dtype, device=x.device)
    dw = torch.empty(n, dtype=torch.float32, device=x.device)
    check(lib.och_rms_norm_grad(types[c["type"]], n, rows, dy.data_ptr(), dy.stride(0), x.data_ptr(), x.stride(0), s["rstd"].data_ptr(), types[c["weight"]],
                                w.data_ptr(), _ptr(r), _ld(r), dx.data_ptr(), n, dw.data_ptr(), _stream()))
    return {"dx": dx, "dw": dw}


def _own_gemm(s):
    lib, check, types = _library()
    c, a, b, sa, sb = s["case"], s["a"], s["b"], s["sa"], s["sb"]
    out = torch.empty(c["n"], c["m"], dtype=TYPES[c["out"]], device=a.device)
    check(lib.och_gemm_scaled(types[c["ca"]], types[c["cb"]], types[c["out"]], c["ta"].encode(), c["tb"].encode(), c["m"], c["n"], c["k"], 1.0,
                              a.data_ptr(), a.stride(0), sa.data_ptr(), sa.stride(0), c["ba"], b.data_ptr(), b.stride(0), sb.data_ptr(), sb.stride(0), c["bb"],
                              0.0, out.data_ptr(), c["m"], _stream()))
    return out


PLAIN = {"quantize": lambda s: dict(zip("qs", _quantize(s["x"].float(), s["case"]["bm"], s["case"]["bn"], s["case"]["code"]))),
         "norm": _plain_norm, "norm_grad": _plain_norm_grad, "gemm": _plain_gemm}
OWN = {"quantize": _own_quantize, "norm": _own_norm, "norm_grad": _own_norm_grad, "gemm": _own_gemm}


def run(state):
    if own:
        return OWN[state["case"]["op"]](state)
    return PLAIN[state["case"]["op"]](state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------

def work(case):
    c = case
    if c["op"] == "quantize":
        scales = -(-c["m"] // c["bm"]) * -(-c["n"] // c["bn"])
        return {"bytes": c["m"] * c["n"] * (SIZE[c["type"]] + 1) + 4 * scales, "flops": 3 * c["m"] * c["n"]}
    if c["op"] in ("norm", "norm_grad"):
        t, e = SIZE[c["type"]], c["n"] * c["rows"]
        weight = c["n"] * SIZE[c["weight"]]
        if c["op"] == "norm":
            out = e * t if c["out"] == "same" else e + 4 * c["rows"] * -(-c["n"] // BLOCK)
            return {"bytes": e * t * (3 if c["residual"] else 1) + out + weight + 4 * c["rows"], "flops": 5 * e}
        return {"bytes": e * t * (4 if c["residual"] else 3) + weight + 4 * c["n"] + 4 * c["rows"], "flops": 9 * e}
    m, n, k = c["m"], c["n"], c["k"]
    kb = -(-k // BLOCK)
    return {"bytes": m * k + n * k + 4 * kb * (-(-m // c["ba"]) + -(-n // c["bb"])) + m * n * SIZE[c["out"]], "flops": 2 * m * n * k}


# ---- the same results in 64 bits --------------------------------------------------------------------------------------

def _spread(s, axis, block, length):
    index = torch.arange(length, device=s.device) // block
    return s.double().index_select(axis, index)


def _exact_scaled(v, bm, bn, code):
    """Scales of float64 values v [n, m] and what every code approximates: the value over its scale."""
    n, m = v.shape
    nb, mb = -(-n // bn), -(-m // bm)
    size = torch.zeros(nb * bn, mb * bm, dtype=torch.float64, device=v.device)
    size[:n, :m] = v.abs()
    largest = size.reshape(nb, bn, mb, bm).permute(0, 2, 1, 3).reshape(nb, mb, bn * bm).max(2).values
    scale = torch.maximum(largest, torch.tensor(SMALLEST, dtype=torch.float64, device=v.device)) / MAX_CODE[code]
    return v / _spread(_spread(scale, 0, bn, n), 1, bm, m), scale


def _nearest(v, code):
    """float64 values on the grid of a code, ties to even: 3 (e4m3) or 2 (e5m2) bits behind the leading one, whose
    exponent is at least -6 or -14."""
    bits, lowest = (3, -6) if code == "e4m3" else (2, -14)
    step = torch.ldexp(torch.ones_like(v), (torch.frexp(v).exponent - 1).clamp(min=lowest) - bits)
    return torch.round(v / step) * step


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "quantize":
        q, scale = _exact_scaled(s["x"].double(), c["bm"], c["bn"], c["code"])
        return {"q": _nearest(q, c["code"]), "s": scale}
    if c["op"] == "norm":
        out, h = {}, s["x"].double()
        if s["r"] is not None:
            h = h + s["r"].double()
            out["h"] = h
            h = h.to(TYPES[c["type"]]).double()         # the norm is that of the stored sum
        mean = torch.sum(h * h, dim=1) / c["n"]
        out["rstd"] = 1.0 / torch.sqrt(mean + EPS)
        y = h * (out["rstd"].unsqueeze(1) * s["w"].double().unsqueeze(0))
        if c["out"] == "same":
            out["y"] = y
        else:
            out["q"], out["s"] = _exact_scaled(y, 128, 1, c["out"])     # before the codes' rounding, like the other outputs
        return out
    if c["op"] == "norm_grad":
        # y_i = w_i h_i / m with m = sqrt(mean h^2 + eps): dL/dh_j = w_j dy_j / m - h_j (sum_i w_i dy_i h_i) / (n m^3)
        h, dy, w, r = s["x"].double(), s["dy"].double(), s["w"].double(), s["rstd"].double().unsqueeze(1)
        inner = torch.sum(w * dy * h, dim=1, keepdim=True)
        dx = w * dy * r - h * (inner * r ** 3 / c["n"])
        return {"dx": dx if s["r"] is None else dx + s["r"].double(), "dw": torch.sum(dy * (h * r), dim=0)}
    m, n, k = c["m"], c["n"], c["k"]
    if c["ta"] == "T":
        a = s["a"].to(torch.float64) * _spread(_spread(s["sa"], 0, c["ba"], m), 1, 128, k)
    else:
        a = (s["a"].to(torch.float64) * _spread(_spread(s["sa"], 0, 128, k), 1, c["ba"], m)).t()
    if c["tb"] == "N":
        b = s["b"].to(torch.float64) * _spread(_spread(s["sb"], 0, c["bb"], n), 1, 128, k)
    else:
        b = (s["b"].to(torch.float64) * _spread(_spread(s["sb"], 0, 128, k), 1, c["bb"], n)).t()
    return torch.matmul(a, b.t()).t().contiguous()
