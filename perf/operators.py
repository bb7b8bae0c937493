"""What the group normalisation and 8-bit operators are measured on.

`listed()` gives the cases, `draw()` more of the same ranges, `prepare()` a
case's inputs on the GPU, `run()` one pass: in plain torch operations where
`own` is false, through the framework's operators where it is true.
`exact()` gives the same outputs from the definitions in 64 bits.

Operators ("op" of a case):
  norm      group normalisation with an activation over channels-last maps
  norm8     the same, written as e4m3 codes with a scale per pixel and 128 channels
  quant     rows (block_rows 1) or weights (block_rows 128) to e4m3 codes and scales
  product   8-bit product of prepared operands, with bias, activation, residual
  linear    quant of 16-bit rows and the product, as a layer runs them
"""

import math
import os
import sys

import torch

own = False

BLOCK = 128  # values that share a scale along the reduction
TOP = 448.0  # largest e4m3 value
TINY = 2.0 ** -100  # blocks below it are stored as zeros with scale 1

NONE, RELU, GELU, SIGMOID, SILU = range(5)
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------- cases
def _norm(op, n, h, w, c, groups, dtype, act, affine=True, pad=0, eps=1e-5):
    # pad: extra channels between pixels (the map is a slice of a wider one)
    return {"op": op, "n": n, "h": h, "w": w, "c": c, "groups": groups, "dtype": dtype, "act": act,
            "affine": affine, "pad": pad, "eps": eps}


def _quant(rows, k, dtype, block_rows=1, pad=0):
    return {"op": "quant", "rows": rows, "k": k, "dtype": dtype, "block_rows": block_rows, "pad": pad}


def _product(op, m, n, k, dtype, act=NONE, bias=True, residual=False):
    return {"op": op, "m": m, "n": n, "k": k, "dtype": dtype, "act": act, "bias": bias, "residual": residual}


def listed():
    named = {
        # the bottleneck of a network on one small tile: latency
        "norm 16x16x512": _norm("norm", 1, 16, 16, 512, 32, "f16", SILU),
        # a batch of 64 x 64 maps of 512 channels, the inpainting network's width
        "norm 4 of 64x64x512": _norm("norm", 4, 64, 64, 512, 32, "f16", SILU),
        # odd sides, groups of 10 channels, f32, a slice of a wider map
        "norm 3 of 37x53x320 f32": _norm("norm", 3, 37, 53, 320, 32, "f32", NONE, affine=False, pad=64),
        # whole images at full resolution: larger than L2
        "norm 2 of 768x512x128 bf16": _norm("norm", 2, 768, 512, 128, 32, "bf16", SILU),
        # the deepest map of a 1024-pixel image on its way into a product
        "norm8 32x32x768": _norm("norm8", 1, 32, 32, 768, 32, "f16", SILU),
        # a batch of maps on their way into a product
        "norm8 8 of 128x128x256": _norm("norm8", 8, 128, 128, 256, 32, "f16", SILU),
        # one pooled vector of the squeeze block's 2880 channels
        "quant 1x2880": _quant(1, 2880, "bf16"),
        # the hidden rows of a transformer level on a large image
        "quant 49152x1536": _quant(49152, 1536, "f16"),
        # one row against a whole weight matrix: weight bandwidth
        "product 1x4096x4096": _product("product", 1, 4096, 4096, "bf16"),
        # nothing a multiple of a tile
        "product 1111x777x1000": _product("product", 1111, 777, 1000, "f16", act=SILU),
        # the first layer of a transformer level's MLP, from 16-bit rows
        "linear 4096x1536x384": _product("linear", 4096, 1536, 384, "f16", act=GELU, residual=True),
        # a wide layer over a large image: tensor rate
        "product 16384x8192x2048": _product("product", 16384, 8192, 2048, "bf16"),
    }
    return [{"name": name, **case} for name, case in named.items()]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "norm8", "quant", "product", "product", "linear"])
    if op in ("norm", "norm8"):
        dtype = rng.choice(["f16", "bf16", "f32"])
        groups = rng.choice([1, 8, 16, 32, 32, 32])
        c = groups * rng.randint(max(1, 32 // groups), max(1, 1024 // groups))
        most = 100_000_000 if dtype != "f32" else 50_000_000
        pixels = _log(rng, 64, most // c)
        n = rng.choice([1, 1, 2, 3, 4, 8])
        h = max(1, int(math.sqrt(pixels / n) * rng.uniform(0.7, 1.4)))
        w = max(1, int(pixels / n / h))
        return _norm(op, n, h, w, c, groups, dtype, rng.choice([NONE, RELU, GELU, SIGMOID, SILU, SILU]),
                     affine=rng.random() < 0.8, pad=rng.choice([0, 0, 8, 40]), eps=rng.choice([1e-5, 1e-6]))
    if op == "quant":
        k = _log(rng, 16, 8192)
        rows = _log(rng, 1, 75_000_000 // k)
        return _quant(rows, k, rng.choice(["f16", "bf16", "f32"]) if rows * k < 35_000_000 else rng.choice(["f16", "bf16"]),
                      block_rows=rng.choice([1, 1, 128]), pad=rng.choice([0, 0, 24]))
    m = rng.choice([_log(rng, 1, 128), _log(rng, 64, 16384)])
    n, k = _log(rng, 32, 8192), _log(rng, 32, 4096)
    if rng.random() < 0.5:
        n, k = _up(n, 64), _up(k, 64)
    m = max(1, min(m, 16384 * 8192 * 2048 // (n * k)))
    return _product(op, m, n, k, rng.choice(["f16", "bf16", "f32"]) if op == "product" else rng.choice(["f16", "bf16"]),
                    act=rng.choice([NONE, NONE, RELU, GELU, SILU]), bias=rng.random() < 0.7, residual=rng.random() < 0.4)


# ------------------------------------------------------------------ inputs
def _up(a, b):
    return -(-a // b) * b


def _codes_like(rows, k):
    """Codes with rows 16 bytes apart or a multiple of it, as the product reads them."""
    return torch.empty((rows, _up(max(k, 1), 16)), dtype=torch.float8_e4m3fn, device="cuda")[:, :k]


def _rows(gen, rows, k, dtype):
    """Activations: channels of different spread, some rows much larger than others."""
    spread = torch.exp(0.5 * torch.randn(k, generator=gen, device="cuda"))
    size = torch.exp(torch.randn(rows, 1, generator=gen, device="cuda"))
    return (torch.randn(rows, k, generator=gen, device="cuda") * spread * size).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = {"case": case}
    op, dtype = case["op"], TYPES[case["dtype"]]
    if op in ("norm", "norm8"):
        n, h, w, c = case["n"], case["h"], case["w"], case["c"]
        x = torch.randn(n, h, w, c + case["pad"], generator=gen, device="cuda")
        offset = torch.randn(c + case["pad"], generator=gen, device="cuda")
        s["x"] = torch.addcmul(offset, x, torch.exp(0.3 * offset)).to(dtype)[..., :c]
        s["gamma"] = 1 + 0.2 * torch.randn(c, generator=gen, device="cuda") if case["affine"] else None
        s["beta"] = 0.2 * torch.randn(c, generator=gen, device="cuda") if case["affine"] else None
        if op == "norm":
            s["out"] = torch.empty((n, h, w, c), dtype=dtype, device="cuda")
        else:
            s["codes"] = _codes_like(n * h * w, c)
            s["scales"] = torch.empty((_up(c, BLOCK) // BLOCK, n * h * w), device="cuda")
    elif op == "quant":
        rows, k, br = case["rows"], case["k"], case["block_rows"]
        s["x"] = _rows(gen, rows, k + case["pad"], dtype)[:, :k]
        s["codes"] = _codes_like(rows, k)
        s["scales"] = torch.empty((_up(k, BLOCK) // BLOCK, rows if br == 1 else _up(rows, br) // br), device="cuda")
    else:
        m, n, k = case["m"], case["n"], case["k"]
        rows = _rows(gen, m, k, torch.float16 if op == "product" else dtype)
        weights = torch.randn(n, k, generator=gen, device="cuda") / math.sqrt(k)
        codes, s["w_scales"] = _plain_quant(weights, 128)
        s["w"] = _codes_like(n, k)
        s["w"].copy_(codes)
        s["a"] = _codes_like(m, k)
        if op == "product":
            codes, s["a_scales"] = _plain_quant(rows, 1)
            s["a"].copy_(codes)
        else:
            s["x"] = rows
            s["a_scales"] = torch.empty((_up(k, BLOCK) // BLOCK, m), device="cuda")
        s["bias"] = 0.2 * torch.randn(n, generator=gen, device="cuda") if case["bias"] else None
        s["residual"] = torch.randn(m, n, generator=gen, device="cuda").to(dtype) if case["residual"] else None
        s["out"] = torch.empty((m, n), dtype=dtype, device="cuda")
    return s


# -------------------------------------------------------------- plain forms
def _plain_act(v, act):
    if act == RELU:
        return torch.clamp_min(v, 0)
    if act == GELU:
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    if act == SIGMOID:
        return 1 / (1 + torch.exp(-v))
    if act == SILU:
        return v / (1 + torch.exp(-v))
    return v


def _plain_norm(s):
    case = s["case"]
    x = s["x"].float()
    n, c, g = case["n"], case["c"], case["groups"]
    v = x.reshape(n, -1, g, c // g)
    mean = v.mean(dim=(1, 3), keepdim=True)
    v = v - mean
    var = (v * v).mean(dim=(1, 3), keepdim=True)
    v = (v / torch.sqrt(var + case["eps"])).reshape(x.shape)
    if case["affine"]:
        v = v * s["gamma"] + s["beta"]
    return _plain_act(v, case["act"])


def _plain_quant(x, block_rows):
    rows, k = x.shape
    kb, rb = _up(k, BLOCK) // BLOCK, _up(rows, block_rows) // block_rows
    v = torch.zeros((rb * block_rows, kb * BLOCK), device=x.device)
    v[:rows, :k] = x
    v = v.reshape(rb, block_rows, kb, BLOCK)
    amax = v.abs().amax(dim=(1, 3), keepdim=True)
    small = amax < TINY
    codes = (v * torch.where(small, 1.0, TOP / amax)).to(torch.float8_e4m3fn)
    scales = torch.where(small, 1.0, amax / TOP).reshape(rb, kb).t().contiguous()
    return codes.reshape(rb * block_rows, kb * BLOCK)[:rows, :k], scales


def _plain_product(s, a, a_scales):
    case = s["case"]
    m, n, k = case["m"], case["n"], case["k"]
    x = a.float() * a_scales.t().repeat_interleave(BLOCK, 1)[:, :k]
    w = s["w"].float() * s["w_scales"].t().repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    v = x @ w.t()
    if case["bias"]:
        v = v + s["bias"]
    v = _plain_act(v, case["act"])
    if case["residual"]:
        v = v + s["residual"].float()
    return v.to(TYPES[case["dtype"]])


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "norm":
        return _plain_norm(s).to(TYPES[case["dtype"]])
    if op == "norm8":
        return _plain_quant(_plain_norm(s).reshape(-1, case["c"]), 1)
    if op == "quant":
        return _plain_quant(s["x"].float(), case["block_rows"])
    if op == "product":
        return _plain_product(s, s["a"], s["a_scales"])
    return _plain_product(s, *_plain_quant(s["x"].float(), 1))


# -------------------------------------------------- the framework's operators
_handle = None


def _ops():
    global _handle
    if _handle is None:
        path = os.path.join(os.getcwd(), "image-engine-native_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        from iec.ops import Ops

        _handle = Ops()
    return _handle


def _own(s):
    ops, case = _ops(), s["case"]
    op = case["op"]
    if op == "norm":
        return ops.group_norm(s["x"], case["groups"], s["gamma"], s["beta"], case["eps"], case["act"], out=s["out"])
    if op == "norm8":
        return ops.group_norm_fp8(s["x"], case["groups"], s["gamma"], s["beta"], case["eps"], case["act"],
                                  codes=s["codes"], scales=s["scales"])
    if op == "quant":
        return ops.quantize_fp8(s["x"], case["block_rows"], codes=s["codes"], scales=s["scales"])
    if op == "linear":
        ops.quantize_fp8(s["x"], codes=s["a"], scales=s["a_scales"])
    return ops.matmul_fp8(s["a"], s["a_scales"], s["w"], s["w_scales"], s["bias"], case["act"], s["residual"],
                          out=s["out"])


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ the work
def work(case):
    op = case["op"]
    size = TYPES[case["dtype"]].itemsize
    if op in ("norm", "norm8"):
        rows, c = case["n"] * case["h"] * case["w"], case["c"]
        affine = 8 * c if case["affine"] else 0
        wrote = rows * c * size if op == "norm" else rows * (c + 4 * (_up(c, BLOCK) // BLOCK))
        return {"bytes": rows * c * size + wrote + affine, "flops": 10 * rows * c}
    if op == "quant":
        rows, k, br = case["rows"], case["k"], case["block_rows"]
        return {"bytes": rows * k * (size + 1) + 4 * (_up(k, BLOCK) // BLOCK) * (_up(rows, br) // br), "flops": 2 * rows * k}
    m, n, k = case["m"], case["n"], case["k"]
    kb = _up(k, BLOCK) // BLOCK
    a = m * (k + 4 * kb) if op == "product" else m * k * size
    extra = (4 * n if case["bias"] else 0) + (m * n * size if case["residual"] else 0)
    return {"bytes": a + n * k + 4 * kb * (_up(n, BLOCK) // BLOCK) + m * n * size + extra, "flops": 2 * m * n * k}


# ------------------------------------------------- the definitions in 64 bits
def _e4m3(v):
    """The nearest e4m3 value (ties to even) of doubles of magnitude up to 448."""
    _, exponent = torch.frexp(v.abs())
    step = torch.ldexp(torch.ones_like(v), torch.clamp_min(exponent - 1, -6) - 3)
    return torch.round(v / step) * step


def _exact_act(v, act):
    if act == RELU:
        return torch.relu(v)
    if act == GELU:
        return v * torch.special.ndtr(v)
    if act == SIGMOID:
        return torch.sigmoid(v)
    if act == SILU:
        return v * torch.sigmoid(v)
    return v


def _exact_blocks(x, block_rows):
    """The codes (as doubles) and scales of `x`, block by block of the columns."""
    rows, k = x.shape
    codes, scales = torch.empty_like(x), []
    starts = range(0, k, BLOCK)
    fill = _up(rows, block_rows) - rows
    for at in starts:
        part = x[:, at:at + BLOCK]
        top = part.abs().max(dim=1).values
        if block_rows > 1:
            top = torch.cat([top, top.new_zeros(fill)]).view(-1, block_rows).max(dim=1).values
        zero = top < TINY
        scales.append(torch.where(zero, torch.ones_like(top), top / TOP))
        rate = torch.where(zero, torch.ones_like(top), TOP / top)
        codes[:, at:at + BLOCK] = _e4m3(part * rate.repeat_interleave(block_rows)[:rows, None])
    return codes, torch.stack(scales)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("norm", "norm8"):
        x = s["x"].double()
        n, c, g = case["n"], case["c"], case["groups"]
        flat = x.view(n, -1, c) if x.is_contiguous() else x.contiguous().view(n, -1, c)
        out = torch.empty_like(flat)
        for i in range(n):
            for j in range(g):
                at = slice(j * (c // g), (j + 1) * (c // g))
                part = flat[i, :, at]
                out[i, :, at] = (part - part.mean()) * torch.rsqrt(part.var(unbiased=False) + case["eps"])
        if case["affine"]:
            out = out * s["gamma"].double() + s["beta"].double()
        out = _exact_act(out, case["act"])
        return out.view(x.shape) if op == "norm" else _exact_blocks(out.view(-1, c), 1)
    if op == "quant":
        return _exact_blocks(s["x"].double(), case["block_rows"])
    m, n, k = case["m"], case["n"], case["k"]
    codes, scales = (s["a"].double(), s["a_scales"].double()) if op == "product" else _exact_blocks(s["x"].double(), 1)
    total = torch.zeros((m, n), dtype=torch.float64, device="cuda")
    w = s["w"].double()
    for b in range(scales.shape[0]):
        at = slice(b * BLOCK, min(k, (b + 1) * BLOCK))
        part = (codes[:, at] @ w[:, at].t()) * scales[b][:, None]
        total += part * s["w_scales"][b].double().repeat_interleave(BLOCK)[:n]
    if case["bias"]:
        total += s["bias"].double()
    total = _exact_act(total, case["act"])
    return total + s["residual"].double() if case["residual"] else total
