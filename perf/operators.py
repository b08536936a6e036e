"""Microscaled numbers (blocks of 32 values that share a power of two) as a user of this package calls them: the
quantisation to 4 and 8 bits, the 4-bit product for prompts and single tokens, and the training step of a layer that
computes in 4 bits and keeps its activations in 8.

``run`` computes each pass by elementary torch operations in 32 bits (``own`` false) or by the package's calls (``own``
true).  ``exact`` gives the same outputs from the definition in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

BLOCK = 32
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
# format: exponent of the largest element (4-bit e2m1: 6 = 1.5 * 2^2, 8-bit integers of 6 fraction bits: 127/64), bits
EMAX = {"fp4": 2, "int8": 0}
BITS = {"fp4": 4, "int8": 8}


# ---- cases -----------------------------------------------------------------------------------------

def _keep(name, fmt, rows, k, dtype):
    return {"name": name, "do": "keep", "fmt": fmt, "rows": rows, "k": k, "dtype": dtype}


def _linear(name, m, k, n, dtype, bias, epilogue):
    return {"name": name, "do": "linear", "m": m, "k": k, "n": n, "dtype": dtype, "bias": bias, "epilogue": epilogue}


def _train(name, m, k, n, dtype, wdtype, bias):
    return {"name": name, "do": "train", "m": m, "k": k, "n": n, "dtype": dtype, "wdtype": wdtype, "bias": bias}


def listed():
    return [
        # the activations of one token: two launches and little else
        _keep("keep fp4 1x4096 bf16", "fp4", 1, 4096, "bf16"),
        # a large weight, as a deployment script quantises it, and back
        _keep("keep fp4 11008x4096 bf16", "fp4", 11008, 4096, "bf16"),
        # an odd number of fp32 activations kept for the backward pass
        _keep("keep int8 4095x1001 f32", "int8", 4095, 1001, "f32"),
        # the activations of a batch of 128 images kept for the backward pass
        _keep("keep int8 25216x768 f16", "int8", 25216, 768, "f16"),
        # one token through a square layer: the weight is read once
        _linear("linear 1x4096->4096 bf16", 1, 4096, 4096, "bf16", False, "none"),
        # a batch of eight single tokens against a large weight
        _linear("linear 8x8192->8192 f16", 8, 8192, 8192, "f16", True, "none"),
        # one image of 197 tokens through a qkv projection
        _linear("linear 197x768->2304 bf16", 197, 768, 2304, "bf16", True, "gelu"),
        # no size a multiple of anything, fp32 in and out
        _linear("linear 1000x1001->999 f32", 1000, 1001, 999, "f32", True, "relu"),
        # a long prompt
        _linear("linear 8192x8192->8192 bf16", 8192, 8192, 8192, "bf16", True, "none"),
        # a small step: launches count
        _train("train 256x1024->1024 bf16", 256, 1024, 1024, "bf16", "bf16", True),
        # fp32 gradients of odd sizes
        _train("train 777x1001->515 f32", 777, 1001, 515, "f32", "f32", True),
        # a step of 8192 tokens, fp32 master weights under bf16 activations
        _train("train 8192x4096->11008 bf16", 8192, 4096, 11008, "bf16", "f32", True),
    ]


def _log(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    # half of the sizes as programs have them, the rest as they fall
    step = rng.choice((1, 1, 8, 64 if v >= 128 else 8))
    return max(lo, min(hi, (v + step - 1) // step * step))


def draw(rng):
    do = rng.choice(("keep", "linear", "linear", "train"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    if do == "keep":
        k = _log(rng, 1, 16384)
        return {"do": do, "fmt": rng.choice(("fp4", "int8")), "rows": _log(rng, 1, max(1, min(32768, (1 << 25) // k))), "k": k,
                "dtype": dtype}
    k, n = _log(rng, 8, 11008), _log(rng, 8, 11008)
    most = 8192 if do == "linear" else min(8192, int(3.6e11 / (k * n)))
    m = _log(rng, 1, 64) if do == "linear" and rng.random() < 0.5 else _log(rng, 1, most)
    if do == "linear":
        return {"do": do, "m": m, "k": k, "n": n, "dtype": dtype, "bias": rng.random() < 0.5,
                "epilogue": rng.choice(("none", "relu", "gelu"))}
    return {"do": do, "m": m, "k": k, "n": n, "dtype": dtype, "wdtype": rng.choice((dtype, "f32")), "bias": rng.random() < 0.7}


# ---- inputs ----------------------------------------------------------------------------------------

def _activations(rows, k, dtype, gen):
    """Unit normal values whose size differs from feature to feature, a few features far above the rest."""
    size = torch.exp(0.5 * torch.randn(k, device="cuda", generator=gen))
    size = torch.where(torch.rand(k, device="cuda", generator=gen) < 0.01, 12 * size, size)
    return (torch.randn(rows, k, device="cuda", generator=gen) * size).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    s = dict(case)
    if case["do"] == "keep":
        s["x"] = _activations(case["rows"], case["k"], dtype, gen)
        return s
    m, k, n = case["m"], case["k"], case["n"]
    s["x"] = _activations(m, k, dtype, gen)
    w = 0.02 * torch.randn(n, k, device="cuda", generator=gen)
    s["bias"] = torch.randn(n, device="cuda", generator=gen).to(dtype) if case["bias"] else None
    if case["do"] == "linear":
        # what a deployed layer keeps: packed codes and their scales
        exponents, values = _quantize(w, "fp4")
        s["codes"], s["scales"] = _pack(values, exponents), _tile(exponents)
        return s
    s["w"] = w.to(DTYPES[case["wdtype"]])
    s["x"].requires_grad_()
    s["w"].requires_grad_()
    if s["bias"] is not None:
        s["bias"].requires_grad_()
    s["dy"] = (torch.randn(m, n, device="cuda", generator=gen) / m).to(dtype)
    return s


def _pack(values, exponents):
    """4-bit codes of block values, two to a byte, the first in the low half: sign, two exponent bits, one mantissa bit."""
    a = torch.ldexp(values.view(values.shape[0], -1, BLOCK), -exponents[:, :, None]).reshape(values.shape)
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=a.device)
    code = torch.searchsorted(grid, a.abs()).to(torch.uint8) | ((a < 0).to(torch.uint8) << 3)
    return code[:, 0::2] | (code[:, 1::2] << 4)


def _tile(exponents):
    """Scale bytes in tiles of 128 rows x 4 blocks: [row tile][block tile][row % 32][row // 32 % 4][block % 4]."""
    rows, blocks = exponents.shape
    rt, bt = -(-rows // 128), -(-blocks // 4)
    b = torch.zeros(rt * 128, bt * 4, dtype=torch.uint8, device=exponents.device)
    b[:rows, :blocks] = (exponents + 127).to(torch.uint8)
    return b.view(rt, 4, 32, bt, 4).permute(0, 3, 2, 1, 4).reshape(rt, bt, 512).contiguous()


def _untile(scales, rows, blocks):
    rt, bt, _ = scales.shape
    b = scales.view(rt, bt, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(rt * 128, bt * 4)
    return b[:rows, :blocks].int() - 127


# ---- the operators in plain torch, 32 bits ---------------------------------------------------------

def _quantize(x, fmt):
    """(exponent of each block of 32, the values the codes stand for, in fp32 and padded to whole blocks)."""
    rows, k = x.shape
    v = torch.nn.functional.pad(x.detach().float(), (0, -k % BLOCK)).view(rows, -1, BLOCK)
    top = v.abs().amax(-1)
    e = ((top.view(torch.int32) >> 23) - 127 - EMAX[fmt]).clamp(min=-127)
    a = torch.ldexp(v, -e[:, :, None])
    if fmt == "fp4":
        step = torch.where(a.abs() < 2, 0.5, torch.where(a.abs() < 4, 1.0, 2.0))
        q = (torch.round(a / step) * step).clamp(-6, 6)
    else:
        q = torch.round(a * 64).clamp(-127, 127) / 64
    return e, torch.ldexp(q, e[:, :, None]).reshape(rows, -1)


def _unpack(codes, scales):
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    grid = torch.cat((grid, -grid))
    rows = codes.shape[0]
    v = torch.stack((grid[(codes & 15).int()], grid[(codes >> 4).int()]), -1).view(rows, -1, BLOCK)
    return torch.ldexp(v, _untile(scales, rows, v.shape[1])[:, :, None]).reshape(rows, -1)


def _activate(y, epilogue):
    if epilogue == "relu":
        return y.clamp(min=0)
    if epilogue == "gelu":
        return 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    return y


def _plain(s):
    x, k = s["x"], s["k"]
    if s["do"] == "keep":
        return _quantize(x, s["fmt"])[1][:, :k].to(x.dtype)
    bias = 0 if s["bias"] is None else s["bias"].detach().float()
    if s["do"] == "linear":
        y = _quantize(x, "fp4")[1] @ _unpack(s["codes"], s["scales"]).t() + bias
        return _activate(y, s["epilogue"]).to(x.dtype)
    w = _quantize(s["w"], "fp4")[1]
    y = _quantize(x, "fp4")[1] @ w.t() + bias
    dy = s["dy"].float()
    dx = (dy @ w)[:, :k]
    dw = (dy.t() @ _quantize(x, "int8")[1])[:, :k]
    db = None if s["bias"] is None else dy.sum(0).to(s["bias"].dtype)
    return _step(y.detach().to(x.dtype), dx.to(x.dtype), dw.to(s["w"].dtype), db)


def _step(y, dx, dw, db):
    out = {"y": y, "dx": dx, "dw": dw}
    if db is not None:
        out["db"] = db
    return out


def run(s):
    if not own:
        return _plain(s)
    from dimq_b200 import ops, qat

    if s["do"] == "keep":
        codes, scales = ops.mx_quantize(s["x"], s["fmt"])
        return ops.mx_dequantize(codes, scales, s["k"], s["fmt"], out_dtype=s["x"].dtype)
    if s["do"] == "linear":
        return ops.mx_linear(s["x"], s["codes"], s["scales"], s["bias"], s["n"], s["k"], out_dtype=s["x"].dtype,
                             epilogue=s["epilogue"])
    leaves = [t for t in (s["x"], s["w"], s["bias"]) if t is not None]
    y = qat.mx_linear(s["x"], s["w"], s["bias"], checkpoint="int8")
    grads = torch.autograd.grad(y, leaves, s["dy"])
    return _step(y.detach(), grads[0], grads[1], grads[2] if len(grads) == 3 else None)


# ---- what a pass cannot do without -----------------------------------------------------------------

def work(case):
    es = SIZE[case["dtype"]]
    if case["do"] == "keep":     # the values in, codes and scales out and in again (the caller keeps them), the values out
        n = case["rows"] * case["k"]
        return {"bytes": 2 * n * es + 2 * n * (BITS[case["fmt"]] / 8 + 1 / BLOCK), "flops": 4 * n}
    m, k, n = case["m"], case["k"], case["n"]
    if case["do"] == "linear":
        return {"bytes": m * k * es + n * k * (0.5 + 1 / BLOCK) + m * n * es + (n * es if case["bias"] else 0), "flops": 2 * m * n * k}
    ws = SIZE[case["wdtype"]]    # x, w, dy in; y, dx, dw, db out
    return {"bytes": 2 * m * k * es + 2 * n * k * ws + 2 * m * n * es + (2 * n * es if case["bias"] else 0), "flops": 6 * m * n * k}


# ---- the definition in 64 bits ---------------------------------------------------------------------

def _blocks64(x, fmt):
    """Nearest representable value of each element, from the format's definition: the block's exponent by frexp, the 4-bit
    code by comparing with the midpoints of the grid (a tie goes to the even code), the 8-bit one by rounding to 1/64."""
    rows, k = x.shape
    v = torch.zeros(rows, (k + BLOCK - 1) // BLOCK * BLOCK, dtype=torch.float64, device=x.device)
    v[:, :k] = x
    v = v.view(rows, -1, BLOCK)
    _, e = torch.frexp(v.abs().max(-1, keepdim=True).values)
    e = torch.where((v != 0).any(-1, keepdim=True), e - 1 - EMAX[fmt], -127).clamp(min=-127).double()
    a = v.abs() * torch.exp2(-e)
    if fmt == "int8":
        q = torch.round(a * 64).clamp(max=127) / 64
    else:
        q = torch.zeros_like(a)
        grid = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
        for i in range(7):
            middle = (grid[i] + grid[i + 1]) / 2
            q += (grid[i + 1] - grid[i]) * (a > middle if i % 2 == 0 else a >= middle)
    return (torch.sign(v) * q * torch.exp2(e)).view(rows, -1)[:, :k]


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].detach()
    if case["do"] == "keep":
        return _blocks64(x.double(), case["fmt"])
    bias = s["bias"].detach().double() if s["bias"] is not None else torch.zeros(case["n"], dtype=torch.float64, device=x.device)
    x4 = _blocks64(x.double(), "fp4")
    if case["do"] == "linear":
        gen = torch.Generator(device="cuda").manual_seed(seed)
        _activations(case["m"], case["k"], x.dtype, gen)
        w = 0.02 * torch.randn(case["n"], case["k"], device="cuda", generator=gen)
        y = torch.addmm(bias, x4, _blocks64(w.double(), "fp4").t())
        if case["epilogue"] == "relu":
            y = torch.relu(y)
        elif case["epilogue"] == "gelu":
            y = y * torch.special.ndtr(y)
        return y
    w4, dy = _blocks64(s["w"].detach().double(), "fp4"), s["dy"].double()
    y = torch.addmm(bias, x4, w4.t())
    del x4
    dx = torch.mm(dy, w4)
    dw = torch.mm(dy.t(), _blocks64(x.double(), "int8"))
    return _step(y, dx, dw, torch.mv(dy.t(), torch.ones(case["m"], dtype=torch.float64, device=x.device)) if case["bias"] else None)
