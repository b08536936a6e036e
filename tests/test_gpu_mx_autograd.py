"""Gradients through the microscaled product of packed weights (`ops.mx_linear`, `MXLinear`) against plain 64-bit torch."""

from __future__ import annotations

import math

import pytest
import torch

from tests import _mx

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _on_grid(rows, cols, seed, top=7):
    """Values that 4-bit blocks hold as they are (block exponent 0): rounding leaves them alone, sums of up to 1000 are exact."""
    gen = torch.Generator().manual_seed(seed)
    v = _mx.GRID.float()[torch.randint(0, top, (rows, cols), generator=gen)]
    v = torch.where(torch.rand(rows, cols, generator=gen) < 0.5, -v, v)
    v[:, ::32] = 4.0
    return v


def _formula(x, w, b, r, epilogue):
    z = x @ w.t()
    if b is not None:
        z = z + b.reshape(-1)
    if epilogue == "add_relu":
        return torch.relu(z + r if r is not None else z)
    if epilogue == "relu":
        z = torch.relu(z)
    if epilogue == "gelu":
        z = torch.nn.functional.gelu(z)
    return z if r is None else z + r


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("epilogue", [None, "relu", "gelu", "add_relu"])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("lead,k,n", [((5,), 96, 40), ((2, 70), 100, 136), ((300,), 64, 33)])
def test_product_gradients(cuda_device, lead, k, n, residual, epilogue, dtype):
    from dimq_b200 import ops

    m = math.prod(lead)
    x = _on_grid(m, k, 1).to(dtype).cuda().view(*lead, k).requires_grad_()
    w = _on_grid(n, k, 2)
    gen = torch.Generator().manual_seed(3)
    b = (torch.randint(-9, 10, (n,), generator=gen) / 4).cuda().requires_grad_()
    r = (torch.randint(-9, 10, (m, n), generator=gen) / 2).to(dtype).cuda().view(*lead, n).requires_grad_() if residual else None
    scale = 1 / 64 if epilogue == "gelu" else 1.0       # where the derivative is neither 0 nor 1
    codes, scales = ops.mx_quantize((w * scale).cuda())
    dy = (torch.randint(-8, 9, (m, n), generator=gen) / 4).to(dtype).cuda().view(*lead, n)
    y = ops.mx_linear(x, codes, scales, b, n, k, out_dtype=dtype, epilogue=epilogue, residual=r)
    assert y.requires_grad
    with torch.no_grad():                                # the same bits as without gradients
        assert torch.equal(y, ops.mx_linear(x, codes, scales, b, n, k, out_dtype=dtype, epilogue=epilogue, residual=r))
    leaves = [t for t in (x, b, r) if t is not None]
    got = torch.autograd.grad(y, leaves, dy)
    x64, b64 = x.detach().cpu().double().view(m, k).requires_grad_(), b.detach().cpu().double().requires_grad_()
    r64 = r.detach().cpu().double().view(m, n).requires_grad_() if residual else None
    want = torch.autograd.grad(_formula(x64, w.double() * scale, b64, r64, epilogue), [t for t in (x64, b64, r64) if t is not None],
                               dy.cpu().double().view(m, n))
    for name, leaf, g, e in zip("xbr", leaves, got, want):
        assert g.dtype == leaf.dtype and g.shape == leaf.shape
        if epilogue != "gelu" or name == "r":            # small multiples of 1/8: exact
            assert torch.equal(g.cpu().reshape(e.shape), e.to(g.dtype)), name
            continue
        # dz: the derivative in fp32 (its argument, its error function and three products, 2^-20 of |dy|) rounded to y's type,
        # then a sum of n (m) terms in fp32, rounded to the leaf's type
        d = dy.cpu().double().view(m, n).abs()
        each = (torch.finfo(dtype).eps / 2 * 1.13 + 2.0 ** -20) * d
        bound = each @ (w.double() * scale).abs() + _mx.product_bound(1.13 * d, (w.double() * scale).abs(), n) if name == "x" else \
            each.sum(0) + (m + 1) * 2.0 ** -23 * 1.13 * d.sum(0)
        _mx.check(g.reshape(e.shape), e, bound + _mx.rounding(e.abs() + bound, g.dtype), name)


def test_only_what_is_needed(cuda_device):
    from dimq_b200 import ops

    m, k, n = 20, 64, 24
    q = ops.mx_quantize(_on_grid(n, k, 4).cuda())
    ts = [_on_grid(m, k, 5).cuda(), torch.randn(n, device="cuda"), torch.randn(m, n, device="cuda")]
    dy = torch.randn(m, n, device="cuda")
    for epilogue in (None, "relu", "gelu", "add_relu"):
        call = lambda x, b, r: ops.mx_linear(x, *q, b, n, k, epilogue=epilogue, residual=r)          # noqa: E731
        full = [t.clone().requires_grad_() for t in ts]
        want = torch.autograd.grad(call(*full), full, dy)
        for i in range(3):
            leaves = [t.clone().requires_grad_(j == i) for j, t in enumerate(ts)]
            (g,) = torch.autograd.grad(call(*leaves), leaves[i], dy)
            assert torch.equal(g, want[i])
    assert not call(*ts).requires_grad
    with torch.no_grad():
        assert not call(*full).requires_grad
    # no rows
    x = torch.zeros(0, k, device="cuda", requires_grad=True)
    b = torch.zeros(n, device="cuda", requires_grad=True)
    ops.mx_linear(x, *q, b, n, k).sum().backward()
    assert x.grad.shape == (0, k) and not b.grad.any()
    # a weight written in place after the forward is noticed
    x = _on_grid(m, k, 5).cuda().requires_grad_()
    y = ops.mx_linear(x, *q, None, n, k)
    q[0].zero_()
    with pytest.raises(RuntimeError):
        y.sum().backward()


def test_second_derivatives_raise(cuda_device):
    from dimq_b200 import ops

    m, k, n = 20, 64, 24
    q = ops.mx_quantize(_on_grid(n, k, 6).cuda())
    x = _on_grid(m, k, 7).cuda().requires_grad_()
    (g,) = torch.autograd.grad(ops.mx_linear(x, *q, None, n, k, epilogue="gelu").square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        g.sum().backward(retain_graph=True)
    with pytest.raises(RuntimeError):      # cut off from x
        torch.autograd.grad(g.sum(), x)
    # the gradients' own entry points, given a gradient that has one
    dy = torch.randn(m, n, device="cuda", requires_grad=True)
    kept = ops.mx_quantize(x.detach(), "int8")
    for call in (lambda: ops.mx_linear_grad_input(dy, *q, k), lambda: ops.mx_linear_grad_weight(dy, *kept, k)):
        with pytest.raises(RuntimeError, match="once"):
            call().sum().backward()
        with torch.no_grad():
            assert not call().requires_grad


def test_frozen_layer_inside_a_trained_model(cuda_device):
    """An adapter in front of a frozen 4-bit layer gets the gradient of the same formula in 64 bits, also from a captured step."""
    from dimq_b200.modules import MXLinear

    torch.manual_seed(0)
    base = torch.nn.Linear(96, 48).cuda()
    layer = MXLinear.from_linear(base, epilogue="relu")
    scale = torch.full((96,), 1.0, device="cuda", requires_grad=True)
    x = _on_grid(37, 96, 8).cuda()
    layer(x * scale).sum().backward()
    w4 = _mx.quantize64(base.weight, "fp4")[2]
    z = x.cpu().double() @ w4.t() + base.bias.detach().cpu().double()
    want = ((z > 0).double() @ w4 * x.cpu().double()).sum(0)
    bound = 40 * 50 * 2.0 ** -23 * ((z > 0).double() @ w4.abs() * x.cpu().double().abs()).sum(0)
    _mx.check(scale.grad, want, bound + 1e-30)
    eager = torch.autograd.grad(layer(x * scale).sum(), scale)[0]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.autograd.grad(layer(x * scale).sum(), scale)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = torch.autograd.grad(layer(x * scale).sum(), scale)[0]
    for _ in range(2):
        got.detach().zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, eager)


def test_forward_mode_tangents_are_refused(cuda_device):
    """There is no forward-mode rule: a tangent raises instead of getting lost."""
    from torch.autograd import forward_ad

    from dimq_b200 import ops, qat

    m, k, n = 20, 64, 24
    w = _on_grid(n, k, 9).cuda()
    q = ops.mx_quantize(w)
    x, b, r = _on_grid(m, k, 10).cuda(), torch.randn(n, device="cuda"), torch.randn(m, n, device="cuda")
    with forward_ad.dual_level():
        dual = [forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, b, r)]
        for call in (lambda: ops.mx_linear(dual[0], *q, b, n, k), lambda: ops.mx_linear(x, *q, dual[1], n, k),
                     lambda: ops.mx_linear(x, *q, b, n, k, residual=dual[2]), lambda: qat.mx_linear(dual[0], w)):
            with pytest.raises((RuntimeError, NotImplementedError)):
                call()
        assert not ops.mx_linear(x, *q, b, n, k).requires_grad
