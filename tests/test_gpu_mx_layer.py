"""The microscaled training layer (`qat.mx_linear`) and the layer deployed from it (`MXLinear`): argument forms, long batches,
equality of the two."""

from __future__ import annotations

import pytest
import torch

from tests import _mx

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("shape", [(1, 24), (24, 1), (2, 3, 4)])
def test_bias_of_any_shape_has_a_gradient(cuda_device, shape):
    """A bias of n values is taken in any shape, and its gradient has that shape."""
    from dimq_b200 import qat

    gen = torch.Generator().manual_seed(1)
    x, w = torch.randn(10, 64, generator=gen).cuda(), torch.randn(24, 64, generator=gen).cuda()
    b = torch.randn(24, generator=gen).cuda()
    dy = torch.randn(10, 24, generator=gen).cuda()
    flat = b.clone().requires_grad_()
    y = qat.mx_linear(x, w, flat)
    y.backward(dy)
    other = b.clone().view(shape).requires_grad_()
    z = qat.mx_linear(x, w, other)
    z.backward(dy)
    assert torch.equal(y, z) and other.grad.shape == shape and torch.equal(other.grad.flatten(), flat.grad)


def test_more_rows_than_a_grid_dimension_has_runs(cuda_device):
    """16.8 million rows: every gradient, the bias's too.  Small integers: sums are exact in any order."""
    from dimq_b200 import ops, qat

    m, n, k = 65536 * 256 + 77, 8, 8
    gen = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randint(-3, 4, (m, k), device="cuda", generator=gen, dtype=torch.int8).to(torch.bfloat16).requires_grad_()
    w = torch.randint(-3, 4, (n, k), device="cuda", generator=gen).float().requires_grad_()
    b = torch.zeros(n, device="cuda", requires_grad=True)
    dy = torch.randint(-2, 3, (m, n), device="cuda", generator=gen, dtype=torch.int8).to(torch.bfloat16)
    dy[-77:] = 2                                         # the last rows count
    dx, dw, db = torch.autograd.grad(qat.mx_linear(x, w, b), (x, w, b), dy)
    assert torch.equal(db, dy.double().sum(0).float())
    x8 = ops.mx_dequantize(*ops.mx_quantize(x.detach(), "int8"), k, "int8")
    assert torch.equal(x8, x.detach().float())           # integers up to 3 are what the 8-bit copy holds
    assert torch.equal(dw, (dy.double().t() @ x8.double()).float())
    w4 = ops.mx_dequantize(*ops.mx_quantize(w.detach()), k)
    assert torch.equal(dx[-300:], (dy[-300:].float() @ w4).to(torch.bfloat16))
