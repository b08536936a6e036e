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
