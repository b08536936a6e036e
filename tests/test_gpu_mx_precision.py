"""How near the microscaled product and its gradients are to 64 bits, with bounds that missing or coarse work does not keep."""

from __future__ import annotations

import pytest
import torch

from tests import _mx

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n", [(4, 200), (20, 77), (200, 264), (200, 131), (300, 10200), (2500, 2568)])
def test_gelu_of_fp32_results(cuda_device, m, n):
    """GELU in fp32 keeps its digits where it is small: a weight of zeros makes the bias the activation's argument.

    Bound: the argument of the error function is off by two roundings, 2^-23 in relative terms, which erfc passes on times
    v^2 + 1; erfc itself by 4 steps of 2^-23; the product with v by half a step."""
    from dimq_b200 import ops

    v = torch.linspace(-12.5, 9.0, n)
    q = ops.mx_quantize(torch.zeros(n, 32, device="cuda"))
    x = torch.randn(m, 32, device="cuda")
    v64 = v.double()
    want = (v64 * 0.5 * torch.special.erfc(-v64 / 2.0 ** 0.5)).expand(m, n)
    bound = want.abs() * (4 + v64.square() + 1 + 0.5) * 2.0 ** -23
    y = ops.mx_linear(x, *q, v.cuda(), n, 32, epilogue="gelu")
    _mx.check(y, want, bound)
    r = torch.randn(m, n, device="cuda")
    y = ops.mx_linear(x, *q, v.cuda(), n, 32, epilogue="gelu", residual=r)
    want = want + r.cpu().double()
    _mx.check(y, want, bound + 2.0 ** -24 * (want.abs() + bound))
