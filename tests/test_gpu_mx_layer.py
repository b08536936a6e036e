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


@pytest.mark.parametrize("dtype,m,n,k", [(torch.float16, 1 << 20, 64, 64), (torch.float16, 20000, 18944, 64), (torch.float16, 20000, 2432, 832),
                                         (torch.float16, 20000, 1920, 1216), (torch.float16, 20000, 1152, 3648),
                                         (torch.bfloat16, 1 << 22, 64, 64), (torch.bfloat16, 140000, 1920, 1216)])
def test_sums_over_many_rows_in_16_bits(cuda_device, m, n, k, dtype):
    """Weight gradients whose terms have one sign, over up to four million rows (in slices, and whole with every tile width):
    half a step of their 16-bit type from 64 bits and little more.

    Little: sums of 512 values take 32 steps of the tensor cores, each off by at most two units of 2^-23 of the sum (7.6e-6),
    and at most 512 + 16 of them are added in fp32 (3.2e-5 of bf16's 3.9e-3; at most 272 for fp16, 1.6e-5 of 4.9e-4)."""
    from dimq_b200 import ops

    gen = torch.Generator(device="cuda").manual_seed(3)
    dy = ((torch.rand(m, n, device="cuda", generator=gen) + 0.5) / 1024).to(dtype)
    kept = ops.mx_quantize((torch.rand(m, k, device="cuda", generator=gen) + 0.5).to(torch.bfloat16), "int8")
    g = ops.mx_linear_grad_weight(dy, *kept, k, "int8", out_dtype=dtype).double()
    x8 = ops.mx_dequantize(*kept, k, "int8")
    want = sum(dy[r:r + 65536].double().t() @ x8[r:r + 65536].double() for r in range(0, m, 65536))
    worst = float(((g - want).abs() / want).max())
    assert worst <= torch.finfo(dtype).eps / 2 + 64 * 2.0 ** -23 + (288 if dtype == torch.float16 else 528) * 2.0 ** -24, worst


def _spread(rows, cols, seed):
    """Normal values whose blocks of 32 differ by up to 2^24: sums that fp32 has to round."""
    gen = torch.Generator().manual_seed(seed)
    e = torch.randint(-12, 13, (rows, (cols + 31) // 32), generator=gen).float().repeat_interleave(32, 1)[:, :cols]
    return (torch.randn(rows, cols, generator=gen) * torch.exp2(e)).cuda()


@pytest.mark.parametrize("checkpoint", ["int8", "fp4", None])
@pytest.mark.parametrize("m,k,n", [(1, 8192, 72), (4, 4100, 40), (16, 8192, 130), (17, 1000, 64), (32, 8192, 72), (40, 8192, 72), (200, 1030, 300)])
def test_trained_and_deployed_products_have_the_same_bits(cuda_device, m, k, n, checkpoint):
    """Whatever the number of rows, and where the order of a sum shows (None: nothing needs a gradient)."""
    from dimq_b200 import ops, qat

    x, w = _spread(m, k, 4), _spread(n, k, 5)
    b = torch.randn(n, device="cuda")
    want = ops.mx_linear(x, *ops.mx_quantize(w), b, n, k)
    if checkpoint is None:
        assert torch.equal(qat.mx_linear(x, w, b), want)
        return
    x.requires_grad_(), w.requires_grad_()
    y = qat.mx_linear(x, w, b, checkpoint=checkpoint)
    assert torch.equal(y, want)
    dy = _spread(m, n, 6)
    dx, dw = torch.autograd.grad(y, (x, w), dy)          # what is kept is what the operators quantise
    kept = ops.mx_quantize(x.detach(), checkpoint)
    assert torch.equal(dw, ops.mx_linear_grad_weight(dy, *kept, k, checkpoint))
    assert torch.equal(dx, ops.mx_linear_grad_input(dy, *ops.mx_quantize(w.detach()), k))


@pytest.mark.parametrize("m", [1, 20, 150])
@pytest.mark.parametrize("dtype", TYPES)
def test_deployed_chain_repeats_the_training_forward(cuda_device, dtype, m):
    """Two layers: the same types and bits, so that the second one quantises the values it was trained on."""
    from dimq_b200 import qat
    from dimq_b200.modules import MXLinear

    torch.manual_seed(0)
    l1, l2 = torch.nn.Linear(1000, 130).cuda(), torch.nn.Linear(130, 40).cuda()
    with torch.no_grad():
        l1.weight.copy_(_spread(130, 1000, 7) * 0.01)
        x = torch.randn(m, 1000, device="cuda").to(dtype)
        h = qat.mx_linear(x, l1.weight, l1.bias)
        want = qat.mx_linear(torch.relu(h), l2.weight, l2.bias)
    d1, d2 = MXLinear.from_linear(l1, epilogue="relu"), MXLinear.from_linear(l2)
    got = d1(x)
    assert got.dtype == h.dtype == dtype and torch.equal(got, torch.relu(h))
    assert d2(got).dtype == dtype and torch.equal(d2(got), want)
    assert MXLinear.from_linear(l2, out_dtype=torch.float32)(got).dtype == torch.float32
