"""Microscaled quantisation, product and gradients against plain 64-bit torch (tests/_mx.py)."""

from __future__ import annotations

import math

import pytest
import torch

from tests import _mx

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _values(rows, cols, dtype, seed=0, spread=2.0):
    gen = torch.Generator().manual_seed(seed * 1009 + rows * 31 + cols)
    x = torch.randn(rows, cols, generator=gen) * torch.exp2(torch.randn(rows, cols, generator=gen) * spread)
    return x.to(dtype).cuda()


# ---- quantise / dequantise ------------------------------------------------------------------------

def _check_codes(x, fmt, codes, scales):
    from dimq_b200 import ops

    rows, cols = x.shape
    byte, code, value = _mx.quantize64(x, fmt)
    assert torch.equal(ops.mx_scale_rows(scales, rows, cols).cpu(), byte)
    padded = ops.mx_scale_rows(scales, scales.shape[0] * 128, scales.shape[1] * 128).cpu()
    padded[:rows, :byte.shape[1]] = 0
    assert not padded.any(), "scale padding is zero"
    got = codes.cpu()
    if fmt == "fp4":
        got = torch.stack((got & 15, got >> 4), -1).view(rows, -1).double()
        signs = (got >= 8) & (got > 8) | (code > 8)
        assert torch.equal(torch.where(signs, got, got % 8), torch.where(signs, code, code % 8))      # -0 is 0
    else:
        assert torch.equal(got.double(), code)
    return value


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("fmt", ["fp4", "int8"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 32), (3, 31), (2, 33), (33, 256), (129, 260), (128, 128), (257, 1000), (5, 8, ), (300, 77)])
def test_quantize_is_exact(cuda_device, rows, cols, fmt, dtype):
    from dimq_b200 import ops

    x = _values(rows, cols, dtype)
    codes, scales = ops.mx_quantize(x, fmt)
    value = _check_codes(x, fmt, codes, scales)
    for out in TYPES:
        y = ops.mx_dequantize(codes, scales, cols, fmt, out_dtype=out)
        assert y.dtype == out and torch.equal(y.cpu().double(), value.to(out).double())
    assert ops.mx_dequantize(codes, scales, cols, fmt).dtype == torch.float32


@pytest.mark.parametrize("fmt", ["fp4", "int8"])
def test_quantize_ties_and_ends(cuda_device, fmt):
    """Every midpoint of the grids, saturation, zeros of both signs, the largest and smallest floats, subnormals."""
    from dimq_b200 import ops

    steps = torch.arange(-512, 513) / 64.0                 # all fp4 midpoints and quarters between
    fine = torch.arange(-255, 256) / 128.0                 # int8: every half step
    rows = []
    for scale in (1.0, 2.0 ** -126, 2.0 ** 120, 2.0 ** -140, 2.0 ** -149, 2.0 ** 126):
        for v in (steps, fine, torch.zeros(64), -torch.zeros(32), torch.tensor([3.4028234663852886e38] * 3 + [1e38, -1e37])):
            v = (v.double() * scale).clamp(-3.4028234663852886e38, 3.4028234663852886e38)
            rows.append(torch.nn.functional.pad(v, (0, 1056 - v.numel())).float())
    x = torch.stack(rows).cuda()
    codes, scales = ops.mx_quantize(x, fmt)
    value = _check_codes(x, fmt, codes, scales)
    assert torch.equal(ops.mx_dequantize(codes, scales, 1056, fmt).cpu().double(), value)
    assert torch.equal(ops.mx_dequantize(codes, scales, 1056, fmt, out_dtype=torch.bfloat16).cpu(), value.to(torch.bfloat16))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("fmt", ["fp4", "int8"])
def test_quantize_non_finite_blocks(cuda_device, fmt, dtype):
    from dimq_b200 import ops

    x = _values(5, 100, dtype)
    x[0, 3], x[1, 99], x[2, 32], x[3, 64] = float("nan"), float("inf"), -float("inf"), float("nan")
    codes, scales = ops.mx_quantize(x, fmt)
    value = _check_codes(x, fmt, codes, scales)
    y = ops.mx_dequantize(codes, scales, 100, fmt).cpu().double()
    assert torch.equal(y.isnan(), value.isnan()) and torch.equal(y.nan_to_num(), value.nan_to_num())
    assert int(value.isnan().sum()) == 32 * 3 + 4


def test_quantize_shapes_strides_and_alignment(cuda_device):
    from dimq_b200 import ops

    x = _values(24, 96, torch.bfloat16)
    want = ops.mx_quantize(x)
    for view in (x.t().contiguous().t(), torch.cat((x, x), 1)[:, :96], torch.cat((x.new_zeros(1), x.flatten()))[1:].view(24, 96)):
        got = ops.mx_quantize(view)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    codes, scales = ops.mx_quantize(x.view(2, 3, 4, 96))
    assert codes.shape == (2, 3, 4, 48) and torch.equal(codes.view(24, 48), want[0]) and torch.equal(scales, want[1])
    assert torch.equal(ops.mx_dequantize(codes, scales, 96), ops.mx_dequantize(*want, 96).view(2, 3, 4, 96))
    one = ops.mx_quantize(x[0])
    assert one[0].shape == (48,) and torch.equal(one[0], want[0][0])
    odd = torch.cat((want[0].new_zeros(1), want[0].flatten()))[1:].view(24, 48)          # codes at an odd address
    assert torch.equal(ops.mx_dequantize(odd, scales, 96), ops.mx_dequantize(*want, 96))
    codes, scales = ops.mx_quantize(x[:0])
    assert codes.shape == (0, 48) and scales.shape == (0, 1, 512) and ops.mx_dequantize(codes, scales, 96).shape == (0, 96)


# ---- product --------------------------------------------------------------------------------------

def _activate(v, epilogue):
    if epilogue in ("relu", "add_relu"):
        return v.clamp(min=0)
    if epilogue == "gelu":
        return 0.5 * v * (1 + torch.erf(v / math.sqrt(2)))
    return v


def _check_linear(y, x4, w4, bias, epilogue, residual, out_dtype):
    rows = x4.shape[0]
    sums = x4.nan_to_num() @ w4.nan_to_num().t()
    sums[x4.isnan().any(1)] = float("nan")
    sums[:, w4.isnan().any(1)] = float("nan")
    if bias is not None:
        sums = sums + bias.detach().cpu().double()
    r = 0 if residual is None else residual.detach().cpu().double().view(rows, -1)
    want = _activate(sums + r, epilogue) if epilogue == "add_relu" else _activate(sums, epilogue) + r
    # the sums, three more fp32 operations, and an error function good to 2^-22 of its argument
    bound = 1.2 * _mx.product_bound(x4.nan_to_num(), w4.nan_to_num().t(), x4.shape[1]) + 2.0 ** -22 * (sums.abs() + want.abs())
    if residual is not None:
        bound = bound + 2.0 ** -23 * r.abs()
    _mx.check(y.reshape(rows, -1), want, bound.nan_to_num() + _mx.rounding(want.nan_to_num() + bound.nan_to_num(), out_dtype), "y")


LINEAR = [(1, 1, 1), (1, 32, 8), (3, 33, 7), (2, 100, 128), (8, 256, 130), (16, 1000, 129), (17, 1024, 64), (32, 16500, 136), (27, 4100, 300), (1, 4096, 256), (5, 8320, 128),
          (33, 520, 257), (64, 2050, 100), (128, 128, 128), (130, 300, 257), (197, 768, 96), (300, 1001, 515), (257, 512, 640),
          (16, 16500, 130), (5, 32768, 40), (3, 33000, 40), (2500, 330, 2568), (1300, 4420, 2600)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", LINEAR)
def test_linear(cuda_device, m, k, n, dtype):
    from dimq_b200 import ops

    x, w = _values(m, k, dtype, 1, 0.5), _values(n, k, torch.float32, 2, 0.5)
    codes, scales = ops.mx_quantize(w)
    x4, w4 = _mx.quantize64(x, "fp4")[2], _mx.quantize64(w, "fp4")[2]
    bias = torch.randn(n, device="cuda").to(dtype)
    _check_linear(ops.mx_linear(x, codes, scales, None, n, k, out_dtype=dtype), x4, w4, None, None, None, dtype)
    _check_linear(ops.mx_linear(x, codes, scales, bias, n, k), x4, w4, bias, None, None, torch.float32)


@pytest.mark.parametrize("out_dtype", TYPES)
@pytest.mark.parametrize("epilogue", ["none", "relu", "gelu", "add_relu"])
@pytest.mark.parametrize("m,k,n", [(4, 288, 136), (150, 320, 264), (7, 65, 33), (140, 65, 131)])
def test_linear_epilogues_and_residual(cuda_device, m, k, n, epilogue, out_dtype):
    from dimq_b200 import ops

    x, w = _values(m, k, torch.bfloat16, 3, 0.5), _values(n, k, torch.float32, 4, 0.5)
    codes, scales = ops.mx_quantize(w)
    x4, w4 = _mx.quantize64(x, "fp4")[2], _mx.quantize64(w, "fp4")[2]
    bias = torch.randn(n, device="cuda")
    residual = (torch.randn(m, n, device="cuda") * 4).to(out_dtype)
    for b, r in ((bias, residual), (None, residual), (bias, None)):
        y = ops.mx_linear(x, codes, scales, b, n, k, out_dtype=out_dtype, epilogue=epilogue, residual=r)
        _check_linear(y, x4, w4, b, epilogue, r, out_dtype)


@pytest.mark.parametrize("m,k,n", [(3, 200, 40), (20, 96, 40), (200, 300, 300)])
def test_linear_non_finite_and_extreme_blocks(cuda_device, m, k, n):
    """A NaN or an infinity of x or w reaches the whole block's products: its row or column is NaN, no other value changes.
    Blocks of the smallest and largest exponents multiply exactly."""
    from dimq_b200 import ops

    x, w = _values(m, k, torch.float32, 5, 0.5), _values(n, k, torch.float32, 6, 0.5)
    x[1, 40], w[7, 0], w[n - 1, k - 1] = float("inf"), float("nan"), -float("inf")
    x[0] *= 2.0 ** -100
    w[3] *= 2.0 ** 110
    w[4] = 0
    codes, scales = ops.mx_quantize(w)
    x4, w4 = _mx.quantize64(x, "fp4")[2], _mx.quantize64(w, "fp4")[2]
    y = ops.mx_linear(x, codes, scales, None, n, k)
    assert torch.equal(y.isnan().any(0).cpu().nonzero().flatten(), torch.arange(n))     # row 1
    _check_linear(y, x4, w4, None, None, None, torch.float32)
    for epilogue in ("relu", "gelu"):                       # a NaN stays one
        z = ops.mx_linear(x, codes, scales, None, n, k, epilogue=epilogue, out_dtype=torch.bfloat16)
        assert torch.equal(z.isnan(), y.isnan())


def test_linear_leading_dimensions_strides_empty(cuda_device):
    from dimq_b200 import ops

    x, w = _values(24, 96, torch.bfloat16, 7), _values(40, 96, torch.float32, 8)
    codes, scales = ops.mx_quantize(w)
    want = ops.mx_linear(x, codes, scales, None, 40, 96)
    assert torch.equal(ops.mx_linear(x.view(2, 3, 4, 96), codes, scales, None, 40, 96), want.view(2, 3, 4, 40))
    assert torch.equal(ops.mx_linear(x.t().contiguous().t(), codes, scales, None, 40, 96), want)
    odd = torch.cat((codes.new_zeros(1), codes.flatten()))[1:].view(40, 48)
    odd_scales = torch.cat((scales.new_zeros(1), scales.flatten()))[1:].view(scales.shape)
    assert torch.equal(ops.mx_linear(torch.cat((x.new_zeros(1), x.flatten()))[1:].view(24, 96), odd, odd_scales, None, 40, 96), want)
    assert ops.mx_linear(x[:0], codes, scales, None, 40, 96).shape == (0, 40)
    assert torch.equal(ops.mx_linear(x[3], codes, scales, None, 40, 96), want[3])
    # the bias may start anywhere
    bias = torch.randn(41, device="cuda").bfloat16()[1:]
    assert torch.equal(ops.mx_linear(x, codes, scales, bias, 40, 96), ops.mx_linear(x, codes, scales, bias.clone(), 40, 96))


@pytest.mark.parametrize("m", [1, 16, 17, 32, 33, 128, 500])
def test_linear_rows_do_not_depend_on_their_neighbours(cuda_device, m):
    """A row's result is the same bits twice, and does not change with the values of the other rows."""
    from dimq_b200 import ops

    x, w = _values(m, 640, torch.bfloat16, 9, 0.5), _values(264, 640, torch.float32, 10, 0.5)
    codes, scales = ops.mx_quantize(w)
    y = ops.mx_linear(x, codes, scales, None, 264, 640)
    assert torch.equal(y, ops.mx_linear(x, codes, scales, None, 264, 640))
    other = x.clone()
    other[1:] = 7
    assert torch.equal(ops.mx_linear(other, codes, scales, None, 264, 640)[0], y[0])


# ---- gradients ------------------------------------------------------------------------------------

GRADS = [(1, 1, 1), (1, 64, 32), (3, 33, 7), (64, 128, 64), (130, 260, 129), (100, 1000, 72), (513, 96, 200), (257, 300, 515), (2000, 64, 40), (700, 2600, 1300), (9000, 200, 264), (40, 136, 5000)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", GRADS)
def test_gradients(cuda_device, m, k, n, dtype):
    from dimq_b200 import ops

    x, w = _values(m, k, dtype, 11, 0.5), _values(n, k, torch.float32, 12, 0.5)
    dy = _values(m, n, dtype, 13, 1.0)
    g64 = dy.cpu().double()
    w4 = _mx.quantize64(w, "fp4")[2]
    w_q = ops.mx_quantize(w)
    for out in (torch.float32, dtype):
        dx = ops.mx_linear_grad_input(dy, *w_q, k, out_dtype=out)
        want, bound = g64 @ w4, _mx.product_bound(g64, w4, 3 * n)
        _mx.check(dx, want, bound + _mx.rounding(want.abs() + bound, out), "dx")
        for fmt in ("int8", "fp4"):
            x8 = _mx.quantize64(x, fmt)[2]
            dw = ops.mx_linear_grad_weight(dy, *ops.mx_quantize(x, fmt), k, fmt, out_dtype=out)
            want, bound = g64.t() @ x8, _mx.product_bound(g64.t(), x8, 3 * m)
            _mx.check(dw, want, bound + _mx.rounding(want.abs() + bound, out), "dw " + fmt)


@pytest.mark.parametrize("checkpoint", ["int8", "fp4"])
@pytest.mark.parametrize("dtype,w_dtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
                                           (torch.float16, torch.float16), (torch.float16, torch.float32)])
@pytest.mark.parametrize("lead,k,n,bias", [((5,), 40, 9, True), ((2, 70), 256, 130, True), ((300,), 513, 264, False), ((1,), 96, 64, True)])
def test_layer_forward_and_backward(cuda_device, lead, k, n, bias, dtype, w_dtype, checkpoint):
    from dimq_b200 import ops, qat

    m = math.prod(lead)
    x = _values(m, k, dtype, 14, 0.5).view(*lead, k).requires_grad_()
    w = _values(n, k, w_dtype, 15, 0.5).requires_grad_()
    b = torch.randn(n, device="cuda").to(dtype).requires_grad_() if bias else None
    y = qat.mx_linear(x, w, b, checkpoint=checkpoint)
    assert y.shape == (*lead, n) and y.dtype == dtype
    x4, w4 = _mx.quantize64(x.view(m, k), "fp4")[2], _mx.quantize64(w, "fp4")[2]
    _check_linear(y, x4, w4, b, None, None, dtype)
    assert torch.equal(y, ops.mx_linear(x.detach(), *ops.mx_quantize(w.detach()), None if b is None else b.detach(), n, k, out_dtype=dtype))
    dy = _values(m, n, dtype, 16, 1.0).view(*lead, n)
    y.backward(dy)
    g = dy.view(m, n).cpu().double()
    x8 = _mx.quantize64(x.view(m, k), checkpoint)[2]
    for name, leaf, want, bound in (("dx", x, g @ w4, _mx.product_bound(g, w4, 3 * n)),
                                    ("dw", w, g.t() @ x8, _mx.product_bound(g.t(), x8, 3 * m))):
        assert leaf.grad.dtype == leaf.dtype and leaf.grad.shape == leaf.shape
        _mx.check(leaf.grad.reshape(want.shape), want, bound + _mx.rounding(want.abs() + bound, leaf.dtype), name)
    if bias:
        want, bound = g.sum(0), (m + 1) * 2.0 ** -23 * g.abs().sum(0)
        _mx.check(b.grad, want, bound + _mx.rounding(want.abs() + bound, b.dtype), "db")


def test_layer_gradient_against_differences(cuda_device):
    """On values the 4-bit grid holds, a step to the next grid value moves y by exactly step * w: differences of the layer's
    own forward give the gradients, and autograd of the same formula in 64 bits does too."""
    from dimq_b200 import qat

    gen = torch.Generator().manual_seed(3)
    grid = _mx.GRID.float()
    m, k, n = 6, 64, 5
    x, w = (grid[torch.randint(0, 7, (r, k), generator=gen)] * torch.where(torch.rand(r, k, generator=gen) < 0.5, -1.0, 1.0) for r in (m, n))
    x[:, ::32], w[:, ::32] = 6.0, 6.0                      # fixes every block's exponent at 0
    dy = torch.randint(-8, 9, (m, n), generator=gen).float()
    x, w, dy = (t.cuda() for t in (x, w, dy))

    def loss(a, b):
        return float((qat.mx_linear(a, b, None) * dy).sum())

    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    qat.mx_linear(xg, wg, None).backward(dy)
    base = loss(x, w)
    for t, grad, at in ((x, xg.grad, [(0, 1), (3, 17), (5, 63)]), (w, wg.grad, [(0, 2), (4, 40), (2, 31)])):
        for r, c in at:
            moved = t.clone()
            i = int((grid == abs(float(t[r, c]))).nonzero())
            moved[r, c] = grid[i + 1] * (1.0 if t[r, c] >= 0 else -1.0)
            step = float(moved[r, c] - t[r, c])
            got = (loss(moved, w) if t is x else loss(x, moved)) - base
            assert got == step * float(grad[r, c])        # small multiples of 1/4: exact in fp32
    x64, w64 = x.double().requires_grad_(), w.double().requires_grad_()
    ((x64 @ w64.t()) * dy.double()).sum().backward()
    assert torch.equal(xg.grad.double(), x64.grad) and torch.equal(wg.grad.double(), w64.grad)


def test_layer_only_what_is_needed(cuda_device):
    from dimq_b200 import qat

    x, w = _values(40, 64, torch.bfloat16, 17), _values(24, 64, torch.float32, 18)
    b = torch.randn(24, device="cuda")
    dy = _values(40, 24, torch.bfloat16, 19)
    full = [t.clone().requires_grad_() for t in (x, w, b)]
    qat.mx_linear(*full).backward(dy)
    for i in range(3):
        leaves = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, w, b))]
        y = qat.mx_linear(*leaves)
        y.backward(dy)
        assert torch.equal(leaves[i].grad, full[i].grad)
        assert all(leaves[j].grad is None for j in range(3) if j != i)
    with torch.no_grad():
        assert not qat.mx_linear(*full).requires_grad
    # a gradient that is broadcast, one with other strides, a layer used twice
    y = qat.mx_linear(full[0], full[1], full[2])
    got = torch.autograd.grad(y.sum(), full)
    y = qat.mx_linear(full[0], full[1], full[2])
    want = torch.autograd.grad(y, full, torch.ones_like(y))
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    y = qat.mx_linear(full[0], full[1], full[2])
    got = torch.autograd.grad(y, full, dy.t().contiguous().t())
    assert all(torch.equal(a, c.grad) for a, c in zip(got, full))
    with pytest.raises(RuntimeError):      # the rounding has no second derivative
        y = qat.mx_linear(full[0], full[1], full[2])
        (g,) = torch.autograd.grad(y.float().square().sum(), full[0], create_graph=True)
        torch.autograd.grad(g.float().sum(), full[1])


def test_layer_under_saved_tensor_hooks_and_recomputation(cuda_device):
    """What the layer keeps may wait on the host, be computed again, or come back wrong (which is refused)."""
    from torch.utils.checkpoint import checkpoint

    from dimq_b200 import qat

    leaves = [t.requires_grad_() for t in (_values(40, 96, torch.bfloat16, 17), _values(24, 96, torch.float32, 18), torch.randn(24, device="cuda"))]
    dy = _values(40, 24, torch.bfloat16, 19)
    want = torch.autograd.grad(qat.mx_linear(*leaves), leaves, dy)
    with torch.autograd.graph.save_on_cpu():
        y = qat.mx_linear(*leaves)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, dy), want))
    y = checkpoint(qat.mx_linear, *leaves, use_reentrant=False)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, dy), want))
    for spoil in (lambda t: t.cpu(), lambda t: t[:-1], lambda t: t.int()):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, spoil):
            y = qat.mx_linear(*leaves)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(y, leaves, dy)
    y = qat.mx_linear(*leaves)
    torch.autograd.grad(y, leaves, dy)
    with pytest.raises(RuntimeError):      # the graph is gone
        torch.autograd.grad(y, leaves, dy)


def test_layer_empty_batch(cuda_device):
    from dimq_b200 import qat

    x, w, b = torch.zeros(0, 64, device="cuda", requires_grad=True), _values(24, 64, torch.float32, 18).requires_grad_(), torch.zeros(24, device="cuda", requires_grad=True)
    y = qat.mx_linear(x, w, b)
    y.sum().backward()
    assert y.shape == (0, 24) and x.grad.shape == (0, 64) and not w.grad.any() and not b.grad.any()


def test_gradients_carry_non_finite_values(cuda_device):
    from dimq_b200 import ops

    x, w = _values(70, 64, torch.float32, 20), _values(40, 64, torch.float32, 21)
    for dtype in TYPES:
        dy = _values(70, 40, dtype, 22, 0.5)
        clean_dx = ops.mx_linear_grad_input(dy, *ops.mx_quantize(w), 64)
        clean_dw = ops.mx_linear_grad_weight(dy, *ops.mx_quantize(x, "int8"), 64)
        dy[3, 5] = float("nan")
        dx = ops.mx_linear_grad_input(dy, *ops.mx_quantize(w), 64)
        dw = ops.mx_linear_grad_weight(dy, *ops.mx_quantize(x, "int8"), 64)
        rows, cols = torch.arange(70, device="cuda") != 3, torch.arange(40, device="cuda") != 5
        assert dx[3].isnan().all() and torch.equal(dx[rows], clean_dx[rows])
        assert dw[5].isnan().all() and torch.equal(dw[cols], clean_dw[cols])
        dy[3, 5] = float("inf")
        w4 = ops.mx_dequantize(*ops.mx_quantize(w), 64)
        dx = ops.mx_linear_grad_input(dy, *ops.mx_quantize(w), 64)
        want = float("inf") * w4[5]
        assert torch.equal(dx[3].isnan(), want.isnan()) and torch.equal(dx[3].nan_to_num(0), want.nan_to_num(0))
        assert torch.equal(dx[rows], clean_dx[rows])


# ---- together -------------------------------------------------------------------------------------

def test_train_then_deploy(cuda_device):
    """Two layers trained for a few steps, then run from their packed weights: the same bits as the trained forward."""
    from dimq_b200 import qat
    from dimq_b200.modules import MXLinear

    torch.manual_seed(0)
    l1, l2 = torch.nn.Linear(96, 160).cuda(), torch.nn.Linear(160, 24).cuda()
    opt = torch.optim.SGD([*l1.parameters(), *l2.parameters()], lr=0.05)
    x, t = torch.randn(50, 96, device="cuda"), torch.randn(50, 24, device="cuda")
    for _ in range(3):
        h = torch.relu(qat.mx_linear(x, l1.weight, l1.bias))
        loss = (qat.mx_linear(h, l2.weight, l2.bias) - t).square().mean()
        opt.zero_grad()
        loss.backward()
        assert all(p.grad.isfinite().all() and p.grad.abs().sum() > 0 for p in [*l1.parameters(), *l2.parameters()])
        opt.step()
    with torch.no_grad():
        want = qat.mx_linear(torch.relu(qat.mx_linear(x, l1.weight, l1.bias)), l2.weight, l2.bias)
    d1, d2 = MXLinear.from_linear(l1, epilogue="relu"), MXLinear.from_linear(l2)
    assert torch.equal(d2(d1(x)), want)
    d3 = MXLinear.from_linear(torch.nn.Linear(96, 160).cuda(), epilogue="relu")
    d3.load_state_dict(d1.state_dict())
    assert torch.equal(d3(x), d1(x))


@pytest.mark.parametrize("m", [1, 8, 40, 300])
def test_capture_and_replay(cuda_device, m):
    """A captured pass of every operator gives the eager results on new inputs; two graphs share no scratch."""
    from dimq_b200 import ops

    k, n = 352, 200
    w = ops.mx_quantize(_values(n, k, torch.float32, 23, 0.5))
    xs, dys = [_values(m, k, torch.bfloat16, 24 + i) for i in range(3)], [_values(m, n, torch.bfloat16, 34 + i) for i in range(3)]

    def work(x, dy):
        kept = ops.mx_quantize(x, "int8")
        return (ops.mx_linear(x, *w, None, n, k), ops.mx_linear_grad_input(dy, *w, k), ops.mx_linear_grad_weight(dy, *kept, k),
                ops.mx_dequantize(*kept, k, "int8"))

    want = [work(x, dy) for x, dy in zip(xs, dys)]
    graphs = []
    for i in range(2):
        x, dy = xs[0].clone(), dys[0].clone()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            work(x, dy)
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = work(x, dy)
        graphs.append((g, x, dy, out))
    for order in ((0, 1), (1, 2), (2, 0)):
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for (g, x, dy, out), i, s in zip(graphs, order, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                x.copy_(xs[i])
                dy.copy_(dys[i])
                g.replay()
        torch.cuda.synchronize()
        for (g, x, dy, out), i in zip(graphs, order):
            assert all(torch.equal(a, b) for a, b in zip(out, want[i]))


def test_captured_training_step(cuda_device):
    from dimq_b200 import qat

    x, w = _values(64, 96, torch.bfloat16, 30).requires_grad_(), _values(48, 96, torch.float32, 31).requires_grad_()
    dy = _values(64, 48, torch.bfloat16, 32)
    want = torch.autograd.grad(qat.mx_linear(x, w), (x, w), dy)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.autograd.grad(qat.mx_linear(x, w), (x, w), dy)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = torch.autograd.grad(qat.mx_linear(x, w), (x, w), dy)
    for _ in range(2):
        for t in got:
            t.detach().zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(qat.mx_linear(x, w), (x, w), dy), want))


def test_threads_and_streams(cuda_device):
    """Calls of different sizes from several threads, each on its own stream."""
    import threading

    from dimq_b200 import ops

    w = ops.mx_quantize(_values(264, 1056, torch.float32, 40, 0.5))
    xs = {m: _values(m, 1056, torch.bfloat16, 41) for m in (1, 12, 100, 700)}
    dys = {m: _values(m, 264, torch.bfloat16, 42) for m in xs}

    def job(m):
        kept = ops.mx_quantize(xs[m], "int8")
        return ops.mx_linear(xs[m], *w, None, 264, 1056), ops.mx_linear_grad_input(dys[m], *w, 1056), ops.mx_linear_grad_weight(dys[m], *kept, 1056)

    want = {m: job(m) for m in xs}
    torch.cuda.synchronize()
    errors = []

    def run(m):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(100):
                    got = job(m)
                torch.cuda.current_stream().synchronize()
            if not all(torch.equal(a, b) for a, b in zip(got, want[m])):
                errors.append(f"wrong result for {m} rows")
        except Exception as e:          # noqa: BLE001 - reported below
            errors.append(repr(e))

    threads = [threading.Thread(target=run, args=(m,)) for m in xs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


def test_offsets_past_32_bits(cuda_device):
    """2.3e9 values: the last rows and columns are what they are in a call of their own."""
    from dimq_b200 import ops

    m, n, k = 70001, 32776, 64
    x, w = _values(m, k, torch.bfloat16, 50, 0.5), _values(n, k, torch.float32, 51, 0.5)
    wq = ops.mx_quantize(w)
    y = ops.mx_linear(x, *wq, None, n, k, out_dtype=torch.bfloat16)
    assert torch.equal(y[-3:], ops.mx_linear(x[-3:], *wq, None, n, k, out_dtype=torch.bfloat16))       # 64 terms of few bits: exact sums
    kept = ops.mx_quantize(x, "int8")
    dx, dw = ops.mx_linear_grad_input(y, *wq, k), ops.mx_linear_grad_weight(y, *kept, k)
    last = y[-3:].cpu().double()
    w4, x8 = _mx.quantize64(w, "fp4")[2], _mx.quantize64(x, "int8")[2]
    _mx.check(dx[-3:], last @ w4, _mx.product_bound(last, w4, n) + 1e-30, "dx")
    last = y[:, -3:].cpu().double()
    _mx.check(dw[-3:], last.t() @ x8, _mx.product_bound(last.t(), x8, m) + 1e-30, "dw")
    del dx, dw
    for fmt in ("fp4", "int8"):
        codes, scales = ops.mx_quantize(y, fmt)
        tail = ops.mx_quantize(y[-3:].contiguous(), fmt)
        assert torch.equal(codes[-3:], tail[0])
        z = ops.mx_dequantize(codes, scales, n, fmt, out_dtype=torch.bfloat16)
        assert torch.equal(z[-3:], ops.mx_dequantize(*tail, n, fmt, out_dtype=torch.bfloat16))
        del codes, scales, z


# ---- refusals -------------------------------------------------------------------------------------

def test_refusals(cuda_device):
    from dimq_b200 import ops, qat

    x, w = _values(4, 96, torch.bfloat16), _values(8, 96, torch.float32)
    codes, scales = ops.mx_quantize(w)
    c8, s8 = ops.mx_quantize(w, "int8")
    dy = torch.zeros(4, 8, device="cuda")
    refused = [
        lambda: ops.mx_quantize(x.double()), lambda: ops.mx_quantize(x.int()), lambda: ops.mx_quantize(x.cpu()),
        lambda: ops.mx_quantize(torch.tensor(1.0, device="cuda")), lambda: ops.mx_quantize(x[:, :0]),
        lambda: ops.mx_dequantize(c8, s8, 96, "fp4"), lambda: ops.mx_dequantize(codes, scales, 96, "int8"),
        lambda: ops.mx_dequantize(codes, scales, 97), lambda: ops.mx_dequantize(codes, scales, 64),
        lambda: ops.mx_dequantize(codes, scales, 0), lambda: ops.mx_dequantize(codes, scales.cpu(), 96),
        lambda: ops.mx_dequantize(codes, scales[:0], 96), lambda: ops.mx_dequantize(codes, scales.int(), 96),
        lambda: ops.mx_dequantize(codes, scales, 96, out_dtype=torch.float64),
        lambda: ops.mx_linear(x.cpu(), codes, scales, None, 8, 96), lambda: ops.mx_linear(x.double(), codes, scales, None, 8, 96),
        lambda: ops.mx_linear(x[:, :64], codes, scales, None, 8, 96), lambda: ops.mx_linear(x, codes, scales, None, 9, 96),
        lambda: ops.mx_linear(x, codes, scales, None, 8, 0), lambda: ops.mx_linear(x, codes.cpu(), scales, None, 8, 96),
        lambda: ops.mx_linear(x, codes[:, :32], scales, None, 8, 96), lambda: ops.mx_linear(x, c8, s8, None, 8, 96),
        lambda: ops.mx_linear(x, codes, scales[:, :, :256], None, 8, 96),
        lambda: ops.mx_linear(x, codes, scales, torch.zeros(7, device="cuda"), 8, 96),
        lambda: ops.mx_linear(x, codes, scales, torch.zeros(8), 8, 96),
        lambda: ops.mx_linear(x, codes, scales, None, 8, 96, residual=torch.zeros(4, 8, device="cuda").half()),
        lambda: ops.mx_linear(x, codes, scales, None, 8, 96, out_dtype=torch.float64),
        lambda: ops.mx_linear_grad_input(dy.double(), codes, scales, 96), lambda: ops.mx_linear_grad_input(dy[:, :7], codes, scales, 96),
        lambda: ops.mx_linear_grad_input(dy.cpu(), codes, scales, 96), lambda: ops.mx_linear_grad_input(dy, c8, s8, 96),
        lambda: ops.mx_linear_grad_weight(dy, *ops.mx_quantize(x[:3], "int8"), 96),
        lambda: ops.mx_linear_grad_weight(dy, *ops.mx_quantize(x, "int8"), 96, "fp4"),
        lambda: qat.mx_linear(x, w[:, :64]), lambda: qat.mx_linear(x, w[0]), lambda: qat.mx_linear(x, w.cpu()),
        lambda: qat.mx_linear(x, w, torch.zeros(7, device="cuda")), lambda: qat.mx_linear(x.double(), w),
        lambda: ops.mx_scale_rows(scales, 200, 96),
    ]
    for i, call in enumerate(refused):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"refusal {i} went through")
    for call in (lambda: ops.mx_quantize(x, "fp8"), lambda: qat.mx_linear(x, w, checkpoint=None), lambda: ops.mx_dequantize(codes, scales, 96, 4)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(KeyError):
        ops.mx_linear(x, codes, scales, None, 8, 96, epilogue="tanh")
    torch.cuda.synchronize()
    assert ops.last_device_status() == 0
