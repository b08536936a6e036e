"""How near the microscaled product and its gradients are to 64 bits, with bounds that missing or coarse work does not keep."""

from __future__ import annotations

import math

import pytest
import torch

from tests import _mx, _mx_forms

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


# ---- sums that are exact: every form has to give them to the bit -----------------------------------

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _grid(rows, cols, gen):
    """4-bit values as they are: signed grid values under block exponents -1, 0 and 1 (multiples of 1/4 up to 12)."""
    blocks = (cols + 31) // 32
    v = _mx.GRID.float().cuda()[torch.randint(0, 8, (rows, blocks, 32), device="cuda", generator=gen)]
    v[:, :, 0] = 4.0 + 2.0 * torch.randint(0, 2, (rows, blocks), device="cuda", generator=gen)     # the block's exponent
    v = torch.where(torch.rand(rows, blocks, 32, device="cuda", generator=gen) < 0.5, -v, v)
    e = torch.randint(-1, 2, (rows, blocks, 1), device="cuda", generator=gen).float()
    return (v * torch.exp2(e)).reshape(rows, -1)[:, :cols].contiguous()


def _bytes(rows, cols, gen):
    """8-bit values as they are: integers up to 127 over 64, one of 64 or more in every block, exponents -1, 0 and 1."""
    blocks = (cols + 31) // 32
    c = torch.randint(-127, 128, (rows, blocks, 32), device="cuda", generator=gen).float()
    c[:, :, 0] = torch.randint(64, 128, (rows, blocks), device="cuda", generator=gen).float()
    e = torch.randint(-1, 2, (rows, blocks, 1), device="cuda", generator=gen).float()
    return (c / 64 * torch.exp2(e)).reshape(rows, -1)[:, :cols].contiguous()


def _assert_exact(y, a, b, unit, what):
    """y = a @ b to the bit: products are multiples of `unit` and no partial sum, in whatever order, needs more than 24 bits."""
    a, b = a.double(), b.double()
    assert float((a.abs() @ b.abs()).max()) < 2.0 ** 24 * unit, "the data of this test"
    assert torch.equal(y, (a @ b).to(y.dtype)), what


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("m,k,n", _mx_forms.PRODUCTS)
def test_products_of_every_form_are_exact(cuda_device, m, k, n, name):
    from dimq_b200 import ops

    gen = torch.Generator(device="cuda").manual_seed(m + k + n)
    x, w = _grid(m, k, gen), _grid(n, k, gen)
    q = ops.mx_quantize(w)
    for out in {torch.float32, TYPES[name]}:
        _assert_exact(ops.mx_linear(x.to(TYPES[name]), *q, None, n, k, out_dtype=out), x, w.t(), 1 / 16, (_mx_forms.product_form(m, k, n), out))


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("m,k,n", _mx_forms.GRADIENTS)
def test_gradients_of_every_form_are_exact(cuda_device, m, k, n, name):
    """dy has as many bits as the sums leave room for: more than one bf16 term of fp16 and fp32 where they are short."""
    from dimq_b200 import ops

    gen = torch.Generator(device="cuda").manual_seed(m + k + n)
    dtype = TYPES[name]
    w, x8, x4 = _grid(n, k, gen), _bytes(m, k, gen), _grid(m, k, gen)

    def grad(depth, unit):       # values up to 2 in steps of 2^-bits, with room for `depth` products of them
        bits = max(0, min(6 if name == "bf16" else 8, int(math.log2(2.0 ** 24 * unit / (8.0 * depth)))))
        return (torch.randint(-2 << bits, (2 << bits) + 1, (m, n), device="cuda", generator=gen) / 2.0 ** bits).to(dtype), 2.0 ** -bits * unit

    for out in {torch.float32, dtype}:
        dy, unit = grad(n, 1 / 4)
        _assert_exact(ops.mx_linear_grad_input(dy, *ops.mx_quantize(w), k, out_dtype=out), dy, w, unit,
                      ("dx", _mx_forms.gradient_form(m, k, n, _mx_forms.TERMS[name])))
        for fmt, x, step in (("int8", x8, 1 / 128), ("fp4", x4, 1 / 4)):
            dy, unit = grad(m, step)
            _assert_exact(ops.mx_linear_grad_weight(dy, *ops.mx_quantize(x, fmt), k, fmt, out_dtype=out), dy.t(), x, unit,
                          ("dw " + fmt, _mx_forms.gradient_form(n, k, m, _mx_forms.TERMS[name])))


@pytest.mark.parametrize("m,k,n", _mx_forms.GRADIENTS)
def test_all_bits_of_an_fp32_gradient_count(cuda_device, m, k, n):
    """Twenty bits of dy, in few places: the three terms of every one of them are in the sums."""
    from dimq_b200 import ops

    gen = torch.Generator(device="cuda").manual_seed(m + k + n + 1)
    w, x8 = _grid(n, k, gen), _bytes(m, k, gen)
    far = torch.randint(-2 ** 20, 2 ** 20 + 1, (m, n), device="cuda", generator=gen).float()
    row = torch.arange(m, device="cuda")
    dy = torch.zeros(m, n, device="cuda")
    col = torch.randint(0, n, (m,), device="cuda", generator=gen)
    dy[row, col] = far[row, col] / 2.0 ** 10            # one value a row: dx is a multiple of a row of w
    dx = ops.mx_linear_grad_input(dy, *ops.mx_quantize(w), k).double()
    want = dy.double() @ w.double()
    # three exact products added up, largest last: two roundings or cuts
    assert float(((dx - want).abs() - 2.0 ** -22 * want.abs()).max()) <= 0
    dy = torch.zeros(m, n, device="cuda")
    other = torch.randint(0, m, (n,), device="cuda", generator=gen)
    at = torch.arange(n, device="cuda")
    dy[other, at] = far[other, at] / 2.0 ** 10          # one value a column: dw is a multiple of a row of x
    dw = ops.mx_linear_grad_weight(dy, *ops.mx_quantize(x8, "int8"), k).double()
    want = dy.double().t() @ x8.double()
    assert float(((dw - want).abs() - 2.0 ** -22 * want.abs()).max()) <= 0


# ---- sums that fp32 has to round -------------------------------------------------------------------

LONG = [(8, 32768, 256), (64, 32768, 256), (200, 11008, 8200), (300, 11008, 10200), (1300, 11008, 2600)]     # one of each form


def _values_of(x, fmt="fp4"):
    from dimq_b200 import ops

    codes, scales = ops.mx_quantize(x, fmt)
    return ops.mx_dequantize(codes, scales, x.shape[1], fmt).double(), int(ops.mx_scale_rows(scales, *x.shape).min()) - 127


@pytest.mark.parametrize("m,k,n", LONG)
def test_long_sums_of_normal_values_are_exact(cuda_device, m, k, n):
    """Normal values, mixed and of one sign: the codes have so few bits that no sum of 32768 products needs more than 24."""
    from dimq_b200 import ops

    gen = torch.Generator(device="cuda").manual_seed(1)
    for sign in (False, True):
        x, w = torch.randn(m, k, device="cuda", generator=gen), 0.02 * torch.randn(n, k, device="cuda", generator=gen)
        if sign:
            x, w = x.abs(), w.abs()
        (a, low_a), (b, low_b) = _values_of(x), _values_of(w)
        _assert_exact(ops.mx_linear(x, *ops.mx_quantize(w), None, n, k), a, b.t(), 2.0 ** (low_a + low_b - 2), sign)


@pytest.mark.parametrize("spread", [4, 12])
@pytest.mark.parametrize("m,k,n", LONG)
def test_long_sums_of_spread_blocks(cuda_device, m, k, n, spread):
    """Blocks up to 2^(4 spread) apart in their products, of mixed and of one sign.

    Bound: 64 products take one step of the tensor cores, each cutting the sum by at most a step of 2^-23 of it, a sum is at
    most sum |a||b|, and up to eight parts are added in fp32.  That is K / 64 + 9 cuts, where a bound over all K additions would
    let a 64-k step go missing."""
    from dimq_b200 import ops

    gen = torch.Generator(device="cuda").manual_seed(2)

    def values(rows):
        e = torch.randint(-spread, spread + 1, (rows, k // 32), device="cuda", generator=gen).float()
        return torch.randn(rows, k, device="cuda", generator=gen) * torch.exp2(e).repeat_interleave(32, 1)

    for sign in (False, True):
        x, w = values(m), values(n)
        if sign:
            x, w = x.abs(), w.abs()
        a, b = _values_of(x)[0], _values_of(w)[0].t()
        y = ops.mx_linear(x, *ops.mx_quantize(w), None, n, k).double()
        bound = (k / 64 + 9) * 2.0 ** -23 * (a.abs() @ b.abs())
        assert float(((y - a @ b).abs() - bound).max()) <= 0, sign


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("m,k,n", [(9000, 200, 264), (40, 136, 5000), (20000, 72, 264), (700, 2600, 1300)])
def test_long_gradient_sums_of_spread_values(cuda_device, m, k, n, name):
    """As above for the gradients: 16 products a step of the tensor cores, each off by at most two units of 2^-23 of a sum that
    is at most sum |a||b|; fp32 results are added up every 512 values of each term (32 steps, and one addition for every 512)."""
    from dimq_b200 import ops

    gen = torch.Generator(device="cuda").manual_seed(3)
    x, w = torch.randn(m, k, device="cuda", generator=gen), torch.randn(n, k, device="cuda", generator=gen)
    x *= torch.exp2(3 * torch.randn(m, 1, device="cuda", generator=gen))       # scales along the reduction
    w *= torch.exp2(3 * torch.randn(n, 1, device="cuda", generator=gen))
    dy = torch.randn(m, n, device="cuda", generator=gen).to(TYPES[name])
    terms = _mx_forms.TERMS[name]
    for out in {torch.float32, TYPES[name]}:
        for got, a, b, depth in ((ops.mx_linear_grad_input(dy, *ops.mx_quantize(w), k, out_dtype=out), dy, _values_of(w)[0], n),
                                 (ops.mx_linear_grad_weight(dy, *ops.mx_quantize(x, "int8"), k, out_dtype=out), dy.t(), _values_of(x, "int8")[0], m)):
            a = a.double()
            steps = 32 + terms * depth / 512 + 18 if out == torch.float32 else terms * depth / 16 + 34
            want = a @ b
            bound = 2 * steps * 2.0 ** -23 * (a.abs() @ b.abs())
            if out != torch.float32:
                bound = bound + torch.finfo(out).eps / 2 * (want.abs() + bound)
            assert float(((got.double() - want).abs() - bound).max()) <= 0, (out, depth)


def test_small_fp32_gradients(cuda_device):
    """An fp32 gradient enters as three bf16 terms, and bf16 has no bits under 2^-133: a value loses less than that, nothing else."""
    from dimq_b200 import ops

    gen = torch.Generator(device="cuda").manual_seed(4)
    m, k, n = 70, 64, 96
    w, x = torch.randn(n, k, device="cuda", generator=gen) * 2.0 ** 60, torch.randn(m, k, device="cuda", generator=gen) * 2.0 ** 60
    for power in (-108, -112, -120, -126, -130):
        dy = torch.randn(m, n, device="cuda", generator=gen) * 2.0 ** power
        for got, a, b, depth in ((ops.mx_linear_grad_input(dy, *ops.mx_quantize(w), k), dy, _values_of(w)[0], n),
                                 (ops.mx_linear_grad_weight(dy, *ops.mx_quantize(x, "int8"), k), dy.t(), _values_of(x, "int8")[0], m)):
            a = a.double()
            lost = 2.0 ** -133 * b.abs().sum(0)
            bound = lost + 2 * (3 * depth / 16 + 20) * 2.0 ** -23 * (a.abs() @ b.abs())
            assert float(((got.double() - a @ b).abs() - bound).max()) <= 0, power
            if power == -108:        # what is lost is under a quarter of a step of 2^-23 of a value of this size
                assert float((lost / (2.0 ** power * b.abs().sum(0))).max()) <= 2.0 ** -25
