"""CPU-only checks of the microscaled operators: sizes, argument errors before any launch, the 64-bit oracle, the scale
tiles' order."""

from __future__ import annotations

import ctypes as C

import pytest
import torch

from tests import _mx


@pytest.fixture(scope="module")
def lib():
    from dimq_b200 import _lib
    from dimq_b200.build import build

    build()
    return _lib.lib()


def test_sizes(lib):
    for rows, cols, fmt, pitch, scales in ((1, 1, 4, 16, 512), (128, 128, 4, 64, 512), (129, 129, 4, 80, 2048), (0, 32, 8, 32, 0), (5, 97, 8, 128, 512)):
        p, s = C.c_int64(0), C.c_int64(0)
        assert lib.dimq_mx_sizes(C.c_int64(rows), C.c_int64(cols), fmt, C.byref(p), C.byref(s)) == 0
        assert (p.value, s.value) == (pitch, scales)
    p = C.c_int64(0)
    assert lib.dimq_mx_sizes(C.c_int64(1), C.c_int64(1), 4, None, C.byref(p)) == -1
    assert lib.dimq_mx_sizes(C.c_int64(-1), C.c_int64(1), 4, C.byref(p), C.byref(p)) == -2
    assert lib.dimq_mx_sizes(C.c_int64(1), C.c_int64(0), 4, C.byref(p), C.byref(p)) == -2
    assert lib.dimq_mx_sizes(C.c_int64(1), C.c_int64(1), 5, C.byref(p), C.byref(p)) == -4
    assert lib.dimq_mx_sizes(C.c_int64(1 << 40), C.c_int64(1 << 40), 4, C.byref(p), C.byref(p)) == -11


def test_argument_errors_are_reported_without_a_gpu(lib):
    null, one, odd = C.c_void_p(0), C.c_void_p(256), C.c_void_p(24)
    i = C.c_int64
    assert lib.dimq_mx_quantize(one, 7, i(1), i(32), 4, one, one, null) == -3
    assert lib.dimq_mx_quantize(one, 0, i(1), i(32), 3, one, one, null) == -4
    assert lib.dimq_mx_quantize(one, 0, i(1), i(0), 4, one, one, null) == -2
    assert lib.dimq_mx_quantize(null, 0, i(1), i(32), 4, one, one, null) == -1
    assert lib.dimq_mx_quantize(one, 0, i(1), i(32), 4, odd, one, null) == -8
    assert lib.dimq_mx_quantize(null, 0, i(0), i(32), 4, null, null, null) == 0          # no rows: nothing to do
    assert lib.dimq_mx_quantize_both(one, 0, i(1), i(32), one, one, null, one, null) == -1
    assert lib.dimq_mx_dequantize(one, one, 4, i(1), i(32), one, 9, null) == -3
    assert lib.dimq_mx_dequantize(one, odd, 4, i(1), i(32), one, 0, null) == -8
    assert lib.dimq_mx_dequantize(null, null, 4, i(0), i(32), null, 0, null) == 0
    need = i(0)
    assert lib.dimq_mx_linear_workspace_bytes(i(4), i(0), i(32), 0, C.byref(need)) == -2
    assert lib.dimq_mx_linear_workspace_bytes(i(4), i(8), i(32), 0, None) == -1

    def linear(x=one, xd=0, xs=null, wc=one, ws=one, y=one, yd=0, m=200, n=8, k=32, epi=0, work=one, size=1 << 30):
        return lib.dimq_mx_linear(x, xd, xs, wc, ws, null, 0, null, y, yd, i(m), i(n), i(k), epi, work, i(size), null)

    assert linear(xd=5) == -3 and linear(yd=5) == -3 and linear(n=0) == -2 and linear(k=-1) == -2 and linear(m=-1) == -2
    assert linear(epi=9) == -7 and linear(x=null) == -1 and linear(wc=null) == -1 and linear(ws=null) == -1 and linear(y=null) == -1
    assert linear(work=null) == -12 and linear(size=0) == -12 and linear(m=0) == 0 and linear(n=1 << 40) == -11
    assert linear(wc=odd) == -8 and linear(ws=odd) == -8 and linear(work=odd) == -8 and linear(xs=odd) == -8

    def grad_in(dy=one, dyd=0, wc=one, ws=one, dx=one, dxd=0, m=2, n=8, k=32, work=one, size=1 << 30):
        return lib.dimq_mx_grad_input(dy, dyd, wc, ws, dx, dxd, i(m), i(n), i(k), work, i(size), null)

    assert grad_in(dyd=4) == -3 and grad_in(dxd=4) == -3 and grad_in(dy=null) == -1 and grad_in(dx=null) == -1 and grad_in(wc=null) == -1
    assert grad_in(k=0) == -2 and grad_in(m=0) == 0 and grad_in(wc=odd) == -8 and grad_in(work=null) == -12 and grad_in(size=8) == -12

    def grad_w(dy=one, dyd=0, xc=one, xs=one, fmt=8, dw=one, dwd=0, db=null, dbd=0, m=2, n=8, k=32, work=one, size=1 << 30):
        return lib.dimq_mx_grad_weight(dy, dyd, xc, xs, fmt, dw, dwd, db, dbd, i(m), i(n), i(k), work, i(size), null)

    assert grad_w(fmt=2) == -4 and grad_w(dyd=4) == -3 and grad_w(dwd=4) == -3 and grad_w(db=one, dbd=4) == -3
    assert grad_w(dw=null) == -1 and grad_w(dy=null) == -1 and grad_w(xc=null) == -1 and grad_w(n=0) == -2
    assert grad_w(xs=odd) == -8 and grad_w(work=null) == -12 and grad_w(size=8) == -12

    def grads(dy=one, wc=one, ws=one, xc=one, xs=one, fmt=8, dx=one, dw=one, db=one, m=2, work=one, size=1 << 30):
        return lib.dimq_mx_grads(dy, 0, wc, ws, xc, xs, fmt, dx, 0, dw, 0, db, 0, i(m), i(8), i(32), work, i(size), null)

    assert grads(dx=null, dw=null, db=null) == -1 and grads(dy=null) == -1 and grads(wc=null) == -1 and grads(xs=null) == -1
    assert grads(fmt=5) == -4 and grads(ws=odd) == -8 and grads(dy=odd) == -8 and grads(work=null) == -12 and grads(m=-1) == -2
    assert lib.dimq_mx_grad_workspace_bytes(5, i(1), i(1), i(1), C.byref(need)) == -3
    assert lib.dimq_mx_grad_workspace_bytes(0, i(1), i(1), i(1), None) == -1


def test_operators_refuse_cpu_tensors_and_unknown_formats(lib):
    from dimq_b200 import ops, qat

    x = torch.zeros(2, 32)
    for call in (lambda: ops.mx_quantize(x), lambda: ops.mx_linear(x, x, x, None, 2, 32), lambda: ops.mx_linear_grad_input(x, x, x, 32),
                 lambda: ops.mx_linear_grad_weight(x, x, x, 32), lambda: qat.mx_linear(x, x), lambda: ops.mx_dequantize(x, x, 32)):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(ValueError):
        ops.mx_quantize(x, "e4m3")
    with pytest.raises(ValueError):
        qat.mx_linear(x, x, checkpoint="bf16")


def test_scale_rows_undoes_the_tiles(lib):
    from dimq_b200 import ops

    rows, cols = 300, 330
    tiles = torch.zeros(3, 3, 512, dtype=torch.uint8)
    byte = torch.randint(1, 255, (rows, 11), dtype=torch.uint8)
    for r in range(rows):
        for b in range(11):
            tiles[r // 128, b // 4, (r % 32) * 16 + (r // 32 % 4) * 4 + b % 4] = byte[r, b]
    assert torch.equal(ops.mx_scale_rows(tiles, rows, cols), byte)


def test_oracle_on_values_worked_by_hand():
    x = torch.zeros(1, 64)
    x[0, :6] = torch.tensor([7.0, 6.9, 2.5, 0.25, -0.75, -5.0])       # exponent 0: 7 is past the largest code
    x[0, 32:35] = torch.tensor([0.01, -0.005, 0.0])
    byte, code, value = _mx.quantize64(x, "fp4")
    assert byte[0, 0] == 127 and value[0, :6].tolist() == [6.0, 6.0, 2.0, 0.0, -1.0, -4.0]
    assert byte[0, 1] == 127 - 9 and value[0, 32:35].tolist() == [6 * 2.0 ** -9, -3 * 2.0 ** -9, 0.0]    # 0.01 = 5.12 * 2^-9, 0.005 = 2.56 * 2^-9
    byte, code, value = _mx.quantize64(x, "int8")
    assert byte[0, 0] == 129 and code[0, :3].tolist() == [112, 110, 40] and value[0, 0] == 7.0
