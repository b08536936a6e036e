"""The sizes that the microscaled tests use reach every kernel form that the dispatch can choose (tests/_mx_forms.py restates it)."""

from __future__ import annotations

from tests import _mx_forms as forms


def test_products_reach_every_form():
    seen = {forms.product_form(*s) for s in forms.PRODUCTS}
    assert seen == {"few rows", "64", "128", "256", "pair"}
    for form in seen:       # short and long sums of each; the second scale tile of a 256-wide tile in and out of the weight
        ks = [k for m, k, n in forms.PRODUCTS if forms.product_form(m, k, n) == form]
        assert min(ks) <= 520 and max(ks) >= 2050, form
    rest = {-(-n // 128) % 2 for m, k, n in forms.PRODUCTS if forms.product_form(m, k, n) == "256"}
    assert rest == {0, 1}


def test_gradients_reach_every_variant():
    seen = set()
    for m, k, n in forms.GRADIENTS:
        for name, terms in forms.TERMS.items():
            for rows, depth in ((m, n), (n, m)):
                for out_bytes in {4, 4 if name == "f32" else 2}:
                    seen.add(forms.gradient_variant(rows, k, depth, terms, out_bytes) + ((out_bytes,)))
    for form in ("64", "128", "256", "pair"):
        for want in (("whole", "added up", 4), ("whole", "one accumulator", 4), ("whole", "one accumulator", 2), ("sliced", "added up", 4),
                     ("sliced", "one accumulator", 2)):
            assert (form, *want) in seen, (form, want)


def test_launch_counts_follow_the_plan():
    """The library's own plan, as far as it shows in the number of kernels, for sizes of all kinds; argument errors."""
    import ctypes as C
    import random

    from dimq_b200 import _lib
    from dimq_b200.build import build

    build()
    lib, rng, i = _lib.lib(), random.Random(0), C.c_int64
    count = C.c_int(0)
    for dtype, terms in ((0, 3), (1, 2), (2, 1)):
        for _ in range(500):
            m, k, n = (int(2 ** rng.uniform(0, 14)) for _ in range(3))
            want = {"db": 1 + (m > 256), "dx": 2 + (forms.gradient_form(m, k, n, terms)[1] > 1), "dw": 2 + (forms.gradient_form(n, k, m, terms)[1] > 1)}
            split = dtype != 2 or n % 8 != 0
            for dx, dw, db in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 1)):
                assert lib.dimq_mx_grad_launches(dtype, i(m), i(n), i(k), dx, dw, db, C.byref(count)) == 0
                assert count.value == dx * want["dx"] + dw * want["dw"] + db * want["db"] + (split and (dx or dw))
    assert lib.dimq_mx_grad_launches(0, i(0), i(8), i(8), 1, 1, 1, C.byref(count)) == 0 and count.value == 0
    assert lib.dimq_mx_grad_launches(7, i(1), i(8), i(8), 1, 1, 1, C.byref(count)) == -3
    assert lib.dimq_mx_grad_launches(0, i(1), i(0), i(8), 1, 1, 1, C.byref(count)) == -2
    assert lib.dimq_mx_grad_launches(0, i(1), i(8), i(8), 1, 1, 1, None) == -1
