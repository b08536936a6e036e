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
