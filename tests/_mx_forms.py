"""Which kernel form a microscaled product or gradient of given sizes runs as: the rules of ``mx_small.cu``, ``mx_gemm.cu`` and
``mx_grad.cu`` restated, so that the tests can show that their sizes reach every form."""

from __future__ import annotations

SMS = 148


def up(a: int, b: int) -> int:
    return -(-a // b)


def product_form(m: int, k: int, n: int) -> str:
    """``"few rows"``, or the tile width of the many-row kernel (``"pair"``: 256 x 256 by two blocks)."""
    steps, row_blocks = up(up(up(k, 32), 4), 2), up(n, 128)
    if m <= 32 and steps <= 128:
        slices = 1
        while slices < 8 and 2 * slices <= steps and (row_blocks * slices * 2 <= 3 * SMS or up(steps, slices) > 16):
            slices *= 2
        if m <= 16 or up(steps, slices) <= 4:
            return "few rows"
    best, least = "", 0.0
    for form, width, rows, side, cost in (("pair", 256, 256, SMS // 2, 600), ("256", 256, 128, SMS, 768), ("128", 128, 128, SMS, 520),
                                          ("64", 64, 128, SMS, 430)):
        c = up(up(m, rows) * up(n, width), side) * cost
        if not best or c < least:
            best, least = form, c
    return best


def gradient_form(rows: int, cols: int, depth: int, terms: int) -> tuple[str, int]:
    """(tile width, slices of the reduction) of a gradient ``[rows, cols]`` over ``depth`` values of ``terms`` terms each."""
    steps = up(depth, 64) * terms
    best, least = ("", 0), -1.0
    for form, width, height, side, cost in (("pair", 256, 256, SMS // 2, 650), ("256", 256, 128, SMS, 750), ("128", 128, 128, SMS, 520),
                                            ("64", 64, 128, SMS, 430)):
        tiles = up(rows, height) * up(cols, width)
        for s in range(1, 17):
            if s > 1 and (s * 8 > steps or tiles * (s - 1) >= side):
                break
            c = up(tiles * s, side) * (up(steps, s) * cost + 2000.0)
            if s > 1:
                c += 6000.0 + rows * cols * 8.0 * s / 3000.0
            if least < 0 or c < least:
                best, least = (form, s), c
    return best


def gradient_variant(rows: int, cols: int, depth: int, terms: int, out_bytes: int) -> tuple[str, str, str]:
    """(tile width, whole or sliced, how the sums are kept) of the kernel that computes the gradient."""
    form, slices = gradient_form(rows, cols, depth, terms)
    blocks = up(depth, 64)
    if out_bytes == 4:
        added = blocks * terms > 8 * slices
    else:
        added = min(up(blocks * terms, slices), blocks) > 256      # fp16's limit; no test here is near bf16's
    return form, "sliced" if slices > 1 else "whole", "added up" if added else "one accumulator"


# (m, k, n) of products that between them run every form, short and long sums, no size a multiple of anything in most
PRODUCTS = [(1, 32768, 72), (5, 300, 40), (16, 16500, 130), (27, 4100, 300), (32, 1000, 264),
            (40, 33000, 72), (33, 520, 257), (130, 2050, 515),
            (197, 330, 8200), (512, 300, 4100), (130, 4420, 8201),
            (300, 330, 10200), (777, 130, 5100), (300, 2100, 10101),
            (2500, 330, 2568), (1300, 4420, 2600), (1300, 11000, 2601)]

# (m, k, n) of layers whose two gradients run every variant
GRADIENTS = [(1, 64, 32), (130, 260, 129), (500, 72, 72), (64, 3600, 264), (64, 3600, 1100), (64, 2000, 5000), (130, 2000, 1100),
             (1000, 1000, 130), (336, 3576, 1914), (9000, 200, 264), (700, 2600, 1300), (64, 500, 5000), (1914, 3576, 336),
             (218, 1060, 3602), (40, 136, 5000), (1600, 1500, 2000), (280, 1540, 1801)]
TERMS = {"bf16": 1, "f16": 2, "f32": 3}
