"""A call for every form of the attention over a quantised cache: the kernel, its name
(qattn_debug_quant_kernel), and sizes that get it.

A call is (name, (D, bits) that have the form, B, positions of the table, tokens per
sequence, q heads per kv head, kv heads, whether a token's heads lie side by side)."""
from __future__ import annotations

PAGE = 16
ALL = [(D, bits) for D in (32, 64, 128) for bits in (4, 8)]
HALF_LINES = [db for db in ALL if db != (128, 8)]     # rows of up to 64 bytes: two heads a line
QUARTERS = [(32, 4), (32, 8), (64, 4)]                # up to 32 bytes: four
ITEM, WIDE, NARROW = "quant_attn_kernel, a workgroup per item", "quant_wide_kernel", "quant_attn_kernel, "

FORMS = [
    (ITEM, ALL, 24, 480, 2, 4, 4, True),
    (ITEM, ALL, 6, 500, 3, 5, 3, False),
    (WIDE, ALL, 24, 3000, 13, 4, 4, True),
    (WIDE, ALL, 5, 9000, 40, 4, 3, False),
    (NARROW + "2 tiles, 1 head", ALL, 24, 3000, 6, 4, 4, True),
    (NARROW + "2 tiles, 1 head", ALL, 5, 5000, 8, 4, 2, False),
    (NARROW + "2 tiles, 2 heads, 2 sets", HALF_LINES, 24, 33000, 3, 4, 4, True),
    (NARROW + "2 tiles, 2 heads, 2 sets", HALF_LINES, 24, 11000, 4, 4, 12, True),
    (NARROW + "2 tiles, 2 heads, 4 sets", HALF_LINES, 24, 33000, 4, 4, 8, True),
    (NARROW + "1 head", ALL, 4, 4000, 4, 4, 8, True),        # drafts of a small batch
    (NARROW + "1 head", ALL, 24, 2000, 1, 4, 4, False),      # heads with gaps between them
    (NARROW + "1 head", ALL, 5, 3000, 2, 4, 3, True),
    (NARROW + "1 head, 2 sets", ALL, 24, 8000, 2, 4, 6, False),
    (NARROW + "1 head, 4 sets", ALL, 24, 8000, 2, 4, 8, False),
    (NARROW + "2 heads", HALF_LINES, 24, 3000, 2, 4, 8, True),
    (NARROW + "2 heads", HALF_LINES, 4, 6000, 1, 5, 2, True),
    (NARROW + "2 heads, 2 sets", HALF_LINES, 24, 11000, 2, 4, 4, True),
    (NARROW + "2 heads, 4 sets", HALF_LINES, 24, 11000, 2, 4, 8, True),
    (NARROW + "4 heads", QUARTERS, 4, 4000, 1, 4, 8, True),  # a decode step of a small batch
    (NARROW + "4 heads", QUARTERS, 24, 2000, 1, 3, 4, True),
    (NARROW + "4 heads, 2 sets", QUARTERS, 24, 11000, 1, 4, 8, True),
    (NARROW + "4 heads, 4 sets", QUARTERS, 24, 11000, 1, 4, 16, True),
]
CALLS = [(name, D, bits, *sizes) for name, sets, *sizes in FORMS for D, bits in sets]


def columns(positions):
    return -(-positions // PAGE)


def kernel_of(D, bits, B, positions, n, group, Hkv, together):
    """The kernel that a call of B sequences of n tokens gets, by the library's rule."""
    from qattention_amd import _lib
    return _lib.lib().qattn_debug_quant_kernel(B, n, B * n, group * Hkv, Hkv, D, columns(positions), PAGE, bits,
                                               together).decode()
