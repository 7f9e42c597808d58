"""The rule that chooses a form of the attention over a quantised cache, on the CPU: every
form that any call gets is one that the GPU tests run."""
from __future__ import annotations

import pytest

from quant_forms import CALLS, ITEM, kernel_of


@pytest.mark.parametrize("call", CALLS, ids=lambda c: "-".join(map(str, c)))
def test_the_forms_calls(call):
    assert kernel_of(*call[1:]) == call[0]


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("bits", [4, 8])
def test_no_form_without_a_call(D, bits):
    tested = {name for name, d, b, *_ in CALLS if (d, b) == (D, bits)}
    seen = {kernel_of(D, bits, B, positions, rows // group, group, Hkv, together)
            for together in (True, False) for Hkv in (1, 2, 3, 4, 6, 8, 12, 16, 32)
            for rows in (1, 2, 3, 4, 5, 8, 9, 12, 16, 17, 24, 32, 33, 60) for group in (1, 4) if rows % group == 0
            for B in (1, 2, 4, 8, 16, 24, 32, 64, 128, 300)
            for positions in (64, 500, 1000, 1024, 1500, 2000, 4000, 8000, 16000, 65536, 262144)}
    assert seen == tested


def test_nothing_to_launch():
    assert kernel_of(64, 4, 0, 500, 1, 4, 2, True) == "" and kernel_of(64, 4, 3, 500, 0, 4, 2, True) == ""


@pytest.mark.parametrize("D,bits", [(32, 4), (32, 8), (64, 4), (64, 8), (128, 4), (128, 8)])
def test_a_workgroup_per_item(D, bits):
    """Up to 4 steps of 8 waves, 1024 positions, of up to 256 (sequence, kv head) pairs; 2 steps
    where rows of 128 bytes belong to 64 pairs or fewer."""
    def items(B, positions, n=1):
        return kernel_of(D, bits, B, positions, n, 4, 8, True) == ITEM
    wide = D * bits == 1024
    for B in (1, 2, 8):
        assert items(B, 512) and items(B, 1024) == (not wide) and items(B, 528) == (not wide)
    for B in (9, 16, 32):
        assert items(B, 1024) and items(B, 1024, 4) and not items(B, 1040) and not items(B, 1024, 5)
    assert not items(33, 512)
