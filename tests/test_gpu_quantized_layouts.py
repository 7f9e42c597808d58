"""Caches whose heads lie side by side in a token are read several heads at a time, as
far as the scales' alignment lets their loads: the kernel that ran, and its results."""
from __future__ import annotations

import pytest
import torch

from attn64 import check
from test_gpu_quantized_context import context, queries, reference

pytestmark = pytest.mark.gpu
DEV = "cuda"


def padded(t, pad):
    """t with pad bytes behind the heads of each token."""
    heads, width = t.shape[2:]
    wide = torch.full(t.shape[:2] + (heads * width + pad,), 255, dtype=torch.uint8, device=DEV)
    view = wide.as_strided(t.shape, (wide.stride(0), wide.stride(1), width, 1))
    view.copy_(t)
    return view


@pytest.mark.parametrize("Hkv,D,bits,pad,heads", [
    # scales of a token: 4 bytes, 2 bytes, 12 bytes
    (4, 32, 4, 0, 4), (2, 64, 4, 0, 2), (4, 32, 8, 0, 4), (2, 32, 4, 0, 2), (2, 32, 8, 0, 2), (12, 32, 4, 0, 4),
    (6, 64, 8, 0, 2), (2, 128, 4, 0, 2),
    # ... and a few more that no head has: off the boundaries of four heads', of two heads'
    (4, 32, 4, 2, 1), (4, 32, 8, 1, 1), (2, 32, 4, 1, 1), (2, 64, 4, 2, 1), (4, 64, 4, 4, 4),
    # one head, or heads that do not pair
    (1, 64, 4, 0, 1), (3, 32, 8, 0, 1),
])
def test_heads_read_together(Hkv, D, bits, pad, heads):
    import qattention_amd as qa
    from qattention_amd import _lib
    ctx = [2111, 1, 0, 1777]
    cache, table, lens, rows = context(ctx, 16, Hkv, D, bits, 800 + D + Hkv)
    cache = cache._replace(K_scale=padded(cache.K_scale, pad), V_scale=padded(cache.V_scale, pad))
    Q = queries(len(ctx), 3 * Hkv, D, torch.bfloat16, 801)
    print("together", Hkv, D, bits, pad, flush=True)
    O, L = qa.prefix_attention_quantized(Q, cache, table, lens)
    assert _lib.last_kernel() == f"quant_attn_kernel, {heads} head{'s' if heads > 1 else ''}"
    check(O, L, reference(Q, rows, [1] * len(ctx)))
