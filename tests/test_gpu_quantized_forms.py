"""Every form of the attention over a quantised cache against dense attention in 64 bits:
ragged contexts and tokens, an empty sequence, a missing page, blocks without a number that
stay in their own head and sequence, no numbers behind the contexts; that the form ran
that the rule names, and gives the same bits again."""
from __future__ import annotations

import pytest
import torch

import quant64
from attn64 import check, offsets
from quant_forms import CALLS, PAGE, columns, kernel_of
from test_gpu_quantized_context import queries, reference

pytestmark = pytest.mark.gpu
DEV = "cuda"


def blocks(g, bits, *shape):
    """Random elements and scales: blocks with largest magnitudes of .75 to 7."""
    D = 32 * shape[-1]
    e = torch.randint(0, 256, shape[:-1] + (D * bits // 8,), dtype=torch.uint8, device=DEV, generator=g)
    if bits == 8:
        e = torch.where(e % 128 == 127, e - 1, e)  # (e4m3's NaN)
    s = torch.randint(*((124, 127) if bits == 4 else (118, 121)), shape, device=DEV, generator=g)
    return e, s.to(torch.uint8)


def spread(t, together):
    """t as it is, or with gaps between the heads of a token."""
    if together:
        return t
    wide = torch.full(t.shape[:2] + (t.shape[2] + 1, 2 * t.shape[3]), 255, dtype=torch.uint8, device=DEV)
    view = wide[:, :, 1:, :t.shape[3]]
    view.copy_(t)
    return view


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("call", CALLS, ids=lambda c: "-".join(map(str, c)))
def test_form(call, dtype):
    import qattention_amd as qa
    from qattention_amd import _lib
    name, D, bits, B, positions, n, group, Hkv, together = call
    assert kernel_of(*call[1:]) == name
    g = torch.Generator(device=DEV).manual_seed(700 + D + bits + Hkv)
    ctx = min(positions - 20, 6000)
    held = [min(477, ctx), min(300, ctx), ctx, ctx - 100]  # two sequences' own, two that the others share
    first = [0]
    for m in held:
        first.append(first[-1] + columns(m))
    cache = qa.quantized_kv_cache(first[-1] + 1, PAGE, Hkv, D, bits=bits)
    order = torch.randperm(first[-1], generator=torch.Generator().manual_seed(701)).to(DEV)
    rows, tables = [], []
    for t in cache:
        t.fill_(255)
    for m, a, e in zip(held, first, first[1:]):
        at = order[a:e][torch.arange(m, device=DEV) // PAGE], torch.arange(m, device=DEV) % PAGE
        pair = []
        for x, s in ((cache.K, cache.K_scale), (cache.V, cache.V_scale)):
            x[at], s[at] = blocks(g, bits, m, Hkv, D // 32)
            pair.append(quant64.decode(x[at], s[at], bits))
        rows.append(tuple(pair))
        # (columns behind the context name the page without a number)
        table = torch.full((columns(positions),), first[-1], dtype=torch.int32, device=DEV)
        table[:e - a] = order[a:e].to(torch.int32)
        tables.append(table)
    # sequence 0 holds a block of K and one of V without a number; sequence 1 lacks a page
    cache.K_scale[int(tables[0][100 // PAGE]), 100 % PAGE, Hkv - 1, D // 32 - 1] = 255
    cache.V_scale[int(tables[0][200 // PAGE]), 200 % PAGE, 0, 0] = 255
    tables[1][3] = -1
    here = torch.ones(held[1], dtype=torch.bool, device=DEV)
    here[3 * PAGE:4 * PAGE] = False
    rows[1] = tuple(x[here] for x in rows[1])
    owner = [0, 1] + [2 + s % 2 for s in range(2, B)]
    lens = held[:2] + [held[2 + s % 2] - (37 * s * s) % (ctx // 2) if s % 9 else (0, 1, 33)[s // 9 % 3]
                       for s in range(2, B)]
    toks = [n, n] + [max(0, n - s % 3) if s % 5 else n for s in range(2, B)]
    views = qa.QuantizedKV(*(spread(t, together) for t in cache))
    page_table = torch.stack([tables[o] for o in owner])
    n_ctx = torch.tensor(lens, dtype=torch.int32, device=DEV)
    cu = offsets(toks).to(DEV)
    Q = queries(sum(toks), group * Hkv, D, dtype, 702)
    print(*call, dtype, flush=True)
    # (as many rows as the call may have: the lengths stay on the device)
    Q = torch.cat([Q, queries(B * n - sum(toks), group * Hkv, D, dtype, 703)])
    O, L = qa.prefix_attention_quantized(Q, views, page_table, n_ctx, cu, max_seqlen=n)
    assert _lib.last_kernel() == name
    T = sum(toks)
    again = qa.prefix_attention_quantized(Q, views, page_table, n_ctx, cu, max_seqlen=n)
    kv = [tuple(x[:m] for x in rows[o]) if o != 1 else rows[1] for o, m in zip(owner, lens)]
    o, lse, to, tl = reference(Q[:T], kv, toks)
    bad = torch.zeros_like(O[:T], dtype=torch.bool)
    bad[:n, (Hkv - 1) * group:] = True      # (K of the last head)
    bad[:n, :group, :32] = True             # (V of the first)
    bad_lse = torch.zeros_like(L[:T], dtype=torch.bool)
    bad_lse[:n, (Hkv - 1) * group:] = True
    O, L = O[:T], L[:T]
    assert torch.equal(torch.isnan(O), bad) and torch.equal(torch.isnan(L), bad_lse)
    clean = lambda x, m: x.masked_fill(m, 0)  # noqa: E731
    check(clean(O, bad), clean(L, bad_lse), (clean(o, bad), clean(lse, bad_lse), clean(to, bad), clean(tl, bad_lse)))
    assert torch.equal(clean(again[0][:T], bad), clean(O, bad))
    assert torch.equal(clean(again[1][:T], bad_lse), clean(L, bad_lse))
