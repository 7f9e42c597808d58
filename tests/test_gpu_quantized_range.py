"""What the calls over a quantised cache say about values and rows at the edges: fp16
queries over values past fp16's range, and rows that a read leaves as they were."""
from __future__ import annotations

import pytest
import torch

import quant64
from attn64 import check, offsets
from test_gpu_quantized_context import context, queries, reference

pytestmark = pytest.mark.gpu
DEV = "cuda"
FP16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("ctx,n", [([300, 200], 1), ([300, 200], 5), ([300, 200], 50), ([3000, 2500], 1),
                                   ([3000, 2500], 5)])
def test_values_past_fp16(ctx, n, bits):
    """Values written from bf16 rows may lie past 65504.  bf16 queries attend them as they
    are; fp16 queries see infinities, in the rows, heads and dims that hold them alone."""
    from qattention_amd import prefix_attention_quantized
    Hkv, D, g = 2, 128, 4
    cache, table, lens, rows = context(ctx, 16, Hkv, D, bits, 811, dtype=BF16)
    # V of sequence 0, head 1, dims 32 .. 63 of key 70: 2^17 times the codes of N(0, 1)
    page, slot = int(table[0, 70 // 16]), 70 % 16
    cache.V_scale[page, slot, 1, 1] += 17
    v = quant64.decode(cache.V[page, slot], cache.V_scale[page, slot], bits)
    rows[0][1][70] = v
    past = v[1].abs() > 65504
    assert 0 < int(past.sum()) < 32 and bool(past[32:64].any())
    cu = offsets([n] * len(ctx)).to(DEV)
    for dtype in (BF16, FP16):
        Q = queries(n * len(ctx), g * Hkv, D, dtype, 812)
        print("range", ctx, n, bits, dtype, flush=True)
        O, L = prefix_attention_quantized(Q, cache, table, lens, cu, max_seqlen=n)
        o, lse, to, tl = reference(Q, rows, [n] * len(ctx))
        inf = torch.zeros_like(O, dtype=torch.bool)
        if dtype is FP16:
            inf[:n, g:] = past
        assert torch.equal(torch.isinf(O), inf) and not bool(torch.isnan(O).any())
        assert torch.equal(torch.signbit(O)[inf], torch.signbit(v[1]).expand_as(O)[inf])
        check(O.masked_fill(inf, 0), L, (o.masked_fill(inf, 0), lse, to.masked_fill(inf, 0), tl))
    # K there as well: scores of fp16 queries that are infinite or no number, in that head alone
    cache.K_scale[page, slot, 1, 0] += 17
    O, L = prefix_attention_quantized(Q, cache, table, lens, cu, max_seqlen=n)
    hit = torch.zeros_like(O, dtype=torch.bool)
    hit[:n, g:] = True
    assert not bool(torch.isfinite(L[:n, g:]).any())
    check(O.masked_fill(hit, 0), L.masked_fill(hit[..., 0], 0),
          (o.masked_fill(hit, 0), lse.masked_fill(hit[..., 0], 0), to.masked_fill(hit, 0),
           tl.masked_fill(hit[..., 0], 0)))


@pytest.mark.parametrize("more", [0, 100])
def test_rows_that_a_read_leaves(more):
    """Rows behind the last sequence, of bad offsets and past max_seqlen are left as they
    were (the Python call hands them back as they were allocated); every other row is written."""
    import qattention_amd as qa
    from qattention_amd import _lib
    Hkv, D, ps = 2, 64, 16
    cache = qa.quantized_kv_cache(8, ps, Hkv, D)
    for t, byte in zip(cache, (0x11, 0x11, 127, 127)):
        t.fill_(byte)
    table = torch.arange(8, dtype=torch.int32, device=DEV).view(1, 8).repeat(5 + more, 1)
    starts = torch.zeros(5 + more, dtype=torch.int32, device=DEV)
    # 9 rows, 3, none, one past the end, one before its start; the last sequence ends at 20 of 24
    cu = [0, 9, 12, 12, 30, 14] + [20] * more
    cu = torch.tensor(cu, dtype=torch.int32, device=DEV)
    T, most = 24, 4
    K, V = (torch.full((T, Hkv, D), 7.0, dtype=FP16, device=DEV) for _ in range(2))
    st = _lib.layout(K.stride())[0]
    cs, ss = (_lib.layout(t.stride()[:3] + (1,))[0] for t in (cache.K, cache.K_scale))
    stream = torch.cuda.current_stream().cuda_stream
    print("left", more, flush=True)
    rc = _lib.lib().qattn_quant_read(
        cache.K.data_ptr(), cache.V.data_ptr(), cs, cache.K_scale.data_ptr(), cache.V_scale.data_ptr(), ss,
        table.data_ptr(), 8, 8, ps, starts.data_ptr(), K.data_ptr(), st, V.data_ptr(), st, cu.data_ptr(), 5 + more, most,
        T, Hkv, D, _lib.DTYPE_F16, 4, stream)
    assert rc == 0
    torch.cuda.synchronize()
    written = torch.zeros(T, dtype=torch.bool, device=DEV)
    for a, e in zip(cu.tolist(), cu.tolist()[1:]):
        if 0 <= a <= e <= T:
            written[a:min(e, a + most)] = True
    assert int(written.sum()) == (11 if more else 7)
    for x in (K, V):
        assert bool((x[written] == 0.5).all()) and bool((x[~written] == 7).all())
