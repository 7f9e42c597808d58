"""prefix_attention_quantized against dense attention in 64 bits over the values that
the cache stands for."""
from __future__ import annotations

import math

import pytest
import torch

import quant64
from attn64 import attend64, check, offsets

pytestmark = pytest.mark.gpu
DEV = "cuda"
FP16, BF16 = torch.float16, torch.bfloat16


def say(*a):
    print(*a, flush=True)


def context(ctx, ps, Hkv, D, bits, seed, extra=3, dtype=FP16, sigma=1.0):
    """A cache in shuffled pages, no numbers in every slot that no context fills (scale
    255, e4m3's NaN), and the contexts' K/V values in fp64."""
    import qattention_amd as qa
    g = torch.Generator().manual_seed(seed)
    pages = [-(-n // ps) for n in ctx]
    total, cols = sum(pages) + extra, max(pages + [1]) + 1
    cache = qa.quantized_kv_cache(total, ps, Hkv, D, bits=bits)
    for t in cache:
        t.fill_(255)
    order = torch.randperm(total, generator=g).to(torch.int32)
    table = torch.full((len(ctx), cols), -1, dtype=torch.int32)
    rows, first = [], 0
    for i, n in enumerate(ctx):
        table[i, :pages[i]] = order[first:first + pages[i]]
        first += pages[i]
        pair = []
        for e, s in ((cache.K, cache.K_scale), (cache.V, cache.V_scale)):
            x, y = quant64.encode((torch.randn(n, Hkv, D, generator=g) * sigma).to(dtype), bits)
            x, y = x.to(DEV), y.to(DEV)
            if n:
                at = table[i].long().to(DEV)[torch.arange(n, device=DEV) // ps], torch.arange(n, device=DEV) % ps
                e[at], s[at] = x, y
            pair.append(quant64.decode(x, y, bits))
        rows.append(tuple(pair))
    return cache, table.to(DEV), torch.tensor(ctx, dtype=torch.int32, device=DEV), rows


def queries(T, Hq, D, dtype, seed, sigma=1.0):
    g = torch.Generator().manual_seed(seed + 1)
    return (torch.randn(T, Hq, D, generator=g) * sigma).to(dtype).to(DEV)


def reference(Q, rows, lens):
    """attend64 with one bound more: a weight below fp32's smallest normal number, 2^-126
    of the row's largest, may count as 0, which takes 2^-126 |v_j| from the output.  It
    shows where the values of all larger weights are 0, as 4-bit elements often are."""
    parts, a = [], 0
    for n, (k, v) in zip(lens, rows):
        o, lse, to, tl = attend64(Q[a:a + n], k, v, torch.ones(n, k.shape[0], dtype=torch.bool, device=DEV))
        g = Q.shape[1] // v.shape[1]
        to = to + 2.0 ** -126 * v.abs().nan_to_num(0).sum(0).repeat_interleave(g, 0)
        parts.append((o, lse, to, tl))
        a += n
    return [torch.cat(x) for x in zip(*parts)]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("ctx,ps,Hq,Hkv,D", [
    ([1], 16, 4, 4, 64),
    ([0], 16, 4, 4, 64),
    ([0, 1, 15, 16, 17, 31, 32, 33], 16, 8, 2, 128),
    ([127, 128, 129, 0, 255, 256, 257], 16, 8, 2, 64),
    ([5, 0, 0, 200], 1, 4, 1, 32),
    ([300, 40], 7, 6, 2, 128),
    ([1000, 3], 64, 32, 8, 128),
    ([4000], 16, 32, 4, 128),
    ([1111, 700, 2], 16, 8, 8, 32),
    ([700, 650], 300, 16, 1, 64),
    ([90, 2000], 16, 24, 1, 128),   # 24 rows: two row blocks
    ([90, 1500], 16, 20, 1, 64),
    ([333, 1], 16, 40, 1, 64),      # 40 rows: the wide kernel
    ([150, 20], 16, 100, 1, 128),
])
def test_one_token(ctx, ps, Hq, Hkv, D, dtype, bits):
    from qattention_amd import prefix_attention_quantized
    cache, table, lens, rows = context(ctx, ps, Hkv, D, bits, 300 + sum(ctx) + D)
    Q = queries(len(ctx), Hq, D, dtype, 300)
    say("one token", ctx, ps, Hq, Hkv, D, dtype, bits)
    O, L = prefix_attention_quantized(Q, cache, table, lens)
    check(O, L, reference(Q, rows, [1] * len(ctx)))
    assert torch.equal(prefix_attention_quantized(Q, cache, table.cpu(), lens.cpu(), return_lse=False), O)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("B,ctx,Hq,Hkv,D", [
    (70, 900, 32, 8, 128), (33, 2100, 8, 2, 64), (300, 130, 4, 4, 32), (20, 5000, 32, 4, 128), (64, 1900, 16, 16, 128),
    (64, 5000, 16, 8, 128), (60, 7000, 16, 8, 64), (64, 9000, 8, 8, 32), (40, 3000, 16, 2, 128), (50, 4000, 8, 2, 32),
])
def test_batches(B, ctx, Hq, Hkv, D, dtype, bits):
    """Contexts of ragged lengths, cut between workgroups, several kv heads each."""
    from qattention_amd import prefix_attention_quantized
    lens = [max(0, ctx - (ctx * 7 * (5 * i % B)) // (10 * B)) if i % 11 else i % 3 for i in range(B)]
    cache, table, n, rows = context(lens, 16, Hkv, D, bits, 500 + B)
    Q = queries(B, Hq, D, dtype, 501)
    say("batch", B, ctx, Hq, Hkv, D, dtype, bits)
    O, L = prefix_attention_quantized(Q, cache, table, n)
    check(O, L, reference(Q, rows, [1] * B))
    again = prefix_attention_quantized(Q, cache, table, n)
    assert torch.equal(again[0], O) and torch.equal(again[1], L)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("ctx,toks,ps,Hq,Hkv,D", [
    ([500], [60], 16, 32, 8, 128),
    ([500, 0, 31], [3, 5, 7], 16, 8, 2, 64),
    ([129, 700, 64], [0, 61, 1], 32, 4, 4, 128),
    ([1, 2], [130, 2], 16, 4, 2, 32),
    ([260, 900], [15, 33], 5, 6, 2, 64),
    ([2100], [100], 16, 4, 1, 128),
    ([63, 64, 65, 127, 128, 129, 191, 193], [40] * 8, 16, 2, 1, 128),
    ([1600], [70], 16, 8, 8, 32),
    ([5000, 100], [300, 2], 16, 8, 2, 128),
])
def test_many_tokens(ctx, toks, ps, Hq, Hkv, D, dtype, bits):
    from qattention_amd import prefix_attention_quantized
    cache, table, lens, rows = context(ctx, ps, Hkv, D, bits, 400 + sum(ctx) + D)
    Q = queries(sum(toks), Hq, D, dtype, 400)
    say("many tokens", ctx, toks, ps, Hq, Hkv, D, dtype, bits)
    O, L = prefix_attention_quantized(Q, cache, table, lens, offsets(toks))
    check(O, L, reference(Q, rows, toks))
    again = prefix_attention_quantized(Q, cache, table, lens, offsets(toks).to(DEV), max_seqlen=max(toks) + 50)
    check(*again, reference(Q, rows, toks))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("many,long,ctx,Hq,Hkv,D", [(79, 600, 200, 8, 2, 128), (300, 90, 700, 16, 2, 64)])
def test_one_long_chunk_among_single_tokens(many, long, ctx, Hq, Hkv, D, bits):
    from qattention_amd import prefix_attention_quantized
    toks = [(1, 1, 0, 2)[i % 4] for i in range(many)]
    ctxs = [(0, 3, 64, 150, 20)[i % 5] for i in range(many)]
    toks[many // 2], ctxs[many // 2] = long, ctx
    cache, table, lens, rows = context(ctxs, 16, Hkv, D, bits, 71)
    Q = queries(sum(toks), Hq, D, BF16, 71)
    say("mixed", many, long, ctx, Hq, Hkv, D, bits)
    check(*prefix_attention_quantized(Q, cache, table, lens, offsets(toks)), reference(Q, rows, toks))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("n", [1, 70])
def test_missing_pages_and_lengths_past_the_table(n, bits):
    """A page outside the cache removes its keys, lengths end at the table's width; rows
    of no sequence stay as they were."""
    from qattention_amd import prefix_attention_quantized
    ps, Hkv, Hq, D = 16, 2, 8, 128
    ctx = [400, 96, 33, 700]
    cache, table, lens, rows = context(ctx, ps, Hkv, D, bits, 81)
    table[0, 3], table[0, 7], table[2] = -1, cache.K.shape[0], 2**31 - 1
    for s, gone in ((0, (3, 7)), (2, range(3))):
        keep = torch.ones(ctx[s], dtype=torch.bool, device=DEV)
        for c in gone:
            keep[c * ps:(c + 1) * ps] = False
        rows[s] = tuple(x[keep] for x in rows[s])
    lens = torch.tensor([400, 96, 33, 2**31 - 1], dtype=torch.int32, device=DEV)
    table = table[:, :44]  # 704 positions: the slots behind 700 hold no numbers
    lens[3] = 700
    Q = queries(4 * n + 3, Hq, D, FP16, 82)
    cu = torch.arange(0, 4 * n + 1, n, dtype=torch.int32, device=DEV)
    say("missing", n, bits)
    O, L = prefix_attention_quantized(Q, cache, table, lens, cu, max_seqlen=n)
    check(O[:4 * n], L[:4 * n], reference(Q, rows, [n] * 4))
    narrow = table[:, :25]
    rows[3] = tuple(x[:400] for x in rows[3])
    lens[3] = 2**31 - 1
    O, L = prefix_attention_quantized(Q, cache, narrow, lens, cu, max_seqlen=n)
    check(O[:4 * n], L[:4 * n], reference(Q, rows, [n] * 4))
    lens.fill_(-5)
    O, L = prefix_attention_quantized(Q, cache, narrow, lens, cu, max_seqlen=n)
    assert not O[:4 * n].any() and bool(torch.isinf(L[:4 * n]).all())


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("B,ctx,n,Hq,Hkv,D", [
    (24, 8000, 4, 32, 8, 64), (40, 8000, 5, 8, 4, 64), (64, 9000, 12, 4, 4, 32), (33, 7000, 3, 16, 4, 32),
    (66, 14000, 5, 16, 8, 128), (64, 14000, 13, 4, 4, 128), (24, 8000, 16, 6, 6, 64),
])
def test_short_drafts_over_long_contexts(B, ctx, n, Hq, Hkv, D, dtype, bits):
    """9 to 16 rows: heads in tiles of their own.  Most sequences read the same pages, to
    lengths of their own; the first one's hold a block without a number in K and in V."""
    from qattention_amd import prefix_attention_quantized
    own = 777
    cache, table, _, rows = context([own, ctx, ctx - 1000], 16, Hkv, D, bits, 600 + B + D)
    table = table[torch.tensor([0] + [1 + s % 2 for s in range(1, B)], device=DEV)].contiguous()
    lens = [own] + [ctx - 1000 - (37 * s * s) % (ctx // 2) if s % 9 else s % 4 for s in range(1, B)]
    toks = [n] + [n - s % 3 if s % 7 else 0 for s in range(1, B)]
    cache.K_scale[int(table[0, 100 // 16]), 100 % 16, 1, 0] = 255
    cache.V_scale[int(table[0, 200 // 16]), 200 % 16, 0, 0] = 255
    Q = queries(sum(toks), Hq, D, dtype, 601)
    say("drafts", B, ctx, n, Hq, Hkv, D, dtype, bits)
    n_ctx = torch.tensor(lens, dtype=torch.int32, device=DEV)
    O, L = prefix_attention_quantized(Q, cache, table, n_ctx, offsets(toks))
    kv = [rows[0]] + [tuple(x[:m] for x in rows[1 + s % 2]) for s, m in zip(range(1, B), lens[1:])]
    o, lse, to, tl = reference(Q, kv, toks)
    g = Hq // Hkv
    bad = torch.zeros_like(O, dtype=torch.bool)
    bad[:n, g:2 * g] = True     # (K of head 1)
    bad[:n, :g, :32] = True     # (V of head 0)
    assert torch.equal(torch.isnan(O), bad)
    bad_lse = torch.zeros_like(L, dtype=torch.bool)
    bad_lse[:n, g:2 * g] = True
    assert torch.equal(torch.isnan(L), bad_lse)
    some = ~bad[..., 0]
    check(O.masked_fill(bad, 0), L.masked_fill(bad_lse, 0),
          (o.masked_fill(bad, 0), lse.masked_fill(bad_lse, 0), to.masked_fill(bad, 0), tl.masked_fill(bad_lse, 0)))
    again = prefix_attention_quantized(Q, cache, table, n_ctx, offsets(toks))
    assert torch.equal(again[0][some], O[some]) and torch.equal(again[1][some], L[some])


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("n,ctx", [(1, [200, 300]), (5, [200, 300]), (50, [200, 300]), (1, [1500, 2900]),
                                   (1, [130] + 39 * [6000])])
def test_no_numbers(n, ctx, bits):
    """A block without a number makes the rows that attend it NaN, of its own head and
    sequence alone."""
    from qattention_amd import prefix_attention_quantized
    B = len(ctx)
    for name, part in (("K_scale", 0), ("V_scale", 1)):
        cache, table, lens, rows = context(ctx, 16, 2, 128, bits, 91)
        getattr(cache, name)[int(table[0, 100 // 16]), 100 % 16, 1, 2] = 255
        Q = queries(B * n, 8, 128, FP16, 92)
        say("no numbers", n, ctx[:2], bits, name)
        cu = torch.arange(0, B * n + 1, n, dtype=torch.int32, device=DEV)
        O, L = prefix_attention_quantized(Q, cache, table, lens, cu, max_seqlen=n)
        o, lse, to, tl = reference(Q, rows, [n] * B)
        bad = torch.zeros_like(O, dtype=torch.bool)
        if part == 0:
            bad[:n, 4:] = True
        else:
            bad[:n, 4:, 64:96] = True
        assert torch.equal(torch.isnan(O), bad)
        assert bool(((O.double() - o).abs() <= to)[~bad].all())
        assert torch.equal(torch.isnan(L), bad[..., 0] if part == 0 else torch.zeros_like(L, dtype=torch.bool))


@pytest.mark.parametrize("bits", [4, 8])
def test_steep_scores_and_scales(bits):
    """Scales far apart in one context, scores of +-hundreds."""
    from qattention_amd import prefix_attention_quantized
    for dtype, sigma in ((FP16, 8.0), (BF16, 40.0), (FP16, 2.0 ** -9)):
        for toks in ([1, 1], [50, 3]):
            cache, table, lens, rows = context([777, 1300], 16, 2, 64, bits, 95, dtype=dtype, sigma=sigma)
            Q = queries(sum(toks), 8, 64, dtype, 96, 2.0)
            say("steep", dtype, sigma, toks, bits)
            check(*prefix_attention_quantized(Q, cache, table, lens, offsets(toks)), reference(Q, rows, toks))


def test_layouts():
    """Layer slices with the layers in each page, gaps between heads, odd query strides."""
    import qattention_amd as qa
    cache, table, lens, rows = context([300, 500], 16, 3, 128, 4, 97)
    wide = [torch.full((t.shape[0], 2, 16, 4, 2 * t.shape[-1]), 255, dtype=torch.uint8, device=DEV) for t in cache]
    views = qa.QuantizedKV(*(t[:, 1, :, 1:, :t.shape[-1] // 2] for t in wide))
    for a, b in zip(views, cache):
        a.copy_(b)
    for toks in ([1, 1], [40, 2]):
        Q = queries(sum(toks), 24, 128, BF16, 98)[:, ::2]
        say("layouts", toks)
        O, L = qa.prefix_attention_quantized(Q, views, table, lens, offsets(toks))
        check(O, L, reference(Q, rows, toks))
        odd = queries(sum(toks), 12, 130, BF16, 99)[..., 1:129]
        check(*qa.prefix_attention_quantized(odd, views, table, lens, offsets(toks)), reference(odd, rows, toks))


def test_offsets_past_32_bits():
    """Rows more than 4 GiB from the cache's start."""
    from qattention_amd import QuantizedKV, prefix_attention_quantized
    ps, Hkv, D, pages = 64, 2, 128, 4
    near, table, lens, rows = context([200], ps, Hkv, D, 4, 101, extra=0)
    room = torch.empty((5 << 30) + (1 << 20), dtype=torch.uint8, device=DEV)
    step = 5 * 2**30 // 4 // 16 * 16
    far = QuantizedKV(*(room.as_strided((pages, ps, Hkv, t.shape[-1]), (step, Hkv * t.shape[-1], t.shape[-1], 1),
                                        i << 16) for i, t in enumerate(near)))
    for a, b in zip(far, near):
        a.copy_(b)
    for toks in ([1], [40]):
        Q = queries(sum(toks), 8, D, FP16, 102)
        say("far", toks)
        check(*prefix_attention_quantized(Q, far, table, lens, offsets(toks)), reference(Q, rows, toks))
