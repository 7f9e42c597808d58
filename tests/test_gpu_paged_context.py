"""prefix_attention_paged against dense attention in 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

from attn64 import attend64, check, offsets

pytestmark = pytest.mark.gpu
DEV = "cuda"


def say(*a):
    print(*a, flush=True)


def paged(ctx, ps, Hkv, D, dtype, seed, extra=3, behind=math.nan):
    """Caches in shuffled pages with `behind` in every slot that no context fills,
    and the contexts' K/V rows in order."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    pages = [-(-n // ps) for n in ctx]
    total, cols = sum(pages) + extra, max(pages + [1]) + 1
    Kc, Vc = (torch.full((total, ps, Hkv, D), behind, dtype=dtype, device=DEV) for _ in range(2))
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.full((len(ctx), cols), -1, dtype=torch.int32)
    rows, first = [], 0
    for i, n in enumerate(ctx):
        k, v = (torch.empty(n, Hkv, D, dtype=dtype, device=DEV).normal_(0, 1, generator=g) for _ in range(2))
        rows.append((k, v))
        table[i, :pages[i]] = order[first:first + pages[i]]
        first += pages[i]
        if n:
            at = table[i].long().to(DEV)[torch.arange(n, device=DEV) // ps], torch.arange(n, device=DEV) % ps
            Kc[at], Vc[at] = k, v
    return Kc, Vc, table.to(DEV), torch.tensor(ctx, dtype=torch.int32, device=DEV), rows


def queries(T, Hq, D, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed + 1)
    return torch.empty(T, Hq, D, dtype=dtype, device=DEV).normal_(0, 1, generator=g)


def reference(Q, rows, lens):
    parts, a = [], 0
    for n, (k, v) in zip(lens, rows):
        parts.append(attend64(Q[a:a + n], k, v, torch.ones(n, k.shape[0], dtype=torch.bool, device=DEV)))
        a += n
    return [torch.cat(x) for x in zip(*parts)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("ctx,ps,Hq,Hkv,D", [
    ([1], 16, 4, 4, 64),
    ([0], 16, 4, 4, 64),
    ([0, 1, 15, 16, 17, 31, 32, 33], 16, 8, 2, 128),
    ([127, 128, 129, 0, 255, 256, 257], 16, 8, 2, 64),
    ([5, 0, 0, 200], 1, 4, 1, 32),
    ([300, 40], 7, 6, 2, 128),
    ([1000, 3], 64, 32, 8, 128),
    ([4000], 16, 32, 4, 128),
    ([700, 650], 300, 16, 1, 64),
    ([90, 2000], 16, 24, 1, 128),   # 24 rows: two row blocks
    ([333, 1], 16, 40, 1, 64),      # 40 rows: four
    ([150, 20], 16, 100, 1, 128),   # 100 rows: two tiles
])
def test_one_token(ctx, ps, Hq, Hkv, D, dtype):
    from qattention_amd import prefix_attention_paged
    Kc, Vc, table, lens, rows = paged(ctx, ps, Hkv, D, dtype, 300 + sum(ctx) + D)
    Q = queries(len(ctx), Hq, D, dtype, 300)
    say("one token", ctx, ps, Hq, Hkv, D, dtype)
    O, L = prefix_attention_paged(Q, Kc, Vc, table, lens)
    check(O, L, reference(Q, rows, [1] * len(ctx)))
    assert torch.equal(prefix_attention_paged(Q, Kc, Vc, table.cpu(), lens.cpu(), return_lse=False), O)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("ctx,toks,ps,Hq,Hkv,D", [
    ([500], [60], 16, 32, 8, 128),
    ([500, 0, 31], [3, 5, 7], 16, 8, 2, 64),
    ([129, 700, 64], [0, 61, 1], 32, 4, 4, 128),
    ([1, 2], [130, 2], 16, 4, 2, 32),
    ([260, 900], [15, 33], 5, 6, 2, 64),
    ([2100], [100], 16, 4, 1, 128),
])
def test_many_tokens(ctx, toks, ps, Hq, Hkv, D, dtype):
    from qattention_amd import prefix_attention_paged
    Kc, Vc, table, lens, rows = paged(ctx, ps, Hkv, D, dtype, 400 + sum(ctx) + D)
    Q = queries(sum(toks), Hq, D, dtype, 400)
    say("many tokens", ctx, toks, ps, Hq, Hkv, D, dtype)
    O, L = prefix_attention_paged(Q, Kc, Vc, table, lens, offsets(toks))
    check(O, L, reference(Q, rows, toks))
    again = prefix_attention_paged(Q, Kc, Vc, table, lens, offsets(toks).to(DEV), max_seqlen=max(toks) + 50)
    check(*again, reference(Q, rows, toks))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("many,long,ctx,Hq,Hkv,D", [
    (79, 600, 200, 8, 2, 128),
    (300, 90, 700, 16, 2, 64),
    (1100, 8, 300, 8, 8, 64),   # few rows
    (900, 7, 0, 16, 8, 32),     # a long one without a context
])
def test_one_long_chunk_among_single_tokens(many, long, ctx, Hq, Hkv, D, dtype):
    from qattention_amd import prefix_attention_paged
    toks = [(1, 1, 0, 2)[i % 4] for i in range(many)]
    ctxs = [(0, 3, 64, 150, 20)[i % 5] for i in range(many)]
    toks[many // 2], ctxs[many // 2] = long, ctx
    Kc, Vc, table, lens, rows = paged(ctxs, 16, Hkv, D, dtype, 71)
    Q = queries(sum(toks), Hq, D, dtype, 71)
    say("mixed", many, long, ctx, Hq, Hkv, D, dtype)
    O, L = prefix_attention_paged(Q, Kc, Vc, table, lens, offsets(toks))
    check(O, L, reference(Q, rows, toks))


@pytest.mark.parametrize("pages", [0, 3])
def test_rows_without_contexts(pages):
    """Chunks and single tokens without a context, with and without a cache."""
    from qattention_amd import prefix_attention_paged
    for toks in ([1] * 5, [100, 1, 0, 3], [40] * 3, [1] * 300 + [500], [6] * 70):
        Q = queries(sum(toks), 8, 64, torch.float16, 73)
        cache = torch.full((pages, 16, 2, 64), math.nan, dtype=torch.float16, device=DEV)
        table = torch.zeros(len(toks), 60, dtype=torch.int32, device=DEV)
        lens = torch.zeros(len(toks), dtype=torch.int32, device=DEV)
        say("no contexts", pages, len(toks))
        O, L = prefix_attention_paged(Q, cache, torch.full_like(cache, math.nan), table, lens, offsets(toks))
        assert not O.any() and (L == -math.inf).all()


def test_large_batch():
    """More sequences than a workgroup has threads, lengths from zero on."""
    from qattention_amd import prefix_attention_paged
    ctx = [(37 * i) % 90 if i % 5 else 0 for i in range(700)]
    Kc, Vc, table, lens, rows = paged(ctx, 16, 2, 64, torch.float16, 31)
    Q = queries(700, 4, 64, torch.float16, 31)
    say("large batch")
    O, L = prefix_attention_paged(Q, Kc, Vc, table, lens)
    check(O, L, reference(Q, rows, [1] * 700))


def test_missing_pages_and_lengths_out_of_range():
    """Keys of pages that do not exist are left out; lengths are taken into what
    the table has columns for."""
    from qattention_amd import prefix_attention_paged
    ctx, ps = [200, 64, 90], 16
    Kc, Vc, table, lens, rows = paged(ctx, ps, 2, 128, torch.bfloat16, 37, behind=0.5)
    Q = queries(3, 8, 128, torch.bfloat16, 37)
    table[0, 3], table[0, 4], table[0, 12] = -1, Kc.shape[0], 2 ** 30
    table[1, :] = -7
    say("missing pages")
    O, L = prefix_attention_paged(Q, Kc, Vc, table, lens)
    masks = [torch.ones(1, n, dtype=torch.bool, device=DEV) for n in ctx]
    masks[0][:, 48:80], masks[0][:, 192:], masks[1][:] = False, False, False
    ref = [torch.cat(x) for x in zip(*[attend64(Q[i:i + 1], *rows[i], masks[i]) for i in range(3)])]
    check(O, L, ref)
    assert bool((O[1] == 0).all())
    # lengths past the table, and negative ones
    table = table[2:, :6].contiguous()
    say("lengths out of range")
    for n in (96, 97, 10 ** 6, 2 ** 31 - 1):
        got = prefix_attention_paged(Q[2:], Kc, Vc, table, torch.tensor([n], dtype=torch.int32))
        full = Kc[table[0].long()].flatten(0, 1), Vc[table[0].long()].flatten(0, 1)
        check(*got, attend64(Q[2:], *full, torch.ones(1, 96, dtype=torch.bool, device=DEV)))
    O, L = prefix_attention_paged(Q[2:], Kc, Vc, table, torch.tensor([-5], dtype=torch.int32))
    assert bool((O == 0).all()) and bool((L == -math.inf).all())


def test_nothing_to_read():
    from qattention_amd import prefix_attention_paged
    Q = queries(3, 4, 64, torch.float16, 41)
    none = torch.empty(0, 16, 2, 64, dtype=torch.float16, device=DEV)
    cache = torch.zeros(2, 16, 2, 64, dtype=torch.float16, device=DEV)
    lens = torch.tensor([4, 0, 9], dtype=torch.int32, device=DEV)
    say("no pages")
    for c, cols in ((none, 2), (cache, 0)):
        O, L = prefix_attention_paged(Q, c, c.clone(), torch.zeros(3, cols, dtype=torch.int32, device=DEV), lens)
        assert bool((O == 0).all()) and bool((L == -math.inf).all())
    O, L = prefix_attention_paged(Q[:0], cache, cache.clone(), torch.zeros(0, 2, dtype=torch.int32), lens[:0])
    assert O.shape == (0, 4, 64) and L.shape == (0, 4)


@pytest.mark.parametrize("toks", [None, [40, 2]])
def test_nonfinite_rows(toks):
    """NaN in one key's row reaches the heads that attend it and no other."""
    from qattention_amd import prefix_attention_paged
    ctx, ps, Hkv = [300, 45], 16, 4
    Kc, Vc, table, lens, rows = paged(ctx, ps, Hkv, 64, torch.float16, 43)
    Q = queries(2 if toks is None else sum(toks), 8, 64, torch.float16, 43)
    cu = None if toks is None else offsets(toks)
    n0 = 1 if toks is None else toks[0]
    O, L = prefix_attention_paged(Q, Kc, Vc, table, lens, cu)
    for pos in (0, 170, 299):
        for bad in (math.nan, math.inf):
            say("nonfinite", toks, pos, bad)
            V2 = Vc.clone()
            V2[table[0, pos // ps].long(), pos % ps, 1, 3] = bad
            O2, L2 = prefix_attention_paged(Q, Kc, V2, table, lens, cu)
            hit = torch.zeros_like(O, dtype=torch.bool)
            hit[:n0, 2:4, 3] = True
            assert torch.equal(~torch.isfinite(O2), hit) and torch.equal(O2[~hit], O[~hit]) and torch.equal(L2, L)
        K2 = Kc.clone()
        K2[table[0, pos // ps].long(), pos % ps, 1, 3] = math.nan
        O2, L2 = prefix_attention_paged(Q, K2, Vc, table, lens, cu)
        hit = torch.zeros_like(O, dtype=torch.bool)
        hit[:n0, 2:4] = True
        assert torch.equal(torch.isnan(O2), hit) and torch.equal(O2[~hit], O[~hit])
        assert torch.equal(torch.isnan(L2), hit[:, :, 0])


def test_strided_caches():
    """Heads outside the slots, one layer of an all-layer cache, K and V interleaved."""
    from qattention_amd import prefix_attention_paged
    ctx = [222, 18]
    Kc, Vc, table, lens, rows = paged(ctx, 16, 2, 128, torch.bfloat16, 47)
    Q = queries(2, 8, 128, torch.bfloat16, 47)
    want = prefix_attention_paged(Q, Kc, Vc, table, lens)
    hnd = [c.transpose(1, 2).contiguous().transpose(1, 2) for c in (Kc, Vc)]
    both = torch.stack([Kc, Vc], 1)
    layers = torch.stack([torch.zeros_like(Kc), Kc, Vc])
    unaligned = [torch.empty(*c.shape[:-1], 129, dtype=c.dtype, device=DEV)[..., 1:].copy_(c) for c in (Kc, Vc)]
    for i, (k, v) in enumerate((hnd, (both[:, 0], both[:, 1]), (layers[1], layers[2]), unaligned)):
        say("cache strides", i)
        O, L = prefix_attention_paged(Q, k, v, table, lens)
        assert torch.equal(O, want[0]) and torch.equal(L, want[1])
    q2 = torch.stack([Q, Q], 2)[:, :, 1]
    O, L = prefix_attention_paged(q2, Kc, Vc, table, lens)
    assert torch.equal(O, want[0]) and torch.equal(L, want[1])


def test_offsets_past_32_bits():
    """Pages past 2^31 elements of the cache."""
    from qattention_amd import prefix_attention_paged
    pages, ps, Hkv, D = 140000, 16, 8, 128
    Kc, Vc = (torch.empty(pages, ps, Hkv, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    table = torch.tensor([[pages - 1, 0, 135000, pages - 2, 131073]], dtype=torch.int32, device=DEV)
    for c in (Kc, Vc):
        c[table[0].long()] = torch.randn(5, ps, Hkv, D, device=DEV).bfloat16()
    Q = queries(1, 32, D, torch.bfloat16, 53)
    say("offsets")
    O, L = prefix_attention_paged(Q, Kc, Vc, table, torch.tensor([77], dtype=torch.int32))
    k, v = (c[table[0].long()].flatten(0, 1)[:77] for c in (Kc, Vc))
    check(O, L, attend64(Q, k, v, torch.ones(1, 77, dtype=torch.bool, device=DEV)))


def test_long_context():
    from qattention_amd import prefix_attention_paged
    Kc, Vc, table, lens, rows = paged([130001], 64, 1, 128, torch.float16, 59)
    Q = queries(1, 8, 128, torch.float16, 59)
    say("long context")
    O, L = prefix_attention_paged(Q, Kc, Vc, table, lens)
    check(O, L, reference(Q, rows, [1]))


@pytest.mark.parametrize("ctx,n", [(300, 1), (3000, 1), (3000, 60)])
def test_largest_values(ctx, n):
    from qattention_amd import prefix_attention_paged
    Kc, Vc, table, lens, rows = paged([ctx], 16, 2, 128, torch.float16, 73)
    Vc.copy_(torch.where(torch.isnan(Vc), Vc, torch.full_like(Vc, 65504.0)))
    Q = queries(n, 8, 128, torch.float16, 73)
    say("largest", ctx, n)
    O = prefix_attention_paged(Q, Kc, Vc, table, lens, None if n == 1 else offsets([n]), return_lse=False)
    assert bool((O == 65504.0).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_steep_scores(dtype):
    """Scores that rise by hundreds along the context, one token and many."""
    from qattention_amd import prefix_attention_paged
    n, D = 1200, 64
    Kc, Vc, table, lens, rows = paged([n], 16, 1, D, dtype, 79)
    steps = torch.tensor([0, 30, 120, 400, 500, 100, 0], dtype=dtype, device=DEV)
    at = table[0].long()[torch.arange(n, device=DEV) // 16], torch.arange(n, device=DEV) % 16
    rows[0][0][:, 0, 0] = steps[torch.arange(n, device=DEV) * 7 // n]
    Kc[at] = rows[0][0]
    for toks in (1, 50):
        Q = queries(toks, 2, D, dtype, 79)
        Q[:, :, 0] = 8.0
        say("steep", dtype, toks)
        O, L = prefix_attention_paged(Q, Kc, Vc, table, lens, None if toks == 1 else offsets([toks]))
        check(O, L, reference(Q, rows, [toks]))


def test_rows_of_no_sequence_stay():
    from qattention_amd import _lib, prefix_attention_paged
    ctx, T, Hq, Hkv, D = [50, 60, 70], 40, 4, 2, 64
    Kc, Vc, table, lens, rows = paged(ctx, 16, Hkv, D, torch.float16, 61)
    Q = queries(T, Hq, D, torch.float16, 61)
    cu = torch.tensor([2, 12, 8, 30], dtype=torch.int32, device=DEV)  # sequence 1's offsets are bad
    O, L = torch.full_like(Q, 7.0), torch.full((T, Hq), 7.0, device=DEV)
    lib = _lib.lib()
    ms = 15
    nb = lib.qattn_prefix_paged_workspace_bytes(3, ms, T, Hq, Hkv, D, table.shape[1], 16)
    ws = torch.empty(nb, dtype=torch.uint8, device=DEV)
    say("no sequence")
    rc = lib.qattn_prefix_paged_fwd(
        Q.data_ptr(), _lib.i64arr(Q.stride()), Kc.data_ptr(), _lib.i64arr(Kc.stride()), Vc.data_ptr(),
        _lib.i64arr(Vc.stride()), table.data_ptr(), table.shape[1], Kc.shape[0], 16, lens.data_ptr(), O.data_ptr(),
        _lib.i64arr(O.stride()), L.data_ptr(), _lib.i64arr(L.stride()), cu.data_ptr(), 3, ms, T, Hq, Hkv, D,
        1 / math.sqrt(D), 0, ws.data_ptr(), nb, torch.cuda.current_stream().cuda_stream)
    _lib.check(rc, "qattn_prefix_paged_fwd")
    done = torch.zeros(T, dtype=torch.bool, device=DEV)
    done[2:12], done[8:23] = True, True
    assert bool((O[~done] == 7).all()) and bool((L[~done] == 7).all())
    check(O[12:23], L[12:23], reference(Q[12:23], rows[2:], [11]))


def test_streams_and_graphs():
    """Two captured calls and eager ones in turn, contexts changing on the device."""
    from qattention_amd import prefix_attention_paged
    ctx = [900, 10, 333]
    Kc, Vc, table, lens, rows = paged(ctx, 16, 2, 128, torch.float16, 67, behind=0.25)
    Q, Q2 = queries(3, 8, 128, torch.float16, 67), queries(9, 8, 128, torch.float16, 68)
    cu = offsets([4, 2, 3]).to(DEV)
    one = lambda: prefix_attention_paged(Q, Kc, Vc, table, lens)  # noqa: E731
    many = lambda: prefix_attention_paged(Q2, Kc, Vc, table, lens, cu, 4)  # noqa: E731
    one(), many()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for f in (one, many):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(f())
        graphs.append(graph)
    side = torch.cuda.Stream()
    for i in range(5):
        say("replay", i)
        lens.copy_(torch.tensor([900 - 200 * i, 10 * i, 333 - 70 * i], dtype=torch.int32))
        graphs[i % 2].replay()
        graphs[1 - i % 2].replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            a = one()
        b = many()
        torch.cuda.current_stream().wait_stream(side)
        for got, want in ((outs[0], a), (outs[1], b)):
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_same_bits_every_time():
    from qattention_amd import prefix_attention_paged
    Kc, Vc, table, lens, rows = paged([5000, 900, 3000, 77], 16, 8, 128, torch.bfloat16, 71)
    Q = queries(4, 32, 128, torch.bfloat16, 71)
    O, L = prefix_attention_paged(Q, Kc, Vc, table, lens)
    for _ in range(5):
        O2, L2 = prefix_attention_paged(Q, Kc, Vc, table, lens)
        assert torch.equal(O, O2) and torch.equal(L, L2)
