"""append_paged_kv, compact_paged_kv and copy_kv_pages against torch indexing: moved
rows bit by bit, every other row as it was."""
from __future__ import annotations

import pytest
import torch

from attn64 import offsets

pytestmark = pytest.mark.gpu
DEV = "cuda"


def say(*a):
    print(*a, flush=True)


def cache(pages, ps, Hkv, D, dtype, seed, layers=None):
    g = torch.Generator(device=DEV).manual_seed(seed)
    shape = (pages, ps, Hkv, D) if layers is None else (layers, pages, ps, Hkv, D)
    return [torch.empty(shape, dtype=dtype, device=DEV).normal_(0, 1, generator=g) for _ in range(2)]


def tables(B, cols, pages, seed):
    return torch.randperm(pages, generator=torch.Generator().manual_seed(seed))[:B * cols].view(B, cols).to(torch.int32)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("ctx,new,ps,Hkv,D", [
    ([0], [1], 16, 8, 128),
    ([5, 16, 0, 31], None, 16, 8, 128),
    ([5, 16, 0, 31], [3, 0, 40, 1], 16, 2, 64),
    ([1, 2, 3], [7, 9, 100], 1, 1, 32),
    ([100, 0], [300, 5], 7, 32, 128),
    ([13], [2000], 64, 8, 64),
    ([3, 1], [5, 64], 16, 3, 32),
    ([4, 0, 9, 17] * 20, [1] * 41 + [230] + [0, 2, 1] * 12 + [1, 1], 16, 8, 128),  # one long among many
    ([4, 0, 9, 17] * 50, [1] * 101 + [900] + [3, 0] * 49, 5, 1, 32),
])
def test_append(ctx, new, ps, Hkv, D, dtype):
    from qattention_amd import append_paged_kv
    B, n = len(ctx), [1] * len(ctx) if new is None else new
    cols = max(-(-(c + x) // ps) for c, x in zip(ctx, n))
    Kc, Vc = cache(B * cols + 4, ps, Hkv, D, dtype, 1)
    table = tables(B, cols, B * cols + 4, 2)
    K, V = cache(1, sum(n), Hkv, D, dtype, 3)
    K, V = K[0], V[0]
    want = [Kc.clone(), Vc.clone()]
    row = 0
    for s in range(B):
        for i in range(n[s]):
            pos = ctx[s] + i
            for w, x in zip(want, (K, V)):
                w[int(table[s, pos // ps]), pos % ps] = x[row]
            row += 1
    lens = torch.tensor(ctx, dtype=torch.int32, device=DEV)
    say("append", ctx, new, ps, Hkv, D, dtype)
    got = append_paged_kv(K, V, Kc, Vc, table.to(DEV), lens, None if new is None else offsets(new))
    assert got.dtype == torch.int32 and got.tolist() == [c + x for c, x in zip(ctx, n)] and lens.tolist() == ctx
    assert torch.equal(Kc, want[0]) and torch.equal(Vc, want[1])


def test_append_what_has_no_place():
    """Past the table, missing pages, negative lengths, bad offsets, max_seqlen."""
    from qattention_amd import append_paged_kv
    ps, Hkv, D = 4, 2, 64
    Kc, Vc = cache(12, ps, Hkv, D, torch.float16, 5)
    table = torch.tensor([[0, 1], [2, 99], [-1, 5], [6, 7], [8, 9], [10, 11]], dtype=torch.int32)
    ctx = torch.tensor([6, 3, 2, -1, 0, 9], dtype=torch.int32)
    cu = torch.tensor([0, 5, 10, 15, 17, 16, 22], dtype=torch.int32)  # sequence 4's offsets are bad
    K, V = (x[0] for x in cache(1, 22, Hkv, D, torch.float16, 6))
    want = [Kc.clone(), Vc.clone()]
    for w, x in zip(want, (K, V)):
        w[1, 2], w[1, 3] = x[0], x[1]            # sequence 0: two of five rows have a place
        w[2, 3] = x[5]                           # sequence 1: its second page is missing
        w[5, 0], w[5, 1] = x[12], x[13]          # sequence 2: its first page is missing, four rows at most
    say("no place")
    got = append_paged_kv(K, V, Kc, Vc, table, ctx, cu, max_seqlen=4)
    assert got.tolist() == [8, 7, 6, -1, 0, 9]
    assert torch.equal(Kc, want[0]) and torch.equal(Vc, want[1])


def test_append_what_has_no_place_among_many():
    """The same for many sequences, most far shorter than the longest."""
    from qattention_amd import append_paged_kv
    ps, Hkv, D, B = 4, 2, 64, 150
    Kc, Vc = cache(2 * B, ps, Hkv, D, torch.float16, 7)
    new = [1] * 70 + [600] + [1] * 79
    table = torch.arange(2 * B, dtype=torch.int32).view(B, 2)
    ctx = torch.tensor([i % 9 for i in range(B)], dtype=torch.int32)
    ctx[5], table[6, 1], table[7, 0], ctx[70] = -3, 2 * B, -1, 2
    cu = offsets(new).cpu()
    cu[101], cu[-1] = cu[100] - 1, sum(new) + 1  # sequence 100 and the last one are none; 101 has three rows
    K, V = (x[0] for x in cache(1, sum(new), Hkv, D, torch.float16, 8))
    want, after = [Kc.clone(), Vc.clone()], ctx.clone()
    for s in range(B):
        a, b = int(cu[s]), int(cu[s + 1])
        if b < a or b > sum(new) or ctx[s] < 0:
            continue
        for i in range(min(b - a, 500)):
            pos = int(ctx[s]) + i
            if pos < 2 * ps:
                after[s] += 1
                page = int(table[s, pos // ps])
                if 0 <= page < 2 * B:
                    for w, x in zip(want, (K, V)):
                        w[page, pos % ps] = x[a + i]
    # (row 99 of the single ones belongs to two sequences now: either may have it)
    say("no place among many")
    got = append_paged_kv(K, V, Kc, Vc, table, ctx, cu, max_seqlen=500)
    assert torch.equal(got.cpu(), after)
    skip = [int(table[s, j]) for s in (99, 101) for j in (0, 1)]
    for w, x in zip(want, (Kc, Vc)):
        w[skip], x[skip] = 0, 0
        assert torch.equal(x, w)


def test_append_strided():
    from qattention_amd import append_paged_kv
    ps, Hkv, D = 16, 2, 64
    Kc, Vc = cache(6, ps, Hkv, D, torch.bfloat16, 7)
    table, lens = tables(2, 3, 6, 8).to(DEV), torch.tensor([10, 0], dtype=torch.int32, device=DEV)
    K, V = (x[0] for x in cache(1, 30, Hkv, D, torch.bfloat16, 9))
    cu = offsets([20, 10])
    want = Kc.clone(), Vc.clone()
    append_paged_kv(K, V, *want, table, lens, cu)
    fused = torch.cat([K, V], 1)
    odd = [torch.empty(30, Hkv, D + 1, dtype=K.dtype, device=DEV)[..., 1:].copy_(x) for x in (K, V)]
    hnd = [torch.empty(6, Hkv, ps, D, dtype=K.dtype, device=DEV) for _ in range(2)]
    for i, (k, v) in enumerate(((fused[:, :Hkv], fused[:, Hkv:]), odd)):
        say("append strides", i)
        views = [h.copy_(c.transpose(1, 2)).transpose(1, 2) for h, c in zip(hnd, (Kc, Vc))]
        append_paged_kv(k, v, *views, table, lens, cu)
        assert torch.equal(views[0], want[0]) and torch.equal(views[1], want[1])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layers,ctx,paths,ps,Hkv,D", [
    (None, [10], [[0, 2, 5]], 16, 8, 128),
    (3, [10, 31, 0], [[0, 1, 2], [0, 3, 4, 9, 20], []], 16, 2, 64),
    (2, [7, 100], [[4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 14, 30, 31], [0]], 8, 32, 128),  # rows move onto rows read later
    (1, [3], [list(range(1, 60))], 1, 1, 32),
    (32, [50, 60], [[0, 4, 11, 40], [2]], 16, 4, 128),
])
def test_compact(layers, ctx, paths, ps, Hkv, D, dtype):
    from qattention_amd import compact_paged_kv
    B, P = len(ctx), max(len(p) for p in paths) + 1
    cols = max(-(-(c + 64) // ps) for c in ctx)
    Kc, Vc = cache(B * cols + 2, ps, Hkv, D, dtype, 11, layers)
    table = tables(B, cols, B * cols + 2, 12)
    acc = torch.full((B, P), -1, dtype=torch.int32)
    for s, p in enumerate(paths):
        acc[s, :len(p)] = torch.tensor(p, dtype=torch.int32)
    want = []
    for c in (Kc, Vc):
        old, w = (c.clone() if layers else c.clone()[None] for _ in range(2))
        for s, p in enumerate(paths):
            for j, node in enumerate(p):
                a, b = ctx[s] + node, ctx[s] + j
                w[:, int(table[s, b // ps]), b % ps] = old[:, int(table[s, a // ps]), a % ps]
        want.append(w if layers else w[0])
    say("compact", layers, ctx, ps, Hkv, D, dtype)
    got = compact_paged_kv(Kc, Vc, table.to(DEV), torch.tensor(ctx, dtype=torch.int32, device=DEV), acc.to(DEV))
    assert got.tolist() == [c + len(p) for c, p in zip(ctx, paths)]
    assert torch.equal(Kc, want[0]) and torch.equal(Vc, want[1])


def test_compact_ends_of_paths():
    """Entries that do not rise, lie past the table or are negative end a path;
    rows of missing pages stay; negative lengths are passed over."""
    from qattention_amd import compact_paged_kv
    ps, Hkv, D = 4, 2, 64
    Kc, Vc = cache(16, ps, Hkv, D, torch.float16, 13)
    table = torch.arange(15, dtype=torch.int32).view(5, 3)
    table[4, 1] = 16
    ctx = torch.tensor([1, 2, 3, -2, 1], dtype=torch.int32)
    acc = torch.tensor([[1, 3, 3, 5], [2, 9, 10, 11], [-1, 0, 1, 2], [0, 1, 2, 3], [2, 4, 7, 8]], dtype=torch.int32)
    want = [Kc.clone(), Vc.clone()]
    for w, old in zip(want, (Kc, Vc)):
        w[0, 1], w[0, 2] = old[0, 2], old[1, 0]  # sequence 0: rows 1 + (1, 3)
        w[3, 2], w[3, 3] = old[4, 0], old[5, 3]  # sequence 1: rows 2 + (2, 9); 12 is past the table
        # sequence 4: row 1 + 2 to 1; rows 5 and 8 sit on the missing page and behind it, row 9 goes to it
        w[12, 1], w[12, 3] = old[12, 3], old[14, 0]
    say("ends of paths")
    got = compact_paged_kv(Kc, Vc, table, ctx, acc)
    assert got.tolist() == [3, 4, 3, -2, 5]
    assert torch.equal(Kc, want[0]) and torch.equal(Vc, want[1])


@pytest.mark.parametrize("layers,n,ps,Hkv,D", [(None, 1, 16, 8, 128), (4, 5, 16, 2, 64), (2, 9, 1, 1, 32),
                                               (3, 3, 100, 32, 128), (1, 2, 7, 3, 64)])
def test_copy(layers, n, ps, Hkv, D):
    from qattention_amd import copy_kv_pages
    Kc, Vc = cache(3 * n + 2, ps, Hkv, D, torch.bfloat16, 17, layers)
    order = torch.randperm(3 * n + 2, generator=torch.Generator().manual_seed(18)).tolist()
    src, dst = [order[i // 2] for i in range(n)], order[n:2 * n]  # a source may serve twice
    want = [Kc.clone(), Vc.clone()]
    for w, c in zip(want, (Kc, Vc)):
        for a, b in zip(src, dst):
            w[..., b, :, :, :] = c[..., a, :, :, :]
    say("copy", layers, n, ps, Hkv, D)
    k, v = Kc.clone(), Vc.clone()
    copy_kv_pages(k, v, src, dst)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    # lists on the GPU; pairs outside the cache and onto themselves change nothing
    more = [[-1, 0, len(order), order[0]], [0, -1, 1, order[0]]]
    src, dst = (torch.tensor(x + m, dtype=torch.int32, device=DEV) for x, m in zip((src, dst), more))
    copy_kv_pages(Kc, Vc, src, dst)
    assert torch.equal(Kc, want[0]) and torch.equal(Vc, want[1])


def test_rows_past_32_bits():
    from qattention_amd import append_paged_kv, compact_paged_kv, copy_kv_pages
    pages, ps, Hkv, D = 140000, 16, 8, 128
    Kc, Vc = (torch.empty(pages, ps, Hkv, D, dtype=torch.float16, device=DEV) for _ in range(2))
    table = torch.tensor([[pages - 1, pages - 3]], dtype=torch.int32, device=DEV)
    K, V = (x[0] for x in cache(1, 20, Hkv, D, torch.float16, 19))
    lens = torch.tensor([4], dtype=torch.int32, device=DEV)
    say("past 32 bits")
    append_paged_kv(K, V, Kc, Vc, table, lens, offsets([20]))
    assert torch.equal(Kc[pages - 1, 4:], K[:12]) and torch.equal(Vc[pages - 3, :8], V[12:])
    compact_paged_kv(Kc, Vc, table, lens, torch.tensor([[3, 15]], dtype=torch.int32))
    assert torch.equal(Kc[pages - 1, 4], K[3]) and torch.equal(Vc[pages - 1, 5], V[15])
    copy_kv_pages(Kc, Vc, [pages - 1], [1])
    copy_kv_pages(Kc, Vc, [pages - 3], [pages - 2])
    assert torch.equal(Kc[1], Kc[pages - 1]) and torch.equal(Vc[pages - 2], Vc[pages - 3])


def test_64_bit_values_do_not_wrap():
    """Pages, lengths and steps past 32 bits on the GPU: outside of everything."""
    from qattention_amd import append_paged_kv, compact_paged_kv, copy_kv_pages, prefix_attention_paged
    ps, Hkv, D = 4, 2, 64
    Kc, Vc = cache(8, ps, Hkv, D, torch.float16, 23)
    K, V = (x[0] for x in cache(1, 2, Hkv, D, torch.float16, 24))
    before, w = (Kc.clone(), Vc.clone()), 2 ** 32
    table, lens = torch.tensor([[0, 1], [2, 3]], device=DEV), torch.tensor([w + 1, 2], device=DEV)
    say("64 bits")
    copy_kv_pages(Kc, Vc, torch.tensor([w + 1, 2], device=DEV), torch.tensor([5, w + 6], device=DEV))
    got = append_paged_kv(K[:1], V[:1], Kc, Vc, table + w, lens[1:])  # no such pages: the row is dropped
    assert got.tolist() == [3] and torch.equal(Kc, before[0]) and torch.equal(Vc, before[1])
    got = append_paged_kv(K, V, Kc, Vc, table, lens)
    assert got.tolist() == [2 ** 31 - 1, 3] and torch.equal(Kc[2, 2], K[1]) and torch.equal(Kc[:2], before[0][:2])
    k = Kc.clone()
    got = compact_paged_kv(Kc, Vc, table, torch.tensor([0, 0], device=DEV), torch.tensor([[1, w + 2], [w, 1]], device=DEV))
    assert got.tolist() == [1, 0] and torch.equal(Kc[0, 0], k[0, 1]) and torch.equal(Kc[2:], k[2:])
    Q = torch.empty(2, 4, D, dtype=torch.float16, device=DEV).normal_()
    O = prefix_attention_paged(Q, Kc, Vc, table, lens, max_seqlen=w)[0]
    assert torch.equal(O, prefix_attention_paged(Q, Kc, Vc, table, torch.tensor([2 * ps, 2], device=DEV))[0])
