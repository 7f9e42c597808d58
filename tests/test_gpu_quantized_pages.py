"""append_quantized_kv and read_quantized_kv against the formats' definitions, and the
moves of a quantised cache's bytes: every byte and value exactly."""
from __future__ import annotations

import math

import pytest
import torch

import quant64
from attn64 import offsets

pytestmark = pytest.mark.gpu
DEV = "cuda"
FP16, BF16 = torch.float16, torch.bfloat16


def say(*a):
    print(*a, flush=True)


def noise(pages, ps, Hkv, D, bits, seed, layers=None):
    """A cache of random bytes."""
    import qattention_amd as qa
    g = torch.Generator().manual_seed(seed)
    shape = (pages, ps, Hkv) if layers is None else (layers, pages, ps, Hkv)
    return qa.QuantizedKV(*(torch.randint(0, 256, shape + (n,), dtype=torch.uint8, generator=g).to(DEV)
                            for n in (D * bits // 8, D * bits // 8, D // 32, D // 32)))


def rows(T, Hkv, D, dtype, seed):
    """Rows whose blocks differ in size by many powers of two, with ties, zeros, the
    type's largest and smallest numbers, infinities and NaN among them."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, Hkv, D // 32, 32, generator=g)
    x *= torch.exp2(torch.randint(-20, 12, (T, Hkv, D // 32, 1), generator=g).float())
    ties = torch.randint(-28, 29, x.shape, generator=g) / 4.0
    x = torch.where(torch.rand(T, Hkv, D // 32, 1, generator=g) < 0.3, ties, x)
    x = x.to(dtype).flatten(0, 2)
    info = torch.finfo(dtype)
    special = [0.0, -0.0, info.max, -info.max, info.tiny, info.smallest_normal / 4, -info.tiny, math.inf, -math.inf,
               math.nan, info.max / 2, 1.75, 1.7578125, 7.0, -7.0, 448.0, 450.0]
    for i, v in enumerate(special):
        at = (5 * i + 3) % x.shape[0]
        if i % 3 == 0:
            x[at] = v
        else:
            x[at, (7 * i) % 32] = v
    return x.view(T, Hkv, D)


def same(a, b):
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(0), b.nan_to_num(0))


def tables(B, cols, pages, seed):
    return torch.randperm(pages, generator=torch.Generator().manual_seed(seed))[:B * cols].view(B, cols).to(torch.int32)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [FP16, BF16])
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
def test_append_and_read(ctx, new, ps, Hkv, D, dtype, bits):
    import qattention_amd as qa
    B, n = len(ctx), [1] * len(ctx) if new is None else new
    cols = max(-(-(c + x) // ps) for c, x in zip(ctx, n))
    cache = noise(B * cols + 4, ps, Hkv, D, bits, 1)
    table = tables(B, cols, B * cols + 4, 2)
    K, V = rows(sum(n), Hkv, D, dtype, 3), rows(sum(n), Hkv, D, dtype, 4)
    want = [t.cpu() for t in cache]
    seq = torch.tensor([s for s in range(B) for _ in range(n[s])])
    pos = torch.tensor([ctx[s] + i for s in range(B) for i in range(n[s])])
    at = table[seq, pos // ps].long(), pos % ps
    for i, x in enumerate((K, V)):
        want[i][at], want[2 + i][at] = quant64.encode(x, bits)
    lens = torch.tensor(ctx, dtype=torch.int32, device=DEV)
    cu = None if new is None else offsets(new)
    say("append", ctx[:5], n[:5], ps, Hkv, D, dtype, bits)
    got = qa.append_quantized_kv(K.to(DEV), V.to(DEV), cache, table.to(DEV), lens, cu)
    assert got.dtype == torch.int32 and got.tolist() == [c + x for c, x in zip(ctx, n)] and lens.tolist() == ctx
    for a, b, what in zip(cache, want, ("K", "V", "K_scale", "V_scale")):
        assert torch.equal(a.cpu(), b), what
    for out in (FP16, BF16):
        say("read", out)
        back = qa.read_quantized_kv(cache, table.to(DEV), lens, cu, dtype=out)
        for x, e, s in zip(back, want[:2], want[2:]):
            assert x.dtype == out and x.shape == K.shape
            assert same(x.cpu(), quant64.decode(e[at], s[at], bits).float().to(out))
    # half a step of the format of the scaled value, or what its largest cuts off
    err = (back[0].cpu().double() - K.double()).abs().unflatten(-1, (-1, 32))
    top = K.double().abs().unflatten(-1, (-1, 32)).amax(-1, keepdim=True)
    inside = (torch.isfinite(top) & (top <= 1.75 * 2.0 ** quant64.LAST[dtype]) & (top > 1e-30)).expand_as(err)
    step = {4: 2.0 ** -2, 8: 2.0 ** -4}[bits]  # of the block's largest, at its worst: 1 of 4, 16 of 256
    assert bool((err <= step * top)[inside].all())


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_every_code_and_scale(D, bits):
    """All bytes under all scales, in both types."""
    import qattention_amd as qa
    cache = noise(40, 16, 2, D, bits, 5)
    scale = torch.arange(40 * 16 * 2 * (D // 32), device=DEV).view(cache.K_scale.shape) % 256
    cache.K_scale.copy_(scale)
    table = torch.arange(40, dtype=torch.int32, device=DEV).view(1, 40)
    for dtype in (FP16, BF16):
        say("codes", D, bits, dtype)
        K, V = qa.read_quantized_kv(cache, table, torch.zeros(1, dtype=torch.int32), offsets([640]), dtype=dtype)
        for x, e, s in ((K, cache.K, cache.K_scale), (V, cache.V, cache.V_scale)):
            want = quant64.decode(e.cpu(), s.cpu(), bits).flatten(0, 1).float().to(dtype)
            assert same(x.cpu(), want)


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("bits", [4, 8])
def test_what_has_no_place(bits, many):
    """Past the table, missing pages, negative lengths, bad offsets, max_seqlen; alone and
    in front of sequences enough that rows are dealt out packed."""
    import qattention_amd as qa
    ps, Hkv, D, more = 4, 2, 64, 100 if many else 0
    cache = noise(12, ps, Hkv, D, bits, 5)
    table = torch.tensor([[0, 1], [2, 99], [-1, 5], [6, 7], [8, 9], [10, 11]] + [[-1, -1]] * more, dtype=torch.int32)
    ctx = torch.tensor([6, 3, 2, -1, 0, 9] + [0] * more, dtype=torch.int32)
    cu = torch.tensor([0, 5, 10, 15, 17, 16, 22] + [22] * more, dtype=torch.int32)  # sequence 4's offsets are bad
    K, V = rows(22, Hkv, D, FP16, 6), rows(22, Hkv, D, FP16, 7)
    want = [t.cpu() for t in cache]
    for i, x in enumerate((K, V)):
        for part, y in zip((want[i], want[2 + i]), quant64.encode(x, bits)):
            part[1, 2], part[1, 3] = y[0], y[1]      # sequence 0: two of five rows have a place
            part[2, 3] = y[5]                        # sequence 1: its second page is missing
            part[5, 0], part[5, 1] = y[12], y[13]    # sequence 2: its first page is missing, four rows at most
    say("no place", bits, many)
    got = qa.append_quantized_kv(K.to(DEV), V.to(DEV), cache, table, ctx, cu, max_seqlen=4)
    assert got.tolist() == [8, 7, 6, -1, 0, 9] + [0] * more
    for a, b in zip(cache, want):
        assert torch.equal(a.cpu(), b)
    # read from the same lengths: sequence 3 starts one before its first row
    start = ctx.clone()
    start[5] = 2**31 - 1
    K, V = (x.cpu() for x in qa.read_quantized_kv(cache, table, start, cu, max_seqlen=4, total_tokens=30, dtype=BF16))
    assert K.shape == (30, Hkv, D)
    for x, e, s in ((K, cache.K, cache.K_scale), (V, cache.V, cache.V_scale)):
        v = quant64.decode(e.cpu(), s.cpu(), bits).float().to(BF16)
        zero = torch.zeros(Hkv, D, dtype=BF16)
        # (row 16 is sequence 3's second and sequence 5's first)
        for row, val in [(0, v[1, 2]), (1, v[1, 3]), (2, zero), (3, zero), (5, v[2, 3]), (6, zero), (10, zero),
                         (11, zero), (12, v[5, 0]), (13, v[5, 1]), (15, zero), (17, zero), (18, zero), (19, zero)]:
            assert same(x[row], val), row


def test_long_starts_and_empty_calls():
    import qattention_amd as qa
    cache = noise(4, 16, 2, 64, 4, 8)
    table = torch.tensor([[0, 1, 2, 3]], dtype=torch.int32, device=DEV)
    for start in (2**40, -2**40, 2**31 - 1, -2**31, 64, 63):
        K, _ = qa.read_quantized_kv(cache, table, torch.tensor([start]), offsets([3]), dtype=BF16)
        want = torch.zeros(3, 2, 64, dtype=BF16)
        if start == 63:
            want[0] = quant64.decode(cache.K[3, 15].cpu(), cache.K_scale[3, 15].cpu(), 4).to(BF16)
        assert same(K.cpu(), want), start
    K, _ = qa.read_quantized_kv(cache, table, torch.tensor([-1]), offsets([2]), dtype=BF16)
    assert not K[0].any() and same(K[1].cpu(), quant64.decode(cache.K[0, 0].cpu(), cache.K_scale[0, 0].cpu(), 4).to(BF16))
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    K, V = qa.read_quantized_kv(cache, table[:0], none)
    assert K.shape == V.shape == (0, 2, 64)
    x = torch.zeros(0, 2, 64, dtype=FP16, device=DEV)
    before = [t.clone() for t in cache]
    assert qa.append_quantized_kv(x, x, cache, table[:0], none).shape == (0,)
    assert qa.append_quantized_kv(x, x, cache, table, torch.tensor([5]), offsets([0])).tolist() == [5]
    empty = qa.quantized_kv_cache(0, 16, 2, 64)
    y = torch.ones(1, 2, 64, dtype=FP16, device=DEV)
    assert qa.append_quantized_kv(y, y, empty, table, torch.tensor([5])).tolist() == [6]
    assert not qa.read_quantized_kv(empty, table, torch.tensor([5]))[0].any()
    assert all(torch.equal(a, b) for a, b in zip(cache, before))


@pytest.mark.parametrize("bits", [4, 8])
def test_layouts(bits):
    """A layer's slice with the layers side by side in each page, rows with gaps between
    heads, rows of the inputs with odd strides."""
    import qattention_amd as qa
    ps, Hkv, D, n = 8, 3, 64, 21
    e, s = D * bits // 8, D // 32
    g = torch.Generator().manual_seed(9)
    big = [torch.randint(0, 256, (6, 2, ps, Hkv + 1, 2 * w), dtype=torch.uint8, generator=g).to(DEV)
           for w in (e, e, s, s)]
    cache = qa.QuantizedKV(*(t[:, 1, :, 1:, :t.shape[-1] // 2] for t in big))
    want = [t.cpu() for t in big]
    table = torch.tensor([[4, 0, 3]], dtype=torch.int32, device=DEV)
    K, V = rows(n, 2 * Hkv, D, FP16, 10)[:, ::2], rows(n, Hkv, 2 * D, FP16, 11)[..., ::2]
    pos = torch.arange(2, 2 + n)
    at = table[0].cpu()[pos // ps].long(), pos % ps
    for i, x in enumerate((K, V)):
        for w, y in zip((want[i], want[2 + i]), quant64.encode(x, bits)):
            w[at[0], 1, at[1], 1:, :w.shape[-1] // 2] = y
    say("layouts", bits)
    lens = torch.tensor([2], dtype=torch.int32, device=DEV)
    Kd, Vd = rows(n, 2 * Hkv, D, FP16, 10).to(DEV)[:, ::2], rows(n, Hkv, 2 * D, FP16, 11).to(DEV)[..., ::2]
    qa.append_quantized_kv(Kd, Vd, cache, table, lens, offsets([n]))
    for a, b in zip(big, want):
        assert torch.equal(a.cpu(), b)
    Kr, Vr = qa.read_quantized_kv(cache, table, lens, offsets([n]), dtype=BF16)
    for x, src in ((Kr, K), (Vr, V)):
        assert same(x.cpu(), quant64.decode(*quant64.encode(src, bits), bits).float().to(BF16))


def test_moves_of_bytes():
    """compact_paged_kv and copy_kv_pages over elements and scales of every width, as
    torch moves them."""
    import qattention_amd as qa
    for bits, D, Hkv, layers, gap in ((4, 128, 8, 3, 0), (8, 128, 2, None, 0), (4, 64, 3, 2, 0), (4, 32, 1, 2, 0),
                                      (8, 32, 5, 2, 1), (4, 128, 3, None, 1), (4, 64, 7, 2, 1)):
        ps, B, cols = 4, 3, 5
        wide = noise(B * cols + 4, ps, Hkv + gap, D, bits, 12, layers)
        cache = qa.QuantizedKV(*(t[..., :Hkv, :] for t in wide))
        table = tables(B, cols, B * cols + 4, 13)
        ctx, path = [3, 0, 9], torch.tensor([[0, 2, 5, -1], [1, 3, 4, 7], [0, 1, 1, 2]], dtype=torch.int32)
        steps = [3, 4, 2]
        want = [t.clone() for t in wide]
        for w in want:
            old = w.clone()
            for s in range(B):
                for j in range(steps[s]):
                    a, b = ctx[s] + int(path[s, j]), ctx[s] + j
                    w[..., int(table[s, b // ps]), b % ps, :Hkv, :] = old[..., int(table[s, a // ps]), a % ps, :Hkv, :]
        lens = torch.tensor(ctx, dtype=torch.int32, device=DEV)
        say("compact", bits, D, Hkv, layers, gap)
        for k, v in ((cache.K, cache.V), (cache.K_scale, cache.V_scale)):
            new = qa.compact_paged_kv(k, v, table.to(DEV), lens, path.to(DEV))
            assert new.tolist() == [c + n for c, n in zip(ctx, steps)]
        assert all(torch.equal(a, b) for a, b in zip(wide, want))
        src, dst = [0, 3, 5], [6, 1, 18]
        for w in want:
            p = w if layers is None else w.transpose(0, 1)
            p[dst, ..., :Hkv, :] = p[src][..., :Hkv, :]
        say("copy", bits, D, Hkv, layers, gap)
        for k, v in ((cache.K, cache.V), (cache.K_scale, cache.V_scale)):
            qa.copy_kv_pages(k, v, src, dst)
        assert all(torch.equal(a, b) for a, b in zip(wide, want))


@pytest.mark.parametrize("bits", [4, 8])
def test_offsets_past_32_bits(bits):
    """Pages 5 GiB from the first one: written, moved, copied and read back."""
    import qattention_amd as qa
    ps, Hkv, D, n = 16, 2, 128, 40
    widths = [Hkv * D * bits // 8] * 2 + [Hkv * D // 32] * 2
    room = torch.empty((5 << 30) + (1 << 20), dtype=torch.uint8, device=DEV)
    step = (5 << 30) // 4
    cache = qa.QuantizedKV(*(room.as_strided((5, ps, Hkv, w // Hkv), (step, w, w // Hkv, 1), i << 16)
                             for i, w in enumerate(widths)))
    for t in cache:
        t.zero_()
    table = torch.tensor([[4, 0, 3]], dtype=torch.int32, device=DEV)
    K, V = rows(n, Hkv, D, FP16, 20).to(DEV), rows(n, Hkv, D, FP16, 21).to(DEV)
    zero = torch.zeros(1, dtype=torch.int32, device=DEV)
    say("far", bits)
    assert qa.append_quantized_kv(K, V, cache, table, zero, offsets([n])).tolist() == [n]
    want = [quant64.decode(*quant64.encode(x, bits), bits).float().to(BF16) for x in (K, V)]
    for x, w in zip(qa.read_quantized_kv(cache, table, zero, offsets([n]), dtype=BF16), want):
        assert same(x.cpu(), w)
    # rows 1, 33 and 39 to places 0, 1 and 2; then page 4 to page 1
    path = torch.tensor([[1, 33, 39]], dtype=torch.int32, device=DEV)
    for k, v in ((cache.K, cache.V), (cache.K_scale, cache.V_scale)):
        assert qa.compact_paged_kv(k, v, table, zero, path).tolist() == [3]
        qa.copy_kv_pages(k, v, [4], [1])
    other = torch.tensor([[1]], dtype=torch.int32, device=DEV)
    for t in (table, other):
        for x, w in zip(qa.read_quantized_kv(cache, t, zero, offsets([ps]), dtype=BF16), want):
            assert same(x.cpu(), torch.cat([w[[1, 33, 39]], w[3:ps]]))
