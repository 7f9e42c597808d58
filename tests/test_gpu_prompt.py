"""prompt_attention against causal attention in 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

from attn64 import attend64, causal, check, offsets

pytestmark = pytest.mark.gpu
DEV = "cuda"


def say(*a):
    print(*a, flush=True)


def inputs(lens, Hq, Hkv, D, dtype, seed, sigma=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    T = sum(lens)
    return [torch.empty(T, h, D, dtype=dtype, device=DEV).normal_(0, sigma, generator=g) for h in (Hq, Hkv, Hkv)]


def reference(Q, K, V, lens):
    parts, a = [], 0
    for n in lens:
        parts.append(attend64(Q[a:a + n], K[a:a + n], V[a:a + n], causal(n)))
        a += n
    return [torch.cat(x) for x in zip(*parts)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,Hq,Hkv,D", [
    ([1], 4, 4, 64),
    ([2, 1, 3], 8, 2, 128),
    ([63, 64, 65], 8, 2, 128),
    ([127, 128, 129], 4, 4, 128),
    ([255, 257, 31, 33], 4, 4, 64),
    ([0, 5, 0, 200, 0], 8, 1, 64),
    ([300, 17], 6, 2, 128),        # 3 heads per kv head: tiles end inside a token's heads
    ([190], 32, 1, 128),           # 4 tokens per tile
    ([77, 130], 200, 1, 32),       # more heads than a tile has rows
    ([513, 100], 4, 2, 32),
    ([1100], 2, 1, 128),
])
def test_against_64_bits(lens, Hq, Hkv, D, dtype):
    from qattention_amd import prompt_attention
    Q, K, V = inputs(lens, Hq, Hkv, D, dtype, 100 + sum(lens) + D)
    say("prompt", lens, Hq, Hkv, D, dtype)
    O, L = prompt_attention(Q, K, V, offsets(lens), return_lse=True)
    check(O, L, reference(Q, K, V, lens))
    assert torch.equal(prompt_attention(Q, K, V, offsets(lens).to(DEV), max_seqlen=max(lens)), O)


@pytest.mark.parametrize("sigma", [0.05, 6.0])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_flat_and_peaked_weights(sigma, dtype):
    from qattention_amd import prompt_attention
    lens = [400, 130]
    Q, K, V = inputs(lens, 8, 2, 128, dtype, 7, sigma)
    say("prompt sigma", sigma, dtype)
    O, L = prompt_attention(Q, K, V, offsets(lens), return_lse=True)
    check(O, L, reference(Q, K, V, lens))


def test_strided_inputs():
    """Slices of one fused projection, heads outermost, a unit stride missing."""
    from qattention_amd import prompt_attention
    lens, Hq, Hkv, D = [150, 90], 8, 2, 64
    Q, K, V = inputs(lens, Hq, Hkv, D, torch.bfloat16, 11)
    cu = offsets(lens)
    want = prompt_attention(Q, K, V, cu, return_lse=True)
    fused = torch.cat([Q, K, V], 1)
    q, k, v = fused.split([Hq, Hkv, Hkv], 1)
    heads_first = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (Q, K, V)]
    odd = [torch.empty(x.shape[0], x.shape[1], D + 1, dtype=x.dtype, device=DEV)[:, :, 1:].copy_(x) for x in (Q, K, V)]
    for i, got in enumerate(((q, k, v), heads_first, odd)):
        say("strides", i)
        O, L = prompt_attention(*got, cu, return_lse=True)
        assert torch.equal(O, want[0]) and torch.equal(L, want[1])


@pytest.mark.parametrize("D,Hkv", [(128, 2), (64, 4), (32, 1)])
def test_later_tokens_never_show(D, Hkv):
    """Infinities and NaN of a later token's K or V stay out of earlier rows, and
    show in exactly the rows and dims that attend them."""
    from qattention_amd import prompt_attention
    lens, Hq = [200, 70], 4
    Q, K, V = inputs(lens, Hq, Hkv, D, torch.float16, 13)
    cu, g = offsets(lens), Hq // Hkv
    ref = reference(Q, K, V, lens)
    for bad in (math.nan, math.inf):
        for t in (0, 1, 63, 64, 130, 199):
            say("later", D, Hkv, bad, t)
            V2 = V.clone()
            V2[t, 0, 5] = bad
            O, L = prompt_attention(Q, K, V2, cu, return_lse=True)
            hit = torch.zeros_like(O, dtype=torch.bool)
            hit[t:200, :g, 5] = True
            assert torch.equal(~torch.isfinite(O), hit)
            check(O.masked_fill(hit, 0), L, [ref[0].masked_fill(hit, 0)] + list(ref[1:]))
            K2 = K.clone()
            K2[t, 0, 5] = math.nan
            O, L = prompt_attention(Q, K2, V, cu, return_lse=True)
            hit[t:200, :g] = True
            assert torch.equal(torch.isnan(O), hit) and torch.equal(torch.isnan(L), hit[:, :, 0])
            check(O.masked_fill(hit, 0), L.masked_fill(hit[:, :, 0], 0),
                  [ref[0].masked_fill(hit, 0), ref[1].masked_fill(hit[:, :, 0], 0)] + list(ref[2:]))


def test_scores_of_minus_infinity():
    """A key whose scores are -inf has no weight, wherever in the row it lies."""
    from qattention_amd import prompt_attention
    n, D = 150, 64
    Q, K, V = inputs([n], 2, 1, D, torch.bfloat16, 17)
    Q[:, :, 0] = Q[:, :, 0].abs() + 0.5
    for t in (0, 40, 80):
        say("minus infinity", t)
        K2 = K.clone()
        K2[t, 0, 0] = -math.inf
        O, L = prompt_attention(Q, K2, V, offsets([n]), return_lse=True)
        mask = causal(n)
        mask[:, t] = False
        K3 = K2.clone()
        K3[t] = 0
        ref = attend64(Q, K3, V, mask)
        alone = ~mask.any(1)  # nothing but -inf scores: -inf - -inf, as the formula has it
        assert bool(torch.isnan(O[alone]).all())
        check(O[~alone], L[~alone], [x[~alone] for x in ref])


def test_largest_values():
    """Means of fp16's largest value stay finite, whole tiles and cut ones."""
    from qattention_amd import prompt_attention
    for n, Hq, Hkv, D in ((300, 4, 2, 64), (2100, 4, 1, 128)):
        Q, K, V = inputs([n], Hq, Hkv, D, torch.float16, 37)
        V.fill_(-65504.0)
        V[:, :, ::2] = 65504.0
        say("largest", n)
        O = prompt_attention(Q, K, V, offsets([n]))
        assert torch.equal(O, V[:, :1].expand(n, Hq, D))


def test_steep_scores():
    """Scores that rise by hundreds from block to block, and fall again."""
    from qattention_amd import prompt_attention
    n, D = 400, 64
    for dtype in (torch.float16, torch.bfloat16):
        Q, K, V = inputs([n], 2, 1, D, dtype, 41)
        Q[:, :, 0], K[:, :, 0] = 8.0, 0.0
        K[:, 0, 0] = torch.tensor([0, 30, 120, 400, 500, 100, 0], device=DEV)[torch.arange(n, device=DEV) // 64]
        say("steep", dtype)
        O, L = prompt_attention(Q, K, V, offsets([n]), return_lse=True)
        check(O, L, reference(Q, K, V, [n]))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,Hkv,n", [(128, 2, 300), (64, 4, 300), (32, 1, 190), (64, 1, 2100)])
def test_infinities_and_nan_of_v(D, Hkv, n, dtype):
    """A row is the finite values' mean plus the infinities and NaN that it attends,
    by their dims; their neighbours in the same block do not change."""
    from qattention_amd import prompt_attention
    Hq = 4
    Q, K, V = inputs([n], Hq, Hkv, D, dtype, 43)
    for t, d, x in ((n - 7, 3, math.inf), (n - 40, 9, -math.inf), (n - 31, 9, math.inf), (n - 31, 20, math.nan),
                    (130, 30, -math.inf), (5, 31, math.inf)):
        V[t, Hkv - 1, d] = x
    say("odd values", D, Hkv, n, dtype)
    O, L = prompt_attention(Q, K, V, offsets([n]), return_lse=True)
    finite = torch.where(V.isfinite(), V, 0)
    odd = torch.where(V.isfinite(), 0, V).float().cumsum(0).repeat_interleave(Hq // Hkv, 1)
    hit = odd != 0
    assert torch.equal(O[hit].float().nan_to_num(9.0, 2.0, -2.0), odd[hit].nan_to_num(9.0, 2.0, -2.0))
    ref = reference(Q, K, finite, [n])
    check(O.masked_fill(hit, 0), L, [ref[0].masked_fill(hit, 0)] + list(ref[1:]))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_low_scores_behind_minus_infinity(dtype):
    """A whole block of -inf scores, then scores of about -100: only rows within
    the block have no mean."""
    from qattention_amd import prompt_attention
    n, D, m = 230, 64, 64
    Q, K, V = inputs([n], 2, 1, D, dtype, 47)
    Q[:, :, 0], K[:, 0, 0], K[:m, 0, 0] = 8.0, -100.0, -math.inf
    say("low", dtype)
    O, L = prompt_attention(Q, K, V, offsets([n]), return_lse=True)
    assert O[:m].isnan().all() and (L[:m] == -math.inf).all()
    check(O[m:], L[m:], reference(Q[m:], K[m:], V[m:], [n - m]))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,Hq,Hkv,D", [
    ([1] * 30 + [700] + [0, 1, 2, 3] * 10, 4, 2, 128),
    ([1] * 30 + [2000] + [1] * 39, 4, 2, 64),      # its tiles are cut
    ([1300] + [1] * 200 + [900, 0], 3, 1, 32),
    ([1] * 127 + [900] + [5] * 3, 9, 3, 64),
])
def test_one_long_prompt_among_short_ones(lens, Hq, Hkv, D, dtype):
    from qattention_amd import prompt_attention
    Q, K, V = inputs(lens, Hq, Hkv, D, dtype, 61)
    cu = offsets(lens)
    say("mixed", len(lens), max(lens), Hq, Hkv, D, dtype)
    O, L = prompt_attention(Q, K, V, cu, return_lse=True)
    check(O, L, reference(Q, K, V, lens))
    # a sequence that is none (its end lies ahead of its start) and one that
    # leaves Q: the others stay what they were
    at = lens.index(max(lens))
    bad = cu.clone()
    bad[-1] = sum(lens) + 5
    bad[at + 1] = cu[at] - 1  # (the next one now starts there)
    keep = torch.ones(sum(lens), dtype=torch.bool, device=DEV)
    keep[cu[at] - 1 if at else 0:cu[at + 2]] = False
    keep[cu[-2]:] = False
    O2, L2 = prompt_attention(Q, K, V, bad, max_seqlen=max(lens), return_lse=True)
    assert torch.equal(O2[keep], O[keep]) and torch.equal(L2[keep], L[keep])


def test_rows_of_no_sequence_stay():
    """Through the C entry: rows in front of, between and behind the sequences keep
    what they held; bad offsets and max_seqlen cut what is computed."""
    from qattention_amd import _lib, prompt_attention
    T, Hq, Hkv, D = 260, 4, 2, 64
    Q, K, V = inputs([T], Hq, Hkv, D, torch.float16, 19)
    cu = torch.tensor([3, 100, 90, 240, 400], dtype=torch.int32, device=DEV)  # sequence 1 and 3 are bad
    O = torch.full_like(Q, 7.0)
    L = torch.full((T, Hq), 7.0, device=DEV)
    say("no sequence")
    rc = _lib.lib().qattn_prompt_fwd(
        Q.data_ptr(), _lib.i64arr(Q.stride()), K.data_ptr(), _lib.i64arr(K.stride()), V.data_ptr(),
        _lib.i64arr(V.stride()), O.data_ptr(), _lib.i64arr(O.stride()), L.data_ptr(), _lib.i64arr(L.stride()),
        cu.data_ptr(), 4, 120, T, Hq, Hkv, D, 1 / math.sqrt(D), 0, None, 0, torch.cuda.current_stream().cuda_stream)
    _lib.check(rc, "qattn_prompt_fwd")
    done = torch.zeros(T, dtype=torch.bool, device=DEV)
    for a, b in ((3, 100), (90, 210)):
        done[a:b] = True
    assert bool((O[~done] == 7).all()) and bool((L[~done] == 7).all())
    # (rows 90 .. 99 belong to sequences 0 and 2 both)
    check(O[3:90], L[3:90], attend64(Q[3:90], K[3:90], V[3:90], causal(87)))
    o, l = prompt_attention(Q[90:210], K[90:210], V[90:210], offsets([120]), return_lse=True)
    assert torch.equal(O[100:210], o[10:]) and torch.equal(L[100:210], l[10:])


def test_long_prompt_rows():
    """Rows of a long prompt, among them the last (more than 2^16 keys)."""
    from qattention_amd import prompt_attention
    n, Hq, Hkv, D = 70001, 2, 1, 64
    Q, K, V = inputs([n], Hq, Hkv, D, torch.bfloat16, 23)
    say("long")
    O, L = prompt_attention(Q, K, V, offsets([n]), return_lse=True)
    rows = torch.tensor([0, 1, 64, 65535, 65536, n - 65, n - 1], device=DEV)
    mask = torch.arange(n, device=DEV)[None, :] <= rows[:, None]
    check(O[rows], L[rows], attend64(Q[rows], K, V, mask))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,Hq,Hkv,D", [
    ([2100], 4, 1, 128),
    ([1900, 1899, 60], 2, 2, 64),
    ([3001], 8, 1, 32),
    ([1801], 3, 1, 128),
])
def test_cut_tiles(lens, Hq, Hkv, D, dtype):
    """Few heads of long prompts: tiles cut into parts that a second kernel joins."""
    from qattention_amd import _lib, prompt_attention
    Q, K, V = inputs(lens, Hq, Hkv, D, dtype, 31)
    say("cut", lens, Hq, Hkv, D, dtype)
    O, L = prompt_attention(Q, K, V, offsets(lens), return_lse=True)
    assert _lib.last_kernel() == "prompt_merge_kernel"
    check(O, L, reference(Q, K, V, lens))
    # what a later token holds stays out of every part
    t = lens[0] // 2
    V2 = V.clone()
    V2[t, 0, 3] = math.nan
    O2, L2 = prompt_attention(Q, K, V2, offsets(lens), return_lse=True)
    hit = torch.zeros_like(O, dtype=torch.bool)
    hit[t:lens[0], :Hq // Hkv, 3] = True
    assert torch.equal(torch.isnan(O2), hit)
    ref = reference(Q, K, V, lens)
    check(O2.masked_fill(hit, 0), L2, [ref[0].masked_fill(hit, 0)] + list(ref[1:]))


def test_other_stream_and_graph():
    from qattention_amd import prompt_attention
    lens = [140, 70]
    Q, K, V = inputs(lens, 8, 2, 128, torch.float16, 29)
    cu = offsets(lens).to(DEV)
    want = prompt_attention(Q, K, V, cu, max_seqlen=140, return_lse=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = prompt_attention(Q, K, V, cu, max_seqlen=140, return_lse=True)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    say("graph")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = prompt_attention(Q, K, V, cu, max_seqlen=140, return_lse=True)
    for i in range(4):
        Q.normal_()
        # shorter prompts in the captured call: the lengths are read on the device
        cu.copy_(offsets([lens[0] - 30 * i, lens[1] - 10 * i]))
        graph.replay()
        want = prompt_attention(Q, K, V, cu, max_seqlen=140, return_lse=True)
        n = int(cu[-1])
        assert torch.equal(got[0][:n], want[0][:n]) and torch.equal(got[1][:n], want[1][:n])


def test_lengths_past_32_bits():
    """max_seqlen counts in full, and an offset of 2^32 and more is not one of Q's rows."""
    from qattention_amd import prompt_attention
    Q, K, V = inputs([50], 4, 2, 64, torch.float16, 53)
    want = prompt_attention(Q, K, V, offsets([20, 30]), return_lse=True)
    say("past 32 bits")
    for ms in (30, 2 ** 31 + 7, 2 ** 40):
        O, L = prompt_attention(Q, K, V, offsets([20, 30]), ms, return_lse=True)
        assert torch.equal(O, want[0]) and torch.equal(L, want[1])
    for device in ("cpu", DEV):
        cu = torch.tensor([0, 20, 2 ** 32 + 50], device=device)
        O, L = prompt_attention(Q, K, V, cu, return_lse=True)
        assert torch.equal(O[:20], want[0][:20]) and torch.equal(L[:20], want[1][:20])


def test_contiguous_inputs_off_a_boundary():
    """Rows that start off a 16-byte boundary, and one token whose unused stride is odd."""
    from qattention_amd import prefix_attention_paged, prompt_attention, ragged_attention
    lens, Hq, Hkv, D = [40, 9], 4, 2, 64
    Q, K, V = inputs(lens, Hq, Hkv, D, torch.float16, 59)
    cu = offsets(lens)
    shifted = [torch.cat([x.new_zeros(3), x.flatten()])[3:].view(x.shape) for x in (Q, K, V)]
    say("off a boundary")
    assert torch.equal(prompt_attention(*shifted, cu), prompt_attention(Q, K, V, cu))
    assert torch.equal(ragged_attention(*shifted, cu, 2, 5), ragged_attention(Q, K, V, cu, 2, 5))
    table, ctx = torch.tensor([[0, 1]], dtype=torch.int32, device=DEV), torch.tensor([20], dtype=torch.int32, device=DEV)
    cache = [x[:32].view(2, 16, Hkv, D) for x in (K, V)]
    wide = Hq * D + 3
    one = torch.cat([Q.view(49, -1), Q.new_zeros(49, 3)], 1).as_strided((1, Hq, D), (wide, D, 1), 8 * wide)
    got, want = (prefix_attention_paged(q, *cache, table, ctx) for q in (one, Q[8:9]))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
