"""Where the softmax of the serving calls can go wrong: scores that rise by about what
fp32 weights hold, and rows in which one key has most of the weight."""
from __future__ import annotations

import math

import pytest
import torch

from attn64 import attend64, causal, check, offsets

pytestmark = pytest.mark.gpu
DEV = "cuda"
RISES = [82 + i / 4 for i in range(33)]  # nats: a weight of e^82 .. e^90, that is 2^118 .. 2^130


def say(*a):
    print(*a, flush=True)


def rising(levels, D, Hq, Hkv, dtype, seed):
    """Packed Q, K, V of one sequence per row of levels [B, n]: q.k / sqrt(D) of key
    j is levels[s, j] nats and noise of about a tenth."""
    B, n = levels.shape
    g = torch.Generator(device=DEV).manual_seed(seed)
    Q, K, V = (torch.empty(B * n, h, D, dtype=dtype, device=DEV).normal_(0, 1, generator=g) for h in (Hq, Hkv, Hkv))
    Q *= 0.1
    whole = levels.floor()  # (whole numbers and quarters: exact in 8 bits)
    Q[:, :, :2] = D ** 0.5
    K[:, :, 0], K[:, :, 1] = (x.to(DEV).reshape(-1, 1) for x in (whole, levels - whole))
    return Q, K, V


def check_each(O, L, Q, K, V, n, what):
    for s in range(Q.shape[0] // n):
        at = slice(s * n, (s + 1) * n)
        check(O[at], L[at], attend64(Q[at], K[at], V[at], causal(n)), (*what, s))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("high", [1, 64])
@pytest.mark.parametrize("blocks,behind", [(5, 20.0), (5, 5.0), (2, 0.0), (3, 60.0)])
def test_one_rise(blocks, behind, high, dtype):
    """Scores of 0, then one key or a block of keys far above, then blocks a little
    below that (or nothing: the rise is in the last block)."""
    from qattention_amd import prompt_attention
    n = 64 * blocks
    levels = torch.zeros(len(RISES), n)
    for s, rise in enumerate(RISES):
        levels[s, 64:64 + high] = rise
        levels[s, 128:] = rise - behind
    Q, K, V = rising(levels, 64, 2, 1, dtype, 83)
    say("one rise", blocks, behind, high, dtype)
    O, L = prompt_attention(Q, K, V, offsets([n] * len(RISES)), return_lse=True)
    check_each(O, L, Q, K, V, n, ("rise", blocks, behind, high))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("first,D", [(640, 64), (700, 128), (1100, 64)])
def test_a_rise_between_the_parts_of_a_cut_prompt(first, D, dtype):
    """Few heads of one long prompt: the joined parts' references differ by the rise."""
    from qattention_amd import _lib, prompt_attention
    n = 2100
    for rise in RISES[::2]:
        levels = torch.zeros(1, n)
        levels[0, first:] = rise
        Q, K, V = rising(levels, D, 2, 1, dtype, 89)
        say("rise between parts", first, D, rise, dtype)
        O, L = prompt_attention(Q, K, V, offsets([n]), return_lse=True)
        assert _lib.last_kernel() == "prompt_merge_kernel"
        check_each(O, L, Q, K, V, n, ("parts", first, rise))


def dominated(q, k, v, mask):
    """attend64's o and bound, but for the key of the row's largest weight: its weight
    is 1 before the division and has no rounding, so half a step per weight counts
    against the other keys' |v| alone."""
    o, _, to, _ = attend64(q, k, v, mask)
    half, g = torch.finfo(q.dtype).eps / 2, q.shape[1] // k.shape[1]
    for h in range(q.shape[1]):
        s = q[:, h].double() @ k[:, h // g].double().T / math.sqrt(q.shape[2])
        p = torch.softmax(s.masked_fill(~mask, -math.inf), 1)
        top, at = p.max(1)
        to[:, h] -= half * top[:, None] * v[:, h // g].double()[at].abs()
    return o, to


@pytest.mark.parametrize("sigma", [2.0, 3.0])
def test_largest_weight_of_bf16_prompts_is_exact(sigma):
    from qattention_amd import prompt_attention
    for n, Hq, Hkv, D in ((700, 8, 2, 128), (1500, 2, 1, 64), (300, 4, 4, 32)):
        g = torch.Generator(device=DEV).manual_seed(97)
        Q, K, V = (torch.empty(n, h, D, dtype=torch.bfloat16, device=DEV).normal_(0, sigma, generator=g)
                   for h in (Hq, Hkv, Hkv))
        say("dominated prompt", sigma, n, D)
        O = prompt_attention(Q, K, V, offsets([n]))
        o, to = dominated(Q, K, V, causal(n))
        off = (O.double() - o).abs() - to
        assert float(off.max()) <= 0, (n, float(off.max()), int((off > 0).sum()))


@pytest.mark.parametrize("sigma", [2.0, 3.0])
@pytest.mark.parametrize("n,ctx", [(1, 700), (1, 5000), (9, 3000), (60, 900), (200, 4000)])
def test_largest_weight_over_bf16_pages_is_exact(n, ctx, sigma):
    """One workgroup per item, runs, tiles of 32 and of 128 rows."""
    from qattention_amd import prefix_attention_paged
    Hq, Hkv, D, ps = 6, 2, 128, 16
    g = torch.Generator(device=DEV).manual_seed(101)
    pages = -(-ctx // ps)
    Kc, Vc = (torch.empty(pages, ps, Hkv, D, dtype=torch.bfloat16, device=DEV).normal_(0, sigma, generator=g)
              for _ in range(2))
    Q = torch.empty(n, Hq, D, dtype=torch.bfloat16, device=DEV).normal_(0, sigma, generator=g)
    table = torch.arange(pages, dtype=torch.int32, device=DEV)[None]
    say("dominated pages", sigma, n, ctx)
    O = prefix_attention_paged(Q, Kc, Vc, table, torch.tensor([ctx], device=DEV, dtype=torch.int32), offsets([n]),
                               return_lse=False)
    o, to = dominated(Q, Kc.flatten(0, 1)[:ctx], Vc.flatten(0, 1)[:ctx], torch.ones(n, ctx, dtype=torch.bool, device=DEV))
    off = (O.double() - o).abs() - to
    assert float(off.max()) <= 0, (n, float(off.max()), int((off > 0).sum()))
