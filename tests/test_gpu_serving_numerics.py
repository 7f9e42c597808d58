"""Where the softmax of the serving calls can go wrong: scores that rise by about what
fp32 weights hold."""
from __future__ import annotations

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
