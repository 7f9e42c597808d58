"""The paged operators and the tree kernels together, as a serving loop uses them:
prompts in, draft trees verified over the paged context, accepted paths kept, single
tokens decoded, a sequence forked.  Every answer is checked in 64 bits against the
rows that a plain list of the kept K/V holds."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from attn64 import attend64, causal, check, offsets

pytestmark = pytest.mark.gpu
DEV = "cuda"
HQ, HKV, D, PS, LAYERS = 8, 2, 64, 16, 2


def say(*a):
    print(*a, flush=True)


def rand(g, *shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device=DEV).normal_(0, 1, generator=g)


def merged(pre, tree):
    """fused_lse_merge over [T, H] states: one batch row per call."""
    from qattention_amd import fused_lse_merge
    heads = lambda x: x.transpose(0, 1)[None]  # noqa: E731
    return fused_lse_merge(heads(pre[1]), heads(tree[1]), heads(pre[0]), heads(tree[0]))[0].transpose(0, 1)


def close(O, ref, what):
    """The merge rounds each half's output once more: one more half step of each."""
    o, _, to, _ = ref
    half = torch.finfo(O.dtype).eps / 2
    off = (O.double() - o).abs() - (3 * to + half * o.abs())
    assert float(off.max()) <= 0, (what, float(off.max()))


def test_serving_loop():
    import qattention_amd as qa
    g = torch.Generator(device=DEV).manual_seed(5)
    B, prompts, b, depth = 3, [45, 16, 130], 2, 3
    N, cols = 15, 16
    Kc, Vc = (torch.full((LAYERS, (B + 1) * cols, PS, HKV, D), float("nan"), dtype=torch.bfloat16, device=DEV)
              for _ in range(2))
    table = torch.randperm((B + 1) * cols, generator=torch.Generator().manual_seed(6)).view(B + 1, cols)
    table = table.to(DEV, torch.int32)
    lens = torch.zeros(B, dtype=torch.int32, device=DEV)
    kept = [[(rand(g, 0, HKV, D), rand(g, 0, HKV, D)) for _ in range(B)] for _ in range(LAYERS)]

    def grow(layer, s, k, v):
        a, c = kept[layer][s]
        kept[layer][s] = torch.cat([a, k]), torch.cat([c, v])

    # prompts
    cu = offsets(prompts).to(DEV)
    for layer in range(LAYERS):
        q, k, v = (rand(g, sum(prompts), h, D) for h in (HQ, HKV, HKV))
        say("prompt", layer)
        O = qa.prompt_attention(q, k, v, cu, max(prompts))
        new = qa.append_paged_kv(k, v, Kc[layer], Vc[layer], table, lens, cu, max(prompts))
        for s in range(B):
            a, e = int(cu[s]), int(cu[s + 1])
            check(O[a:e], None, attend64(q[a:e], k[a:e], v[a:e], causal(e - a)))
            grow(layer, s, k[a:e], v[a:e])
    lens = new
    assert lens.tolist() == prompts

    # a second chunk of the prompt: causal within it, merged with the context before it
    chunk = [20, 3, 70]
    cu = offsets(chunk).to(DEV)
    for layer in range(LAYERS):
        q, k, v = (rand(g, sum(chunk), h, D) for h in (HQ, HKV, HKV))
        say("chunk", layer)
        O = merged(qa.prefix_attention_paged(q, Kc[layer], Vc[layer], table, lens, cu, max(chunk)),
                   qa.prompt_attention(q, k, v, cu, max(chunk), return_lse=True))
        new = qa.append_paged_kv(k, v, Kc[layer], Vc[layer], table, lens, cu, max(chunk))
        for s in range(B):
            a, e = int(cu[s]), int(cu[s + 1])
            pre = kept[layer][s][0].shape[0]
            grow(layer, s, k[a:e], v[a:e])
            mask = torch.cat([torch.ones(e - a, pre, dtype=torch.bool, device=DEV), causal(e - a)], 1)
            close(O[a:e], attend64(q[a:e], *kept[layer][s], mask), "chunk")
    lens = new

    # verified drafts: heap trees over the paged context, then the accepted path kept
    paths = torch.tensor([[0, 2, 5, 12], [0, 1, -1, -1], [0, 2, 6, -1]], dtype=torch.int32, device=DEV)
    steps = [4, 2, 3]
    cu = offsets([N] * B).to(DEV)
    anc = torch.zeros(N, N, dtype=torch.bool, device=DEV)
    for x in range(N):
        c = x
        while True:
            anc[x, c] = True
            if c == 0:
                break
            c = (c - 1) // b
    for step in range(2):
        rows = []
        for layer in range(LAYERS):
            q, k, v = (rand(g, B * N, h, D) for h in (HQ, HKV, HKV))
            say("verify", step, layer)
            O = merged(qa.prefix_attention_paged(q, Kc[layer], Vc[layer], table, lens, cu, N),
                       qa.ragged_attention_with_lse(q, k, v, cu, b, depth, N))
            drafted = qa.append_paged_kv(k, v, Kc[layer], Vc[layer], table, lens, cu, N)
            for s in range(B):
                at = slice(s * N, (s + 1) * N)
                ks, vs = kept[layer][s]
                mask = torch.cat([torch.ones(N, ks.shape[0], dtype=torch.bool, device=DEV), anc], 1)
                close(O[at], attend64(q[at], torch.cat([ks, k[at]]), torch.cat([vs, v[at]]), mask), "verify")
            rows.append((k, v))
        assert drafted.tolist() == [n + N for n in lens.tolist()]
        new = qa.compact_paged_kv(Kc, Vc, table, lens, paths)
        assert new.tolist() == [n + x for n, x in zip(lens.tolist(), steps)]
        lens = new
        for layer, (k, v) in enumerate(rows):
            for s in range(B):
                at = paths[s, :steps[s]].long() + s * N
                grow(layer, s, k[at], v[at])

    # decode steps, recorded once: the new row is appended, then attended with the rest
    Q, K, V = (rand(g, LAYERS, B, h, D) for h in (HQ, HKV, HKV))
    static = lens.clone()

    def decode():
        outs = []
        for layer in range(LAYERS):
            new = qa.append_paged_kv(K[layer], V[layer], Kc[layer], Vc[layer], table, static)
            outs.append(qa.prefix_attention_paged(Q[layer], Kc[layer], Vc[layer], table, new))
        static.copy_(new)
        return outs

    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        outs = decode()
    for step in range(4):
        for x in (Q, K, V):
            x.normal_(0, 1, generator=g)
        say("decode", step)
        graph.replay()
        for layer in range(LAYERS):
            for s in range(B):
                grow(layer, s, K[layer, s:s + 1], V[layer, s:s + 1])
                mask = torch.ones(1, kept[layer][s][0].shape[0], dtype=torch.bool, device=DEV)
                check(outs[layer][0][s:s + 1], outs[layer][1][s:s + 1],
                      attend64(Q[layer, s:s + 1], *kept[layer][s], mask))
    lens = static.clone()
    assert lens.tolist() == [kept[0][s][0].shape[0] for s in range(B)]

    # sequence 2 forked: full pages shared, the last one copied; both go on
    n = int(lens[2])
    full = n // PS
    assert n % PS
    own = table[3, full].clone()
    table[3, :full] = table[2, :full]
    say("fork")
    qa.copy_kv_pages(Kc, Vc, table[2, full:full + 1], own[None])
    lens = torch.cat([lens, lens[2:3]])
    for layer in range(LAYERS):
        q, k, v = (rand(g, B + 1, h, D) for h in (HQ, HKV, HKV))
        kept[layer].append(kept[layer][2])
        new = qa.append_paged_kv(k, v, Kc[layer], Vc[layer], table, lens)
        O, L = qa.prefix_attention_paged(q, Kc[layer], Vc[layer], table, new)
        for s in range(B + 1):
            grow(layer, s, k[s:s + 1], v[s:s + 1])
            mask = torch.ones(1, kept[layer][s][0].shape[0], dtype=torch.bool, device=DEV)
            check(O[s:s + 1], L[s:s + 1], attend64(q[s:s + 1], *kept[layer][s], mask))
    assert np.all(new.tolist() == lens.cpu().numpy() + 1)


def test_host_operands_are_taken_at_the_call():
    """Tables, lengths, offsets and paths on the host, pinned and not, that change while
    the stream is still busy ahead of the call."""
    import qattention_amd as qa
    g = torch.Generator(device=DEV).manual_seed(9)
    B, cols, toks = 3, 8, [4, 2, 3]
    Kc, Vc = (rand(g, B * cols, PS, HKV, D, dtype=torch.float16) for _ in range(2))
    Q, K, V = (rand(g, sum(toks), h, D, dtype=torch.float16) for h in (HQ, HKV, HKV))
    wide = torch.zeros(B, 300000, dtype=torch.int32)  # (some MB: not what a copy holds by the way)
    wide[:, :cols] = torch.arange(B * cols).view(B, cols)
    host = dict(table=wide, lens=torch.tensor([100, 3, 57], dtype=torch.int32),
                cu=offsets(toks).cpu(), path=torch.tensor([[0, 2], [1, 3], [2, -1]], dtype=torch.int32),
                src=torch.tensor([0, 9], dtype=torch.int32), dst=torch.tensor([7, 15], dtype=torch.int32))
    big = torch.ones(8192, 8192, dtype=torch.bfloat16, device=DEV)

    def step(o):
        kc, vc = Kc.clone(), Vc.clone()
        out = [*qa.prefix_attention_paged(Q, kc, vc, o["table"], o["lens"], o["cu"], 4),
               qa.prompt_attention(Q, K, V, o["cu"], 4),
               qa.append_paged_kv(K, V, kc, vc, o["table"], o["lens"], o["cu"], 4),
               qa.compact_paged_kv(kc, vc, o["table"], o["lens"], o["path"])]
        qa.copy_kv_pages(kc, vc, o["src"], o["dst"])
        return out + [kc, vc]

    want = step({n: t.to(DEV) for n, t in host.items()})
    for kind in ("pinned", "pageable"):
        o = {n: t.clone().pin_memory() if kind == "pinned" else t.clone() for n, t in host.items()}
        torch.cuda.synchronize()
        say("host operands", kind)
        for _ in range(30):
            big @ big
        got = step(o)
        for t in o.values():  # (other rows of the same tensors: nothing out of range either way)
            t.zero_()
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(got, want)):
            same = torch.equal(a, b)
            assert same, (kind, i)


def test_host_operands_stay_out_of_graphs():
    """A graph would read host memory at each replay, whatever it holds by then."""
    import qattention_amd as qa
    g = torch.Generator(device=DEV).manual_seed(10)
    Kc, Vc = (rand(g, 4, PS, HKV, D, dtype=torch.float16) for _ in range(2))
    Q, K, V = (rand(g, 2, h, D, dtype=torch.float16) for h in (HQ, HKV, HKV))
    table, lens, cu = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32), torch.tensor([5, 20]), offsets([1, 1]).cpu()
    dev = [t.to(DEV, torch.int32) for t in (table, lens, cu)]
    want = qa.prefix_attention_paged(Q, Kc, Vc, *dev, 1)
    calls = [lambda t=t, l=l, c=c: qa.prefix_attention_paged(Q, Kc, Vc, t, l, c, 1)
             for t, l, c in ((table, *dev[1:]), (dev[0], lens.pin_memory(), dev[2]), (*dev[:2], cu))]
    calls += [lambda: qa.prompt_attention(Q, K, V, cu, 1), lambda: qa.copy_kv_pages(Kc, Vc, [0], [1]),
              lambda: qa.append_paged_kv(K, V, Kc, Vc, dev[0], lens),
              lambda: qa.compact_paged_kv(Kc, Vc, dev[0], dev[1], torch.tensor([[0], [1]]))]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        for i, f in enumerate(calls):
            say("in a graph", i)
            with pytest.raises(RuntimeError, match="on the GPU while a graph is captured"):
                f()
        got = qa.prefix_attention_paged(Q, Kc, Vc, *dev, 1)
    for _ in range(3):
        graph.replay()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
