"""The calls over a quantised cache together, as a serving loop uses them: prompts in,
chunks and draft trees over the context, accepted paths kept, rows read back, single
tokens decoded in a graph, a sequence forked.  And the ways the calls are reached: the
call module and Python, host operands, graphs, other streams, two calls at once."""
from __future__ import annotations

import types

import pytest
import torch

import quant64
from attn64 import attend64, causal, check, offsets

pytestmark = pytest.mark.gpu
DEV = "cuda"
FP16, BF16 = torch.float16, torch.bfloat16
HQ, HKV, D, PS, LAYERS = 8, 2, 64, 16, 2


def say(*a):
    print(*a, flush=True)


def rand(g, *shape, dtype=BF16):
    return torch.empty(*shape, dtype=dtype, device=DEV).normal_(0, 1, generator=g)


def held(x, bits):
    """The values that rows x are kept as, in fp64."""
    return quant64.decode(*quant64.encode(x, bits), bits).to(DEV)


def merged(pre, tree):
    from qattention_amd import fused_lse_merge
    heads = lambda x: x.transpose(0, 1)[None]  # noqa: E731
    return fused_lse_merge(heads(pre[1]), heads(tree[1]), heads(pre[0]), heads(tree[0]))[0].transpose(0, 1)


def close(O, ref, what):
    """The merge rounds each half's output once more: one more half step of each."""
    o, _, to, _ = ref
    half = torch.finfo(O.dtype).eps / 2
    off = (O.double() - o).abs() - (3 * to + half * o.abs())
    assert float(off.max()) <= 0, (what, float(off.max()))


@pytest.mark.parametrize("bits,dtype", [(4, BF16), (8, FP16)])
def test_serving_loop(bits, dtype):
    import qattention_amd as qa
    g = torch.Generator(device=DEV).manual_seed(5)
    B, prompts, b, depth = 3, [45, 16, 130], 2, 3
    N, cols = 15, 16
    caches = qa.quantized_kv_cache((B + 1) * cols, PS, HKV, D, bits=bits, layers=LAYERS)
    for t in caches:
        t.fill_(255)  # no numbers
    table = torch.randperm((B + 1) * cols, generator=torch.Generator().manual_seed(6)).view(B + 1, cols)
    table = table.to(DEV, torch.int32)
    lens = torch.zeros(B, dtype=torch.int32, device=DEV)
    none = torch.zeros(0, HKV, D, dtype=torch.float64, device=DEV)
    kept = [[(none, none) for _ in range(B)] for _ in range(LAYERS)]
    half = lambda *h: tuple(rand(g, *x, dtype=dtype) for x in h)  # noqa: E731

    def grow(layer, s, k, v):
        a, c = kept[layer][s]
        kept[layer][s] = torch.cat([a, held(k, bits)]), torch.cat([c, held(v, bits)])

    def read_back(layer, lens, upto):
        """Everything a sequence holds, exactly."""
        cu = offsets(upto)
        K, V = qa.read_quantized_kv(caches.layer(layer), table[:len(upto)], torch.zeros_like(lens), cu, dtype=dtype)
        for s in range(len(upto)):
            for x, want in zip((K, V), kept[layer][s]):
                assert torch.equal(x[int(cu[s]):int(cu[s + 1])].double(), want)

    # prompts
    cu = offsets(prompts).to(DEV)
    for layer in range(LAYERS):
        q, k, v = half(*((sum(prompts), h, D) for h in (HQ, HKV, HKV)))
        say("prompt", layer)
        O = qa.prompt_attention(q, k, v, cu, max(prompts))
        new = qa.append_quantized_kv(k, v, caches.layer(layer), table, lens, cu, max(prompts))
        for s in range(B):
            a, e = int(cu[s]), int(cu[s + 1])
            check(O[a:e], None, attend64(q[a:e], k[a:e], v[a:e], causal(e - a)))
            grow(layer, s, k[a:e], v[a:e])
        read_back(layer, new, prompts)
    lens = new
    assert lens.tolist() == prompts

    # a second chunk of the prompt: causal within it, merged with the context before it
    chunk = [20, 3, 70]
    cu = offsets(chunk).to(DEV)
    for layer in range(LAYERS):
        q, k, v = half(*((sum(chunk), h, D) for h in (HQ, HKV, HKV)))
        say("chunk", layer)
        O = merged(qa.prefix_attention_quantized(q, caches.layer(layer), table, lens, cu, max(chunk)),
                   qa.prompt_attention(q, k, v, cu, max(chunk), return_lse=True))
        new = qa.append_quantized_kv(k, v, caches.layer(layer), table, lens, cu, max(chunk))
        for s in range(B):
            a, e = int(cu[s]), int(cu[s + 1])
            ks, vs = kept[layer][s]
            mask = torch.cat([torch.ones(e - a, ks.shape[0], dtype=torch.bool, device=DEV), causal(e - a)], 1)
            close(O[a:e], attend64(q[a:e], torch.cat([ks, k[a:e].double()]), torch.cat([vs, v[a:e].double()]), mask),
                  "chunk")
            grow(layer, s, k[a:e], v[a:e])
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
            q, k, v = half(*((B * N, h, D) for h in (HQ, HKV, HKV)))
            say("verify", step, layer)
            O = merged(qa.prefix_attention_quantized(q, caches.layer(layer), table, lens, cu, N),
                       qa.ragged_attention_with_lse(q, k, v, cu, b, depth, N))
            drafted = qa.append_quantized_kv(k, v, caches.layer(layer), table, lens, cu, N)
            for s in range(B):
                at = slice(s * N, (s + 1) * N)
                ks, vs = kept[layer][s]
                mask = torch.cat([torch.ones(N, ks.shape[0], dtype=torch.bool, device=DEV), anc], 1)
                close(O[at], attend64(q[at], torch.cat([ks, k[at].double()]), torch.cat([vs, v[at].double()]), mask),
                      "verify")
            rows.append((k, v))
        assert drafted.tolist() == [n + N for n in lens.tolist()]
        new = qa.compact_paged_kv(caches.K, caches.V, table, lens, paths)
        assert torch.equal(qa.compact_paged_kv(caches.K_scale, caches.V_scale, table, lens, paths), new)
        assert new.tolist() == [n + x for n, x in zip(lens.tolist(), steps)]
        lens = new
        for layer, (k, v) in enumerate(rows):
            for s in range(B):
                at = paths[s, :steps[s]].long() + s * N
                grow(layer, s, k[at], v[at])
            read_back(layer, lens, lens.tolist())

    # decode steps, recorded once: the new row is appended, then attended with the rest
    Q, K, V = half(*((LAYERS, B, h, D) for h in (HQ, HKV, HKV)))
    static = lens.clone()

    def decode():
        outs = []
        for layer in range(LAYERS):
            new = qa.append_quantized_kv(K[layer], V[layer], caches.layer(layer), table, static)
            outs.append(qa.prefix_attention_quantized(Q[layer], caches.layer(layer), table, new))
            outs[-1] += qa.read_quantized_kv(caches.layer(layer), table, static, dtype=dtype)
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
            O, L, k, v = outs[layer]
            for s in range(B):
                grow(layer, s, K[layer, s:s + 1], V[layer, s:s + 1])
                ks, vs = kept[layer][s]
                mask = torch.ones(1, ks.shape[0], dtype=torch.bool, device=DEV)
                check(O[s:s + 1], L[s:s + 1], attend64(Q[layer, s:s + 1], ks, vs, mask))
                assert torch.equal(k[s].double(), ks[-1]) and torch.equal(v[s].double(), vs[-1])
    lens = static.clone()
    assert lens.tolist() == [kept[0][s][0].shape[0] for s in range(B)]

    # sequence 2 forked: full pages shared, the last one copied; both go on
    full = int(lens[2]) // PS
    assert int(lens[2]) % PS
    own = table[3, full].clone()
    table[3, :full] = table[2, :full]
    say("fork")
    for k, v in ((caches.K, caches.V), (caches.K_scale, caches.V_scale)):
        qa.copy_kv_pages(k, v, table[2, full:full + 1], own[None])
    lens = torch.cat([lens, lens[2:3]])
    for layer in range(LAYERS):
        q, k, v = half(*((B + 1, h, D) for h in (HQ, HKV, HKV)))
        kept[layer].append(kept[layer][2])
        new = qa.append_quantized_kv(k, v, caches.layer(layer), table, lens)
        O, L = qa.prefix_attention_quantized(q, caches.layer(layer), table, new)
        for s in range(B + 1):
            grow(layer, s, k[s:s + 1], v[s:s + 1])
            mask = torch.ones(1, kept[layer][s][0].shape[0], dtype=torch.bool, device=DEV)
            check(O[s:s + 1], L[s:s + 1], attend64(q[s:s + 1], *kept[layer][s], mask))
        read_back(layer, new, new.tolist())


# ---------------------------------------------------------------------------
# the ways the calls are reached
# ---------------------------------------------------------------------------

def operands(bits, dtype=FP16):
    import qattention_amd as qa
    g = torch.Generator(device=DEV).manual_seed(3)
    o = dict(Q=rand(g, 50, HQ, D, dtype=dtype), K=rand(g, 50, HKV, D, dtype=dtype), V=rand(g, 50, HKV, D, dtype=dtype))
    o["cache"] = qa.quantized_kv_cache(12, PS, HKV, D, bits=bits, layers=2)
    for t in o["cache"]:
        t.random_(120, 127, generator=g)  # (scales near 1; 127 is e4m3's NaN, which equals nothing)
    o["cu"] = offsets([20, 30]).to(DEV)
    o["table"] = torch.randperm(12, generator=torch.Generator().manual_seed(4)).to(DEV, torch.int32).view(2, 6)
    o["ctx"] = torch.tensor([33, 60], dtype=torch.int32, device=DEV)
    o["path"] = torch.tensor([[0, 2, 5], [1, 3, -1]], dtype=torch.int32, device=DEV)
    o["src"], o["dst"] = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([0, 1], [7, 8]))
    return o


def all_calls(o):
    import qattention_amd as qa
    c = qa.QuantizedKV(*(t.clone() for t in o["cache"]))
    a, b = c.layer(0), c.layer(1)
    out = [qa.prefix_attention_quantized(o["Q"][:2], a, o["table"], o["ctx"], return_lse=False),
           *qa.prefix_attention_quantized(o["Q"], b, o["table"], o["ctx"], o["cu"], 30),
           qa.append_quantized_kv(o["K"], o["V"], a, o["table"], o["ctx"], o["cu"], 30),
           qa.append_quantized_kv(o["K"][:2], o["V"][:2], b, o["table"], o["ctx"]),
           *qa.read_quantized_kv(a, o["table"], o["ctx"], o["cu"], 30, 50, dtype=o["K"].dtype),
           *qa.read_quantized_kv(b, o["table"], o["ctx"]),
           qa.compact_paged_kv(c.K, c.V, o["table"], o["ctx"], o["path"]),
           qa.compact_paged_kv(a.K_scale, a.V_scale, o["table"], o["ctx"], o["path"])]
    qa.copy_kv_pages(c.K, c.V, o["src"], o["dst"])
    qa.copy_kv_pages(b.K_scale, b.V_scale, o["dst"], o["src"])
    return out + list(c)


def equal(got, want):
    for i, (a, b) in enumerate(zip(got, want)):
        assert a.dtype == b.dtype and a.shape == b.shape and a.stride() == b.stride() and torch.equal(a, b), i


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [FP16, BF16])
def test_same_as_in_python(monkeypatch, dtype, bits):
    from qattention_amd import _lib
    o = operands(bits, dtype)
    all_calls(o)  # (the device is set up)
    say("direct", bits, dtype)
    direct = all_calls(o)
    c = _lib.calls()
    cache = o["cache"].layer(0)
    assert c.quant_paged(o["Q"][:2], cache, o["table"], o["ctx"], None, None, True) is not None
    assert c.quant_append(o["K"][:2], o["V"][:2], cache, o["table"], o["ctx"], None, None) is not None
    assert c.quant_read(cache, o["table"], o["ctx"], o["cu"], 30, 50, FP16) is not None
    assert c.compact(o["cache"].K, o["cache"].V, o["table"], o["ctx"], o["path"]) is not None
    assert c.copy(cache.K_scale, cache.V_scale, o["src"], o["dst"]) is True
    o = operands(bits, dtype)
    names = ("compact", "copy", "quant_append", "quant_read", "quant_paged")
    monkeypatch.setattr(_lib, "_calls", types.SimpleNamespace(**{n: lambda *a: None for n in names},
                                                              set_ready=lambda d: None))
    say("python", bits, dtype)
    equal(direct, all_calls(o))


def test_same_without_the_call_module(tmp_path, monkeypatch):
    from qattention_amd import _lib
    o = operands(4)
    direct = all_calls(o)
    monkeypatch.setattr(_lib, "CALLS_PATH", str(tmp_path / "_calls.so"))
    monkeypatch.setattr(_lib, "_calls", None)
    say("no module")
    with pytest.warns(RuntimeWarning, match="go through Python"):
        python = all_calls(o)
    equal(direct, python)


def test_leaves_the_rest_to_python():
    """Operands that need a copy, a conversion or an error, one at a time."""
    from qattention_amd import _lib
    all_calls(operands(4))
    c, o = _lib.calls(), operands(4)
    caches = o["cache"]
    before = [t.clone() for t in caches]
    q = caches.layer(0)
    odd = torch.zeros(50, HQ, D + 1, dtype=FP16, device=DEV)[..., 1:]
    bad = (caches, q[:3], list(q), None, (*q[:3], None), (*q[:3], q.V_scale.cpu()), q._replace(K=q.K.view(torch.int8)),
           q._replace(V=q.V[:5]), q._replace(K_scale=q.K_scale[..., :1]), q._replace(K=q.K[..., :16], V=q.V[..., :16]),
           q._replace(K=q.K[..., ::2], V=q.V[..., ::2]), q._replace(K=q.K.transpose(1, 2).contiguous().transpose(1, 2)),
           q._replace(K=torch.zeros(12, PS, HKV, 33, dtype=torch.uint8, device=DEV)[..., 1:]))
    paged = dict(Q=o["Q"], cache=q, table=o["table"], ctx=o["ctx"], cu=o["cu"], ms=30, lse=True)
    for i, kw in enumerate([dict(cache=x) for x in bad] + [
            dict(Q=odd), dict(Q=o["Q"].cpu()), dict(Q=o["Q"].float()), dict(Q=o["Q"][:, :7]), dict(Q=None),
            dict(Q=o["Q"].clone().requires_grad_()), dict(table=o["table"].cpu()), dict(table=o["table"][:, ::2]),
            dict(table=o["table"][:1]), dict(ctx=o["ctx"].long()), dict(cu=None), dict(cu=o["cu"][:2]),
            dict(cu=o["cu"].cpu()), dict(ms=None), dict(ms=-1), dict(ms=1 << 40), dict(ms=30.0), dict(lse=1)]):
        say("attend", i)
        assert c.quant_paged(*{**paged, **kw}.values()) is None
    append = dict(K=o["K"], V=o["V"], cache=q, table=o["table"], ctx=o["ctx"], cu=o["cu"], ms=30)
    for i, kw in enumerate([dict(cache=x) for x in bad] + [
            dict(cache=q._replace(V=q.K)), dict(cache=q._replace(K_scale=q.V_scale)),
            dict(cache=type(q)(*(t[:1].expand(12, -1, -1, -1) for t in q))), dict(K=o["K"][:, :1]), dict(cu=None),
            dict(K=o["K"].cpu()), dict(V=o["V"].bfloat16()), dict(V=o["V"][:40]),
            dict(K=o["K"].clone().requires_grad_())]):
        say("append", i)
        assert c.quant_append(*{**append, **kw}.values()) is None
    read = dict(cache=q, table=o["table"], start=o["ctx"], cu=o["cu"], ms=30, total=50, dtype=FP16)
    for i, kw in enumerate([dict(cache=x) for x in bad] + [
            dict(total=None), dict(total=-1), dict(total=1 << 31), dict(total=50.0), dict(cu=None), dict(dtype=None),
            dict(dtype=torch.float32), dict(table=o["table"].cpu()), dict(start=o["ctx"].long()), dict(ms=None)]):
        say("read", i)
        assert c.quant_read(*{**read, **kw}.values()) is None
    assert c.quant_read() is None and c.quant_append(1, 2, 3, 4, 5, 6, 7) is None
    for kw in (dict(a=q.K, b=q.K), dict(a=q.K, b=q.V_scale), dict(a=q.K[..., ::2], b=q.V[..., ::2])):
        assert c.copy(*kw.values(), o["src"], o["dst"]) is None
    with pytest.raises(TypeError):
        c.bind_quantized(1, 2)
    equal(caches, before)


def test_gradients_and_tangents_are_refused():
    import torch.autograd.forward_ad as fwd
    import qattention_amd as qa
    o = operands(4)
    q = o["cache"].layer(0)
    before = [t.clone() for t in q]
    calls = [(qa.prefix_attention_quantized, [o["Q"][:2]], [q, o["table"], o["ctx"]]),
             (qa.append_quantized_kv, [o["K"][:2], o["V"][:2]], [q, o["table"], o["ctx"]])]
    for f, ts, rest in calls:
        for i in range(len(ts)):
            say("gradients", f.__name__, i)
            with pytest.raises(RuntimeError):
                f(*[t.clone().requires_grad_() if j == i else t for j, t in enumerate(ts)], *rest)
            with fwd.dual_level(), pytest.raises(RuntimeError, match="no forward derivative"):
                f(*[fwd.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(ts)], *rest)
    equal(q, before)


def test_host_operands_are_taken_at_the_call():
    """Tables, lengths and offsets on the host, pinned and not, that change while the
    stream is still busy ahead of the call."""
    import qattention_amd as qa
    g = torch.Generator(device=DEV).manual_seed(9)
    B, cols, toks = 3, 8, [4, 2, 3]
    base = qa.quantized_kv_cache(B * cols, PS, HKV, D)
    for t in base:
        t.random_(120, 127, generator=g)
    Q, K, V = (rand(g, sum(toks), h, D, dtype=FP16) for h in (HQ, HKV, HKV))
    wide = torch.zeros(B, 300000, dtype=torch.int32)  # (some MB: not what a copy holds by the way)
    wide[:, :cols] = torch.arange(B * cols).view(B, cols)
    host = dict(table=wide, lens=torch.tensor([100, 3, 57], dtype=torch.int32), cu=offsets(toks).cpu())
    big = torch.ones(8192, 8192, dtype=BF16, device=DEV)

    def step(o):
        c = qa.QuantizedKV(*(t.clone() for t in base))
        return [*qa.prefix_attention_quantized(Q, c, o["table"], o["lens"], o["cu"], 4),
                qa.append_quantized_kv(K, V, c, o["table"], o["lens"], o["cu"], 4),
                *qa.read_quantized_kv(c, o["table"], o["lens"], o["cu"], 4, 9), *c]

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
        equal(got, want)


def test_host_operands_stay_out_of_graphs():
    import qattention_amd as qa
    o = operands(8)
    c = o["cache"].layer(0)
    table, lens, cu = (o[n].cpu() for n in ("table", "ctx", "cu"))
    Q, K, V = o["Q"], o["K"], o["V"]
    dev = o["table"], o["ctx"], o["cu"]
    want = qa.prefix_attention_quantized(Q, c, *dev, 30)
    back = qa.read_quantized_kv(c, *dev, 30, 50)
    calls = [lambda t=t, l=l, c_=c_: qa.prefix_attention_quantized(Q, c, t, l, c_, 30)
             for t, l, c_ in ((table, *dev[1:]), (dev[0], lens.pin_memory(), dev[2]), (*dev[:2], cu))]
    calls += [lambda: qa.append_quantized_kv(K[:2], V[:2], c, dev[0], lens),
              lambda: qa.read_quantized_kv(c, table, dev[1]), lambda: qa.read_quantized_kv(c, *dev[:2], cu, 30, 50)]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        for i, f in enumerate(calls):
            say("in a graph", i)
            with pytest.raises(RuntimeError, match="on the GPU while a graph is captured"):
                f()
        got = qa.prefix_attention_quantized(Q, c, *dev, 30)
        rows = qa.read_quantized_kv(c, *dev, 30, 50)
    for _ in range(3):
        graph.replay()
        equal((*got, *rows), (*want, *back))


def cut(seed, B, n, ctx, Hq=16, Hkv=2, bits=4):
    """A call whose contexts are cut between workgroups (it has a workspace)."""
    import qattention_amd as qa
    g = torch.Generator(device=DEV).manual_seed(seed)
    cols = -(-ctx // PS)
    c = qa.quantized_kv_cache(B * cols, PS, Hkv, 128, bits=bits)
    for t in c:
        t.random_(118, 127, generator=g)
    table = torch.randperm(B * cols, generator=torch.Generator().manual_seed(seed)).to(DEV, torch.int32).view(B, cols)
    lens = torch.full((B,), ctx - 5, dtype=torch.int32, device=DEV)
    Q = rand(g, B * n, Hq, 128, dtype=FP16)
    cu = torch.arange(0, B * n + 1, n, dtype=torch.int32, device=DEV)
    return lambda: qa.prefix_attention_quantized(Q, c, table, lens, cu, n)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("n", [1, 40])
def test_streams_and_graphs_side_by_side(n, bits):
    """Calls with workspaces: on a stream of their own, two at once, in two graphs that
    replay in turn and at once."""
    calls = [cut(i, 5 - i, n, 3000 + 777 * i, bits=bits) for i in range(2)]
    want = [f() for f in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    say("streams", n, bits)
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(calls[i]())
    torch.cuda.synchronize()
    for i in range(2):
        for x in got[i]:
            equal(x, want[i])
    say("graphs", n, bits)
    graphs, outs = [], []
    for f in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(f())
    for round_ in range(4):
        for o in outs:
            for x in o:
                x.zero_()
        torch.cuda.synchronize()
        for i, s in enumerate(streams):
            with torch.cuda.stream(s if round_ % 2 else torch.cuda.current_stream()):
                graphs[i].replay()
        eager = calls[0]()
        torch.cuda.synchronize()
        equal(eager, want[0])
        for i in range(2):
            equal(outs[i], want[i])


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("n", [1, 3, 40])
def test_rows_of_no_sequence_stay(n, bits):
    """Rows behind the last sequence, and those past max_seqlen, as the output held them:
    written to a buffer that was filled before, through the library's own call."""
    import math
    from qattention_amd import _lib, quantized_kv
    import qattention_amd as qa
    o = operands(bits)
    c = o["cache"].layer(0)
    T = 2 * n + 7
    g = torch.Generator(device=DEV).manual_seed(21)
    Q = rand(g, T, HQ, D, dtype=FP16)
    cu = torch.tensor([0, n, 2 * n], dtype=torch.int32, device=DEV)
    want = qa.prefix_attention_quantized(Q[:2 * n], c, o["table"], o["ctx"], cu, n)
    *_, b, at = quantized_kv._check_cache(c, False)
    L = _lib.lib()
    for ms in (n, max(n - 1, 1)):
        O, lse = torch.full_like(Q, 7.0), torch.full((T, HQ), 7.0, device=DEV)
        st, ls = _lib.layout(Q.stride())[0], _lib.layout(lse.stride())[0]
        bytes_ = L.qattn_prefix_quant_workspace_bytes(2, ms, T, HQ, HKV, D, 6, PS, b)
        ws = torch.empty(bytes_, dtype=torch.uint8, device=DEV) if bytes_ else None
        say("rows", n, bits, ms)
        assert L.qattn_prefix_quant_fwd(
            Q.data_ptr(), st, *at, o["table"].data_ptr(), 6, 12, PS, o["ctx"].data_ptr(), O.data_ptr(), st,
            lse.data_ptr(), ls, cu.data_ptr(), 2, ms, T, HQ, HKV, D, 1 / math.sqrt(D), 0, b, _lib.ptr(ws), bytes_,
            torch.cuda.current_stream().cuda_stream) == 0
        rows = torch.arange(T, device=DEV)
        mine = (rows < 2 * n) & (rows % n < ms)
        assert torch.equal(O[mine], want[0][mine[:2 * n]]) and torch.equal(lse[mine], want[1][mine[:2 * n]])
        assert bool((O[~mine] == 7).all()) and bool((lse[~mine] == 7).all())
