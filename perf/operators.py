"""Measured cases of the serving operators around tree verification.

  op       prompt   causal attention over packed prompts (lse: the log-sum-exp is asked for too)
           paged    attention of each sequence's query tokens over its context in a paged K/V cache, O and LSE:
                    n = 1 token per sequence (a decode step) or n draft nodes (the context half of a verification)
           append   the new K/V rows of a layer stored in the pages behind each context
           compact  the rows of the accepted draft path moved together behind each context, in every layer
           copy     whole pages copied inside the cache (the shared last page of forked sequences), in every layer
  B        sequences; L their prompt length or context (the longest where they are ragged); n rows per sequence
           (query tokens, new rows, steps of the path, pages to copy); N nodes of the draft tree (compact)
  layers   layers of the cache (compact, copy)
  Hq, Hkv, D, page, dtype, ragged

Inputs are N(0, 1) of the case's element type; pages lie in shuffled physical order, the slots behind a
context hold other numbers of the same kind.
"""
from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"


def _case(name=None, **kw):
    c = dict(op="prompt", B=1, L=512, n=1, N=0, layers=1, Hq=32, Hkv=8, D=128, page=16, dtype="fp16", ragged=False,
             lse=False)
    c.update(kw)
    return dict(name=name, **c) if name else c


def listed():
    return [
        # a few short chat turns of odd lengths, each far below a tile of anything: latency counts
        _case("prompt_short", B=4, L=93, ragged=True),
        # a batch of ordinary prompts, no two of one length, 64-wide heads, with the LSE that a merge
        # with an earlier chunk needs
        _case("prompt_batch_lse", B=16, L=2011, D=64, dtype="bf16", ragged=True, lse=True),
        # one long document
        _case("prompt_long", B=1, L=16384, dtype="bf16"),
        # a decode step of two young conversations
        _case("decode_small", op="paged", B=2, L=731, ragged=True),
        # a decode step of a large batch whose contexts differ by a factor of three
        _case("decode_batch", op="paged", B=64, L=16000, dtype="bf16", ragged=True),
        # the context half of verifying 60-node drafts over long contexts
        _case("verify_tree", op="paged", B=4, L=10240, n=60),
        # one layer's new rows of a decode step
        _case("append_step", op="append", B=32, L=2000, n=1, ragged=True),
        # one layer's rows of long prompts, from the first page on or behind an earlier chunk
        _case("append_prompt", op="append", B=8, L=500, n=4003, dtype="bf16"),
        # the path kept of one verified 60-node draft, 32 layers
        _case("compact_one", op="compact", B=1, L=1000, n=6, N=60, layers=32),
        # the same for a batch
        _case("compact_batch", op="compact", B=48, L=100, n=8, N=60, layers=32, dtype="bf16", ragged=True),
        # two forks of one conversation: a page each, in 32 layers
        _case("fork_pages", op="copy", B=2, L=320, n=1, layers=32),
        # beams exchanged across a batch: many pages
        _case("copy_pages", op="copy", B=32, L=320, n=8, layers=16, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges, no dearer than the largest listed."""
    while True:
        op = rng.choice(["prompt", "prompt", "prompt", "paged", "paged", "paged", "append", "compact", "copy"])
        Hkv = rng.choice([4, 8, 32])
        Hq = 32 if Hkv != 4 else rng.choice([4, 32])
        c = _case(op=op, Hq=Hq, Hkv=Hkv, D=rng.choice([64, 128, 128]), dtype=rng.choice(["fp16", "bf16"]),
                  page=rng.choice([16, 16, 32, 64]), ragged=rng.random() < 0.6)
        if op == "prompt":
            c.update(B=_log(rng, 1, 32), L=_log(rng, 30, 16384), lse=rng.random() < 0.4)
            if c["B"] * c["Hq"] * c["L"] ** 2 > 32 * 16384 ** 2:  # what the plain form's score matrix takes
                continue
        elif op == "paged":
            c.update(B=_log(rng, 1, 64), L=_log(rng, 60, 131072), n=rng.choice([1, 1, 1, _log(rng, 2, 100)]))
            if c["B"] * c["L"] * c["Hkv"] * c["D"] > 64 * 16000 * 8 * 128 or c["B"] * c["n"] * c["L"] > 4 * 60 * 10240:
                continue
        elif op == "append":
            c.update(B=_log(rng, 1, 64), L=_log(rng, 30, 4000), n=rng.choice([1, _log(rng, 2, 8000)]))
            if c["B"] * (c["L"] + c["n"]) * c["Hkv"] * c["D"] > 8 * 4503 * 32 * 128:
                continue
        elif op == "compact":
            N = _log(rng, 15, 120)
            c.update(B=_log(rng, 1, 48), L=_log(rng, 30, 1000), N=N, n=rng.randint(3, 9), layers=rng.choice([8, 32]))
        else:
            c.update(B=_log(rng, 1, 32), L=_log(rng, 160, 1000), n=rng.randint(1, 8), layers=rng.choice([8, 32]))
            c.update(L=max(c["L"], c["n"] * c["page"]), ragged=False)
        if op in ("compact", "copy") and c["layers"] * c["B"] * (c["L"] + c["N"]) * Hkv * c["D"] > 5e8:
            continue
        w = work(c)
        if w["bytes"] <= 2.9e9 and w["flops"] <= 2.3e12:
            return c


# ---------------------------------------------------------------------------
# shapes
# ---------------------------------------------------------------------------

def _lens(c):
    """Length per sequence: L each, or spread over [0.3 L, L] in a fixed order."""
    B, L = c["B"], c["L"]
    if not c["ragged"] or B == 1:
        return [L] * B
    return [max(1, L - (L * 7 * ((5 * i) % B)) // (10 * B)) for i in range(B)]


def _steps(c):
    """Accepted nodes per sequence: between one and n."""
    return [1 + (3 * i + c["n"] - 1) % c["n"] for i in range(c["B"])]


def _dtype(c):
    return torch.bfloat16 if c["dtype"] == "bf16" else torch.float16


def _pages(c):
    """Pages of each sequence: its context and what is put behind it."""
    more = {"append": c["n"], "compact": c["N"], "copy": 0, "paged": 0}[c["op"]]
    return [-(-(n + more) // c["page"]) for n in _lens(c)]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def prepare(case, seed):
    c, g = case, torch.Generator(device=DEV).manual_seed(int(seed))
    dt, B, Hq, Hkv, D = _dtype(c), c["B"], c["Hq"], c["Hkv"], c["D"]
    lens, n, op = _lens(c), c["n"], c["op"]

    def rand(*shape):
        return torch.empty(shape, dtype=dt, device=DEV).normal_(0.0, 1.0, generator=g)

    s = {"c": c}
    if op == "prompt":
        T = sum(lens)
        s.update(Q=rand(T, Hq, D), K=rand(T, Hkv, D), V=rand(T, Hkv, D), max=max(lens))
        s["cu"] = torch.tensor([0] + lens).cumsum(0).to(device=DEV, dtype=torch.int32)
        return s
    pages = _pages(c)
    spare = B * n if op == "copy" else 0
    total = sum(pages) + spare
    shape = (total, c["page"], Hkv, D)
    if op in ("compact", "copy"):
        shape = (c["layers"],) + shape
    s["Kc"], s["Vc"] = rand(*shape), rand(*shape)
    order = torch.randperm(total, generator=g, device=DEV, dtype=torch.int32)
    table = torch.zeros(B, max(pages), dtype=torch.int32)
    first = torch.tensor([0] + pages).cumsum(0)
    col = torch.arange(max(pages))[None, :]
    at = (first[:-1, None] + col).clamp(max=total - 1).to(DEV)
    s["table"] = torch.where((col < torch.tensor(pages)[:, None]).to(DEV), order[at.long()], table.to(DEV))
    s["ctx"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    if op == "paged":
        s["Q"] = rand(B * n, Hq, D)
    elif op == "append":
        s["K"], s["V"] = rand(B * n, Hkv, D), rand(B * n, Hkv, D)
    elif op == "compact":
        # a path: the root, then one node per step further down the breadth-first order
        gaps = torch.randint(1, max(2, (c["N"] - 1) // max(1, n - 1)), (B, n), generator=g, device=DEV)
        gaps[:, 0] = 0
        path = gaps.cumsum(1).to(torch.int32)
        past = torch.arange(n, device=DEV)[None, :] >= torch.tensor(_steps(c), device=DEV)[:, None]
        s["path"] = path.masked_fill(past, -1)
    else:
        s["src"] = s["table"][:, :n].reshape(-1).contiguous()
        s["dst"] = order[sum(pages):].contiguous()
    if op in ("paged", "append") and n > 1:
        s["cu"] = torch.arange(0, (B + 1) * n, n, dtype=torch.int32, device=DEV)
        s["max"] = n
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    s, op = state, state["c"]["op"]
    if own:
        return _own(s, op)
    return {"prompt": _prompt, "paged": _paged, "append": _append, "compact": _compact, "copy": _copy}[op](s)


def _own(s, op):
    import qattention_amd as qa

    if op == "prompt":
        return qa.prompt_attention(s["Q"], s["K"], s["V"], s["cu"], max_seqlen=s["max"], return_lse=s["c"]["lse"])
    if op == "paged":
        return qa.prefix_attention_paged(s["Q"], s["Kc"], s["Vc"], s["table"], s["ctx"], cu_seqlens=s.get("cu"),
                                         max_seqlen=s.get("max"))
    if op == "append":
        return s["Kc"], s["Vc"], qa.append_paged_kv(s["K"], s["V"], s["Kc"], s["Vc"], s["table"], s["ctx"],
                                                    cu_seqlens=s.get("cu"), max_seqlen=s.get("max"))
    if op == "compact":
        return s["Kc"], s["Vc"], qa.compact_paged_kv(s["Kc"], s["Vc"], s["table"], s["ctx"], s["path"])
    qa.copy_kv_pages(s["Kc"], s["Vc"], s["src"], s["dst"])
    return s["Kc"], s["Vc"]


def _softmax_rows(x, dead):
    """exp(x - max) with the dead places at 0, the rows' sums and their log-sum-exp (x is overwritten)."""
    x.masked_fill_(dead, -math.inf)
    m = x.amax(-1, keepdim=True)
    x.sub_(m).exp_()
    z = x.sum(-1, keepdim=True)
    return x, z, (m + z.log()).squeeze(-1)


def _prompt(s):
    """Prompts padded to the longest: softmax(Q K^T / sqrt(D) + causal mask) V in fp32."""
    c, cu = s["c"], s["cu"].long()
    B, L, Hq, Hkv, D = c["B"], s["max"], c["Hq"], c["Hkv"], c["D"]
    T, i = s["Q"].shape[0], torch.arange(s["max"], device=DEV)
    tok = (cu[:-1, None] + i).clamp(max=T - 1)

    def heads(x):  # [B, H, L, D], each kv head once per q head that reads it
        return x[tok].float().repeat_interleave(Hq // x.shape[1], 2).transpose(1, 2)

    score = torch.matmul(heads(s["Q"]) / math.sqrt(D), heads(s["K"]).transpose(-1, -2))
    p, z, lse = _softmax_rows(score, i[None, :] > i[:, None])
    o = torch.matmul(p, heads(s["V"])) / z
    t = torch.arange(T, device=DEV)
    seq = torch.searchsorted(cu[1:], t, right=True)
    at = t - cu[seq]
    O = o[seq, :, at].to(s["Q"].dtype)
    return (O, lse[seq, :, at]) if c["lse"] else O


def _paged(s):
    """Each sequence's pages gathered: softmax(Q K^T / sqrt(D) + length mask) V in fp32."""
    c, table = s["c"], s["table"].long()
    B, n, Hq, Hkv, D = c["B"], c["n"], c["Hq"], c["Hkv"], c["D"]

    def rows(x):  # [B, Hkv, rows, D]
        return x[table].flatten(1, 2).transpose(1, 2).float()

    q = s["Q"].float().view(B, n, Hkv, Hq // Hkv, D).permute(0, 2, 1, 3, 4).flatten(2, 3) / math.sqrt(D)
    score = torch.matmul(q, rows(s["Kc"]).transpose(-1, -2))
    j = torch.arange(score.shape[-1], device=DEV)
    p, z, lse = _softmax_rows(score, (j[None, :] >= s["ctx"][:, None])[:, None, None, :])
    o = torch.matmul(p, rows(s["Vc"])) / z
    O = o.view(B, Hkv, n, Hq // Hkv, D).permute(0, 2, 1, 3, 4).reshape(B * n, Hq, D).to(s["Q"].dtype)
    return O, lse.view(B, Hkv, n, Hq // Hkv).permute(0, 2, 1, 3).reshape(B * n, Hq)


def _append(s):
    n, page = s["c"]["n"], s["c"]["page"]
    pos = s["ctx"].long()[:, None] + torch.arange(n, device=DEV)
    at = s["table"].long().gather(1, pos // page), pos % page
    for_layer = (s["c"]["B"], n) + s["K"].shape[1:]
    s["Kc"][at], s["Vc"][at] = s["K"].view(for_layer), s["V"].view(for_layer)
    return s["Kc"], s["Vc"], s["ctx"] + n


def _compact(s):
    page, path = s["c"]["page"], s["path"].long()
    kept = path >= 0
    dst = s["ctx"].long()[:, None] + torch.arange(path.shape[1], device=DEV)
    src = torch.where(kept, s["ctx"].long()[:, None] + path, dst)  # past the path: a row onto itself
    table = s["table"].long()
    to, of = (table.gather(1, dst // page), dst % page), (table.gather(1, src // page), src % page)
    s["Kc"][:, to[0], to[1]] = s["Kc"][:, of[0], of[1]]
    s["Vc"][:, to[0], to[1]] = s["Vc"][:, of[0], of[1]]
    return s["Kc"], s["Vc"], s["ctx"] + kept.sum(1, dtype=torch.int32)


def _copy(s):
    src, dst = s["src"].long(), s["dst"].long()
    s["Kc"][:, dst] = s["Kc"][:, src]
    s["Vc"][:, dst] = s["Vc"][:, src]
    return s["Kc"], s["Vc"]


# ---------------------------------------------------------------------------
# the definition in 64 bits, sequence by sequence
# ---------------------------------------------------------------------------

def _attend64(q, k, v, first):
    """q [a, D] over k, v [b, D]: row i attends keys j < first + i + 1 (first None: all of them)."""
    o, lse = torch.empty_like(q), q.new_empty(q.shape[0])
    step = max(1, (1 << 27) // max(1, k.shape[0]))
    for a in range(0, q.shape[0], step):
        b = min(a + step, q.shape[0])
        end = k.shape[0] if first is None else first + b
        w = q[a:b] @ k[:end].T / math.sqrt(q.shape[1])
        if first is not None:
            w = w.masked_fill(torch.ones_like(w, dtype=torch.bool).triu(first + a + 1), -math.inf)
        lse[a:b] = torch.logsumexp(w, 1)
        o[a:b] = torch.exp(w - lse[a:b, None]) @ v[:end]
    return o, lse


def exact(case, seed):
    c, s = case, prepare(case, seed)
    group, op, lens = c["Hq"] // c["Hkv"], c["op"], _lens(c)
    if op == "prompt":
        O, S = torch.empty_like(s["Q"], dtype=torch.float64), s["Q"].new_empty(s["Q"].shape[:2], dtype=torch.float64)
        for i, (a, b) in enumerate(zip(s["cu"].tolist(), s["cu"].tolist()[1:])):
            for h in range(c["Hq"]):
                k, v = s["K"][a:b, h // group].double(), s["V"][a:b, h // group].double()
                O[a:b, h], S[a:b, h] = _attend64(s["Q"][a:b, h].double(), k, v, 0)
        return (O, S) if c["lse"] else O
    page, table = c["page"], s["table"].tolist()
    if op == "paged":
        n = c["n"]
        O, S = torch.empty_like(s["Q"], dtype=torch.float64), s["Q"].new_empty(s["Q"].shape[:2], dtype=torch.float64)
        for i, ctx in enumerate(lens):
            own_pages = table[i][: -(-ctx // page)]
            for kv in range(c["Hkv"]):
                k = s["Kc"][own_pages, :, kv].reshape(-1, c["D"])[:ctx].double()
                v = s["Vc"][own_pages, :, kv].reshape(-1, c["D"])[:ctx].double()
                q = s["Q"][i * n:(i + 1) * n, kv * group:(kv + 1) * group].double()
                o, lse = _attend64(q.reshape(-1, c["D"]), k, v, None)
                O[i * n:(i + 1) * n, kv * group:(kv + 1) * group] = o.view(n, group, -1)
                S[i * n:(i + 1) * n, kv * group:(kv + 1) * group] = lse.view(n, group)
        return O, S
    out = []
    for name in ("Kc", "Vc"):  # moves: every number is one of the inputs'
        x = s[name].double()
        if op == "copy":
            for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
                x[:, b] = s[name][:, a].double()
        elif op == "append":
            new = s["K" if name == "Kc" else "V"].double()
            for i, ctx in enumerate(lens):
                for p in range(ctx // page, -(-(ctx + c["n"]) // page)):
                    a, b = max(ctx, p * page), min(ctx + c["n"], (p + 1) * page)
                    x[table[i][p], a - p * page:b - p * page] = new[i * c["n"] + a - ctx:i * c["n"] + b - ctx]
        else:
            for i, (ctx, path) in enumerate(zip(lens, s["path"].tolist())):
                for j, node in enumerate([v for v in path if v >= 0]):
                    a, b = ctx + node, ctx + j
                    x[:, table[i][b // page], b % page] = s[name][:, table[i][a // page], a % page].double()
        out.append(x)
    return tuple(out) if op == "copy" else (*out, None)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    c, lens = case, _lens(case)
    B, n, Hq, Hkv, D, op = c["B"], c["n"], c["Hq"], c["Hkv"], c["D"], c["op"]
    if op == "prompt":
        T = sum(lens)
        return {"bytes": 4 * T * (Hq + Hkv) * D + 4 * T * Hq * c["lse"],
                "flops": 4 * D * Hq * sum(x * (x + 1) // 2 for x in lens)}
    if op == "paged":
        return {"bytes": 4 * sum(lens) * Hkv * D + B * n * Hq * (4 * D + 4) + 4 * sum(_pages(c)),
                "flops": 4 * D * Hq * n * sum(lens)}
    rows = {"append": B * n, "compact": sum(_steps(c)), "copy": B * n * c["page"]}[op] * c["layers"]
    return {"bytes": 2 * rows * Hkv * D * 4 + 8 * B, "flops": 0}
