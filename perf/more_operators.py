"""Measured cases of the paged K/V cache that is held in 4 or 8 bits.

  op       store    new K/V rows of a layer quantised into the pages behind each context, and the same rows read back as
                    the cache holds them (what a prompt's own attention takes, so that it sees what later steps will see)
           read     whole contexts read back into packed 16-bit rows
           attend   attention of each sequence's query tokens over its context in the cache, O and LSE:
                    n = 1 token per sequence (a decode step), draft nodes or the tokens of a prompt's chunk
  B        sequences; L their context (the longest where they are ragged); n rows per sequence (new rows, query tokens)
  bits     of an element: 4 (e2m1) or 8 (e4m3); 32 elements along the head share a scale, a power of two in a byte (e8m0)
  Hq, Hkv, D, page, dtype, ragged

The cache holds N(0, 1) rows as append_quantized_kv writes them; pages lie in shuffled physical order, the slots behind a
context hold other rows of the same kind.
"""
from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"
BLOCK = 32                           # elements of a scale
TOP = {4: 2, 8: 8}                   # exponent of the largest element: 1.5 * 2^2, 1.75 * 2^8
LAST = {torch.float16: 15, torch.bfloat16: 127}  # exponent of a type's largest: a block's elements lie in its rows' range


def _case(name=None, **kw):
    c = dict(op="attend", B=1, L=512, n=1, bits=4, Hq=32, Hkv=8, D=128, page=16, dtype="fp16", ragged=False)
    c.update(kw)
    return dict(name=name, **c) if name else c


def listed():
    return [
        # one layer's new rows of a decode step
        _case("store_step", op="store", B=32, L=2000, ragged=True),
        # one layer's rows of long prompts behind an earlier chunk
        _case("store_prompt", op="store", B=8, L=500, n=4003, dtype="bf16"),
        # the same of prompts of a few hundred tokens, 64-wide heads, 8 bits
        _case("store_chunk8", op="store", B=5, L=1203, n=317, bits=8, D=64, ragged=True),
        # a young conversation's context handed to something that takes 16-bit rows
        _case("read_one", op="read", L=731),
        # the contexts of a batch
        _case("read_batch", op="read", B=16, L=10007, dtype="bf16", ragged=True),
        # 64-wide heads, 8 bits
        _case("read_batch8", op="read", B=12, L=5003, bits=8, D=64, Hkv=4, ragged=True),
        # a decode step of two young conversations
        _case("decode_small", B=2, L=731, ragged=True),
        # a decode step of a large batch whose contexts differ by a factor of three
        _case("decode_batch", B=64, L=16000, dtype="bf16", ragged=True),
        # the same in 8 bits
        _case("decode_batch8", B=48, L=12001, bits=8, ragged=True),
        # one very long context, few kv heads of 64
        _case("decode_long", L=131072, Hkv=4, D=64, dtype="bf16"),
        # the context half of verifying 60-node drafts over long contexts
        _case("verify_tree", B=4, L=10240, n=60),
        # a prompt's next chunk over the chunks before it, 8 bits
        _case("chunk8", B=2, L=6007, n=1009, bits=8, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges, no dearer than the largest listed."""
    while True:
        op = rng.choice(["store", "store", "read", "read", "attend", "attend", "attend", "attend"])
        Hkv = rng.choice([2, 4, 8, 32])
        Hq = 32 if Hkv != 4 else rng.choice([4, 32])
        c = _case(op=op, Hq=Hq, Hkv=Hkv, D=rng.choice([32, 64, 128, 128]), bits=rng.choice([4, 4, 8]),
                  dtype=rng.choice(["fp16", "bf16"]), page=rng.choice([16, 16, 32, 64]), ragged=rng.random() < 0.6)
        if op == "store":
            c.update(B=_log(rng, 1, 64), L=_log(rng, 30, 4000), n=rng.choice([1, _log(rng, 2, 8000)]))
            if c["B"] * (c["L"] + c["n"]) * c["Hkv"] * c["D"] > 8 * 4503 * 32 * 128:
                continue
        elif op == "read":
            c.update(B=_log(rng, 1, 32), L=_log(rng, 30, 40000))
            if c["B"] * c["L"] * c["Hkv"] * c["D"] > 16 * 10007 * 8 * 128:
                continue
        else:
            c.update(B=_log(rng, 1, 64), L=_log(rng, 60, 131072), n=rng.choice([1, 1, 1, _log(rng, 2, 1009)]))
            if c["B"] * c["L"] * c["Hkv"] * c["D"] > 64 * 16000 * 8 * 128 or c["B"] * c["n"] * c["L"] > 2 * 1009 * 6007:
                continue
        w = work(c)
        if w["bytes"] <= 8.0e8 and w["flops"] <= 2.0e11:
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


def _dtype(c):
    return torch.bfloat16 if c["dtype"] == "bf16" else torch.float16


# ---------------------------------------------------------------------------
# the cache's format, plainly
# ---------------------------------------------------------------------------

def _quantize(x, bits):
    """Codes and scales of rows [..., D].  The scale's exponent is the largest magnitude's, less TOP, one more where that
    magnitude is above 1.75 times its power of two; elements are rounded to nearest, ties to the even code, and end at the
    format's largest; a block with an infinity or a NaN gets the scale that is no number."""
    b = x.float().unflatten(-1, (-1, BLOCK))
    amax = b.abs().amax(-1)
    code = ((amax.view(torch.int32) + 0x1FFFFF) >> 23) - TOP[bits]
    code = code.clamp(1, 127 + LAST[x.dtype] - TOP[bits])
    y = torch.ldexp(b, (127 - code).unsqueeze(-1))
    if bits == 4:
        a = y.abs()
        q = (a > 0.25).to(torch.uint8)
        for edge, even in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
            q += (a >= edge) if even else (a > edge)
        q = (q | torch.signbit(y).to(torch.uint8) << 3).flatten(-2)
        q = q[..., 0::2] | q[..., 1::2] << 4
    else:
        q = y.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8).flatten(-2)
    code = torch.where(torch.isfinite(amax), code, 255)
    return q, code.to(torch.uint8)


def _values(q, code, bits):
    """The rows that codes and scales stand for, in fp32."""
    if bits == 4:
        table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=q.device)
        x = torch.stack((table[(q & 15).int()], table[(q >> 4).int()]), -1).flatten(-2)
    else:
        x = q.view(torch.float8_e4m3fn).float()
    scale = torch.exp2(code.float() - 127.0).masked_fill(code == 255, math.nan)
    return (x.unflatten(-1, (-1, BLOCK)) * scale.unsqueeze(-1)).flatten(-2)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def prepare(case, seed):
    c, g = case, torch.Generator(device=DEV).manual_seed(int(seed))
    dt, B, Hq, Hkv, D, page, bits = _dtype(c), c["B"], c["Hq"], c["Hkv"], c["D"], c["page"], c["bits"]
    lens, n, op = _lens(c), c["n"], c["op"]

    def rand(*shape):
        return torch.empty(shape, dtype=dt, device=DEV).normal_(0.0, 1.0, generator=g)

    pages = [-(-(x + (n if op == "store" else 0)) // page) for x in lens]
    total = sum(pages)

    def cache():
        q = torch.empty(total, page, Hkv, D * bits // 8, dtype=torch.uint8, device=DEV)
        code = torch.empty(total, page, Hkv, D // BLOCK, dtype=torch.uint8, device=DEV)
        step = max(1, (1 << 26) // (page * Hkv * D))
        for i in range(0, total, step):
            q[i:i + step], code[i:i + step] = _quantize(rand(min(step, total - i), page, Hkv, D), bits)
        return q, code

    s = {"c": c, "max": n, "total": B * n}
    (s["Kc"], s["Ks"]), (s["Vc"], s["Vs"]) = cache(), cache()
    order = torch.randperm(total, generator=g, device=DEV, dtype=torch.int32)
    first = torch.tensor([0] + pages).cumsum(0)
    col = torch.arange(max(pages))[None, :]
    at = (first[:-1, None] + col).clamp(max=total - 1).to(DEV)
    there = (col < torch.tensor(pages)[:, None]).to(DEV)
    s["table"] = torch.where(there, order[at], torch.zeros_like(order[at]))
    s["ctx"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    if op == "store":
        s["K"], s["V"] = rand(B * n, Hkv, D), rand(B * n, Hkv, D)
    elif op == "attend":
        s["Q"] = rand(B * n, Hq, D)
    else:
        s["start"] = torch.zeros(B, dtype=torch.int32, device=DEV)
        s["cu"] = torch.tensor([0] + lens).cumsum(0).to(device=DEV, dtype=torch.int32)
        s["max"], s["total"] = max(lens), sum(lens)
    if op != "read" and n > 1:
        s["cu"] = torch.arange(0, (B + 1) * n, n, dtype=torch.int32, device=DEV)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    s, op = state, state["c"]["op"]
    if own:
        return _own(s, op)
    return {"store": _store, "read": _read, "attend": _attend}[op](s)


def _own(s, op):
    import qattention_amd as qa

    cache, cu, ms = qa.QuantizedKV(s["Kc"], s["Vc"], s["Ks"], s["Vs"]), s.get("cu"), s["max"]
    if op == "attend":
        return qa.prefix_attention_quantized(s["Q"], cache, s["table"], s["ctx"], cu_seqlens=cu, max_seqlen=ms)
    if op == "read":
        return qa.read_quantized_kv(cache, s["table"], s["start"], cu, max_seqlen=ms, total_tokens=s["total"],
                                    dtype=_dtype(s["c"]))
    lens = qa.append_quantized_kv(s["K"], s["V"], cache, s["table"], s["ctx"], cu_seqlens=cu, max_seqlen=ms)
    K, V = qa.read_quantized_kv(cache, s["table"], s["ctx"], cu, max_seqlen=ms, total_tokens=s["total"],
                                dtype=s["K"].dtype)
    return K, V, lens


def _store(s):
    c, (n, page) = s["c"], (s["c"]["n"], s["c"]["page"])
    pos = s["ctx"].long()[:, None] + torch.arange(n, device=DEV)
    at = s["table"].long().gather(1, pos // page), pos % page
    out = []
    for x, q, code in ((s["K"], s["Kc"], s["Ks"]), (s["V"], s["Vc"], s["Vs"])):
        q[at], code[at] = (t.unflatten(0, (c["B"], n)) for t in _quantize(x, c["bits"]))
        out.append(_values(q[at], code[at], c["bits"]).flatten(0, 1).to(x.dtype))
    return out[0], out[1], s["ctx"] + n


def _read(s):
    c, cu = s["c"], s["cu"].long()
    t = torch.arange(s["total"], device=DEV)
    seq = torch.searchsorted(cu[1:], t, right=True)
    pos = s["start"].long()[seq] + t - cu[seq]
    at = s["table"].long()[seq, pos // c["page"]], pos % c["page"]
    return tuple(_values(q[at], code[at], c["bits"]).to(_dtype(c))
                 for q, code in ((s["Kc"], s["Ks"]), (s["Vc"], s["Vs"])))


def _attend(s):
    """Each sequence's pages gathered: softmax(Q K^T / sqrt(D) + length mask) V in fp32."""
    c, table = s["c"], s["table"].long()
    B, n, Hq, Hkv, D = c["B"], c["n"], c["Hq"], c["Hkv"], c["D"]

    def rows(q, code):  # [B, Hkv, rows, D]
        return _values(q[table], code[table], c["bits"]).flatten(1, 2).transpose(1, 2)

    q = s["Q"].float().view(B, n, Hkv, Hq // Hkv, D).permute(0, 2, 1, 3, 4).flatten(2, 3) / math.sqrt(D)
    score = torch.matmul(q, rows(s["Kc"], s["Ks"]).transpose(-1, -2))
    j = torch.arange(score.shape[-1], device=DEV)
    score.masked_fill_((j[None, :] >= s["ctx"][:, None])[:, None, None, :], -math.inf)
    m = score.amax(-1, keepdim=True)
    p = score.sub_(m).exp_()
    z = p.sum(-1, keepdim=True)
    o = torch.matmul(p, rows(s["Vc"], s["Vs"])) / z
    O = o.view(B, Hkv, n, Hq // Hkv, D).permute(0, 2, 1, 3, 4).reshape(B * n, Hq, D).to(s["Q"].dtype)
    return O, (m + z.log()).view(B, Hkv, n, Hq // Hkv).permute(0, 2, 1, 3).reshape(B * n, Hq)


# ---------------------------------------------------------------------------
# the definition in 64 bits, sequence by sequence
# ---------------------------------------------------------------------------

def _levels(bits):
    """Every magnitude of the format, by code."""
    e, m = (2, 1) if bits == 4 else (4, 3)
    bias = (1 << (e - 1)) - 1
    out = []
    for i in range(1 << (e + m)):
        x, f = i >> m, (i & ((1 << m) - 1)) / (1 << m)
        out.append(math.ldexp(f, 1 - bias) if x == 0 else math.ldexp(1 + f, x - bias))
    return torch.tensor(out if bits == 4 else out[:-1], dtype=torch.float64, device=DEV)  # (e4m3's last is no number)


def _held64(x, bits):
    """What the cache holds of rows [..., D]: per block of 32 the smallest power of two that brings its largest magnitude
    to no more than 1.75 times the format's top power, then the nearest level (of two, the even one)."""
    b = x.double().unflatten(-1, (-1, BLOCK))
    amax = b.abs().amax(-1, keepdim=True)
    mant, e = torch.frexp(amax)  # amax = mant 2^e, mant in [0.5, 1)
    e = e.long() - 1 + (mant > 0.875) - TOP[bits]
    low, high = 1 - 127, LAST[x.dtype] - TOP[bits]
    unit = torch.exp2(torch.where(amax == 0, low, e).clamp(low, high).double())
    levels, a = _levels(bits), (b / unit).abs()
    up = torch.searchsorted(levels, a.contiguous()).clamp(max=len(levels) - 1)
    down = (up - 1).clamp(min=0)
    d_up, d_down = levels[up] - a, a - levels[down]
    pick = torch.where((d_down < d_up) | ((d_down == d_up) & (down % 2 == 0)), down, up)
    return (torch.sign(b) * levels[pick] * unit).flatten(-2)


def _rows64(q, code, bits):
    """Rows [..., D] of codes and scales."""
    x = torch.stack((q % 16, q // 16), -1).flatten(-2) if bits == 4 else q
    half = 8 if bits == 4 else 128
    v = torch.cat((_levels(bits), torch.full((bits // 8,), math.nan, dtype=torch.float64, device=DEV)))
    v = v[(x % half).long()] * (1.0 - 2.0 * (x // half).double())
    return (v.unflatten(-1, (-1, BLOCK)) * torch.exp2(code.double() - 127)[..., None]).flatten(-2)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    group, op, lens, page, bits = c["Hq"] // c["Hkv"], c["op"], _lens(c), c["page"], c["bits"]
    if op == "store":
        return _held64(s["K"], bits), _held64(s["V"], bits), None
    table = s["table"].tolist()

    def context(i, ctx, h, q, code):
        own_pages = table[i][: -(-ctx // page)]
        x, y = q[own_pages][:, :, h].flatten(0, 1)[:ctx], code[own_pages][:, :, h].flatten(0, 1)[:ctx]
        return _rows64(x, y, bits)

    if op == "read":
        return tuple(torch.cat([context(i, ctx, slice(None), s[q], s[code]) for i, ctx in enumerate(lens)])
                     for q, code in (("Kc", "Ks"), ("Vc", "Vs")))
    n = c["n"]
    O, S = torch.empty_like(s["Q"], dtype=torch.float64), s["Q"].new_empty(s["Q"].shape[:2], dtype=torch.float64)
    for i, ctx in enumerate(lens):
        for kv in range(c["Hkv"]):
            k, v = context(i, ctx, kv, s["Kc"], s["Ks"]), context(i, ctx, kv, s["Vc"], s["Vs"])
            heads = slice(kv * group, (kv + 1) * group)
            q = s["Q"][i * n:(i + 1) * n, heads].double().reshape(-1, c["D"])
            w = q @ k.T / math.sqrt(c["D"])
            lse = torch.logsumexp(w, 1)
            S[i * n:(i + 1) * n, heads] = lse.view(n, group)
            O[i * n:(i + 1) * n, heads] = (torch.exp(w - lse[:, None]) @ v).view(n, group, -1)
    return O, S


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    c, lens = case, _lens(case)
    B, n, Hq, Hkv, D, op = c["B"], c["n"], c["Hq"], c["Hkv"], c["D"], c["op"]
    held = 2 * Hkv * (D * c["bits"] // 8 + D // BLOCK)  # bytes of a position's K and V row in the cache
    plain = 4 * Hkv * D                                 # and in 16 bits
    if op == "store":
        return {"bytes": B * n * (2 * plain + held) + 8 * B, "flops": 0}
    if op == "read":
        return {"bytes": sum(lens) * (plain + held) + 8 * B, "flops": 0}
    return {"bytes": sum(lens) * held + B * n * Hq * (4 * D + 4) + 4 * sum(-(-x // c["page"]) for x in lens),
            "flops": 4 * D * Hq * n * sum(lens)}
