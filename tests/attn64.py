"""Dense attention in 64 bits with the bounds that the kernels' arithmetic allows.

The kernels form scores, exponentials, sums and products in fp32, round each
softmax weight to the inputs' type for its product with V, and round the output
once.  With u = 2^-24 and h = eps / 2 of the inputs' type, per output element:
  scores   |ds| <= (D + 2) u scale sum_d |q_d k_d|            (a D-term sum, one scaling)
  weights  relative 2 max|ds| + 2^-21 (exp2, its argument's rounding) + n u (their sum)
  product  h per weight, and 2^-25 for fp16 weights below 2^-14 of the largest, all
           against A = sum_j p_j |v_j|
  output   h |o|
The argument s c - m c of the exponential adds u |s c| on top: 4 u max|s|.
"""
from __future__ import annotations

import math

import torch

U = 2.0 ** -24


def attend64(q, k, v, mask):
    """q [n, Hq, D], k, v [m, Hkv, D] (any type), mask [n, m] (True: attends).
    Returns o [n, Hq, D], lse [n, Hq] in fp64 and their bounds; rows that attend
    nothing give 0 and -inf."""
    n, Hq, D = q.shape
    g = Hq // k.shape[1]
    half = torch.finfo(q.dtype).eps / 2
    fp16 = q.dtype == torch.float16
    scale = 1 / math.sqrt(D)
    o = torch.zeros(n, Hq, D, dtype=torch.float64, device=q.device)
    lse = torch.full((n, Hq), -math.inf, dtype=torch.float64, device=q.device)
    to, tl = torch.zeros_like(o), torch.zeros_like(lse)
    if not mask.numel():
        return o, lse, to, tl
    some = mask.any(1)
    for h in range(Hq):
        qh, kh, vh = q[:, h].double(), k[:, h // g].double(), v[:, h // g].double()
        s = (qh @ kh.T * scale).masked_fill(~mask, -math.inf)
        mag = (qh.abs() @ kh.abs().T * scale).masked_fill(~mask, 0.0)
        m = s.amax(1, keepdim=True)
        e = torch.exp(s - torch.where(some[:, None], m, torch.zeros_like(m)))
        l = e.sum(1, keepdim=True)
        p = torch.where(some[:, None], e / l, torch.zeros_like(e))
        live = s.masked_fill(~mask, 0.0).abs().amax(1)
        ds = (D + 2) * U * mag.amax(1) + 4 * U * live
        rel = 2 * ds + 2.0 ** -21 + k.shape[0] * U
        o[:, h] = p @ vh
        A = p @ vh.abs()
        small = (2.0 ** -25 / l.clamp(min=1)) * (mask.double() @ vh.abs()) if fp16 else 0.0
        to[:, h] = half * (o[:, h].abs() + A) + rel[:, None] * A + small
        lse[:, h] = torch.where(some, (m + l.log())[:, 0], torch.full_like(live, -math.inf))
        tl[:, h] = ds + 2.0 ** -21 + k.shape[0] * U + 4 * U * torch.where(some, lse[:, h].abs(), live)
    return o, lse, to, tl


def check(O, L, ref, what=""):
    o, lse, to, tl = ref
    assert O.shape == o.shape and bool(torch.isfinite(O).all()), what
    off = (O.double() - o).abs() - to
    assert float(off.max()) <= 0 if off.numel() else True, (what, float(off.max()))
    if L is not None:
        empty = torch.isinf(lse)
        assert torch.equal(torch.isinf(L) & (L < 0), empty), what
        off = ((L.double() - lse).abs() - tl)[~empty]
        assert float(off.max()) <= 0 if off.numel() else True, (what, float(off.max()))


def causal(n, device="cuda"):
    return torch.ones(n, n, dtype=torch.bool, device=device).tril()


def offsets(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32)
