"""Rows in blocks of 32 elements with a scale, from the formats' definitions in 64 bits.

e2m1 and e4m3 codes are sign, exponent, mantissa; a scale byte c stands for
2^(c - 127), 255 for no number.  Writing: the scale is the smallest power of two s,
2^-126 at least, with the block's largest magnitude <= 1.75 2^T s (T = 2, 8), at most
2^(E - T) (E: exponent of the rows' type's largest number); elements are the code
nearest to x / s, of two the even one, the largest finite one past it."""
from __future__ import annotations

import math

import torch

BLOCK = 32
TOP = {4: 2, 8: 8}
LAST = {torch.float16: 15, torch.bfloat16: 127}


def magnitudes(bits):
    """Value of every code without its sign; NaN where it is none."""
    e, m = (2, 1) if bits == 4 else (4, 3)
    bias = 2 ** (e - 1) - 1
    v = []
    for code in range(2 ** (e + m)):
        x, f = code >> m, (code % 2 ** m) / 2 ** m
        v.append(f * 2.0 ** (1 - bias) if x == 0 else (1 + f) * 2.0 ** (x - bias))
    if bits == 8:
        v[-1] = math.nan
    return torch.tensor(v, dtype=torch.float64)


def encode(x, bits):
    """Bytes of elements [..., D * bits / 8] and of scales [..., D / 32] of fp16 or bf16
    rows x [..., D], on the CPU."""
    b = x.cpu().double().unflatten(-1, (-1, BLOCK))
    amax = b.abs().amax(-1)
    good = torch.isfinite(amax)
    exps = torch.arange(-126, LAST[x.dtype] - TOP[bits] + 1)
    fits = amax.nan_to_num(posinf=0)[..., None] <= 1.75 * 2.0 ** TOP[bits] * torch.exp2(exps.double())
    first = torch.where(fits.any(-1), fits.double().argmax(-1), torch.tensor(len(exps) - 1))
    exp = exps[first]
    a = (b.nan_to_num(posinf=0, neginf=0) / torch.exp2(exp.double())[..., None]).abs()
    table = magnitudes(bits)[:(8 if bits == 4 else 127)]
    above = torch.searchsorted(table, a.contiguous()).clamp(max=len(table) - 1)
    below = (above - 1).clamp(min=0)
    up, down = table[above] - a, a - table[below]
    code = torch.where((down < up) | ((down == up) & (below % 2 == 0)), below, above)
    code = code + torch.signbit(b).long() * (8 if bits == 4 else 128)
    code = torch.where(good[..., None], code, 0).flatten(-2).to(torch.uint8)
    if bits == 4:
        code = code[..., 0::2] + 16 * code[..., 1::2]
    return code, torch.where(good, exp + 127, 255).to(torch.uint8)


def decode(elements, scales, bits):
    """The values in fp64, on the elements' device."""
    x = torch.stack((elements % 16, elements // 16), -1).flatten(-2) if bits == 4 else elements
    half = 8 if bits == 4 else 128
    v = magnitudes(bits).to(x.device)[(x % half).long()] * torch.where(x >= half, -1.0, 1.0)
    s = torch.exp2(scales.double() - 127).masked_fill(scales == 255, math.nan)
    return (v.unflatten(-1, (-1, BLOCK)) * s[..., None]).flatten(-2)
