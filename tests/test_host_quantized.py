"""Refusals of the calls over a quantised cache, on the CPU: nothing is launched.  And
the oracle of its formats, against torch's e4m3, every code and mistakes on purpose."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

import qattention_amd as qa
import quant64
from qattention_amd import _lib, quantized_kv

ARG, DTYPE, HEAD_DIM, LAYOUT, WORKSPACE = -1, -2, -3, -4, -5
FP16, BF16 = torch.float16, torch.bfloat16


def i64(*v):
    return (C.c_int64 * len(v))(*v)


def test_exports():
    import src.ragged_attn as sra
    for name in ("QuantizedKV", "quantized_kv_cache", "append_quantized_kv", "read_quantized_kv",
                 "prefix_attention_quantized"):
        assert getattr(sra, name) is getattr(qa, name)


# strides of a cache of 2 heads of 128 in 4 bits, pages of 16
CS, SS = (2048, 128, 64, 1), (128, 8, 4, 1)


def append(k=16, v=16, kst=(256, 128, 1), kc=16, vc=16, cs=CS, ks=16, vs=16, ss=SS, table=16, cols=4, pages=8, ps=16,
           ctx=16, new=16, cu=16, B=1, ms=8, T=8, Hkv=2, D=128, dtype=0, bits=4):
    st = None if kst is None else i64(*kst)
    return _lib.lib().qattn_quant_append(k, st, v, st, kc, vc, cs and i64(*cs), ks, vs, ss and i64(*ss), table, cols,
                                         pages, ps, ctx, new, cu, B, ms, T, Hkv, D, dtype, bits, None)


def read(k=16, v=16, kst=(256, 128, 1), kc=16, vc=16, cs=CS, ks=16, vs=16, ss=SS, table=16, cols=4, pages=8, ps=16,
         ctx=16, cu=16, B=1, ms=8, T=8, Hkv=2, D=128, dtype=0, bits=4):
    st = None if kst is None else i64(*kst)
    return _lib.lib().qattn_quant_read(kc, vc, cs and i64(*cs), ks, vs, ss and i64(*ss), table, cols, pages, ps, ctx,
                                       k, st, v, st, cu, B, ms, T, Hkv, D, dtype, bits, None)


COMMON = [
    (DTYPE, dict(dtype=2)), (DTYPE, dict(bits=5)), (DTYPE, dict(bits=16)), (HEAD_DIM, dict(D=96)), (ARG, dict(ps=0)),
    (ARG, dict(pages=-1)), (ARG, dict(cols=-1)), (ARG, dict(cols=1 << 27)), (ARG, dict(Hkv=0)), (ARG, dict(B=-1)),
    (ARG, dict(ms=-1)), (ARG, dict(T=1 << 31)), (ARG, dict(k=None)), (ARG, dict(kst=None)), (ARG, dict(kc=None)),
    (ARG, dict(vs=None)), (ARG, dict(cs=None)), (ARG, dict(ss=None)), (ARG, dict(ctx=None)), (ARG, dict(table=None)),
    (LAYOUT, dict(k=24)), (LAYOUT, dict(kst=(255, 128, 1))), (LAYOUT, dict(kc=24)), (LAYOUT, dict(cs=(2048, 128, 64, 2))),
    (LAYOUT, dict(cs=(2040, 128, 64, 1))), (LAYOUT, dict(ks=18)), (LAYOUT, dict(ss=(128, 8, 2, 1))),
    (LAYOUT, dict(ss=(128, 8, 4, 4))), (0, dict(B=0)),
]


@pytest.mark.parametrize("rc,kw", COMMON + [(ARG, dict(new=None))])
def test_append_abi(rc, kw):
    assert append(**kw) == rc
    assert rc == 0 or _lib.last_error()


@pytest.mark.parametrize("rc,kw", COMMON + [(0, dict(T=0)), (0, dict(ms=0))])
def test_read_abi(rc, kw):
    assert read(**kw) == rc
    assert rc == 0 or _lib.last_error()


def attend(q=16, qs=(512, 128, 1), kc=16, vc=16, cs=CS, ks=16, vs=16, ss=SS, table=16, cols=4, pages=8, ps=16, ctx=16,
           o=16, lse=None, cu=16, B=1, ms=8, T=8, Hq=4, Hkv=2, D=128, scale=0.1, dtype=0, bits=4, ws=256,
           ws_bytes=1 << 40):
    return _lib.lib().qattn_prefix_quant_fwd(
        q, i64(*qs), kc, vc, cs and i64(*cs), ks, vs, ss and i64(*ss), table, cols, pages, ps, ctx, o, i64(*qs), lse,
        None, cu, B, ms, T, Hq, Hkv, D, scale, dtype, bits, ws, ws_bytes, None)


@pytest.mark.parametrize("rc,kw", [
    (DTYPE, dict(dtype=2)), (DTYPE, dict(bits=6)), (HEAD_DIM, dict(D=256)), (ARG, dict(Hq=3)), (ARG, dict(ps=0)),
    (ARG, dict(cols=-1)), (ARG, dict(cols=1 << 27)), (ARG, dict(pages=-1)), (ARG, dict(scale=0.0)),
    (ARG, dict(scale=float("nan"))), (ARG, dict(T=1 << 31)), (ARG, dict(q=None)), (ARG, dict(o=None)),
    (ARG, dict(ctx=None)), (ARG, dict(table=None)), (ARG, dict(ks=None)), (ARG, dict(cs=None)), (ARG, dict(lse=16)),
    (LAYOUT, dict(o=8)), (LAYOUT, dict(qs=(511, 128, 1))), (LAYOUT, dict(vc=8)), (LAYOUT, dict(vs=17)),
    (LAYOUT, dict(cs=(-2048, 128, 64, 1))), (LAYOUT, dict(cs=(1 << 38, 128, 64, 1))), (LAYOUT, dict(ss=(-128, 8, 4, 1))),
    (LAYOUT, dict(ss=(1 << 34, 8, 4, 1))), (WORKSPACE, dict(ws=None, cols=500)), (WORKSPACE, dict(ws=264, cols=500)),
    (WORKSPACE, dict(ws_bytes=100, cols=500)), (0, dict(B=0)), (0, dict(T=0)), (0, dict(ms=0)),
])
def test_attend_abi(rc, kw):
    assert attend(**kw) == rc
    assert rc == 0 or _lib.last_error()


def test_workspace():
    ws = _lib.lib().qattn_prefix_quant_workspace_bytes
    for bits in (4, 8):
        assert ws(0, 1, 0, 32, 8, 128, 10, 16, bits) == 0 and ws(4, 1, 4, 32, 7, 128, 10, 16, bits) == 0
        assert ws(1, 1, 1, 32, 8, 128, 8, 16, bits) == 0  # a workgroup per item: no state leaves it
        small, large = ws(1, 1, 1, 32, 8, 128, 200, 16, bits), ws(64, 1, 64, 32, 8, 128, 1000, 16, bits)
        # at most two states of 16 rows (D floats, a maximum, a sum) for each of the 8 kv
        # heads that a workgroup takes, 512 workgroups: 68.2 MB, and a row of boundaries
        assert 0 < small < large < 512 * 2 * 8 * 16 * (128 + 2) * 4 + (1 << 16)
        assert ws(64, 1, 64, 32, 8, 128, 1000, 16, bits) == ws(64, 1, 64, 32, 8, 128, 60000, 16, bits)


def moves(kc=16, st=(0, 2048, 128, 64, 1), Hkv=2, D=64, dtype=2, layers=1, B=0):
    return _lib.lib().qattn_kv_compact(kc, i64(*st), kc + 4096, i64(*st), layers, 16, 4, 8, 16, 16, 16, 3, 16, B, Hkv,
                                       D, dtype, None)


@pytest.mark.parametrize("rc,kw", [
    (0, dict()), (0, dict(kc=17)), (0, dict(D=3, Hkv=3, st=(0, 144, 9, 3, 1))), (0, dict(D=1, st=(0, 32, 2, 1, 1))),
    (0, dict(st=(0, 4096, 256, 128, 1))), (DTYPE, dict(dtype=3)), (HEAD_DIM, dict(D=0)), (HEAD_DIM, dict(D=2000)),
    (HEAD_DIM, dict(dtype=0, D=96)), (LAYOUT, dict(st=(0, 2048, 128, 64, 2))),
    (LAYOUT, dict(D=48, st=(0, 2048, 128, 64, 1))), (LAYOUT, dict(D=12, st=(0, 2048, 128, 64, 1))),
    (ARG, dict(layers=0)), (ARG, dict(Hkv=0)),
])
def test_moves_of_bytes_abi(rc, kw):
    assert moves(**kw) == rc


def test_caches_of_zeros():
    c = qa.quantized_kv_cache(5, 16, 2, 64, device="cpu")
    assert [tuple(t.shape) for t in c] == [(5, 16, 2, 32)] * 2 + [(5, 16, 2, 2)] * 2 and not any(t.any() for t in c)
    c = qa.quantized_kv_cache(5, 16, 2, 64, bits=8, layers=3, device="cpu")
    assert c.K.shape == (3, 5, 16, 2, 64) and c.K_scale.dtype == torch.uint8
    one = c.layer(1)
    assert one.V.shape == (5, 16, 2, 64) and one.V.data_ptr() == c.V[1].data_ptr()
    for kw in (dict(bits=3), dict(head_dim=96)):
        with pytest.raises(ValueError):
            qa.quantized_kv_cache(**{**dict(num_pages=5, page_size=16, num_kv_heads=2, head_dim=64, device="cpu"), **kw})


def cache(bits=4, D=64):
    return qa.quantized_kv_cache(6, 16, 2, D, bits=bits, device="cpu")


def test_what_a_cache_is():
    for bits in (4, 8):
        for D in (32, 64, 128):
            pages, ps, heads, dim, b, at = quantized_kv._check_cache(cache(bits, D), True)
            assert (pages, ps, heads, dim, b) == (6, 16, 2, D, bits)
            assert list(at[2]) == [32 * D * bits // 8, 2 * D * bits // 8, D * bits // 8, 1]
            assert list(at[5]) == [32 * D // 32, 2 * D // 32, D // 32, 1]
    c = cache()
    wide = torch.zeros(6, 16, 4, 64, dtype=torch.uint8)
    bad = [
        None, c[:3], [*c], (*c[:3], 5),
        c._replace(K=c.K.short()), c._replace(K=c.K[0]), c._replace(V=c.V[:5]), c._replace(K_scale=c.K_scale[:, :8]),
        c._replace(K=c.K[..., :16], V=c.V[..., :16]),                      # 2 bits
        c._replace(K=wide[:, :, :2, :24], V=wide[:, :, 2:, :24]),          # 3 bits
        c._replace(K=wide[:, :, ::2, :32]),                                # strides of K and V differ
        c._replace(K=wide[:, :, :2, :32].transpose(1, 2).contiguous().transpose(1, 2)),
        c._replace(K=wide[:, :, :2, ::2], V=wide[:, :, 2:, ::2]),          # no bytes side by side
        c._replace(K=wide[:, :, :2, 1:33], V=wide[:, :, 2:, 1:33]),        # off the boundaries
        c._replace(K_scale=torch.zeros(6, 16, 2, 5, dtype=torch.uint8)[..., 1:3],
                   V_scale=torch.zeros(6, 16, 2, 5, dtype=torch.uint8)[..., 1:3]),
    ]
    for x in bad:
        with pytest.raises(ValueError):
            quantized_kv._check_cache(x, False)
    for x in (c._replace(V=c.K), c._replace(V_scale=c.K_scale),
              qa.QuantizedKV(*(t[:, :, :1].expand(-1, -1, 2, -1) for t in c)),
              qa.QuantizedKV(*(t[:1].expand(6, -1, -1, -1) for t in c))):
        quantized_kv._check_cache(x, False)  # (may be read)
        with pytest.raises(ValueError):
            quantized_kv._check_cache(x, True)


def test_refusals():
    c, x = cache(), torch.zeros(3, 2, 64, dtype=FP16)
    table, lens = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    for f in (lambda: qa.append_quantized_kv(x, x, c, table, lens), lambda: qa.read_quantized_kv(c, table, lens),
              lambda: qa.prefix_attention_quantized(x, c, table, lens)):
        with pytest.raises(RuntimeError, match="GPU only"):
            f()
    with pytest.raises(AssertionError, match="fp16 or bf16"):
        qa.append_quantized_kv(x.float(), x.float(), c, table, lens)
    with pytest.raises(AssertionError, match="fp16 or bf16"):
        qa.append_quantized_kv(x, x.bfloat16(), c, table, lens)
    with pytest.raises(AssertionError, match="fp16 or bf16"):
        qa.prefix_attention_quantized(x.double(), c, table, lens)
    with pytest.raises(ValueError, match="fp16 or bf16"):
        qa.read_quantized_kv(c, table, lens, dtype=torch.float32)
    for f in (lambda: qa.append_paged_kv(x, x, c.K, c.V, table, lens),
              lambda: qa.prefix_attention_paged(x, c.K, c.V, table, lens)):
        with pytest.raises(AssertionError, match="fp16 or bf16"):
            f()


def test_moves_of_bytes_refusals():
    c = cache()
    table, lens, path = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.zeros(3, 2)
    for k, v in ((c.K, c.K), (c.K, c.V[:3]), (c.K, c.V_scale), (c.K, c.V.short()), (c.K[0], c.V[0]),
                 (c.K[..., ::2], c.V[..., ::2]), (c.K[:1].expand(6, -1, -1, -1), c.V)):
        for f in (lambda: qa.compact_paged_kv(k, v, table, lens, path.int()),
                  lambda: qa.copy_kv_pages(k, v, [0], [1])):
            with pytest.raises(ValueError):
                f()
    with pytest.raises(RuntimeError, match="GPU only"):
        qa.copy_kv_pages(c.K, c.V, [0], [1])


# ---------------------------------------------------------------------------
# the oracle
# ---------------------------------------------------------------------------

def test_oracle_codes():
    assert quant64.magnitudes(4).tolist() == [0, 0.5, 1, 1.5, 2, 3, 4, 6]
    every = torch.arange(256, dtype=torch.uint8)
    want = every.view(torch.float8_e4m3fn).double()
    got = quant64.decode(every.view(8, 32), torch.full((8, 1), 127, dtype=torch.uint8), 8).flatten()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(9), want.nan_to_num(9))
    low = torch.tensor([[0x10 * h + h for h in range(16)]], dtype=torch.uint8)
    got = quant64.decode(low, torch.tensor([[128]], dtype=torch.uint8), 4)[0, ::2]
    assert got.tolist() == [0, 1, 2, 3, 4, 6, 8, 12, 0, -1, -2, -3, -4, -6, -8, -12]
    assert torch.isnan(quant64.decode(low, torch.tensor([[255]], dtype=torch.uint8), 4)).all()


@pytest.mark.parametrize("dtype", [FP16, BF16])
def test_oracle_rounding(dtype):
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(3000, 32, generator=g) * torch.exp2(torch.randint(-12, 12, (3000, 1), generator=g))).to(dtype)
    # e4m3: torch's own cast of the scaled rows
    code, s = quant64.encode(x, 8)
    y = x.float() * torch.exp2(127.0 - s.float())
    assert torch.equal(code, y.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8))
    top = y.abs().amax(1)
    assert bool(((top > 224) & (top <= 448)).all())
    # e2m1: no code is nearer, and the largest scaled magnitude is in (3.5, 7]
    code, s = quant64.encode(x, 4)
    y = (x.double() * torch.exp2(127.0 - s.double()))
    top = y.abs().amax(1)
    assert bool(((top > 3.5) & (top <= 7)).all())
    held = quant64.decode(code, torch.full_like(s, 127), 4)
    d = (y.abs()[..., None] - quant64.magnitudes(4)).abs().amin(-1)
    assert torch.equal((held - y).abs(), d)


def test_oracle_ends():
    # ties to the even code; what lies past the scale's end; blocks of zeros; no numbers
    x = torch.zeros(1, 32, dtype=FP16)
    x[0, :9] = torch.tensor([4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -5.0])
    code, s = quant64.encode(x, 4)
    assert s.item() == 127
    assert quant64.decode(code, s, 4)[0, :9].tolist() == [4, 0, 1, 1, 2, 2, 4, 4, -4]
    x = torch.full((1, 32), 65504.0, dtype=FP16)
    for bits, scale, held in ((4, 127 + 13, 49152.0), (8, 127 + 7, 57344.0)):
        code, s = quant64.encode(x, bits)
        assert s.item() == scale and quant64.decode(code, s, bits)[0, 0].item() == held
    code, s = quant64.encode(torch.zeros(1, 32, dtype=BF16), 4)
    assert s.item() == 1 and not code.any()
    x[0, 3] = float("nan")
    assert quant64.encode(x, 8)[1].item() == 255


@pytest.mark.parametrize("mistake", ["ties away", "floor scale", "halves swapped"])
def test_oracle_notices(mistake):
    """Mistakes in the oracle's place change what it says."""
    g = torch.Generator().manual_seed(2)
    x = (torch.randint(-28, 29, (200, 32), generator=g) / 4).to(FP16)
    code, s = quant64.encode(x, 4)
    if mistake == "halves swapped":
        wrong = quant64.decode(code // 16 + code % 16 * 16, s, 4)
    else:
        b = x.double()
        amax = b.abs().amax(1, keepdim=True)
        exp = torch.floor(torch.log2(amax)) - 2 + (amax > 1.75 * 2 ** torch.floor(torch.log2(amax)))
        if mistake == "floor scale":
            exp = torch.floor(torch.log2(amax)) - 2
        a = (b / 2 ** exp).abs()
        d = (a[..., None] - quant64.magnitudes(4)).abs()
        near = 7 - d.flip(-1).argmin(-1) if mistake == "ties away" else d.argmin(-1)
        wrong = torch.sign(b) * quant64.magnitudes(4)[near] * 2 ** exp
    assert not torch.equal(wrong, quant64.decode(code, s, 4))
