"""Refusals of the serving calls, on the CPU: nothing is launched."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

import qattention_amd as qa
from qattention_amd import _lib, paged_kv

ARG, DTYPE, HEAD_DIM, LAYOUT, WORKSPACE = -1, -2, -3, -4, -5


def i64(*v):
    return (C.c_int64 * len(v))(*v)


def test_exports():
    import src.ragged_attn as sra
    for name in ("prompt_attention", "prefix_attention_paged", "append_paged_kv", "compact_paged_kv", "copy_kv_pages"):
        assert getattr(sra, name) is getattr(qa, name)


def prompt(q=16, k=16, v=16, o=16, qs=(512, 128, 1), ks=(256, 128, 1), cu=16, B=1, ms=8, T=8, Hq=4, Hkv=2, D=128,
           scale=0.1, dtype=0, lse=None, ws=None, ws_bytes=0):
    return _lib.lib().qattn_prompt_fwd(q, i64(*qs), k, i64(*ks), v, i64(*ks), o, i64(*qs), lse, None, cu, B, ms, T, Hq,
                                       Hkv, D, scale, dtype, ws, ws_bytes, None)


@pytest.mark.parametrize("rc,kw", [
    (DTYPE, dict(dtype=2)), (HEAD_DIM, dict(D=96)), (ARG, dict(Hq=5)), (ARG, dict(B=-1)), (ARG, dict(T=1 << 31)),
    (ARG, dict(scale=0.0)), (ARG, dict(scale=float("nan"))), (ARG, dict(scale=float("inf"))), (ARG, dict(q=None)),
    (ARG, dict(cu=None)), (ARG, dict(lse=16)), (LAYOUT, dict(q=18)), (LAYOUT, dict(qs=(512, 127, 1))),
    (LAYOUT, dict(ks=(256, 128, 2))), (LAYOUT, dict(ks=(1 << 25, 128, 1))), (0, dict(B=0)), (0, dict(ms=0)),
    (0, dict(T=0)), (WORKSPACE, dict(ms=4000, T=4000)), (WORKSPACE, dict(ms=4000, T=4000, ws=256, ws_bytes=100)),
    (WORKSPACE, dict(ms=4000, T=4000, ws=264, ws_bytes=1 << 40)),
])
def test_prompt_abi(rc, kw):
    assert prompt(**kw) == rc
    assert rc == 0 or _lib.last_error()


def test_prompt_workspace():
    ws = _lib.lib().qattn_prompt_workspace_bytes
    assert ws(1, 8, 8, 4, 2, 128) == 0 and ws(0, 4000, 4000, 4, 2, 128) == 0 and ws(1, 4000, 4000, 5, 2, 128) == 0
    assert ws(64, 4000, 256000, 32, 8, 128) == 0  # tiles enough for every slot
    rows = -(-4000 * 2 // 128) * 2 * 128
    assert ws(1, 4000, 4000, 4, 2, 128) % (rows * 4 * 130) == 0 < ws(1, 4000, 4000, 4, 2, 128)
    # one long prompt among short ones: its tiles are cut, unless the short ones are thousands
    assert 0 < ws(70, 2000, 2069, 4, 2, 64) < 1 << 29 and ws(10001, 2000, 12000, 1, 1, 64) == 0


def paged(q=16, kc=16, vc=16, o=16, qs=(512, 128, 1), cs=(4096, 256, 128, 1), table=16, cols=4, pages=8, ps=16,
          ctx=16, cu=16, B=1, ms=8, T=8, Hq=4, Hkv=2, D=128, scale=0.1, dtype=0, ws=256, ws_bytes=1 << 40, lse=None):
    return _lib.lib().qattn_prefix_paged_fwd(
        q, i64(*qs), kc, i64(*cs), vc, i64(*cs), table, cols, pages, ps, ctx, o, i64(*qs), lse, None, cu, B, ms, T, Hq,
        Hkv, D, scale, dtype, ws, ws_bytes, None)


@pytest.mark.parametrize("rc,kw", [
    (DTYPE, dict(dtype=3)), (HEAD_DIM, dict(D=256)), (ARG, dict(Hq=3)), (ARG, dict(ps=0)), (ARG, dict(cols=-1)),
    (ARG, dict(pages=-1)), (ARG, dict(cols=1 << 27)), (ARG, dict(scale=-1.0)), (ARG, dict(ctx=None)),
    (ARG, dict(table=None)), (ARG, dict(kc=None)), (ARG, dict(lse=16)), (LAYOUT, dict(o=8)),
    (LAYOUT, dict(cs=(4096, 255, 128, 1))), (LAYOUT, dict(cs=(-4096, 256, 128, 1))),
    (LAYOUT, dict(cs=(1 << 35, 256, 128, 1))), (WORKSPACE, dict(ws=None, cols=500)),
    (WORKSPACE, dict(ws=264, cols=500)), (WORKSPACE, dict(ws_bytes=100, cols=500)), (0, dict(B=0)), (0, dict(T=0)), (0, dict(ms=0)),
])
def test_paged_abi(rc, kw):
    assert paged(**kw) == rc
    assert rc == 0 or _lib.last_error()


def test_paged_workspace():
    ws = _lib.lib().qattn_prefix_paged_workspace_bytes
    assert ws(0, 1, 0, 32, 8, 128, 10, 16) == 0 and ws(4, 1, 4, 32, 7, 128, 10, 16) == 0
    assert ws(1, 1, 1, 32, 8, 128, 8, 16) == 0  # a workgroup per item: no state leaves it
    small, large = ws(1, 1, 1, 32, 8, 128, 200, 16), ws(64, 1, 64, 32, 8, 128, 1000, 16)
    assert 0 < small < large < 64 << 20
    # it does not grow with the table past what the launch can share out
    assert ws(64, 1, 64, 32, 8, 128, 8000, 16) == large


def pages_call(which, kc=16, vc=16, cs=(32768, 4096, 256, 128, 1), layers=2, table=16, cols=4, pages=8, ps=16, ctx=16,
               acc=16, pcols=4, new=16, B=2, Hkv=2, D=128, dtype=0, k=16, ks=(256, 128, 1), cu=16, ms=4, T=8, n=3):
    L = _lib.lib()
    if which == "append":
        return L.qattn_kv_append(k, i64(*ks), k, i64(*ks), kc, i64(*cs), vc, i64(*cs), table, cols, pages, ps,
                                 ctx, new, cu, B, ms, T, Hkv, D, dtype, None)
    if which == "compact":
        return L.qattn_kv_compact(kc, i64(*cs), vc, i64(*cs), layers, table, cols, pages, ps, ctx, acc, pcols, new, B,
                                  Hkv, D, dtype, None)
    return L.qattn_kv_copy_pages(kc, i64(*cs), vc, i64(*cs), layers, pages, ps, acc, acc, n, Hkv, D, dtype, None)


@pytest.mark.parametrize("which", ["append", "compact", "copy"])
@pytest.mark.parametrize("rc,kw", [
    (DTYPE, dict(dtype=7)), (HEAD_DIM, dict(D=80)), (ARG, dict(Hkv=0)), (ARG, dict(ps=0)), (ARG, dict(pages=-1)),
    (ARG, dict(kc=None)), (LAYOUT, dict(vc=24)), (LAYOUT, dict(cs=(32768, 4096, 250, 128, 1))),
    (LAYOUT, dict(cs=(32768, 4096, 256, 128, 2))), (ARG, dict(ps=1 << 28)),
])
def test_pages_abi(which, rc, kw):
    assert pages_call(which, **kw) == rc and _lib.last_error()


@pytest.mark.parametrize("which,rc,kw", [
    ("append", ARG, dict(B=-1)), ("append", ARG, dict(cols=1 << 27)), ("append", ARG, dict(ctx=None)),
    ("append", ARG, dict(new=None)), ("append", ARG, dict(table=None)), ("append", ARG, dict(ms=-1)),
    ("append", ARG, dict(T=1 << 31)), ("append", ARG, dict(k=None)), ("append", LAYOUT, dict(ks=(255, 128, 1))),
    ("append", 0, dict(B=0)),
    ("compact", ARG, dict(pcols=-1)), ("compact", ARG, dict(acc=None)), ("compact", ARG, dict(layers=0)),
    ("compact", ARG, dict(new=None)), ("compact", 0, dict(B=0)),
    ("copy", ARG, dict(n=-1)), ("copy", ARG, dict(acc=None)), ("copy", 0, dict(n=0)), ("copy", 0, dict(layers=0)),
])
def test_pages_abi_own(which, rc, kw):
    assert pages_call(which, **kw) == rc


def T(*shape, dtype=torch.float16):
    return torch.zeros(*shape, dtype=dtype)


def test_cpu_tensors_fail_loudly():
    cu = torch.tensor([0, 4], dtype=torch.int32)
    cache, table, lens = (T(3, 16, 2, 64), T(3, 16, 2, 64)), torch.zeros(1, 2, dtype=torch.int32), cu[1:]
    with pytest.raises(RuntimeError, match="GPU only"):
        qa.prompt_attention(T(4, 4, 64), T(4, 2, 64), T(4, 2, 64), cu)
    with pytest.raises(RuntimeError, match="GPU only"):
        qa.prefix_attention_paged(T(1, 4, 64), *cache, table, lens)
    with pytest.raises(RuntimeError, match="GPU only"):
        qa.append_paged_kv(T(1, 2, 64), T(1, 2, 64), *cache, table, lens)
    with pytest.raises(RuntimeError, match="GPU only"):
        qa.compact_paged_kv(*cache, table, lens, table)
    with pytest.raises(RuntimeError, match="GPU only"):
        qa.copy_kv_pages(*cache, [0], [1])


def test_types_and_caches():
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(AssertionError, match="fp16 or bf16"):
        qa.prompt_attention(T(4, 4, 64, dtype=torch.float32), T(4, 2, 64), T(4, 2, 64), cu)
    chk = paged_kv._check_caches
    good = T(3, 16, 2, 64)
    with pytest.raises(ValueError, match="one shape"):
        chk(good, T(3, 16, 2, 32), (4,))
    with pytest.raises(ValueError, match="4-D"):
        chk(T(1, 3, 16, 2, 64), T(1, 3, 16, 2, 64), (4,))
    with pytest.raises(AssertionError, match="fp16 or bf16"):
        chk(good, good.bfloat16(), (4,))
    with pytest.raises(ValueError, match="16-byte rows"):
        chk(good, T(3, 16, 2, 65)[..., 1:], (4,))
    with pytest.raises(ValueError, match="overlap"):
        chk(good, T(1, 16, 2, 64).expand(3, 16, 2, 64), (4,))
    with pytest.raises(ValueError, match="same memory"):
        chk(good, good, (4,))
    chk(good, T(3, 16, 2, 64), (4,))


def test_row_offsets():
    rows, lens = paged_kv._rows, torch.tensor([0, 2, 3], dtype=torch.int32)
    with pytest.raises(ValueError, match="one row per sequence"):
        rows(3, 2, None, None, "cpu")
    with pytest.raises(ValueError, match="must have 4 entries"):
        rows(3, 3, lens, None, "cpu")
    assert rows(2, 2, None, None, "cpu") == (1, None) and rows(3, 2, lens, None, "cpu")[0] == 2
    with pytest.raises(ValueError, match="B >= 3"):
        paged_kv._table(torch.zeros(2, 4), 3, "cpu")
    with pytest.raises(ValueError, match=r"must be \[B\]"):
        paged_kv._lengths(torch.zeros(2, 4), "cpu")
    with pytest.raises(ValueError, match="must be integers"):
        paged_kv._lengths(torch.zeros(2), "cpu")
    with pytest.raises(ValueError, match="must be integers"):
        paged_kv._page_lists([1.5], torch.tensor([2.0]), 8, "cpu")


@pytest.mark.parametrize("src,dst,what", [
    ([0, 1], [2], "one length"), ([0, 9], [1, 2], "outside"), ([0, -1], [1, 2], "outside"), ([0, 1], [2, 9], "outside"),
    ([0, 1], [2, 2], "two copies"), ([0, 2], [2, 3], "source of another"), ([1, 2], [2, 1], "source of another"),
])
def test_page_lists(src, dst, what):
    with pytest.raises(ValueError, match=what):
        paged_kv._page_lists(src, dst, 8, "cpu")


def test_page_lists_taken():
    for src, dst in (([0, 0, 3], [1, 2, 3]), ([], []), (torch.tensor([4]), [5])):
        a, b = paged_kv._page_lists(src, dst, 8, "cpu")
        assert a.tolist() == list(src) and b.tolist() == list(dst) and a.dtype == b.dtype == torch.int32


def test_gradients_refused():
    from qattention_amd.ragged_attn import _no_grad
    x = torch.zeros(2, requires_grad=True)
    with pytest.raises(RuntimeError, match="no backward pass"):
        _no_grad(torch.zeros(2), x)
    _no_grad(torch.zeros(2))
    with torch.no_grad():
        _no_grad(x)


@pytest.mark.parametrize("src,dst", [([1.7], [2]), ([1], [2.0]), ([1], torch.tensor([2.5])), ([0, 1.0], [2, 3]),
                                     (torch.tensor([1.0]), [2])])
def test_page_lists_of_fractions(src, dst):
    with pytest.raises(ValueError, match="must be integers"):
        paged_kv._page_lists(src, dst, 8, "cpu")


def test_offsets_are_a_list_of_integers():
    from qattention_amd.ragged_attn import _offsets
    for cu in (torch.tensor([0.0, 2.5, 4.0]), torch.tensor([0, 4]).half()):
        with pytest.raises(ValueError, match="must be integers"):
            _offsets(cu, "cpu", 4)
        with pytest.raises(ValueError, match="must be integers"):
            paged_kv._rows(4, cu.shape[0] - 1, cu, 4, "cpu")
    for cu in (torch.tensor([[0, 4], [0, 4]]), torch.tensor(4), torch.empty(0, dtype=torch.int32)):
        with pytest.raises(ValueError, match=r"\[B \+ 1\]"):
            _offsets(cu, "cpu", 4)
    ms, cu = _offsets(torch.tensor([0, 3, 4], dtype=torch.int16), "cpu", None)
    assert ms == 3 and cu.dtype == torch.int32 and cu.tolist() == [0, 3, 4]


def test_values_past_32_bits_do_not_wrap():
    from qattention_amd.ragged_attn import _offsets
    top, low = 2 ** 31 - 1, -2 ** 31
    wide = torch.tensor([3, 2 ** 31 - 1, 2 ** 31, 2 ** 32 + 3, 2 ** 33 + 5, -1, -2 ** 32 + 1, -2 ** 63])
    assert paged_kv._int32(wide, wide.device).tolist() == [3, top, top, top, top, -1, low, low]
    assert paged_kv._lengths(wide[3:5], wide.device).tolist() == [top, top]
    assert paged_kv._table(wide[None], 1, wide.device).tolist()[0][4] == top
    assert paged_kv._int32(torch.tensor([7, 2 ** 32 - 1]).to(torch.uint32), wide.device).tolist() == [7, top]
    assert paged_kv._int32(torch.tensor([7, -1]).view(torch.uint64), wide.device).tolist() == [7, top]
    assert paged_kv._int32(torch.tensor([-3, 200], dtype=torch.int16), wide.device).tolist() == [-3, 200]
    for pages in ([2 ** 32 + 3], torch.tensor([2 ** 32 + 3])):
        with pytest.raises(ValueError, match="outside"):
            paged_kv._page_lists(pages, [1], 8, "cpu")
    ms, cu = _offsets(torch.tensor([0, 4, 2 ** 32 + 5]), "cpu", None)
    assert ms == top - 4 and cu.tolist() == [0, 4, top]
    # (the C entries take 32 bits: 2^40 would arrive as 0)
    assert _offsets(torch.tensor([0, 4]), "cpu", 2 ** 40)[0] == top and paged_kv._rows(4, 1, cu[:2], 2 ** 33, "cpu")[0] == top


def test_tangents_refused():
    import torch.autograd.forward_ad as fwd
    from qattention_amd.ragged_attn import _no_grad
    x = torch.zeros(2)
    with fwd.dual_level():
        _no_grad(x)
        dual = fwd.make_dual(x, torch.ones(2))
        with pytest.raises(RuntimeError, match="no forward derivative"):
            _no_grad(x, dual)
        with torch.no_grad(), pytest.raises(RuntimeError, match="no forward derivative"):
            _no_grad(dual)
    _no_grad(x)


@pytest.mark.parametrize("broken", ["compiler fails", "no compiler", "no headers"])
def test_library_is_built_without_the_call_module(broken, tmp_path, monkeypatch, capsys):
    """hipcc is a stand-in that writes what it is asked for."""
    from qattention_amd import build
    hipcc = tmp_path / "hipcc"
    hipcc.write_text('#!/bin/sh\nwhile [ "$1" != -o ]; do shift; done\necho built > "$2"\n')
    hipcc.chmod(0o755)
    for name, to in (("LIB_PATH", "lib.so"), ("CALLS_PATH", "calls.so"), ("OBJ_DIR", "obj")):
        monkeypatch.setattr(build, name, str(tmp_path / to))
    monkeypatch.setattr(build, "_hipcc", lambda: str(hipcc))
    (tmp_path / "calls.so").write_text("of another build")
    if broken == "no headers":
        def gone(out):
            raise ImportError("no torch headers")
        monkeypatch.setattr(build, "calls_command", gone)
    else:
        monkeypatch.setenv("CXX", "/bin/false" if broken == "compiler fails" else str(tmp_path / "not there"))
    assert build.build(verbose=False) == str(tmp_path / "lib.so")
    assert (tmp_path / "lib.so").read_text() == "built\n" and not (tmp_path / "calls.so").exists()
    assert "serving calls go through Python" in capsys.readouterr().err


@pytest.mark.parametrize("there", [False, True])
def test_calls_go_on_without_the_call_module(there, tmp_path, monkeypatch):
    """Not built, and built for something else."""
    path = tmp_path / "_calls.so"
    if there:
        path.write_text("no module")
    monkeypatch.setattr(_lib, "CALLS_PATH", str(path))
    monkeypatch.setattr(_lib, "_calls", None)
    x, cu = T(4, 2, 64), torch.tensor([0, 4], dtype=torch.int32)
    with pytest.warns(RuntimeWarning, match="go through Python"), pytest.raises(RuntimeError, match="GPU only"):
        qa.prompt_attention(x, x, x, cu)
    assert _lib.calls().append() is None and _lib.calls().set_ready(0) is None
    with pytest.raises(RuntimeError, match="GPU only"):  # (told once)
        qa.copy_kv_pages(T(3, 16, 2, 64), T(3, 16, 2, 64), [0], [1])


def test_workgroup_per_item_limits():
    """Two steps of 256 keys, four where the items fill half the chip: no workspace."""
    ws = _lib.lib().qattn_prefix_paged_workspace_bytes
    items = lambda B, cols: ws(B, 1, B, 32, 8, 128, cols, 16) == 0  # noqa: E731
    assert items(2, 32) and not items(2, 33) and items(15, 32) and not items(15, 33)
    assert items(16, 64) and not items(16, 65) and items(32, 64) and not items(33, 64)
