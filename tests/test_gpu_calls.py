"""The direct way of the serving calls (csrc/calls.cpp) against the Python one: the
same bits, and None for whatever needs a conversion, a copy or an error."""
from __future__ import annotations

import types

import pytest
import torch

from attn64 import offsets

DEV = "cuda"


def say(*a):
    print(*a, flush=True)


@pytest.fixture
def in_python(monkeypatch):
    """Within it every call goes through Python."""
    from qattention_amd import _lib
    _lib.calls()
    never = types.SimpleNamespace(**{n: lambda *a: None for n in ("prompt", "paged", "append", "compact", "copy")},
                                  set_ready=lambda d: None)

    class Switch:
        def __enter__(self):
            self.real = _lib._calls
            _lib._calls = never

        def __exit__(self, *exc):
            _lib._calls = self.real

    return Switch()


def operands(dtype=torch.float16):
    g = torch.Generator(device=DEV).manual_seed(3)
    r = lambda *s: torch.empty(s, dtype=dtype, device=DEV).normal_(0, 1, generator=g)  # noqa: E731
    o = dict(Q=r(50, 8, 64), K=r(50, 2, 64), V=r(50, 2, 64), Kc=r(2, 12, 16, 2, 64), Vc=r(2, 12, 16, 2, 64))
    o["cu"] = offsets([20, 30]).to(DEV)
    o["table"] = torch.randperm(12, generator=torch.Generator().manual_seed(4)).to(DEV, torch.int32).view(2, 6)
    o["ctx"] = torch.tensor([33, 60], dtype=torch.int32, device=DEV)
    o["path"] = torch.tensor([[0, 2, 5], [1, 3, -1]], dtype=torch.int32, device=DEV)
    o["src"], o["dst"] = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([0, 1], [7, 8]))
    return o


def all_calls(o):
    import qattention_amd as qa
    kc, vc = o["Kc"].clone(), o["Vc"].clone()
    out = [qa.prompt_attention(o["Q"], o["K"], o["V"], o["cu"], 30),
           *qa.prompt_attention(o["Q"], o["K"], o["V"], o["cu"], 30, return_lse=True),
           qa.prefix_attention_paged(o["Q"][:2], kc[0], vc[0], o["table"], o["ctx"], return_lse=False),
           *qa.prefix_attention_paged(o["Q"], kc[1], vc[1], o["table"], o["ctx"], o["cu"], 30),
           qa.append_paged_kv(o["K"], o["V"], kc[0], vc[0], o["table"], o["ctx"], o["cu"], 30),
           qa.append_paged_kv(o["K"][:2], o["V"][:2], kc[1], vc[1], o["table"], o["ctx"]),
           qa.compact_paged_kv(kc, vc, o["table"], o["ctx"], o["path"]),
           qa.compact_paged_kv(kc[0], vc[0], o["table"], o["ctx"], o["path"])]
    qa.copy_kv_pages(kc, vc, o["src"], o["dst"])
    qa.copy_kv_pages(kc[1], vc[1], o["dst"], o["src"])
    return out + [kc, vc]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_same_as_in_python(in_python, dtype):
    from qattention_amd import _lib
    o = operands(dtype)
    all_calls(o)  # (the device is set up)
    say("direct")
    direct = all_calls(o)
    with in_python:
        say("python")
        python = all_calls(o)
    for a, b in zip(direct, python):
        assert a.dtype == b.dtype and a.shape == b.shape and a.stride() == b.stride() and torch.equal(a, b)
    # the direct way answered these calls
    c = _lib.calls()
    assert c.prompt(o["Q"], o["K"], o["V"], o["cu"], 30, False) is not None
    assert c.paged(o["Q"][:2], o["Kc"][0], o["Vc"][0], o["table"], o["ctx"], None, None, True) is not None
    assert c.append(o["K"][:2], o["V"][:2], o["Kc"][0], o["Vc"][0], o["table"], o["ctx"], None, None) is not None
    assert c.compact(o["Kc"], o["Vc"], o["table"], o["ctx"], o["path"]) is not None
    assert c.copy(o["Kc"], o["Vc"], o["src"], o["dst"]) is True


@pytest.mark.gpu
def test_leaves_the_rest_to_python():
    """Operands that need a copy, a conversion or an error, one at a time."""
    from qattention_amd import _lib
    all_calls(operands())
    c, o = _lib.calls(), operands()
    before = [o[n].clone() for n in ("Kc", "Vc")]
    odd = torch.zeros(50, 8, 65, dtype=torch.float16, device=DEV)[..., 1:]
    grad = o["K"].clone().requires_grad_()
    prompt = dict(Q=o["Q"], K=o["K"], V=o["V"], cu=o["cu"], ms=30, lse=False)
    for i, kw in enumerate((dict(Q=odd), dict(Q=o["Q"].cpu()), dict(Q=o["Q"].float()), dict(K=o["K"].bfloat16()),
                            dict(K=grad), dict(V=o["V"][:40]), dict(cu=o["cu"].cpu()), dict(cu=o["cu"].long()),
                            dict(ms=None), dict(ms=-1), dict(ms=1 << 40), dict(ms=30.0), dict(Q=o["Q"][:, :7]),
                            dict(Q=o["Q"][:0], K=o["K"][:0], V=o["V"][:0]), dict(lse=1), dict(Q=None),
                            dict(cu=o["cu"][:1]))):
        say("prompt", i)
        assert c.prompt(*{**prompt, **kw}.values()) is None
    paged = dict(Q=o["Q"], Kc=o["Kc"][0], Vc=o["Vc"][0], table=o["table"], ctx=o["ctx"], cu=o["cu"], ms=30, lse=True)
    for i, kw in enumerate((dict(Kc=o["Kc"]), dict(table=o["table"].cpu()), dict(table=o["table"][:, ::2]),
                            dict(ctx=o["ctx"].long()), dict(cu=None), dict(cu=o["cu"][:2]), dict(table=o["table"][:1]),
                            dict(Vc=o["Vc"][0][:5]), dict(Kc=o["Kc"][0][..., :32], Vc=o["Vc"][0][..., :32]))):
        say("paged", i)
        assert c.paged(*{**paged, **kw}.values()) is None
    append = dict(K=o["K"], V=o["V"], Kc=o["Kc"][0], Vc=o["Vc"][0], table=o["table"], ctx=o["ctx"], cu=o["cu"], ms=30)
    for i, kw in enumerate((dict(Vc=o["Kc"][0]), dict(Kc=o["Kc"][0][:1].expand(12, 16, 2, 64)), dict(Kc=o["Kc"]),
                            dict(K=o["K"][:, :1]), dict(cu=None), dict(K=o["K"].cpu()))):
        say("append", i)
        assert c.append(*{**append, **kw}.values()) is None
    assert c.compact(o["Kc"], o["Vc"], o["table"], o["ctx"], o["path"][:1]) is None
    assert c.compact(o["K"], o["V"], o["table"], o["ctx"], o["path"]) is None
    assert c.copy(o["Kc"], o["Vc"], [0, 1], [7, 8]) is None
    assert c.copy(o["Kc"], o["Vc"], o["src"], o["dst"][:1]) is None
    assert torch.equal(o["Kc"], before[0]) and torch.equal(o["Vc"], before[1])


def test_host_operands():
    """On the CPU: nothing is answered, nothing is launched."""
    from qattention_amd import _lib
    c, x, i = _lib.calls(), torch.zeros(4, 2, 64, dtype=torch.float16), torch.zeros(2, dtype=torch.int32)
    assert c.prompt(x, x, x, i, 4, True) is None and c.prompt() is None and c.prompt(1, 2, 3, 4, 5, 6) is None
    assert c.paged(x, x, x, i, i, None, None, True) is None and c.append(x, x, x, x, i, i, None, None) is None
    assert c.compact(x, x, i, i, i) is None and c.copy(x, x, i, i) is None
    with pytest.raises(TypeError):
        c.bind(1, 2)
    with pytest.raises(ValueError):
        c.bind(*[0] * 7, len, len)


@pytest.mark.gpu
def test_tangents_are_refused():
    """A dual tensor in every place of every call; the caches stay as they are."""
    import torch.autograd.forward_ad as fwd
    import qattention_amd as qa
    all_calls(operands())
    o = operands()
    kc, vc = o["Kc"], o["Vc"]
    calls = [(qa.prompt_attention, [o["Q"], o["K"], o["V"]], [o["cu"], 30]),
             (qa.prefix_attention_paged, [o["Q"][:2], kc[0], vc[0]], [o["table"], o["ctx"]]),
             (qa.append_paged_kv, [o["K"][:2], o["V"][:2], kc[0], vc[0]], [o["table"], o["ctx"]]),
             (qa.compact_paged_kv, [kc, vc], [o["table"], o["ctx"], o["path"]]),
             (qa.copy_kv_pages, [kc, vc], [o["src"], o["dst"]])]
    before = kc.clone(), vc.clone()
    for f, ts, rest in calls:
        for i in range(len(ts)):
            with fwd.dual_level():
                dual = [fwd.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(ts)]
                say("tangent", f.__name__, i)
                with pytest.raises(RuntimeError, match="no forward derivative"):
                    f(*dual, *rest)
    assert torch.equal(kc, before[0]) and torch.equal(vc, before[1])


@pytest.mark.gpu
def test_same_without_the_call_module(tmp_path, monkeypatch):
    """All calls where the module is missing: the same bits, by the same kernels."""
    from qattention_amd import _lib
    o = operands()
    direct = all_calls(o)
    monkeypatch.setattr(_lib, "CALLS_PATH", str(tmp_path / "_calls.so"))
    monkeypatch.setattr(_lib, "_calls", None)
    say("no module")
    with pytest.warns(RuntimeWarning, match="go through Python"):
        python = all_calls(o)
    assert _lib.calls().prompt(o["Q"], o["K"], o["V"], o["cu"], 30, False) is None
    for a, b in zip(direct, python):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["prompt", "paged", "append", "compact", "copy"])
def test_other_threads_run_meanwhile(name):
    """A library entry that waits (pause() in its place, until a timer's signal): Python's
    other threads go on.  Nothing is launched."""
    import ctypes
    import signal
    import threading
    import time

    from qattention_amd import _lib
    all_calls(operands())
    c, o = _lib.calls(), operands()
    args = {"prompt": (o["Q"], o["K"], o["V"], o["cu"], 30, True),
            "paged": (o["Q"], o["Kc"][0], o["Vc"][0], o["table"], o["ctx"], o["cu"], 30, True),
            "append": (o["K"], o["V"], o["Kc"][0], o["Vc"][0], o["table"], o["ctx"], o["cu"], 30),
            "compact": (o["Kc"], o["Vc"], o["table"], o["ctx"], o["path"]),
            "copy": (o["Kc"], o["Vc"], o["src"], o["dst"])}[name]
    address = lambda f: ctypes.cast(f, ctypes.c_void_p).value  # noqa: E731
    real = [address(getattr(_lib.lib(), n)) for n in _lib._BOUND]
    fake = list(real)
    fake[("", "prompt", "", "paged", "append", "compact", "copy").index(name)] = address(ctypes.CDLL(None).pause)
    torch_fns = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
    ticks, stop = [], threading.Event()

    def tick():
        while not stop.wait(0.002):
            ticks.append(time.perf_counter())

    thread = threading.Thread(target=tick)
    handler = signal.signal(signal.SIGALRM, lambda *a: None)
    c.bind(*fake, *torch_fns)
    thread.start()
    say("waiting entry", name)
    try:
        timer = signal.setitimer(signal.ITIMER_REAL, 0.3, 0.1)
        a = time.perf_counter()
        out = getattr(c, name)(*args)
        b = time.perf_counter()
    finally:
        signal.setitimer(signal.ITIMER_REAL, *timer)
        signal.signal(signal.SIGALRM, handler)
        c.bind(*real, *torch_fns)
        stop.set()
        thread.join()
    assert out is None and b - a > 0.2  # (pause() ends in an error: the call is left to Python)
    assert sum(a + 0.05 < t < b - 0.05 for t in ticks) >= 10
