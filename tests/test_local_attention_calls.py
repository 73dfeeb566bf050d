"""The local attention operators as they are called: buffers of the caller's, the
registered forms, the C entry points, and what is refused."""

import pytest

torch = pytest.importorskip("torch")

BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def kda():
    import kda as k
    return k


@pytest.fixture(autouse=True)
def no_device_error(request, kda):
    yield
    if "gpu" in request.keywords:
        torch.cuda.synchronize()
        assert kda.device_error() == 0


def rows(*shape, seed=0, dtype=BF16):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("ws", ["expanded", "strided"])
def test_a_workspace_whose_bytes_do_not_lie_together_is_refused(kda, ws):
    """Its size counts bytes that it does not have, or that belong to its neighbours."""
    q, kv = rows(1, 40, 4, 128), rows(1, 40, 2, 128, seed=1)
    out, lse = kda.gqa_window_lse(q, kv, kv, 9)
    g, table = torch.ones(128, device="cuda"), kda.rope_table(40, 128)
    n = 1 << 26
    ws = (torch.empty(1, dtype=torch.uint8, device="cuda").expand(n) if ws == "expanded"
          else torch.empty(2 * n, dtype=torch.uint8, device="cuda")[::2])
    with pytest.raises(ValueError, match="contiguous"):
        kda.gqa_window_backward(out, q, kv, kv, out, lse, 9, workspace=ws)
    with pytest.raises(ValueError, match="contiguous"):
        kda.qk_norm_rope_backward(q, kv, q, kv, g, g, table, workspace=ws)


def test_the_other_operators_do_not_need_the_native_binding():
    """It is compiled against one torch; they are called through libkda.so alone."""
    import os
    import subprocess
    import sys

    from conftest import PKG_ROOT
    code = """
import sys
sys.modules["kda._binding"] = None  # as if the file were missing, or did not load
import torch
import kda
try:
    kda.matmul(torch.zeros(4, 4), torch.zeros(4, 4))
except ValueError:
    print("matmul checked its arguments")
try:
    kda.gqa_window(torch.zeros(1, 4, 2, 128), None, None, 2)
except ImportError as e:
    print(e)
"""
    r = subprocess.run([sys.executable, "-c", code], env={**os.environ, "PYTHONPATH": str(PKG_ROOT)},
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    assert "matmul checked its arguments" in r.stdout and "_binding.so is missing" in r.stdout


def test_the_library_builds_without_torch(monkeypatch, tmp_path):
    """For callers of the C ABI alone; the compiler and the linker are stand-ins here."""
    import importlib.util
    import sys

    from conftest import PKG_ROOT
    spec = importlib.util.spec_from_file_location("kda_build", PKG_ROOT / "build.py")
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    obj = tmp_path / "one.o"
    obj.touch()
    monkeypatch.setattr(b, "BUILD", tmp_path)
    monkeypatch.setattr(b, "LIB", tmp_path / "libkda.so")
    monkeypatch.setattr(b, "BINDING", tmp_path / "_binding.so")
    monkeypatch.setattr(b, "_compile", lambda *a: obj)
    ran = []
    monkeypatch.setattr(b.subprocess, "run", lambda cmd, **kw: ran.append(cmd) or type("R", (), {"returncode": 0})())
    monkeypatch.setitem(sys.modules, "torch", None)
    assert b.build() == tmp_path / "libkda.so"
    assert len(ran) == 1 and "-soname=libkda.so" in ran[0]  # the link, nothing else


def strides(*s):
    import ctypes as C
    return (C.c_int64 * 3)(*s)


@pytest.mark.gpu
@pytest.mark.parametrize("odd", [7, -3])
def test_c_entries_take_any_stride_of_an_axis_of_one_entry(kda, odd):
    from kda import _lib
    B, QH, KH, D, T = 1, 4, 1, 128, 24
    g, table = torch.ones(D, device="cuda"), kda.rope_table(T, D)
    stream = torch.cuda.current_stream().cuda_stream

    def call(fn, *args):
        _lib.call(fn, *(a.data_ptr() if isinstance(a, torch.Tensor) else a for a in args), stream)

    for S in (1, 5):
        tok = odd if S == 1 else QH * D, odd if S == 1 else KH * D
        qs, ks = strides(odd, tok[0], D), strides(odd, tok[1], odd)
        q, k, v = rows(B, S, QH, D), rows(B, S, KH, D, seed=1), rows(B, S, KH, D, seed=2)
        qr, kr = kda.qk_norm_rope(q, k, g, g, table)
        a, b = torch.empty_like(q), torch.empty_like(k)
        call("kda_qk_norm_rope", q, k, g, g, table, T, None, 1e-6, a, b, B, S, QH, KH, D, qs, ks, 0)
        assert torch.equal(a, qr) and torch.equal(b, kr)

        kc, vc, kc2, vc2 = (torch.zeros(B, T, KH, D, dtype=BF16, device="cuda") for _ in range(4))
        n = torch.tensor([3], dtype=torch.int32, device="cuda")
        want = kda.qk_norm_rope_append(q, k, v, g, g, table, kc, vc, n)
        cs = strides(odd, KH * D, odd)
        call("kda_qk_norm_rope_append_bf16", q, k, v, g, g, table, T, n, 1e-6, a, kc2, vc2, T, B, S, QH, KH, D, qs, ks, ks,
             cs, cs)
        assert torch.equal(a, want) and torch.equal(kc, kc2) and torch.equal(vc, vc2)

        dq, dk, dgq, dgk = kda.qk_norm_rope_backward(qr, kr, q, k, g, g, table)
        c, d = torch.empty_like(g), torch.empty_like(g)
        nb = _lib._attach(_lib.lib(), "kda_qk_norm_rope_backward_workspace_size")(B, S, QH, KH, D, 0)
        call("kda_qk_norm_rope_backward", qr, kr, q, k, g, g, table, T, None, 1e-6, a, b, c, d, B, S, QH, KH, D, qs, ks, 0,
             torch.empty(nb, dtype=torch.uint8, device="cuda"), nb)
        assert torch.equal(a, dq) and torch.equal(b, dk) and torch.equal(c, dgq) and torch.equal(d, dgk)

        out, lse = kda.gqa_window_lse(q, k, v, 3, 1)
        lse2 = torch.empty_like(lse)
        call("kda_gqa_window_bf16", q, k, v, a, lse2, B, S, QH, KH, D, 3, 1, qs, ks, ks)
        assert torch.equal(a, out) and torch.equal(lse, lse2)

        grads = kda.gqa_window_backward(qr, q, k, v, out, lse, 3, 1)
        e = torch.empty_like(v)
        nb = _lib._attach(_lib.lib(), "kda_gqa_window_backward_workspace_size")(B, S, QH, KH, D, 3, 1)
        call("kda_gqa_window_backward_bf16", qr, q, k, v, out, lse, a, b, e, B, S, QH, KH, D, 3, 1, qs, ks, ks,
             torch.empty(nb, dtype=torch.uint8, device="cuda"), nb)
        assert all(torch.equal(x, y) for x, y in zip((a, b, e), grads))

        y, row = kda.gqa_window_decode(q[:, 0], kc, vc, n + S, 3, 1), torch.empty(B, QH, D, dtype=BF16, device="cuda")
        call("kda_gqa_window_decode_bf16", q, kc, vc, n + S, row, B, T, QH, KH, D, 3, 1, strides(odd, D, 0), cs, cs)
        assert torch.equal(row, y)


@pytest.mark.gpu
def test_a_position_outside_its_table_is_not_called_an_expired_wait(kda):
    import ctypes as C

    from kda import _lib
    t, g = rows(1, 3, 2, 128), torch.ones(128, device="cuda")
    pos = torch.tensor([[0, 1, 4]], dtype=torch.int32, device="cuda")
    kda.qk_norm_rope(t, t, g, g, kda.rope_table(4, 128), positions=pos)
    torch.cuda.synchronize()
    word, h = C.c_uint(0), _lib.lib()
    assert h.kda_device_error(C.byref(word), 1) == 1 and word.value == 8  # KDA_INVALID_ARG
    assert "outside its table" in h.kda_last_error().decode()
    assert h.kda_device_error(C.byref(word), 1) == 0 and word.value == 0


@torch.no_grad()
def _stand_in_norm(q, k, gq, gk, table, positions=None, eps=1e-6):
    return q * gq, k * gk


@torch.no_grad()
def _stand_in_norm_backward(dq, dk, q, k, gq, gk, table, positions=None, eps=1e-6):
    return dq * gq, dk * gk, (dq * q).sum((0, 1, 2)), (dk * k).sum((0, 1, 2))


@torch.no_grad()
def _stand_in_window(q, k, v, window, sinks):
    return q * k * v, q[..., 0].float()


@torch.no_grad()
def _stand_in_window_backward(dout, q, k, v, out, lse, window, sinks):
    return dout * k * v, dout * q * v, dout * q * k


@pytest.mark.parametrize("op", ["norm", "window"])
@pytest.mark.parametrize("loss", ["sum", "square"])
def test_second_derivatives_raise(kda, monkeypatch, op, loss):
    """The kernels give first derivatives.  What depends on a gradient must not lose that
    gradient's own part silently (stand-ins for the kernels: no GPU)."""
    import kda.autograd as ka
    for name, fn in (("qk_norm_rope", _stand_in_norm), ("qk_norm_rope_backward", _stand_in_norm_backward),
                     ("gqa_window_lse", _stand_in_window), ("gqa_window_backward", _stand_in_window_backward)):
        monkeypatch.setattr(ka.ops, name, fn)
    gen = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(1, 3, 2, 4, generator=gen).to(BF16).requires_grad_() for _ in range(3))
    gq, gk = torch.ones(4, dtype=BF16, requires_grad=True), torch.ones(4, dtype=BF16)

    def value():
        y = ka.qk_norm_rope(q, k, gq, gk, None)[0] if op == "norm" else ka.gqa_window(q, k, v, 2)
        return y.sum() if loss == "sum" else y.square().sum()

    want = torch.autograd.grad(value(), q)[0]
    first, = torch.autograd.grad(value(), q, create_graph=True)
    assert torch.equal(first, want)  # first derivatives as ever
    with pytest.raises(RuntimeError, match="second derivatives"):
        (first.square().sum() + q.square().sum()).backward()


@pytest.mark.gpu
def test_registered_forms_are_the_functions(kda):
    """torch.ops.kda.<op>; the append's caches are written in place."""
    q, k, v = rows(2, 20, 4, 128), rows(2, 20, 2, 128, seed=1), rows(2, 20, 2, 128, seed=2)
    g, table = torch.full((128,), 0.5, device="cuda"), kda.rope_table(64, 128)
    pos = torch.arange(40, dtype=torch.int32, device="cuda").view(2, 20)
    for got, want in ((torch.ops.kda.qk_norm_rope(q, k, g, g, table), kda.qk_norm_rope(q, k, g, g, table)),
                      (torch.ops.kda.qk_norm_rope(q, k, g, g, table, pos, 1e-3),
                       kda.qk_norm_rope(q, k, g, g, table, positions=pos, eps=1e-3)),
                      ((torch.ops.kda.gqa_window(q, k, v, 7, 3),), (kda.gqa_window(q, k, v, 7, 3),))):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    caches = [[rows(2, 64, 2, 128, seed=s) for s in (3, 4)] for _ in range(2)]
    n = torch.tensor([0, 31], dtype=torch.int32, device="cuda")
    got = torch.ops.kda.qk_norm_rope_append(q, k, v, g, g, table, *caches[0], n)
    want = kda.qk_norm_rope_append(q, k, v, g, g, table, *caches[1], n)
    assert torch.equal(got, want)
    for a, b, s in zip(*caches, (3, 4)):
        assert torch.equal(a, b) and not torch.equal(a, rows(2, 64, 2, 128, seed=s))
    got = torch.ops.kda.gqa_window_decode(q[:, 0], *caches[0], n + 20, 9, 2)
    assert torch.equal(got, kda.gqa_window_decode(q[:, 0], *caches[1], n + 20, 9, 2))


@pytest.mark.gpu
def test_the_callers_buffers_are_used(kda):
    """out, q_out, k_out and workspace: written there, the same bits, whatever was in them."""
    q, k, v = rows(2, 300, 4, 128), rows(2, 300, 2, 128, seed=1), rows(2, 300, 2, 128, seed=2)
    dout = rows(2, 300, 4, 128, seed=3)
    g, table = torch.full((128,), 0.5, device="cuda"), kda.rope_table(300, 128)

    def nan(t):
        return torch.full_like(t, float("nan"), memory_format=torch.contiguous_format)

    def same(got, buffers, want):
        for a, b, c in zip(got, buffers, want):
            assert a.data_ptr() == b.data_ptr() and torch.equal(a, c) and torch.equal(b, c)

    a, b = nan(q), nan(k)
    same(kda.qk_norm_rope(q, k, g, g, table, q_out=a, k_out=b), (a, b), kda.qk_norm_rope(q, k, g, g, table))
    a = nan(q)
    same((kda.gqa_window(q, k, v, 70, 3, out=a),), (a,), (kda.gqa_window(q, k, v, 70, 3),))
    n = torch.tensor([200, 300], dtype=torch.int32, device="cuda")
    a = nan(q[:, 0])
    same((kda.gqa_window_decode(q[:, 0], k, v, n, 70, 3, out=a),), (a,), (kda.gqa_window_decode(q[:, 0], k, v, n, 70, 3),))
    kc, vc = rows(2, 304, 2, 128), rows(2, 304, 2, 128)
    a, n = nan(q[:, :4]), torch.tensor([3, 300], dtype=torch.int32, device="cuda")
    args = (q[:, :4], k[:, :4], v[:, :4], g, g, kda.rope_table(304, 128), kc, vc, n)
    same((kda.qk_norm_rope_append(*args, q_out=a),), (a,), (kda.qk_norm_rope_append(*args),))

    out, lse = kda.gqa_window_lse(q, k, v, 70, 3)
    calls = ((kda.gqa_window_backward, (dout, q, k, v, out, lse, 70, 3)),
             (kda.qk_norm_rope_backward, (dout, v, q, k, g, g, table)))
    for fn, args in calls:
        want = fn(*args)
        for fill in (0x00, 0x7f, 0xff):
            ws = torch.full((1 << 26,), fill, dtype=torch.uint8, device="cuda")
            for _ in range(2):  # the second time with what the first has left
                assert all(torch.equal(x, y) for x, y in zip(fn(*args, workspace=ws), want))
        with pytest.raises(ValueError, match="bytes required"):
            fn(*args, workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    for bad in (lambda: kda.gqa_window(q, k, v, 70, 3, out=nan(k)),
                lambda: kda.gqa_window(q, k, v, 70, 3, out=torch.empty(2, 4, 300, 128, dtype=BF16, device="cuda").transpose(1, 2)),
                lambda: kda.qk_norm_rope(q, k, g, g, table, q_out=nan(q).float()),
                lambda: kda.gqa_window_decode(q[:, 0], k, v, n, 70, 3, out=nan(q[:, 0]).cpu())):
        with pytest.raises(ValueError):
            bad()
