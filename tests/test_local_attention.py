"""Local attention: the per-head norms with rotation, the sliding window with
sinks, and its decode form, against the float64 restatements in ``oracle.ops``
(which are themselves checked against autograd and differences on the CPU).

Tolerances, relative L2 of a whole output.  Rounding a value to bf16 (8
significant bits) moves it by at most u = 2^-8 of itself, so an output whose
chain rounds k times to bf16 (the result itself, the softmax weights that meet
the tensor core, dS, the saved output) is off by k u at most, and no output may
pass the bf16 gate of the other operators: norms 1; attention and decode 2
(weights, result); dv 2 (weights, result); dq and dk 4 (weights, saved output in
rowsum(dout out), dS, result).  Outputs that stay fp32 (fp32 norms, dgq, dgk) are
held to 1e-5, the fp32 gate of the other operators; the log2-sum-exp of at most
2^11 weights of ex2.approx (2^-22 each) to 1e-5 absolute plus 2^-21 of its value.
"""

import numpy as np
import pytest

from oracle import ops as ref
from oracle.bf16 import to_bf16_rne
from oracle.metrics import GATE_BF16, GATE_FP32, rel_l2

torch = pytest.importorskip("torch")

BF16 = torch.bfloat16


def rounds(k):
    """The bound of an output whose chain rounds k times to bf16."""
    return min(k * 2.0 ** -8, GATE_BF16)


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


def draw(rng, *shape, scale=1.0):
    return to_bf16_rne((scale * rng.normal(size=shape)).astype(np.float32))


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a))
    return (t if dtype is None else t.to(dtype)).cuda()


def host(t):
    return t.detach().double().cpu().numpy()


# --------------------------------------------------------------- the oracle
def test_norm_rope_backward_restatement_matches_autograd():
    rng = np.random.default_rng(0)
    B, S, QH, KH, D = 2, 5, 3, 1, 8
    q, k = rng.normal(size=(B, S, QH, D)), rng.normal(size=(B, S, KH, D))
    gq, gk = rng.normal(size=D), rng.normal(size=D)
    table = ref.rope_table(16, D)
    pos = rng.integers(0, 16, size=(B, S))
    t = [torch.tensor(a, requires_grad=True) for a in (q, k, gq, gk)]
    cs = torch.tensor(table[pos])

    def rows(x, g):
        n = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * g
        z = torch.complex(n[..., : D // 2], n[..., D // 2:]) * torch.view_as_complex(cs.contiguous())[:, :, None]
        return torch.cat([z.real, z.imag], -1)

    yq, yk = rows(t[0], t[2]), rows(t[1], t[3])
    want = ref.qk_norm_rope(q, k, gq, gk, table, pos)
    np.testing.assert_allclose(yq.detach(), want[0], atol=1e-12)
    np.testing.assert_allclose(yk.detach(), want[1], atol=1e-12)
    dq, dk = rng.normal(size=q.shape), rng.normal(size=k.shape)
    torch.autograd.backward([yq, yk], [torch.tensor(dq), torch.tensor(dk)])
    for got, w in zip(ref.qk_norm_rope_backward(dq, dk, q, k, gq, gk, table, pos), t):
        np.testing.assert_allclose(got, w.grad, atol=1e-12)


@pytest.mark.parametrize("S,window,sinks", [(9, 3, 2), (9, 1, 0), (9, 20, 4), (7, 2, 7)])
def test_window_backward_restatement_matches_differences(S, window, sinks):
    rng = np.random.default_rng(S + window)
    q, k, v = rng.normal(size=(1, S, 4, 8)), rng.normal(size=(1, S, 2, 8)), rng.normal(size=(1, S, 2, 8))
    dout = rng.normal(size=q.shape)
    grads = ref.gqa_window_backward(dout, q, k, v, window, sinks)
    for i, g in enumerate(grads):
        for _ in range(6):
            at = tuple(rng.integers(0, n) for n in g.shape)
            f = []
            for step in (1e-5, -1e-5):
                args = [a.copy() for a in (q, k, v)]
                args[i][at] += step
                f.append(np.sum(dout * ref.gqa_window(*args, window, sinks)[0]))
            assert abs((f[0] - f[1]) / 2e-5 - g[at]) < 1e-7


def test_window_restatement_equals_full_attention_and_decode():
    rng = np.random.default_rng(3)
    q, k, v = rng.normal(size=(2, 10, 4, 128)), rng.normal(size=(2, 10, 2, 128)), rng.normal(size=(2, 10, 2, 128))
    full = ref.gqa_full(q, k, v, causal=True, out_layout="bshd")
    np.testing.assert_allclose(ref.gqa_window(q, k, v, 10)[0], full, atol=1e-5)
    out = ref.gqa_window(q, k, v, 3, 2)[0]
    for n in (1, 4, 10):
        got = ref.gqa_window_decode(q[:, n - 1], k, v, [n, n], 3, 2)
        np.testing.assert_allclose(got, out[:, n - 1], atol=1e-12)


# ------------------------------------------------------- refusals on the host
def test_c_entries_reject_bad_arguments(kda):
    """Checked before any launch, so they run without a GPU."""
    import ctypes as C
    from kda import _lib
    s3 = (C.c_int64 * 3)(1024, 512, 128)
    odd = (C.c_int64 * 3)(1024, 511, 128)

    def norm(B=1, S=2, D=128, eps=1e-6, q=16, st=s3, tab=2):
        _lib.call("kda_qk_norm_rope", q, 16, 16, 16, 16, tab, None, eps, 16, 16, B, S, 4, 1, D, st, s3, 0, None)

    def window(S=2, D=128, QH=4, w=1, sinks=0, q=16, st=s3):
        _lib.call("kda_gqa_window_bf16", q, 16, 16, 16, None, 1, S, QH, 1, D, w, sinks, st, s3, s3, None)

    def decode(T=2, D=128, QH=4, w=1, sinks=0, q=16, st=s3):
        _lib.call("kda_gqa_window_decode_bf16", q, 16, 16, 16, 16, 1, T, QH, 1, D, w, sinks, s3, st, s3, None)

    def backward(S=2, w=1, nb=0):
        _lib.call("kda_gqa_window_backward_bf16", 16, 16, 16, 16, 16, 16, 16, 16, 16, 1, S, 4, 1, 128, w, 0, s3, s3,
                  s3, 16, nb, None)

    for bad in (lambda: norm(B=0), lambda: norm(S=0), lambda: norm(eps=-1.0), lambda: norm(q=None),
                lambda: norm(tab=1), lambda: window(S=0), lambda: window(w=0), lambda: window(sinks=-1),
                lambda: window(q=None), lambda: decode(T=0), lambda: decode(w=0), lambda: decode(q=None), lambda: backward(S=0), lambda: backward(w=0),
                lambda: backward(nb=8)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: norm(D=96), lambda: norm(q=8), lambda: norm(st=odd), lambda: window(D=64),
                lambda: window(q=8), lambda: window(st=odd), lambda: decode(D=64), lambda: decode(st=odd)):
        with pytest.raises(kda.KdaError):
            bad()
    with pytest.raises(ValueError):
        window(QH=0)


def test_host_checks_raise_value_error(kda):
    cpu = torch.zeros(1, 4, 2, 128, dtype=BF16)
    with pytest.raises(ValueError, match="CUDA"):
        kda.gqa_window(cpu, cpu, cpu, 2)
    with pytest.raises(ValueError, match="CUDA"):
        torch.ops.kda.gqa_window(cpu, cpu, cpu, 2)
    with pytest.raises(TypeError):
        kda.qk_norm_rope(1.0, cpu, None, None, None)
    with pytest.raises(ValueError):
        kda.rope_table(0, 128)
    with pytest.raises(ValueError):
        kda.rope_table(4, 127)


def test_fake_kernels_give_the_shapes(kda):
    def t(*s, dtype=BF16):
        return torch.empty(*s, device="meta", dtype=dtype)
    g, tab = t(128, dtype=torch.float32), t(16, 64, 2, dtype=torch.float32)
    q, k, cache, n = t(2, 3, 8, 128), t(2, 3, 4, 128), t(2, 16, 4, 128), t(2, dtype=torch.int32)
    a, b = torch.ops.kda.qk_norm_rope(q, k, g, g, tab)
    assert a.shape == q.shape and b.shape == k.shape
    assert torch.ops.kda.qk_norm_rope_append(q, k, k, g, g, tab, cache, cache.clone(), n).shape == q.shape
    assert torch.ops.kda.gqa_window(q, k, k, 4, 1).shape == q.shape
    assert torch.ops.kda.gqa_window_decode(q[:, 0], cache, cache, n, 4, 1).shape == (2, 8, 128)


# ---------------------------------------------------------------------- GPU
@pytest.mark.gpu
@pytest.mark.parametrize("length,D,theta", [(1, 64, 1e4), (300, 128, 1e4), (5000, 256, 5e5), (7, 6, 10.0)])
def test_rope_table(kda, length, D, theta):
    got = host(kda.rope_table(length, D, theta))
    np.testing.assert_allclose(got, ref.rope_table(length, D, theta), rtol=0, atol=2.0 ** -23)


def packed(rng, B, S, QH, KH, D, dtype):
    """q, k, v as slices of one projection, and their values."""
    x = rng.normal(size=(B, S, (QH + 2 * KH) * D)).astype(np.float32)
    if dtype == BF16:
        x = to_bf16_rne(x)
    t = dev(x, dtype).split((QH * D, KH * D, KH * D), dim=-1)
    n = np.split(x, [QH * D, (QH + KH) * D], axis=-1)
    heads = (QH, KH, KH)
    return ([a.unflatten(-1, (h, D)) for a, h in zip(t, heads)],
            [a.reshape(B, S, h, D) for a, h in zip(n, heads)])


NORM_CASES = [(1, 1, 1, 1, 128), (2, 37, 5, 3, 128), (3, 9, 6, 2, 64), (1, 130, 4, 1, 256), (4, 3, 17, 1, 64),
              (1, 700, 32, 8, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("B,S,QH,KH,D", NORM_CASES)
@pytest.mark.parametrize("docs", [False, True])
def test_qk_norm_rope_and_backward(kda, B, S, QH, KH, D, dtype, docs):
    rng = np.random.default_rng(S + D)
    (q, k, _), (nq, nk, _) = packed(rng, B, S, QH, KH, D, dtype)
    nq, nk = nq.copy(), nk.copy()
    gq, gk = (rng.normal(size=D).astype(np.float32) for _ in range(2))
    P = S + 5
    table = kda.rope_table(P, D)
    pos = rng.integers(0, P, size=(B, S)).astype(np.int32) if docs else None
    tpos = dev(pos) if docs else None
    tol = rounds(1) if dtype == BF16 else GATE_FP32
    ntab = host(table)
    got = kda.qk_norm_rope(q, k, dev(gq), dev(gk), table, positions=tpos)
    for a, w in zip(got, ref.qk_norm_rope(nq, nk, gq, gk, ntab, pos)):
        assert a.dtype == dtype and a.shape == w.shape
        assert rel_l2(host(a), w) <= tol
    dq, dk = (rng.normal(size=a.shape).astype(np.float32) for a in (nq, nk))
    if dtype == BF16:
        dq, dk = to_bf16_rne(dq), to_bf16_rne(dk)
    args = (dev(dq, dtype), dev(dk, dtype), q, k, dev(gq), dev(gk), table)
    got = kda.qk_norm_rope_backward(*args, positions=tpos)
    want = ref.qk_norm_rope_backward(dq, dk, nq, nk, gq, gk, ntab, pos)
    for a, w, t in zip(got, want, (tol, tol, GATE_FP32, GATE_FP32)):
        assert a.shape == w.shape
        assert rel_l2(host(a), w) <= t
    # a fixed order of summation: the same bits again
    for a, c in zip(got, kda.qk_norm_rope_backward(*args, positions=tpos)):
        assert torch.equal(a, c)


@pytest.mark.gpu
def test_qk_norm_rope_rows_of_zeros_and_large_values(kda):
    """Zero rows stay zero (eps > 0) with finite gradients; rows of 1e4 norm like rows of 1."""
    rng = np.random.default_rng(5)
    q = draw(rng, 1, 3, 2, 128)
    q[0, 0], q[0, 1] = 0.0, to_bf16_rne(q[0, 1] * 1e4)
    g = np.ones(128, np.float32)
    table = kda.rope_table(3, 128)
    t = dev(q, BF16)
    y, _ = kda.qk_norm_rope(t, t, dev(g), dev(g), table)
    assert rel_l2(host(y), ref.qk_norm_rope(q, q, g, g, host(table))[0]) <= rounds(1)
    assert not host(y)[0, 0].any()
    dy = draw(rng, 1, 3, 2, 128)
    got = kda.qk_norm_rope_backward(dev(dy, BF16), dev(dy, BF16), t, t, dev(g), dev(g), table)
    want = ref.qk_norm_rope_backward(dy, dy, q, q, g, g, host(table))
    for s in range(3):  # each row on its own: their gradients are of very different size
        assert rel_l2(host(got[0])[:, s], want[0][:, s]) <= rounds(1)


@pytest.mark.gpu
def test_positions_outside_the_table_are_reported(kda):
    t = torch.ones(1, 3, 2, 128, dtype=BF16, device="cuda")
    g = torch.ones(128, device="cuda")
    pos = torch.tensor([[0, 4, -1]], dtype=torch.int32, device="cuda")
    y, _ = kda.qk_norm_rope(t, t, g, g, kda.rope_table(4, 128), positions=pos)
    torch.cuda.synchronize()
    assert torch.isfinite(y[:, 0]).all() and torch.isnan(y[:, 1:]).all()
    assert kda.device_error() == 8 and kda.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("B,S,QH,KH,D,layout", [(5, 1, 8, 2, 128, "bthd"), (2, 33, 4, 4, 64, "bhtd"),
                                                (3, 2, 16, 1, 256, "bthd")])
def test_qk_norm_rope_append(kda, B, S, QH, KH, D, layout):
    rng = np.random.default_rng(B + S)
    (q, k, v), (nq, nk, nv) = packed(rng, B, S, QH, KH, D, BF16)
    T = S + 40
    lens = rng.integers(0, T - S + 1, size=B).astype(np.int32)
    lens[1], lens[0] = -1, T - S
    shape = (2, B, T, KH, D) if layout == "bthd" else (2, B, KH, T, D)
    cache = torch.randn(shape, device="cuda").to(BF16)
    before = cache.clone()
    kc, vc = (c if layout == "bthd" else c.transpose(1, 2) for c in cache)
    kb, vb = (c if layout == "bthd" else c.transpose(1, 2) for c in before)
    gq, gk = (rng.normal(size=D).astype(np.float32) for _ in range(2))
    table = kda.rope_table(T, D)
    qo = kda.qk_norm_rope_append(q, k, v, dev(gq), dev(gk), table, kc, vc, dev(lens))
    pos = np.maximum(lens, 0)[:, None] + np.arange(S)
    wq, wk = ref.qk_norm_rope(nq, nk, gq, gk, host(table), pos)
    for b in range(B):
        if lens[b] < 0:
            assert not qo[b].any() and torch.equal(kc[b], kb[b]) and torch.equal(vc[b], vb[b])
            continue
        sl = slice(lens[b], lens[b] + S)
        assert rel_l2(host(qo[b]), wq[b]) <= rounds(1) and rel_l2(host(kc[b, sl]), wk[b]) <= rounds(1)
        assert np.array_equal(host(vc[b, sl]), nv[b].astype(np.float64))
        keep = np.setdiff1d(np.arange(T), np.arange(lens[b], lens[b] + S))
        assert torch.equal(kc[b, keep], kb[b, keep]) and torch.equal(vc[b, keep], vb[b, keep])


@pytest.mark.gpu
def test_append_past_the_cache_is_reported_and_writes_nothing_there(kda):
    t = torch.ones(1, 3, 1, 128, dtype=BF16, device="cuda")
    g = torch.ones(128, device="cuda")
    # one buffer holds both caches and a guard row behind each
    buf = torch.zeros(2, 1, 9, 1, 128, dtype=BF16, device="cuda")
    kc, vc = buf[0, :, :8], buf[1, :, :8]
    n = torch.tensor([6], dtype=torch.int32, device="cuda")
    y = kda.qk_norm_rope_append(t, t, t, g, g, kda.rope_table(16, 128), kc, vc, n)
    torch.cuda.synchronize()
    assert torch.isfinite(y[:, :2]).all() and torch.isnan(y[:, 2]).all()
    assert not buf[:, :, 8].any() and vc[0, 6:8].all()
    assert kda.device_error() == 8


WINDOW_CASES = [
    # B, S, QH, KH, window, sinks
    (1, 1, 1, 1, 1, 0), (1, 2, 2, 1, 1, 0), (2, 128, 4, 2, 128, 0), (1, 129, 2, 2, 64, 1), (1, 256, 3, 1, 1, 3),
    (2, 333, 6, 1, 100, 5), (1, 257, 4, 4, 1000, 4), (1, 700, 4, 2, 128, 130), (1, 1025, 2, 1, 129, 0),
    (1, 640, 8, 2, 255, 256), (3, 515, 2, 2, 384, 128), (1, 900, 2, 1, 17, 900), (1, 300, 16, 1, 40, 1),
]


def window_inputs(B, S, QH, KH, seed, scale=1.5):
    rng = np.random.default_rng(seed)
    return draw(rng, B, S, QH, 128, scale=scale), draw(rng, B, S, KH, 128, scale=scale), draw(rng, B, S, KH, 128), rng


@pytest.mark.gpu
@pytest.mark.parametrize("B,S,QH,KH,window,sinks", WINDOW_CASES)
def test_gqa_window(kda, B, S, QH, KH, window, sinks):
    q, k, v, _ = window_inputs(B, S, QH, KH, S + window)
    out, lse = kda.gqa_window_lse(dev(q, BF16), dev(k, BF16), dev(v, BF16), window, sinks)
    assert torch.equal(out, kda.gqa_window(dev(q, BF16), dev(k, BF16), dev(v, BF16), window, sinks))
    wout, wlse = ref.gqa_window(q, k, v, window, sinks)
    assert rel_l2(host(out), wout) <= rounds(2)
    np.testing.assert_allclose(host(lse), wlse, rtol=2.0 ** -21, atol=1e-5)
    # every row on its own: none may hide behind the others
    row = np.linalg.norm(host(out) - wout, axis=-1) / np.linalg.norm(wout, axis=-1)
    assert row.max() <= 2 * rounds(2)  # a single row of 128 values may be twice the whole's bound


@pytest.mark.gpu
@pytest.mark.parametrize("B,S,QH,KH,window,sinks", [c for c in WINDOW_CASES if c[1] > 1 and c[4] + c[5] > 1])
def test_gqa_window_backward(kda, B, S, QH, KH, window, sinks):
    q, k, v, rng = window_inputs(B, S, QH, KH, S + window)
    dout = draw(rng, B, S, QH, 128)
    args = [dev(a, BF16) for a in (q, k, v)]
    out, lse = kda.gqa_window_lse(*args, window, sinks)
    got = kda.gqa_window_backward(dev(dout, BF16), *args, out, lse, window, sinks)
    want = ref.gqa_window_backward(dout, q, k, v, window, sinks)
    for name, a, w, n in zip(("dq", "dk", "dv"), got, want, (4, 4, 2)):
        assert a.shape == w.shape, name
        assert rel_l2(host(a), w) <= rounds(n), name


@pytest.mark.gpu
def test_window_backward_of_rows_that_see_themselves_alone(kda):
    """window 1, no sinks: the weight is 1, dv = dout summed over the group, dq and dk zero up to rounding."""
    q, k, v, rng = window_inputs(1, 140, 4, 2, 8)
    dout = draw(rng, 1, 140, 4, 128)
    args = [dev(a, BF16) for a in (q, k, v)]
    out, lse = kda.gqa_window_lse(*args, 1, 0)
    assert np.array_equal(host(out), np.repeat(v, 2, axis=2).astype(np.float64))
    dq, dk, dv = kda.gqa_window_backward(dev(dout, BF16), *args, out, lse, 1, 0)
    assert rel_l2(host(dv), dout.reshape(1, 140, 2, 2, 128).sum(3)) <= rounds(2)
    # dP - di cancels to fp32 rounding of two 128-term sums of products: 128 x 2^-24 x |dout| |v| ~ 1e-3
    assert np.abs(host(dq)).max() < 1e-3 and np.abs(host(dk)).max() < 1e-3


@pytest.mark.gpu
def test_gqa_window_with_the_whole_sequence_is_full_attention(kda):
    q, k, v, _ = window_inputs(2, 520, 4, 2, 1, scale=1.0)
    args = [dev(a, BF16) for a in (q, k, v)]
    full = kda.gqa_full(*args, causal=True, out_layout="bshd")
    for w, s in ((520, 0), (10 ** 6, 7), (1, 520)):
        assert rel_l2(host(kda.gqa_window(*args, w, s)), host(full)) <= rounds(2)


@pytest.mark.gpu
def test_gqa_window_strided_operands(kda):
    """q, k, v as slices of one packed projection give the bits of their copies; gradients too."""
    rng = np.random.default_rng(11)
    (q, k, v), _ = packed(rng, 2, 300, 4, 2, 128, BF16)
    c = [t.contiguous() for t in (q, k, v)]
    out, lse = kda.gqa_window_lse(q, k, v, 90, 3)
    cout, clse = kda.gqa_window_lse(*c, 90, 3)
    assert torch.equal(out, cout) and torch.equal(lse, clse)
    dout = dev(draw(rng, 2, 300, 4, 128), BF16)
    for a, b in zip(kda.gqa_window_backward(dout, q, k, v, out, lse, 90, 3),
                    kda.gqa_window_backward(dout, *c, cout, clse, 90, 3)):
        assert rel_l2(host(a), host(b)) <= rounds(1)  # dq adds its blocks in the order they arrive


@pytest.mark.gpu
def test_gqa_window_extreme_scores(kda):
    """Scores of some hundreds: the running maximum carries the row; one key takes all the weight."""
    q, k, v, _ = window_inputs(1, 400, 2, 1, 6, scale=8.0)
    args = [dev(a, BF16) for a in (q, k, v)]
    out, lse = kda.gqa_window_lse(*args, 100, 4)
    wout, wlse = ref.gqa_window(q, k, v, 100, 4)
    assert rel_l2(host(out), wout) <= rounds(2)
    np.testing.assert_allclose(host(lse), wlse, rtol=2.0 ** -21, atol=1e-4)


DECODE_CASES = [
    # B, T, QH, KH, window, sinks, lengths
    (1, 16, 1, 1, 1, 0, [1]), (4, 50, 8, 2, 16, 3, [0, 1, 17, 50]), (3, 700, 12, 4, 300, 130, [700, 301, -1]),
    (2, 5000, 32, 8, 4096, 4, [5000, 4097]), (1, 1500, 16, 1, 900, 1, [1333]), (2, 300, 40, 2, 64, 300, [300, 77]),
    (5, 40, 3, 3, 8, 0, [8, 9, 15, 16, 40]), (1, 260, 6, 2, 10 ** 6, 0, [259]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,QH,KH,window,sinks,lengths", DECODE_CASES)
@pytest.mark.parametrize("layout", ["bthd", "bhtd"])
def test_gqa_window_decode(kda, B, T, QH, KH, window, sinks, lengths, layout):
    rng = np.random.default_rng(T + QH)
    q, k, v = draw(rng, B, QH, 128, scale=1.5), draw(rng, B, T, KH, 128), draw(rng, B, T, KH, 128)
    n = np.array(lengths, np.int32)
    tk, tv = dev(k, BF16), dev(v, BF16)
    for b in range(B):  # what lies past the valid tokens may be anything
        tk[b, max(n[b], 0):] = float("nan")
        tv[b, max(n[b], 0):] = float("nan")
    for b in range(B):  # and what the window has left behind, too
        lo, hi = min(sinks, T), max(n[b] - window, 0)
        tk[b, lo:hi] = float("nan")
        tv[b, lo:hi] = float("inf")
    if layout == "bhtd":
        tk, tv = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (tk, tv))
    out = kda.gqa_window_decode(dev(q, BF16), tk, tv, dev(n), window, sinks)
    want = ref.gqa_window_decode(q, k, v, n, window, sinks)
    assert out.shape == want.shape
    for b in range(B):
        if n[b] <= 0:
            assert not out[b].any()
        else:
            assert rel_l2(host(out[b]), want[b]) <= rounds(2)
    assert torch.equal(out, kda.gqa_window_decode(dev(q, BF16), tk, tv, dev(n), window, sinks))


@pytest.mark.gpu
def test_decode_length_past_the_cache_is_cut_and_reported(kda):
    rng = np.random.default_rng(2)
    q, k, v = (dev(draw(rng, *s), BF16) for s in ((1, 4, 128), (1, 20, 2, 128), (1, 20, 2, 128)))
    n = torch.tensor([21], dtype=torch.int32, device="cuda")
    got = kda.gqa_window_decode(q, k, v, n, 8, 2)
    torch.cuda.synchronize()
    assert kda.device_error() == 8
    assert torch.equal(got, kda.gqa_window_decode(q, k, v, n - 1, 8, 2))


@pytest.mark.gpu
def test_decode_of_a_cache_past_32_bit_offsets(kda):
    """The last rows of a cache of more than 2^31 elements (4.3 GB in bf16)."""
    T, KH = (1 << 31) // (8 * 128) + 64, 8
    k = torch.empty(1, T, KH, 128, dtype=BF16, device="cuda")
    v = torch.empty_like(k)
    k[:, :8], v[:, :8] = 0, 1
    k[:, -200:], v[:, -200:] = 0, 3
    q = torch.ones(1, 8, 128, dtype=BF16, device="cuda")
    n = torch.tensor([T], dtype=torch.int32, device="cuda")
    out = kda.gqa_window_decode(q, k, v, n, 24, 8)  # equal scores: (24 x 3 + 8 x 1) / 32
    assert (out == 2.5).all()
    # and the append that writes there
    new = torch.ones(1, 1, KH, 128, dtype=BF16, device="cuda")
    g = torch.ones(128, device="cuda")
    kda.qk_norm_rope_append(new, new, 5 * new, g, g, kda.rope_table(T, 128), k, v, n - 1)
    assert (v[0, -1] == 5).all() and (v[0, -2] == 3).all()


@pytest.mark.gpu
def test_autograd_layer_and_decode_agree_with_prefill(kda):
    """Norms, rotation and windowed attention as one differentiable layer; then the same
    tokens one at a time through the cache give the prefill's rows."""
    import kda.autograd as ka
    rng = np.random.default_rng(9)
    B, S, QH, KH, W, sinks = 2, 45, 4, 2, 16, 3
    (q, k, v), (nq, nk, nv) = packed(rng, B, S, QH, KH, 128, BF16)
    gq, gk = (1 + 0.1 * rng.normal(size=128).astype(np.float32) for _ in range(2))
    table = kda.rope_table(S, 128)
    leaf = [t.detach().clone().requires_grad_() for t in (q, k, v, dev(gq.astype(np.float32)),
                                                          dev(gk.astype(np.float32)))]
    q1, k1 = ka.qk_norm_rope(leaf[0], leaf[1], leaf[3], leaf[4], table)
    out = ka.gqa_window(q1, k1, leaf[2], W, sinks)
    dout = draw(rng, B, S, QH, 128)
    out.backward(dev(dout, BF16))
    rq, rk = ref.qk_norm_rope(nq, nk, gq, gk, host(table))
    wout = ref.gqa_window(rq, rk, nv, W, sinks)[0]
    assert rel_l2(host(out), wout) <= rounds(4)  # the rotated q and k round too
    dq1, dk1, dv = ref.gqa_window_backward(dout, rq, rk, nv, W, sinks)
    want = ref.qk_norm_rope_backward(dq1, dk1, nq, nk, gq, gk, host(table))
    for t, w in zip(leaf, (want[0], want[1], dv, want[2], want[3])):
        assert rel_l2(host(t.grad), w) <= rounds(8)
    # token by token
    kc = torch.zeros(B, S, KH, 128, dtype=BF16, device="cuda")
    vc = torch.zeros_like(kc)
    n = torch.zeros(B, dtype=torch.int32, device="cuda")
    g1, g2 = leaf[3].detach(), leaf[4].detach()
    for s in range(S):
        qs = kda.qk_norm_rope_append(q[:, s:s + 1], k[:, s:s + 1], v[:, s:s + 1], g1, g2, table, kc, vc, n)
        n += 1
        row = kda.gqa_window_decode(qs[:, 0], kc, vc, n, W, sinks)
        assert rel_l2(host(row), host(out[:, s])) <= rounds(4)
    assert torch.equal(kc, k1.detach())


@pytest.mark.gpu
def test_calls_on_another_stream_and_in_a_graph(kda):
    """Each call runs on the current stream and can be captured."""
    rng = np.random.default_rng(4)
    (q, k, v), _ = packed(rng, 1, 200, 4, 2, 128, BF16)
    g = torch.ones(128, device="cuda")
    table = kda.rope_table(200, 128)
    dout = dev(draw(rng, 1, 200, 4, 128), BF16)
    n = torch.tensor([200], dtype=torch.int32, device="cuda")

    def step():
        a, b = kda.qk_norm_rope(q, k, g, g, table)
        o, lse = kda.gqa_window_lse(a, b, v, 50, 2)
        grads = kda.gqa_window_backward(dout, a, b, v, o, lse, 50, 2)
        return o, kda.gqa_window_decode(a[:, -1], b, v, n, 50, 2), *grads[1:]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_refusals(kda):
    q = torch.zeros(1, 4, 4, 128, dtype=BF16, device="cuda")
    kv = torch.zeros(1, 4, 2, 128, dtype=BF16, device="cuda")
    g = torch.ones(128, device="cuda")
    table = kda.rope_table(4, 128)
    n = torch.ones(1, dtype=torch.int32, device="cuda")
    wide = torch.zeros(1, 4, 2, 132, dtype=BF16, device="cuda")
    for bad in (
        lambda: kda.gqa_window(q, kv, kv, 0), lambda: kda.gqa_window(q, kv, kv, 4, -1),
        lambda: kda.gqa_window(q.float(), kv, kv, 4), lambda: kda.gqa_window(q, kv[:, :3], kv, 4),
        lambda: kda.gqa_window(q[:, :, :3], kv, kv, 4), lambda: kda.gqa_window(q[:, :0], kv[:, :0], kv[:, :0], 4),
        lambda: kda.gqa_window(q[..., :64], kv[..., :64], kv[..., :64], 4),
        lambda: kda.gqa_window(q, wide[..., 4:], kv, 4),          # rows off 16 bytes
        lambda: kda.gqa_window(q, kv[:, :, :1].expand(-1, -1, 2, -1), kv, 4),
        lambda: kda.gqa_window(q, kv, kv.transpose(2, 3).contiguous().transpose(2, 3), 4),
        lambda: kda.gqa_window_backward(q, q, kv, kv, q, torch.zeros(1, 4, 4, device="cuda"), 4,
                                        workspace=torch.empty(8, dtype=torch.uint8, device="cuda")),
        lambda: kda.gqa_window_backward(q, q, kv, kv, q, torch.zeros(1, 4, 5, device="cuda"), 4),
        lambda: kda.qk_norm_rope(q, kv, g[:64], g, table), lambda: kda.qk_norm_rope(q, kv, g, g.to(BF16), table),
        lambda: kda.qk_norm_rope(q, kv, g, g, table[:3]), lambda: kda.qk_norm_rope(q, kv, g, g, table[:, :32]),
        lambda: kda.qk_norm_rope(q, kv.float(), g, g, table), lambda: kda.qk_norm_rope(q, kv, g, g, table, eps=-1.0),
        lambda: kda.qk_norm_rope(q, kv, g, g, table, positions=n),
        lambda: kda.qk_norm_rope(q, kv, g, g, table, positions=torch.zeros(1, 4, dtype=torch.int64, device="cuda")),
        lambda: kda.qk_norm_rope_append(q, kv, kv, g, g, table, kv, kv[:, :3], n),
        lambda: kda.qk_norm_rope_append(q.float(), kv.float(), kv, g, g, table, kv, kv, n),
        lambda: kda.qk_norm_rope_append(q, kv, kv, g, g, table, kv, kv, n.long()),
        lambda: kda.gqa_window_decode(q[:, 0], kv, kv, n, 0), lambda: kda.gqa_window_decode(q, kv, kv, n, 4),
        lambda: kda.gqa_window_decode(q[:, 0], kv, kv, n.float(), 4),
        lambda: kda.gqa_window_decode(q[:, 0, :3], kv, kv, n, 4),
        lambda: kda.gqa_window_decode(q[:, 0], kv.cpu(), kv, n, 4),
    ):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.gpu
def test_example_runs():
    import runpy

    from conftest import REPO
    worst = runpy.run_path(str(REPO / "examples" / "local_attention.py"))["main"]()
    assert worst <= 4 * 2.0 ** -8


def _window64(q, k, v, window, sinks, dout):
    """Output and gradients of one batch entry in 64 bits, on the GPU."""
    S, QH, KH = q.shape[0], q.shape[1], k.shape[1]
    q, k, v = (t.double().transpose(0, 1).requires_grad_() for t in (q, k, v))
    i = torch.arange(S, device="cuda")
    seen = (i[None] <= i[:, None]) & ((i[:, None] - i[None] < window) | (i[None] < sinks))
    outs = []
    for h in range(QH):
        s = (q[h] @ k[h // (QH // KH)].T) * 128 ** -0.5
        outs.append(torch.softmax(s.masked_fill(~seen, -torch.inf), dim=-1) @ v[h // (QH // KH)])
    out = torch.stack(outs)
    grads = torch.autograd.grad(out, (q, k, v), dout.double().transpose(0, 1))
    return tuple(t.transpose(0, 1) for t in (out.detach(), *grads))


# Many units per CTA, each of one or two key blocks: the pipelines run across the
# units' ends all the time.  Every call has to give the same bits.
@pytest.mark.gpu
@pytest.mark.parametrize("B,S,QH,KH,window,sinks", [(1, 4000, 8, 8, 62, 0), (3, 2724, 4, 4, 62, 0), (3, 971, 16, 8, 1, 64),
                                                    (2, 3000, 8, 2, 128, 1), (1, 5000, 12, 4, 1, 0)])
def test_gqa_window_short_units(kda, B, S, QH, KH, window, sinks):
    gen = torch.Generator(device="cuda").manual_seed(5)
    q, dout = (torch.randn(B, S, QH, 128, generator=gen, device="cuda").to(torch.bfloat16) for _ in range(2))
    k, v = (torch.randn(B, S, KH, 128, generator=gen, device="cuda").to(torch.bfloat16) for _ in range(2))
    first = None
    for _ in range(20):
        out, lse = kda.gqa_window_lse(q, k, v, window, sinks)
        got = (out, *kda.gqa_window_backward(dout, q, k, v, out, lse, window, sinks))
        if first is None:
            first = got
        assert all(torch.equal(a, b) for a, b in zip(first, got))
    b = B - 1
    want = _window64(q[b], k[b], v[b], window, sinks, dout[b])
    for name, g, w in zip(("out", "dq", "dk", "dv"), first, want):
        if name in ("dq", "dk") and window + sinks == 1:  # zero up to rounding, as above
            assert g[b].abs().max() < 1e-3
            continue
        # the output's own rounding, the weights' and, for the gradients, dS's and di's
        assert (g[b].double() - w).norm() <= rounds(4) * w.norm(), name
