"""Attention of packed sequences against the float64 restatements in ``oracle.ops``
(checked on the CPU against differences, through those of the windowed attention).

Tolerances, relative L2, as for the windowed attention (``test_local_attention``): rounding
to bf16 moves a value by at most 2^-8 of itself, so an output whose chain rounds k times is
off by k 2^-8 at most, and never past the bf16 gate: the forward 2 (weights, result), dv 2,
dq and dk 4 (weights, saved output in rowsum(dout out), dS, result).  The log2-sum-exp of at
most 2^11 weights of ex2.approx (2^-22 each): 1e-5 absolute plus 2^-21 of its value.
"""

import numpy as np
import pytest

from oracle import ops as ref
from oracle.bf16 import to_bf16_rne
from oracle.metrics import GATE_BF16, rel_l2

torch = pytest.importorskip("torch")

BF16 = torch.bfloat16


def rounds(k):
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


def dev(a, dtype=BF16):
    return torch.from_numpy(np.ascontiguousarray(a)).to(dtype).cuda()


def host(t):
    return t.detach().double().cpu().numpy()


def offsets_of(lens, first=0):
    return np.concatenate([[first], first + np.cumsum(lens)]).astype(np.int32)


# lengths, QH, KH, rows before the first and behind the last
CASES = [
    ([1], 1, 1, 0, 0),
    ([1], 4, 2, 3, 5),
    ([2, 1, 1, 3], 2, 1, 0, 0),
    ([128], 2, 2, 0, 1),
    ([129, 127], 2, 1, 0, 0),
    ([0, 5, 0, 0, 200, 0], 6, 3, 0, 40),
    ([256, 255, 257], 3, 1, 7, 0),
    ([640], 8, 8, 0, 0),
    ([31, 700, 1, 1, 129, 64], 4, 4, 2, 2),
    ([385], 5, 1, 0, 130),
    ([100] * 9, 16, 2, 0, 0),
    ([1] * 40, 2, 2, 0, 1),
    ([1025, 3], 2, 1, 0, 0),
]


def inputs(lens, QH, KH, before, behind, scale=1.5, seed=0):
    rng = np.random.default_rng(sum(lens) + QH + seed)
    T = before + sum(lens) + behind
    q, k, v = draw(rng, T, QH, 128, scale=scale), draw(rng, T, KH, 128, scale=scale), draw(rng, T, KH, 128)
    return q, k, v, offsets_of(lens, before), rng


# --------------------------------------------------------------- the oracle
def test_packed_restatement_is_each_sequence_alone():
    q, k, v, off, rng = inputs([3, 0, 5], 4, 2, 1, 2)
    out, lse = ref.gqa_packed(q, k, v, off)
    assert not out[0].any() and not out[9:].any() and not lse[:, 9:].any()
    for a, b in ((1, 4), (4, 9)):
        full = ref.gqa_full(q[None, a:b], k[None, a:b], v[None, a:b], causal=True, out_layout="bshd")[0]
        np.testing.assert_allclose(out[a:b], full, atol=1e-5)
    dout = draw(rng, *q.shape)
    grads = ref.gqa_packed_backward(dout, q, k, v, off)
    args = [x.astype(np.float64) for x in (q, k, v)]
    for i, g in enumerate(grads):
        assert not g[0].any() and not g[9:].any()
        for at in ((2, 0, 7), (5, 1, 3)):
            f = []
            for step in (1e-5, -1e-5):
                moved = [x.copy() for x in args]
                moved[i][at] += step
                f.append(np.sum(dout * ref.gqa_packed(*moved, off)[0]))
            assert abs((f[0] - f[1]) / 2e-5 - g[at]) < 1e-6


# ------------------------------------------------------- refusals on the host
def test_c_entries_reject_bad_arguments(kda):
    """Checked before any launch, so they run without a GPU."""
    import ctypes as C
    from kda import _lib
    lib = _lib.lib()
    size = _lib._attach(lib, "kda_packed_plan_size")
    work = _lib._attach(lib, "kda_gqa_packed_backward_workspace_size")
    s2, odd = (C.c_int64 * 2)(512, 128), (C.c_int64 * 2)(511, 128)
    nb = size(8, 2)

    def plan(off=16, n=2, T=8, p=16, size=nb):
        _lib.call("kda_packed_plan", off, n, T, p, size, None)

    def forward(q=16, p=16, size=nb, out=16, T=8, QH=4, KH=2, D=128, st=s2):
        _lib.call("kda_gqa_packed_bf16", q, 16, 16, p, size, out, None, 0, T, QH, KH, D, st, s2, s2, None)

    def backward(size=nb, T=8, KH=2, D=128, lse=16, st=s2, ws=16, wb=None):
        wb = work(8, nb, 4, 2, 128) if wb is None else wb
        _lib.call("kda_gqa_packed_backward_bf16", 16, 16, 16, 16, 16, lse, 16, size, 16, 16, 16, 0, T, 4, KH, D, st,
                  s2, s2, ws, wb, None)

    for bad in (lambda: plan(off=None), lambda: plan(p=None), lambda: plan(n=0), lambda: plan(T=0),
                lambda: plan(size=nb - 4), lambda: plan(size=nb + 4), lambda: forward(q=None), lambda: forward(p=None),
                lambda: forward(out=None), lambda: forward(T=0), lambda: forward(KH=3), lambda: forward(size=0),
                lambda: forward(size=nb + 4), lambda: forward(size=2 ** 41), lambda: forward(size=2 ** 64 - 1),
                lambda: forward(T=1000), lambda: backward(size=8), lambda: backward(T=0), lambda: backward(KH=3),
                lambda: backward(lse=None), lambda: backward(ws=None), lambda: backward(wb=64)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: plan(p=8), lambda: plan(T=2 ** 24), lambda: plan(n=2 ** 24), lambda: forward(D=64),
                lambda: forward(q=8), lambda: forward(p=24), lambda: forward(out=8), lambda: forward(st=odd),
                lambda: forward(T=2 ** 24), lambda: backward(D=64), lambda: backward(st=odd), lambda: backward(ws=8)):
        with pytest.raises(kda.KdaError):
            bad()
    assert size(0, 1) == 0 and size(8, 0) == 0 and size(2 ** 24, 1) == 0 and work(8, nb, 4, 3, 128) == 0
    assert work(8, 0, 4, 2, 128) == 0 and work(8, nb, 4, 2, 64) == 0 and work(8, nb + 4, 4, 2, 128) == 0
    # a plan of every size is told apart: the entry reads the number of sequences off its bytes
    for T in (1, 127, 128, 5000):
        assert len({size(T, n) for n in range(1, 200)}) == 199


def test_host_checks_and_fake_kernels(kda):
    cpu = torch.zeros(4, 2, 128, dtype=BF16)
    with pytest.raises(ValueError, match="CUDA"):
        kda.packed_plan(torch.zeros(2, dtype=torch.int32), 4)
    with pytest.raises(ValueError, match="CUDA"):
        torch.ops.kda.gqa_packed(cpu, cpu, cpu, torch.zeros(32, dtype=torch.int32))
    off = torch.empty(6, dtype=torch.int32, device="meta")
    plan = torch.ops.kda.packed_plan(off, 1000)
    from kda import _lib
    assert plan.numel() * 4 == _lib._attach(_lib.lib(), "kda_packed_plan_size")(1000, 5)
    q, k = torch.empty(1000, 8, 128, device="meta", dtype=BF16), torch.empty(1000, 2, 128, device="meta", dtype=BF16)
    assert torch.ops.kda.gqa_packed(q, k, k, plan).shape == q.shape


# ---------------------------------------------------------------------- GPU
@pytest.mark.gpu
@pytest.mark.parametrize("lens,T", [([1], 1), ([0, 0, 3, 0], 9), ([128, 129, 127, 1000], 1390), ([1] * 1500, 1501),
                                    ([5, 0] * 1100, 5600), ([70000, 600000, 1], 700000)])
def test_plan_tables(kda, lens, T):
    off = offsets_of(lens)
    plan = kda.packed_plan(dev(off, torch.int32), T).cpu().numpy()
    n = [(x + 127) // 128 for x in lens]
    E, most = sum(n), T // 128 + len(lens)
    assert plan[1] == E and tuple(plan[3:6]) == (0, off[-1], T)
    assert plan[2] == sum((x + 1) // 2 for x in n)
    assert plan[6:8].view(np.int64)[0] == sum(x * (x + 1) // 2 for x in n)
    want, base, before, steps = [], 0, [], 0
    for s, x in enumerate(n):
        for z in range(x):
            want.append((off[s], lens[s], z, base))
            before.append(steps)
            steps += x - z
        base += x
    want = np.array(want, np.int32).reshape(-1, 4)
    at = 8
    assert np.array_equal(plan[at:at + 4 * E].reshape(-1, 4), want)
    for rows, keep in ((plan[at + 4 * most:][:4 * E], slice(None)),
                       (plan[at + 8 * most:][:4 * plan[2]], want[:, 2] % 2 == 0)):
        rows = rows.reshape(-1, 4)
        assert (np.diff(np.minimum(rows[:, 2], 1023)) <= 0).all()
        assert np.array_equal(rows[np.lexsort(rows.T)], want[keep][np.lexsort(want[keep].T)])
    assert np.array_equal(plan[at + 12 * most:][:2 * E].view(np.int64), before)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [[0, 5, 4, 8], [-1, 3, 4, 8], [0, 3, 4, 9], [0, 2 ** 31 - 1, 4, 8]])
def test_offsets_that_do_not_fit_are_reported(kda, bad):
    plan = kda.packed_plan(torch.tensor(bad, dtype=torch.int32, device="cuda"), 8)
    torch.cuda.synchronize()
    assert kda.device_error() == 8
    q, k, v = (torch.ones(8, 2, 128, dtype=BF16, device="cuda") for _ in range(3))
    out, lse = kda.gqa_packed_lse(q, k, v, plan)  # of no sequence
    assert not out.any() and not lse.any()
    assert not any(g.any() for g in kda.gqa_packed_backward(q, q, k, v, out, lse, plan))


@pytest.mark.gpu
@pytest.mark.parametrize("lens,QH,KH,before,behind", CASES)
def test_gqa_packed_and_backward(kda, lens, QH, KH, before, behind):
    q, k, v, off, rng = inputs(lens, QH, KH, before, behind)
    dout = draw(rng, *q.shape)
    args = [dev(x) for x in (q, k, v)]
    used = np.zeros(len(q), bool)
    used[off[0]:off[-1]] = True
    for x in args:  # rows of no sequence may hold anything
        x[torch.from_numpy(~used).cuda()] = float("nan")
    plan = kda.packed_plan(dev(off, torch.int32), len(q))
    out, lse = kda.gqa_packed_lse(*args, plan)
    assert torch.equal(out, kda.gqa_packed(*args, plan))
    wout, wlse = ref.gqa_packed(q, k, v, off)
    assert not out[torch.from_numpy(~used).cuda()].any()
    np.testing.assert_allclose(host(lse), wlse, rtol=2.0 ** -21, atol=1e-5)
    row = np.linalg.norm(host(out) - wout, axis=-1)[used] / np.linalg.norm(wout, axis=-1)[used]
    assert rel_l2(host(out), wout) <= rounds(2)
    assert row.max() <= 2 * rounds(2)  # a single row of 128 values may be twice the whole's bound
    tdout = dev(dout)
    tdout[torch.from_numpy(~used).cuda()] = float("nan")
    got = kda.gqa_packed_backward(tdout, *args, out, lse, plan)
    want = ref.gqa_packed_backward(dout, q, k, v, off)
    for name, a, w, n in zip(("dq", "dk", "dv"), got, want, (4, 4, 2)):
        assert a.shape == w.shape and not a[torch.from_numpy(~used).cuda()].any(), name
        if name != "dv" and max(lens) == 1:
            # dP - di cancels to fp32 rounding of two 128-term sums of products: 128 x 2^-24 x |dout| |v| ~ 1e-3
            assert np.abs(host(a)).max() < 1e-3
        else:
            assert rel_l2(host(a), w) <= rounds(n), name
    # the same bits again
    for a, b in zip((out, lse, *got), (*kda.gqa_packed_lse(*args, plan),
                                       *kda.gqa_packed_backward(tdout, *args, out, lse, plan))):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_rows_of_no_sequence_stay_in_a_given_output(kda):
    q, k, v, off, _ = inputs([150, 9], 4, 2, 4, 7)
    plan = kda.packed_plan(dev(off, torch.int32), len(q))
    out = torch.full(q.shape, 3.0, dtype=BF16, device="cuda")
    got = kda.gqa_packed(dev(q), dev(k), dev(v), plan, out=out)
    assert got is out or got.data_ptr() == out.data_ptr()
    assert (out[:4] == 3).all() and (out[-7:] == 3).all()
    assert torch.equal(out[4:-7], kda.gqa_packed(dev(q), dev(k), dev(v), plan)[4:-7])


@pytest.mark.gpu
@pytest.mark.parametrize("QH,KH", [(4, 2), (3, 1)])
def test_a_sequence_does_not_depend_on_its_neighbours(kda, QH, KH):
    """NaN, infinities and large values in every other sequence: the same bits."""
    lens = [200, 77, 300, 1, 60]
    q, k, v, off, rng = inputs(lens, QH, KH, 0, 3)
    dout = draw(rng, *q.shape)
    plan = kda.packed_plan(dev(off, torch.int32), len(q))

    def run(q, k, v, dout):
        out, lse = kda.gqa_packed_lse(q, k, v, plan)
        return (out, *kda.gqa_packed_backward(dout, q, k, v, out, lse, plan)), lse

    clean = [dev(x) for x in (q, k, v, dout)]
    want, wlse = run(*clean)
    for s in range(len(lens)):
        keep = slice(off[s], off[s + 1])
        for junk in (float("nan"), float("inf"), 1e30):
            dirty = [torch.full_like(x, junk) for x in clean]
            for d, c in zip(dirty, clean):
                d[keep] = c[keep]
            got, lse = run(*dirty)
            for a, b in zip(got, want):
                assert torch.equal(a[keep], b[keep])
            assert torch.equal(lse[:, keep], wlse[:, keep])


@pytest.mark.gpu
@pytest.mark.parametrize("QH,KH", [(16, 8), (14, 14), (18, 2)])
def test_a_sequence_among_many_is_the_sequence_alone(kda, QH, KH):
    """More blocks than SMs, where a unit has two tiles: the bits of the sequence by itself, whatever
    the others hold, from strided operands, rows of no sequence untouched."""
    lens = [200, 77, 300, 1, 60, 128, 257, 513, 90, 129, 31, 640]
    q, k, v, off, rng = inputs(lens, QH, KH, 5, 9)
    T = len(q)
    qkv = dev(np.concatenate([q, k, v], 1))
    args = qkv.split((QH, KH, KH), dim=1)
    plan = kda.packed_plan(dev(off, torch.int32), T)
    out, lse = kda.gqa_packed_lse(*args, plan)
    for s, n in enumerate(lens):
        keep = slice(off[s], off[s + 1])
        one = kda.packed_plan(torch.tensor([0, n], dtype=torch.int32, device="cuda"), n)
        want, wlse = kda.gqa_packed_lse(*(x[keep].contiguous() for x in args), one)
        assert torch.equal(out[keep], want) and torch.equal(lse[:, keep], wlse)
        dirty = torch.full_like(qkv, (float("nan"), float("inf"), 1e30)[s % 3])
        dirty[keep] = qkv[keep]
        given = torch.full_like(out, 3.0)
        kda.gqa_packed(*dirty.split((QH, KH, KH), dim=1), plan, out=given)
        assert torch.equal(given[keep], want)
        assert (given[:5] == 3).all() and (given[-9:] == 3).all()
    wout, wl = ref.gqa_packed(q, k, v, off)
    assert rel_l2(host(out)[5:-9], wout[5:-9]) <= rounds(2)
    np.testing.assert_allclose(host(lse)[:, 5:-9], wl[:, 5:-9], rtol=2.0 ** -21, atol=1e-5)


@pytest.mark.gpu
def test_a_sequence_alone_is_full_attention(kda):
    rng = np.random.default_rng(1)
    q, k, v = draw(rng, 520, 4, 128), draw(rng, 520, 2, 128), draw(rng, 520, 2, 128)
    plan = kda.packed_plan(torch.tensor([0, 520], dtype=torch.int32, device="cuda"), 520)
    out = kda.gqa_packed(dev(q), dev(k), dev(v), plan)
    full = kda.gqa_full(dev(q)[None], dev(k)[None], dev(v)[None], causal=True, out_layout="bshd")
    assert rel_l2(host(out), host(full[0])) <= rounds(2)


@pytest.mark.gpu
def test_strided_operands(kda):
    """q, k, v as slices of one packed projection give the bits of their copies; gradients too."""
    rng = np.random.default_rng(11)
    T, QH, KH = 333, 4, 2
    qkv = dev(draw(rng, T, QH + 2 * KH, 128))
    q, k, v = qkv.split((QH, KH, KH), dim=1)
    by_head = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    c = [x.contiguous() for x in (q, k, v)]
    plan = kda.packed_plan(torch.tensor([0, 130, 333], dtype=torch.int32, device="cuda"), T)
    dout = dev(draw(rng, T, QH, 128))
    want = kda.gqa_packed_lse(*c, plan)
    wgrad = kda.gqa_packed_backward(dout, *c, *want, plan)
    for x in ((q, k, v), by_head):
        got = kda.gqa_packed_lse(*x, plan)
        for a, b in zip((*got, *kda.gqa_packed_backward(dout, *x, *got, plan)), (*want, *wgrad)):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_extreme_scores(kda):
    """Scores of some hundreds: the running maximum carries the row; one key takes all the weight."""
    q, k, v, off, _ = inputs([400, 130], 2, 1, 0, 0, scale=8.0)
    plan = kda.packed_plan(dev(off, torch.int32), len(q))
    out, lse = kda.gqa_packed_lse(dev(q), dev(k), dev(v), plan)
    wout, wlse = ref.gqa_packed(q, k, v, off)
    assert rel_l2(host(out), wout) <= rounds(2)
    np.testing.assert_allclose(host(lse), wlse, rtol=2.0 ** -21, atol=1e-4)


@pytest.mark.gpu
def test_autograd(kda):
    """Gradients through autograd, of a broadcast input among them; second derivatives raise."""
    import kda.autograd as ka
    q, k, v, off, rng = inputs([90, 140], 4, 2, 0, 6)
    dout = draw(rng, *q.shape)
    plan = kda.packed_plan(dev(off, torch.int32), len(q))
    leaf = [dev(x).requires_grad_() for x in (q, k[:, :1], v)]
    out = ka.gqa_packed(leaf[0], leaf[1].expand(-1, 2, -1).contiguous(), leaf[2], plan)
    out.backward(dev(dout))
    kk = np.repeat(k[:, :1], 2, axis=1)
    want = ref.gqa_packed_backward(dout, q, kk, v, off)
    for t, w, n in zip(leaf, (want[0], want[1].sum(1, keepdims=True), want[2]), (4, 5, 2)):
        assert rel_l2(host(t.grad), w) <= rounds(n)
    with pytest.raises(ValueError, match="expanded"):
        kda.gqa_packed(leaf[0], leaf[1].expand(-1, 2, -1), leaf[2], plan)
    leaf = [dev(x).requires_grad_() for x in (q, k, v)]
    out = ka.gqa_packed(*leaf, plan)
    kda.packed_plan(dev(off, torch.int32), len(q), out=plan)  # perhaps of other sequences: the backward cannot know
    with pytest.raises(RuntimeError, match="inplace operation"):
        out.float().sum().backward()
    with torch.inference_mode():
        kda.packed_plan(dev(off, torch.int32), len(q), out=torch.empty_like(plan))
    g = torch.autograd.grad(ka.gqa_packed(*leaf, plan).float().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        g[0].float().sum().backward()


@pytest.mark.gpu
def test_streams_and_graph_replays_with_new_offsets(kda):
    """Plan, forward and backward on a side stream and in a graph; a replay works on what
    its buffers hold then, the offsets among them."""
    q, k, v, off, rng = inputs([100, 300, 20], 4, 2, 0, 30)
    T = len(q)
    other = offsets_of([1, 350, 64])
    dout = draw(rng, *q.shape)
    args = [dev(x) for x in (q, k, v, dout)]
    toff = dev(off, torch.int32)

    def step():
        plan = kda.packed_plan(toff, T)
        out, lse = kda.gqa_packed_lse(*args[:3], plan)
        return (out, lse, *kda.gqa_packed_backward(args[3], *args[:3], out, lse, plan))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    toff[:len(other)] = dev(other, torch.int32)
    args[0].mul_(0.5)
    for _ in range(3):
        graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, step()))


# Many units and walks per CTA, most of one or two blocks: the pipelines run across their
# ends all the time.  Every call has to give the same bits.
@pytest.mark.gpu
@pytest.mark.parametrize("lens,QH,KH", [([62] * 300, 8, 8), ([130, 1, 255, 128] * 20, 6, 2), ([700, 3] * 12, 16, 2),
                                        ([40] * 500, 4, 4), ([2600], 12, 4), ([5, 1500, 256] * 3, 3, 3)])
def test_many_short_units(kda, lens, QH, KH):
    gen = torch.Generator(device="cuda").manual_seed(5)
    T = sum(lens) + 11
    q, dout = (torch.randn(T, QH, 128, generator=gen, device="cuda").to(BF16) for _ in range(2))
    k, v = (torch.randn(T, KH, 128, generator=gen, device="cuda").to(BF16) for _ in range(2))
    off = offsets_of(lens)
    first = None
    for _ in range(20):
        plan = kda.packed_plan(dev(off, torch.int32), T)  # equal blocks may be in another order
        out, lse = kda.gqa_packed_lse(q, k, v, plan)
        got = (out, *kda.gqa_packed_backward(dout, q, k, v, out, lse, plan))
        first = got if first is None else first
        assert all(torch.equal(a, b) for a, b in zip(first, got))
    for s in {0, len(lens) // 2, len(lens) - 1}:
        a, b = int(off[s]), int(off[s + 1])
        leaf = [t[a:b].double().transpose(0, 1).requires_grad_() for t in (q, k, v)]
        rep = QH // KH
        s_ = leaf[0] @ leaf[1].repeat_interleave(rep, 0).transpose(1, 2) * 128 ** -0.5
        mask = torch.ones(b - a, b - a, dtype=torch.bool, device="cuda").triu(1)
        o = torch.softmax(s_.masked_fill(mask, -torch.inf), -1) @ leaf[2].repeat_interleave(rep, 0)
        want = (o.detach(), *torch.autograd.grad(o, leaf, dout[a:b].double().transpose(0, 1)))
        for name, g, w in zip(("out", "dq", "dk", "dv"), first, want):
            # the output's own rounding, the weights' and, for the gradients, dS's and di's
            assert (g[a:b].double().transpose(0, 1) - w).norm() <= rounds(4) * w.norm(), name


@pytest.mark.gpu
def test_plan_for_other_rows_does_nothing_and_is_reported(kda):
    """24 rows and 25 take plans of one size: only the kernel can tell."""
    q, k, v = (torch.ones(25, 2, 128, dtype=BF16, device="cuda") for _ in range(3))
    plan = kda.packed_plan(torch.tensor([0, 24], dtype=torch.int32, device="cuda"), 24)
    out = torch.full_like(q, 7.0)
    kda.gqa_packed(q, k, v, plan, out=out)
    torch.cuda.synchronize()
    assert kda.device_error() == 8 and (out == 7).all()
    good = kda.packed_plan(torch.tensor([0, 25], dtype=torch.int32, device="cuda"), 25)
    got, lse = kda.gqa_packed_lse(q, k, v, good)
    assert (got == 1).all()
    kda.gqa_packed_backward(q, q, k, v, got, lse, plan)
    torch.cuda.synchronize()
    assert kda.device_error() == 8
    # junk of a plan's size
    kda.gqa_packed(q, k, v, torch.full_like(plan, 12345), out=out)
    torch.cuda.synchronize()
    assert kda.device_error() == 8 and (out == 7).all()


@pytest.mark.gpu
def test_refusals(kda):
    q = torch.zeros(8, 4, 128, dtype=BF16, device="cuda")
    kv = torch.zeros(8, 2, 128, dtype=BF16, device="cuda")
    off = torch.tensor([0, 3, 8], dtype=torch.int32, device="cuda")
    plan = kda.packed_plan(off, 8)
    lse = torch.zeros(4, 8, device="cuda")
    wide = torch.zeros(8, 2, 132, dtype=BF16, device="cuda")
    for bad in (
        lambda: kda.packed_plan(off.long(), 8), lambda: kda.packed_plan(off[:1], 8), lambda: kda.packed_plan(off, 0),
        lambda: kda.packed_plan(off[None], 8), lambda: kda.packed_plan(off.repeat(2)[::2], 8),
        lambda: kda.packed_plan(off, 2 ** 24), lambda: kda.packed_plan(off, 8, out=plan[:-1]),
        lambda: kda.gqa_packed(q, kv, kv, plan[:-1]), lambda: kda.gqa_packed(q, kv, kv, plan.float()),
        lambda: kda.gqa_packed(q, kv, kv, plan.cpu()), lambda: kda.gqa_packed(q, kv, kv, off),
        lambda: kda.gqa_packed(q.float(), kv, kv, plan), lambda: kda.gqa_packed(q[:7], kv, kv, plan),
        lambda: kda.gqa_packed(q[:, :3], kv, kv, plan), lambda: kda.gqa_packed(q[:0], kv[:0], kv[:0], plan),
        lambda: kda.gqa_packed(q[None], kv, kv, plan), lambda: kda.gqa_packed(q[..., :64], kv[..., :64], kv[..., :64], plan),
        lambda: kda.gqa_packed(q, wide[..., 4:], kv, plan), lambda: kda.gqa_packed(q, kv[:, :1].expand(-1, 2, -1), kv, plan),
        lambda: kda.gqa_packed(q, kv, kv, plan, out=q[:, :2]),
        lambda: kda.gqa_packed_backward(q, q, kv, kv, q, lse[:, :7], plan),
        lambda: kda.gqa_packed_backward(q[:, :2], q, kv, kv, q, lse, plan),
        lambda: kda.gqa_packed_backward(q, q, kv, kv, q, lse, off),
        lambda: kda.gqa_packed_backward(q, q, kv, kv, q, lse, plan,
                                        workspace=torch.empty(8, dtype=torch.uint8, device="cuda")),
    ):
        with pytest.raises(ValueError):
            bad()
