"""The local attention kernels where they run as in large calls -- many items, units and
pieces for each CTA -- against their formulas in 64 bits, row by row or value by value,
and their order among streams, graphs and launches.

Bounds.  u = 2^-8 is the most that rounding to bf16 moves a value by, relative to it.
Norms, each row's error: u of the row for bf16, and 1e-5 of |r t| (|y| in the forward), the
scale of the terms that fp32 subtracts, for 30 roundings of 2^-24 or so along a row's sums,
rsqrt and the products.  dg, whole: 1e-5, the fp32 gate.
Attention, each value: a product of 128 terms is off by at most 2^-16 of the sum of its
terms' sizes (fp32, truncated additions), which enters the softmax weights as a relative
error eps; weights and dS round to bf16 (u) where they meet the tensor core, sums over up
to 2^11 steps of 16 keys or queries are off by 2^-12 of the sum of their terms' sizes, and
the result rounds (u).  The gradients are checked as functions of the saved out and lse.
"""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

BF16, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -8


@pytest.fixture(scope="module")
def kda():
    import kda as k
    return k


@pytest.fixture(autouse=True)
def no_device_error(request, kda):
    yield
    torch.cuda.synchronize()
    assert kda.device_error() == 0


def normal(gen, *shape, dtype=BF16):
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


def packed(gen, B, S, heads, D, dtype=BF16):
    """Head rows as slices of one projection."""
    x = normal(gen, B, S, sum(heads) * D, dtype=dtype)
    return [t.unflatten(-1, (-1, D)) for t in x.split([h * D for h in heads], dim=-1)]


# ------------------------------------------------------------------ the norms
def norm64(x, g, cs, dy, eps=1e-6):
    """y, dx, dg and the rows' |r t| in 64 bits; cs: cos, sin of each token."""
    x, g, dy = x.double(), g.double(), dy.double()
    c, s = cs.double()[:, :, None, :, 0], cs.double()[:, :, None, :, 1]
    h = x.shape[-1] // 2
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    n = x * r * g
    y = torch.cat([n[..., :h] * c - n[..., h:] * s, n[..., :h] * s + n[..., h:] * c], -1)
    dn = torch.cat([dy[..., :h] * c + dy[..., h:] * s, dy[..., h:] * c - dy[..., :h] * s], -1)
    t = g * dn
    dx = r * t - x * r ** 3 * (x * t).mean(-1, keepdim=True)
    return y, dx, (x * r * dn).sum((0, 1, 2)), (r * t).norm(dim=-1)


@pytest.mark.gpu
def test_rope_table_of_a_theta_that_no_float_holds(kda):
    """Angles in double precision: theta too.  (sincos and exp2 are good to a few 2^-53 of angles
    of up to 2^17; the entries round to fp32.)"""
    from oracle import ops as ref
    theta = 10000.0 * 8.0 ** (128 / 126)
    got = kda.rope_table(1 << 17, 128, theta)[-64:].double().cpu().numpy()
    assert np.abs(got - ref.rope_table(1 << 17, 128, theta)[-64:]).max() <= 2.0 ** -23


# Enough rows that the forward takes its items in two rounds and the backward's CTAs loop
# over items, queries and keys sharing the CTAs; tokens and heads that leave remainders.
@pytest.mark.gpu
@pytest.mark.parametrize("B,S,QH,KH,D,dtype,docs", [(2, 4099, 33, 5, 128, BF16, False), (1, 5003, 12, 3, 256, F32, True),
                                                    (3, 3001, 18, 2, 64, F32, False), (4, 4099, 25, 4, 64, BF16, True),
                                                    (1, 4501, 17, 3, 256, BF16, False), (1, 9001, 1, 17, 128, F32, True)])
def test_norms_of_many_rows(kda, B, S, QH, KH, D, dtype, docs):
    gen = torch.Generator(device="cuda").manual_seed(S)
    q, k = packed(gen, B, S, (QH, KH), D, dtype)
    gq, gk = (normal(gen, D, dtype=F32) for _ in range(2))
    dq, dk = normal(gen, B, S, QH, D, dtype=dtype), normal(gen, B, S, KH, D, dtype=dtype)
    table = kda.rope_table(S + 3, D)
    pos = torch.randint(0, S + 3, (B, S), generator=gen, device="cuda", dtype=torch.int32) if docs else None
    cs = table[pos.long()] if docs else table[None, :S]
    y = kda.qk_norm_rope(q, k, gq, gk, table, positions=pos)
    grads = kda.qk_norm_rope_backward(dq, dk, q, k, gq, gk, table, positions=pos)
    u = U if dtype == BF16 else 0.0
    for i, (x, g, dy) in enumerate(((q, gq, dq), (k, gk, dk))):
        wy, wdx, wdg, rt = norm64(x, g, cs, dy)
        err = (y[i].double() - wy).norm(dim=-1)
        assert (err <= (u + 1e-5) * wy.norm(dim=-1)).all()
        err = (grads[i].double() - wdx).norm(dim=-1)
        assert (err <= u * wdx.norm(dim=-1) + 1e-5 * rt).all()
        assert (grads[2 + i].double() - wdg).norm() <= 1e-5 * wdg.norm()
    for a, b in zip(grads, kda.qk_norm_rope_backward(dq, dk, q, k, gq, gk, table, positions=pos)):
        assert torch.equal(a, b)


# -------------------------------------------------------------- the attention
def check_window(q, k, v, dout, out, lse, grads, window, sinks):
    """One batch entry, every value of the output and the gradients against its bound."""
    S, QH, D = q.shape
    KH, scale = k.shape[1], 128 ** -0.5
    i = torch.arange(S, device="cuda")
    seen = (i[None] <= i[:, None]) & ((i[:, None] - i[None] < window) | (i[None] < sinks))
    want = {n: 0.0 for n in ("dk", "dv")}
    bound = {n: 0.0 for n in ("dk", "dv")}

    def within(name, got, want, err):
        # (a value whose terms are all zero has a bound of zero, and meets it)
        off = (got.double() - want).abs() - 1.01 * (err + U * want.abs())
        assert (off <= 0.0).all(), (name, off.max().item())

    for h in range(QH):
        g = h // (QH // KH)
        qh, kh, vh, dh, oh = (t.double() for t in (q[:, h], k[:, g], v[:, g], dout[:, h], out[:, h]))
        s = scale * (qh @ kh.T)
        eps = 2.0 ** -16 * scale * (qh.abs() @ kh.abs().T) + 2.0 ** -20
        p = torch.softmax(s.masked_fill(~seen, -torch.inf), dim=-1)
        within("out", out[:, h], p @ vh, (p * (U + 2.0 ** -12 + 2 * eps)) @ vh.abs())
        # gradients, given out and lse
        p = torch.exp2(s / np.log(2.0) - lse[h].double()[:, None]).masked_fill(~seen, 0.0)
        dp, di = dh @ vh.T, (dh * oh).sum(-1, keepdim=True)
        ds = p * (dp - di)
        eta = 2.0 ** -16 * (dh.abs() @ vh.abs().T + (dh * oh).abs().sum(-1, keepdim=True))
        ds_err = (U + 2.0 ** -12 + eps) * ds.abs() + p * eta
        within("dq", grads[0][:, h], scale * (ds @ kh), scale * (ds_err @ kh.abs()))
        want["dk"] = want["dk"] + scale * (ds.T @ qh)
        bound["dk"] = bound["dk"] + scale * (ds_err.T @ qh.abs())
        want["dv"] = want["dv"] + p.T @ dh
        bound["dv"] = bound["dv"] + (p * (U + 2.0 ** -12 + eps)).T @ dh.abs()
        if (h + 1) % (QH // KH) == 0:
            within("dk", grads[1][:, g], want["dk"], bound["dk"])
            within("dv", grads[2][:, g], want["dv"], bound["dv"])
            for d in (want, bound):
                d.update(dk=0.0, dv=0.0)


# Five units of the forward and more for each CTA: short ones, and long ones of uneven walks.
@pytest.mark.gpu
@pytest.mark.parametrize("B,S,QH,KH,window,sinks", [(4, 2100, 32, 8, 62, 0), (2, 1500, 64, 16, 1, 3),
                                                    (3, 4700, 16, 2, 500, 0), (1, 9000, 24, 8, 1000, 130),
                                                    (2, 2100, 48, 3, 2100, 4)])
def test_window_of_many_units(kda, B, S, QH, KH, window, sinks):
    gen = torch.Generator(device="cuda").manual_seed(S)
    q, dout = normal(gen, B, S, QH, 128), normal(gen, B, S, QH, 128)
    k, v = normal(gen, B, S, KH, 128), normal(gen, B, S, KH, 128)

    def step():
        out, lse = kda.gqa_window_lse(q, k, v, window, sinks)
        return out, lse, *kda.gqa_window_backward(dout, q, k, v, out, lse, window, sinks)

    first = step()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, step()))
    out, lse, *grads = first
    for b in range(B):
        check_window(q[b], k[b], v[b], dout[b], out[b], lse[b], [t[b] for t in grads], window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["packed", "heads first"])
def test_window_of_views_gives_the_bits_of_their_copies(kda, layout):
    gen = torch.Generator(device="cuda").manual_seed(11)
    B, S, QH, KH = 2, 700, 6, 2
    if layout == "packed":
        q, k, v = packed(gen, B, S, (QH, KH, KH), 128)
    else:
        q, k, v = (normal(gen, B, h, S, 128).transpose(1, 2) for h in (QH, KH, KH))
    dout = normal(gen, B, S, QH, 128)
    copies = [t.contiguous() for t in (q, k, v)]
    got, want = [], []
    for args, to in (((q, k, v), got), (copies, want)):
        out, lse = kda.gqa_window_lse(*args, 90, 140)
        to += [out, lse, *kda.gqa_window_backward(dout, *args, out, lse, 90, 140)]
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def layer(kda, q, k, v, dout, g, table, n):
    """Every kernel of the forward, the backward and the decode, one behind the other."""
    a, b = kda.qk_norm_rope(q, k, g, g, table)
    out, lse = kda.gqa_window_lse(a, b, v, 150, 2)
    da, db, dv = kda.gqa_window_backward(dout, a, b, v, out, lse, 150, 2)
    return out, lse, da, db, dv, *kda.qk_norm_rope_backward(da, db, q, k, g, g, table), \
        kda.gqa_window_decode(a[:, -1], b, v, n, 150, 2)


@pytest.mark.gpu
def test_streams_and_graph_replays_give_the_bits_of_plain_calls(kda):
    """The kernels start while the ones before them drain.  A graph replayed with other inputs
    each time must not find what an earlier replay left."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    B, S, QH, KH = 2, 900, 8, 4
    x, dout = normal(gen, B, S, (QH + 2 * KH) * 128), normal(gen, B, S, QH, 128)
    q, k, v = (t.unflatten(-1, (-1, 128)) for t in x.split([QH * 128, KH * 128, KH * 128], dim=-1))
    args = (kda, q, k, v, dout, torch.ones(128, device="cuda"), kda.rope_table(S, 128),
            torch.full((B,), S, dtype=torch.int32, device="cuda"))
    layer(*args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        replayed = layer(*args)
    side = torch.cuda.Stream()
    for _ in range(8):
        x.normal_(generator=gen)
        dout.normal_(generator=gen)
        graph.replay()
        got = [t.clone() for t in replayed]
        torch.cuda.synchronize()
        want = layer(*args)
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            aside = layer(*args)
        torch.cuda.current_stream().wait_stream(side)
        for a, b, c in zip(got, want, aside):
            assert torch.equal(a, b) and torch.equal(c, b)


@pytest.mark.gpu
def test_backward_positions_outside_the_table_give_nan_and_are_reported(kda):
    gen = torch.Generator(device="cuda").manual_seed(7)
    q, k = normal(gen, 2, 3, 5, 128), normal(gen, 2, 3, 2, 128)
    dq, dk = normal(gen, 2, 3, 5, 128), normal(gen, 2, 3, 2, 128)
    g, table = torch.ones(128, device="cuda"), kda.rope_table(4, 128)
    good = torch.tensor([[0, 3, 1], [2, 0, 3]], dtype=torch.int32, device="cuda")
    bad = good.clone()
    bad[0, 1], bad[1, 2] = 4, -1
    want = kda.qk_norm_rope_backward(dq, dk, q, k, g, g, table, positions=good)
    got = kda.qk_norm_rope_backward(dq, dk, q, k, g, g, table, positions=bad)
    torch.cuda.synchronize()
    assert kda.device_error() == 8
    off = good != bad
    for a, b in zip(got[:2], want[:2]):
        assert torch.isnan(a[off]).all() and torch.equal(a[~off], b[~off])
    for a in got[2:]:  # sums over those rows too
        assert torch.isnan(a).all()
