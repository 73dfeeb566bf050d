"""Cases of the local-attention operators, to time and compare them.

Three operators of one decoder layer with local attention (head_dim D, QH query
heads that share KH key/value heads):

* the norms of queries and keys for each head with the position rotation in the
  same pass: forward, backward, and the form that appends to a key/value cache;
* causal attention inside a sliding window whose first tokens (sinks) stay
  visible: forward and backward;
* the same attention for one new token of each request, read from the cache.

``own`` selects between the plain form (elementary torch operations in 32 bits,
rounded once) and the calls a user makes of the ``kda`` package.
"""

import math
import random
import sys
from pathlib import Path

import torch

own = False

EPS = 1e-6
THETA = 10000.0
LOG2E = 1.4426950408889634
BF16 = torch.bfloat16
F32 = torch.float32


def listed():
    return [
        # training / prefill of the grouped-query configuration: q and k are
        # slices of one packed projection
        {"name": "norm_b8s4096", "op": "norm", "dtype": "bf16", "B": 8, "S": 4096, "QH": 32, "KH": 8, "D": 128,
         "docs": False},
        # fp32 activations of a small model, ragged token count, packed documents
        {"name": "norm_f32_odd", "op": "norm", "dtype": "f32", "B": 3, "S": 1001, "QH": 12, "KH": 4, "D": 64,
         "docs": True},
        # one training step's gradient at the attention backward's configuration, twice the heads
        {"name": "norm_bwd_b2s4096", "op": "norm_bwd", "dtype": "bf16", "B": 2, "S": 4096, "QH": 32, "KH": 8,
         "D": 128, "docs": False},
        # wide heads, a single key head, a ragged sequence of packed documents
        {"name": "norm_bwd_d256", "op": "norm_bwd", "dtype": "bf16", "B": 1, "S": 777, "QH": 8, "KH": 1, "D": 256,
         "docs": True},
        # a decode step of 64 requests: one token each, latency counts
        {"name": "append_decode", "op": "append", "B": 64, "S": 1, "QH": 32, "KH": 8, "D": 128, "T": 2048},
        # a prefill chunk of a few requests goes to the cache
        {"name": "append_chunk", "op": "append", "B": 4, "S": 1000, "QH": 16, "KH": 8, "D": 128, "T": 4096},
        # a short ragged prompt batch: a launch-bound prefill, one key head
        {"name": "window_short", "op": "window", "B": 3, "S": 333, "QH": 6, "KH": 1, "W": 100, "sinks": 5},
        # a long document: the window is a sixteenth of it
        {"name": "window_s32768", "op": "window", "B": 1, "S": 32768, "QH": 32, "KH": 8, "W": 2048, "sinks": 4},
        # a training step at the attention backward's configuration
        {"name": "window_bwd_s4096", "op": "window_bwd", "B": 1, "S": 4096, "QH": 16, "KH": 8, "W": 1024,
         "sinks": 4},
        # every head its own keys, ragged length, a window and sinks that end inside a block
        {"name": "window_bwd_odd", "op": "window_bwd", "B": 2, "S": 2051, "QH": 8, "KH": 8, "W": 300, "sinks": 130},
        # one conversation: the smallest decode call
        {"name": "decode_b1", "op": "decode", "B": 1, "T": 8192, "QH": 32, "KH": 8, "W": 4096, "sinks": 4,
         "lo": 7001, "hi": 7001, "idle": 0},
        # a full server: ragged lengths up to the cache's, some slots idle
        {"name": "decode_b64", "op": "decode", "B": 64, "T": 16384, "QH": 32, "KH": 8, "W": 4096, "sinks": 4,
         "lo": 100, "hi": 16384, "idle": 3},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    kh = rng.choice([1, 2, 4, 8])
    rep = rng.choice([1, 2, 3, 4, 6, 8, 16])
    while kh * rep > 64:
        rep = rng.choice([1, 2, 3, 4])
    return kh * rep, kh


def draw(rng):
    limit = {}
    for c in listed():
        w = work(c)
        b, f = limit.get(c["op"], (0, 0))
        limit[c["op"]] = (max(b, w["bytes"]), max(f, w["flops"]))
    op = rng.choice(sorted(limit))
    while True:
        QH, KH = _heads(rng)
        c = {"op": op, "B": _log_int(rng, 1, 64 if op in ("append", "decode") else 8), "QH": QH, "KH": KH}
        if op in ("norm", "norm_bwd"):
            c.update(dtype=rng.choice(["bf16", "bf16", "f32"]), S=_log_int(rng, 1, 16384),
                     D=rng.choice([64, 128, 256]), docs=rng.random() < 0.5)
        elif op == "append":
            c.update(S=1 if rng.random() < 0.5 else _log_int(rng, 2, 2048), D=rng.choice([64, 128, 256]))
            c["T"] = c["S"] + _log_int(rng, 16, 4096)
        elif op in ("window", "window_bwd"):
            # where every query sees itself alone the gradients of q and k are zero,
            # and what is computed for them is rounding noise: two tokens at least
            least = 2 if op == "window_bwd" else 1
            c.update(S=_log_int(rng, least, 32768), W=_log_int(rng, least, 4096),
                     sinks=rng.choice([0, 1, 4, 16, 64, 130, 256]))
        else:
            c.update(T=_log_int(rng, 16, 16384), W=_log_int(rng, 1, 8192), sinks=rng.choice([0, 1, 4, 64, 130]))
            c["hi"] = rng.randint(1, c["T"])
            c["lo"] = rng.randint(1, c["hi"])
            c["idle"] = rng.randint(0, c["B"] // 4)
        w = work(c)
        size = c["B"] * c.get("T", 0) * KH * c.get("D", 128)
        if w["bytes"] <= limit[op][0] and w["flops"] <= limit[op][1] and size <= 64 * 16384 * 8 * 128:
            return c


# ------------------------------------------------------------------ inputs
def _dtype(case):
    return F32 if case.get("dtype") == "f32" else BF16


def _lengths(case):
    """Valid tokens of each request after the new one; idle slots have none."""
    B = case["B"]
    n = B - case["idle"]
    step = (case["hi"] - case["lo"]) / max(n - 1, 1)
    return [int(round(case["lo"] + i * step)) for i in range(n)] + [0] * case["idle"]


def _table(length, D, device):
    """cos and sin of every position and frequency, (length, D/2, 2)."""
    inv = THETA ** (-2.0 * torch.arange(D // 2, dtype=torch.float64, device=device) / D)
    ang = torch.arange(length, dtype=torch.float64, device=device)[:, None] * inv
    return torch.stack((ang.cos(), ang.sin()), dim=-1).to(F32).contiguous()


def _gamma(D, gen):
    return 1.0 + 0.1 * torch.randn(D, generator=gen, device="cuda")


def _unit_rows(shape, gen, scale):
    """Rows as the norm and rotation leave them: root mean square `scale`."""
    x = torch.randn(shape, generator=gen, device="cuda")
    return (scale * x / x.square().mean(-1, keepdim=True).sqrt()).to(BF16)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    op, B, QH, KH = case["op"], case["B"], case["QH"], case["KH"]
    st = {"case": case}
    if op in ("norm", "norm_bwd", "append"):
        S, D, dt = case["S"], case["D"], _dtype(case)
        qkv = torch.randn(B, S, (QH + 2 * KH) * D, generator=gen, device="cuda", dtype=dt)
        q, k, v = qkv.split((QH * D, KH * D, KH * D), dim=-1)
        st.update(q=q.unflatten(-1, (QH, D)), k=k.unflatten(-1, (KH, D)), v=v.unflatten(-1, (KH, D)),
                  gq=_gamma(D, gen), gk=_gamma(D, gen))
    if op in ("norm", "norm_bwd"):
        st["table"] = _table(S, D, "cuda")
        st["positions"] = None
        if case["docs"]:  # packed documents: positions restart at each one
            rows = []
            for _ in range(B):
                row = []
                while len(row) < S:
                    row.extend(range(min(rng.randint(1, max(1, S // 3)), S - len(row))))
                rows.append(row)
            st["positions"] = torch.tensor(rows, dtype=torch.int32, device="cuda")
        if op == "norm_bwd":
            st["dq"] = torch.randn(B, S, QH, D, generator=gen, device="cuda", dtype=dt)
            st["dk"] = torch.randn(B, S, KH, D, generator=gen, device="cuda", dtype=dt)
    elif op == "append":
        T = case["T"]
        st["table"] = _table(T, D, "cuda")
        # tokens already in the cache; -1 marks an idle slot
        lens = [rng.randint(0, T - S) for _ in range(B)]
        if B > 4:
            lens[rng.randrange(B)] = -1
        st["lengths"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        st["k_cache"] = torch.randn(B, T, KH, D, generator=gen, device="cuda", dtype=BF16)
        st["v_cache"] = torch.randn(B, T, KH, D, generator=gen, device="cuda", dtype=BF16)
    elif op in ("window", "window_bwd"):
        S = case["S"]
        st.update(q=_unit_rows((B, S, QH, 128), gen, 1.5), k=_unit_rows((B, S, KH, 128), gen, 1.5),
                  v=torch.randn(B, S, KH, 128, generator=gen, device="cuda", dtype=BF16))
        if op == "window_bwd":
            st["dout"] = torch.randn(B, S, QH, 128, generator=gen, device="cuda", dtype=BF16)
            st["out"], st["lse"] = _plain_window(st)  # what the forward left
    else:
        T = case["T"]
        lens = _lengths(case)
        rng.shuffle(lens)
        st["lengths"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        st["q"] = _unit_rows((B, QH, 128), gen, 1.5)
        st["k_cache"] = torch.randn(B, T, KH, 128, generator=gen, device="cuda", dtype=BF16)
        st["v_cache"] = torch.randn(B, T, KH, 128, generator=gen, device="cuda", dtype=BF16)
    return st


# ------------------------------------------------------------- plain forms
def _norm_rope_rows(x, g, cs):
    """x (..., H, D) in 32 bits; cs (..., D/2, 2) of its positions."""
    n = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * g
    a, b = n.chunk(2, dim=-1)
    c, s = cs[..., None, :, 0], cs[..., None, :, 1]
    return torch.cat((a * c - b * s, a * s + b * c), dim=-1)


def _angles(st):
    S = st["case"]["S"]
    if st.get("positions") is not None:
        return st["table"][st["positions"].long()]
    return st["table"][:S][None]


def _plain_norm(st):
    cs = _angles(st)
    dt = st["q"].dtype
    return (_norm_rope_rows(st["q"].to(F32), st["gq"], cs).to(dt),
            _norm_rope_rows(st["k"].to(F32), st["gk"], cs).to(dt))


def _norm_rope_grad(dy, x, g, cs):
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    a, b = dy.chunk(2, dim=-1)
    c, s = cs[..., None, :, 0], cs[..., None, :, 1]
    dn = torch.cat((a * c + b * s, b * c - a * s), dim=-1)
    t = g * dn
    dx = r * t - x * (r * r * r) * (x * t).mean(-1, keepdim=True)
    return dx, (x * r * dn).sum(dim=(0, 1, 2))


def _plain_norm_bwd(st):
    cs = _angles(st)
    dt = st["q"].dtype
    dq, dgq = _norm_rope_grad(st["dq"].to(F32), st["q"].to(F32), st["gq"], cs)
    dk, dgk = _norm_rope_grad(st["dk"].to(F32), st["k"].to(F32), st["gk"], cs)
    return dq.to(dt), dk.to(dt), dgq, dgk


def _plain_append(st):
    B, S = st["case"]["B"], st["case"]["S"]
    lens = st["lengths"].long()
    live = lens >= 0
    pos = lens.clamp(min=0)[:, None] + torch.arange(S, device=lens.device)
    cs = st["table"][pos]
    q = _norm_rope_rows(st["q"].to(F32), st["gq"], cs).to(BF16)
    q = torch.where(live[:, None, None, None], q, torch.zeros_like(q))
    k = _norm_rope_rows(st["k"].to(F32), st["gk"], cs).to(BF16)
    b = torch.arange(B, device=lens.device)[:, None].expand(B, S)
    keep = live[:, None, None, None]
    st["k_cache"][b, pos] = torch.where(keep, k, st["k_cache"][b, pos])
    st["v_cache"][b, pos] = torch.where(keep, st["v"], st["v_cache"][b, pos])
    return q, st["k_cache"], st["v_cache"]


def _query_chunks(case, rows):
    """(first query, end, first window key) of consecutive chunks of queries: all
    scores of a long sequence at once would not fit the card."""
    S, W = case["S"], case["W"]
    for i0 in range(0, S, rows):
        yield i0, min(i0 + rows, S), max(0, i0 - W + 1)


def _chunk_keys(case, i0, i1, lo, device):
    """Key indexes a chunk reads (sinks before the window, then the window's
    keys) and which of them each of its queries sees."""
    n = min(case["sinks"], lo)
    keys = torch.cat((torch.arange(n, device=device), torch.arange(lo, i1, device=device)))
    i = torch.arange(i0, i1, device=device)[:, None]
    seen = (keys <= i) & ((i - keys < case["W"]) | (keys < case["sinks"]))
    return keys, seen


def _plain_window(st):
    case = st["case"]
    B, S, QH, KH = case["B"], case["S"], case["QH"], case["KH"]
    q = st["q"].to(F32).unflatten(2, (KH, QH // KH)).permute(0, 2, 3, 1, 4)  # B KH rep S D
    k = st["k"].to(F32).transpose(1, 2)[:, :, None]
    v = st["v"].to(F32).transpose(1, 2)[:, :, None]
    out = torch.empty(B, S, QH, 128, dtype=BF16, device=q.device)
    lse = torch.empty(B, QH, S, dtype=F32, device=q.device)
    for i0, i1, lo in _query_chunks(case, 512):
        keys, seen = _chunk_keys(case, i0, i1, lo, q.device)
        s = torch.matmul(q[..., i0:i1, :], k[..., keys, :].transpose(-1, -2)) * (128 ** -0.5)
        s = torch.where(seen, s, torch.full_like(s, -math.inf))
        m = s.amax(-1, keepdim=True)
        p = torch.exp(s - m)
        z = p.sum(-1, keepdim=True)
        o = torch.matmul(p / z, v[..., keys, :])
        out[:, i0:i1] = o.permute(0, 3, 1, 2, 4).flatten(2, 3).to(BF16)
        lse[:, :, i0:i1] = ((m + torch.log(z)) * LOG2E).squeeze(-1).flatten(1, 2)
    return out, lse


def _plain_window_bwd(st):
    case = st["case"]
    B, S, QH, KH = case["B"], case["S"], case["QH"], case["KH"]

    def split(x):
        return x.to(F32).unflatten(2, (KH, QH // KH)).permute(0, 2, 3, 1, 4)

    scale = 128 ** -0.5
    q, do, o = split(st["q"]), split(st["dout"]), split(st["out"])
    k = st["k"].to(F32).transpose(1, 2)[:, :, None]
    v = st["v"].to(F32).transpose(1, 2)[:, :, None]
    lse = st["lse"].unflatten(1, (KH, QH // KH))[..., None]
    di = (do * o).sum(-1, keepdim=True)
    dq = torch.empty_like(q)
    dk = torch.zeros(B, KH, S, 128, dtype=F32, device=q.device)
    dv = torch.zeros(B, KH, S, 128, dtype=F32, device=q.device)
    for i0, i1, lo in _query_chunks(case, 512):
        keys, seen = _chunk_keys(case, i0, i1, lo, q.device)
        qc, doc, kc, vc = q[..., i0:i1, :], do[..., i0:i1, :], k[..., keys, :], v[..., keys, :]
        s = torch.matmul(qc, kc.transpose(-1, -2)) * scale
        p = torch.where(seen, torch.exp(s - lse[..., i0:i1, :] / LOG2E), torch.zeros_like(s))
        ds = p * (torch.matmul(doc, vc.transpose(-1, -2)) - di[..., i0:i1, :]) * scale
        dq[..., i0:i1, :] = torch.matmul(ds, kc)
        dk[:, :, keys] += torch.matmul(ds.transpose(-1, -2), qc).sum(2)
        dv[:, :, keys] += torch.matmul(p.transpose(-1, -2), doc).sum(2)
    return (dq.permute(0, 3, 1, 2, 4).flatten(2, 3).to(BF16), dk.transpose(1, 2).to(BF16),
            dv.transpose(1, 2).to(BF16))


def _plain_decode(st):
    case = st["case"]
    B, QH, KH, T = case["B"], case["QH"], case["KH"], case["T"]
    lens = st["lengths"].long()[:, None]
    # window slots of each request (past its start: masked), then the sinks before the window
    n = min(case["W"], T)
    ns = min(case["sinks"], T)
    start = (lens - case["W"]).clamp(min=0)
    win = start + torch.arange(n, device=lens.device)
    sink = torch.arange(ns, device=lens.device).expand(B, ns)
    idx = torch.cat((sink, win), dim=1)
    seen = torch.cat((sink < torch.minimum(start, lens), win < lens), dim=1)
    b = torch.arange(B, device=lens.device)[:, None]
    idx = idx.clamp(max=T - 1)
    k = st["k_cache"][b, idx].to(F32).permute(0, 2, 1, 3)  # B KH n D
    v = st["v_cache"][b, idx].to(F32).permute(0, 2, 1, 3)
    q = st["q"].to(F32).unflatten(1, (KH, QH // KH))
    s = torch.matmul(q, k.transpose(-1, -2)) * (128 ** -0.5)
    s = torch.where(seen[:, None, None], s, torch.full_like(s, -math.inf))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    z = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(z == 0, torch.ones_like(z), z)
    return o.flatten(1, 2).to(BF16)


# ------------------------------------------------------------------- calls
def _kda():
    path = str(Path(__file__).resolve().parent.parent / "kda-for-trainium_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import kda
    return kda


def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        return {"norm": _plain_norm, "norm_bwd": _plain_norm_bwd, "append": _plain_append, "window": _plain_window,
                "window_bwd": _plain_window_bwd, "decode": _plain_decode}[op](state)
    kda = _kda()
    s = state
    if op == "norm":
        return kda.qk_norm_rope(s["q"], s["k"], s["gq"], s["gk"], s["table"], positions=s["positions"], eps=EPS)
    if op == "norm_bwd":
        return kda.qk_norm_rope_backward(s["dq"], s["dk"], s["q"], s["k"], s["gq"], s["gk"], s["table"],
                                         positions=s["positions"], eps=EPS)
    if op == "append":
        q = kda.qk_norm_rope_append(s["q"], s["k"], s["v"], s["gq"], s["gk"], s["table"], s["k_cache"],
                                    s["v_cache"], s["lengths"], eps=EPS)
        return q, s["k_cache"], s["v_cache"]
    if op == "window":
        return kda.gqa_window_lse(s["q"], s["k"], s["v"], case["W"], case["sinks"])
    if op == "window_bwd":
        return kda.gqa_window_backward(s["dout"], s["q"], s["k"], s["v"], s["out"], s["lse"], case["W"],
                                       case["sinks"])
    return kda.gqa_window_decode(s["q"], s["k_cache"], s["v_cache"], s["lengths"], case["W"], case["sinks"])


# -------------------------------------------------------------------- work
def _pairs(S, W, sinks):
    """Visible (query, key) pairs of one head."""
    i = torch.arange(S, dtype=torch.int64)
    seen = torch.minimum(i + 1, torch.tensor(W)) + (i - W + 1).clamp(min=0, max=sinks)
    return int(seen.sum())


def work(case):
    op, B, QH, KH = case["op"], case["B"], case["QH"], case["KH"]
    D = case.get("D", 128)
    if op in ("norm", "norm_bwd"):
        S, es = case["S"], 4 if case["dtype"] == "f32" else 2
        n = B * S * (QH + KH) * D
        extra = S * D * 4 + 2 * D * 4 + (B * S * 4 if case["docs"] else 0)
        if op == "norm":
            return {"bytes": 2 * n * es + extra, "flops": 8 * n}
        return {"bytes": 3 * n * es + extra + 2 * D * 4, "flops": 18 * n}
    if op == "append":
        n = B * case["S"]
        return {"bytes": 2 * n * (QH + 2 * KH) * D * 2 + min(n, case["T"]) * D * 4 + 2 * D * 4 + 4 * B,
                "flops": 8 * n * (QH + KH) * D}
    if op in ("window", "window_bwd"):
        S = case["S"]
        q, kv, row = B * S * QH * D * 2, B * S * KH * D * 2, B * S * QH * 4
        pairs = B * QH * _pairs(S, case["W"], case["sinks"])
        if op == "window":
            return {"bytes": 2 * q + 2 * kv + row, "flops": 4 * D * pairs}
        return {"bytes": 4 * q + 4 * kv + row, "flops": 10 * D * pairs}
    seen = sum(min(n, case["W"]) + max(0, min(case["sinks"], n - case["W"])) for n in _lengths(case))
    return {"bytes": seen * KH * D * 4 + 2 * B * QH * D * 2 + 4 * B, "flops": 4 * seen * QH * D}


# ------------------------------------------------------------ 64-bit values
def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    return {"norm": _exact_norm, "norm_bwd": _exact_norm_bwd, "append": _exact_append, "window": _exact_window,
            "window_bwd": _exact_window_bwd, "decode": _exact_decode}[op](st)


def _exact_rotation(st, pos):
    """Rows rotated as complex numbers (first half + i second half)."""
    t = st["table"].double()
    return torch.complex(t[..., 0], t[..., 1])[pos][..., None, :]


def _exact_positions(st):
    if st.get("positions") is not None:
        return st["positions"].long()
    return torch.arange(st["case"]["S"], device="cuda")[None].expand(st["case"]["B"], -1)


def _exact_rows(x, g, rot):
    x = x.double()
    n = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS) * g.double()
    h = x.shape[-1] // 2
    z = torch.complex(n[..., :h], n[..., h:]) * rot
    return torch.cat((z.real, z.imag), dim=-1)


def _exact_norm(st):
    rot = _exact_rotation(st, _exact_positions(st))
    return _exact_rows(st["q"], st["gq"], rot), _exact_rows(st["k"], st["gk"], rot)


def _exact_norm_bwd(st):
    rot = _exact_rotation(st, _exact_positions(st))
    dx, dg = [], []
    for x, g, dy in ((st["q"], st["gq"], st["dq"]), (st["k"], st["gk"], st["dk"])):
        x, g, dy = x.double(), g.double(), dy.double()
        D = x.shape[-1]
        z = torch.complex(dy[..., :D // 2], dy[..., D // 2:]) * rot.conj()
        dn = torch.cat((z.real, z.imag), dim=-1)
        rms = torch.sqrt((x * x).sum(-1, keepdim=True) / D + EPS)
        unit = x / rms
        t = dn * g
        dx.append((t - unit * ((unit * t).sum(-1, keepdim=True) / D)) / rms)
        dg.append((unit * dn).flatten(0, 2).sum(0))
    return dx[0], dx[1], dg[0], dg[1]


def _exact_append(st):
    S = st["case"]["S"]
    kc, vc = st["k_cache"].double(), st["v_cache"].double()
    q = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(st["lengths"].tolist()):
        if n >= 0:
            rot = _exact_rotation(st, torch.arange(n, n + S, device="cuda"))
            q[b] = _exact_rows(st["q"][b], st["gq"], rot)
            kc[b, n:n + S] = _exact_rows(st["k"][b], st["gk"], rot)
            vc[b, n:n + S] = st["v"][b].double()
    return q, kc, vc


def _exact_scores(st, b, h, i0, i1):
    """Scaled scores of queries [i0, i1) of one head over keys [0, i1), hidden ones -inf."""
    case = st["case"]
    g = h // (case["QH"] // case["KH"])
    lo = 0 if i0 < case["W"] + case["sinks"] else i0 - case["W"] + 1
    j = torch.arange(lo, i1, device="cuda")
    if lo > 0:
        j = torch.cat((torch.arange(case["sinks"], device="cuda"), j))
    i = torch.arange(i0, i1, device="cuda")[:, None]
    k = st["k"][b, j, g].double()
    s = st["q"][b, i0:i1, h].double() @ k.T / math.sqrt(128.0)
    hidden = (j > i) | ((j <= i - case["W"]) & (j >= case["sinks"]))
    return s.masked_fill(hidden, -math.inf), j, g


def _exact_blocks(case):
    rows = 1024 if case["S"] > 1024 else case["S"]
    for b in range(case["B"]):
        for h in range(case["QH"]):
            for i0 in range(0, case["S"], rows):
                yield b, h, i0, min(i0 + rows, case["S"])


def _exact_window(st):
    case = st["case"]
    out = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(case["B"], case["QH"], case["S"], dtype=torch.float64, device="cuda")
    for b, h, i0, i1 in _exact_blocks(case):
        s, j, g = _exact_scores(st, b, h, i0, i1)
        z = torch.logsumexp(s, dim=-1)
        out[b, i0:i1, h] = torch.exp(s - z[:, None]) @ st["v"][b, j, g].double()
        lse[b, h, i0:i1] = z / math.log(2.0)
    return out, lse


def _exact_window_bwd(st):
    case = st["case"]
    dq = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")
    dk = torch.zeros(st["k"].shape, dtype=torch.float64, device="cuda")
    dv = torch.zeros(st["v"].shape, dtype=torch.float64, device="cuda")
    for b, h, i0, i1 in _exact_blocks(case):
        s, j, g = _exact_scores(st, b, h, i0, i1)
        p = torch.softmax(s, dim=-1)
        do = st["dout"][b, i0:i1, h].double()
        dp = do @ st["v"][b, j, g].double().T
        ds = p * (dp - (p * dp).sum(-1, keepdim=True)) / math.sqrt(128.0)
        dq[b, i0:i1, h] = ds @ st["k"][b, j, g].double()
        dk[b, j, g] += ds.T @ st["q"][b, i0:i1, h].double()
        dv[b, j, g] += p.T @ do
    return dq, dk, dv


def _exact_decode(st):
    case = st["case"]
    rep = case["QH"] // case["KH"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(st["lengths"].tolist()):
        if n == 0:
            continue
        lo = max(0, n - case["W"])
        j = torch.arange(lo, n, device="cuda")
        j = torch.cat((torch.arange(min(case["sinks"], lo), device="cuda"), j))
        k = st["k_cache"][b, j].double().transpose(0, 1)
        v = st["v_cache"][b, j].double().transpose(0, 1)
        q = st["q"][b].double().unflatten(0, (case["KH"], rep))
        p = torch.softmax(q @ k.transpose(-1, -2) / math.sqrt(128.0), dim=-1)
        out[b] = (p @ v).flatten(0, 1)
    return out
