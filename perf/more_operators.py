"""Cases of packed-prompt attention and of the 4-bit key/value cache, to time and compare them.

Four operators of a decoder's attention over whole contexts (head_dim 128, QH
query heads that share KH key/value heads):

* causal attention of sequences of different lengths that lie one behind the
  other in one buffer of tokens: forward and backward;
* the append that holds new key and value rows in 4 bits, with the values that
  the cache then stands for;
* attention of one new token of each request against that cache.

``own`` selects between the plain form (elementary torch operations in 32 bits,
rounded once) and the calls a user makes of the ``kda`` package.
"""

import math
import random
import sys
from pathlib import Path

import torch

own = False

D = 128
LOG2E = 1.4426950408889634
BLOCK = 16  # tokens of a cache block
BF16 = torch.bfloat16
F32 = torch.float32


def listed():
    return [
        # a handful of short ragged prompts that arrive together, in a buffer with
        # room behind them: latency counts
        {"name": "packed_prompts", "op": "packed", "QH": 6, "KH": 1, "N": 7, "T": 800, "spread": 2.0, "rest": 45},
        # a training batch of documents, packed to 16,384 tokens
        {"name": "packed_docs", "op": "packed", "QH": 32, "KH": 8, "N": 24, "T": 16384, "spread": 1.0, "rest": 0},
        # one long document
        {"name": "packed_long", "op": "packed", "QH": 32, "KH": 8, "N": 1, "T": 32768, "spread": 0.0, "rest": 0},
        # short documents, each head its own keys, ragged, padding behind the last
        {"name": "bwd_odd", "op": "packed_bwd", "QH": 8, "KH": 8, "N": 9, "T": 2051, "spread": 1.0, "rest": 77},
        # a training step's gradients at the attention backward's configuration
        {"name": "bwd_docs", "op": "packed_bwd", "QH": 16, "KH": 8, "N": 12, "T": 8192, "spread": 1.0, "rest": 0},
        # a long document and what fits behind it, more query heads
        {"name": "bwd_long", "op": "packed_bwd", "QH": 32, "KH": 8, "N": 2, "T": 16384, "spread": 0.5, "rest": 0},
        # a decode step: one token of each request, some slots idle
        {"name": "append_step", "op": "append", "B": 16, "KH": 8, "T": 256, "group": 32, "most": 1, "idle": 2},
        # prompts of different lengths go to the cache
        {"name": "append_prompts", "op": "append", "B": 16, "KH": 8, "T": 2048, "group": 64, "most": 1900, "idle": 0},
        # one conversation: the smallest decode call
        {"name": "decode_b1", "op": "decode", "B": 1, "QH": 32, "KH": 8, "T": 8192, "group": 64, "lo": 7001,
         "hi": 7001, "idle": 0, "window": 0, "sinks": 0},
        # a window with sinks, ragged lengths, heads that do not fill the operand
        {"name": "decode_window", "op": "decode", "B": 7, "QH": 12, "KH": 4, "T": 10000, "group": 128, "lo": 300,
         "hi": 9990, "idle": 1, "window": 4096, "sinks": 4},
        # one very long context
        {"name": "decode_long", "op": "decode", "B": 1, "QH": 32, "KH": 8, "T": 131072, "group": 64, "lo": 130001,
         "hi": 130001, "idle": 0, "window": 0, "sinks": 0},
        # a full server: ragged lengths up to the cache's, some slots idle
        {"name": "decode_b64", "op": "decode", "B": 64, "QH": 32, "KH": 8, "T": 16384, "group": 64, "lo": 100,
         "hi": 16384, "idle": 3, "window": 0, "sinks": 0},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    kh = rng.choice([1, 2, 4, 8])
    rep = rng.choice([1, 2, 3, 4, 5, 6, 8, 16])
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
        c = {"op": op, "KH": KH}
        if op in ("packed", "packed_bwd"):
            # where every query sees itself alone the gradients of q and k are zero,
            # and what is computed for them is rounding noise
            least = 2 if op == "packed_bwd" else 1
            c.update(QH=QH, N=_log_int(rng, 1, 64), spread=rng.choice([0.0, 0.5, 1.0, 2.0]))
            c["T"] = _log_int(rng, least * c["N"], 32768)
            c["rest"] = rng.choice([0, 0, 1, rng.randint(0, 300)])
        else:
            c.update(B=_log_int(rng, 1, 64), group=rng.choice([32, 64, 128]))
            c["T"] = _log_int(rng, 16, 131072 if op == "decode" else 8192)
            c["idle"] = rng.randint(0, c["B"] // 4)
            if op == "append":
                c["most"] = 1 if rng.random() < 0.5 else rng.randint(1, c["T"])
            else:
                c.update(QH=QH, window=rng.choice([0, 0, _log_int(rng, 1, 8192)]), sinks=rng.choice([0, 0, 1, 4, 130]))
                c["hi"] = rng.randint(1, c["T"])
                c["lo"] = rng.randint(1, c["hi"])
        w = work(c)
        size = c.get("B", 0) * c["T"] * KH
        if w["bytes"] <= limit[op][0] and w["flops"] <= limit[op][1] and size <= 64 * 16384 * 8:
            return c


# --------------------------------------------------------------- the lengths
def _packed_lengths(case):
    """Lengths of the sequences, T tokens together, all at least 1 (2 for the
    backward); spread 0: equal ones, 2: from a token to most of the buffer."""
    N, T = case["N"], case["T"]
    least = 2 if case["op"] == "packed_bwd" else 1
    rng = random.Random(N * 1000003 + T)
    parts = [math.exp(case["spread"] * rng.gauss(0.0, 1.0)) for _ in range(N)]
    left = T - least * N
    ends, total = [], 0.0
    for p in parts:
        total += p
        ends.append(total)
    cut = [int(left * e / total) for e in ends[:-1]] + [left]
    return [least + b - a for a, b in zip([0] + cut, cut)]


def _decode_lengths(case):
    """Valid tokens of each request, the new one among them; idle slots have none."""
    n = case["B"] - case["idle"]
    step = (case["hi"] - case["lo"]) / max(n - 1, 1)
    return [int(round(case["lo"] + i * step)) for i in range(n)] + [0] * case["idle"]


def _append_counts(case):
    """(cached tokens, new ones) of each request; -1 cached: an idle slot."""
    rng = random.Random(case["B"] * 1000003 + case["T"])
    rows = []
    for _ in range(case["B"] - case["idle"]):
        new = rng.randint(max(1, case["most"] // 4), case["most"])
        rows.append((rng.randint(0, case["T"] - new), new))
    return rows + [(-1, 1)] * case["idle"]


# -------------------------------------------------------------- 4-bit caches
# A cache is (B, KH, blocks, bytes): 16 tokens of a head are 64 bytes of codes
# each and behind them each token's (step, low) pairs, two bfloat16 for a group
# of channels.  A value is code * step + low.
def _code_places(device):
    """Byte and shift of each channel's code in a block: (16, 128) and (128,)."""
    ch = torch.arange(D, device=device)
    t = torch.arange(BLOCK, device=device)[:, None]
    chunk = (ch % 32) // 8 ^ ((t // 2) % 4)
    return t * 64 + chunk * 16 + ch // 32 * 4 + ch % 8 // 2, ch % 2 * 4


def _cache_codes(cache):
    """(B, KH, tokens, 128) whole numbers."""
    at, shift = _code_places(cache.device)
    codes = cache[..., at.flatten()].unflatten(-1, (BLOCK, D))
    return torch.bitwise_and(torch.bitwise_right_shift(codes, shift.to(torch.uint8)), 15).flatten(2, 3)


def _cache_pairs(cache):
    """step and low of every group: (B, KH, tokens, groups) each, in 32 bits."""
    s = cache[..., BLOCK * 64:].contiguous().view(BF16).unflatten(-1, (BLOCK, -1, 2)).flatten(2, 3).to(F32)
    return s[..., 0], s[..., 1]


def _cache_values(cache):
    """(B, KH, tokens, 128) in 32 bits."""
    step, low = _cache_pairs(cache)
    codes = _cache_codes(cache).to(F32).unflatten(-1, (step.shape[-1], -1))
    return (codes * step[..., None] + low[..., None]).flatten(-2)


def _blocks(T):
    return (T + BLOCK - 1) // BLOCK


def _random_cache(B, T, KH, group, gen):
    """A cache whose values are spread as normed keys and values are."""
    n = _blocks(T)
    cache = torch.empty(B, KH, n, BLOCK * (64 + 4 * (D // group)), dtype=torch.uint8, device="cuda")
    cache[..., :BLOCK * 64] = torch.randint(0, 256, (B, KH, n, BLOCK * 64), generator=gen, device="cuda",
                                            dtype=torch.uint8)
    step = 0.3 + 0.1 * torch.rand(B, KH, n, BLOCK * (D // group), generator=gen, device="cuda")
    low = -step * (7.0 + torch.rand(step.shape, generator=gen, device="cuda"))
    cache[..., BLOCK * 64:] = torch.stack((step, low), dim=-1).to(BF16).flatten(-2).view(torch.uint8)
    return cache


# ------------------------------------------------------------------ inputs
def _unit_rows(shape, gen, scale):
    """Rows as the head norms leave them: root mean square `scale`."""
    x = torch.randn(shape, generator=gen, device="cuda")
    return (scale * x / x.square().mean(-1, keepdim=True).sqrt()).to(BF16)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    op, KH = case["op"], case["KH"]
    st = {"case": case}
    if op in ("packed", "packed_bwd"):
        lens = _packed_lengths(case)
        rng.shuffle(lens)
        T = case["T"] + case["rest"]
        st["lens"] = lens
        st["offsets"] = torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)
        st.update(q=_unit_rows((T, case["QH"], D), gen, 1.5), k=_unit_rows((T, KH, D), gen, 1.5),
                  v=torch.randn(T, KH, D, generator=gen, device="cuda", dtype=BF16))
        if op == "packed_bwd":
            st["dout"] = torch.randn(T, case["QH"], D, generator=gen, device="cuda", dtype=BF16)
            st["out"], st["lse"] = _plain_packed(st)  # what the forward left
    elif op == "append":
        rows = _append_counts(case)
        rng.shuffle(rows)
        st["rows"] = rows
        st["lengths"] = torch.tensor([r[0] for r in rows], dtype=torch.int32, device="cuda")
        st["offsets"] = torch.tensor([0] + [r[1] for r in rows], device="cuda").cumsum(0).to(torch.int32)
        n = sum(r[1] for r in rows)
        st["k"] = _unit_rows((n, KH, D), gen, 1.5)
        st["v"] = torch.randn(n, KH, D, generator=gen, device="cuda", dtype=BF16)
        for c in ("k_cache", "v_cache"):
            st[c] = _random_cache(case["B"], case["T"], KH, case["group"], gen)
    else:
        lens = _decode_lengths(case)
        rng.shuffle(lens)
        st["lens"] = lens
        st["lengths"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        st["q"] = _unit_rows((case["B"], case["QH"], D), gen, 1.0)
        for c in ("k_cache", "v_cache"):
            st[c] = _random_cache(case["B"], case["T"], KH, case["group"], gen)
    return st


# ------------------------------------------------------------- plain forms
def _chunks(lens, rows):
    """(first query, end, first key) of runs of queries of one sequence each:
    all scores of a long sequence at once would not fit the card."""
    at = 0
    for n in lens:
        for i0 in range(at, at + n, rows):
            yield i0, min(i0 + rows, at + n), at
        at += n


def _split(x, KH):
    return x.to(F32).unflatten(1, (KH, -1)).permute(1, 2, 0, 3)  # KH rep T D


def _plain_packed(st):
    case = st["case"]
    KH = case["KH"]
    q, k, v = _split(st["q"], KH), _split(st["k"], KH), _split(st["v"], KH)
    out = torch.zeros_like(st["q"])
    lse = torch.zeros(case["QH"], q.shape[2], dtype=F32, device=q.device)
    for i0, i1, lo in _chunks(st["lens"], 512):
        s = torch.matmul(q[:, :, i0:i1], k[:, :, lo:i1].transpose(-1, -2)) * (D ** -0.5)
        hidden = torch.arange(lo, i1, device=q.device) > torch.arange(i0, i1, device=q.device)[:, None]
        s = s.masked_fill(hidden, -math.inf)
        m = s.amax(-1, keepdim=True)
        p = torch.exp(s - m)
        z = p.sum(-1, keepdim=True)
        o = torch.matmul(p / z, v[:, :, lo:i1])
        out[i0:i1] = o.permute(2, 0, 1, 3).flatten(1, 2).to(BF16)
        lse[:, i0:i1] = ((m + torch.log(z)) * LOG2E).squeeze(-1).flatten(0, 1)
    return out, lse


def _plain_packed_bwd(st):
    case = st["case"]
    KH = case["KH"]
    q, k, v = _split(st["q"], KH), _split(st["k"], KH), _split(st["v"], KH)
    do = _split(st["dout"], KH)
    lse = st["lse"].unflatten(0, (KH, -1))[..., None]
    di = (do * _split(st["out"], KH)).sum(-1, keepdim=True)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k[:, 0]), torch.zeros_like(v[:, 0])
    scale = D ** -0.5
    for i0, i1, lo in _chunks(st["lens"], 512):
        qc, doc, kc, vc = q[:, :, i0:i1], do[:, :, i0:i1], k[:, :, lo:i1], v[:, :, lo:i1]
        s = torch.matmul(qc, kc.transpose(-1, -2)) * scale
        hidden = torch.arange(lo, i1, device=q.device) > torch.arange(i0, i1, device=q.device)[:, None]
        p = torch.exp(s - lse[:, :, i0:i1] / LOG2E).masked_fill(hidden, 0.0)
        ds = p * (torch.matmul(doc, vc.transpose(-1, -2)) - di[:, :, i0:i1]) * scale
        dq[:, :, i0:i1] = torch.matmul(ds, kc)
        dk[:, lo:i1] += torch.matmul(ds.transpose(-1, -2), qc).sum(1)
        dv[:, lo:i1] += torch.matmul(p.transpose(-1, -2), doc).sum(1)
    return (dq.permute(2, 0, 1, 3).flatten(1, 2).to(BF16), dk.transpose(0, 1).to(BF16), dv.transpose(0, 1).to(BF16))


def _quantise(x, groups):
    """Codes (whole numbers in 32 bits), steps and lows (bfloat16) of rows (n, KH, 128)."""
    x = x.to(F32).unflatten(-1, (groups, -1))
    low = x.amin(-1)
    step = ((x.amax(-1) - low) * (1.0 / 15.0)).to(BF16).to(F32)
    step = torch.where(step < 2.0 ** -126, torch.zeros_like(step), step)
    inv = torch.where(step > 0, torch.reciprocal(step), torch.zeros_like(step))
    codes = torch.round((x - low[..., None]) * inv[..., None]).clamp(0, 15)
    return codes.flatten(-2), step.to(BF16), low.to(BF16)


def _append_places(st):
    """Source row, request and position of every token that is written."""
    new = (st["offsets"][1:] - st["offsets"][:-1]).long()
    n = st["k"].shape[0]
    b = torch.repeat_interleave(torch.arange(len(new), device=new.device), new, output_size=n)
    pos = st["lengths"].long()[b] + torch.arange(n, device=new.device) - st["offsets"].long()[b]
    live = torch.nonzero(st["lengths"][b] >= 0).squeeze(-1)
    return live, b[live], pos[live]


def _plain_append(st):
    groups = D // st["case"]["group"]
    live, b, pos = _append_places(st)
    at, _ = _code_places(pos.device)
    for x, cache in ((st["k"], st["k_cache"]), (st["v"], st["v_cache"])):
        codes, step, low = _quantise(x[live], groups)
        pairs = codes.to(torch.uint8).unflatten(-1, (-1, 2))
        byte = pairs[..., 0] + pairs[..., 1] * 16  # (n, KH, 64): channels 2 i and 2 i + 1
        heads = torch.arange(x.shape[1], device=pos.device)[None, :, None]
        block, t = (pos // BLOCK)[:, None, None], pos % BLOCK
        cache[b[:, None, None], heads, block, at[t][:, None, ::2]] = byte
        side = torch.stack((step, low), dim=-1).flatten(-2).view(torch.uint8)  # (n, KH, 4 groups)
        where = BLOCK * 64 + t[:, None] * 4 * groups + torch.arange(4 * groups, device=pos.device)
        cache[b[:, None, None], heads, block, where[:, None]] = side
    return tuple(_cache_values(st[c]).to(BF16).transpose(1, 2) for c in ("k_cache", "v_cache"))


def _plain_decode(st):
    case = st["case"]
    KH = case["KH"]
    k, v = _cache_values(st["k_cache"]), _cache_values(st["v_cache"])
    j = torch.arange(k.shape[2], device=k.device)
    n = st["lengths"][:, None]
    window = case["window"] or case["T"]
    seen = (j < n) & ((j >= n - window) | (j < case["sinks"]))
    q = st["q"].to(F32).unflatten(1, (KH, -1))
    s = torch.matmul(q, k.transpose(-1, -2)) * (D ** -0.5)
    s = s.masked_fill(~seen[:, None, None], -math.inf)
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
    s = state
    case = s["case"]
    op = case["op"]
    if not own:
        return {"packed": _plain_packed, "packed_bwd": _plain_packed_bwd, "append": _plain_append,
                "decode": _plain_decode}[op](s)
    kda = _kda()
    if op == "packed":
        plan = kda.packed_plan(s["offsets"], s["q"].shape[0])
        return kda.gqa_packed_lse(s["q"], s["k"], s["v"], plan)
    if op == "packed_bwd":
        plan = kda.packed_plan(s["offsets"], s["q"].shape[0])
        return kda.gqa_packed_backward(s["dout"], s["q"], s["k"], s["v"], s["out"], s["lse"], plan)
    if op == "append":
        kda.kv_append_q4(s["k"], s["v"], s["k_cache"], s["v_cache"], s["lengths"], s["offsets"])
        return kda.kv_read_q4(s["k_cache"]), kda.kv_read_q4(s["v_cache"])
    return kda.gqa_decode_q4(s["q"], s["k_cache"], s["v_cache"], s["lengths"], case["window"] or None, case["sinks"])


# -------------------------------------------------------------------- work
def work(case):
    op, KH = case["op"], case["KH"]
    if op in ("packed", "packed_bwd"):
        QH, T = case["QH"], case["T"]
        q, kv, row = T * QH * D * 2, T * KH * D * 2, T * QH * 4
        pairs = QH * sum(n * (n + 1) // 2 for n in _packed_lengths(case))
        if op == "packed":
            return {"bytes": 2 * q + 2 * kv + row, "flops": 4 * D * pairs}
        return {"bytes": 4 * q + 4 * kv + row, "flops": 10 * D * pairs}
    held = 64 + 4 * (D // case["group"])  # bytes of a row
    if op == "append":
        new = sum(n for at, n in _append_counts(case) if at >= 0)
        slots = case["B"] * _blocks(case["T"]) * BLOCK
        # rows in, held rows out; then every slot is read and its values written
        return {"bytes": 2 * KH * (new * (2 * D + held) + slots * (held + 2 * D)),
                "flops": 2 * KH * D * (6 * new + 2 * slots)}
    seen = 0
    for n in _decode_lengths(case):
        window = case["window"] or case["T"]
        seen += min(n, window) + max(0, min(case["sinks"], n - window))
    return {"bytes": 2 * seen * KH * held + 4 * case["B"] * case["QH"] * D, "flops": 4 * seen * case["QH"] * D}


# ------------------------------------------------------------ 64-bit values
def exact(case, seed):
    st = prepare(case, seed)
    return {"packed": _exact_packed, "packed_bwd": _exact_packed_bwd, "append": _exact_append,
            "decode": _exact_decode}[case["op"]](st)


def _exact_rows(st):
    """(sequence start, first query, end) and the scaled scores' pieces."""
    at = 0
    for n in st["lens"]:
        step = min(n, 2048)
        for i in range(0, n, step):
            yield at, at + i, at + min(i + step, n)
        at += n


def _exact_scores(st, h, lo, i0, i1):
    g = h * st["case"]["KH"] // st["case"]["QH"]
    s = st["q"][i0:i1, h].double() @ st["k"][lo:i1, g].double().T / math.sqrt(float(D))
    return s.masked_fill(torch.ones_like(s, dtype=torch.bool).triu(i0 - lo + 1), -math.inf), g


def _exact_packed(st):
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(st["q"].shape[1], st["q"].shape[0], dtype=torch.float64, device="cuda")
    for lo, i0, i1 in _exact_rows(st):
        for h in range(st["case"]["QH"]):
            s, g = _exact_scores(st, h, lo, i0, i1)
            z = torch.logsumexp(s, dim=-1)
            out[i0:i1, h] = torch.exp(s - z[:, None]) @ st["v"][lo:i1, g].double()
            lse[h, i0:i1] = z / math.log(2.0)
    return out, lse


def _exact_packed_bwd(st):
    dq = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    dk = torch.zeros(st["k"].shape, dtype=torch.float64, device="cuda")
    dv = torch.zeros_like(dk)
    for lo, i0, i1 in _exact_rows(st):
        for h in range(st["case"]["QH"]):
            s, g = _exact_scores(st, h, lo, i0, i1)
            p = torch.softmax(s, dim=-1)
            do = st["dout"][i0:i1, h].double()
            dp = do @ st["v"][lo:i1, g].double().T
            ds = p * (dp - (p * dp).sum(-1, keepdim=True)) / math.sqrt(float(D))
            dq[i0:i1, h] = ds @ st["k"][lo:i1, g].double()
            dk[lo:i1, g] += ds.T @ st["q"][i0:i1, h].double()
            dv[lo:i1, g] += p.T @ do
    return dq, dk, dv


def _exact_cache(cache):
    """Every value of a cache, channel by channel from the block's definition."""
    B, KH, n, size = cache.shape
    per = (size // BLOCK - 64) // 4
    side = cache[..., BLOCK * 64:].contiguous().view(BF16).double().reshape(B, KH, n, BLOCK, per, 2)
    out = torch.empty(B, n, BLOCK, KH, D, dtype=torch.float64, device="cuda")
    for t in range(BLOCK):
        for ch in range(D):
            word = 16 * ((ch // 8) % 4 ^ (t >> 1) & 3) + 4 * (ch // 32)
            code = (cache[..., 64 * t + word + (ch % 8) // 2] >> (4 * (ch % 2))) & 15
            pair = side[..., t, ch * per // D, :]
            out[:, :, t, :, ch] = (code.double() * pair[..., 0] + pair[..., 1]).transpose(1, 2)
    return out.flatten(1, 2)


def _exact_append(st):
    """The codes are whole numbers that the format defines by operations in 32
    bits: low and step as bfloat16, code = round((x - low) * (1 / step))."""
    group = st["case"]["group"]
    outs = []
    for x, cache in ((st["k"], st["k_cache"]), (st["v"], st["v_cache"])):
        values = _exact_cache(cache)
        rows = x.float().reshape(x.shape[0], x.shape[1], D // group, group)
        low, high = rows.min(-1).values, rows.max(-1).values
        step = ((high - low) * torch.tensor(1.0 / 15.0, dtype=F32, device="cuda")).bfloat16().float()
        fine = step >= 2.0 ** -126
        inv = torch.where(fine, 1.0 / step, torch.zeros_like(step))
        code = torch.round((rows - low[..., None]) * inv[..., None]).clamp(max=15.0).double()
        held = (code * torch.where(fine, step, torch.zeros_like(step)).double()[..., None] + low.double()[..., None])
        held = held.reshape(x.shape)
        at = 0
        for b, (cached, new) in enumerate(st["rows"]):
            if cached >= 0:
                values[b, cached:cached + new] = held[at:at + new]
            at += new
        outs.append(values)
    return tuple(outs)


def _exact_decode(st):
    case = st["case"]
    KH, rep = case["KH"], case["QH"] // case["KH"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    keys, values = _exact_cache(st["k_cache"]), _exact_cache(st["v_cache"])
    for b, n in enumerate(st["lens"]):
        if n == 0:
            continue
        lo = max(0, n - (case["window"] or case["T"]))
        j = torch.cat((torch.arange(min(case["sinks"], lo), device="cuda"), torch.arange(lo, n, device="cuda")))
        k, v = keys[b, j].transpose(0, 1), values[b, j].transpose(0, 1)
        q = st["q"][b].double().unflatten(0, (KH, rep))
        p = torch.softmax(q @ k.transpose(-1, -2) / math.sqrt(float(D)), dim=-1)
        out[b] = (p @ v).flatten(0, 1)
    return out
