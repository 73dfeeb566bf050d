"""The 4-bit decode over the range of numbers that a cache and a query may hold: steps
from 2^-60 to 2^120 and such as differ between a head's groups and between tokens, queries from
2^-100 to 2^119; and a long context.

The bound of a channel, from the kernel's chain.  With weights p (softmax over the visible tokens,
in 64 bits), A = sum p code step, L = sum p |low| and n tokens:
  * the result is rounded to bf16: 2^-8 |want|;
  * weight times step is rounded to fp16: 2^-11 A, and 2^-25 where it falls below the normal numbers,
    in a unit in which the largest weight times step of the head, M, is 2^5 or more: 15 n 2^-30 M;
  * fp32 sums of n terms, and the tensor core's, which are cut off: n 2^-23 (A + A' + L), A' the
    neighbouring channel's (two codes share an operand);
  * scores: a dozen fp32 operations on numbers of S = sum over groups of |step (q . code)| + |low sum q| in
    units of log2: weights are off by 12 x 2^-24 (S + 64) log 2 of themselves, their sum as much.
The queries are small whole numbers times a power of two, exact in the fp16 operands.
"""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_q4_cache import DECODE_CASES, LONG_CASES  # noqa: E402

BF16 = torch.bfloat16
LOG2E = 1.4426950408889634
GROUPS = [32, 64, 128]
# B, blocks, QH, KH: a cluster's walks of 8 warps and of 16, with more than 8 heads, runs, runs of two kv
# heads together, runs with more than 8 heads
WALKS = [(2, 40, 8, 2), (1, 512, 16, 8), (1, 94, 16, 1), (1, 1400, 6, 1), (64, 260, 16, 8), (1, 2600, 16, 1)]


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


def pack(codes, step, low):
    """The bytes of codes (B,KH,T,128) and of steps and lows (B,KH,T,groups), as kda.h lays them out."""
    B, KH, T, _ = codes.shape
    c = codes.reshape(B, KH, T // 16, 16, 128).to(torch.uint8)
    t, ch = torch.arange(16)[:, None], torch.arange(0, 128, 2)
    at = (64 * t + 16 * ((ch % 32 // 8) ^ (t // 2 % 4)) + 4 * (ch // 32) + ch % 8 // 2).flatten()
    rows = torch.empty(B, KH, T // 16, 1024, dtype=torch.uint8, device=codes.device)
    rows[..., at.to(codes.device)] = (c[..., ::2] | c[..., 1::2] << 4).flatten(-2)
    side = torch.stack([step, low], -1).to(BF16).reshape(B, KH, T // 16, -1).view(torch.uint8)
    return torch.cat([rows, side], -1)


class Cache:
    """Random codes with given steps (B,KH,T,groups; powers of two or bf16 numbers) and lows."""

    def __init__(self, gen, step, low, codes=None):
        B, KH, T, n = step.shape
        self.step, self.low = step.to(BF16).double(), low.to(BF16).double()
        if codes is None:
            codes = torch.randint(0, 16, (B, KH, T, 128), generator=gen, device=step.device)
        self.codes, self.group = codes, 128 // n
        self.raw = pack(codes, step, low)

    def head(self, b, g):
        """Code times step and low of every value of a kv head, (T,128) each."""
        wide = [x[b, g].repeat_interleave(self.group, -1) for x in (self.step, self.low)]
        return self.codes[b, g].double() * wide[0], wide[1]


def whole(gen, *shape):
    return torch.randint(-3, 4, shape, generator=gen, device="cuda").double()


def compare(out, q, k, v, lengths, requests=None):
    """Every channel of out (B,QH,128) against the 64-bit value, within the bound above."""
    rep = q.shape[1] // k.raw.shape[1]
    for b in requests if requests is not None else range(q.shape[0]):
        n = int(lengths[b])
        for g in range(k.raw.shape[1]):
            kc, kl = (x[:n] for x in k.head(b, g))
            vc, vl = (x[:n] for x in v.head(b, g))
            for h in range(g * rep, (g + 1) * rep):
                qh = q[b, h].double()
                unit = LOG2E / np.sqrt(128.0)
                s = (kc + kl) @ qh * unit
                groups = [((kc @ (qh * m)).abs() + (kl @ (qh * m)).abs()) * unit
                          for m in torch.eye(128 // k.group, device=q.device, dtype=torch.float64)
                          .repeat_interleave(k.group, 1)]
                size = float(sum(groups).max())
                p = torch.softmax(s / LOG2E, 0)
                want, A, L = p @ (vc + vl), p @ vc, p @ vl.abs()
                M = float((p[:, None] * v.step[b, g, :n]).max())
                A2 = A.unflatten(0, (-1, 2)).flip(1).flatten()
                bound = (2.0 ** -8 * want.abs() + 2.0 ** -11 * A + 15 * n * 2.0 ** -30 * M
                         + n * 2.0 ** -23 * (A + A2 + L)
                         + 2 * 12 * 2.0 ** -24 * (size + 64) * np.log(2.0) * (A + L))
                got = out[b, h].double()
                assert torch.isfinite(got).all(), (b, h)
                off = (got - want).abs() / bound
                assert float(off.max()) <= 1, (b, h, int(off.argmax()), float(off.max()))


def lengths_of(B, T):
    return [max(1, T - 37 * b - (b > 0) * (T // 3)) for b in range(B)]


def spread(B, KH, T, groups, exponents):
    """Steps 2^e, the exponents by group and token as the function gives them."""
    t, g = torch.arange(T, device="cuda")[:, None], torch.arange(groups, device="cuda")
    e = exponents(t, g).double().expand(T, groups)
    return torch.exp2(e).expand(B, KH, T, groups).contiguous()


def test_pack_is_the_layout_of_the_oracle():
    from oracle import ops as ref
    rng = np.random.default_rng(0)
    codes = rng.integers(0, 16, size=(2, 3, 32, 128))
    step = np.exp2(rng.integers(-4, 5, size=(2, 3, 32, 2))).astype(np.float32)
    low = -7 * step
    got = pack(torch.from_numpy(codes), torch.from_numpy(step), torch.from_numpy(low))
    assert np.array_equal(got.numpy(), ref.q4_pack(codes, step, low))


@pytest.mark.gpu
@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("e", [-60, 0, 60, 103, 104, 120])
def test_decode_at_every_size_of_values(kda, group, e):
    """Steps of 2^e: values of -7 to 8 of them, up to 2^123, finite in fp32 and in bf16."""
    gen = torch.Generator(device="cuda").manual_seed(e + 100)
    for B, blocks, QH, KH in ((2, 40, 8, 2), (1, 94, 16, 1), (1, 1400, 6, 1)):
        T = 16 * blocks
        k = Cache(gen, *(spread(B, KH, T, 128 // group, lambda t, g: 0 * t + 0 * g - 3) * f for f in (1, -7)))
        v = Cache(gen, *(spread(B, KH, T, 128 // group, lambda t, g: 0 * t + 0 * g + e) * f for f in (1, -7)))
        q, lengths = whole(gen, B, QH, 128).to(BF16), lengths_of(B, T)
        n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        compare(kda.gqa_decode_q4(q, k.raw, v.raw, n), q, k, v, lengths)


@pytest.mark.gpu
@pytest.mark.parametrize("group", GROUPS)
def test_decode_of_constant_groups(kda, group):
    """Steps of zero beside lows of 2^100, of zero and of -2^120; a lone step among them."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    B, KH, T, groups = 2, 2, 640, 128 // group
    k = Cache(gen, *(spread(B, KH, T, groups, lambda t, g: 0 * t + 0 * g - 3) * f for f in (1, -7)))
    q = whole(gen, B, 8, 128).to(BF16)
    n = torch.tensor([640, 333], dtype=torch.int32, device="cuda")
    for value in (2.0 ** 100, 0.0, -2.0 ** 120):
        step = torch.zeros(B, KH, T, groups, device="cuda", dtype=torch.float64)
        low = torch.full_like(step, value)
        step[:, :, 301], low[:, :, 301] = 1.0, -7.0
        v = Cache(gen, step, low)
        compare(kda.gqa_decode_q4(q, k.raw, v.raw, n), q, k, v, [640, 333])


@pytest.mark.gpu
@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("e", [-100, -60, 60, 107, 118])
def test_decode_of_large_and_small_queries(kda, group, e):
    """|q| up to 3 x 2^e against keys as much smaller: ordinary scores.  (Keys' steps are bf16
    numbers from 2^-121 on.)"""
    gen = torch.Generator(device="cuda").manual_seed(e + 100)
    for B, blocks, QH, KH in ((2, 40, 8, 2), (1, 94, 16, 1)):
        T = 16 * blocks
        k = Cache(gen, *(spread(B, KH, T, 128 // group, lambda t, g: 0 * t + 0 * g - e - 3) * f for f in (1, -7)))
        v = Cache(gen, *(spread(B, KH, T, 128 // group, lambda t, g: 0 * t + 0 * g) * f for f in (1, -7)))
        q = (whole(gen, B, QH, 128) * 2.0 ** e).to(BF16)
        lengths = lengths_of(B, T)
        n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        compare(kda.gqa_decode_q4(q, k.raw, v.raw, n), q, k, v, lengths)


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64])
@pytest.mark.parametrize("e", [8, 12, 20])
def test_decode_where_groups_of_a_head_differ(kda, group, e):
    """Steps 2^e apart between a head's groups: each group is its own outputs, within its own bound."""
    gen = torch.Generator(device="cuda").manual_seed(e)
    for B, blocks, QH, KH in ((2, 40, 8, 2), (1, 94, 16, 1), (1, 1400, 6, 1), (64, 260, 16, 8)):
        T, groups = 16 * blocks, 128 // group
        k = Cache(gen, *(spread(B, KH, T, groups, lambda t, g: 0 * t + 0 * g - 3) * f for f in (1, -7)))
        v = Cache(gen, *(spread(B, KH, T, groups, lambda t, g: 0 * t - e * (g % 2)) * f for f in (1, -7)))
        q, lengths = whole(gen, B, QH, 128).to(BF16), lengths_of(B, T)
        n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        compare(kda.gqa_decode_q4(q, k.raw, v.raw, n), q, k, v, lengths, range(0, B, 31))


@pytest.mark.gpu
@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("B,blocks,QH,KH", WALKS)
def test_decode_where_scores_rise_past_large_steps(kda, group, B, blocks, QH, KH):
    """The first blocks have steps 2^18 larger; scores then rise all the way, so that those blocks' weights
    vanish and what stays is small beside them: the scale of a head's weights has to follow."""
    gen = torch.Generator(device="cuda").manual_seed(blocks)
    T, groups = 16 * blocks, 128 // group
    step = spread(B, KH, T, groups, lambda t, g: 18.0 * (t < T // 4) + 0 * g)
    v = Cache(gen, step, -7 * step)
    # keys: lows that rise, by 1/16 a token or so that they do not pass 188; codes are noise
    rise = min(3000.0 / T, 1.0)
    t = torch.arange(T, device="cuda").double()[:, None]
    low = (t * rise / 16).to(BF16).double().expand(B, KH, T, groups).contiguous()
    k = Cache(gen, spread(B, KH, T, groups, lambda t, g: 0 * t + 0 * g - 6), low)
    q = whole(gen, B, QH, 128)
    q[..., 0] += 14 - q.sum(-1)  # the sum is 14: a rise of 14 log2e / sqrt(128) = 1.8 for each unit of low
    q = q.to(BF16)
    lengths = [T - 16 * (b % 5) for b in range(B)]
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    compare(kda.gqa_decode_q4(q, k.raw, v.raw, n), q, k, v, lengths, range(0, B, 31))


@pytest.mark.gpu
@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("e", [8, 12, 16])
@pytest.mark.parametrize("B,blocks,QH,KH", WALKS)
def test_decode_where_tokens_differ(kda, group, e, B, blocks, QH, KH):
    """Small steps, then some blocks with steps 2^e larger, in one group or in all, then small ones: a
    warp's sums are rescaled with sums there already.  In every other pair of channels the large
    tokens hold zeros (code 0, low 0), so the small tokens' sums alone are the output there."""
    gen = torch.Generator(device="cuda").manual_seed(e * blocks)
    T, groups = 16 * blocks, 128 // group
    lengths = [T - 16 * (b % 5) for b in range(B)]
    for which in (0, groups):  # the last group alone, or every one

        def large(t, g):
            return ((t // 16 % 19 >= 14) & (t // 16 % 19 < 16) | (t == 2 * T // 3)) & (g >= groups - 1 - which)

        big = spread(B, KH, T, groups, large) > 1.5
        step = torch.where(big, 2.0 ** e, 1.0)
        codes = torch.randint(0, 16, (B, KH, T, 128), generator=gen, device="cuda")
        off = torch.arange(128, device="cuda") // 2 % 2 == 1
        codes[big.repeat_interleave(group, -1) & off] = 0
        v = Cache(gen, step, 0 * step, codes)
        k = Cache(gen, *(spread(B, KH, T, groups, lambda t, g: 0 * t + 0 * g - 4) * f for f in (1, -7)))
        q = whole(gen, B, QH, 128).to(BF16)
        n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        out = kda.gqa_decode_q4(q, k.raw, v.raw, n)
        compare(out, q, k, v, lengths, range(0, B, 31))
        assert torch.equal(out, kda.gqa_decode_q4(q, k.raw, v.raw, n))


@pytest.mark.gpu
@pytest.mark.parametrize("group", GROUPS)
def test_decode_of_131072_tokens(kda, group):
    """Random queries and values, relative L2 over 32 heads.  Rounding the result: at most 2^-8 / sqrt(3) of the
    values' (every error uniform in half a step, every value at the bottom of its binade), 5 % more for 4,096
    samples; the weights' and queries' rounding to fp16, 2^-11 each."""
    gen = torch.Generator(device="cuda").manual_seed(group)
    T, KH, QH, n = 131072, 8, 32, 131001
    caches = []
    for _ in range(2):
        step = 0.3 + 0.1 * torch.rand(1, KH, T, 128 // group, generator=gen, device="cuda")
        caches.append(Cache(gen, step, -7.5 * step))
    k, v = caches
    q = torch.randn(1, QH, 128, generator=gen, device="cuda").to(BF16)
    out = kda.gqa_decode_q4(q, k.raw, v.raw, torch.tensor([n], dtype=torch.int32, device="cuda"))
    want = torch.empty(QH, 128, dtype=torch.float64, device="cuda")
    for g in range(KH):
        kv, vv = (sum(c.head(0, g))[:n] for c in (k, v))
        qs = q[0, 4 * g:4 * g + 4].double()
        want[4 * g:4 * g + 4] = torch.softmax(qs @ kv.T / np.sqrt(128.0), -1) @ vv
    err = float((out[0].double() - want).norm() / want.norm())
    assert err <= 1.05 * 2.0 ** -8 / np.sqrt(3.0) + 2.0 ** -10, err


@pytest.mark.gpu
@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("case", range(len(DECODE_CASES) + len(LONG_CASES)))
def test_decode_of_random_values(kda, group, case):
    """Relative L2 of a request: rounding the result, 2^-8 at most, and 2^-10 for the fp16 operands: queries
    and weights are off by 2^-11 of themselves each, independently of one another."""
    B, blocks, QH, KH, window, sinks, *lens = (DECODE_CASES + LONG_CASES)[case]
    gen = torch.Generator(device="cuda").manual_seed(case)
    T, seen = 16 * blocks, 10 ** 9 if window is None else window
    lens = lens[0] if lens else [T - (77 * b) % T for b in range(B)]
    caches = []
    for _ in range(2):
        step = 0.3 + 0.1 * torch.rand(B, KH, T, 128 // group, generator=gen, device="cuda")
        caches.append(Cache(gen, step, -step * (7 + torch.rand(step.shape, generator=gen, device="cuda"))))
    k, v = caches
    q = torch.randn(B, QH, 128, generator=gen, device="cuda").to(BF16)
    out = kda.gqa_decode_q4(q, k.raw, v.raw, torch.tensor(lens, dtype=torch.int32, device="cuda"), window, sinks)
    for b in range(0, B, 1 + B // 8):
        n = lens[b]
        if n <= 0:
            assert not out[b].any()
            continue
        j = torch.arange(n, device="cuda")
        want = []
        for g in range(KH):
            kv, vv = (sum(c.head(b, g))[:n] for c in caches)
            s = q[b, g * QH // KH:(g + 1) * QH // KH].double() @ kv.T / np.sqrt(128.0)
            want.append(torch.softmax(s.masked_fill((j < n - seen) & (j >= sinks), -torch.inf), -1) @ vv)
        want = torch.cat(want)
        assert float((out[b].double() - want).norm() / want.norm()) <= 2.0 ** -8 + 2.0 ** -10
