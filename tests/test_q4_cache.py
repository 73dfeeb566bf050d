"""The 4-bit key/value cache: append, reading back and the decode against it, against the
restatements in ``oracle.ops`` (codes by the same fp32 operations, attention in float64).

What the append writes is compared byte for byte.  Values read back are code * step + low,
exact in fp32 up to its rounding and then rounded to bf16: 2^-8 of the value.  The decode's
chain rounds twice to bf16 (weight times step, the result): relative L2 2 x 2^-8 at most.
"""

import numpy as np
import pytest

from oracle import ops as ref
from oracle.bf16 import to_bf16_rne
from oracle.metrics import rel_l2

torch = pytest.importorskip("torch")

BF16 = torch.bfloat16
U = 2.0 ** -8


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


def ints(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


# --------------------------------------------------------------- the oracle
@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantised_values_are_within_half_a_step(group):
    rng = np.random.default_rng(group)
    x = draw(rng, 3, 2, 5, 128)
    codes, step, low = ref.q4_quantise(x, group)
    assert codes.min() == 0 and codes.max() == 15
    off = np.abs(ref.q4_values(codes, step, low) - x).reshape(*step.shape, group).max(-1)
    # half a step, and at the group's top 15 times what step itself was rounded by
    assert (off <= step * (0.5 + 15 * U)).all()


def test_quantised_corner_cases():
    x = np.zeros((6, 128), np.float32)
    x[1] = 3.0                       # constant: low alone
    x[2, :32], x[3, 5], x[4, 40] = np.linspace(0, 15, 32), np.nan, np.inf
    x[5, :2] = to_bf16_rne(np.array([1e-39, 2e-39], np.float32))  # a step below 2^-126
    x = to_bf16_rne(x)
    codes, step, low = ref.q4_quantise(x, 32)
    v = ref.q4_values(codes, step, low)
    assert not v[0].any() and (v[1] == 3).all() and not codes[1].any()
    assert step[2, 0] == 1 and np.abs(v[2] - x[2]).max() <= 0.5
    assert np.isnan(v[3, :32]).all() and not np.isnan(v[3, 32:]).any()
    assert np.isnan(v[4, 32:64]).all() and not np.isnan(v[4, :32]).any()
    assert (step[5] == 0).all() and (v[5] == low[5].repeat(32)).all()


def test_packed_bytes_read_back():
    """The layout that kda.h states, nibble by nibble."""
    rng = np.random.default_rng(0)
    codes, step, low = ref.q4_quantise(draw(rng, 2, 3, 32, 128), 64)
    raw = ref.q4_pack(codes, step, low)
    assert raw.shape == (2, 3, 2, 1152)
    for _ in range(200):
        b, h, t, ch = (int(rng.integers(n)) for n in (2, 3, 32, 128))
        block, u = raw[b, h, t // 16], t % 16
        at = 64 * u + 16 * ((ch % 32 // 8) ^ (u // 2 & 3)) + 4 * (ch // 32)
        word = int.from_bytes(block[at:at + 4].tobytes(), "little")
        assert (word >> 4 * (ch % 8)) & 15 == codes[b, h, t, ch]
        pair = block[1024 + (u * 2 + ch // 64) * 4:][:4].view("<u2").astype(np.uint32) << 16
        assert np.array_equal(pair.view(np.float32), [step[b, h, t, ch // 64], low[b, h, t, ch // 64]])


# ------------------------------------------------------- refusals on the host
def test_c_entries_reject_bad_arguments(kda):
    """Checked before any launch, so they run without a GPU."""
    import ctypes as C
    from kda import _lib
    lib = _lib.lib()
    rows, odd = (C.c_int64 * 3)(1024, 256, 128), (C.c_int64 * 3)(1024, 255, 128)
    cs, codd = (C.c_int64 * 2)(4608, 2304), (C.c_int64 * 2)(4608, 2300)
    work = _lib._attach(lib, "kda_gqa_decode_q4_workspace_size")
    assert [_lib._attach(lib, "kda_q4_block_bytes")(g) for g in (32, 64, 128, 16, 0)] == [1280, 1152, 1088, 0, 0]

    def append(k=16, off=None, n=16, kc=16, T=8, B=2, blocks=2, KH=2, D=128, group=64, ks=rows, kcs=cs):
        _lib.call("kda_kv_append_q4", k, 16, off, n, kc, 16, T, B, blocks, KH, D, group, ks, rows, kcs, cs, None)

    def read(c=16, out=16, B=2, blocks=2, KH=2, D=128, group=64, st=cs):
        _lib.call("kda_kv_read_q4", c, out, B, blocks, KH, D, group, st, None)

    def decode(q=16, n=16, B=2, blocks=2, QH=4, KH=2, D=128, group=64, w=32, sinks=0, st=cs, ws=16, wb=None):
        s2 = (C.c_int64 * 2)(512, 128)
        wb = work(4, 2) if wb is None else wb
        _lib.call("kda_gqa_decode_q4", q, 16, 16, n, 16, B, blocks, QH, KH, D, group, w, sinks, s2, st, cs, ws, wb,
                  None)

    for bad in (lambda: append(k=None), lambda: append(n=None), lambda: append(kc=None), lambda: append(T=0),
                lambda: append(T=7), lambda: append(B=0), lambda: append(blocks=0), lambda: append(KH=0),
                lambda: append(group=16), lambda: append(group=0), lambda: read(c=None), lambda: read(out=None),
                lambda: read(B=0), lambda: read(blocks=0), lambda: read(group=48), lambda: decode(q=None),
                lambda: decode(n=None), lambda: decode(B=0), lambda: decode(blocks=0), lambda: decode(KH=3),
                lambda: decode(group=256), lambda: decode(w=0), lambda: decode(sinks=-1), lambda: decode(ws=None),
                lambda: decode(wb=64)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: append(k=8), lambda: append(kc=8), lambda: append(D=64), lambda: append(ks=odd),
                lambda: append(kcs=codd), lambda: append(blocks=2 ** 26), lambda: read(c=8), lambda: read(out=8),
                lambda: read(D=64), lambda: read(st=codd), lambda: read(blocks=2 ** 26), lambda: decode(q=8),
                lambda: decode(D=64), lambda: decode(st=codd), lambda: decode(ws=8), lambda: decode(B=65536)):
        with pytest.raises(kda.KdaError):
            bad()
    assert work(0, 1) == 0 and work(5, 2) == 0


def test_host_checks_and_fake_kernels(kda):
    for bad in (lambda: kda.kv_cache_q4(0, 1, 1), lambda: kda.kv_cache_q4(1, 0, 1), lambda: kda.kv_cache_q4(1, 1, 0),
                lambda: kda.kv_cache_q4(1, 1, 1, 16, device="cpu"),
                lambda: kda.kv_read_q4(kda.kv_cache_q4(1, 1, 1, device="cpu"))):
        with pytest.raises(ValueError):
            bad()
    c = kda.kv_cache_q4(3, 33, 2, 128, device="meta")
    assert c.shape == (3, 2, 3, 1088) and c.dtype == torch.uint8
    got = torch.ops.kda.kv_read_q4(c)
    assert got.shape == (3, 48, 2, 128) and got.dtype == BF16
    q, n = torch.empty(3, 4, 128, device="meta", dtype=BF16), torch.empty(3, device="meta", dtype=torch.int32)
    assert torch.ops.kda.gqa_decode_q4(q, c, c.clone(), n).shape == q.shape
    k = torch.empty(3, 1, 2, 128, device="meta", dtype=BF16)
    assert torch.ops.kda.kv_append_q4(k, k, c, c.clone(), n) is None


# ---------------------------------------------------------------------- GPU
def noise(rng, *shape):
    return torch.from_numpy(rng.integers(0, 256, size=shape, dtype=np.uint8)).cuda()


def expected_bytes(before, x, group, lengths, starts):
    """The cache's bytes after rows x (n,KH,128): row i of request b from starts[b] on."""
    raw = before.copy()
    codes, step, low = ref.q4_quantise(x, group)
    n = codes.shape[0]
    # the rows as a cache of n requests of 16 equal tokens: row t of block i is what token t would be
    one = ref.q4_pack(np.repeat(codes[:, :, None], 16, 2), np.repeat(step[:, :, None], 16, 2),
                      np.repeat(low[:, :, None], 16, 2))[:, :, 0]
    per = 4 * (128 // group)
    for b, (a, e) in enumerate(zip(starts[:-1], starts[1:])):
        for i in range(a, min(e, n)):
            p = lengths[b] + i - a
            if lengths[b] < 0 or p >= 16 * raw.shape[2]:
                continue
            t = p % 16
            raw[b, :, p // 16, 64 * t:64 * t + 64] = one[i, :, 64 * t:64 * t + 64]
            raw[b, :, p // 16, 1024 + per * t:1024 + per * (t + 1)] = one[i, :, 1024 + per * t:1024 + per * (t + 1)]
    return raw


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("counts,KH,lengths,blocks", [
    ([1], 1, [0], 1), ([1, 1, 1], 8, [15, -1, 16], 2), ([5, 0, 40, 1, 16], 2, [3, 7, 0, -4, 17], 3),
    ([70], 3, [10], 5), ([0, 0, 2], 1, [0, 0, 14], 1), ([3] * 50, 2, list(range(50)), 4), ([1] * 300, 1, [5] * 300, 1),
])
def test_append_packed_rows(kda, group, counts, KH, lengths, blocks):
    rng = np.random.default_rng(sum(counts) + group)
    starts = np.concatenate([[0], np.cumsum(counts)])
    n, B = int(starts[-1]) + 3, len(counts)  # three rows of no request
    k, v = draw(rng, n, KH, 128, scale=2.0), draw(rng, n, KH, 128)
    v[:, :, :16] = 0.25  # ties and constant runs
    caches = [noise(rng, B, KH, blocks, 1024 + 8192 // group) for _ in range(2)]
    before = [c.cpu().numpy() for c in caches]
    kda.kv_append_q4(dev(k), dev(v), *caches, ints(lengths), ints(starts))
    for c, b, x in zip(caches, before, (k, v)):
        assert np.array_equal(c.cpu().numpy(), expected_bytes(b, x, group, lengths, starts))


@pytest.mark.gpu
@pytest.mark.parametrize("S", [1, 19])
def test_append_rows_of_each_request_and_views(kda, S):
    """(B,S,KH,128) slices of a packed projection into layers of a larger cache."""
    rng = np.random.default_rng(S)
    B, KH, blocks, group = 4, 2, 3, 64
    qkv = draw(rng, B, S, 3 * KH, 128)
    t = dev(qkv)
    cache = noise(rng, B, 2, 2 * KH, blocks, 1152)
    before = cache.cpu().numpy()
    kc, vc = cache[:, 0, KH:], cache[:, 1, :KH]
    lengths = [0, 11, -1, 29]
    kda.kv_append_q4(t[:, :, KH:2 * KH], t[:, :, 2 * KH:], kc, vc, ints(lengths))
    starts = np.arange(B + 1) * S
    after = cache.cpu().numpy()
    for at, sl in (((slice(None), 0, slice(KH, None)), slice(KH, 2 * KH)), ((slice(None), 1, slice(0, KH)), slice(2 * KH, None))):
        want = expected_bytes(before[at], qkv[:, :, sl].reshape(B * S, KH, 128), group, lengths, starts)
        assert np.array_equal(after[at], want)
        before[at] = after[at]
    assert np.array_equal(after, before)  # and nothing else


@pytest.mark.gpu
@pytest.mark.parametrize("T,KH,group", [(3000, 9, 32), (20000, 9, 64), (40000, 5, 128)])
def test_append_of_many_rows_is_each_head_alone(kda, T, KH, group):
    """Several heads to a CTA: the bytes of appends of one head, requests of any length, rows of
    none, an idle slot and rows past the cache among them."""
    gen = torch.Generator(device="cuda").manual_seed(T)
    kv = torch.randn(T, 2 * KH + 1, 128, generator=gen, device="cuda").to(BF16)
    k, v = kv[:, :KH], kv[:, KH + 1:]
    B, length = 11, T // 4
    cuts = np.sort(np.random.default_rng(T).integers(5, T - 9, size=B + 1))
    cuts[4] = cuts[3]
    off, lens = ints(cuts.tolist()), ints([0, 3, 16, 7, -1, 0, 40, 1, 250, 0, length - 2])
    got = [kda.kv_cache_q4(B, length, KH, group) for _ in range(2)]
    want = [kda.kv_cache_q4(B, length, KH, group) for _ in range(2)]
    kda.kv_append_q4(k, v, *got, lens, off)
    for h in range(KH):
        kda.kv_append_q4(k[:, h:h + 1], v[:, h:h + 1], *(c[:, h:h + 1] for c in want), lens, off)
    torch.cuda.synchronize()
    assert kda.device_error() == 8
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and got[0].any()
    step = T // B  # the same rows for each request
    k2, v2 = (x[:step * B].unflatten(0, (B, step)) for x in (k, v))
    lens = ints([17, -3] + [5] * (B - 2))
    kda.kv_append_q4(k2, v2, *got, lens)
    for h in range(KH):
        kda.kv_append_q4(k2[:, :, h:h + 1], v2[:, :, h:h + 1], *(c[:, h:h + 1] for c in want), lens)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_append_past_the_cache_is_reported_and_writes_nothing_there(kda):
    rng = np.random.default_rng(3)
    buf = noise(rng, 3, 1, 1, 1152)  # one request's cache between two others
    before = buf.cpu().numpy()
    x = draw(rng, 5, 1, 128)
    kda.kv_append_q4(dev(x), dev(x), buf[1:2], buf[1:2].clone(), ints([13]), ints([0, 5]))
    torch.cuda.synchronize()
    assert kda.device_error() == 8
    want = before.copy()
    want[1:2] = expected_bytes(before[1:2], x, 64, [13], [0, 5])
    assert np.array_equal(buf.cpu().numpy(), want)
    # lengths and offsets far outside
    kda.kv_append_q4(dev(x), dev(x), buf[1:2], buf[1:2].clone(), ints([2 ** 31 - 1]), ints([0, 5]))
    torch.cuda.synchronize()
    assert kda.device_error() == 8
    for off in ([9, 20], [-7, -2], [5, 0], [0, 0]):
        kda.kv_append_q4(dev(x), dev(x), buf[1:2], buf[1:2].clone(), ints([0]), ints(off))
    assert np.array_equal(buf.cpu().numpy(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
def test_append_corner_values(kda, group):
    """Constant rows, NaN, infinities, the widest range, values below the normal ones."""
    x = np.zeros((8, 1, 128), np.float32)
    x[1] = -2.5
    x[2, 0, 7], x[3, 0, 100], x[4, 0, 3] = np.nan, np.inf, -np.inf
    x[5, 0, ::2], x[5, 0, 1::2] = 3.3e38, -3.3e38
    x[6, 0, ::3] = 3e-39
    x[7, 0] = np.arange(128) * 2.0 ** -120
    x = to_bf16_rne(x)
    kc, vc = kda.kv_cache_q4(1, 16, 1, group), kda.kv_cache_q4(1, 16, 1, group)
    kda.kv_append_q4(dev(x), dev(x), kc, vc, ints([2]), ints([0, 8]))
    want = ref.q4_values(*ref.q4_quantise(x, group))
    got = host(kda.kv_read_q4(kc))[0, 2:10]
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = ~np.isnan(want)
    assert (np.abs(got - want)[fine] <= U * np.abs(want)[fine]).all()
    assert torch.equal(kc, vc) or not torch.equal(kc, kc)  # the same rows give the same bytes
    assert not host(kda.kv_read_q4(kc))[0, :2].any()


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("B,KH,blocks", [(1, 1, 1), (3, 2, 5), (2, 8, 33)])
def test_read(kda, group, B, KH, blocks):
    rng = np.random.default_rng(B + group)
    codes, step, low = ref.q4_quantise(draw(rng, B, KH, 16 * blocks, 128), group)
    raw = torch.from_numpy(ref.q4_pack(codes, step, low)).cuda()
    want = to_bf16_rne(ref.q4_values(codes, step, low).astype(np.float32)).transpose(0, 2, 1, 3)
    assert np.array_equal(host(kda.kv_read_q4(raw)), want)
    wide = torch.zeros(B, 2 * KH, blocks, raw.shape[-1], dtype=torch.uint8, device="cuda")
    wide[:, KH:] = raw
    assert np.array_equal(host(kda.kv_read_q4(wide[:, KH:])), want)


DECODE_CASES = [
    # B, blocks, QH, KH, window, sinks, lengths
    (1, 1, 1, 1, None, 0, [1]), (1, 1, 2, 1, None, 0, [16]), (2, 2, 8, 8, None, 0, [17, 3]),
    (4, 4, 8, 2, 16, 3, [0, 1, 17, 50]), (3, 44, 12, 4, 300, 130, [700, 301, -1]), (1, 94, 16, 1, 900, 1, [1333]),
    (2, 19, 40, 2, 64, 300, [300, 77]), (5, 3, 3, 3, 8, 0, [8, 9, 15, 16, 40]), (1, 17, 6, 2, 10 ** 6, 0, [259]),
    (1, 320, 32, 8, None, 0, [5111]), (2, 200, 20, 4, 1, 0, [3200, 1600]), (1, 600, 8, 1, None, 0, [9600]),
    (70, 4, 4, 2, None, 0, [0] * 33 + [64, 1, 33] + [0] * 33 + [5]), (1, 300, 9, 1, None, 0, [4800]),
    (300, 1, 2, 1, None, 0, [b % 17 for b in range(300)]), (1, 40, 5, 1, 17, 15, [640]),
    # many requests
    (256, 2, 8, 2, None, 0, [b % 33 for b in range(256)]), (130, 3, 12, 4, 9, 3, [(7 * b) % 49 for b in range(130)]),
    (64, 5, 8, 8, None, 0, [80 - b for b in range(64)]), (86, 9, 12, 6, 100, 20, [144 - b for b in range(86)]),
]


def random_cache(rng, B, KH, blocks, group):
    codes = rng.integers(0, 16, size=(B, KH, 16 * blocks, 128))
    step = to_bf16_rne((0.3 + 0.1 * rng.random((B, KH, 16 * blocks, 128 // group))).astype(np.float32))
    low = to_bf16_rne((-step * (7 + rng.random(step.shape))).astype(np.float32))
    return ref.q4_pack(codes, step, low), ref.q4_values(codes, step, low).transpose(0, 2, 1, 3)


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("B,blocks,QH,KH,window,sinks,lengths", DECODE_CASES)
def test_decode(kda, group, B, blocks, QH, KH, window, sinks, lengths):
    rng = np.random.default_rng(blocks + QH)
    q = draw(rng, B, QH, 128)
    (rk, k), (rv, v) = (random_cache(rng, B, KH, blocks, group) for _ in range(2))
    per = 4 * (128 // group)
    seen = 10 ** 9 if window is None else window
    for raw in (rk, rv):  # what lies past the valid tokens, or what the window has left behind, may be anything
        for b, n in enumerate(lengths):
            for t in range(16 * blocks):
                if t >= n or (t < n - seen and t >= sinks):
                    at = 1024 + per * (t % 16)
                    raw[b, :, t // 16, at:at + per] = 0xff  # NaN pairs
    args = (dev(q), torch.from_numpy(rk).cuda(), torch.from_numpy(rv).cuda(), ints(lengths), window, sinks)
    out = kda.gqa_decode_q4(*args)
    want = ref.gqa_window_decode(q, k, v, lengths, seen, sinks)
    for b in range(B):
        if lengths[b] <= 0:
            assert not out[b].any()
        else:
            assert rel_l2(host(out[b]), want[b]) <= 2 * U
    assert torch.equal(out, kda.gqa_decode_q4(*args))


def values64(raw):
    """Every value of a cache (B,KH,blocks,bytes) on the GPU: (B,KH,T,128) in 64 bits."""
    t, ch = torch.arange(16, device="cuda")[:, None], torch.arange(128, device="cuda")
    at = 64 * t + 16 * ((ch % 32 // 8) ^ (t // 2 % 4)) + 4 * (ch // 32) + ch % 8 // 2
    codes = (raw[..., at.flatten()].unflatten(-1, (16, 128)) >> (4 * (ch % 2)).to(torch.uint8)) & 15
    side = raw[..., 1024:].contiguous().view(BF16).double().unflatten(-1, (16, -1, 2))
    v = codes.double().unflatten(-1, (side.shape[-2], -1)) * side[..., :1] + side[..., 1:]
    return v.flatten(-2).flatten(2, 3)


# Walks too long for a cluster: runs over all CTAs, cut walks joined by a second launch.  The second,
# third, seventh and ninth take two kv heads together, the eighth and ninth have some walks to a
# run; the last two are clusters.
LONG_CASES = [
    # B, blocks, QH, KH, window, sinks
    (1, 1400, 6, 1, None, 0), (64, 260, 16, 8, None, 0), (4, 4200, 16, 8, 50000, 33), (3, 700, 5, 5, None, 0),
    (2, 1300, 34, 2, 20000, 1), (1, 2600, 16, 1, None, 0), (130, 259, 8, 4, None, 0), (700, 260, 4, 1, None, 0),
    (520, 260, 4, 2, None, 0), (300, 66, 8, 4, None, 0), (9, 400, 48, 6, None, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("B,blocks,QH,KH,window,sinks", LONG_CASES)
def test_decode_of_long_walks(kda, group, B, blocks, QH, KH, window, sinks):
    gen = torch.Generator(device="cuda").manual_seed(blocks)
    rng = np.random.default_rng(blocks)
    T, seen = 16 * blocks, 10 ** 9 if window is None else window
    lens = rng.integers(0, T + 1, size=B)
    lens[0] = T
    if B > 2:
        lens[1], lens[2] = 0, -5
    caches = []
    for _ in range(2):
        c = torch.randint(0, 256, (B, KH, blocks, 1024 + 8192 // group), generator=gen, device="cuda", dtype=torch.uint8)
        step = 0.3 + 0.1 * torch.rand(B, KH, blocks, 16 * (128 // group), generator=gen, device="cuda")
        c[..., 1024:] = torch.stack([step, -7.5 * step], -1).to(BF16).flatten(-2).view(torch.uint8)
        caches.append(c)
    q = torch.randn(B, QH, 128, generator=gen, device="cuda").to(BF16)
    args = (q, *caches, ints(lens.tolist()), window, sinks)
    out = kda.gqa_decode_q4(*args)
    for b in range(B):
        n = int(lens[b])
        if n <= 0:
            assert not out[b].any()
            continue
        if b > 3 and b % 17:
            continue
        k, v = (values64(c[b:b + 1])[0, :, :n] for c in caches)
        j = torch.arange(n, device="cuda")
        s = q[b].double().unflatten(0, (KH, -1)) @ k.transpose(-1, -2) / np.sqrt(128.0)
        s = s.masked_fill((j < n - seen) & (j >= sinks), -torch.inf)
        want = (torch.softmax(s, -1) @ v).flatten(0, 1)
        assert (out[b].double() - want).norm() <= 2 * U * want.norm()
    for _ in range(3):
        assert torch.equal(out, kda.gqa_decode_q4(*args))


@pytest.mark.gpu
def test_decode_of_long_walks_strides_ends_and_graphs(kda):
    """Runs: strided caches, a length past the cache, a NaN in one kv head, a workspace that two
    graphs share with a call of short walks."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    B, QH, KH, blocks = 2, 4, 2, 1400
    both = torch.randint(0, 256, (B, blocks, 2 * KH, 1152), generator=gen, device="cuda", dtype=torch.uint8)
    both[..., 1024:] = ints([0x3e80, 0xbf80]).to(torch.int16).repeat(32).view(torch.uint8)  # c / 4 - 1
    kc, vc = (both.permute(0, 2, 1, 3)[:, i::2].contiguous() for i in range(2))
    wide = torch.empty(B, KH + 1, blocks + 3, 1152, dtype=torch.uint8, device="cuda")
    wide[:, 1:, :blocks] = kc
    q = torch.randn(B, QH, 128, generator=gen, device="cuda").to(BF16)
    n, T = ints([16 * blocks, 9001]), 16 * blocks
    want = kda.gqa_decode_q4(q, kc, vc, n)
    assert torch.equal(want, kda.gqa_decode_q4(q, wide[:, 1:].narrow(2, 0, blocks), vc, n))
    assert torch.equal(want, kda.gqa_decode_q4(q, kc, vc, ints([T + 9, 9001])))
    torch.cuda.synchronize()
    assert kda.device_error() == 8
    bad = vc.clone()
    bad[0, 1, 700, 1030:1032] = 0xff
    got = kda.gqa_decode_q4(q, kc, bad, n)
    assert torch.equal(got[0, :2], want[0, :2]) and torch.equal(got[1], want[1])
    nan = torch.isnan(got[0, 2:]).any(0)
    assert nan.sum() == 64 and (nan[:64].all() or nan[64:].all())
    ws = torch.full((4 << 20,), 0xff, dtype=torch.uint8, device="cuda")
    short = [c[:, :, :9].contiguous() for c in (kc, vc)]
    few = ints([130, 77])
    small = kda.gqa_decode_q4(q, *short, few)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, kda.gqa_decode_q4(q, kc, vc, n, workspace=ws),
                           kda.gqa_decode_q4(q, *short, few, workspace=ws),
                           kda.gqa_decode_q4(q, kc, vc, n, workspace=ws)))
    for _ in range(3):
        for graph, *_ in graphs:
            graph.replay()
        assert all(torch.equal(a, b) for _, *got in graphs for a, b in zip(got, (want, small, want)))


@pytest.mark.gpu
def test_decode_extreme_scores_and_nan(kda):
    """Scores of some hundreds; a NaN among the visible rows reaches its own head alone."""
    rng = np.random.default_rng(8)
    q = draw(rng, 1, 4, 128, scale=30.0)
    (rk, k), (rv, v) = (random_cache(rng, 1, 2, 60, 64) for _ in range(2))
    tk, tv = torch.from_numpy(rk).cuda(), torch.from_numpy(rv).cuda()
    want = ref.gqa_window_decode(q, k, v, [950], 10 ** 6)
    out = kda.gqa_decode_q4(dev(q), tk, tv, ints([950]))
    assert rel_l2(host(out), want) <= 2 * U
    for cache in (tk, tv):
        bad = cache.clone()
        bad[0, 1, 30, 1024 + 8 * 5:1024 + 8 * 6] = 0xff
        got = kda.gqa_decode_q4(dev(q), *((bad, tv) if cache is tk else (tk, bad)), ints([950]))
        assert torch.equal(got[:, :2], out[:, :2]) and torch.isnan(got[:, 2:]).all()


@pytest.mark.gpu
def test_decode_length_past_the_cache_is_cut_and_reported(kda):
    rng = np.random.default_rng(2)
    q = dev(draw(rng, 2, 4, 128))
    kc, vc = (torch.from_numpy(random_cache(rng, 2, 2, 2, 64)[0]).cuda() for _ in range(2))
    got = kda.gqa_decode_q4(q, kc, vc, ints([33, 2 ** 31 - 1]), 8, 2)
    torch.cuda.synchronize()
    assert kda.device_error() == 8
    assert torch.equal(got, kda.gqa_decode_q4(q, kc, vc, ints([32, 32]), 8, 2))


@pytest.mark.gpu
def test_decode_strided_operands_and_output(kda):
    rng = np.random.default_rng(12)
    B, QH, KH = 3, 8, 2
    q = dev(draw(rng, B, 2 * QH, 128))[:, QH:]
    cache = noise(rng, B, 2, 2 * KH, 5, 1152)
    for c in (cache[:, 0, KH:], cache[:, 1, :KH]):  # finite pairs
        c.copy_(torch.from_numpy(random_cache(rng, B, KH, 5, 64)[0]))
    kc, vc = cache[:, 0, KH:], cache[:, 1, :KH]
    want = kda.gqa_decode_q4(q.contiguous(), kc.contiguous(), vc.contiguous(), ints([80, 1, 41]))
    out = torch.empty_like(want)
    ws = torch.full((4 << 20,), 0xff, dtype=torch.uint8, device="cuda")
    assert kda.gqa_decode_q4(q, kc, vc, ints([80, 1, 41]), out=out, workspace=ws) is not None
    assert torch.equal(out, want)


@pytest.mark.gpu
def test_caches_past_32_bit_offsets(kda):
    """The last rows of caches of more than 2^32 bytes, of one head and of many."""
    for B, KH, blocks in ((1, 2, (1 << 31) // 1152 + 40), (1100, 2, 1800)):
        kc = torch.zeros(B, KH, blocks, 1152, dtype=torch.uint8, device="cuda")
        vc = torch.zeros_like(kc)
        T = 16 * blocks
        x = torch.ones(1, KH, 128, dtype=BF16, device="cuda")
        lens = torch.full((B,), -1, dtype=torch.int32, device="cuda")
        lens[-1] = T - 1
        off = torch.zeros(B + 1, dtype=torch.int32, device="cuda")
        off[-1] = 1
        kda.kv_append_q4(x, 6 * x, kc, vc, lens, off)
        q = torch.zeros(B, KH, 128, dtype=BF16, device="cuda")
        n = torch.zeros(B, dtype=torch.int32, device="cuda")
        n[-1] = T
        out = kda.gqa_decode_q4(q, kc, vc, n, 3, 0)  # equal scores: 6 / 3
        assert (out[-1] == 2).all() and not out[:-1].any()
        del kc, vc


@pytest.mark.gpu
def test_prompts_to_cache_to_decode(kda):
    """As they are used together: a batch of prompts, packed; its keys and values to the caches by
    the same offsets; then one token at a time.  Against the values that the cache stands for."""
    rng = np.random.default_rng(21)
    lens, QH, KH, group = [37, 1, 130], 8, 2, 64
    off = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    T, B = int(off[-1]), len(lens)
    q, k, v = draw(rng, T, QH, 128, scale=1.5), draw(rng, T, KH, 128, scale=1.5), draw(rng, T, KH, 128)
    g = torch.ones(128, device="cuda")
    table = kda.rope_table(200, 128)
    pos = np.concatenate([np.arange(n) for n in lens]).astype(np.int32)
    tq, tk = kda.qk_norm_rope(dev(q)[None], dev(k)[None], g, g, table, positions=dev(pos, torch.int32)[None])
    tq, tk, tv = tq[0], tk[0], dev(v)
    plan = kda.packed_plan(dev(off, torch.int32), T)
    out = kda.gqa_packed(tq, tk, tv, plan)
    want = ref.gqa_packed(host(tq), host(tk), v, off)[0]
    assert rel_l2(host(out), want) <= 2 * U
    caches = [kda.kv_cache_q4(B, 140, KH, group) for _ in range(2)]
    n = torch.zeros(B, dtype=torch.int32, device="cuda")
    kda.kv_append_q4(tk, tv, *caches, n, dev(off, torch.int32))
    n += ints(lens)
    for _ in range(4):
        new = [dev(draw(rng, B, 1, h, 128)) for h in (QH, KH, KH)]
        q1, k1 = kda.qk_norm_rope(new[0], new[1], g, g, table, positions=n[:, None].contiguous())
        kda.kv_append_q4(k1, new[2], *caches, n)
        n += 1
        got = kda.gqa_decode_q4(q1[:, 0], *caches, n)
        held = []
        for c in caches:  # the bytes' values in 64 bits
            raw = c.cpu().numpy()
            t, ch = np.arange(16)[:, None], np.arange(128)
            at = 64 * t + 16 * ((ch % 32 // 8) ^ (t // 2 & 3)) + 4 * (ch // 32) + ch % 8 // 2
            codes = (raw[..., at] >> (4 * (ch % 2))) & 15
            pairs = (np.ascontiguousarray(raw[..., 1024:]).view("<u2").astype(np.uint32) << 16).view(np.float32)
            pairs = pairs.reshape(*raw.shape[:3], 16, 128 // group, 2)
            val = ref.q4_values(codes, pairs[..., 0], pairs[..., 1])
            held.append(val.reshape(B, KH, -1, 128).transpose(0, 2, 1, 3))
        wd = ref.gqa_window_decode(host(q1[:, 0]), *held, n.cpu().numpy(), 10 ** 6)
        assert rel_l2(host(got), wd) <= 2 * U
        assert torch.equal(torch.ops.kda.gqa_decode_q4(q1[:, 0], *caches, n), got)


@pytest.mark.gpu
def test_streams_and_graph_replays(kda):
    """Append and decode on a side stream and in two graphs that share caches and a workspace."""
    rng = np.random.default_rng(4)
    B, QH, KH = 3, 8, 2
    kc, vc = (torch.from_numpy(random_cache(rng, B, KH, 12, 64)[0]).cuda() for _ in range(2))
    q, k, v = dev(draw(rng, B, QH, 128)), dev(draw(rng, B, 1, KH, 128)), dev(draw(rng, B, 1, KH, 128))
    n = ints([100, 0, 191])
    ws = torch.empty(4 << 20, dtype=torch.uint8, device="cuda")

    def step():
        kda.kv_append_q4(k, v, kc, vc, n)
        return kda.gqa_decode_q4(q, kc, vc, n + 1, workspace=ws), kda.kv_read_q4(kc)

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, step()))
    for turn in range(3):
        n.copy_(ints([100 + turn, turn, 191 - turn]))
        k.mul_(0.75)
        for graph, got in graphs:
            graph.replay()
        want = step()
        assert all(torch.equal(a, b) for _, got in graphs for a, b in zip(got, want))


@pytest.mark.gpu
def test_refusals(kda):
    q = torch.zeros(2, 4, 128, dtype=BF16, device="cuda")
    kv = torch.zeros(2, 1, 2, 128, dtype=BF16, device="cuda")
    kc, vc = kda.kv_cache_q4(2, 40, 2), kda.kv_cache_q4(2, 40, 2)
    other = kda.kv_cache_q4(2, 40, 2, 32)
    n = torch.ones(2, dtype=torch.int32, device="cuda")
    off = ints([0, 1, 2])
    for bad in (
        lambda: kda.kv_append_q4(kv, kv, kc, other, n), lambda: kda.kv_append_q4(kv, kv, kc, vc[:, :, :2], n),
        lambda: kda.kv_append_q4(kv, kv, kc[:1], vc[:1], n[:1]), lambda: kda.kv_append_q4(kv, kv, kc, vc, n.long()),
        lambda: kda.kv_append_q4(kv[:, :, :1], kv[:, :, :1], kc, vc, n),
        lambda: kda.kv_append_q4(kv, kv[:, :, :1], kc, vc, n), lambda: kda.kv_append_q4(kv.float(), kv, kc, vc, n),
        lambda: kda.kv_append_q4(kv, kv, kc, vc, n, off), lambda: kda.kv_append_q4(kv[:, 0], kv[:, 0], kc, vc, n),
        lambda: kda.kv_append_q4(kv[:, 0], kv[:, 0], kc, vc, n, off[:2]),
        lambda: kda.kv_append_q4(kv[:, 0], kv[:, 0], kc, vc, n, off.long()),
        lambda: kda.kv_append_q4(kv[:0, 0], kv[:0, 0], kc, vc, n, off),
        lambda: kda.kv_append_q4(kv, kv, kc.to(torch.int8), vc, n), lambda: kda.kv_append_q4(kv, kv, kc.cpu(), vc, n),
        lambda: kda.kv_append_q4(kv, kv, kc[..., :1100], vc[..., :1100], n),
        lambda: kda.kv_append_q4(kv, kv, kc[:, :, ::2], vc[:, :, ::2], n),
        lambda: kda.kv_append_q4(kv, kv, kc[:1].expand(2, -1, -1, -1), vc, n),
        lambda: kda.kv_read_q4(kc[0]), lambda: kda.kv_read_q4(kc[:0]), lambda: kda.kv_read_q4(kc.float()),
        lambda: kda.kv_read_q4(kc, out=torch.empty(2, 40, 2, 128, dtype=BF16, device="cuda")),
        lambda: kda.gqa_decode_q4(q, kc, vc, n, 0), lambda: kda.gqa_decode_q4(q, kc, vc, n, 4, -1),
        lambda: kda.gqa_decode_q4(q, kc, other, n), lambda: kda.gqa_decode_q4(q[:, :3], kc, vc, n),
        lambda: kda.gqa_decode_q4(q[:1], kc, vc, n[:1]), lambda: kda.gqa_decode_q4(q.float(), kc, vc, n),
        lambda: kda.gqa_decode_q4(q, kc, vc, n[:1]), lambda: kda.gqa_decode_q4(q, kc, vc, n.float()),
        lambda: kda.gqa_decode_q4(q[:, None], kc, vc, n),
        lambda: kda.gqa_decode_q4(q, kc, vc, n, workspace=torch.empty(8, dtype=torch.uint8, device="cuda")),
    ):
        with pytest.raises(ValueError):
            bad()
