"""The decode operators on the GPU against plain 64-bit implementations (tests/operators_ref.py).

Tolerances.  The cache's codes and exponents are compared exactly.  Attention: with S the largest
scale * sum |q||k| of a call, a score comes out of 2 * dim / 16 <= 16 accumulation steps in f32, each
off by at most 2^-23 of the running sum (truncation), from q in two f16 parts (2^-22) scaled by
log2(e) (2^-24 twice), so it is off by at most (16 + 3) * 2^-23 * S; with exp2's 2^-22 and the weights'
two f16 parts (2^-22) a weight is off by 19 * 2^-23 * S + 4 * 2^-23, numerator and denominator together
by twice that, plus the accumulation of the keys (at most 2^-23 per 16 keys of a warp's share, 64 such
steps at the lengths used here) and of the merges (under 64 * 2^-24): in all
(2 * (19 * S + 4) + 128) * 2^-23 of the largest |v|.  The output's rounding adds eps / 2 of its value.
Where queries and output have 16 bits and a K/V head has more than 8 query rows, the weights of the
numerator may be f16: 2^-12 of each (and 2^-31 of the largest below f16's normal range, at most 2^12
keys), so at most 2^-12 + 2^-19 of the largest |v|.  (The longest of these cases take up to 160 steps of 16
keys, 2^-16 more; a weight's rounding is 2^-13 on average, so that the bound of 2^-12 has room for it.)"""
import numpy as np
import pytest

import operators_ref as R
import stt_b200
from stt_b200 import BeamSelector, Kv8Cache, SttError, beam_reorder
from stt_b200._lib import STT_E_DEVICE_FLAG, STT_E_INVALID_ARG

pytestmark = pytest.mark.gpu

NAMES = {"f32": "float32", "bf16": "bfloat16", "f16": "float16"}


def dt(name):
    import torch
    return getattr(torch, NAMES[name])


def i32(v):
    import torch
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Pair:
    """A cache over memory of the test's own and its 64-bit counterpart."""

    def __init__(self, seqs, heads, dim, cap, seed=0, fill=True):
        import torch
        self.shape = (seqs, heads, cap, dim)
        n = Kv8Cache.bytes(seqs, heads, dim, cap)
        gen = np.random.default_rng(seed)
        a, b = seqs * heads * cap * dim, seqs * heads * cap // 16
        raw = np.zeros(n, np.int8)
        if fill:
            raw[:2 * a] = gen.integers(-127, 128, 2 * a)
            raw[2 * a:] = gen.integers(-9, -4, 2 * b)
        self.mem = torch.from_numpy(raw).cuda()
        self.cache = Kv8Cache(seqs, heads, dim, cap, memory=self.mem)
        self.a, self.b = a, b
        self.k, self.v = self.halves(raw)

    def halves(self, raw):
        seqs, heads, cap, dim = self.shape
        a, b = self.a, self.b
        es = (seqs, heads, cap // 16)
        return (R.RefCache(raw[:a].reshape(self.shape), raw[2 * a:2 * a + b].reshape(es)),
                R.RefCache(raw[a:2 * a].reshape(self.shape), raw[2 * a + b:].reshape(es)))

    def same(self):
        k, v = self.halves(self.mem.cpu().numpy())
        for got, exp in ((k, self.k), (v, self.v)):
            assert np.array_equal(got.codes, exp.codes)
            assert np.array_equal(got.exps, exp.exps)

    def append(self, x, y, pos, count, seqs):
        for i, s in enumerate(seqs):
            self.k.append(s, pos[i], x[i, :count[i]].double().cpu().numpy())
            self.v.append(s, pos[i], y[i, :count[i]].double().cpu().numpy())


def rand(shape, dtype, seed, spread=1.0):
    import torch
    g = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * spread).to(dt(dtype))


# ------------------------------------------------------------------------------------ the cache


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 17, 40])
def test_append_writes_the_definitions_codes(dim, dtype, tokens):
    p = Pair(5, 3, dim, 64, seed=tokens)
    seqs, pos = [4, 0, 3, 1], [0, 7, 63, 1000]
    count = [tokens, max(0, tokens - 1), tokens, tokens // 2]
    x, y = rand((4, tokens, 3, dim), dtype, 1, 0.5), rand((4, tokens, 3, dim), dtype, 2, 3.0)
    p.cache.append(x, y, i32(pos), count=i32(count), seqs=i32(seqs))
    p.cache.status()
    p.append(x, y, pos, count, seqs)
    p.same()


def test_append_token_by_token_stays_within_a_step_and_reads_back():
    import torch
    p = Pair(2, 2, 64, 32, fill=False)
    x = rand((2, 40, 2, 64), "f32", 3) * torch.linspace(0.01, 4, 40, device="cuda")[:, None, None]
    for t in range(40):
        xt = x[:, t:t + 1]
        p.cache.append(xt, xt, i32([t, t]))
        p.append(xt, xt, [t, t], [1, 1], [0, 1])
    p.same()
    k, v = (torch.full((2, 20, 2, 64), 7.0, device="cuda") for _ in range(2))
    p.cache.read(k, v, i32([20, 24]), count=i32([20, 16]))
    p.cache.status()
    for i, (first, many) in enumerate([(20, 20), (24, 16)]):
        got = k[i].cpu().double().numpy()
        exp = p.k.values(i, range(first, first + many))
        assert np.array_equal(got[:many], exp)
        assert (got[many:] == 7.0).all()
        step = np.ldexp(1.0, p.k.exps[i][:, (np.arange(first, first + many) % 32) // 16]).T[..., None]
        assert (np.abs(exp - x[i, first:first + many].cpu().double().numpy()) < step).all()


def test_append_and_read_take_strided_tensors():
    import torch
    p = Pair(3, 2, 128, 48)
    wide = rand((3, 5, 3, 2, 128), "bf16", 4)
    x, y = wide[:, :, 1], wide[:, :, 2]
    p.cache.append(x, y, i32([3, 14, 40]))
    p.append(x, y, [3, 14, 40], [5, 5, 5], [0, 1, 2])
    p.same()
    heads_first = rand((3, 2, 5, 128), "f32", 5).transpose(1, 2)
    p.cache.append(heads_first, heads_first, i32([8, 19, 45]))
    p.append(heads_first, heads_first, [8, 19, 45], [5, 5, 5], [0, 1, 2])
    p.same()
    # V laid out another way than K
    p.cache.append(x, heads_first.to(torch.bfloat16), i32([13, 24, 50]))
    p.append(x, heads_first.to(torch.bfloat16), [13, 24, 50], [5, 5, 5], [0, 1, 2])
    p.same()
    out = torch.zeros(3, 5, 3, 2, 128, device="cuda")
    p.cache.read(out[:, :, 0], out[:, :, 2], i32([8, 19, 45]))
    for i, first in enumerate([8, 19, 45]):
        assert np.array_equal(out[i, :, 0].cpu().double().numpy(), p.k.values(i, range(first, first + 5)))
        assert np.array_equal(out[i, :, 2].cpu().double().numpy(), p.v.values(i, range(first, first + 5)))
    assert (out[:, :, 1] == 0).all()


@pytest.mark.parametrize("value", [0.0, 1e-38, 127.0, 127.00001, 1.0, 3e38, 2.0 ** -106, -255.0])
def test_append_at_the_borders_of_the_exponent(value):
    import torch
    p = Pair(1, 1, 64, 16, fill=False)
    x = torch.zeros(1, 3, 1, 64, device="cuda")
    x[0, 1, 0, 5] = value
    x[0, 2, 0, 6] = value / 3
    p.cache.append(x, -x, i32([0]))
    p.append(x, -x, [0], [3], [0])
    p.same()
    p.cache.status()


def test_append_reports_what_is_not_finite():
    import torch
    p = Pair(1, 1, 64, 16, fill=False)
    x = torch.ones(1, 2, 1, 64, device="cuda")
    x[0, 0, 0, 0], x[0, 1, 0, 1], x[0, 1, 0, 2] = float("inf"), float("nan"), -float("inf")
    p.cache.append(x, x, i32([4]))
    p.append(x, x, [4], [2], [0])
    p.same()
    with pytest.raises(SttError) as e:
        p.cache.status()
    assert e.value.code == STT_E_DEVICE_FLAG
    p.cache.status()  # reported once


def test_rows_out_of_range_are_skipped_and_reported():
    import torch
    p = Pair(4, 2, 64, 32)
    x = rand((3, 2, 2, 64), "f32", 6)
    out = torch.full((3, 2, 2, 64), 5.0, device="cuda")
    good_pos, good_count, good_seqs = [3, 4, 5], [2, 2, 2], [0, 1, 2]
    for name, bad in [("seqs", -1), ("seqs", 4), ("pos", -1), ("pos", 2 ** 31 - 2), ("count", 3), ("count", -1)]:
        a = dict(pos=list(good_pos), count=list(good_count), seqs=list(good_seqs))
        a[name][1] = bad
        t = {k: i32(v) for k, v in a.items()}
        p.cache.append(x, x, **t)
        for i in (0, 2):
            p.k.append(good_seqs[i], good_pos[i], x[i].double().cpu().numpy())
            p.v.append(good_seqs[i], good_pos[i], x[i].double().cpu().numpy())
        p.same()
        with pytest.raises(SttError) as e:
            p.cache.status()
        assert e.value.code == STT_E_INVALID_ARG
        p.cache.read(out, out.clone(), **t)
        p.cache.attention(x, out, **t)
        assert (out[1] == 5.0).all() and not (out[0] == 5.0).all()
        with pytest.raises(SttError):
            p.cache.status()
    p.cache.append(x, x, i32(good_pos), seqs=i32([2, 0, 2]))
    with pytest.raises(SttError):
        p.cache.status()
    # more new tokens than the ring holds from that position on
    many = rand((1, 32, 2, 64), "f32", 7)
    p = Pair(4, 2, 64, 32)
    p.cache.append(many, many, i32([1]))
    p.same()
    with pytest.raises(SttError):
        p.cache.status()
    p.cache.append(many, many, i32([32]))
    p.append(many, many, [32], [32], [0])
    p.same()
    p.cache.status()


# ------------------------------------------------------------------------------------ attention


def check_attention(p, q, out, before, pos, count, seqs, scale, window=0, start=None):
    import torch
    eps = torch.finfo(out.dtype).eps / 2 if out.dtype != torch.float32 else 0.0
    got = out.double().cpu().numpy()
    for i, s in enumerate(seqs):
        exp, S = R.attention(p.k, p.v, s, pos[i], q[i, :count[i]].double().cpu().numpy(), scale, window,
                             start[i] if start else 0)
        total = pos[i] + count[i]
        big = np.abs(p.v.values(s, range(max(0, total - p.shape[2]), max(1, total)))).max()
        tol = (2 * (19 * S + 4) + 128) * 2.0 ** -23 * big
        # (weights of 16 bits: 2^-12 of each, on either side of the division)
        if eps and q.dtype != torch.float32 and q.shape[1] * q.shape[2] // p.shape[1] > 8:
            tol += (2.0 ** -12 + 2.0 ** -19) * big
        assert (np.abs(got[i, :count[i]] - exp) <= tol + eps * np.abs(exp) + 2.0 ** -24 * (eps > 0)).all(), \
            (i, np.abs(got[i, :count[i]] - exp).max(), tol)
        assert torch.equal(out[i, count[i]:], before[i, count[i]:])


ATTENTION = [
    # heads, group, dim, tokens, positions (last tokens' first), cap, window, start, q, out
    (2, 1, 128, 1, [0, 1, 15, 16, 17, 120], 128, 0, None, "f32", "f32"),
    (2, 1, 64, 1, [0, 1, 15, 16, 17, 120], 128, 0, None, "f32", "f32"),
    (1, 8, 128, 1, [0, 300, 511], 512, 0, None, "bf16", "bf16"),
    (2, 3, 64, 1, [0, 300, 511], 512, 0, None, "f16", "f32"),
    (1, 1, 128, 1, [2000, 4095], 4096, 0, None, "f32", "f32"),       # split over CTAs
    (2, 4, 64, 1, [31, 700, 19999], 20000, 0, None, "bf16", "f32"),  # and joined through memory
    (1, 6, 128, 1, [12345], 20000, 0, None, "f32", "f32"),
    (3, 5, 64, 1, [100, 1000, 5000], 128, 0, None, "f32", "f16"),     # rings that wrapped
    (2, 1, 128, 1, [100, 1000, 5000], 128, 33, None, "f32", "f32"),   # and a window in them
    (2, 1, 128, 1, [100, 1000, 5000], 128, 1, None, "f32", "f32"),    # a window of the position itself
    (2, 4, 128, 7, [0, 9, 40], 64, 0, None, "f32", "f32"),
    (1, 3, 64, 37, [0, 5, 200], 256, 0, None, "f16", "f16"),
    (2, 1, 128, 37, [0, 5, 200], 256, 20, None, "bf16", "bf16"),
    (2, 1, 64, 16, [0, 16, 48], 64, 0, [3, 20, 60], "f32", "f32"),    # rows that start behind themselves are empty
    (1, 2, 128, 33, [0, 90], 128, 0, [40, 0], "f32", "bf16"),
    (2, 2, 128, 130, [0, 33, 100], 256, 0, [0, 7, 0], "bf16", "bf16"),
    (1, 16, 64, 100, [0, 33, 1000], 256, 77, [0, 7, 0], "f16", "f32"),
    (1, 1, 128, 200, [0, 57], 272, 0, None, "f32", "f32"),
    # many rows of 16 bits: tiles of 128 rows and steps of 128 keys
    (1, 1, 128, 64, [0], 64, 0, None, "bf16", "bf16"),
    (1, 1, 64, 64, [0], 64, 0, None, "f16", "f16"),
    (2, 1, 128, 128, [0, 1, 900], 1040, 0, None, "f16", "f16"),
    (1, 1, 128, 300, [0, 57, 700], 1024, 0, None, "bf16", "f16"),
    (1, 4, 64, 150, [0, 15, 333], 512, 0, None, "f16", "bf16"),
    (2, 5, 128, 77, [3, 600, 1000], 160, 0, None, "f16", "f16"),     # rings that wrapped inside a step
    (1, 3, 64, 40, [3, 600, 1000], 80, 0, None, "f16", "f16"),       # a ring shorter than a step
    (1, 2, 128, 260, [0, 200, 1000], 1280, 100, None, "f16", "f16"),
    (1, 2, 64, 260, [0, 200, 1000], 1280, 1, None, "f16", "f16"),
    (2, 1, 128, 140, [0, 200, 500], 640, 0, [0, 330, 100], "bf16", "bf16"),
    (1, 1, 64, 129, [0, 10], 160, 0, [200, 100], "f16", "f16"),      # no row sees anything; some rows do not
    # keys shared by clusters of 2, 4 and 8, runs without a step among them
    (8, 1, 128, 300, [0, 57, 3700], 4096, 0, None, "bf16", "bf16"),
    (4, 1, 128, 300, [0, 57, 3700], 4096, 0, [0, 300, 3500], "f16", "f16"),
    (1, 4, 64, 130, [5, 3900], 4096, 0, [0, 4020], "f16", "bf16"),
    (1, 8, 128, 9, [16000], 20000, 0, None, "bf16", "f16"),
    (2, 5, 128, 61, [50000, 2000], 4112, 0, None, "f16", "f16"),     # rings that wrapped
    (1, 2, 128, 200, [9000], 16384, 5000, None, "bf16", "bf16"),
]


@pytest.mark.parametrize("heads,group,dim,tokens,pos,cap,window,start,qt,ot", ATTENTION)
def test_attention_matches_the_formula(heads, group, dim, tokens, pos, cap, window, start, qt, ot):
    n = len(pos)
    p = Pair(n + 1, heads, dim, cap, seed=tokens + cap)
    seqs = list(range(n, 0, -1))
    count = [tokens if i == 0 else max(0, tokens - 3 * i) if tokens > 1 else 1 for i in range(n)]
    wide = rand((n, tokens, 2, heads * group, dim), qt, 8)
    q = wide[:, :, 1]
    out = rand((n, tokens, heads * group, dim), ot, 9)
    before = out.clone()
    scale = 0.7 / dim ** 0.5
    p.cache.attention(q, out, i32(pos), count=i32(count), seqs=i32(seqs), window=window,
                      start=None if start is None else i32(start), scale=scale)
    p.cache.status()
    check_attention(p, q, out, before, pos, count, seqs, scale, window, start)
    again = before.clone()
    p.cache.attention(q, again, i32(pos), count=i32(count), seqs=i32(seqs), window=window,
                      start=None if start is None else i32(start), scale=scale)
    import torch
    assert torch.equal(out, again)  # the order of the sums does not depend on the run


def test_long_sums_do_not_drift():
    """More items than CTAs fit, 60,000 positions each.  A product's accumulator is truncated at every block of 16 keys, by half a
    unit on average, at most 2^-24 of the running sum: runs of 128 blocks stay within 128 * 2^-24 of the output's norm (runs of
    all 938 blocks of a warp do not), and the softmax's 22 bits and exponents add under 2^-20."""
    import torch
    n, heads, dim, cap = 80, 8, 128, 60000
    p = Pair(1, heads, dim, cap, seed=3)
    q, out = rand((n, 1, heads, dim), "f32", 37), torch.zeros(n, 1, heads, dim, device="cuda")
    p.cache.attention(q, out, i32([cap - 1] * n), seqs=i32([0] * n), scale=0.01)
    p.cache.status()
    k, v = (torch.from_numpy(x.values(0, range(cap))).cuda() for x in (p.k, p.v))
    w = torch.softmax(torch.einsum("nhd,phd->nhp", q[:, 0].double(), k) * 0.01, -1)
    exact = torch.einsum("nhp,phd->nhd", w, v)
    error = ((out[:, 0].double() - exact).norm() / exact.norm()).item()
    assert error < 128 * 2.0 ** -24 + 2.0 ** -20, error


def test_attention_of_codes_in_masked_slots_and_uneven_exponents():
    """Exponents far apart between blocks, all-zero V blocks, and slots behind the last position that hold the largest codes."""
    import torch
    p = Pair(2, 1, 64, 64)
    raw = p.mem.cpu().numpy()
    a, b = p.a, p.b
    raw[2 * a:2 * a + b] = np.resize([-20, -6, -9, -8], b)
    raw[2 * a + b:] = np.resize([-100, 3, -30, -7], b)
    raw[a:a + 16 * 64] = 0       # sequence 0's first block of V
    raw[33 * 64:64 * 64] = 127   # sequence 0's K behind position 32
    p.mem.copy_(torch.from_numpy(raw))
    p.k, p.v = p.halves(raw)
    q = rand((2, 1, 1, 64), "f32", 10)
    for pos in ([5, 15], [20, 32], [32, 63]):
        out = torch.zeros(2, 1, 1, 64, device="cuda")
        p.cache.attention(q, out, i32(pos), scale=0.125)
        check_attention(p, q, out, out, pos, [1, 1], [0, 1], 0.125)
    q = rand((2, 1, 64, 64), "f16", 10)
    for pos in ([5, 15], [20, 32], [32, 63]):
        for scale in (0.125, -0.25, 0.0):
            out = torch.zeros(2, 1, 64, 64, dtype=torch.float16, device="cuda")
            p.cache.attention(q, out, i32(pos), scale=scale)
            check_attention(p, q, out, out, pos, [1, 1], [0, 1], scale)


def test_attention_with_large_and_small_queries_and_nan():
    import torch
    p = Pair(1, 1, 128, 64)
    for mul in (1e-30, 1e-3, 1e4):
        q = rand((1, 1, 8, 128), "f32", 11) * mul
        out = torch.zeros(1, 1, 8, 128, device="cuda")
        p.cache.attention(q, out, i32([50]), scale=1.0)
        check_attention(p, q, out, out, [50], [1], [0], 1.0)
    q = rand((1, 80, 3, 128), "bf16", 11)
    q[0, 5, 1, 5], q[0, 79, 2, 7] = float("nan"), float("inf")
    out = torch.zeros(1, 80, 3, 128, dtype=torch.bfloat16, device="cuda")
    p = Pair(1, 1, 128, 128)
    p.cache.attention(q, out, i32([40]))
    assert torch.isnan(out[0, 5, 1]).all() and torch.isnan(out[0, 79, 2]).all()
    assert int(torch.isnan(out).sum()) == 2 * 128
    q = rand((1, 2, 8, 128), "f32", 11)
    q[0, 0, 3, 5] = float("nan")
    out = torch.zeros(1, 2, 8, 128, device="cuda")
    p.cache.attention(q, out, i32([40]))
    assert torch.isnan(out[0, 0, 3]).all()
    rest = out.clone()
    rest[0, 0, 3] = 0
    assert torch.isfinite(rest).all()


def test_empty_calls_change_nothing():
    import torch
    p = Pair(2, 2, 64, 32)
    z = torch.zeros(0, 1, 2, 64, device="cuda")
    p.cache.append(z, z, i32([]))
    p.cache.attention(z, z.clone(), i32([]))
    p.cache.read(z, z.clone(), i32([]))
    p.same()


def test_operators_in_a_captured_graph_follow_the_positions():
    import torch
    p = Pair(2, 2, 128, 64)
    s = torch.cuda.Stream()
    x, q = rand((2, 1, 2, 128), "f32", 12), rand((2, 1, 4, 128), "f32", 13)
    out, pos = torch.zeros(2, 1, 4, 128, device="cuda"), i32([10, 30])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        h = torch.cuda.current_stream().cuda_stream
        p.cache.append(x, x, pos, stream=h)
        p.cache.attention(q, out, pos, stream=h)
    for step in range(5):
        at = [10 + 9 * step, 30 + 5 * step]
        pos.copy_(i32(at))
        x.copy_(rand((2, 1, 2, 128), "f32", 20 + step))
        g.replay()
        torch.cuda.synchronize()
        p.append(x, x, at, [1, 1], [0, 1])
        p.same()
        check_attention(p, q, out, out, at, [1, 1], [0, 1], 128 ** -0.5)


# ------------------------------------------------------------------------------------ beam search


def test_chunks_that_share_keys_in_a_captured_graph():
    """The tensor-core kernel in clusters, replayed for positions whose runs of keys are of other lengths (some empty)."""
    import torch
    p = Pair(1, 4, 128, 4096)
    q, out = rand((1, 300, 4, 128), "bf16", 30), rand((1, 300, 4, 128), "bf16", 31)
    pos = i32([0])
    p.cache.attention(q, out, pos)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        p.cache.attention(q, out, pos, stream=torch.cuda.current_stream().cuda_stream)
    for at in (0, 130, 3700, 1):
        pos.fill_(at)
        g.replay()
        torch.cuda.synchronize()
        check_attention(p, q, out, out, [at], [300], [0], 1 / 128 ** 0.5)
    p.cache.status()


@pytest.mark.parametrize("tokens,dtype", [(1, "f32"), (9, "bf16"), (300, "bf16"), (300, "f32")])
def test_starts_at_both_ends_of_the_integers(tokens, dtype):
    import torch
    p = Pair(3, 2, 64, 4096)
    q, out = rand((3, tokens, 2, 64), dtype, 35), rand((3, tokens, 2, 64), dtype, 36)
    pos, start = [3000, 100, 2500], [2 ** 31 - 1, -2 ** 31, 2600]
    before = out.clone()
    p.cache.attention(q, out, i32(pos), start=i32(start), window=2 ** 31 - 1)
    p.cache.status()
    assert not out[0].any()
    check_attention(p, q, out, before, pos, [tokens] * 3, [0, 1, 2], 0.125, 2 ** 31 - 1, start)


def test_two_caches_and_selectors_at_once_on_streams_of_their_own():
    import torch
    caches = [Pair(2, 2, 128, 20000, seed=s) for s in (1, 2)]
    beams = [BeamSelector(4, 8, 9000) for _ in range(2)]
    q = rand((2, 1, 8, 128), "f32", 32)
    chunk = rand((2, 40, 8, 128), "f16", 33)
    logits = rand((32, 9000), "f32", 34, 3.0)
    pos, chunk_pos = i32([19000, 12345]), i32([19000, 300])
    scores = torch.zeros(4, 8, device="cuda")
    streams = [torch.cuda.Stream() for _ in range(2)]

    def outputs():
        return (torch.empty_like(q), torch.empty_like(chunk), torch.empty_like(scores),
                torch.empty(4, 8, dtype=torch.int32, device="cuda"), torch.empty(4, 8, dtype=torch.int32, device="cuda"))

    def call(k, o, stream):
        caches[k].cache.attention(q, o[0], pos, stream=stream)
        caches[k].cache.attention(chunk, o[1], chunk_pos, stream=stream)
        beams[k].select(logits, scores, o[2], o[3], o[4], stream=stream)

    alone = [outputs() for _ in range(2)]
    for k in range(2):
        call(k, alone[k], 0)
        torch.cuda.synchronize()
    together = [[outputs() for _ in range(8)] for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(8):
        for k in range(2):
            call(k, together[k][i], streams[k].cuda_stream)
    torch.cuda.synchronize()
    for k in range(2):
        for o in together[k]:
            assert all(torch.equal(x, y) for x, y in zip(o, alone[k]))


def test_allocation_failures_of_the_handles_release_everything():
    import torch
    from stt_b200._lib import STT_E_OOM, lib
    torch.cuda.synchronize()
    free0 = torch.cuda.mem_get_info()[0]
    for make, least in ((lambda: Kv8Cache(64, 8, 128, 16384), 2), (lambda: BeamSelector(64, 32, 65537), 1)):
        failures = 0
        for k in range(10):
            assert lib().stt_debug_fail_allocation(k) == 0
            h = None
            try:
                h = make()
            except SttError as e:
                assert e.code == STT_E_OOM, e
                failures += 1
            finally:
                lib().stt_debug_fail_allocation(-1)
            done = h is not None
            if done:
                h.close()
            torch.cuda.synchronize()
            assert abs(torch.cuda.mem_get_info()[0] - free0) < (64 << 20), k
            if done:
                break
        assert failures == least and done


def run_select(logits, scores, done=None, eos=-1, selector=None):
    import torch
    batch, beams = scores.shape
    sel = selector or BeamSelector(batch, beams, logits.shape[1])
    out = [torch.full((batch, beams), 77, dtype=d, device="cuda") for d in (torch.float32, torch.int32, torch.int32, torch.uint8)]
    sel.select(logits, scores, *out[:3], done=done, next_done=out[3], eos=eos)
    return sel, out


def check_select(logits, scores, done, eos, out):
    batch, beams = scores.shape
    exp = R.select(logits.double().cpu().numpy().reshape(batch, beams, -1), scores.cpu().numpy(),
                   None if done is None else done.cpu().numpy(), eos)
    got = [o.cpu().numpy() for o in out]
    assert np.array_equal(got[1], exp[1]) and np.array_equal(got[2], exp[2])
    assert np.array_equal(got[3].astype(bool), exp[3])
    # the log sum's exponentials are f32 sums of up to 16, each term and step off by 2^-23 at most, then
    # 64 bits: 2^-18 of the sum; the score itself is rounded to f32 once
    fin = np.isfinite(exp[0])
    assert np.array_equal(np.isfinite(got[0]), fin)
    assert (np.abs(got[0][fin] - exp[0][fin]) <= 2.0 ** -18 + 2.0 ** -24 * np.abs(exp[0][fin])).all()


@pytest.mark.parametrize("batch,beams,vocab", [(1, 1, 1), (1, 1, 8000), (3, 4, 8000), (2, 8, 4096), (2, 8, 4097), (1, 32, 33),
                                               (2, 3, 2), (1, 5, 1), (4, 16, 12289), (1, 32, 70001)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_select_matches_a_stable_sort(batch, beams, vocab, dtype):
    logits = rand((batch * beams, vocab), dtype, vocab, 3.0)
    scores = rand((batch, beams), "f32", 1, 5.0)
    sel, out = run_select(logits, scores)
    sel.status()
    check_select(logits, scores, None, -1, out)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_select_of_ties_takes_the_lowest_index(dtype):
    import torch
    logits = torch.zeros(2 * 6, 5000, dtype=dt(dtype), device="cuda")
    logits[3, 4321] = 1.0
    logits[4, 4321] = 1.0
    logits[7:9] = -0.0
    scores = torch.zeros(2, 6, device="cuda")
    sel, out = run_select(logits, scores)
    check_select(logits, scores, None, -1, out)
    sel.status()


def test_select_with_masked_logits_and_first_steps():
    import torch
    inf = float("inf")
    logits = rand((3 * 4, 9000), "f32", 2, 3.0)
    logits[0:4, 3:] = -inf      # fewer finite candidates than beams in a row
    logits[5] = -inf            # a row that its mask leaves empty
    logits[8:12] = torch.finfo(torch.float32).min
    logits[9, 17] = 0.0
    scores = rand((3, 4), "f32", 3, 2.0)
    scores[1, 1:] = -inf
    sel, out = run_select(logits, scores)
    check_select(logits, scores, None, -1, out)
    scores[1] = -inf            # nothing finite: the lowest candidates
    sel, out = run_select(logits, scores, selector=sel)
    check_select(logits, scores, None, -1, out)
    logits[4:8] = -inf
    scores[1] = 0.0
    sel, out = run_select(logits, scores, selector=sel)
    check_select(logits, scores, None, -1, out)
    sel.status()


@pytest.mark.parametrize("eos", [0, 5, 8999])
def test_select_with_beams_that_ended(eos):
    import torch
    logits = rand((4 * 5, 9000), "bf16", 4, 3.0)
    scores = rand((4, 5), "f32", 5, 2.0)
    done = torch.zeros(4, 5, dtype=torch.uint8, device="cuda")
    done[0, 2] = done[1, 0] = done[1, 1] = 1
    done[2] = 1
    scores[0, 2] = 50.0
    logits[15:20, eos] = 40.0
    logits[11] = float("nan")   # a beam that ended: its logits are not looked at
    sel, out = run_select(logits, scores, done, eos)
    logits[11] = 0
    check_select(logits, scores, done, eos, out)
    sel.status()
    # in place: the next scores and flags over the present ones
    nxt = [torch.zeros(4, 5, dtype=torch.int32, device="cuda") for _ in range(2)]
    s2, d2 = scores.clone(), done.clone()
    sel.select(logits, s2, s2, nxt[0], nxt[1], done=d2, next_done=d2, eos=eos)
    assert torch.equal(s2, out[0]) and torch.equal(d2, out[3]) and torch.equal(nxt[0], out[1])


def test_select_when_poor_chunks_pull_the_bound_down():
    """32 beams over 32 chunks of which every last one is masked: the bound lets more through than the list holds."""
    logits = rand((32, 32 * 4096 - 8), "f32", 6, 1.0)
    logits[:, 31 * 4096:] = -float("inf")
    scores = rand((1, 32), "f32", 7, 0.01)
    _, out = run_select(logits, scores)
    check_select(logits, scores, None, -1, out)


def test_select_reports_nan_and_infinite_rows():
    import torch
    for bad, where in [(float("nan"), "logit"), (float("inf"), "logit"), (float("nan"), "score"), (float("inf"), "score")]:
        logits, scores = rand((2 * 3, 500), "f32", 8, 3.0), rand((2, 3), "f32", 9)
        if where == "logit":
            logits[1, 400] = bad
        else:
            scores[0, 1] = bad
        sel, out = run_select(logits, scores)
        check_select(logits, scores, None, -1, out)
        with pytest.raises(SttError) as e:
            sel.status()
        assert e.value.code == STT_E_DEVICE_FLAG
        sel.status()


def test_select_takes_strided_and_unaligned_rows():
    import torch
    for dtype, off in (("bf16", 1), ("bf16", 3), ("f32", 1), ("f16", 7)):
        wide = rand((6, 4200), dtype, 10, 3.0)
        logits = wide.view(-1)[off:off + 5 * 4200 + 4111].as_strided((6, 4111), (4200, 1))
        scores = rand((2, 3), "f32", 11)
        sel = BeamSelector(4, 8, 5000)
        _, out = run_select(logits, scores, selector=sel)
        check_select(logits, scores, None, -1, out)
        sel.status()


def ref_reorder(states, parents, held=None):
    got = states.clone()
    g, beams = parents.shape
    for i in range(g):
        for b in range(beams):
            p = int(parents[i, b])
            if 0 <= p < beams:
                m = states.shape[2] if held is None else max(0, min(states.shape[2], int(held[i, b])))
                got[i * beams + b, :, :m] = states[i * beams + p, :, :m]
    return got


@pytest.mark.parametrize("groups,beams,segments,units,unit,dtype", [
    (1, 1, 2, 5, 8, "f32"), (3, 2, 3, 700, 64, "bf16"), (2, 4, 5, 33, 72, "bf16"), (2, 5, 1, 1, 1, "f32"), (2, 8, 3, 257, 3, "f16"),
    (1, 16, 4, 100, 128, "f32"), (2, 32, 2, 65, 16, "bf16"), (1, 7, 2, 3, 33, "f16")])
def test_reorder_in_place(groups, beams, segments, units, unit, dtype):
    import torch
    rng = np.random.default_rng(beams)
    states = rand((groups * beams, segments, units, unit), dtype, 12)
    parents = i32(rng.integers(0, beams, (groups, beams)).tolist())
    for held in (None, i32(rng.integers(-1, units + 2, (groups, beams)).tolist())):
        exp = ref_reorder(states, parents.cpu(), None if held is None else held.cpu())
        beam_reorder(states, parents, held=held)
        assert torch.equal(states, exp)
    parents[0, beams - 1] = beams
    parents[0, 0] = -1
    exp = ref_reorder(states, parents.cpu())
    beam_reorder(states, parents)
    assert torch.equal(states, exp)


def test_reorder_of_interleaved_rows_leaves_the_gaps():
    import torch
    wide = rand((3, 12, 40, 16), "f32", 13)
    states = wide.transpose(0, 1)[:, :, :33]  # [12 rows, 3 segments, 33, 16], the rows inside the segments
    parents = i32([[1, 0, 1, 1], [3, 3, 3, 3], [0, 1, 2, 3]])
    exp = wide.clone()
    exp.transpose(0, 1)[:, :, :33] = ref_reorder(states, parents.cpu())
    beam_reorder(states, parents)
    assert torch.equal(wide, exp)


def test_cache_reorder_moves_sequences():
    p = Pair(7, 2, 64, 48)
    parents, held = [[2, 2, 0], [1, 0, 9]], [[20, 48, 33], [100, 0, 5]]
    k0, v0 = (c.codes.copy() for c in (p.k, p.v)), None
    k0, v0, ke, ve = p.k.codes.copy(), p.v.codes.copy(), p.k.exps.copy(), p.v.exps.copy()
    p.cache.reorder(i32(parents), held=i32(held))
    for g in range(2):
        for b in range(3):
            src, dst = parents[g][b], 3 * g + b
            if src > 2:
                continue
            blocks = min(3, -(-held[g][b] // 16))
            for c, c0, e0 in ((p.k, k0, ke), (p.v, v0, ve)):
                c.codes[dst, :, :16 * blocks] = c0[3 * g + src, :, :16 * blocks]
                c.exps[dst, :, :blocks] = e0[3 * g + src, :, :blocks]
    p.same()


# ------------------------------------------------------------------------------------ together


def test_beam_decoding_over_the_cache_matches_64_bits():
    """Two utterances with three beams each step together: append, attention, a projection to logits,
    selection, reordering, with a table of token embeddings for q, k and v, against the same loop on
    the 64-bit operators.  The table is small whole numbers / 8, so every run has clear margins."""
    import torch
    G, B, H, D, V, STEPS = 2, 3, 2, 64, 50, 40
    rng = np.random.default_rng(14)
    table = torch.from_numpy(rng.integers(-8, 9, (V, 3, H, D)) / 8.0).float().cuda()
    head = torch.from_numpy(rng.integers(-8, 9, (H * D, V)) / 8.0).float().cuda()
    p = Pair(G * B, H, D, 32, fill=False)
    sel = BeamSelector(G, B, V)
    scores = torch.tensor([[0.0] + [-float("inf")] * (B - 1)] * G, device="cuda")
    tokens = i32([[1] * B, [2] * B])
    parents = i32([[0] * B] * G)
    out = torch.zeros(G * B, 1, H, D, device="cuda")
    r_scores, r_tokens = scores.cpu().numpy(), tokens.cpu().numpy()
    for step in range(STEPS):
        x = table[tokens.view(-1).long()]
        pos = i32([step] * (G * B))
        p.cache.append(x[:, None, 1], x[:, None, 2], pos)
        p.cache.attention(x[:, None, 0], out, pos, window=20)
        logits = out.view(G * B, -1) @ head
        sel.select(logits, scores, scores, parents, tokens)
        p.cache.reorder(parents, held=i32([[step + 1] * B] * G))
        # the same on the plain operators
        rx = table.double().cpu().numpy()[r_tokens.reshape(-1)]
        rl = np.zeros((G * B, V))
        for i in range(G * B):
            p.k.append(i, step, rx[i, None, 1])
            p.v.append(i, step, rx[i, None, 2])
            rl[i] = R.attention(p.k, p.v, i, step, rx[i, None, 0], D ** -0.5, 20)[0].reshape(-1) @ head.double().cpu().numpy()
        r_scores, r_parents, r_tokens, _ = R.select(rl.reshape(G, B, V), r_scores)
        src = (np.arange(G)[:, None] * B + r_parents).reshape(-1)
        p.k, p.v = (R.RefCache(c.codes[src], c.exps[src]) for c in (p.k, p.v))
        assert np.array_equal(parents.cpu().numpy(), r_parents) and np.array_equal(tokens.cpu().numpy(), r_tokens), step
        assert np.abs(scores.cpu().numpy() - r_scores).max() < 1e-3
    k, v = p.halves(p.mem.cpu().numpy())
    held = np.arange(max(0, (STEPS + 15) // 16 * 16 - 32), STEPS)
    for i in range(G * B):
        assert np.array_equal(k.values(i, held), p.k.values(i, held))
        assert np.array_equal(v.values(i, held), p.v.values(i, held))
    sel.status()
    p.cache.status()
