"""The decode operators at the ends of their ranges, on the GPU, against the plain 64-bit implementations
of tests/operators_ref.py: exponents and positions near their limits, peaked and masked rows of logits,
padded batches.  Tolerances are those of tests/test_gpu_operators.py unless a test derives its own."""
import numpy as np
import pytest

import operators_ref as R
from stt_b200 import BeamSelector, SttError
from stt_b200._lib import STT_E_DEVICE_FLAG, STT_E_INVALID_ARG
from test_gpu_operators import Pair, check_attention, check_select, dt, i32, rand, run_select

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_read_is_exact_for_every_exponent(dim, dtype):
    """A value is a whole number of at most 7 bits times a power of two: exact in f32 and bf16 (the largest here
    is 127 * 2^121 < 2^128), and in f16 the nearest f16 (infinity beyond 65,504)."""
    import torch
    exps = [-100, -60, -27, 0, 9, 60, 103, 104, 105, 106, 113, 120, 121, 121, -99, 105]
    p = Pair(1, 2, dim, 16 * len(exps), seed=1)
    raw = p.mem.cpu().numpy()
    raw[2 * p.a:] = np.tile(np.array(exps, np.int8), 4)
    raw[0:p.a:dim] = 0  # a zero in every row
    p.mem.copy_(torch.from_numpy(raw))
    p.k, p.v = p.halves(raw)
    out = torch.zeros(2, 1, p.shape[2], 2, dim, dtype=dt(dtype), device="cuda")
    p.cache.read(out[0], out[1], i32([0]))
    p.cache.status()
    for got, half in ((out[0, 0], p.k), (out[1, 0], p.v)):
        exp = half.values(0, range(p.shape[2]))
        if dtype == "f16":
            with np.errstate(over="ignore"):
                exp = exp.astype(np.float16).astype(np.float64)
        assert np.array_equal(got.double().cpu().numpy(), exp)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("value", [2.5e33, 2.7e33, -1e36, 3e38])
def test_the_largest_values_are_read_back_as_they_were_appended(dtype, value):
    import torch
    p = Pair(1, 2, 64, 32, fill=False)
    x = rand((1, 5, 2, 64), dtype, 2, 1e33)
    x[0, 1, 0, 5] = value
    x[0, 3, 1, 9] = 0.0
    out = torch.zeros(2, 1, 5, 2, 64, dtype=dt(dtype), device="cuda")
    p.cache.append(x, -x, i32([7]))
    p.append(x, -x, [7], [5], [0])
    p.same()
    p.cache.read(out[0], out[1], i32([7]))
    p.cache.status()
    assert np.array_equal(out[0, 0].double().cpu().numpy(), p.k.values(0, range(7, 12)))
    assert np.array_equal(out[1, 0].double().cpu().numpy(), p.v.values(0, range(7, 12)))


@pytest.mark.parametrize("dtype,largest", [("f32", 3.4e38), ("bf16", 3.3895313892515355e38), ("f16", 65504.0), ("f32", 1e-38)])
def test_an_infinity_next_to_the_largest_values_is_the_largest_code(dtype, largest):
    """The block's exponent is then 122 in f32 and bf16, where 127 steps are more than an f32 holds."""
    import torch
    for infinite in (float("inf"), -float("inf")):
        p = Pair(1, 1, 64, 16, fill=False)
        x = torch.ones(1, 3, 1, 64, dtype=dt(dtype), device="cuda")
        x[0, 0, 0, 0], x[0, 1, 0, 1], x[0, 2, 0, 2] = largest, infinite, float("nan")
        p.cache.append(x, -x, i32([3]))
        p.append(x, -x, [3], [3], [0])
        p.same()
        assert p.k.codes[0, 0, 4, 1] == (127 if infinite > 0 else -127)
        with pytest.raises(SttError) as e:
            p.cache.status()
        assert e.value.code == STT_E_DEVICE_FLAG


def select_error(logits, scores, tolerance):
    """Checks a selection, its scores to `tolerance` and their rounding to f32."""
    sel, out = run_select(logits, scores)
    check_select(logits, scores, None, -1, out)
    sel.status()
    exp = R.select(logits.double().cpu().numpy().reshape(*scores.shape, -1), scores.cpu().numpy())[0]
    got = out[0].double().cpu().numpy()
    fin = np.isfinite(exp)
    off = np.abs(got[fin] - exp[fin]) - 2.0 ** -24 * np.abs(exp[fin])
    assert off.max() <= tolerance, off.max()


@pytest.mark.parametrize("dtype,vocab,tile", [("f32", 8000, 2048), ("bf16", 16000, 4096), ("f16", 16000, 4096)])
def test_log_sums_of_rows_with_one_large_logit(dtype, vocab, tile):
    """A trained model's rows: one logit far above the others, in a later tile of a CTA that takes several.  The
    large logit is the sum's reference, its term 1: a thread's at most 32 terms, added in two chains, are off by
    16 * 2^-24 of the sum, the powers by 2^-22 of themselves, and the arguments of the others (d below the
    reference, d * 3 * 2^-24 off) weigh e^-d: 2^-20 + 2^-22 + 2^-23 in all."""
    rng = np.random.default_rng(vocab)
    logits = rand((64 * 8, vocab), dtype, 3, 1.0)
    scores = rand((64, 8), "f32", 4, 2.0)
    for row in range(64 * 8):
        at = int(rng.integers(tile, 2 * tile) if row % 2 else rng.integers(3 * tile, vocab))
        logits[row, at] = float(rng.uniform(25.0, 62.0))
    select_error(logits, scores, 2.0 ** -20 + 2.0 ** -22 + 2.0 ** -23)


@pytest.mark.parametrize("tokens", [1, 3, 20])
def test_padding_rows_do_not_count_as_repeated_sequences(tokens):
    p = Pair(4, 2, 64, 64)
    x = rand((5, tokens, 2, 64), "f32", 5)
    seqs, pos, count = [2, 0, 0, 2, 0], [5, 0, 9, 17, 0], [tokens, 0, tokens, 0, 0]
    p.cache.append(x, x, i32(pos), count=i32(count), seqs=i32(seqs))
    p.append(x, x, pos, count, seqs)
    p.same()
    p.cache.status()
    count[3] = 1  # now sequence 2 does come twice
    p.cache.append(x, x, i32(pos), count=i32(count), seqs=i32(seqs))
    with pytest.raises(SttError) as e:
        p.cache.status()
    assert e.value.code == STT_E_INVALID_ARG


def test_outputs_whose_rows_lie_on_one_another_are_refused():
    import torch
    p = Pair(2, 2, 64, 32)
    q = rand((2, 3, 4, 64), "f32", 6)
    wide = torch.zeros(2, 3, 4, 128, device="cuda")
    flat = torch.zeros(64 * 64, device="cuda")

    def refused(call, text):
        with pytest.raises(SttError) as e:
            call()
        assert e.value.code == STT_E_INVALID_ARG and text in str(e.value)

    bad = [torch.zeros(1, 3, 4, 64, device="cuda").expand(2, 3, 4, 64), torch.zeros(2, 1, 4, 64, device="cuda").expand(2, 3, 4, 64),
           torch.zeros(2, 3, 1, 64, device="cuda").expand(2, 3, 4, 64), flat.as_strided((2, 3, 4, 64), (768, 256, 60, 1)),
           flat.as_strided((2, 3, 4, 64), (768, 128, 64, 1)), flat.as_strided((2, 3, 4, 64), (512, 256, 64, 1))]
    for out in bad:
        refused(lambda: p.cache.attention(q, out, i32([5, 6])), "on one another")
    k = torch.zeros(2, 3, 2, 64, device="cuda")
    for out in (torch.zeros(1, 3, 2, 64, device="cuda").expand(2, 3, 2, 64), flat.as_strided((2, 3, 2, 64), (384, 64, 64, 1))):
        refused(lambda: p.cache.read(out, k, i32([5, 6])), "on one another")
        refused(lambda: p.cache.read(k, out, i32([5, 6])), "on one another")
    refused(lambda: p.cache.read(k, k, i32([5, 6])), "one memory")
    # gaps, another order of the dimensions, and strides of dimensions of one entry are as good as any
    p.cache.attention(q, wide[..., :64], i32([5, 6]))
    p.cache.attention(q, torch.zeros(4, 3, 2, 64, device="cuda").permute(2, 1, 0, 3), i32([5, 6]))
    one = flat.as_strided((1, 1, 4, 64), (0, 0, 64, 1))
    p.cache.attention(q[:1, :1], one, i32([5]))
    # inputs may repeat: one query, key and value for all rows
    p.cache.attention(q[:1].expand(2, 3, 4, 64), torch.zeros(2, 3, 4, 64, device="cuda"), i32([5, 6]))
    p.cache.append(k[:1].expand(2, 3, 2, 64), k[:1].expand(2, 3, 2, 64), i32([5, 6]))
    p.cache.status()


@pytest.mark.parametrize("tokens,group,dtype", [(20, 16, "bf16"), (20, 16, "f16"), (20, 16, "f32"), (1, 1, "f32"), (5, 1, "bf16")])
def test_attention_at_the_last_positions(tokens, group, dtype):
    """Positions up to the largest that a batch may have, the last step of 128 keys reaching past 2^31."""
    heads, cap = 2, 4096
    pos = 2 ** 31 - 1 - 32 - tokens
    end = -(-(pos + tokens) // 16) * 16
    p = Pair(1, heads, 128, cap, seed=7)
    q, out = (rand((1, tokens, heads * group, 128), dtype, seed) for seed in (8, 9))
    for start in (0, end - cap + 64):
        p.cache.attention(q, out, i32([pos]), start=i32([start]), scale=0.05)
        p.cache.status()
        check_attention(p, q, out, out, [pos], [tokens], [0], 0.05, 0, [start])


@pytest.mark.parametrize("tokens,group,dtype", [(1, 1, "f32"), (3, 2, "f32"), (20, 16, "bf16")])
def test_attention_of_queries_near_the_least_normal_values(tokens, group, dtype):
    """Keys near the largest values: the scores are ordinary numbers."""
    import torch
    p = Pair(1, 2, 128, 4096, seed=10)
    raw = p.mem.cpu().numpy()
    raw[2 * p.a:2 * p.a + p.b] = 114
    p.mem.copy_(torch.from_numpy(raw))
    p.k, p.v = p.halves(raw)
    q, out = rand((1, tokens, 2 * group, 128), dtype, 11, 1e-36), rand((1, tokens, 2 * group, 128), dtype, 12)
    p.cache.attention(q, out, i32([3700]), scale=0.25)
    p.cache.status()
    check_attention(p, q, out, out, [3700], [tokens], [0], 0.25)


@pytest.mark.parametrize("dim,tokens,window,spread", [(128, 20, 0, 1.0), (128, 20, 0, 12.0), (64, 24, 0, 4.0), (128, 30, 3000, 4.0), (128, 3, 0, 4.0)])
@pytest.mark.parametrize("qt", ["f16", "bf16"])
def test_f16_chunks_are_as_near_as_their_rounding_allows(dim, tokens, window, spread, qt):
    """An f16 output holds 11 bits and is rounded once: the result may be no further from the 64-bit values than those
    rounded to f16 are, but for sums in f32 and weights in two f16 parts.  These are off by e <= 2^-17 of a value here
    (18 S 2^-23 of it and less, S under 100), independent of the rounding of up to 2^-11, in the mean over an output
    2^-11 / sqrt(3) * about 0.7: together sqrt(1 + (2^-17 / 2^-12.3)^2) < 1.001 times the rounding alone."""
    import torch
    heads, group, pos = 2, 16, 3700
    p = Pair(1, heads, dim, 4096, seed=13)
    q = rand((1, tokens, heads * group, dim), qt, 14, spread)
    out = torch.zeros(1, tokens, heads * group, dim, dtype=torch.float16, device="cuda")
    scale = dim ** -0.5
    p.cache.attention(q, out, i32([pos]), window=window, scale=scale)
    p.cache.status()
    exact, _ = R.attention(p.k, p.v, 0, pos, q[0].double().cpu().numpy(), scale, window)
    least = np.linalg.norm(exact.astype(np.float16).astype(np.float64) - exact)
    off = np.linalg.norm(out[0].double().cpu().numpy() - exact)
    print("error", off, "rounding alone", least)
    assert off <= 1.001 * least


def test_append_takes_a_batch_padded_beyond_the_capacity():
    p = Pair(3, 2, 64, 32)
    x = rand((3, 50, 2, 64), "bf16", 50)
    p.cache.append(x, x, i32([5, 16, 0]), count=i32([20, 32, 0]))
    p.append(x, x, [5, 16, 0], [20, 32, 0], [0, 1, 2])
    p.same()
    p.cache.status()
    with pytest.raises(SttError) as e:
        p.cache.append(x, x, i32([0, 0, 0]))
    assert e.value.code == STT_E_INVALID_ARG and "capacity" in str(e.value)
    p.cache.append(x, x, i32([0, 3, 0]), count=i32([33, 32, 1]))  # two rows that the ring does not hold
    p.append(x, x, [0, 0, 0], [0, 0, 1], [0, 1, 2])
    p.same()
    with pytest.raises(SttError) as e:
        p.cache.status()
    assert e.value.code == STT_E_INVALID_ARG


@pytest.mark.parametrize("tokens,group,dtype", [(1, 1, "f32"), (5, 1, "f32"), (20, 16, "bf16")])
def test_attention_over_blocks_of_v_110_binades_apart(tokens, group, dtype):
    """The widest spread that the softmax's sum is promised to hold: blocks of nothing but zeros (exponent -100) beside
    blocks of values up to 127 * 2^10, the zeros' scores below the others' and above them."""
    import torch
    heads = 2
    for high in (0, 1):
        p = Pair(1, heads, 128, 4096, seed=15)
        raw = p.mem.cpu().numpy()
        codes = raw[p.a:2 * p.a].reshape(heads, 256, 16 * 128)
        codes[:, ::2] = 0
        raw[2 * p.a + p.b:] = np.tile(np.array([-100, 10], np.int8), heads * 128)
        keys = raw[:p.a].reshape(heads, 256, 16, 128)
        keys[..., 0] = 100
        keys[:, high::2, :, 0] = 127  # these blocks' scores are the higher ones
        p.mem.copy_(torch.from_numpy(raw))
        p.k, p.v = p.halves(raw)
        q, out = rand((1, tokens, heads * group, 128), dtype, 16, 0.1), rand((1, tokens, heads * group, 128), dtype, 17)
        q[..., 0] = 10.0
        p.cache.attention(q, out, i32([3700]), scale=1.0)
        p.cache.status()
        check_attention(p, q, out, out, [3700], [tokens], [0], 1.0)


@pytest.mark.parametrize("beams", [1, 2, 4, 8])
@pytest.mark.parametrize("vocab,dtype", [(65537, "f32"), (65537, "bf16"), (130000, "bf16")])
def test_select_joins_many_chunks_of_a_row(beams, vocab, dtype):
    """One utterance's rows in 9 to 32 chunks each: whole chunks masked, chunks with fewer finite logits than beams,
    beams that ended, and ties across chunks."""
    import torch
    inf = float("inf")
    eos = vocab - 3
    for case in range(5):
        logits = rand((beams, vocab), dtype, 20 + case, 3.0)
        scores = rand((1, beams), "f32", 30 + case, 2.0)
        done = None
        if case == 1:    # all but the row's ends
            logits[:, 1000:vocab - 1000] = -inf
        elif case == 2:  # a chunk or more with a single finite logit, the others' ones poor
            logits[:, vocab // 4:vocab // 2] = -inf
            logits[:, vocab // 3] = 20.0
            logits[0, vocab // 2:] = -inf
        elif case == 3:  # fewer finite logits in the whole row than beams
            logits[:] = -inf
            logits[0, vocab - 1] = 1.0
            logits[beams - 1, 5] = 1.0
        elif case == 4:
            logits[:] = 0.0
            logits[:, vocab // 2] = 1.0
            done = torch.zeros(1, beams, dtype=torch.uint8, device="cuda")
            done[0, beams // 2] = 1
        sel, out = run_select(logits, scores, done, eos if case == 4 else -1)
        check_select(logits, scores, done, eos if case == 4 else -1, out)
        sel.status()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_select_when_a_chunk_is_masked_behind_a_poor_one(dtype):
    """32 beams: four chunks a row, one of them masked whole, one with fewer finite logits than beams: their bounds stay at
    -inf, which more logits reach than a list takes."""
    inf = float("inf")
    logits = rand((32, 131064), dtype, 40, 0.001)
    logits[:, 32768:65536] = -inf
    logits[:, 65536 + 20:98304] = -inf
    logits[5] = 0.25   # ties all over a row
    logits[6, 40000:] = -inf
    scores = rand((1, 32), "f32", 41, 0.001)
    _, out = run_select(logits, scores)
    check_select(logits, scores, None, -1, out)


@pytest.mark.parametrize("n,group,tokens,cap", [(80, 1, 1, 60000), (80, 1, 1, 16000), (16, 8, 1, 60000), (6, 1, 24, 60000), (80, 1, 1, 2048)])
def test_the_error_of_f32_outputs_does_not_grow_with_the_context(n, group, tokens, cap):
    """Relative to the outputs' norm: weights in two f16 parts and their exponentials 2^-22, a block's product 2^-24, and a
    warp's additions, at most 938 here and each rounded to nearest (0.29 of 2^-24 in the mean) over a sum that grows like
    the root of their number, 0.29 * sqrt(938 / 2) * 2^-24; runs of up to 32 blocks may truncate instead, 32 * 2^-26."""
    import torch
    heads, dim = 8, 128
    p = Pair(1, heads, dim, cap, seed=3)
    q, out = rand((n, tokens, heads * group, dim), "f32", 37), torch.zeros(n, tokens, heads * group, dim, device="cuda")
    p.cache.attention(q, out, i32([cap - tokens] * n), seqs=i32([0] * n), scale=0.01)
    p.cache.status()
    k, v = (torch.from_numpy(x.values(0, range(cap))).cuda().permute(1, 0, 2) for x in (p.k, p.v))
    hidden = torch.arange(cap, device="cuda") > cap - tokens + torch.arange(tokens, device="cuda")[:, None]
    error = []
    for i in range(0, n, max(1, n // 12)):
        s = torch.einsum("thgd,hpd->htgp", q[i].double().view(tokens, heads, group, dim), k) * 0.01
        w = torch.softmax(s.masked_fill(hidden[None, :, None], -float("inf")), -1)
        exact = torch.einsum("htgp,hpd->thgd", w, v)
        error.append(((out[i].double().view_as(exact) - exact).norm() / exact.norm()).item())
    print("errors", error)
    assert np.mean(error) < 2.0 ** -22 + 2.0 ** -24 + max(0.29 * (938 / 2) ** 0.5 * 2.0 ** -24, 32 * 2.0 ** -26), error


def test_more_tokens_than_positions_are_refused():
    """The counts of such a batch could be small, but its grid has no size."""
    from stt_b200._lib import KV8_BATCH, KV8_TENSOR, lib
    p = Pair(1, 1, 64, 32)
    x, one = rand((1, 1, 1, 64), "f32", 60), i32([0])
    tensor = KV8_TENSOR.pack(x.data_ptr(), 256, 64, 64, 0, 0)
    out = KV8_TENSOR.pack(rand((1, 1, 1, 64), "f32", 61).data_ptr(), 2 ** 40, 64, 64, 0, 0)
    for tokens in (2 ** 31 - 1, 2 ** 31 - 31, 2 ** 31 - 1000):
        batch = KV8_BATCH.pack(0, one.data_ptr(), one.data_ptr(), 1, tokens)
        assert lib().stt_kv8_append_device(p.cache._h, batch, tensor, tensor, None) == STT_E_INVALID_ARG
        assert lib().stt_kv8_read_device(p.cache._h, batch, out, tensor, None) == STT_E_INVALID_ARG
        assert lib().stt_kv8_attention_device(p.cache._h, batch, tensor, 1, None, 0, 1.0, out, None) == STT_E_INVALID_ARG
    p.cache.status()
    p.same()
