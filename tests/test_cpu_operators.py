"""Refusals of the decode operators that need no device, and the plain implementations that their GPU
tests compare with, checked on cases worked out by hand."""
import ctypes as C
import math

import numpy as np
import pytest

import operators_ref as R
from stt_b200 import BeamSelector, Kv8Cache, SttError, beam_reorder
from stt_b200._lib import BEAM_STATES, STT_E_INVALID_ARG, lib


def refused(rc, text):
    msg = lib().stt_last_error().decode()
    assert rc == STT_E_INVALID_ARG and text in msg, (rc, msg)


@pytest.mark.parametrize("args", [(0, 1, 64, 16), (1, 0, 64, 16), (1, 1, 96, 16), (1, 1, 64, 0), (1, 1, 64, 24),
                                  (-1, 1, 64, 16), (1, 1, 64, -16), (2 ** 30, 2 ** 10, 128, 2 ** 20)])
def test_cache_shapes_are_checked(args):
    n, out = C.c_size_t(7), C.c_void_p(1)
    refused(lib().stt_kv8_cache_bytes(*args, C.byref(n)), "no 8-bit cache")
    refused(lib().stt_kv8_cache_create(0, *args, None, C.byref(out)), "no 8-bit cache")
    assert n.value == 7 and not out.value


def test_cache_bytes():
    assert Kv8Cache.bytes(3, 2, 64, 48) == 2 * (3 * 2 * 48 * 64 + 3 * 2 * 3)
    assert Kv8Cache.bytes(512, 16, 128, 65536) == 2 * (512 * 16 * 65536 * 128 + 512 * 16 * 4096)  # past 32 bits
    refused(lib().stt_kv8_cache_bytes(1, 1, 64, 16, None), "NULL")
    refused(lib().stt_kv8_cache_create(0, 1, 1, 64, 16, C.c_void_p(8), C.byref(C.c_void_p())), "16-byte aligned")
    refused(lib().stt_kv8_cache_create(0, 1, 1, 64, 16, None, None), "NULL")
    with pytest.raises(SttError):
        Kv8Cache.bytes(1, 1, 65, 16)


def test_calls_without_a_handle_are_refused():
    L = lib()
    refused(L.stt_kv8_append_device(None, None, None, None, None), "bad arguments")
    refused(L.stt_kv8_read_device(None, None, None, None, None), "bad arguments")
    refused(L.stt_kv8_attention_device(None, None, None, 1, None, 0, 1.0, None, None), "bad arguments")
    refused(L.stt_kv8_reorder_device(None, None, 1, 1, None, None), "bad arguments")
    refused(L.stt_kv8_cache_status(None), "NULL")
    refused(L.stt_kv8_cache_get_info(None, None), "NULL")
    refused(L.stt_beam_select_device(None, None, None), "bad arguments")
    refused(L.stt_beam_reorder_device(0, None, None), "bad arguments")
    refused(L.stt_beam_status(None), "NULL")
    assert L.stt_kv8_cache_destroy(None) == 0 and L.stt_beam_destroy(None) == 0


@pytest.mark.parametrize("args", [(0, 1, 1), (1, 0, 1), (1, 33, 1), (1, 1, 0), (1, 32, 2 ** 27), (2 ** 30, 32, 8000)])
def test_selector_sizes_are_checked(args):
    out = C.c_void_p(1)
    assert lib().stt_beam_create(0, *args, C.byref(out)) == STT_E_INVALID_ARG and not out.value


def test_reorder_layouts_are_checked():
    def call(**k):
        f = dict(states=16, row=64, segment=32, units=4, unit=8, parents=16, held=0, segments=2, groups=1, beams=2, reserved=0)
        return lib().stt_beam_reorder_device(0, BEAM_STATES.pack(*{**f, **k}.values()), None)

    refused(call(states=0), "bad arguments")
    refused(call(parents=0), "bad arguments")
    refused(call(unit=0), "bad arguments")
    refused(call(units=-1), "bad arguments")
    refused(call(beams=0), "beams")
    refused(call(beams=33), "beams")
    refused(call(segment=31), "segments overlap")
    refused(call(row=63), "rows overlap")
    refused(call(row=-64), "overlap")
    refused(call(units=2 ** 40, row=2 ** 60, segment=2 ** 50), "too large")


class FakeTensor:
    def __init__(self, shape, dtype="torch.float32", device=("cuda", 0), stride=None):
        self.shape, self.dtype = tuple(shape), dtype
        self.device = type("D", (), {"type": device[0], "index": device[1], "__str__": lambda s: f"{s.type}:{s.index}"})()
        dense = [int(np.prod(shape[i + 1:])) for i in range(len(shape))]
        self._stride = tuple(stride) if stride else tuple(dense)
        self._dense = list(self._stride) == dense

    def stride(self): return self._stride
    def get_device(self): return -1 if self.device.index is None else self.device.index
    def numel(self): return int(np.prod(self.shape))
    def element_size(self): return 4 if "32" in self.dtype else 2
    def is_contiguous(self): return self._dense
    def data_ptr(self): return 256


def cache():
    c = Kv8Cache.__new__(Kv8Cache)
    c._prepare()
    c._h, c.n_seqs, c.n_kv_heads, c.head_dim, c.capacity, c.device = None, 4, 2, 64, 32, 0
    return c


def test_the_binding_checks_tensors_before_it_calls():
    c, pos = cache(), FakeTensor([3], "torch.int32")
    k = FakeTensor([3, 1, 2, 64])
    for bad, text in [(FakeTensor([3, 1, 2, 32]), "tensors are"), (FakeTensor([3, 2, 64]), "tensors are"),
                      (FakeTensor([3, 1, 1, 64]), "tensors are"), (FakeTensor([3, 1, 2, 64], device=("cpu", None)), "on cpu"),
                      (FakeTensor([3, 1, 2, 64], device=("cuda", 1)), "cuda:1"),
                      (FakeTensor([3, 1, 2, 64], stride=[256, 256, 128, 2]), "contiguous"),
                      (FakeTensor([3, 1, 2, 64], "torch.int8"), "")]:
        with pytest.raises(SttError) as e:
            c.append(bad, k, pos)
        assert text in str(e.value) and e.value.code == STT_E_INVALID_ARG
    with pytest.raises(SttError):
        c.append(k, FakeTensor([3, 1, 2, 64], "torch.bfloat16"), pos)
    for bad in (FakeTensor([2], "torch.int32"), FakeTensor([3], "torch.int64"), FakeTensor([3], "torch.int32", stride=[2]),
                FakeTensor([3], "torch.int32", device=("cpu", None))):
        for name in ("pos", "count", "seqs"):
            with pytest.raises(SttError):
                c.append(k, k, **{**dict(pos=pos), name: bad})
        with pytest.raises(SttError):
            c.attention(k, k, pos, start=bad)
    with pytest.raises(SttError):
        c.attention(k, FakeTensor([3, 1, 4, 64]), pos)
    with pytest.raises(SttError):
        c.reorder(FakeTensor([4], "torch.int32"))
    s = BeamSelector.__new__(BeamSelector)
    s._prepare()
    s._h, s.device = None, 0
    f = lambda d="torch.float32", shape=(2, 3): FakeTensor(shape, d)  # noqa: E731
    good = dict(logits=f(shape=(6, 9)), scores=f(), next_scores=f(), parents=f("torch.int32"), tokens=f("torch.int32"))
    for name, bad in [("logits", f(shape=(5, 9))), ("logits", FakeTensor((6, 9), stride=(18, 2))), ("logits", f("torch.int8", (6, 9))),
                      ("scores", f("torch.float16")), ("scores", f(shape=(6,))), ("parents", f("torch.int64")),
                      ("tokens", f("torch.int32", (2, 2))), ("done", f("torch.bool")), ("next_done", f())]:
        with pytest.raises(SttError):
            s.select(**{**good, name: bad})
    with pytest.raises(SttError):
        beam_reorder(f(shape=(5, 2, 3)), f("torch.int32"))
    with pytest.raises(SttError):
        beam_reorder(f(shape=(6, 2)), f("torch.int32"))
    with pytest.raises(SttError):
        beam_reorder(FakeTensor((6, 2, 3, 4), stride=(24, 12, 5, 1)), f("torch.int32"))


def test_reference_exponents_and_codes():
    assert R.exponent(127.0) == 0 and R.exponent(math.nextafter(127.0, 200)) == 1 and R.exponent(1.0) == -6
    assert R.exponent(63.5) == -1 and R.exponent(0.0) == -100 and R.exponent(1e-40) == -100
    c = R.RefCache(np.zeros((1, 1, 16, 1)), np.zeros((1, 1, 1)))
    c.append(0, 0, np.array([[[1.0]]]))
    assert c.exps[0, 0, 0] == -6 and c.codes[0, 0, 0, 0] == 64
    c.append(0, 1, np.array([[[3.0]]]))           # the block's exponent grows: 64 -> 32
    assert c.exps[0, 0, 0] == -5 and list(c.codes[0, 0, :2, 0]) == [32, 96]
    c.append(0, 2, np.array([[[0.1]]]))           # and stays
    assert list(c.codes[0, 0, :3, 0]) == [32, 96, 3]
    c.append(0, 16, np.array([[[0.5]]]))          # a new lap begins the block anew
    assert c.exps[0, 0, 0] == -7 and c.codes[0, 0, 0, 0] == 64


def test_reference_selection():
    s, p, t, d = R.select(np.log([[[0.5, 0.25, 0.25], [0.8, 0.1, 0.1]]]), np.array([[0.0, -1.0]]))
    assert p.tolist() == [[0, 1]] and t.tolist() == [[0, 0]]
    assert np.allclose(s, [[math.log(0.5), math.log(0.8) - 1]])
    s, p, t, d = R.select(np.zeros((1, 2, 4)), np.array([[0.0, 0.0]]), np.array([[0, 1]]), 2)
    assert p.tolist() == [[1, 0]] and t.tolist() == [[2, 0]] and d.tolist() == [[True, False]]


def test_oracle_int8_rings_are_close_to_f32_ones(tiny_ref_gguf):
    """The oracle's 8-bit rings round K and V by at most a step of 1/64 of a block's largest value: its
    logits stay near, and are not, the f32 rings' (the GPU tests compare with them exactly that way)."""
    from oracle import oracle as O
    om = O.OracleModel(tiny_ref_gguf, num_layers=2, num_heads=2, num_codebooks=4, text_start_token=1000, sliding_window=20)
    a, b = om.stream(0), om.stream(O.KV_INT8)
    rng = np.random.default_rng(0)
    far = 0.0
    for _ in range(40):
        audio, text = rng.integers(0, 300, 4), int(rng.integers(0, 1000))
        x, y = a.forward(audio, text)[0], b.forward(audio, text)[0]
        far = max(far, float(np.abs(x - y).max() / np.abs(x).max()))
    assert 1e-6 < far < 1 / 16


def test_beam_calls_without_a_set_are_refused():
    L = lib()
    refused(L.stt_streams_reorder(None, None, 1, 1, None), "NULL")
    refused(L.stt_streams_beam_frame(None, None, None, 1, 1, None, None, None, None), "NULL")
