"""What stt_streams_beam_frame reports, and what the streams and outputs are then: a host that is told of an
error must still know which stream carries what."""
import numpy as np
import pytest

import stt_b200
from gguf_tools import read_gguf
from stt_b200 import BeamSelector, SttError
from stt_b200._lib import I32P, F32P, U32P, STT_E_DEVICE_FLAG, STT_E_INVALID_ARG, lib
from stt_b200.model import SttConfig

pytestmark = pytest.mark.gpu

NAN = 0x7E00  # an f16 scale


def model_with(change=None):
    spec = stt_b200.SynthSpec(seed=21, num_layers=2, hidden_size=256, num_heads=2, ffn_hidden=512, vocab_size=40,
                              text_in_vocab_size=41, num_codebooks=4, audio_vocab_size=300, weight_std=0.1)
    g = stt_b200.synth_gguf(spec)
    buf = np.array(g.array)
    _, tensors, data = read_gguf(buf.tobytes())
    if change:
        name, row = change
        t = tensors[name]
        at = data + t["offset"] + row * (256 // 32 * 18)  # the row's first block: its scale
        buf[at:at + 2] = np.frombuffer(np.uint16(NAN).tobytes(), np.uint8)
    cfg = SttConfig(num_layers=2, hidden_size=256, num_heads=2, num_kv_heads=2, num_codebooks=4, vocab_size=40,
                    text_in_vocab_size=41, audio_vocab_size=300, text_start_token=40, sliding_window=20)
    return stt_b200.SttModel.from_shards([buf], config=cfg)


def frame(cache, sel, ids, audio, scores):
    """The C call with outputs of the caller's own: (status, text, scores, parents, tokens)."""
    ids, audio = np.ascontiguousarray(ids, np.int32), np.ascontiguousarray(audio, np.uint32)
    sc = np.array(scores, np.float32)
    par, tok = np.full(ids.shape, 77, np.int32), np.full(ids.shape, 78, np.int32)
    rc = lib().stt_streams_beam_frame(cache._h, sel._h, ids.ctypes.data_as(I32P), *ids.shape, audio.ctypes.data_as(U32P),
                                      sc.ctypes.data_as(F32P), par.ctypes.data_as(I32P), tok.ctypes.data_as(I32P))
    return rc, lib().stt_last_error().decode(), sc, par, tok


def states(cache, n):
    return [{k: cache.state(i)[k] for k in ("offset", "frame_count", "last_text_token")} for i in range(n)]


IDS = [[3, 0, 4], [1, 5, 2]]
START = [[0.0, -np.inf, -np.inf]] * 2


@pytest.mark.parametrize("kv", ["bf16", "int8"])
def test_nan_logits_are_reported_by_the_frame_that_met_them(kv):
    """A NaN scale in the head's row 7: every beam's logits hold a NaN.  The frame is done, with -inf scores."""
    cache = model_with(("text_linear.weight", 7)).create_cache(6, kv)
    sel = BeamSelector(2, 3, 40)
    audio = np.random.default_rng(1).integers(0, 300, (2, 4))
    rc, text, sc, par, tok = frame(cache, sel, IDS, audio, START)
    assert rc == STT_E_DEVICE_FLAG and "NaN" in text, (rc, text)
    assert (sc == -np.inf).all() and par.tolist() == [[0, 0, 0]] * 2 and tok.tolist() == [[0, 1, 2]] * 2
    for ids, t in zip(IDS, tok):
        for b, i in enumerate(ids):
            st = cache.state(i)
            assert (st["offset"], st["frame_count"], st["last_text_token"]) == (1, 1, t[b])
    sel.status()  # reported once, by the frame
    with pytest.raises(SttError) as e:
        cache.beam_frame(sel, IDS, audio, sc)
    assert e.value.code == STT_E_DEVICE_FLAG
    assert (e.value.frame[0] == -np.inf).all() and e.value.frame[2].tolist() == [[0, 1, 2]] * 2


def test_an_error_of_the_step_leaves_the_streams_in_their_order():
    """A NaN scale in layer 1's K rows: the 8-bit rings report what they were given.  Nothing is chosen or moved."""
    cache = model_with(("transformer.layers.1.self_attn.in_proj_weight", 256 + 3)).create_cache(6, "int8")
    sel = BeamSelector(2, 3, 40)
    audio = np.random.default_rng(2).integers(0, 300, (2, 4))
    for i in range(6):
        assert lib().stt_stream_set_last_text_token(cache._h, i, 10 + i) == 0
    rc, text, sc, par, tok = frame(cache, sel, IDS, audio, START)
    assert rc == STT_E_DEVICE_FLAG, (rc, text)
    assert np.array_equal(sc, np.float32(START)) and (par == 77).all() and (tok == 78).all()
    assert states(cache, 6) == [dict(offset=1, frame_count=0, last_text_token=10 + i) for i in range(6)]
    with pytest.raises(SttError) as e:
        cache.beam_frame(sel, IDS, audio, START)
    assert e.value.frame[1].tolist() == [[0, 1, 2]] * 2 and (e.value.frame[2] == -1).all()
    assert states(cache, 6) == [dict(offset=2, frame_count=0, last_text_token=10 + i) for i in range(6)]


def test_what_an_earlier_selection_left_does_not_fail_a_frame():
    import torch
    cache = model_with().create_cache(6, "bf16")
    sel = BeamSelector(2, 3, 40)
    bad = torch.full((3, 40), float("nan"), device="cuda")
    s, i = torch.zeros(1, 3, device="cuda"), [torch.zeros(1, 3, dtype=torch.int32, device="cuda") for _ in range(2)]
    sel.select(bad, s, s.clone(), i[0], i[1])
    torch.cuda.synchronize()
    rc, text, sc, par, tok = frame(cache, sel, IDS, np.zeros((2, 4)), START)
    assert rc == 0, text
    assert np.isfinite(sc).all()
    with pytest.raises(SttError) as e:
        sel.status()  # the selection's own
    assert e.value.code == STT_E_DEVICE_FLAG


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_scores_that_are_no_scores_are_refused_before_the_frame(value):
    cache = model_with().create_cache(6, "bf16")
    sel = BeamSelector(2, 3, 40)
    scores = np.zeros((2, 3), np.float32)
    scores[1, 2] = value
    rc, text, sc, par, tok = frame(cache, sel, IDS, np.zeros((2, 4)), scores)
    assert rc == STT_E_INVALID_ARG and "score" in text
    assert (par == 77).all() and (tok == 78).all()
    assert [s["offset"] for s in states(cache, 6)] == [0] * 6
    sel.status()
