"""The talker's key/value cache in 8 bits (LoaderConfig.kv_cache, qtts_model_set_kv_cache) through generate.

The oracle holds its keys and values in the same format.  The bar is that of bf16 runs (logits within 2e-2 max-abs): keys and
values of the two sides differ by about 2^-16 relative before they are held, so about 2^-12 of the codes (steps of 2^-4) come out one
step apart, which adds less than rounding every key and value to bf16 does in the runs that the bar was set for."""
import ctypes as C

import numpy as np
import pytest

from conftest import make_oracle
from golden.make_golden import GREEDY
from test_gpu_continuous import _model, _requests
from test_gpu_generate import BF16_LOGIT_TOL, _req, _sampling

pytestmark = pytest.mark.gpu
TOP = {"e4m3": 448.0, "int8": 127.0}


@pytest.fixture
def hold(bind):
    def set_top(top):
        for fast in (False, True):
            bind.lib(fast).orc_set_kv_hold(C.c_float(top))
    yield set_top
    set_top(0.0)


def _icl_request(golden, ref):
    from qwen3_tts_rs_amd import GenerationRequest
    return GenerationRequest(text_ids=golden["text_ids"], language="english", speaker_embed=golden["xvector"], ref_codes=ref,
                             ref_text_ids=golden["ref_text_ids"], non_streaming_mode=False)


def _compare(out, r, frames):
    agree = 0
    while agree < frames and np.array_equal(r["codes"][agree], out.codes[0, agree]):
        agree += 1
    n = min(frames, agree + 1)  # the first diverging frame still has identical inputs to the talker
    assert np.abs(r["logits"][:n] - out.logits[0, :n]).max() <= BF16_LOGIT_TOL


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("shape", ["T0", "M0"])
def test_logits_match_an_oracle_that_holds_the_same(bind, hold, shape, fmt):
    from qwen3_tts_rs_amd import synth, synthetic_model
    m, cfg, _, tmpl = synthetic_model(shape, dtype="bf16", codec=False, round_to_bf16=True, kv_cache=fmt)
    o, _, _, _ = make_oracle(bind, shape, "bf16", talker=True, codec=False)
    try:
        text = synth.synthetic_text_ids(tmpl, 14, 3)
        hold(TOP[fmt])
        r = o.generate(text, bind.resolve_codec_prefill(cfg, "english", "speaker1"), GREEDY, 8,
                       speaker_token=bind.resolve_speaker_token(cfg, "speaker1"), trace=True)
        out = m.generate([_req(text)], _sampling(GREEDY), 8, trace=True)
        _compare(out, r, 8)
        m.set_kv_cache(None)  # and back: another cache, other logits
        plain = m.generate([_req(text)], _sampling(GREEDY), 8, trace=True)
        assert not np.array_equal(plain.logits, out.logits)
        m.set_kv_cache(fmt)
        again = m.generate([_req(text)], _sampling(GREEDY), 8, trace=True)
        assert np.array_equal(again.logits, out.logits)
    finally:
        m.close()


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_contexts_of_several_parts(bind, hold, golden, fmt):
    """A reference of 600 frames in the prompt: the decode steps join parts of the key range, the prompt spans many tiles; a short
    utterance shares the batch."""
    from qwen3_tts_rs_amd import synthetic_model
    m, cfg, _, _ = synthetic_model("T0", dtype="bf16", codec=False, round_to_bf16=True, kv_cache=fmt)
    o, _, _, _ = make_oracle(bind, "T0", "bf16", talker=True, codec=False)
    try:
        ref = np.resize(golden["ref_codes"], (600, golden["ref_codes"].shape[1]))
        req = _icl_request(golden, ref)
        out = m.generate([req, _req(golden["text_ids"])], _sampling(GREEDY), 6, trace=True)
        hold(TOP[fmt])
        r = o.generate(golden["text_ids"], bind.resolve_codec_prefill(cfg, "english", None), GREEDY, 6, speaker_embed=golden["xvector"],
                       ref_text_ids=golden["ref_text_ids"], ref_codes=ref, non_streaming=False, trace=True)
        _compare(out, r, 6)
    finally:
        m.close()


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_sliding_window(bind, hold, golden, fmt):
    """A talker with a window of 20 keys: prompt rows and decode steps beyond it."""
    from conftest import SEED
    from qwen3_tts_rs_amd import LoaderConfig, Model, round_bf16, synth
    cfg, _, tmpl = synth.shape_set("T0")
    cfg["talker_config"]["sliding_window"] = 20
    m = Model(cfg, None, LoaderConfig(dtype="bf16", kv_cache=fmt))
    m.load_weights((k, round_bf16(a)) for k, a in synth.iter_weights(synth.talker_keys(cfg), SEED))
    m.finalize()
    o, _, _, _ = make_oracle(bind, "T0", "bf16", talker=True, codec=False)
    o.set_model_config(cfg)
    try:
        ref = np.resize(golden["ref_codes"], (90, golden["ref_codes"].shape[1]))
        req = _icl_request(golden, ref)
        out = m.generate([req], _sampling(GREEDY), 8, trace=True)
        hold(TOP[fmt])
        r = o.generate(golden["text_ids"], bind.resolve_codec_prefill(cfg, "english", None), GREEDY, 8, speaker_embed=golden["xvector"],
                       ref_text_ids=golden["ref_text_ids"], ref_codes=ref, non_streaming=False, trace=True)
        _compare(out, r, 8)
    finally:
        m.close()


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_schedules_agree(fmt):
    """Graph and eager frames, a session, and continuous batching against the plain batch of as many rows: the same codes bit for
    bit (a row's attention does not depend on what shares its launch)."""
    from qwen3_tts_rs_amd import SamplingConfig
    m, tmpl = _model("bf16")
    try:
        m.set_kv_cache(fmt)
        reqs = _requests(tmpl, 12)
        sampling = SamplingConfig(temperature=1.0, top_k=0)
        plain = [m.generate(reqs[4 * i:4 * i + 4], sampling, 40) for i in range(3)]
        eager = m.generate(reqs[:4], sampling, 40, use_graph=False)
        assert np.array_equal(plain[0].codes, eager.codes)
        ses = m.open_session()
        try:
            assert np.array_equal(ses.generate(reqs[:4], sampling, 40).codes, plain[0].codes)
        finally:
            ses.close()
        out = m.generate(reqs, sampling, 40, slots=4)
        for u in range(12):
            n = out.steps_per_utterance[u]
            assert np.array_equal(out.codes[u, :n], plain[u // 4].codes[u % 4, :n]), u
    finally:
        m.close()


def test_refusals():
    from qwen3_tts_rs_amd import QttsError, synthetic_model
    with pytest.raises(QttsError, match="bf16 model"):
        synthetic_model("T0", dtype="f32", codec=False, talker=False, kv_cache="int8")
    m, _, _, _ = synthetic_model("T0", dtype="bf16", codec=False)
    try:
        with pytest.raises(QttsError, match="Unknown"):
            m.set_kv_cache("fp4")
        assert m.lib.qtts_model_set_kv_cache(m._m, 7) == -1 and m.lib.qtts_model_set_kv_cache(None, 1) == -1
    finally:
        m.close()
