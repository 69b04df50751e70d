"""The talker over its 8-bit cache rounds keys and values, and nothing else that its 16-bit cache does not round.

Yardstick: the oracle holding the same codes, and the same oracle with queries and attention probabilities rounded to bf16 (what one
product of bf16 numbers each would do).  The GPU's logits have to lie within half of that distance, root mean square, from the
oracle that does not round them: queries and probabilities in bf16 alone are about the whole of it away.

What is left without them are f32 sums and inputs that carry 16 bits, so that keys and values differ by about 2^-17 before they are held
and some codes come out one step apart.  int8: a fraction 2^-17 * 127 = 2^-10 of the codes at most, each by 2^-7 of the block's
largest element, root mean square 2^-12 of it; rounding costs 2^-10 relative each for queries and probabilities, 2^-11 of the largest.
e4m3: a fraction 2^-17 / 2^-3.5 = 2^-13.5 of the codes, each by 2^-3.5 of its value.  A short prompt of T0 or M0 has few such codes among
many elements.  Over hundreds of keys the two come to the same: one V code of one of n keys moves one of the 256 output channels by
2^-3.5 v / n, a root mean square of 2^-7.5 v / n over them, and rounding all probabilities moves each by 2^-10 v / sqrt(n); for n = 20 keys
in view that is 2^-11.8 v from a single code against 2^-12.2 v, and 600 keys have 2^18 codes, 2^4.7 of them a step apart:
2^(-7.5 - 9.2 + 2.3) = 2^-14.4 v against 2^-14.6 v.  There the yardstick says nothing, and e4m3 is held to the bar of bf16 runs alone.

Every case compares the prompt's logits (tiles of 128 rows) and at least one decode step's (tiles of 16 rows, parts of the key range
joined), whose inputs are the same on both sides because all codes before it are."""
import ctypes as C

import numpy as np
import pytest

from conftest import SEED, make_oracle
from golden.make_golden import GREEDY
from test_gpu_generate import BF16_LOGIT_TOL, _req, _sampling
from test_gpu_kv_generate import TOP, _icl_request

pytestmark = pytest.mark.gpu
QUERIES, PROBABILITIES = 16, 32  # bits of the oracle's rounding probe
FRAMES = 6


def _same_inputs(a, b):
    """Frames whose inputs are the same for both code sequences: those with equal codes and the one behind them."""
    n = 0
    while n < FRAMES and np.array_equal(a[n], b[n]):
        n += 1
    return min(FRAMES, n + 1)


def _rms(xs):
    return float(np.sqrt(np.mean(np.concatenate([x.ravel() for x in xs]).astype(np.float64) ** 2)))


def _check(bind, m, fmt, runs, yardstick=True):
    """runs: (request, oracle call) pairs."""
    lib = bind.lib(False)
    far, near = {"prompt": [], "decode": []}, {"prompt": [], "decode": []}
    for req, oracle in runs:
        try:
            lib.orc_set_kv_hold(C.c_float(TOP[fmt]))
            exact = oracle()
            lib.orc_set_round_probe(QUERIES | PROBABILITIES)
            rounded = oracle()
        finally:
            lib.orc_set_kv_hold(C.c_float(0.0))
            lib.orc_set_round_probe(0)
        out = m.generate([req], _sampling(GREEDY), FRAMES, trace=True)
        n = min(_same_inputs(exact["codes"], out.codes[0]), _same_inputs(exact["codes"], rounded["codes"]))
        assert n >= 2, "no decode step to compare"
        assert np.abs(out.logits[0, :n] - exact["logits"][:n]).max() <= BF16_LOGIT_TOL
        for part, s in (("prompt", slice(0, 1)), ("decode", slice(1, n))):
            near[part].append(out.logits[0, s] - exact["logits"][s])
            far[part].append(rounded["logits"][s] - exact["logits"][s])
    if yardstick:
        for part in near:
            assert _rms(near[part]) <= 0.5 * _rms(far[part]), part


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("shape", ["T0", "M0"])
def test_texts(bind, shape, fmt):
    from qwen3_tts_rs_amd import synth, synthetic_model
    m, cfg, _, tmpl = synthetic_model(shape, dtype="bf16", codec=False, round_to_bf16=True, kv_cache=fmt)
    o, _, _, _ = make_oracle(bind, shape, "bf16", talker=True, codec=False)
    try:
        runs = []
        for n, seed in ((14, 3), (60, 4), (31, 5)):
            text = synth.synthetic_text_ids(tmpl, n, seed)
            runs.append((_req(text), lambda text=text: o.generate(
                text, bind.resolve_codec_prefill(cfg, "english", "speaker1"), GREEDY, FRAMES,
                speaker_token=bind.resolve_speaker_token(cfg, "speaker1"), trace=True)))
        _check(bind, m, fmt, runs)
    finally:
        m.close()


@pytest.mark.parametrize("frames,window", [(600, 0), (90, 20)])
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_reference_codes_in_the_prompt(bind, golden, fmt, frames, window):
    """Decode steps over several parts of the key range, and with a sliding window."""
    from qwen3_tts_rs_amd import LoaderConfig, Model, round_bf16, synth
    cfg, _, _ = synth.shape_set("T0")
    if window:
        cfg["talker_config"]["sliding_window"] = window
    m = Model(cfg, None, LoaderConfig(dtype="bf16", kv_cache=fmt))
    m.load_weights((k, round_bf16(a)) for k, a in synth.iter_weights(synth.talker_keys(cfg), SEED))
    m.finalize()
    o, _, _, _ = make_oracle(bind, "T0", "bf16", talker=True, codec=False)
    o.set_model_config(cfg)
    try:
        ref = np.resize(golden["ref_codes"], (frames, golden["ref_codes"].shape[1]))
        _check(bind, m, fmt, [(_icl_request(golden, ref), lambda: o.generate(
            golden["text_ids"], bind.resolve_codec_prefill(cfg, "english", None), GREEDY, FRAMES, speaker_embed=golden["xvector"],
            ref_text_ids=golden["ref_text_ids"], ref_codes=ref, non_streaming=False, trace=True))], yardstick=fmt == "int8")
    finally:
        m.close()


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_many_heads_on_one_kv_head(bind, fmt):
    """20 query heads share a kv head: a decode step's rows fill more than one tile of 16."""
    from qwen3_tts_rs_amd import LoaderConfig, Model, round_bf16, synth
    cfg, _, tmpl = synth.shape_set("T0")
    cfg["talker_config"].update(num_attention_heads=20, num_key_value_heads=1)
    m = Model(cfg, None, LoaderConfig(dtype="bf16", kv_cache=fmt))
    o = bind.Oracle(fast=False)
    for k, a in synth.iter_weights(synth.talker_keys(cfg), SEED):
        a = round_bf16(a)
        m.load_tensor(k, a)
        o.load_tensor(k, a)
    m.finalize()
    o.set_model_config(cfg)
    try:
        text = synth.synthetic_text_ids(tmpl, 40, 3)
        _check(bind, m, fmt, [(_req(text), lambda: o.generate(text, bind.resolve_codec_prefill(cfg, "english", "speaker1"), GREEDY, FRAMES,
                                                              speaker_token=bind.resolve_speaker_token(cfg, "speaker1"), trace=True))],
               yardstick=fmt == "int8")
    finally:
        m.close()


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_prompts_of_more_than_one_pass(golden, fmt):
    """Eight prompts of 5000 tokens in all, one of which is cut between two prefill passes: which one depends on the order of the
    requests, the logits and codes do not."""
    from qwen3_tts_rs_amd import SamplingConfig, synthetic_model
    m, _, _, _ = synthetic_model("T0", dtype="bf16", codec=False, kv_cache=fmt)
    try:
        reqs = [_icl_request(golden, np.resize(np.roll(golden["ref_codes"], i, 0), (500 + 37 * i, golden["ref_codes"].shape[1]))) for i in range(8)]
        a = m.generate(reqs, SamplingConfig.cli_greedy(), 4, trace=True)
        b = m.generate(reqs[::-1], SamplingConfig.cli_greedy(), 4, trace=True)
        assert np.array_equal(a.logits, b.logits[::-1]) and np.array_equal(a.codes, b.codes[::-1])
    finally:
        m.close()
