"""Greedy generation under sampling rules (chpe_generate_processed): without a
rule it is chpe_generate; with penalties, biases and a mask every token equals
the one that the same rules, applied on the host to the logits of the same
steps, choose; a mask that leaves nothing is an error and the context stays
usable."""
import ctypes as C

import numpy as np
import pytest

import chpe_qwen_engine_b200 as chpe
from _ops_ref import logits
from _util import archive

pytestmark = pytest.mark.gpu

PROMPT = np.array([11, 2222, 33333, 11, 2222, 151000, 7, 11, 2222], np.uint32)


@pytest.fixture(scope="module", params=[chpe.SYNTH_3B_W4, chpe.SYNTH_3B_FP16_RAW])
def eng(request):
    e = chpe.Engine.from_bytes(archive(request.param), chpe.SYNTH_ARCH[request.param], 128)
    yield e
    e.close()


def on_host(e, n_gen, rep, freq, pres, bias, mask):
    """The same rules in f32, one rounding each, on every step's logits."""
    e.forward_tokens(PROMPT)
    said = [int(t) for t in PROMPT]
    out = []
    for i in range(n_gen):
        if i:
            e.forward_decode(out[-1], len(said) - 1)
        ids = np.array([list(bias)], np.int64) if bias else None
        vals = np.array([list(bias.values())], np.float32) if bias else None
        _, t = logits(e.logits()[None], np.array([said]), [PROMPT.size], None, np.float32([rep]), np.float32([freq]),
                      np.float32([pres]), ids, vals, None if mask is None else mask.view(np.int32)[None], kind=np.float32)
        out.append(int(t[0]))
        said.append(out[-1])
    return out


def test_without_rules_it_is_greedy_generation(eng):
    assert np.array_equal(eng.generate_processed(PROMPT, 20), eng.generate(PROMPT, 20))
    assert eng.position() == PROMPT.size + 19
    assert eng.generate_processed(PROMPT, 0).size == 0


@pytest.mark.parametrize("rep, freq, pres, biased, masked", [
    (1.3, 0.0, 0.0, False, False), (1.0, 0.4, 0.3, False, False), (1.2, 0.2, -0.1, True, False), (0.8, 0.0, 0.5, True, True)])
def test_rules_choose_what_they_choose_on_the_host(eng, rep, freq, pres, biased, masked):
    rng = np.random.default_rng(3)
    plain = eng.generate(PROMPT, 4)
    bias = {int(plain[0]): -3.0, 500: 1.5, 151935: 0.5, 7: -100.0} if biased else None
    mask = rng.integers(0, 2 ** 32, (eng.vocab + 31) // 32, dtype=np.uint64).astype(np.uint32) if masked else None
    got = eng.generate_processed(PROMPT, 24, rep, freq, pres, bias, mask)
    assert got.tolist() == on_host(eng, 24, rep, freq, pres, bias, mask)
    if masked:
        assert all(mask[t // 32] >> (t % 32) & 1 for t in got)


def test_a_mask_of_one_token_and_of_none(eng):
    mask = np.zeros((eng.vocab + 31) // 32, np.uint32)
    with pytest.raises(chpe.ChpeError, match="no token is allowed at generated token 0"):
        eng.generate_processed(PROMPT, 3, mask=mask)
    mask[777 // 32] = 1 << (777 % 32)
    assert eng.generate_processed(PROMPT, 5, repetition=2.0, mask=mask).tolist() == [777] * 5
    assert eng.last_result().argmax_token == 777
    assert np.array_equal(eng.generate_processed(PROMPT, 6), eng.generate(PROMPT, 6))


def test_refusals(eng):
    for kw in (dict(repetition=0.0), dict(repetition=float("nan")), dict(frequency=float("inf")), dict(presence=float("nan"))):
        with pytest.raises(chpe.ChpeError, match="penalties"):
            eng.generate_processed(PROMPT, 2, **kw)
    with pytest.raises(chpe.ChpeError, match="max_seq_len"):
        eng.generate_processed(PROMPT, 120)
    with pytest.raises(ValueError, match="mask"):
        eng.generate_processed(PROMPT, 2, mask=np.zeros(3, np.uint32))
    out = np.zeros(2, np.uint32).ctypes.data_as(C.POINTER(C.c_uint32))
    f = chpe.lib().chpe_generate_processed
    p = PROMPT.ctypes.data_as(C.POINTER(C.c_uint32))
    assert f(None, p, 3, 2, 1.0, 0.0, 0.0, None, None, 0, None, out) == -1
    assert f(eng.ctx, p, 0, 2, 1.0, 0.0, 0.0, None, None, 0, None, out) == -1
    assert f(eng.ctx, p, 3, 2, 1.0, 0.0, 0.0, None, None, 1, None, out) == -1
