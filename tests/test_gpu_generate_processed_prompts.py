"""chpe_generate_processed after prompts that go through the single-token step, the
batched step or both, and with another device current."""
import ctypes as C
import threading
from contextlib import closing

import numpy as np
import pytest

import chpe_qwen_engine_b200 as chpe
from _ops_ref import logits
from _util import archive

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

WORDS = np.array([11, 2222, 33333, 11, 2222, 151000, 7, 11, 2222, 5, 5, 90000, 7, 11, 42, 2222, 11], np.uint32)
RULES = dict(repetition=1.3, frequency=0.25, presence=0.5, bias={500: 1.5, 2222: -2.0})


def engine(device=0):
    return chpe.Engine.from_bytes(archive(chpe.SYNTH_3B_W4), chpe.SYNTH_ARCH[chpe.SYNTH_3B_W4], 64, device=device)


def on_host(e, prompt, n_gen):
    """The rules in f32, one rounding each, on every step's logits."""
    e.forward_tokens(prompt)
    said, ids, vals = [int(t) for t in prompt], np.array([list(RULES["bias"])]), np.float32([list(RULES["bias"].values())])
    for i in range(n_gen):
        if i:
            e.forward_decode(said[-1], len(said) - 1)
        _, t = logits(e.logits()[None], np.array([said]), [len(prompt)], None, np.float32([1.3]), np.float32([0.25]), np.float32([0.5]),
                      ids, vals, kind=np.float32)
        said.append(int(t[0]))
    return said[len(prompt):]


@pytest.mark.parametrize("n", [1, 3, 7, 8, 9, 16, 17])
def test_prompts_of_every_path(n):
    with closing(engine()) as e:
        first = e.generate_processed(WORDS[:n], 10, **RULES).tolist()  # the engine's first call
        assert first == on_host(e, WORDS[:n], 10)
        assert e.generate_processed(WORDS[:n], 10, **RULES).tolist() == first
        assert np.array_equal(e.generate_processed(WORDS[:n], 10), e.generate(WORDS[:n], 10))


def test_called_from_another_thread():
    with closing(engine()) as e:
        want = e.generate_processed(WORDS[:3], 6, **RULES).tolist()
        got = []
        t = threading.Thread(target=lambda: got.extend(e.generate_processed(WORDS[:3], 6, **RULES).tolist()))
        t.start()
        t.join()
        assert got == want


@pytest.mark.skipif(torch is None or torch.cuda.device_count() < 2, reason="needs two GPUs")
@pytest.mark.parametrize("device", [0, 1])
def test_with_another_device_current(device):
    """Prompts below 8 tokens do not pass the batched step, which makes the engine's device current."""
    with closing(engine(device)) as e:
        want = e.generate_processed(WORDS[:3], 6, **RULES).tolist()
        with torch.cuda.device(1 - device):
            torch.zeros(1, device=f"cuda:{1 - device}")
            assert e.generate_processed(WORDS[:3], 6, **RULES).tolist() == want
            assert torch.cuda.current_device() == 1 - device


@pytest.mark.parametrize("n_gen", [-1, -3, 2 ** 64 - 3, 2 ** 63, 62])
def test_lengths_whose_sum_wraps_are_refused(n_gen):
    """A negative number of tokens arrives as a size_t near 2^64."""
    u32 = lambda a: a.ctypes.data_as(C.POINTER(C.c_uint32))  # noqa: E731
    out = np.full(64, 7, np.uint32)
    with closing(engine()) as e:
        e.generate(WORDS[:3], 2)
        n, L = C.c_size_t(n_gen), chpe.lib()
        assert L.chpe_generate_processed(e.ctx, u32(WORDS), 3, n, 1.0, 0.0, 0.0, None, None, 0, None, u32(out)) == -1
        assert L.chpe_generate(e.ctx, u32(WORDS), 3, n, u32(out)) == -1
        assert L.chpe_speculative_generate(e.ctx, u32(WORDS), 3, n, 4, 3, u32(out), None) == -1
        assert "max_seq_len" in L.chpe_last_error(e.ctx).decode()
        assert L.chpe_speculative_generate(e.ctx, u32(WORDS), 3, 4, 2 ** 32 - 1, 3, u32(out), None) == -1
        assert L.chpe_bench_greedy(e.ctx, n, C.byref(C.c_float())) == -1
        assert (out == 7).all()
        assert e.generate_processed(WORDS[:3], 61).size == 61  # to the last position


def test_the_last_result_is_of_the_chosen_token():
    with closing(engine()) as e:
        for n in (3, 8):  # the last prompt token by the single-token step, by the batched one
            for n_gen in (1, 2, 7):
                got = e.generate_processed(WORDS[:n], n_gen, **RULES)
                r = e.last_result()
                assert r.argmax_token == got[-1] and r.max_logit == e.logits()[got[-1]]
            mask = np.zeros((e.vocab + 31) // 32, np.uint32)
            mask[777 // 32] = 1 << (777 % 32)
            e.generate_processed(WORDS[:n], 3, mask=mask)
            r, x = e.last_result(), e.logits()
            assert r.argmax_token == 777 and r.max_logit == x[777] < x.max()
            e.generate_processed(WORDS[:n], 3)
            assert e.last_result().max_logit == e.logits().max()
