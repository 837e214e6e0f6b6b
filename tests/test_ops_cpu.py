"""The batched decode operators' host side, without a GPU: what the entry points
refuse (each with its message), what needs no launch, and the 64-bit
definitions the GPU tests compare with, against differently written ones."""
import ctypes as C

import numpy as np
import pytest

import chpe_qwen_engine_b200 as chpe
from _ops_ref import attention, logits, norm_rope

F32, F16, BF16 = 0, 1, 2
HOST = np.zeros(1 << 16, np.float32)
P = (HOST.ctypes.data + 63) & ~63  # an aligned host address: refused as a device buffer


def err():
    return chpe.lib().chpe_last_error(None).decode()


def qk(**kw):
    freq = np.ones(64)
    a = dict(q=P, k=P, v=P, dtype=F16, qs=1024, ks=256, vs=256, T=2, H=8, KV=2, D=128, qw=None, kw=None, off=0.0,
             eps=1e-6, pos=P, freq=freq.ctypes.data, rope=128, qo=P, qos=1024, ko=None, kos=0, kc=P, vc=P, ct=F16,
             rows=64, slots=P, stream=None)
    a.update(kw)
    return chpe.lib().chpe_qk_norm_rope(*a.values())


@pytest.mark.parametrize("change, said", [
    (dict(dtype=7), "dtype"), (dict(D=96), "head_dim"), (dict(H=0), "num_heads"), (dict(KV=0), "num_kv_heads"),
    (dict(rope=8), "rope_dim"), (dict(rope=144), "rope_dim"), (dict(vc=None), "go together"),
    (dict(kc=None, vc=None), "k_out"), (dict(ct=F32), "FP16 or BF16"), (dict(ct=BF16), "type"),
    (dict(qs=1000), "q_stride"), (dict(ks=260), "k_stride"), (dict(vs=128), "v_stride"), (dict(qos=8), "q_out_stride"),
    (dict(ko=P, kos=4), "k_out_stride"), (dict(qs=2 ** 62), "q_stride"), (dict(freq=None), "inv_freq"),
    (dict(rows=2 ** 63), "cache_rows"), (dict(q=None), "q is NULL"), (dict(q=P + 8), "aligned"), (dict(), "q"),
])
def test_qk_refusals(change, said):
    assert qk(**change) == -1
    assert err().startswith("chpe_qk_norm_rope: ") and said in err()


@pytest.mark.parametrize("bad", [np.nan, np.inf, -17.0, 1e9])
def test_qk_refuses_frequencies(bad):
    f = np.ones(64)
    f[63] = bad
    assert qk(freq=f.ctypes.data) == -1 and "inv_freq[63]" in err()


def paged(**kw):
    ws = chpe.lib().chpe_attention_decode_paged_workspace(128)
    a = dict(q=P, dtype=F16, qs=1024, kc=P, vc=P, ct=F16, pages=4, page=64, table=P, ts=2, mp=2, lens=P, B=2, H=8, KV=2,
             D=128, scale=0.1, out=P, os=1024, lse=None, ws=P, wb=ws, stream=None)
    a.update(kw)
    return chpe.lib().chpe_attention_decode_paged(*a.values())


@pytest.mark.parametrize("change, rc, said", [
    (dict(dtype=3), -1, "dtype"), (dict(ct=F32), -1, "FP16 or BF16"), (dict(ct=BF16), -1, "type"),
    (dict(D=192), -1, "head_dim"), (dict(H=9), -1, "multiple"), (dict(KV=0), -1, "multiple"), (dict(H=0), -1, "multiple"),
    (dict(page=8), -1, "page_size"), (dict(page=48), -1, "page_size"), (dict(page=131072), -1, "page_size"),
    (dict(B=70000), -1, "batch"), (dict(ts=1), -1, "table_stride"), (dict(ts=-1), -1, "table_stride"),
    (dict(scale=float("nan")), -1, "scale"), (dict(qs=512), -1, "q_stride"), (dict(os=1), -1, "out_stride"),
    (dict(wb=1000), -2, "workspace"), (dict(q=None), -1, "q is NULL"), (dict(), -1, "q"),
])
def test_paged_refusals(change, rc, said):
    assert paged(**change) == rc
    assert err().startswith("chpe_attention_decode_paged: ") and said in err()


def test_paged_workspace_sizes():
    f = chpe.lib().chpe_attention_decode_paged_workspace
    assert [f(d) > 0 for d in (64, 128, 256)] == [True] * 3
    assert f(0) == f(96) == f(512) == 0


def rules(**kw):
    a = dict(x=P, dtype=F32, ls=1000, B=2, V=1000, hist=P, hs=8, hl=8, pl=None, tl=None, rep=P, freq=None, pres=None,
             ids=P, vals=P, bs=4, nb=4, mask=P, ms=32, out=P, os=1000, am=P, stream=None)
    a.update(kw)
    return chpe.lib().chpe_logits_process(*a.values())


@pytest.mark.parametrize("change, said", [
    (dict(dtype=-1), "dtype"), (dict(V=0), "vocab"), (dict(V=2 ** 31), "vocab"), (dict(B=2 ** 25), "batch"),
    (dict(out=None, am=None), "neither"), (dict(hist=None), "without a history"), (dict(vals=None), "go together"),
    (dict(nb=65536, bs=65536), "65535"), (dict(ls=999), "logits_stride"), (dict(os=999), "out_stride"),
    (dict(hs=7), "history_stride"), (dict(bs=3), "bias_stride"), (dict(ms=31), "mask_stride"), (dict(ms=-32), "mask_stride"),
    (dict(x=None), "logits is NULL"), (dict(x=P + 2), "aligned"), (dict(), "logits"),
])
def test_logits_refusals(change, said):
    assert rules(**change) == -1
    assert err().startswith("chpe_logits_process: ") and said in err()


def test_nothing_to_do_needs_no_gpu():
    assert qk(T=0) == 0 and paged(B=0) == 0 and rules(B=0) == 0
    assert err() == ""


def test_torch_layer_refuses_host_tensors():
    torch = pytest.importorskip("torch")
    from chpe_qwen_engine_b200 import ops
    with pytest.raises(ValueError, match="CUDA"):
        ops.logits_process(torch.zeros(2, 8))
    with pytest.raises(ValueError, match="CUDA"):
        ops.attention_decode_paged(torch.zeros(1, 2, 64), None, None, None, None)
    with pytest.raises(ValueError, match="CUDA"):
        ops.qk_norm_rope(torch.zeros(1, 2, 64), None, None, None, None)
    with pytest.raises(ValueError, match="head_dim"):
        ops.attention_workspace(96)
    f = ops.rope_inv_freq(1e6, 128)
    assert f.dtype == np.float64 and f.shape == (64,) and f[0] == 1.0 and abs(f[32] - 1e-3) < 1e-18


# ---- the definitions themselves ------------------------------------------------
def test_definition_of_the_rotation():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((3, 2, 64))
    pos = np.array([0, 5, 100003])
    f = 1e4 ** (-np.arange(0, 32, 2) / 32)
    y, _ = norm_rope(x, None, 0, 0, pos, f)
    assert np.array_equal(y[0], x[0]) and np.array_equal(y[..., 32:], x[..., 32:])
    z = (x[..., :16] + 1j * x[..., 16:32]) * np.exp(1j * pos[:, None, None] * f)
    assert np.allclose(y[..., :16], z.real, atol=1e-9) and np.allclose(y[..., 16:32], z.imag, atol=1e-9)
    n, _ = norm_rope(3 * x, np.ones(64), 1.0, 0.0, pos, None)
    assert np.allclose((n ** 2).mean(-1), 4)


def test_definition_of_the_attention():
    rng = np.random.default_rng(2)
    kc, vc = rng.standard_normal((2, 5, 16, 2, 64))
    q = rng.standard_normal((3, 4, 64))
    table = np.array([[3, 1], [4, -1], [0, 0]])
    lens = np.array([20, 32, 0])
    vc[1, 4:] = np.nan  # behind the first sequence
    out, lse, bo, bl = attention(q, kc, vc, table, lens, 0.125, 16, "f32", "f16")
    k = np.concatenate((kc[3], kc[1][:4]))[:, 1]
    v = np.concatenate((vc[3], vc[1][:4]))[:, 1]
    e = np.exp(k @ q[0, 3] * 0.125)
    assert np.allclose(out[0, 3], e @ v / e.sum()) and np.isclose(lse[0, 3], np.log(e.sum()))
    e = np.exp(kc[4][:, 0] @ q[1, 0] * 0.125)  # the second page is not there
    assert np.isclose(lse[1, 0], np.log(e.sum()))
    assert not out[2].any() and np.all(np.isneginf(lse[2]))
    assert np.all(bo[:2] > 0) and np.all(bo < 1e-3) and np.all(bl < 1e-3)


def test_definition_of_the_rules():
    x = np.array([[1.0, -2.0, 3.0, 3.0, 0.5, -1.0]])
    h = np.array([[0, 1, 1, 2, 9, -1, 1]])
    y, a = logits(x, h, [2], [6], [2.0], [0.25], [0.5], np.array([[4, 5, 4, -1]]), np.array([[9.0, 1.0, 2.0, 5.0]]))
    # 0 and 1 in the prompt; 1 once and 2 once after it (9 and -1 are no tokens, the last 1 lies behind the length)
    assert np.allclose(y, [[0.5, -4.75, 0.75, 3.0, 2.5, 0.0]]) and a[0] == 3
    m = np.array([[0b010011]])
    y, a = logits(x, mask=m)
    assert np.array_equal(np.isneginf(y[0]), [False, False, True, True, False, True]) and a[0] == 0
    assert logits(x, mask=np.zeros((1, 1), np.int64))[1][0] == -1


def test_torch_layer_arguments():
    torch = pytest.importorskip("torch")
    from chpe_qwen_engine_b200 import ops
    x = torch.zeros(2, 8)
    with pytest.raises(TypeError, match="unknown argument penalty"):
        ops.logits_process(x, penalty=1)
    with pytest.raises(TypeError, match="by position"):
        ops.logits_process(x, None)
    with pytest.raises(TypeError, match="given twice"):
        ops.qk_norm_rope(x, x, q=x)
    with pytest.raises(TypeError, match="logits is missing"):
        ops.logits_process()
    with pytest.raises(TypeError, match="must be a tensor"):
        ops.logits_process(3)
