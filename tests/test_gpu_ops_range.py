"""The batched decode operators at the ends of their range.  References and bounds
as in test_gpu_ops.py."""
import numpy as np
import pytest

from _ops_ref import attention
from test_gpu_ops import DEV, check_paged, close, f64, i32, paged_case, put

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
if torch is not None:
    from chpe_qwen_engine_b200 import ops


# ---- precision of the attention's operands -------------------------------------------
def bf16(x):
    return torch.tensor(x, dtype=torch.float64).bfloat16().double().numpy()


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_probabilities_keep_f32_bits_over_a_bf16_cache(kind, D):
    """Weights 1, 1 and p with values -hi, -lo and 1, where hi + lo are the two BF16 parts of
    p: the output is what 16 bits of p leave out."""
    rng = np.random.default_rng(1)
    x = np.unique(bf16(-rng.uniform(0.25, 1.0, 4000)))
    p = np.exp(x)
    hi = bf16(p)
    lo = bf16(p - hi)
    at = np.argsort(-np.abs(p - hi - lo) / p)[:8]  # those whose rest is largest
    assert np.all(np.abs(p - hi - lo)[at] > 0.75 * 2.0 ** -18 * p[at])
    x, p, hi, lo = x[at], p[at], hi[at], lo[at]
    q, k, v = np.zeros((1, 8, D)), np.zeros((1, 16, 8, D)), np.zeros((1, 16, 8, D))
    q[0, :, 0] = 1.0
    k[0, 2, :, 0] = x
    v[0, 0], v[0, 1], v[0, 2] = -hi[:, None], -lo[:, None], 1.0
    tq, tk, tv = put(q, kind)[0], put(k, "bf16")[0], put(v, "bf16")[0]
    out = ops.attention_decode_paged(tq, tk, tv, i32([[0]]), i32([3]), scale=1.0)
    ref = ((p - hi - lo) / (2 + p))[None, :, None] * np.ones((1, 8, D))
    # p is off by: log2 e and its product with x (2^-24 each of |x| log2 e < 1.5), the sum of
    # the exponent's argument (half a step below 16: 2^-21), exp2 (2 ulp); the products are summed in f32, cut
    e = np.log(2) * (1.5 * 2.0 ** -23 + 2.0 ** -21) + 2.0 ** -22 + 4 * 2.0 ** -23
    close(out, ref, e * (2 * p / (2 + p))[None, :, None], kind)


def test_the_longest_batch_repeats_its_bits():
    g = torch.Generator(DEV).manual_seed(5)
    n, page = 131071, 64
    table = torch.randperm(2048, generator=g, device=DEV).int()[None]
    kc, vc = (torch.randn(2048, page, 8, 128, generator=g, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    q = torch.randn(1, 64, 128, generator=g, device=DEV, dtype=torch.bfloat16)
    first, lse = None, torch.empty(1, 64, device=DEV)
    for _ in range(20):
        out = ops.attention_decode_paged(q, kc, vc, table, i32([n]), lse=lse)
        first = first or (out, lse.clone())
        assert torch.equal(out, first[0]) and torch.equal(lse, first[1])


@pytest.mark.parametrize("cache", ["f16", "bf16"])
@pytest.mark.parametrize("D, H, KV", [(64, 4, 2), (128, 16, 2), (256, 4, 4), (128, 32, 2)])
@pytest.mark.parametrize("large", [1e3, 4e4, 1e6])
def test_paged_attention_one_large_query_dimension(cache, D, H, KV, large):
    """A dimension far above the others, which the keys do not have: the others count alone."""
    rng = np.random.default_rng(D)
    lens = [300, 17]
    q, tk, tv, table, xq, xk, xv = paged_case(rng, "f32", cache, lens, H, KV, D, 16)
    q[:, :, 5] = large
    tk[..., 5] = 0
    check_paged(q, tk, tv, table, lens, f64(q), f64(tk), xv, "f32", cache, 16)


@pytest.mark.parametrize("largest", [2.0 ** 127, 2.0 ** 100, 2.0 ** -100, 2.0 ** -126, 2.0 ** -140])
@pytest.mark.parametrize("cache", ["f16", "bf16"])
def test_paged_attention_queries_of_every_size(cache, largest):
    """The scale brings the scores back to ordinary ones, as far as f32 holds it."""
    rng = np.random.default_rng(2)
    lens = [100]
    q, tk, tv, table, xq, xk, xv = paged_case(rng, "f32", cache, lens, 4, 2, 64, 16)
    q = (q / q.abs().max() * 1.5).double().mul(largest).float()
    scale = float(np.clip(0.2 / largest, 2.0 ** -126, 1e6))
    check_paged(q, tk, tv, table, lens, f64(q), xk, xv, "f32", cache, 16, scale=scale)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("lens, H, KV, D", [([100, 7], 8, 2, 128), ([2000], 4, 4, 64), ([2000], 8, 2, 256), ([600] * 30, 8, 8, 128)])
def test_paged_attention_large_bf16_values(kind, lens, H, KV, D):
    """Values of 2^112 over some thousand positions: their sums are within f32."""
    rng = np.random.default_rng(3)
    q, tk, tv, table, xq, xk, xv = paged_case(rng, kind, "bf16", lens, H, KV, D, 16)
    tv = tv * 2.0 ** 112
    check_paged(q, tk, tv, table, lens, xq, xk, f64(tv), kind, "bf16", 16)


# ---- what is not finite ----------------------------------------------------------------
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("n, B", [(40, 1), (3000, 1), (3000, 70)])  # in one CTA, cut into many and into few records
@pytest.mark.parametrize("H, KV, D", [(4, 2, 64), (8, 8, 128), (4, 1, 256)])
def test_paged_attention_infinite_scores(kind, n, B, H, KV, D):
    inf = float("inf")
    rng = np.random.default_rng(4)
    G = H // KV
    page, each = 64, -(-n // 64)
    tk, _ = put(rng.standard_normal((each, page, KV, D)), kind)
    tv, _ = put(rng.standard_normal((each, page, KV, D)), kind)
    q, _ = put(np.abs(rng.standard_normal((B, H, D))) + 0.1, kind)  # the sign of a key's infinity is its score's
    table = i32(np.arange(each)[None]).expand(B, -1)
    lens = i32([n] * B)
    lse = torch.empty(B, H, device=DEV)

    def call(k, v=tv, qq=q):
        return ops.attention_decode_paged(qq, k, v, table, lens, lse=lse).clone(), lse.clone()
    clean, clean_lse = call(tk)
    others = torch.arange(H, device=DEV) >= G
    at = n - 5
    for value, kind_of in ((float("nan"), "nan"), (inf, "nan"), (-inf, "gone")):
        k = tk.clone()
        k[at // page, at % page, 0, 3] = value  # kv head 0
        out, l = call(k)
        assert torch.equal(out[:, others], clean[:, others]) and torch.equal(l[:, others], clean_lse[:, others])
        if kind_of == "nan":
            assert torch.isnan(out[:, :G]).all() and torch.isnan(l[:, :G]).all()
        else:  # weight 0: as if the position were not there
            keep = np.arange(n) != at
            kk, vv = (f64(t).reshape(-1, KV, D)[:n][keep] for t in (tk, tv))
            pad = np.zeros((each * page - n + 1, KV, D))
            for b in (0, B - 1):
                ref, rl, bo, bl = attention(f64(q)[b:b + 1], np.concatenate((kk, pad)).reshape(each, page, KV, D),
                                            np.concatenate((vv, pad)).reshape(each, page, KV, D), np.arange(each)[None], [n - 1],
                                            D ** -0.5, page, kind, kind)
                close(out[b:b + 1, :G], ref[:, :G], bo[:, :G], kind)
                assert np.all(np.abs(f64(l)[b, :G] - rl[0, :G]) <= bl[0, :G])
    k = tk.clone()
    k[:, :, 0, 3] = -inf  # every score of kv head 0
    out, l = call(k)
    assert not out[:, :G].any() and torch.isneginf(l[:, :G]).all()
    assert torch.equal(out[:, others], clean[:, others])
    k[0, :, 0, 3] = 1.0  # all but the first page's
    out, l = call(k)
    assert torch.isfinite(out).all() and torch.isfinite(l).all()
    v = tv.clone()
    v[at // page, at % page, 0, 9] = inf
    out, l = call(tk, v)
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[:, :G, 9] = True
    assert torch.equal(~torch.isfinite(out), bad) and torch.equal(out[~bad], clean[~bad]) and torch.equal(l, clean_lse)
    qq = q.clone()
    qq[0, 0, 3] = inf
    out, l = call(tk, tv, qq)
    assert torch.isnan(out[0, 0]).all() and torch.isnan(l[0, 0])
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[0, 0] = True
    assert torch.equal(out[~bad], clean[~bad])


@pytest.mark.parametrize("cache", ["f16", "bf16"])
def test_paged_attention_infinite_keys_under_float_queries(cache):
    """The parts of a float query meet an infinite key one by one: 0 times infinity among them."""
    tk = torch.zeros(1, 16, 1, 64, device=DEV, dtype=torch.float16 if cache == "f16" else torch.bfloat16)
    tv = torch.ones_like(tk)
    tk[0, 2, 0, 0] = -float("inf")
    q = torch.ones(1, 1, 64, device=DEV)
    lse = torch.zeros(1, 1, device=DEV)
    out = ops.attention_decode_paged(q, tk, tv, i32([[0]]), i32([5]), lse=lse)
    assert torch.isnan(out).all() and torch.isnan(lse).all()
    assert torch.equal(ops.attention_decode_paged(q, tk, tv, i32([[0]]), i32([2])), torch.ones_like(q))
