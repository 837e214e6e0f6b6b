"""The batched decode operators at the ends of their range.  References and bounds
as in test_gpu_ops.py."""
import numpy as np
import pytest

import chpe_qwen_engine_b200 as chpe
from _ops_ref import attention, logits
from test_gpu_ops import DEV, check_paged, close, f64, i32, on_gpu, paged_case, put, rules_case

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


@pytest.mark.parametrize("cache", ["f16", "bf16"])
@pytest.mark.parametrize("KV, D", [(8, 64), (8, 128), (4, 256)])
def test_sums_over_positions_are_rounded_not_cut(cache, KV, D):
    """All weights 1, the first value 16, then every 16 positions three quarters of a step of
    the sum: cut, none of them would count."""
    m, B, page = 40, 300, 16
    k = np.zeros((m, page, KV, D))
    v = np.zeros((m, page, KV, D))
    v[0, 0], v[1:, 0] = 16.0, 0.75 * 2.0 ** -19
    tk, tv = put(k, cache)[0], put(v, cache)[0]
    q = torch.zeros(B, KV, D, device=DEV)
    n = page * m
    out = ops.attention_decode_paged(q, tk, tv, i32(np.arange(m)[None]).expand(B, -1), i32([n] * B))
    ref = (16.0 + (m - 1) * 0.75 * 2.0 ** -19) / n * np.ones((B, KV, D))
    # an addition for every 16 positions, each off by half a step (2^-24 of the sum); the joins
    # of a few records, the quotient and its product
    close(out, ref, ref * (m - 1 + 8) * 2.0 ** -24, "f32")


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


# ---- angles ----------------------------------------------------------------------------
@pytest.mark.parametrize("theta", [1e4, 1e7])
def test_angles_of_every_size_keep_f32_bits(theta):
    """Pairs (1, 0) turn into the cosine and the sine, each right to its own last bits, those
    of an angle of 1e-7 too."""
    pos = np.array([1, 2, 7, 1000, 131071, 2 ** 30 + 1, -5])
    f = ops.rope_inv_freq(theta, 128)
    x = torch.zeros(len(pos), 1, 128, device=DEV)
    x[..., :64] = 1.0
    out, _ = ops.qk_norm_rope(x, x, None, i32(pos), f)
    a = pos[:, None].astype(np.longdouble) * f.astype(np.longdouble)
    for got, ref in ((out[:, 0, :64], np.cos(a)), (out[:, 0, 64:], np.sin(a))):
        # the angle's rounding and sincospi's 2 ulp of the result; the fixed point's 2^-65 turn of a
        # position, and the reference's 2^-63 of the angle
        tol = (1 + 4) * 2.0 ** -24 * np.abs(ref) + np.abs(pos)[:, None] * 2.0 ** -61
        assert np.all(np.abs(f64(got) - ref) <= tol)


# ---- one long sequence among many short ones ----------------------------------------------
@pytest.mark.parametrize("kind, H, KV, D", [("f16", 8, 2, 64), ("bf16", 16, 8, 128), ("f16", 8, 4, 256), ("bf16", 32, 2, 128)])
@pytest.mark.parametrize("B, n", [(7, 20000), (32, 20000), (64, 20000), (200, 9000), (400, 9000)])
def test_paged_attention_one_long_among_short(kind, H, KV, D, B, n):
    """The long one is cut into far more records than the others."""
    rng = np.random.default_rng(B)
    page, each = 64, -(-n // 64)
    lens = [10] * B
    lens[B // 3] = n
    table = np.full((B, each), -1, np.int32)
    pages = rng.permutation(each + B)
    table[B // 3] = pages[:each]
    table[np.arange(B) != B // 3, 0] = pages[each:each + B - 1]
    tk, xk = put(rng.standard_normal((each + B, page, KV, D)), kind)
    tv, xv = put(rng.standard_normal((each + B, page, KV, D)), kind)
    q, xq = put(rng.standard_normal((B, H, D)), kind)
    check_paged(q, tk, tv, table, lens, xq, xk, xv, kind, kind, page)


# ---- the largest tables of the logits rules ---------------------------------------------
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("B, V, L, n", [(1, 500003, 20000, 40000), (16, 300001, 17000, 33000), (1, 458752, 40000, 65535)])
def test_logits_rules_largest_tables(kind, B, V, L, n):
    """Counts of 32 bits, a bias place and a list entry for every token of a full slice, by 16 and by 8 CTAs per row."""
    rng = np.random.default_rng(V)
    x, x64, a = rules_case(rng, B, V, L, n, True, kind)
    out, am = ops.logits_process(x, **on_gpu(a))
    want, wam = logits(x64, **a, kind=np.float32)
    assert np.array_equal(out.cpu().numpy(), want) and np.array_equal(am.cpu().numpy(), wam)


# ---- buffers that overlap ------------------------------------------------------------
def refused(what, f, *a, **kw):
    with pytest.raises(chpe.ChpeError, match=what):
        f(*a, **kw)


def test_qk_refuses_overlaps():
    T, H, KV, D = 5, 4, 2, 64
    wide = torch.randn(T, (H + 2 * KV) * D + 2 * D, device=DEV).half()
    part = lambda first, heads: wide[:, first * D:(first + heads) * D].unflatten(1, (heads, D))  # noqa: E731
    q, k, v = part(0, H), part(H, KV), part(H + KV, KV)
    freq, pos = ops.rope_inv_freq(1e4, D), i32(range(T))
    kc, vc = torch.zeros(2, 2, 16, KV, D, device=DEV, dtype=torch.float16)
    slots = torch.arange(T, device=DEV)
    a = (q, k, v, pos, freq)
    cache = dict(k_cache=kc, v_cache=vc, slots=slots)
    want = [t.clone() for t in ops.qk_norm_rope(*a)]
    before = wide.clone()
    refused("q_out overlaps k", ops.qk_norm_rope, *a, q_out=part(H, H))
    refused("q_out overlaps q", ops.qk_norm_rope, *a, q_out=part(1, H))
    refused("q_out overlaps v", ops.qk_norm_rope, *a, q_out=part(H + KV, H), **cache)
    both = torch.zeros(T, (H + KV) * D, device=DEV, dtype=torch.float16)
    refused("k_out overlaps q_out", ops.qk_norm_rope, *a, q_out=both[:, :H * D].unflatten(1, (H, D)),
            k_out=both[:, (H - 1) * D:(H + 1) * D].unflatten(1, (KV, D)))
    refused("k_cache overlaps q", ops.qk_norm_rope, q, k, v, pos, freq, k_cache=wide.view(-1)[:16 * KV * D].view(1, 16, KV, D),
            v_cache=vc[:1], slots=slots)
    refused("v_cache overlaps k_cache", ops.qk_norm_rope, *a, k_cache=kc, v_cache=kc, slots=slots)
    rows = torch.zeros(T, 2, KV, D, device=DEV, dtype=torch.float16)
    refused("q_out overlaps positions", ops.qk_norm_rope, rows[:, 0].contiguous(), rows[:, 0].contiguous(), None, rows.view(-1).view(torch.int32)[:T],
            freq, q_out=rows.view(-1)[:T * KV * D].view(T, KV, D))
    torch.cuda.synchronize()
    assert torch.equal(wide, before) and not kc.any()
    # side by side in one buffer they share nothing, and in place is allowed
    out, _ = ops.qk_norm_rope(*a, q_out=q, k_out=k, **cache)
    assert torch.equal(out, want[0]) and torch.equal(k, want[1]) and torch.equal(wide[:, (H + KV) * D:], before[:, (H + KV) * D:])
    wide.copy_(before)
    tail = wide[:, -2 * D:].unflatten(1, (KV, D))  # behind v in the same rows
    assert torch.equal(ops.qk_norm_rope(*a, k_out=tail)[1], want[1])


def test_attention_refuses_overlaps():
    B, H, KV, D = 3, 4, 2, 64
    g = torch.randn(B, 3 * H * D, device=DEV).half()
    q = g[:, :H * D].unflatten(1, (H, D))
    kc, vc = torch.randn(2, 4, 16, KV, D, device=DEV).half()
    table, lens = i32([[0, 1], [2, 3], [1, 0]]), i32([20, 30, 1])
    a = (q, kc, vc, table, lens)
    want = ops.attention_decode_paged(*a)
    refused("out overlaps q", ops.attention_decode_paged, *a, out=q)
    refused("out overlaps q", ops.attention_decode_paged, *a, out=g[:, D:(H + 1) * D].unflatten(1, (H, D)))
    refused("out overlaps k_cache", ops.attention_decode_paged, *a, out=kc.view(-1)[:B * H * D].view(B, H, D))
    refused("out overlaps v_cache", ops.attention_decode_paged, *a, out=vc.view(-1)[-B * H * D:].view(B, H, D))
    ws = ops.attention_workspace(D, DEV)
    refused("lse overlaps seq_lens", ops.attention_decode_paged, *a[:4], ws[:12].view(torch.int32), lse=ws[:4 * B * H].view(torch.float32).view(B, H))
    refused("workspace overlaps out", ops.attention_decode_paged, *a, out=ws[64:64 + 2 * B * H * D].view(torch.float16).view(B, H, D), workspace=ws)
    refused("workspace overlaps page_table", ops.attention_decode_paged, q, kc, vc, ws[-24:].view(torch.int32).view(3, 2), lens, workspace=ws)
    out = g[:, H * D:2 * H * D].unflatten(1, (H, D))  # behind the queries in the same rows
    assert torch.equal(ops.attention_decode_paged(*a, out=out), want)
    assert torch.equal(ops.attention_decode_paged(q, kc, kc, table, lens), ops.attention_decode_paged(q, kc, kc.clone(), table, lens))


def test_logits_refuse_overlaps():
    B, V = 3, 256
    room = torch.randn(B, 3 * V, device=DEV)
    x = room[:, :V]
    want, am = ops.logits_process(x)
    refused("out overlaps logits", ops.logits_process, x, out=room[:, 8:V + 8])
    refused("out overlaps logits", ops.logits_process, x, out=room.view(-1)[:B * V].view(B, V))
    half = torch.zeros(B, 2 * V, device=DEV, dtype=torch.float16)
    refused("out overlaps logits", ops.logits_process, half[:, :V], out=half.view(torch.float32))
    hist = torch.zeros(B, V, device=DEV, dtype=torch.int32)
    refused("out overlaps history", ops.logits_process, x, history=hist, out=hist.view(torch.float32))
    refused("out overlaps mask", ops.logits_process, x, mask=room.view(torch.int32)[:, V + 3:V + 11], out=room[:, V:2 * V])
    few = torch.zeros(8, device=DEV, dtype=torch.int32)
    refused("argmax overlaps total_lens", ops.logits_process, x, history=hist, total_lens=few[:B], argmax=few[1:B + 1])
    refused("argmax overlaps history", ops.logits_process, x, history=hist, argmax=hist.view(-1)[:B])
    refused("out overlaps argmax", ops.logits_process, x, out=room[:, V:2 * V], argmax=room.view(torch.int32)[0, V:V + B])
    y, t = ops.logits_process(x, out=room[:, V:2 * V])
    assert torch.equal(y, want) and torch.equal(t, am)
    # one row's token behind the tokens so far
    one, h = room[:1, :V], hist.view(-1)[:8].view(1, 8)
    ops.logits_process(one, history=h, total_lens=i32([5]), argmax=h[0, 5:6], want_logits=False)
    assert h[0, 5] == am[0] and not h[0, :5].any()
    y, t = ops.logits_process(x, out=x)
    assert torch.equal(room[:, :V], want) and torch.equal(t, am)


# ---- the torch layer ---------------------------------------------------------------------
def test_gradients_are_refused_and_no_grad_is_not():
    p = torch.nn.Parameter
    q, kc = torch.randn(2, 2, 64, device=DEV).half(), torch.randn(2, 16, 2, 64, device=DEV).half()
    pos, freq, w = i32([0, 1]), ops.rope_inv_freq(1e4, 64), p(torch.ones(64, device=DEV))
    table, lens, x = i32([[0], [1]]), i32([3, 4]), torch.randn(2, 40, device=DEV)
    one = torch.ones(2, device=DEV)
    calls = [("q_weight", lambda: ops.qk_norm_rope(q, q, None, pos, freq, q_weight=w)),
             ("k", lambda: ops.qk_norm_rope(q, p(q.clone()), None, pos, freq)),
             ("inv_freq", lambda: ops.qk_norm_rope(q, q, None, pos, p(torch.from_numpy(freq)))),
             ("q", lambda: ops.attention_decode_paged(p(q.clone()), kc, kc, table, lens)),
             ("v_cache", lambda: ops.attention_decode_paged(q, kc, p(kc.clone()), table, lens)),
             ("out", lambda: ops.attention_decode_paged(q, kc, kc, table, lens, out=p(q.clone()))),
             ("logits", lambda: ops.logits_process(x.clone().requires_grad_() * 2)),
             ("repetition", lambda: ops.logits_process(x, history=i32([[1], [2]]), repetition=p(one)))]
    for name, call in calls:
        with pytest.raises(ValueError, match=f"^{name} requires a gradient"):
            call()
        with torch.no_grad():
            call()
        with torch.inference_mode():
            call()


def test_what_is_written_counts_as_written():
    """torch refuses a backward pass through values that an in-place write has replaced since."""
    q, k = (torch.randn(2, 2, 64, device=DEV).half() for _ in range(2))
    kc, vc = (torch.randn(2, 16, 2, 64, device=DEV).half() for _ in range(2))
    lse, x = torch.zeros(2, 2, device=DEV), torch.randn(2, 40, device=DEV)
    out, tok, base = torch.zeros_like(x), i32([0, 0]), torch.zeros(4, 2, 64, device=DEV).half()
    at = lambda *ts: [t._version for t in ts]  # noqa: E731
    v = at(q, k, kc, vc)
    ops.qk_norm_rope(q, k, k, i32([0, 1]), None, q_out=base[:2], k_cache=kc, v_cache=vc, slots=torch.tensor([3, 17], device=DEV))
    assert at(q, k, kc, vc) == [v[0], v[1], v[2] + 1, v[3] + 1] and base._version == 1
    ops.qk_norm_rope(q, k, None, i32([0, 1]), None, q_out=q, k_out=k)
    assert at(q, k) == [v[0] + 1, v[1] + 1]
    v = at(q, kc, vc, lse, base)
    ops.attention_decode_paged(q, kc, vc, i32([[0], [1]]), i32([3, 4]), out=base[2:], lse=lse)
    assert at(q, kc, vc, lse, base) == [v[0], v[1], v[2], v[3] + 1, v[4] + 1]
    v = at(x, out, tok)
    ops.logits_process(x, out=out, argmax=tok)
    assert at(x, out, tok) == [v[0], v[1] + 1, v[2] + 1]
    w = torch.ones(2, 40, device=DEV, requires_grad=True)
    y = (w * out).sum()  # needs `out` for w's gradient
    ops.logits_process(x, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        held = torch.zeros_like(x)
    ops.logits_process(x, out=held)
    assert torch.equal(held, out)


def test_norm_weights_at_any_float():
    """A layer's weights out of one packed buffer."""
    q, k = (torch.randn(3, 2, 64, device=DEV) for _ in range(2))
    packed = torch.randn(1 + 64 + 2 + 64, device=DEV)
    wq, wk = packed[1:65], packed[67:]
    a = ops.qk_norm_rope(q, k, None, i32([0, 1, 2]), ops.rope_inv_freq(1e4, 64), q_weight=wq, k_weight=wk)
    b = ops.qk_norm_rope(q, k, None, i32([0, 1, 2]), ops.rope_inv_freq(1e4, 64), q_weight=wq.clone(), k_weight=wk.clone())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
