"""The batched decode operators on the GPU (chpe_qk_norm_rope,
chpe_attention_decode_paged, chpe_logits_process through
chpe_qwen_engine_b200.ops) against their 64-bit definitions, at the sizes and
masks where they can go wrong.  A bound is half a rounding step of the output's
type plus what the f32 steps before it can be off by (tests/_ops_ref.py)."""
import math

import numpy as np
import pytest

import chpe_qwen_engine_b200 as chpe
from _ops_ref import HALF_STEP, SMALLEST, attention, logits, norm_rope

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
if torch is not None:
    from chpe_qwen_engine_b200 import ops

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEV = "cuda:0"


def f64(t):
    return t.double().cpu().numpy()


def put(a, kind):
    """numpy -> (device tensor of the type, its values in 64 bits)"""
    t = torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(DEV).to(DT[kind])
    return t, f64(t)


def i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(DEV)


def close(got, ref, before, kind, what=""):
    """|got - ref| within half a step of the type plus the f32 error before the rounding."""
    got = f64(got) if torch.is_tensor(got) else got
    tol = HALF_STEP[kind] * (np.abs(ref) + before) + before + SMALLEST[kind]
    worst = np.max(np.abs(got - ref) / tol) if got.size else 0.0
    assert worst <= 1, f"{what}: {worst:.3g} times the bound"


# ---- q/k norm, rotation, append --------------------------------------------------
@pytest.mark.parametrize("kind, cache", [("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("T, H, KV, D, rope", [
    (1, 16, 4, 256, 64), (1, 16, 2, 128, 128), (3, 5, 3, 64, 32), (7, 64, 8, 128, 128), (2, 1, 1, 64, 0),
    (5, 3, 1, 256, 16), (4, 9, 3, 128, 48), (130, 40, 40, 64, 64), (33, 100, 20, 256, 256)])
def test_qk_norm_rope(kind, cache, T, H, KV, D, rope):
    rng = np.random.default_rng(T * H + D)
    packed, x = put(rng.standard_normal((T, (H + 2 * KV) * D + 16)) * np.exp(rng.uniform(-3, 3, (T, 1))), kind)
    at = np.cumsum([0, H * D, KV * D, KV * D])
    q, k, v = (packed[:, at[i]:at[i + 1]].unflatten(1, (-1, D)) for i in range(3))
    xq, xk, xv = (x[:, at[i]:at[i + 1]].reshape(T, -1, D) for i in range(3))
    w = (1 + 0.2 * rng.standard_normal((2, D))).astype(np.float32)
    pos = rng.integers(0, 2 ** 20, T).astype(np.int32)
    pos[0] = 2 ** 31 - 1 if T > 1 else 131071
    f = ops.rope_inv_freq(1e6, rope) if rope else None
    page, pages = 16, (T + 15) // 16 + 1
    slots = rng.permutation(page * pages)[:T].astype(np.int64)
    if T > 2:
        slots[1] = -1  # a padded token
    if T > 4:
        slots[3] = page * pages  # behind the cache
    kc, vc = (torch.full((pages, page, KV, D), 7.0, dtype=DT[cache], device=DEV) for _ in range(2))
    q_out, k_out = ops.qk_norm_rope(q, k, v, i32(pos), f, q_weight=torch.from_numpy(w[0]).to(DEV),
                                    k_weight=torch.from_numpy(w[1]).to(DEV), eps=1e-6, weight_offset=0.25, k_cache=kc,
                                    v_cache=vc, slots=torch.from_numpy(slots).to(DEV))
    assert k_out is None
    rq, bq = norm_rope(xq, w[0], 0.25, 1e-6, pos, f)
    rk, bk = norm_rope(xk, w[1], 0.25, 1e-6, pos, f)
    close(q_out, rq, bq, kind, "q")
    wk, wv, bound = np.full((page * pages, KV, D), 7.0), np.full((page * pages, KV, D), 7.0), np.zeros((page * pages, KV, D))
    fine = (slots >= 0) & (slots < page * pages)
    wk[slots[fine]], wv[slots[fine]], bound[slots[fine]] = rk[fine], xv[fine], bk[fine]
    close(kc.view(-1, KV, D), wk, bound, cache, "k")
    close(vc.view(-1, KV, D), wv, 0 * wv, cache, "v")
    # without norm and cache, in place
    q2, k2 = q.clone(), k.clone()
    a, b = ops.qk_norm_rope(q2, k2, None, i32(pos), f, q_out=q2, k_out=k2)
    assert a is q2 and b is k2
    close(q2, *norm_rope(xq, None, 0, 0, pos, f), kind, "q in place")
    close(k2, *norm_rope(xk, None, 0, 0, pos, f), kind, "k in place")


def test_qk_values_at_the_type_limits():
    """Zero heads, the largest halves, subnormals: the norm in f32 neither overflows nor loses them."""
    x = np.zeros((4, 2, 64), np.float32)
    x[1] = 65504.0
    x[2] = 2.0 ** -24
    x[3, :, ::2] = -65504.0
    q, xq = put(x, "f16")
    w = torch.ones(64, device=DEV)
    out, k = ops.qk_norm_rope(q, q, None, i32([0, 1, -5, 7]), ops.rope_inv_freq(1e4, 64), q_weight=w, k_weight=w, eps=1e-12)
    ref, b = norm_rope(xq, np.ones(64), 0, 1e-12, np.array([0, 1, -5, 7]), ops.rope_inv_freq(1e4, 64))
    close(out, ref, b, "f16")
    assert torch.equal(out, k)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D, rope", [(64, 0), (64, 32), (128, 48), (256, 64)])
def test_qk_what_is_not_rotated_stays(kind, D, rope):
    """Bit for bit, whatever stands beside it: infinities, NaN, zeros of both signs."""
    x = np.random.default_rng(D).standard_normal((3, 2, D)).astype(np.float32)
    x[:, :, rope + 1::7], x[:, :, rope + 2::7], x[:, :, rope + 3::7] = np.inf, np.nan, -0.0
    q, _ = put(x, kind)
    kc, vc = (torch.zeros(1, 16, 2, D, dtype=DT["f16" if kind == "f32" else kind], device=DEV) for _ in range(2))
    out, _ = ops.qk_norm_rope(q, q, q, i32([1, 2, 3]), ops.rope_inv_freq(1e4, rope) if rope else None, k_cache=kc, v_cache=vc,
                              slots=torch.tensor([3, 4, 5], device=DEV))
    bits = lambda t: t[..., rope:].contiguous().view(torch.int32 if t.dtype == torch.float32 else torch.int16)  # noqa: E731
    number = ~torch.isnan(q[..., rope:])
    assert torch.equal(bits(out)[number], bits(q)[number]) and torch.isnan(out[..., rope:][~number]).all()
    row = q.to(kc.dtype)
    assert torch.equal(bits(kc[0, 3:6])[number], bits(row)[number]) and torch.equal(bits(vc[0, 3:6])[number], bits(row)[number])


def test_qk_more_tokens_than_a_grid_row():
    T = 70001
    q = torch.randn(T, 1, 64, device=DEV, dtype=torch.bfloat16)
    pos = torch.arange(T, device=DEV, dtype=torch.int32)
    f = ops.rope_inv_freq(1e4, 64)
    out, k = ops.qk_norm_rope(q, q, None, pos, f)
    at = np.array([0, 65535, 65536, T - 1])
    ref, b = norm_rope(f64(q)[at], None, 0, 0, at, f)
    close(f64(out)[at], ref, b, "bf16")
    assert torch.equal(out, k)


# ---- paged attention ---------------------------------------------------------------
def paged_case(rng, kind, cache, lens, H, KV, D, page, spare=2, spread=1.0):
    """Tensors of a batch whose pages lie in a shuffled order; every cache entry that
    no sequence uses is NaN or infinite."""
    B, each = len(lens), max(1, -(-max(max(lens), 1) // page))
    pages = B * each + spare
    table = rng.permutation(pages)[:B * each].reshape(B, each).astype(np.int32)
    kc, vc = rng.standard_normal((2, pages, page, KV, D)).astype(np.float32)
    used = np.zeros((pages, page), bool)
    for b, n in enumerate(lens):
        for p in range(max(n, 0)):
            used[table[b, p // page], p % page] = True
    kc[~used], vc[~used] = np.nan, np.inf
    q, xq = put(spread * rng.standard_normal((B, H, D)), kind)
    tk, xk = put(kc, cache)
    tv, xv = put(vc, cache)
    return q, tk, tv, table, xq, xk, xv


def check_paged(q, tk, tv, table, lens, xq, xk, xv, kind, cache, page, scale=None, what=""):
    D = q.shape[2]
    lse = torch.full(q.shape[:2], 5.0, device=DEV)
    out = ops.attention_decode_paged(q, tk, tv, i32(table), i32(lens), scale=scale, lse=lse)
    ref, rl, bo, bl = attention(xq, xk, xv, table, lens, D ** -0.5 if scale is None else scale, page, kind, cache)
    empty = np.isneginf(rl)
    assert np.array_equal(np.isneginf(f64(lse)), empty), what
    assert not f64(out)[empty].any()
    close(out, ref, bo, kind, what + " out")
    assert np.all(np.abs(f64(lse)[~empty] - rl[~empty]) <= bl[~empty]), what + " lse"
    return out, lse


@pytest.mark.parametrize("kind, cache", [("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("H, KV, D", [(16, 2, 128), (16, 4, 256), (4, 4, 64), (12, 4, 128), (24, 2, 64), (9, 1, 256), (64, 4, 128),
                                      (40, 2, 64), (33, 1, 128)])
@pytest.mark.parametrize("page", [16, 64])
def test_paged_attention(kind, cache, H, KV, D, page):
    rng = np.random.default_rng(H + D + page)
    lens = [1, 0, 15, 16, 17, 63, 64, 65, 200, -3, 129]
    check_paged(*(c := paged_case(rng, kind, cache, lens, H, KV, D, page))[:4], lens, *c[4:], kind, cache, page)


@pytest.mark.parametrize("lens", [[1], [16], [20001], [0, 0, 0], [0, 9000, 0, 3], [5000, 1, 5001, 64], [3] * 300,
                                  list(range(130)), [700] * 65])
def test_paged_attention_shares_of_the_work(lens):
    """One long sequence, many short ones, none at all: every way the line of tiles is cut."""
    rng = np.random.default_rng(len(lens))
    c = paged_case(rng, "f16", "f16", lens, 4, 2, 64, 64)
    check_paged(*c[:4], lens, *c[4:], "f16", "f16", 64)


@pytest.mark.parametrize("kind, cache", [("f32", "f16"), ("bf16", "bf16")])
def test_paged_attention_sharp_and_flat(kind, cache):
    """Scores hundreds apart (one entry takes all), all alike, and a head of tiny or huge queries."""
    rng = np.random.default_rng(7)
    lens = [300, 300]
    c = paged_case(rng, kind, cache, lens, 8, 2, 128, 16, spread=40.0)
    check_paged(*c[:4], lens, *c[4:], kind, cache, 16, what="sharp")
    q, xq = put(np.full((2, 8, 128), 1e-30 if kind == "f32" else 2.0 ** -100), kind)
    check_paged(q, *c[1:4], lens, xq, *c[5:], kind, cache, 16, what="flat")
    if kind == "f32":  # beyond FP16's range
        q, xq = put(1e7 * rng.standard_normal((2, 8, 128)), kind)
        check_paged(q, *c[1:4], lens, xq, *c[5:], kind, cache, 16, scale=1e-7 / 11, what="huge")


def test_paged_attention_keeps_small_weights():
    """One entry of weight 1 and 20000 of 2e-7: together 0.4 % of the sum."""
    n, D = 20001, 64
    pages = -(-n // 64)
    k = np.zeros((pages, 64, 1, D), np.float32)
    v = np.ones((pages, 64, 1, D), np.float32)
    k[0, 0, 0, 0], v[0, 0] = 1.0, 0.0
    q = np.zeros((1, 1, D), np.float32)
    q[0, 0, 0] = math.log(5e6)
    tq, xq = put(q, "f32")
    tk, xk = put(k, "f16")
    tv, xv = put(v, "f16")
    table = np.arange(pages, dtype=np.int32)[None]
    check_paged(tq, tk, tv, table, [n], xq, xk, xv, "f32", "f16", 64, scale=1.0)


def test_paged_attention_bad_pages_and_lengths_beyond_the_table():
    rng = np.random.default_rng(3)
    lens = [100, 100, 100]
    q, tk, tv, table, xq, xk, xv = paged_case(rng, "f16", "f16", lens, 8, 2, 64, 16)
    table[0, 2], table[1, :], table[2, 6] = -1, 10 ** 9, tk.shape[0]
    given = [100, 100, 2 ** 31 - 1]  # the last: as long as its table, whose last page is bad
    kept = [100, 100, 112]
    out, lse = check_paged(q, tk, tv, table, kept, xq, xk, xv, "f16", "f16", 16)
    lse2 = torch.empty_like(lse)
    out2 = ops.attention_decode_paged(q, tk, tv, i32(table), i32(given), lse=lse2)
    assert torch.equal(out, out2) and torch.equal(lse, lse2)
    # a table without entries, a cache without pages: all empty
    for t, a, b in ((torch.empty(3, 0, dtype=torch.int32, device=DEV), tk, tv), (i32(table), tk[:0], tv[:0])):
        o = ops.attention_decode_paged(q, a, b, t, i32(given), lse=lse2)
        assert not o.any() and torch.isneginf(lse2).all()


def test_paged_attention_nan_and_infinite_entries():
    """A NaN query makes its head NaN and no other; NaN in K or V its sequence's kv head."""
    rng = np.random.default_rng(4)
    lens = [70, 70]
    q, tk, tv, table, xq, xk, xv = paged_case(rng, "f16", "f16", lens, 4, 2, 64, 16)
    clean = ops.attention_decode_paged(q, tk, tv, i32(table), i32(lens))
    q2 = q.clone()
    q2[0, 1, 5] = float("nan")
    out = ops.attention_decode_paged(q2, tk, tv, i32(table), i32(lens))
    assert torch.isnan(out[0, 1]).all()
    keep = torch.ones(2, 4, dtype=torch.bool, device=DEV)
    keep[0, 1] = False
    assert torch.equal(out[keep], clean[keep])
    v2 = tv.clone()
    v2[table[1, 2], 3, 1, 7] = float("nan")
    out = ops.attention_decode_paged(q, tk, v2, i32(table), i32(lens))
    assert torch.isnan(out[1, 2:, 7]).all() and torch.isnan(out).sum() == 2


def test_paged_attention_strides_and_shared_pages():
    rng = np.random.default_rng(5)
    B, H, KV, D, page = 3, 8, 2, 128, 32
    lens = [50, 64, 33]
    _, tk, tv, table, _, xk, xv = paged_case(rng, "bf16", "bf16", [64], H, KV, D, page)
    table = np.repeat(table, B, 0)  # one prefix for all
    wide, xw = put(rng.standard_normal((B, H * D + 64)), "bf16")
    q, xq = wide[:, :H * D].unflatten(1, (H, D)), xw[:, :H * D].reshape(B, H, D)
    room = torch.full((B, H * D + 8), 3.0, dtype=torch.bfloat16, device=DEV)
    out = room[:, :H * D].unflatten(1, (H, D))
    got = ops.attention_decode_paged(q, tk, tv, i32(table[:1]).expand(B, -1), i32(lens), out=out)
    assert got is out and (room[:, H * D:] == 3).all()
    ref, _, bo, _ = attention(xq, xk, xv, table, lens, D ** -0.5, page, "bf16", "bf16")
    close(out, ref, bo, "bf16")
    big = torch.full((B, table.shape[1] + 5), -1, dtype=torch.int32, device=DEV)
    big[:, :table.shape[1]] = i32(table)
    assert torch.equal(out, ops.attention_decode_paged(q, tk, tv, big[:, :table.shape[1]], i32(lens)))


def test_paged_attention_offsets_beyond_32_bits():
    """Cache rows whose element offset passes 2^32: 5 GB of cache, a few pages of it used."""
    KV, D, page = 8, 128, 64
    pages = (2 ** 32) // (page * KV * D) + 40
    tk = torch.zeros(pages, page, KV, D, dtype=torch.float16, device=DEV)
    tv = torch.zeros(pages, page, KV, D, dtype=torch.float16, device=DEV)
    ids = np.array([pages - 1, 3, pages - 2, pages - 40])
    k, v = np.random.default_rng(6).standard_normal((2, 4, page, KV, D)).astype(np.float32)
    at = torch.from_numpy(ids).to(DEV)
    slots = (at[:, None] * page + torch.arange(page, device=DEV)).reshape(-1)
    (sk, xk), (sv, xv) = put(k, "f16"), put(v, "f16")
    pos = torch.zeros(4 * page, dtype=torch.int32, device=DEV)
    ops.qk_norm_rope(sk.view(-1, KV, D), sk.view(-1, KV, D), sv.view(-1, KV, D), pos, None, k_cache=tk, v_cache=tv,
                     slots=slots)
    assert torch.equal(tk[at], sk) and torch.equal(tv[at], sv)
    q, xq = put(np.random.default_rng(8).standard_normal((1, 16, D)), "f16")
    out = ops.attention_decode_paged(q, tk, tv, i32(ids)[None], i32([250]))
    ref, _, bo, _ = attention(xq, xk, xv, np.arange(4)[None], [250], D ** -0.5, page, "f16", "f16")
    close(out, ref, bo, "f16")


# ---- logits rules --------------------------------------------------------------------
def rules_case(rng, B, V, L, n, mask, kind):
    x, x64 = put(4 * rng.standard_normal((B, V)), kind)
    a = dict(history=None, prompt=None, total=None, rep=None, freq=None, pres=None, ids=None, vals=None, mask=None)
    if L:
        h = np.minimum((rng.random((B, L)) ** 6 * V).astype(np.int64), V - 1)
        h[rng.random((B, L)) < 0.05] = -1
        h[rng.random((B, L)) < 0.02] = V
        a["history"], a["total"] = h, rng.integers(-2, L + 3, B)
        a["prompt"] = rng.integers(-1, L + 2, B)
        a["rep"], a["freq"], a["pres"] = (rng.uniform(lo, hi, B).astype(np.float32) for lo, hi in ((0.7, 1.6), (-1, 1), (-1, 1)))
    if n:
        a["ids"] = rng.integers(-1, min(V + 1, 3 * n), (B, n))
        a["vals"] = rng.standard_normal((B, n)).astype(np.float32)
    if mask:
        a["mask"] = rng.integers(-2 ** 31, 2 ** 31, (B, (V + 31) // 32))
        a["mask"][B // 2] = 0  # a row whose mask leaves nothing
    return x, x64, a


def on_gpu(a):
    f = lambda k, dt: None if a[k] is None else torch.from_numpy(np.ascontiguousarray(a[k]).astype(dt)).to(DEV)  # noqa: E731
    return dict(history=f("history", np.int32), prompt_lens=f("prompt", np.int32), total_lens=f("total", np.int32),
                repetition=f("rep", np.float32), frequency=f("freq", np.float32), presence=f("pres", np.float32),
                bias_ids=f("ids", np.int32), bias_values=f("vals", np.float32), mask=f("mask", np.int32))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("B, V, L, n, mask", [
    (1, 1, 1, 1, True), (2, 31, 5, 0, False), (3, 32, 0, 4, False), (2, 33, 7, 3, True), (5, 1000, 40, 10, True),
    (3, 1003, 300, 0, True), (2, 50257, 1000, 300, False), (2, 151936, 2000, 0, False), (1, 151936, 0, 0, True),
    (2, 300000, 500, 65, True), (1, 300001, 8000, 0, True), (4, 4096, 0, 0, False),
    # counts beyond 14 bits; slices counted in two goes, by 16 and by 8 CTAs per row; batches beyond 14 and 32 rows
    (1, 40, 40000, 3, False), (2, 151936, 16384, 4, False), (2, 500003, 3000, 50, True), (16, 300001, 200, 5, True),
    (15, 1003, 30, 0, True), (33, 3000, 50, 4, True)])
def test_logits_rules(kind, B, V, L, n, mask):
    rng = np.random.default_rng(V + L)
    x, x64, a = rules_case(rng, B, V, L, n, mask, kind)
    out, am = ops.logits_process(x, **on_gpu(a))
    # the same steps in f32, one rounding each: equal to the last bit
    want, wam = logits(x64, **a, kind=np.float32)
    got = out.cpu().numpy()
    assert got.dtype == np.float32 and np.array_equal(got, want)
    assert np.array_equal(am.cpu().numpy(), wam)
    # and the definition in 64 bits: five roundings of values within the largest one met
    ref, _ = logits(x64, **a)
    fine = np.isfinite(ref)
    size = np.abs(x64).max() * 2 + (L + 1) * 1.0 + 6
    assert np.array_equal(fine, np.isfinite(got)) and np.abs(got[fine] - ref[fine]).max(initial=0) <= 5 * 2.0 ** -24 * size
    # the token alone
    none, am2 = ops.logits_process(x, **on_gpu(a), want_logits=False)
    assert none is None and torch.equal(am, am2)


def test_logits_each_rule_alone():
    rng = np.random.default_rng(9)
    x, x64, a = rules_case(rng, 3, 700, 50, 6, True, "f32")
    g = on_gpu(a)
    sets = [("history", "rep"), ("history", "freq"), ("history", "pres"), ("history", "total", "rep"), ("history", "prompt", "freq"),
            ("ids", "vals"), ("mask",), ("history",)]
    name = dict(rep="repetition", freq="frequency", pres="presence", total="total_lens", prompt="prompt_lens", ids="bias_ids", vals="bias_values")
    for keys in sets:
        out, am = ops.logits_process(x, **{name.get(k, k): g[name.get(k, k)] for k in keys})
        want, wam = logits(x64, **{k: a[k] for k in keys}, kind=np.float32)
        assert np.array_equal(out.cpu().numpy(), want) and np.array_equal(am.cpu().numpy(), wam), keys


def test_logits_special_values():
    inf, nan = math.inf, math.nan
    x = np.array([[nan, 1, 1, -0.0], [nan, nan, nan, nan], [-inf, -inf, -inf, -inf], [-0.0, 0.0, -1, nan],
                  [1, inf, inf, 2], [-3.4e38, -3.4e38, nan, -inf], [5, 5, 5, 5]], np.float32)
    out, am = ops.logits_process(torch.from_numpy(x).to(DEV))
    assert np.array_equal(out.cpu().numpy(), x, equal_nan=True)
    assert am.tolist() == [1, -1, -1, 0, 1, 0, 0]
    # biases of -inf ban, +inf force, the last of equal ids counts, +inf - inf is NaN
    ids = torch.tensor([[0, 1, 0, 2]] * 7, dtype=torch.int32, device=DEV)
    vals = torch.tensor([[-inf, inf, 2.0, -inf]] * 7, device=DEV)
    out, am = ops.logits_process(torch.from_numpy(x).to(DEV), bias_ids=ids, bias_values=vals)
    want, wam = logits(x, ids=ids.cpu().numpy(), vals=vals.cpu().numpy(), kind=np.float32)
    assert np.array_equal(out.cpu().numpy(), want, equal_nan=True) and am.tolist() == wam.tolist()


def test_logits_strides_in_place_and_shared_lists():
    rng = np.random.default_rng(10)
    B, V = 5, 2001
    x, x64, a = rules_case(rng, B, V, 30, 7, True, "f32")
    g = on_gpu(a)
    want, wam = logits(x64, **a, kind=np.float32)
    for wide in (V, V + 1, V + 3, 2 * V + 7):  # aligned and unaligned rows
        room = torch.full((B, wide), 9.0, device=DEV)
        room[:, :V] = x
        out, am = ops.logits_process(room[:, :V], **g, out=room[:, :V])
        assert np.array_equal(room[:, :V].cpu().numpy(), want) and (room[:, V:] == 9).all()
        assert am.tolist() == wam.tolist()
    hist = torch.full((B, 64), 3, dtype=torch.int32, device=DEV)
    hist[:, :30] = g["history"]
    a1 = dict(a, ids=a["ids"][:1].repeat(B, 0), vals=a["vals"][:1].repeat(B, 0), mask=a["mask"][:1].repeat(B, 0))
    g1 = dict(g, history=hist[:, :30], bias_ids=g["bias_ids"][:1].expand(B, -1), bias_values=g["bias_values"][:1].expand(B, -1),
              mask=g["mask"][:1].expand(B, -1))
    out, am = ops.logits_process(x, **g1)
    want, wam = logits(x64, **a1, kind=np.float32)
    assert np.array_equal(out.cpu().numpy(), want) and am.tolist() == wam.tolist()


def test_logits_many_biases():
    """65535 entries, the most: the last of each id counts."""
    rng = np.random.default_rng(11)
    ids = rng.integers(0, 500, (1, 65535)).astype(np.int32)
    vals = rng.standard_normal((1, 65535)).astype(np.float32)
    x, x64 = put(rng.standard_normal((1, 600)), "f32")
    out, am = ops.logits_process(x, bias_ids=i32(ids), bias_values=torch.from_numpy(vals).to(DEV))
    want, wam = logits(x64, ids=ids, vals=vals, kind=np.float32)
    assert np.array_equal(out.cpu().numpy(), want) and am.tolist() == wam.tolist()


# ---- refusals on the GPU, streams, graphs -------------------------------------------------
def test_refusals_of_host_and_misaligned_buffers():
    q = torch.zeros(2, 8, 64, dtype=torch.float16, device=DEV)
    kc = torch.zeros(4, 16, 2, 64, dtype=torch.float16, device=DEV)
    t, n = i32(np.zeros((2, 2))), i32([1, 1])
    ws = ops.attention_workspace(64, DEV)
    with pytest.raises(chpe.ChpeError, match="workspace"):
        ops.attention_decode_paged(q, kc, kc, t, n, workspace=ws[:100])
    with pytest.raises(chpe.ChpeError, match="aligned"):
        ops.attention_decode_paged(q, kc, kc, t, n, workspace=torch.empty(ws.numel() + 1, dtype=torch.uint8, device=DEV)[1:])
    with pytest.raises(ValueError):
        ops.attention_decode_paged(q, kc, kc, t.cpu(), n)
    with pytest.raises(ValueError):
        ops.attention_decode_paged(q, kc, kc.float(), t, n)
    with pytest.raises(chpe.ChpeError, match="multiple"):
        ops.attention_decode_paged(q[:, :7].contiguous(), kc, kc, t, n)
    with pytest.raises(chpe.ChpeError, match="type"):
        ops.attention_decode_paged(q.bfloat16(), kc, kc, t, n)
    host = np.zeros(64, np.int32)
    rc = chpe.lib().chpe_attention_decode_paged(
        q.data_ptr(), 1, 512, kc.data_ptr(), kc.data_ptr(), 1, 4, 16, t.data_ptr(), 2, 2, host.ctypes.data, 2, 8, 2, 64,
        1.0, q.data_ptr(), 512, None, ws.data_ptr(), ws.numel(), None)
    assert rc == -1 and b"seq_lens is not device memory" in chpe.lib().chpe_last_error(None)
    x = torch.zeros(2, 40, device=DEV)
    with pytest.raises(ValueError):
        ops.logits_process(x, mask=i32(np.zeros((2, 1))))
    with pytest.raises(chpe.ChpeError, match="without a history"):
        ops.logits_process(x, repetition=torch.ones(2, device=DEV))


def step(s):
    """One decode step: the three operators one after the other on the batch's state."""
    q, _ = ops.qk_norm_rope(s["q"], s["k"], s["v"], s["pos"], s["freq"], q_weight=s["w"], k_weight=s["w"], k_cache=s["kc"],
                            v_cache=s["vc"], slots=s["slots"], q_out=s["q_out"])
    a = ops.attention_decode_paged(q, s["kc"], s["vc"], s["table"], s["lens"], out=s["a"], lse=s["lse"], workspace=s["ws"])
    torch.matmul(a.view(s["B"], -1), s["head"], out=s["x"])
    ops.logits_process(s["x"], history=s["hist"], total_lens=s["lens"], repetition=s["rep"], mask=s["mask"], out=s["y"],
                       argmax=s["tok"])


def step_state(seed, B=5, H=8, KV=2, D=128, V=997, page=16, cap=8):
    g = torch.Generator(DEV).manual_seed(seed)
    r = lambda *n: torch.randn(*n, generator=g, device=DEV)  # noqa: E731
    s = dict(B=B, q=r(B, H, D).half(), k=r(B, KV, D).half(), v=r(B, KV, D).half(), w=1 + 0.1 * r(D), freq=ops.rope_inv_freq(1e4, D),
             kc=torch.full((B * cap, page, KV, D), math.nan, device=DEV).half(), table=torch.randperm(B * cap, generator=g, device=DEV).int().view(B, cap),
             head=(r(H * D, V) / 8).half(), rep=torch.full((B,), 1.3, device=DEV), mask=torch.full((B, (V + 31) // 32), 0x5DF7BEEF, device=DEV, dtype=torch.int32))
    s["vc"] = s["kc"].clone()
    z = lambda *n, dt=torch.float32: torch.zeros(*n, device=DEV, dtype=dt)  # noqa: E731
    s.update(pos=z(B, dt=torch.int32), lens=z(B, dt=torch.int32), slots=z(B, dt=torch.int64), q_out=torch.empty_like(s["q"]), a=torch.empty_like(s["q"]),
             lse=z(B, H), x=z(B, V, dt=torch.float16), y=z(B, V), tok=z(B, dt=torch.int32), hist=z(B, cap * page, dt=torch.int32),
             ws=ops.attention_workspace(D, DEV))
    return s


def advance(s, i, seed):
    """The host's part between steps: new projections, positions, slots, lengths."""
    g = torch.Generator(DEV).manual_seed(seed)
    page = s["kc"].shape[1]
    for name in ("q", "k", "v"):
        s[name].copy_(torch.randn(s[name].shape, generator=g, device=DEV))
    if i:
        s["hist"][torch.arange(s["B"]), s["lens"].long() - 1] = s["tok"]
    s["pos"].fill_(i)
    s["slots"].copy_(s["table"][:, i // page].long() * page + i % page)
    s["lens"].fill_(i + 1)


def test_a_run_of_steps_matches_the_definitions():
    s = step_state(1)
    B, KV, D, page = s["B"], 2, 128, 16
    table = s["table"].cpu().numpy()
    kc, vc = np.zeros((2, B * 8 * page, KV, D))
    for i in range(40):
        advance(s, i, 100 + i)
        step(s)
        torch.cuda.synchronize()
        w, pos, slots = s["w"].cpu().numpy(), s["pos"].cpu().numpy(), s["slots"].cpu().numpy()
        rq, bq = norm_rope(f64(s["q"]), w, 0, 1e-6, pos, s["freq"])
        close(s["q_out"], rq, bq, "f16", f"step {i}: q")
        rk, bk = norm_rope(f64(s["k"]), w, 0, 1e-6, pos, s["freq"])
        row = s["kc"].view(-1, KV, D)[s["slots"]]
        close(row, rk, bk, "f16", f"step {i}: k")
        kc[slots], vc[slots] = f64(row), f64(s["v"])
        n = np.full(B, i + 1)
        ref, rl, bo, bl = attention(f64(s["q_out"]), kc.reshape(-1, page, KV, D), vc.reshape(-1, page, KV, D), table, n, D ** -0.5, page, "f16", "f16")
        close(s["a"], ref, bo, "f16", f"step {i}: attention")
        assert np.all(np.abs(f64(s["lse"]) - rl) <= bl)
        want, tok = logits(f64(s["x"]), s["hist"].cpu().numpy(), None, n, np.full(B, np.float32(1.3)), mask=s["mask"].cpu().numpy(), kind=np.float32)
        assert np.array_equal(s["y"].cpu().numpy(), want) and s["tok"].tolist() == tok.tolist(), i


def test_a_captured_step_replays_as_the_sequences_grow():
    """One graph for all steps; two graphs with workspaces of their own on two streams."""
    eager, caught = [step_state(k) for k in (1, 2)], [step_state(k) for k in (1, 2)]
    for s in caught:
        advance(s, 0, 0)
        step(s)  # attributes and handles are set up before the capture
    torch.cuda.synchronize()
    graphs, streams = [], [torch.cuda.Stream() for _ in caught]
    for s, st in zip(caught, streams):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=st):
            step(s)
        graphs.append(gr)
    for i in range(70):
        for s in eager + caught:
            advance(s, i, 7 * i)
        for s in eager:
            step(s)
        torch.cuda.synchronize()
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for a, b in zip(eager, caught):
            for name in ("q_out", "a", "lse", "y", "tok"):
                assert torch.equal(a[name], b[name]), (i, name)


def test_calls_on_two_streams_at_once():
    a, b = step_state(3, B=40), step_state(4, B=33)
    for s in (a, b):
        advance(s, 0, 1)
    want = []
    for s in (a, b):
        step(s)
        torch.cuda.synchronize()
        want.append([s[n].clone() for n in ("a", "lse", "y", "tok")])
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(30):
        for s, st in zip((a, b), streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                step(s)
    torch.cuda.synchronize()
    for s, w in zip((a, b), want):
        assert all(torch.equal(s[n], x) for n, x in zip(("a", "lse", "y", "tok"), w))


def test_the_same_call_gives_the_same_bits():
    rng = np.random.default_rng(12)
    lens = [3000, 1, 777, 0, 2049]
    q, tk, tv, table, *_ = paged_case(rng, "bf16", "bf16", lens, 16, 2, 128, 64)
    first = None
    for _ in range(20):
        lse = torch.empty(5, 16, device=DEV)
        out = ops.attention_decode_paged(q, tk, tv, i32(table), i32(lens), lse=lse)
        first = first or (out, lse)
        assert torch.equal(out, first[0]) and torch.equal(lse, first[1])


@pytest.mark.parametrize("B, n", [(1, 9000), (2, 3000), (5, 1500), (9, 1500), (30, 400), (70, 150)])
def test_paged_attention_joins(B, n):
    """Sequences cut into hundreds, dozens and a few records, joined by the kernel for each."""
    rng = np.random.default_rng(B)
    for kind, H, KV, D in (("bf16", 8, 8, 64), ("f16", 16, 4, 256), ("f16", 8, 1, 128), ("bf16", 24, 2, 64)):
        lens = [int(x) for x in rng.integers(n // 2, n + 1, B)]
        c = paged_case(rng, kind, kind, lens, H, KV, D, 16)
        check_paged(*c[:4], lens, *c[4:], kind, kind, 16)


@pytest.mark.parametrize("kind, cache", [("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("H, KV", [(12, 1), (32, 2), (33, 1), (60, 4)])
def test_paged_attention_many_heads_per_kv_head_and_wide_tables(kind, cache, H, KV):
    """More than 8 query heads per kv head behind tables with room for long sequences."""
    rng = np.random.default_rng(H)
    lens = [700, 0, 16, 333, 1]
    q, tk, tv, table, xq, xk, xv = paged_case(rng, kind, cache, lens, H, KV, 128, 64)
    room = np.full((5, 64 * 2 ** 20 // (5 * 64 * KV * 128 * 4) + 1), -1, np.int32)
    room[:, :table.shape[1]] = table
    check_paged(q, tk, tv, room, lens, xq, xk, xv, kind, cache, 64)


def test_paged_attention_workspace_of_any_content():
    """Garbage in the workspace, and calls of other shapes before, change nothing."""
    rng = np.random.default_rng(14)
    ws = ops.attention_workspace(128, DEV)
    for lens, H, KV in (([2500, 3, 0, 900], 16, 2), ([9] * 200, 8, 8), ([5000], 8, 1)):
        q, tk, tv, table, *_ = paged_case(rng, "f16", "f16", lens, H, KV, 128, 32)
        want = ops.attention_decode_paged(q, tk, tv, i32(table), i32(lens))
        for fill in (0xFF, 0x7F, None):
            if fill is not None:
                ws.fill_(fill)
            assert torch.equal(want, ops.attention_decode_paged(q, tk, tv, i32(table), i32(lens), workspace=ws))


def test_calls_without_rows():
    e = lambda *n, dt=torch.float16: torch.empty(*n, dtype=dt, device=DEV)  # noqa: E731
    kc = torch.full((2, 16, 2, 64), 5.0, dtype=torch.float16, device=DEV)
    q, k = ops.qk_norm_rope(e(0, 4, 64), e(0, 2, 64), e(0, 2, 64), e(0, dt=torch.int32), ops.rope_inv_freq(1e4, 64),
                            k_cache=kc, v_cache=kc.clone(), slots=e(0, dt=torch.int64))
    assert q.shape == (0, 4, 64) and k is None and (kc == 5).all()
    assert ops.attention_decode_paged(e(0, 4, 64), kc, kc, e(0, 3, dt=torch.int32), e(0, dt=torch.int32)).shape == (0, 4, 64)
    x, t = ops.logits_process(e(0, 100), history=e(0, 5, dt=torch.int32))
    assert x.shape == (0, 100) and t.shape == (0,)
    x = torch.randn(3, 100, device=DEV)
    y, t = ops.logits_process(x, history=e(3, 0, dt=torch.int32), repetition=torch.ones(3, device=DEV),
                              bias_ids=e(3, 0, dt=torch.int32), bias_values=e(3, 0, dt=torch.float32))
    assert torch.equal(x, y) and torch.equal(t, x.argmax(1).int())
