"""The operators of a batched decode step on torch CUDA tensors: q/k norm with
rotation and cache append (chpe_qk_norm_rope), paged decode attention
(chpe_attention_decode_paged) and the logits rules (chpe_logits_process).

include/chpe.h states what each computes and what it refuses.  The functions
here take shapes, strides and types from the tensors, check that they fit
together, run on the current stream of the tensors' device (which need not be
the current device), and raise ChpeError for what the library refuses and
ValueError for tensors that do not fit.  Nothing is allocated when the outputs
and the workspace are passed.  A cache is a pair of contiguous tensors
[num_pages, page_size, num_kv_heads, head_dim].
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import torch

from . import ChpeError, lib

_DTYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _check(rc: int) -> None:
    if rc != 0:
        raise ChpeError(lib().chpe_last_error(None).decode())


def _want(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _dtype(t: torch.Tensor, name: str) -> int:
    d = _DTYPE.get(t.dtype)
    if d is None:
        raise ValueError(f"{name} must be float32, float16 or bfloat16, not {t.dtype}")
    return d


def _vec(t, name: str, dtype, n: int, dev):
    """Address of a contiguous 1-D tensor of n values (None: NULL)."""
    if t is None:
        return None
    if t.dtype != dtype or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous() or t.device != dev:
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of {n} values on {dev}")
    return t.data_ptr()


def _heads(t: torch.Tensor, name: str, dtype, dev, n: int, heads: int, d: int) -> int:
    """Stride between the tokens of [n, heads, d] whose heads are contiguous."""
    if t.dtype != dtype or t.device != dev or t.dim() != 3 or t.shape != (n, heads, d):
        raise ValueError(f"{name} must be a {dtype} tensor [{n}, {heads}, {d}] on {dev}")
    s = t.stride()
    if t.numel() and (s[2] != 1 or (heads > 1 and s[1] != d)):
        raise ValueError(f"{name}: the heads of a token must be contiguous")
    return s[0]


def _rows(t: torch.Tensor, name: str, dtype, dev, n: int, width: int | None) -> int:
    """Stride between the rows of [n, width] with contiguous rows (0 for a row
    that is expanded over all n)."""
    if t.dtype != dtype or t.device != dev or t.dim() != 2 or t.shape[0] != n or (width is not None and t.shape[1] != width):
        raise ValueError(f"{name} must be a {dtype} tensor [{n}, {'any' if width is None else width}] on {dev}")
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"{name}: rows must be contiguous")
    return t.stride(0)


def _cache(k_cache: torch.Tensor, v_cache: torch.Tensor, kv: int, d: int, dev) -> int:
    if (k_cache.dim() != 4 or k_cache.shape != v_cache.shape or k_cache.dtype != v_cache.dtype
            or k_cache.shape[2:] != (kv, d) or not k_cache.is_contiguous() or not v_cache.is_contiguous()
            or k_cache.device != dev or v_cache.device != dev):
        raise ValueError(f"the caches must be two contiguous tensors [pages, page size, {kv}, {d}] of one type on {dev}")
    return _dtype(k_cache, "the cache")


def _cuda(t: torch.Tensor, name: str) -> torch.device:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    return t.device


def rope_inv_freq(theta: float, rope_dim: int) -> np.ndarray:
    """theta^(-2 i / rope_dim), i < rope_dim / 2, in 64 bits."""
    return np.asarray(float(theta) ** (-np.arange(0, rope_dim, 2, dtype=np.float64) / rope_dim))


def qk_norm_rope(q, k, v, positions, inv_freq, *, q_weight=None, k_weight=None, eps: float = 1e-6,
                 weight_offset: float = 0.0, k_cache=None, v_cache=None, slots=None, q_out=None, k_out=None):
    """chpe_qk_norm_rope.  q [T, H, D], k and v [T, KV, D] (v may be None
    without a cache); positions [T] int32; inv_freq: 64-bit values on the host
    (numpy array or CPU tensor) or None for no rotation; slots [T] int64.
    Returns (q_out, k_out); k_out is made when there is no cache, else it is the one
    passed."""
    dev = _cuda(q, "q")
    dt = _dtype(q, "q")
    _want(q.dim() == 3 and k.dim() == 3, "q and k must be [tokens, heads, head dim]")
    T, H, D = q.shape
    KV = k.shape[1]
    qs, ks = _heads(q, "q", q.dtype, dev, T, H, D), _heads(k, "k", q.dtype, dev, T, KV, D)
    if q_out is None:
        q_out = torch.empty(T, H, D, dtype=q.dtype, device=dev)
    if k_out is None and k_cache is None:
        k_out = torch.empty(T, KV, D, dtype=q.dtype, device=dev)
    qos = _heads(q_out, "q_out", q.dtype, dev, T, H, D)
    kos = _heads(k_out, "k_out", q.dtype, dev, T, KV, D) if k_out is not None else 0
    vs, ct, rows = 0, dt, 0
    if k_cache is not None:
        _want(v is not None and v_cache is not None and slots is not None, "a cache needs v, v_cache and slots")
        vs = _heads(v, "v", q.dtype, dev, T, KV, D)
        ct = _cache(k_cache, v_cache, KV, D, dev)
        rows = k_cache.shape[0] * k_cache.shape[1]
    if inv_freq is None:
        freq, r = None, 0
    else:
        if isinstance(inv_freq, torch.Tensor):
            _want(inv_freq.device.type == "cpu", "inv_freq must be on the host")
            inv_freq = inv_freq.numpy()
        _want(inv_freq.dtype == np.float64 and inv_freq.ndim == 1 and inv_freq.flags.c_contiguous,
              "inv_freq must be a contiguous array of 64-bit values")
        freq, r = inv_freq.ctypes.data, 2 * inv_freq.shape[0]
    _check(lib().chpe_qk_norm_rope(
        q.data_ptr(), k.data_ptr(), v.data_ptr() if vs or k_cache is not None else None, dt, qs, ks, vs, T, H, KV, D,
        _vec(q_weight, "q_weight", torch.float32, D, dev), _vec(k_weight, "k_weight", torch.float32, D, dev),
        weight_offset, eps, _vec(positions, "positions", torch.int32, T, dev) if r else None, freq, r,
        q_out.data_ptr(), qos, k_out.data_ptr() if k_out is not None else None, kos,
        k_cache.data_ptr() if k_cache is not None else None, v_cache.data_ptr() if k_cache is not None else None, ct,
        rows, _vec(slots, "slots", torch.int64, T, dev) if k_cache is not None else None,
        torch.cuda.current_stream(dev).cuda_stream))
    return q_out, k_out


def attention_workspace(head_dim: int, device="cuda") -> torch.Tensor:
    """A workspace for attention_decode_paged; calls that may overlap on the GPU
    need one each."""
    n = lib().chpe_attention_decode_paged_workspace(head_dim)
    _want(n > 0, f"head_dim {head_dim} is not 64, 128 or 256")
    return torch.empty(n, dtype=torch.uint8, device=device)


def attention_decode_paged(q, k_cache, v_cache, page_table, seq_lens, *, scale: float | None = None, out=None,
                           lse=None, workspace=None):
    """chpe_attention_decode_paged.  q [B, H, D]; page_table [B, pages] int32;
    seq_lens [B] int32; scale 1/sqrt(D) unless given; lse: a float32 tensor [B, H]
    to fill, or None.  Returns out."""
    dev = _cuda(q, "q")
    dt = _dtype(q, "q")
    _want(q.dim() == 3, "q must be [batch, heads, head dim]")
    B, H, D = q.shape
    _want(k_cache.dim() == 4, "the caches must be [pages, page size, kv heads, head dim]")
    pages, page, KV, _ = k_cache.shape
    ct = _cache(k_cache, v_cache, KV, D, dev)
    qs = _heads(q, "q", q.dtype, dev, B, H, D)
    if out is None:
        out = torch.empty(B, H, D, dtype=q.dtype, device=dev)
    os_ = _heads(out, "out", q.dtype, dev, B, H, D)
    width = _rows(page_table, "page_table", torch.int32, dev, B, None)
    if lse is not None:
        _want(lse.dtype == torch.float32 and lse.shape == (B, H) and lse.is_contiguous() and lse.device == dev,
              "lse must be a contiguous float32 tensor [batch, heads]")
    if workspace is None:
        workspace = attention_workspace(D, dev)
    _want(workspace.dtype == torch.uint8 and workspace.is_contiguous() and workspace.device == dev,
          "workspace must be a contiguous uint8 tensor on q's device")
    _check(lib().chpe_attention_decode_paged(
        q.data_ptr(), dt, qs, k_cache.data_ptr(), v_cache.data_ptr(), ct, pages, page, page_table.data_ptr(),
        width, page_table.shape[1], _vec(seq_lens, "seq_lens", torch.int32, B, dev), B, H, KV, D,
        D ** -0.5 if scale is None else scale, out.data_ptr(), os_, lse.data_ptr() if lse is not None else None,
        workspace.data_ptr(), workspace.numel(), torch.cuda.current_stream(dev).cuda_stream))
    return out


def logits_process(logits, *, history=None, prompt_lens=None, total_lens=None, repetition=None, frequency=None,
                   presence=None, bias_ids=None, bias_values=None, mask=None, out=None, argmax=None,
                   want_logits: bool = True):
    """chpe_logits_process.  logits [B, V]; history [B, L] int32; lengths [B]
    int32; penalties [B] float32; bias_ids [B, n] int32 with bias_values [B, n]
    float32; mask [B, ceil(V/32)] int32 words.  A bias list or mask expanded
    over the rows (stride 0) is shared.  Returns (processed logits or None,
    winning tokens [B] int32)."""
    dev = _cuda(logits, "logits")
    dt = _dtype(logits, "logits")
    _want(logits.dim() == 2, "logits must be [batch, vocab]")
    B, V = logits.shape
    ls = _rows(logits, "logits", logits.dtype, dev, B, V)
    if out is None and want_logits:
        out = torch.empty(B, V, dtype=torch.float32, device=dev)
    os_ = _rows(out, "out", torch.float32, dev, B, V) if out is not None else 0
    if argmax is None:
        argmax = torch.empty(B, dtype=torch.int32, device=dev)
    hs = hl = bs = nb = ms = 0
    if history is not None:
        hs, hl = _rows(history, "history", torch.int32, dev, B, None), history.shape[1]
    if bias_ids is not None:
        _want(bias_values is not None, "bias_ids and bias_values go together")
        nb = bias_ids.shape[1]
        bs = _rows(bias_ids, "bias_ids", torch.int32, dev, B, None)
        _want(_rows(bias_values, "bias_values", torch.float32, dev, B, nb) == bs or B <= 1,
              "bias_ids and bias_values must have one stride")
    if mask is not None:
        ms = _rows(mask, "mask", torch.int32, dev, B, (V + 31) // 32)
    f32, i32 = torch.float32, torch.int32
    _check(lib().chpe_logits_process(
        logits.data_ptr(), dt, ls, B, V, history.data_ptr() if history is not None else None, hs, hl,
        _vec(prompt_lens, "prompt_lens", i32, B, dev), _vec(total_lens, "total_lens", i32, B, dev),
        _vec(repetition, "repetition", f32, B, dev), _vec(frequency, "frequency", f32, B, dev),
        _vec(presence, "presence", f32, B, dev), bias_ids.data_ptr() if bias_ids is not None else None,
        bias_values.data_ptr() if bias_ids is not None else None, bs, nb,
        mask.data_ptr() if mask is not None else None, ms, out.data_ptr() if out is not None else None, os_,
        _vec(argmax, "argmax", i32, B, dev), torch.cuda.current_stream(dev).cuda_stream))
    return out, argmax
