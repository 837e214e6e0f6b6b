"""The operators of a batched decode step on torch CUDA tensors: q/k norm with
rotation and cache append (chpe_qk_norm_rope), paged decode attention
(chpe_attention_decode_paged) and the logits rules (chpe_logits_process).

include/chpe.h states what each computes and what it refuses.  The functions
(native, csrc/ops_torch.cpp) take shapes, strides and types from the tensors,
check that they fit together, run on the current stream of the tensors' device
(which need not be the current device), and raise ChpeError for what the
library refuses and ValueError for tensors that do not fit.  They have no
gradients: where gradients are recorded, tensors that require one are refused.
Nothing is allocated when the outputs and the workspace are passed.  A cache is a pair of
contiguous tensors [num_pages, page_size, num_kv_heads, head_dim].
"""
from __future__ import annotations

import numpy as np
import torch  # loads the libraries _ops is linked with

from . import lib

try:
    from ._ops import attention_decode_paged, logits_process, qk_norm_rope
except ImportError as e:
    raise RuntimeError(f"chpe_qwen_engine_b200/_ops is missing or does not load ({e}): "
                       "run python -m chpe_qwen_engine_b200.build") from e

__all__ = ["attention_decode_paged", "attention_workspace", "logits_process", "qk_norm_rope", "rope_inv_freq"]


def rope_inv_freq(theta: float, rope_dim: int) -> np.ndarray:
    """theta^(-2 i / rope_dim), i < rope_dim / 2, in 64 bits."""
    return float(theta) ** (-np.arange(0, rope_dim, 2, dtype=np.float64) / rope_dim)


def attention_workspace(head_dim: int, device="cuda") -> torch.Tensor:
    """A workspace for attention_decode_paged; calls that may overlap on the GPU
    need one each."""
    n = lib().chpe_attention_decode_paged_workspace(head_dim)
    if n == 0:
        raise ValueError(f"head_dim {head_dim} is not 64, 128 or 256")
    return torch.empty(n, dtype=torch.uint8, device=device)
