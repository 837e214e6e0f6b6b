"""The torch layer's refusals that need no GPU."""
import pytest

torch = pytest.importorskip("torch")


def test_a_gradient_that_autograd_expects_is_refused():
    from chpe_qwen_engine_b200 import ops
    x = torch.zeros(2, 8, requires_grad=True)
    with pytest.raises(ValueError, match="logits requires a gradient"):
        ops.logits_process(x)
    with pytest.raises(ValueError, match="q requires a gradient"):
        ops.attention_decode_paged(x, None, None, None, None)
    with pytest.raises(ValueError, match="q requires a gradient"):
        ops.qk_norm_rope(x, None, None, None, None)
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
        ops.logits_process(x)
    with pytest.raises(ValueError, match="CUDA"):
        ops.logits_process(x.detach())
