"""CPU: what the norm + rotation and the 8-bit cache refuse or trace, on tensors without data."""

import pytest
import torch


def test_a_table_that_wants_gradients_is_refused():
    """No backward pass: like the rows and weights, the table must not be left without its gradient in silence."""
    from waminfer_b200.rope import qk_norm_rope

    q, w = torch.zeros(1, 4, 256, dtype=torch.bfloat16), torch.ones(128, dtype=torch.bfloat16)
    rope = torch.zeros(4, 64, dtype=torch.complex64, requires_grad=True)
    with pytest.raises(RuntimeError, match="backward"):
        qk_norm_rope(q, None, w, None, rope, None, 2)
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
        qk_norm_rope(q, None, w, None, rope, None, 2)
