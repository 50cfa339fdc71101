"""What the gradient of windows does not take is told by the call that it belongs to, not by the backward pass: no GPU needed."""
import pytest
import torch

from lapis_amd import attention


@pytest.mark.parametrize("leaf", [0, 1, 2])
def test_too_many_queries_for_a_gradient(leaf):
    q = torch.zeros((1, 1, 1, 8), dtype=torch.bfloat16).expand(1, 2 ** 23, 128, 8)
    k, v = (torch.zeros((1, 9, 2, 8), dtype=torch.bfloat16) for _ in range(2))
    operands = [q, k, v]
    operands[leaf].requires_grad_()
    with pytest.raises(ValueError, match="8388608 queries of 64 heads"):
        attention.attend_window(*operands, 3)
