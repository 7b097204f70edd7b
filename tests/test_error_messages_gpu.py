"""A refusal whose message holds numbers is an exception, not the end of the process."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_numbers_in_messages():
    from vagus_b200.ops import native
    a, b, c = (torch.zeros(s, device="cuda", dtype=torch.bfloat16) for s in ((128, 64), (128, 72), (128, 128)))
    with pytest.raises(RuntimeError, match="K mismatch .64 vs 72"):
        native().gemm(a, False, b, False, c, None, 1.0, 0.0, False, 0, 0)
    x = torch.zeros(1, 1, 1, 2, device="cuda")
    with pytest.raises(ValueError, match="R <= 2"):
        native().rotary(x, None, None, 0, torch.zeros(2, device="cuda"), True, 1.0, 1.0)
