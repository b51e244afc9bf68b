"""cafe_amd.adamw.AdamW loads its own states only (no GPU needed)."""
import pytest
import torch

from cafe_amd.adamw import AdamW


def test_adamw_refuses_other_optimizers():
    p = torch.nn.Parameter(torch.zeros(4))
    for other in (torch.optim.AdamW([p]), torch.optim.SGD([p], lr=0.1)):
        with pytest.raises(ValueError, match="not a state"):
            AdamW([p]).load_state_dict(other.state_dict())
