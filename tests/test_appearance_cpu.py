"""AppearanceHead's refusals that need no GPU."""
from __future__ import annotations

import pytest
import torch

from msplat_amd.appearance import AppearanceHead


def test_training_in_float16_is_refused():
    """Its gradients vanish: at a view of 1297 x 840 all but the output layer's are 0."""
    head = AppearanceHead(1, dtype=torch.float16, device="cpu")
    view = torch.zeros(4, 5, 3)
    with pytest.raises(ValueError, match="float16"):
        head(view, 0, training=True)
    before = [p.detach().clone() for p in head.parameters()]
    with pytest.raises(ValueError, match="float16"):
        head.fit([view], [view], steps=1)
    assert head.step == 0 and all(torch.equal(p, q) for p, q in zip(before, head.parameters()))
