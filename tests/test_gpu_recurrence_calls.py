"""How the gated recurrence is called: refusals, what it keeps and what it allocates."""

import pytest
import torch

from wiretorch_b200 import recurrence

pytestmark = pytest.mark.gpu


def test_dimensions_are_refused_whatever_comes_with_them():
    for shape in ((5,), (4, 5), (2, 3, 4, 5)):
        x = torch.zeros(shape, device="cuda")
        for kw in ({}, {"lengths": torch.ones(shape[0], dtype=torch.int64, device="cuda")},
                   {"starts": torch.zeros(shape[:2], dtype=torch.bool, device="cuda")}):  # fmt: skip
            with pytest.raises(ValueError, match="dimensions"):
                recurrence.gated_scan(x, x, **kw)
