"""Refusals of the gated recurrence that need no GPU."""

import pytest
import torch

from wiretorch_b200 import recurrence


def test_what_is_not_three_dimensional_is_refused_whatever_comes_with_it():
    x = torch.zeros((4, 5))
    more = [{}, {"lengths": torch.ones(4, dtype=torch.int64)}, {"lengths": torch.ones(4, dtype=torch.int32)},
            {"starts": torch.zeros((4, 5), dtype=torch.bool)}, {"state": torch.zeros((4, 5))}]  # fmt: skip
    for kw in more:
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            recurrence.gated_scan(x, x, **kw)
