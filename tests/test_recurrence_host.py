"""Refusals on the way to the kernels that need no GPU."""

import ctypes

import pytest
import torch

from wiretorch_b200 import _lib, build, recurrence


def test_what_is_not_three_dimensional_is_refused_whatever_comes_with_it():
    x = torch.zeros((4, 5))
    more = [{}, {"lengths": torch.ones(4, dtype=torch.int64)}, {"lengths": torch.ones(4, dtype=torch.int32)},
            {"starts": torch.zeros((4, 5), dtype=torch.bool)}, {"state": torch.zeros((4, 5))}]  # fmt: skip
    for kw in more:
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            recurrence.gated_scan(x, x, **kw)


def test_a_device_that_is_not_a_gpu_has_no_stream():
    for device in ("cpu", torch.device("cpu"), torch.device("cpu", 0), "meta"):
        with pytest.raises(ValueError, match="no CUDA stream"):
            _lib.stream_of(device)


def test_sizes_past_the_kernels_numbers_are_refused():
    build.build()
    lib = _lib.lib()
    for cls, call in ((recurrence._Scan, lib.wt_gated_scan), (recurrence._Grad, lib.wt_gated_grad), (recurrence._Step, lib.wt_gated_step)):
        for name in ("B", "N"):
            for size in (recurrence.MOST + 1, (1 << 31) - 1):
                s = cls(B=1, N=1)
                setattr(s, name, size)
                assert call(ctypes.byref(s), None) == _lib.ERR_ARGS
                assert b"bad recurrence" in lib.wt_last_error()
    assert lib.wt_gated_parts(1, 10_000, (1 << 31) - 1, 0, 0) == 1
