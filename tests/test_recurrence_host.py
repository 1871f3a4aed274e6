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


def threads_held(N, kind, backward):
    """Of the threads that walk the columns of a trial's rows: how many a trial takes, and how many the GPU holds at
    once: blocks of 256 for rows that four elements divide, else of 128 (a warp for 128 columns), as
    many as an SM's 227 KB take of their slots (16 operands' steps a stage of 8 steps: two stages of 4-byte
    elements or of three operands, else three; a sixteenth and 1 KB on top), at most 1,024 threads an SM."""
    wide, ops, size = N % 4 == 0, 3 if backward else 2, 2 if kind else 4
    block = 256 if wide else 128
    stage = ops * 8 * block * 4 * size
    blocks = (227 << 10) // ((2 if size == 4 or ops == 3 else 3) * stage * 17 // 16 + 1024)
    return N // 4 if wide else -(-N // 128) * 32, 148 * min(blocks * block, 1024)


@pytest.mark.parametrize("kind", [0, 1, 2])
@pytest.mark.parametrize("backward", [0, 1])
def test_parts_fill_the_gpu_and_no_more(kind, backward):
    build.build()
    lib = _lib.lib()
    assert threads_held(256, kind, backward)[1] == (75_776 if kind else 37_888)
    assert threads_held(333, kind, backward)[1] == (75_776 if kind else 37_888 if backward else 56_832)
    for B in (1, 2, 5, 32, 64, 1000):
        for T in (63, 64, 100, 500, 1237, 10_000, 131_072, 1 << 30):
            for N in (1, 4, 17, 33, 64, 256, 333, 1000, 20_000, 20_001):
                parts = lib.wt_gated_parts(B, T, N, kind, backward)
                columns, held = threads_held(N, kind, backward)
                asked = min(held // (B * columns), T // 16, 2048)
                if T < 64 or asked < 2:
                    assert parts == 1
                    continue
                steps = -(-(-(-T // asked)) // 8) * 8  # whole tiles
                assert parts == -(-T // steps) and 2 <= parts <= asked
                assert B * parts * columns <= held


def test_parts_of_named_cases():
    build.build()
    parts = _lib.lib().wt_gated_parts
    for backward in (0, 1):
        assert parts(32, 10_000, 256, 1, backward) == 37 and parts(32, 10_000, 256, 0, backward) == 18
        assert parts(1, 131_072, 64, 0, backward) == 2048 and parts(1, 32_768, 4, 0, backward) == 2048
        assert parts(5, 1237, 333, 2, backward) == 52
        assert parts(64, 500, 20_000, 0, backward) == 1
