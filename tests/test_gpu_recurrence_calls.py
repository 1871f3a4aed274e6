"""How the gated recurrence is called: refusals, what it keeps and what it allocates."""

import pytest
import torch

from wiretorch_b200 import _lib, recurrence

pytestmark = pytest.mark.gpu


def test_dimensions_are_refused_whatever_comes_with_them():
    for shape in ((5,), (4, 5), (2, 3, 4, 5)):
        x = torch.zeros(shape, device="cuda")
        for kw in ({}, {"lengths": torch.ones(shape[0], dtype=torch.int64, device="cuda")},
                   {"starts": torch.zeros(shape[:2], dtype=torch.bool, device="cuda")}):  # fmt: skip
            with pytest.raises(ValueError, match="dimensions"):
                recurrence.gated_scan(x, x, **kw)


@pytest.mark.parametrize("which", ["scalar", "1", "B11", "N", "every other"])
def test_a_broadcast_decay_is_not_written_out(which):
    """A call with a decay that is one value, one a trial or one a neuron takes no memory beyond its results
    (and keeps none beside x and h for the backward pass), a decay read with a stride that of its own size."""
    B, T, N = 8, 50, 20_000
    x = torch.rand((B, T, N), device="cuda")
    a = torch.rand({"scalar": (), "1": (1,), "B11": (B, 1, 1), "N": (N,), "every other": (2 * N,)}[which], device="cuda")
    a = (a[::2] if which == "every other" else a).requires_grad_(True)
    size, rows = 4 * B * T * N, 4 * B * N
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    h, last = recurrence.gated_scan(a, x)
    assert torch.cuda.max_memory_allocated() - before <= size + 4 * rows + (1 << 21)
    want, end = recurrence.gated_scan(a.detach().expand(B, T, N).contiguous(), x)
    assert torch.equal(h, want) and torch.equal(last, end)
    (da,) = torch.autograd.grad(last.sum(), a)
    assert da.shape == a.shape and bool(torch.isfinite(da).all())
    state = torch.zeros((B, N), device="cuda")
    step = recurrence.gated_step(a.detach().expand(B, 1, N)[:, 0] if which == "B11" else a.detach(), x[:, 0], state)
    assert torch.equal(step, h[:, 0].detach())


def test_decays_that_do_not_expand_are_refused():
    x = torch.zeros((2, 3, 4), device="cuda")
    for shape in ((5,), (3, 3, 1), (2, 2, 4), (1, 2, 3, 4), (2, 3, 0)):
        with pytest.raises(ValueError, match="expand"):
            recurrence.gated_scan(torch.zeros(shape, device="cuda"), x)
    with pytest.raises(ValueError, match="expand"):  # x smaller than a
        recurrence.gated_scan(torch.zeros((2, 3, 4), device="cuda"), x[..., :1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("form", ["decay", "sigmoid"])
def test_h_may_be_changed_in_place_where_the_backward_pass_does_not_read_it(dtype, form):
    """Chunks of at most 8 steps, and 16-bit ones of any length."""
    for T in (1, 5, 8, 9, 200):
        a, x = (torch.rand((3, T, 10), device="cuda").to(dtype).requires_grad_(True) for _ in range(2))
        state = torch.rand((3, 10), device="cuda", requires_grad=True)
        grads = []
        for change in (False, True):
            h, last = recurrence.gated_scan(a, x, state, form=form)
            out = (h.mul_(0.5) if change else h * 0.5).float().sum() + last.sum()
            if change and T > 8 and dtype == torch.float32:
                with pytest.raises(RuntimeError, match="inplace operation"):
                    torch.autograd.grad(out, [a, x, state])
            else:
                grads.append(torch.autograd.grad(out, [a, x, state]))
        assert all(torch.equal(p, q) for p, q in zip(grads[0], grads[-1]))


def test_the_current_stream_of_a_device_by_every_name():
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for device in (0, None, "cuda", "cuda:0", torch.device("cuda"), torch.device("cuda", 0), side.device):
            assert _lib.stream_of(device) == side.cuda_stream


def test_sizes_past_the_kernels_numbers_are_refused():
    """Sizes that 32 bits would cut: broadcast inputs, so that nothing of the size is ever held."""
    one = torch.zeros((1, 1, 1), device="cuda")
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    for shape in ((2**32 + 8, 1, 1), (1, 1, 2**32 + 8), (2**31 - 255, 1, 1), (1, 1, 2**31 - 255), (1, 2**30 + 1, 1)):
        with pytest.raises(ValueError, match="at most"):
            recurrence.gated_scan(one[0, 0, 0], one.expand(shape))
        if shape[1] == 1:
            x = one.expand(shape)[:, 0]
            with pytest.raises(ValueError, match="at most"):
                recurrence.gated_step(one[0, 0, 0], x, x)
    assert torch.cuda.max_memory_allocated() == before
