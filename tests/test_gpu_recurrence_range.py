"""The gated recurrence where products of decays leave float32's range, time cut into parts:
against the definition step by step in 64 bits.

Tolerances. u = 2^-24. Every value here is one input carried through at most 40 steps (each a
product and a sum with 0, two roundings) and, in da, a product of two such: 2 x 80 + 1 roundings,
so 256 u of itself bounds it, besides the rounding of the result to its type. What is 0 in the
definition has to be 0."""

import pytest
import torch

from wiretorch_b200 import _lib, recurrence

pytestmark = pytest.mark.gpu

U = 2.0**-24
UNIT = {torch.float32: U, torch.bfloat16: 2.0**-8}


def definition(a, x, state, dh, dlast, form="decay"):
    """h, last, da, dx, dstate in 64 bits on the CPU (no starts, no lengths)."""
    a, x, state, dh, dlast = (t.detach().double().cpu() for t in (a, x, state, dh, dlast))
    f = torch.sigmoid(a) if form == "sigmoid" else a
    u = torch.sigmoid(-a) * x if form == "sigmoid" else x
    h, dx, da = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    s = state
    for t in range(x.shape[1]):
        s = h[:, t] = f[:, t] * s + u[:, t]
    adj = dlast
    for t in range(x.shape[1] - 1, -1, -1):
        tot = adj + dh[:, t]
        prev = h[:, t - 1] if t else state
        if form == "sigmoid":
            dx[:, t] = tot * torch.sigmoid(-a[:, t])
            da[:, t] = tot * f[:, t] * torch.sigmoid(-a[:, t]) * (prev - x[:, t])
        else:
            dx[:, t], da[:, t] = tot, tot * prev
        adj = tot * f[:, t]
    return h, s, da, dx, adj


def run(a, x, state, dh, dlast, form="decay"):
    leaves = [t.detach().requires_grad_(True) for t in (a, x, state)]
    h, last = recurrence.gated_scan(*leaves, form=form)
    return h, last, *torch.autograd.grad([h, last], leaves, [dh, dlast])


def check(a, x, state, dh, dlast):
    for name, got, want in zip(("h", "last", "da", "dx", "dstate"), run(a, x, state, dh, dlast), definition(a, x, state, dh, dlast)):
        unit = UNIT[got.dtype] if got.dtype != torch.float32 else 0.0
        got = got.detach().double().cpu()
        assert torch.isfinite(got).all(), name
        over = (got - want).abs() - (unit + 256 * U) * want.abs()
        assert float(over.max()) <= 0, f"{name}: over by {float(over.max())}"


SHAPES = [(8, 6000, 64), (4, 3000, 1000), (1, 32_768, 4), (2, 10_000, 17)]


def parts(B, T, N, dtype, backward):
    return _lib.lib().wt_gated_parts(B, T, N, recurrence.TYPES[dtype], backward)


@pytest.mark.parametrize("decay", [1.125, 2.0, 9.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,N", SHAPES)
def test_growing_decays_leave_zero_at_zero(B, T, N, dtype, decay):
    """Zero inputs, zero state; one spike 20 steps ahead of the end, one of the gradient 20 steps
    behind the beginning, which grow over what is left."""
    assert parts(B, T, N, dtype, 0) > 1 and parts(B, T, N, dtype, 1) > 1
    a = torch.full((B, T, N), decay, device="cuda", dtype=dtype)
    x, dh = torch.zeros_like(a), torch.zeros_like(a)
    state, dlast = (torch.zeros((B, N), device="cuda") for _ in range(2))
    check(a, x, state, dh, dlast)
    x[:, T - 20, 1:] = 1.5
    dh[:, 19, ::2] = -0.75
    check(a, x, state, dh, dlast)


@pytest.mark.parametrize("decay", [2.0, 9.0, -9.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,N", SHAPES)
def test_growth_that_a_decay_of_zero_ends(B, T, N, dtype, decay):
    """Every 150th decay is 0 (9^149 is far past the range); a spike 10 steps ahead of it and one of
    the gradient 10 steps behind it grow over those steps alone."""
    a = torch.full((B, T, N), decay, device="cuda", dtype=dtype)
    a[:, 149::150] = 0.0
    x, dh = torch.zeros_like(a), torch.zeros_like(a)
    x[:, 139::150] = 1.0
    x[:, 140::150, ::3] = -3.0
    dh[:, 10::150, 1:] = 0.5
    state, dlast = (torch.zeros((B, N), device="cuda") for _ in range(2))
    check(a, x, state, dh, dlast)


def test_a_stretch_of_growth_among_ordinary_decays():
    """Decays of 0.5 (0 ahead of the growth), then 1,000 of 1.125 which nothing enters, then 0.5 again:
    an ordinary state on both sides, forward and backward."""
    B, T, N = 4, 10_000, 260
    a = torch.full((B, T, N), 0.5, device="cuda")
    a[:, 4000:5000] = 1.125
    a[:, 3999] = a[:, 5000] = 0.0
    x, dh = torch.zeros_like(a), torch.zeros_like(a)
    x[:, 100::100], dh[:, 50::100] = 1.0, 2.0
    x[:, 3960:5000] = dh[:, 4000:5040] = 0.0
    state, dlast = torch.full((B, N), 3.0, device="cuda"), torch.full((B, N), -1.0, device="cuda")
    got, want = run(a, x, state, dh, dlast), definition(a, x, state, dh, dlast)
    for name, g, w in zip(("h", "last", "da", "dx", "dstate"), got, want):
        g = g.detach().double().cpu()
        assert torch.isfinite(g).all(), name
        # sums of up to three inputs that overlap within 100 steps of a half each; below 2^-100 nothing counts
        assert float(((g - w).abs() - 1024 * U * w.abs()).max()) <= 2.0**-100, name


@pytest.mark.parametrize("form,value", [("decay", 0.5), ("decay", -0.5), ("sigmoid", 0.0)])
@pytest.mark.parametrize("B,T,N", [(2, 6000, 64), (3, 4000, 9)])
def test_infinities_stay_where_products_of_decays_underflow(B, T, N, form, value):
    """An infinite state, input or gradient is infinite, of the definition's sign, to the end (or to the
    beginning); a decay of 0 makes it NaN. Elsewhere sums of inputs halved from step to step: below 2 in
    size, 16 u of that."""
    gen = torch.Generator("cuda").manual_seed(1)
    a = torch.full((B, T, N), value, device="cuda")
    x, dh = (torch.rand((B, T, N), device="cuda", generator=gen) for _ in range(2))
    state, dlast = (torch.rand((B, N), device="cuda", generator=gen) for _ in range(2))
    inf = float("inf")
    state[:, 0], state[:, 1] = inf, -inf
    x[:, 100, 2], x[:, 2500, 3] = inf, -inf
    dlast[:, 4], dh[:, 2700, 5] = -inf, inf
    if form == "decay":
        x[:, 50, 6], a[:, 1999, 6] = inf, 0.0
        state[:, 7], a[:, 60, 7] = inf, 0.0
    assert parts(B, T, N, a.dtype, 0) > 1 and parts(B, T, N, a.dtype, 1) > 1
    h, last, _, dx, dstate = (t.detach().double().cpu() for t in run(a, x, state, dh, dlast, form))
    rh, rlast, _, rdx, rdstate = definition(a, x, state, dh, dlast, form)
    assert torch.isinf(rh[..., :4]).any(1).all() and torch.isinf(rdx[..., 4:6]).any(1).all()
    for name, got, want in (("h", h, rh), ("last", last, rlast), ("dx", dx, rdx), ("dstate", dstate, rdstate)):
        assert torch.allclose(got, want, rtol=0.0, atol=32 * U, equal_nan=True), name


@pytest.mark.parametrize("form,cuts", [("decay", True), ("sigmoid", False)])
def test_as_many_parts_as_there_can_be(form, cuts):
    """2,048 parts of 16 steps, against the definition with the tolerances of the gated recurrence's tests."""
    import test_gpu_recurrence as general

    B, T, N = 1, 32_768, 4
    assert parts(B, T, N, torch.float32, 0) == parts(B, T, N, torch.float32, 1) == 2048
    a, x, state, dh, dlast = general.inputs(B, T, N, form, torch.float32, 3)
    starts = None
    if cuts:
        starts = torch.rand((B, T), device="cuda", generator=torch.Generator("cuda").manual_seed(2)) < 2e-4
    general.check(a, x, state, dh, dlast, form, starts=starts)
