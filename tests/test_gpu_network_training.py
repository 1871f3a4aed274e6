"""Both training operators on the network's own parts: a loss behind a gated recurrence over its spikes,
through the engine's backward pass, stepped by AdamW on its scales and per-synapse weights.

Tolerances. The gradient that enters the engine is a sum over at most T steps of float32 products, by the
kernel's order or by the loop's: T x 4 u of its largest value (u = 2^-24); what leaves the engine is linear
in it, and is compared like the engine's gradients elsewhere, to 1e-3 of the largest entry."""

import pytest
import torch

import golden_io
from wiretorch_b200 import engine, optim, recurrence

pytestmark = pytest.mark.gpu

NAMES = [n for n in golden_io.cases() if n in ("recurrent_learnt_weights", "recurrent_gradients", "feedforward_learnt_weights")]


class Network:
    """A golden case with its scales and weights as parameters."""

    def __init__(self, name):
        drive, self.p, d, meta = golden_io.load(name, "cuda")
        T = meta["grad_steps"]
        self.x = torch.from_numpy(d["in.x"][:, :T]).cuda()
        self.drive, made = drive, {}
        drive.scale = torch.nn.Parameter(drive.scale.detach().clone())
        for part in ("recurrent", "feedforward"):
            pairs = [(r, made.setdefault(id(W), torch.nn.Parameter(W.detach().clone()))) for r, W in getattr(drive, part)]
            setattr(drive, part, pairs)
        self.weights = list(made.values())
        self.kw = {key: torch.from_numpy(d[f"in.{key}"]).cuda() for key in ("refractory", "gating", "adaptation") if f"in.{key}" in d}
        self.v, self.g = torch.from_numpy(d["in.v"]).cuda(), torch.from_numpy(d["in.g"]).cuda()

    def spikes(self):
        return engine.simulate(self.v, self.g, self.x, self.drive, self.p, **self.kw).output

    def parameters(self):
        return [self.drive.scale, *self.weights]


def loop(a, x):
    h, out = torch.zeros_like(x[:, 0]), []
    for t in range(x.shape[1]):
        h = a * h + x[:, t]
        out.append(h)
    return torch.stack(out, 1)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("name", NAMES)
def test_a_filtered_loss_trains_the_network(name, bits):
    net = Network(name)
    N = net.v.shape[1]
    decay = torch.nn.Parameter(torch.full((N,), 0.9, device="cuda"))
    params = [*net.parameters(), decay]
    target = torch.rand((N,), device="cuda", generator=torch.Generator("cuda").manual_seed(0))
    grads = []
    for filtered in (lambda s: recurrence.gated_scan(decay, s)[0], lambda s: loop(decay, s)):
        for p in params:
            p.grad = None
        (filtered(net.spikes()) - target).square().mean().backward()
        grads.append([None if p.grad is None else p.grad.clone() for p in params])
    assert any(float(g.abs().max()) > 0 for g in grads[0][:-1] if g is not None)
    for got, want, p in zip(*grads, params):
        assert (got is None) == (want is None)
        if got is not None:
            there = p.detach() != 0
            assert float((got - want)[there].abs().max()) <= 1e-3 * max(float(want[there].abs().max()), 1e-12)
    # a step, and what the engine makes of the stepped tensors: what it makes of copies of them
    before = [p.detach().clone() for p in params]
    for p, g in zip(params, grads[0]):
        p.grad = g
    optim.AdamW(params, lr=1e-2, state_bits=bits, weight_decay=0.0, max_norm=1.0).step()
    for p, b, g in zip(params, before, grads[0]):
        assert torch.equal(p, b) == (g is None or not bool(g.any()))
    with torch.no_grad():
        stepped = net.spikes()
        copies = {id(p): torch.nn.Parameter(p.detach().clone()) for p in net.parameters()}
        net.drive.scale = copies[id(net.drive.scale)]
        for part in ("recurrent", "feedforward"):
            setattr(net.drive, part, [(r, copies[id(W)]) for r, W in getattr(net.drive, part)])
        assert torch.equal(stepped, net.spikes())
