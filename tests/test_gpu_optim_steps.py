"""What the AdamW step counts and keeps: steps that were refused, left out or that a tensor had no part in,
and settings that change between steps. Runs that must agree use the same kernels on the same
values, so they are compared bit for bit."""

import pytest
import torch

from wiretorch_b200 import optim

pytestmark = pytest.mark.gpu


def tensors(sizes, dtype, seed, scale=1.0):
    gen = torch.Generator("cuda").manual_seed(seed)
    return [(torch.randn(s, device="cuda", generator=gen) * scale).to(dtype) for s in sizes]


def params_of(values):
    return [torch.nn.Parameter(v.clone()) for v in values]


def take(opt, params, grads):
    for p, g in zip(params, grads):
        p.grad = g
    opt.step()


def same_state(a, b):
    return a.keys() == b.keys() and all(torch.equal(a[k].view(torch.uint8), b[k].view(torch.uint8)) for k in a)


@pytest.mark.parametrize("dtype,bits,max_norm", [(torch.float32, 32, None), (torch.bfloat16, 32, 1.0),
                                                 (torch.float16, 8, None), (torch.float32, 8, 1.0)])  # fmt: skip
def test_a_refused_capture_leaves_nothing_behind(dtype, bits, max_norm):
    """A first step that is tried under capture makes no state: the next step is a first one."""
    values, grads = tensors([1000, (7, 9)], dtype, 1), tensors([1000, (7, 9)], dtype, 2, 0.1)
    ours, other = params_of(values), params_of(values)
    opt, ref = (optim.AdamW(ps, lr=1e-2, state_bits=bits, max_norm=max_norm) for ps in (ours, other))
    for p, g in zip(ours, grads):
        p.grad = g.clone()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    assert not opt.state and opt.steps == 0 and opt.skipped == 0 and opt.grad_norm is None
    for k in range(2):
        take(opt, ours, grads)
        take(ref, other, grads)
    for p, q in zip(ours, other):
        assert torch.equal(p, q) and same_state(opt.state[p], ref.state[q])


def left_out(opt, params, grads):
    """A step that its norm leaves out."""
    bad = [g.clone() for g in grads]
    bad[0].view(-1)[0] = float("nan")
    take(opt, params, bad)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_steps_that_were_left_out_do_not_count_without_a_limit_either(dtype):
    """Steps left out, then the limit taken off, or the state loaded by an optimiser without one, a
    group added: as if the steps that were left out had not been. An optimiser that never had a limit takes
    its corrections from the host, in 64 bits: the steps, of at most 3e-2, agree within 40 u of themselves and
    the parameter's own roundings, 3 u of it in each (u = 2^-24)."""
    values, more = tensors([1000, (7, 9)], dtype, 1), tensors([33], dtype, 3)
    grads = [tensors([1000, (7, 9), 33], dtype, 4 + k, 1e-3) for k in range(6)]

    def train(skip, limit, load):
        ps, qs = params_of(values), params_of(more)
        opt = optim.AdamW(ps, lr=1e-2, weight_decay=0.0, max_norm=limit)
        for k in range(2):
            take(opt, ps, grads[k])
            for _ in range(3 if skip else 0):
                left_out(opt, ps, grads[k])
        assert opt.skipped == (6 if skip else 0)
        if load:
            saved, held = opt.state_dict(), opt
            opt = optim.AdamW(ps, lr=1e-2, weight_decay=0.0)
            opt.load_state_dict(saved)
            assert opt.skipped == held.skipped
        opt.max_norm = None
        opt.add_param_group({"params": qs, "lr": 1e-2, "weight_decay": 0.0})
        for k in range(2, 6):
            take(opt, ps + qs, grads[k])
        return [opt.state[p].get("master", p).detach() for p in ps + qs]

    want, plain = train(False, 1e6, False), train(False, None, False)
    for load in (False, True):
        for p, w, v in zip(train(True, 1e6, load), want, plain):
            assert torch.equal(p, w)
            assert bool(((p - v).abs() <= 6 * 2.0**-24 * (40 * 3e-2 + 3 * v.abs())).all())
