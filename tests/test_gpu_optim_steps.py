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
