"""What the AdamW step counts and keeps: steps that were refused, left out or that a tensor had no part in,
and settings that change between steps. Runs that must agree use the same kernels on the same
values, so they are compared bit for bit."""

import copy

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


@pytest.mark.parametrize("dtype,bits,limit", [(torch.float32, 32, None), (torch.bfloat16, 32, 1e6), (torch.float32, 8, None),
                                              (torch.float16, 8, 1e6)])  # fmt: skip
def test_a_late_tensor_steps_as_a_new_one(dtype, bits, limit):
    """A tensor whose first gradient comes after 40 steps, two more left out where there is a limit: its
    steps are those of a new optimiser. Without a limit that one's corrections come from the host: the
    steps, of at most 3e-2, then agree within 40 u of themselves and three roundings of the parameter in each."""
    values = tensors([1000, (7, 9)], dtype, 1)
    grads = [tensors([1000, (7, 9)], dtype, 4 + k, 1e-3) for k in range(3)]
    ours, other = params_of(values), params_of(values[1:])
    opt = optim.AdamW(ours, lr=1e-2, state_bits=bits, max_norm=limit)
    for k in range(40):
        take(opt, ours[:1], grads[0][:1])
        if limit is not None and k % 20 == 0:
            left_out(opt, ours[:1], grads[0][:1])
    assert ours[1] not in opt.state
    ref = optim.AdamW(other, lr=1e-2, state_bits=bits, max_norm=limit)
    for k in range(3 if bits == 32 else 1):  # 8 bits: rounded by another step's bits from then on
        take(opt, ours, grads[k])
        take(ref, other, grads[k][1:])
        got, want = (o.state[p].get("master", p).detach() for o, p in ((opt, ours[1]), (ref, other[0])))
        if limit is None:
            assert bool(((got - want).abs() <= (k + 1) * 2.0**-24 * (40 * 3e-2 + 3 * want.abs())).all())
        else:
            assert torch.equal(got, want)


def test_a_late_tensor_is_saved_and_copied_with_its_count():
    """Tensors that began at the first step, at the fourth and, after a save, at the sixth, steps left out
    in between: the loaded and the copied optimiser go on as the one that was saved."""
    sizes = [300, 40, (3, 5)]
    values = tensors(sizes, torch.float32, 1)
    grads = [tensors(sizes, torch.float32, 4 + k, 1e-3) for k in range(8)]
    ours = params_of(values)
    opt = optim.AdamW(ours, lr=1e-2, max_norm=1e6)
    for k in range(5):
        take(opt, ours[: 1 if k < 3 else 2], grads[k])
        if k in (1, 3):
            left_out(opt, ours[: 1 if k < 3 else 2], grads[k])
            ours[1].grad = None if k < 3 else ours[1].grad
    assert [int(opt.state[p]["before"]) if "before" in opt.state[p] else 0 for p in ours[:2]] == [0, 3]
    saved = copy.deepcopy(opt.state_dict())
    theirs = [torch.nn.Parameter(p.detach().clone()) for p in ours]
    other = optim.AdamW(theirs, lr=1e-2, max_norm=1e6)
    other.load_state_dict(saved)
    copies, third = copy.deepcopy((ours, opt))
    for k in range(5, 8):
        for o, ps in ((opt, ours), (other, theirs), (third, copies)):
            take(o, ps, grads[k])
    for p, q, r in zip(ours, theirs, copies):
        assert torch.equal(p, q) and torch.equal(p, r)
    assert int(opt.state[ours[2]]["before"]) == 5
    # the third tensor against a new optimiser's
    new = params_of(values[2:])
    ref = optim.AdamW(new, lr=1e-2, max_norm=1e6)
    for k in range(5, 8):
        take(ref, new, grads[k][2:])
    assert torch.equal(new[0], ours[2])


def test_groups_that_were_used_before_and_states_that_count_by_group():
    """The groups of another optimiser start a new one at its first step; a state that was saved with the
    step at which a group was added counts from there."""
    values = tensors([100, 50], torch.float32, 1)
    grads = tensors([100, 50], torch.float32, 2, 1e-3)
    ps = params_of(values)
    opt = optim.AdamW(ps[:1], lr=1e-2)
    for _ in range(5):
        take(opt, ps[:1], grads[:1])
    opt.add_param_group({"params": ps[1:]})
    for _ in range(3):
        take(opt, ps, grads)
    saved = copy.deepcopy(opt.state_dict())
    del saved["state"][1]["before"]
    saved["param_groups"][0]["born"], saved["param_groups"][1]["born"] = 0, 5
    theirs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    other = optim.AdamW([{"params": theirs[:1]}, {"params": theirs[1:]}], lr=1e-2)
    other.load_state_dict(saved)
    new = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    again = optim.AdamW([{**group, "params": [q], "born": 5} for group, q in zip(other.param_groups, new)])
    ref = optim.AdamW([torch.nn.Parameter(p.detach().clone()) for p in ps], lr=1e-2)
    for o in (opt, other, again, ref):
        take(o, [p for group in o.param_groups for p in group["params"]], grads)
    for p, q in zip(ps, theirs):
        assert torch.equal(p, q)
    for p, q in zip(new, ref.param_groups[0]["params"]):
        assert torch.equal(p, q)


def test_settings_that_change_between_steps_are_taken():
    """A group's dict put in the place of another with other rates, betas changed within their list."""
    values = tensors([300], torch.float32, 1)
    grads = [tensors([300], torch.float32, 4 + k, 1e-3) for k in range(4)]
    (p,), (q,) = params_of(values), params_of(values)
    opt = optim.AdamW([p], lr=1e-2, betas=[0.9, 0.999])
    ref = optim.AdamW([q], lr=1e-2, betas=(0.9, 0.999))
    for k in range(4):
        if k == 1:
            opt.param_groups[0] = {**opt.param_groups[0], "lr": 1e-3, "weight_decay": 0.5}
            ref.param_groups[0].update(lr=1e-3, weight_decay=0.5)
        if k == 2:
            opt.param_groups = [dict(group, lr=0.0) for group in opt.param_groups]
            ref.param_groups[0]["lr"] = 0.0
        if k == 3:
            opt.param_groups[0]["lr"] = ref.param_groups[0]["lr"] = 1e-2
            opt.param_groups[0]["betas"][0] = 0.5
            ref.param_groups[0]["betas"] = (0.5, 0.999)
        take(opt, [p], grads[k])
        take(ref, [q], grads[k])
        assert torch.equal(p, q), k


def test_tensors_without_a_gradient_keep_their_numbers():
    """What the 8-bit rounding numbers an element by includes the tensors ahead that have no gradient: one
    of another size in their place, and the numbers follow."""
    (v, g) = tensors([500, 500], torch.float32, 1)
    ahead = tensors([300, 900], torch.float32, 2)
    p = torch.nn.Parameter(v.clone())
    first, second = params_of(ahead)
    opt = optim.AdamW([first, p], state_bits=8)
    take(opt, [p], [g])
    q = torch.nn.Parameter(p.detach().clone())
    ref = optim.AdamW([second, q], state_bits=8)
    ref.state[q] = {k: t.clone() for k, t in opt.state[p].items()}
    ref.steps = 1
    opt.param_groups[0]["params"][0] = second
    take(opt, [p], [g])
    take(ref, [q], [g])
    assert torch.equal(p, q) and same_state(opt.state[p], ref.state[q])
