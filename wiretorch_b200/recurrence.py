"""A gated linear recurrence over trains ``(B, T, N)``, with its gradients.

``filtering.double_exponential`` filters with decays that are constants of the program; here
they are data. In the decay form ``h_t = a_t h_{t-1} + x_t``, ``a`` given per trial, step and
neuron, or learnt per neuron (a time constant); in the sigmoid form ``f_t = sigmoid(a_t)``,
``h_t = f_t h_{t-1} + (1 - f_t) x_t``, ``a`` the logits. The reference has the recurrence with
one decay for all steps, without gradients to it (``utils/recurrences.py:7-43``
``ar1_trajectory``).

``gated_scan`` runs whole chunks and carries the state from one to the next (as the reference's
filters do, ``training_utils/filtering.py:28-48``), trials of different lengths and trials
packed behind one another included; ``gated_step`` advances one step in place, for closed loops.
"""

from __future__ import annotations

import torch

from wiretorch_b200 import _lib

_C = _lib.C
SEGMENT = 8  # WT_GATED_SEGMENT: steps between the states saved for the backward pass
TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # WT_F32, WT_BF16, WT_F16
FORMS = {"decay": 0, "sigmoid": 1}
MOST, MOST_STEPS = (1 << 31) - 256, 1 << 30  # trials or columns, and steps, of a call


class _Scan(_C.Structure):
    _fields_ = [
        ("B", _C.c_int32), ("T", _C.c_int32), ("N", _C.c_int32), ("type", _C.c_int32), ("form", _C.c_int32),
        ("a", _lib.P), ("a_b", _C.c_int64), ("a_t", _C.c_int64),
        ("x", _lib.P), ("x_b", _C.c_int64), ("x_t", _C.c_int64),
        ("state", _lib.P), ("starts", _lib.P), ("lengths", _lib.P),
        ("h", _lib.P), ("last", _lib.P), ("saved", _lib.P), ("scratch", _lib.P),
    ]  # fmt: skip


class _Grad(_C.Structure):
    _fields_ = [
        ("B", _C.c_int32), ("T", _C.c_int32), ("N", _C.c_int32), ("type", _C.c_int32), ("form", _C.c_int32),
        ("reduce", _C.c_int32), ("da_type", _C.c_int32),
        ("a", _lib.P), ("a_b", _C.c_int64), ("a_t", _C.c_int64),
        ("x", _lib.P), ("x_b", _C.c_int64), ("x_t", _C.c_int64),
        ("state", _lib.P), ("starts", _lib.P), ("lengths", _lib.P), ("h", _lib.P), ("saved", _lib.P),
        ("dh", _lib.P), ("dh_b", _C.c_int64), ("dh_t", _C.c_int64), ("dlast", _lib.P),
        ("da", _lib.P), ("dx", _lib.P), ("dstate", _lib.P), ("scratch", _lib.P),
    ]  # fmt: skip


class _Step(_C.Structure):
    _fields_ = [
        ("B", _C.c_int32), ("N", _C.c_int32), ("type", _C.c_int32), ("form", _C.c_int32),
        ("a", _lib.P), ("a_b", _C.c_int64), ("x", _lib.P), ("x_b", _C.c_int64),
        ("state", _lib.P), ("h", _lib.P),
    ]  # fmt: skip


def _form(form):
    if form not in FORMS:
        raise ValueError(f"form must be one of {sorted(FORMS)}, not {form!r}")
    return FORMS[form]


def _checked(a, x, dims):
    """``a`` expanded to ``x``'s shape, both with unit (or copied to unit) last stride."""
    if not x.is_cuda:
        raise RuntimeError("wiretorch_b200 runs on CUDA tensors only (no CPU path)")
    if x.dim() != dims:
        raise ValueError(f"x must have {dims} dimensions, not {tuple(x.shape)}")
    if x.dtype not in TYPES:
        raise TypeError(f"the recurrence takes float32, bfloat16 and float16, not {x.dtype}")
    if a.dtype != x.dtype or a.device != x.device:
        raise TypeError(f"a and x must have one type and device: {a.dtype} on {a.device}, {x.dtype} on {x.device}")
    if a.shape == x.shape:
        return _unit(a), _unit(x)
    try:  # rows are written out before they are broadcast over trials and time
        row = _unit(a.expand(*a.shape[:-1], x.shape[-1]))
        return row.expand(x.shape), _unit(x)
    except RuntimeError:
        raise ValueError(f"a of shape {tuple(a.shape)} does not expand to x's {tuple(x.shape)}") from None


def _unit(t):
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _too_large(x):
    return ValueError(f"a call takes at most {MOST} trials or columns and {MOST_STEPS} steps, not {tuple(x.shape)}")


def _per_trial(name, t, shape, dtypes, x):
    if t is None:
        return None
    if t.dtype not in dtypes or t.device != x.device or tuple(t.shape) != shape:
        raise ValueError(f"{name} must be of shape {shape}, {' or '.join(str(d) for d in dtypes)}, on {x.device}")
    return t


def _at(t):
    return None if t is None else t.data_ptr()


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, a, x, state, starts, lengths, form, want_grad):
        given = a.shape
        a, x = _checked(a, x, 3)
        B, T, N = x.shape
        lib, kind, dev = _lib.lib(), TYPES[x.dtype], x.device
        h = torch.empty_like(x, memory_format=torch.contiguous_format)
        last = torch.empty((B, N), device=dev) if state is None else torch.empty_like(state)
        # the states that enter each segment (kept for the backward pass), then the call's scratch
        saves = B * -(-T // SEGMENT) * N if want_grad and kind and T > SEGMENT else 0
        need = saves + (lib.wt_gated_scratch_bytes(B, T, N, kind, 0) + 3) // 4
        work = torch.empty(need, device=dev) if need else None
        at = _at(work)
        s = _Scan(B, T, N, kind, form, a.data_ptr(), a.stride(0), a.stride(1), x.data_ptr(), x.stride(0), x.stride(1),
                  _at(state), _at(starts), _at(lengths), h.data_ptr(), last.data_ptr(),
                  at if saves else None, at + 4 * saves if need > saves else None)  # fmt: skip
        with _lib.timed("wt_gated_scan"):
            rc = lib.wt_gated_scan(_C.byref(s), _C.c_void_p(_lib.stream_of(x.get_device())))
        if rc:
            _lib.check(rc, "wt_gated_scan")
        _lib.count_launches(1)
        if want_grad:
            # a chunk of one segment needs neither h nor saved states
            ctx.save_for_backward(a, x, state, starts, lengths, work if saves else h if T > SEGMENT else None)
            ctx.form, ctx.given, ctx.from_h = form, given, not saves
        return h, last

    @staticmethod
    def backward(ctx, dh, dlast):
        if torch.is_grad_enabled():
            raise RuntimeError("gated_scan has no second derivatives (create_graph)")
        a, x, state, starts, lengths, kept = ctx.saved_tensors
        B, T, N = x.shape
        lib, kind, dev, given = _lib.lib(), TYPES[x.dtype], x.device, ctx.given
        dh = _unit(dh if dh.dtype == x.dtype else dh.to(x.dtype))
        dlast = dlast.float().contiguous()
        # a without a time axis: its gradient summed over time where it is made
        reduce = T > 1 and (len(given) < 2 or given[-2] == 1)
        dx = torch.empty_like(x, memory_format=torch.contiguous_format)
        if reduce:
            da = torch.empty((B, lib.wt_gated_parts(B, T, N, kind, 1), N), device=dev)
        else:
            da = dx.new_empty(dx.shape, dtype=torch.float32) if given != x.shape else torch.empty_like(dx)
        dstate = torch.empty_like(dlast) if ctx.needs_input_grad[2] else None
        size = lib.wt_gated_scratch_bytes(B, T, N, kind, 1)
        scratch = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
        h, saved = (_at(kept), None) if ctx.from_h else (None, _at(kept))
        s = _Grad(B, T, N, kind, ctx.form, reduce, TYPES[da.dtype],
                  a.data_ptr(), a.stride(0), 0 if reduce else a.stride(1), x.data_ptr(), x.stride(0), x.stride(1),
                  _at(state), _at(starts), _at(lengths), h, saved, dh.data_ptr(), dh.stride(0), dh.stride(1),
                  dlast.data_ptr(), da.data_ptr(), dx.data_ptr(), _at(dstate), _at(scratch))  # fmt: skip
        with _lib.timed("wt_gated_grad"):
            rc = lib.wt_gated_grad(_C.byref(s), _C.c_void_p(_lib.stream_of(x.get_device())))
        if rc:
            _lib.check(rc, "wt_gated_grad")
        _lib.count_launches(1)
        if given != x.shape:
            da = (da.sum(1, keepdim=True) if reduce else da).sum_to_size(given).to(x.dtype)
        return da, dx, dstate, None, None, None, None


def gated_scan(a, x, state=None, *, form="decay", starts=None, lengths=None):
    """``(h, last)``: the recurrence over a chunk ``x`` ``(B, T, N)`` (float32, bfloat16 or
    float16), ``h`` of ``x``'s shape and type, ``last`` ``(B, N)`` float32 the state after it.

    ``a``: of ``x``'s type, its shape or one that expands to it (``(N,)``: a decay per neuron,
    constant in time). Any strides; a chunk cut from a larger tensor is read in place as long
    as its last dimension has unit stride. ``state`` ``(B, N)`` float32 enters (zero without).
    ``starts`` ``(B, T)`` bool: steps that begin a new trial, which take the state as 0.
    ``lengths`` ``(B,)`` int32 or int64: a trial's steps from its length on (held to 0..T) have
    ``h`` 0, keep the state and get no gradient, whatever they contain.

    Gradients flow to ``a``, ``x`` and ``state`` (detach it between chunks to truncate), first
    ones only; the state and the sums are float32, each result rounded once. Decays of size up to
    about 1 are what it is for: where some are larger, the product of the decays over any stretch
    of time has to stay in float32's range, or the state that enters the stretch has to be 0. An
    infinite decay gives an infinity or NaN."""
    code = _form(form)
    if x.is_cuda and x.get_device() != torch.cuda.current_device():
        with torch.cuda.device(x.get_device()):
            return gated_scan(a, x, state, form=form, starts=starts, lengths=lengths)
    if x.dim() == 3:
        B, T, N = x.shape
        if B > MOST or N > MOST or T > MOST_STEPS:
            raise _too_large(x)
        if state is not None and (state.dtype != torch.float32 or state.device != x.device or tuple(state.shape) != (B, N)):
            raise ValueError(f"state must be float32 of shape {(B, N)} on {x.device}")
        starts = _per_trial("starts", starts, (B, T), (torch.bool,), x)
        lengths = _per_trial("lengths", lengths, (B,), (torch.int32, torch.int64), x)
        if state is not None:
            state = state.contiguous()
        if starts is not None:
            starts = starts.contiguous()
        if lengths is not None:
            lengths = (lengths if lengths.dtype == torch.int32 else lengths.clamp(0, T).int()).contiguous()
    want = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (a, x, state))
    return _GatedScan.apply(a, x, state, starts, lengths, code, want)


def gated_step(a, x, state, *, form="decay"):
    """One step: advances ``state`` ``(B, N)`` float32 in place and returns ``h`` ``(B, N)``, its
    value in the type of ``x`` ``(B, N)``. ``a`` as in ``gated_scan``. No gradient."""
    code = _form(form)
    if x.is_cuda and x.get_device() != torch.cuda.current_device():
        with torch.cuda.device(x.get_device()):
            return gated_step(a, x, state, form=form)
    if torch.is_grad_enabled() and (a.requires_grad or x.requires_grad or state.requires_grad):
        raise RuntimeError("gated_step has no gradient: use gated_scan, or call it under torch.no_grad()")
    if x.dim() == 2:
        B, N = x.shape
        if B > MOST or N > MOST:
            raise _too_large(x)
    a, x = _checked(a, x, 2)
    if state.dtype != torch.float32 or state.shape != x.shape or state.device != x.device or not state.is_contiguous():
        raise ValueError(f"state must be contiguous float32 of shape {tuple(x.shape)} on {x.device}")
    h = torch.empty_like(x, memory_format=torch.contiguous_format)
    s = _Step(B, N, TYPES[x.dtype], code, a.data_ptr(), a.stride(0), x.data_ptr(), x.stride(0), state.data_ptr(), h.data_ptr())
    with _lib.timed("wt_gated_step"):
        rc = _lib.lib().wt_gated_step(_C.byref(s), _C.c_void_p(_lib.stream_of(x.get_device())))
    if rc:
        _lib.check(rc, "wt_gated_step")
    _lib.count_launches(1)
    torch.autograd.graph.increment_version(state)
    return h
