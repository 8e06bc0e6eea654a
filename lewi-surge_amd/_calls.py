"""What the operators' Python surfaces share: argument checks, the call on the current stream, rows by strides, and calls
without a gradient as steps of a trace."""
from __future__ import annotations

import math

import torch
from torch.autograd import forward_ad

import _lib as L


def check_device(what, first, *rest):
    device = first.get_device()  # a number; a device object for each tensor would take as long as a short call's launch
    if device < 0:
        L.require_cuda(first)
    for t in rest:
        if t is not None and t.get_device() != device:
            L.require_cuda(t)
            raise ValueError(f"{what}: all tensors must be on one device (got {first.device} and {t.device})")


def check_dtype(what, *ts):
    dt = ts[0].dtype
    for t in ts:
        if t.dtype is not dt or dt is not torch.bfloat16 and dt is not torch.float16:
            raise TypeError(f"{what}: tensors must all be bfloat16 or all float16 (got {[str(t.dtype) for t in ts]})")


def check_no_grad(what, *ts):
    if torch.is_grad_enabled():
        for t in ts:
            if t.requires_grad:
                raise ValueError(f"{what}: no gradient; call it under torch.no_grad() or on detached tensors")
    # no level is open outside of forward-mode code (unpack_dual would say so too, 0.3 us a tensor)
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in ts):
        raise ValueError(f"{what}: no gradient, of the forward mode neither; call it on detached tensors")


def check_index(what, name, t, shape):
    if t.dtype is not torch.int32 or t.shape != shape:
        raise ValueError(f"{what}: {name} must be int32 of shape {shape} (got {t.dtype}, {tuple(t.shape)})")
    return L.contig(t)


def packed(what, rows, cu_seqlens, state, state_slots):
    """The number of sequences of `rows` packed rows (cu_seqlens None: one row each), and the checked cu_seqlens and
    state_slots (None: sequence b has slot b)."""
    nseq = rows if cu_seqlens is None else cu_seqlens.numel() - 1
    if cu_seqlens is not None:
        if nseq < 0:
            raise ValueError(f"{what}: cu_seqlens must hold the sequences' ends, from 0 (got no entry)")
        cu_seqlens = check_index(what, "cu_seqlens", cu_seqlens, (nseq + 1,))
    if state_slots is not None:
        state_slots = check_index(what, "state_slots", state_slots, (nseq,))
    elif state.shape[0] < nseq:
        raise ValueError(f"{what}: {nseq} sequences in {state.shape[0]} slots need state_slots")
    return nseq, cu_seqlens, state_slots


def slot_stride(what, state, unit):
    """Elements from one slot of `state` to the next; a slot's must be contiguous, 16-byte aligned and apart from the others."""
    if state.is_contiguous():
        size = apart = math.prod(state.shape[1:])
        ok = apart % unit == 0
    else:
        size, apart = state[0].numel(), state.stride(0)
        ok = state[0].is_contiguous() and apart >= size and apart % unit == 0
    if not ok or state.data_ptr() % 16:
        raise ValueError(f"{what}: a slot's state must be contiguous, 16-byte aligned and apart from the others "
                         f"(shape {tuple(state.shape)}, strides {state.stride()})")
    return apart


def call(what, device, fn, *args):
    """fn(*args, the current stream of `device`), with `device` current while its kernels are launched.  The stream's bare
    handle: a Stream object around it costs 2 us, as much as a short call's launch."""
    stream = torch._C._cuda_getCurrentRawStream(device.index)
    if device.index == torch.cuda.current_device():
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, stream)
    if rc:
        L.check(rc, what)


def ptr(t):
    return None if t is None else t.data_ptr()


def rows(t, min_row=None):
    """t [rows, heads, D] as the kernels read it, by strides: a copy only where its last axis is not contiguous, a row or
    head does not start on 16 bytes, or (min_row) rows overlap or lie too far apart."""
    if t.is_contiguous():
        return aligned(t)
    ok = t.stride(2) == 1 and t.data_ptr() % 16 == 0 and t.stride(0) % 8 == 0 and t.stride(1) % 8 == 0
    if min_row is not None:
        ok = ok and min_row <= t.stride(0) < 1 << 22
    return t if ok else t.contiguous()


def aligned(t):
    return t if t.data_ptr() % 16 == 0 else t.clone()


def rows_arg(t):
    row, head = (t.shape[1] * t.shape[2], t.shape[2]) if t.is_contiguous() else t.stride()[:2]
    return L.AttnRows(t.data_ptr(), row, head)


def row_args(t, min_row=0, most=1 << 40):
    """rows(t) and its pointer, row stride and head stride, with as few calls as that takes."""
    row, head, one = t.stride()
    p = t.data_ptr()
    if one == 1 and (p | row << 1 | head << 1) % 16 == 0 and min_row <= row < most:
        return t, p, row, head
    t = t.contiguous()
    if t.data_ptr() % 16:
        t = t.clone()
    return t, t.data_ptr(), t.shape[1] * t.shape[2], t.shape[2]


class _Step(torch.autograd.Function):
    """fn(*args) as one step of a trace."""

    @staticmethod
    def forward(ctx, fn, *args):
        return fn(*args)


def step(fn, *args):
    """fn(*args), which has no gradient: plainly, 3 us less than an autograd function takes, but as one where torch.jit
    traces, which would otherwise record the empty output and not the call that fills it."""
    return _Step.apply(fn, *args) if torch.jit.is_tracing() else fn(*args)
