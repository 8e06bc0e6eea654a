"""Causal depthwise Conv1D of the Gated DeltaNet block on the HIP library (mirrors modal/fast_conv.py).

The reference replaces flax `nnx.Conv(padding="CAUSAL", feature_group_count=C)` on [B, T, C] inputs by K shifted
multiply-adds (fast_conv.py:14-31):  y[b, t, c] = sum_{j<K} w[j, 0, c] x[b, t-(K-1)+j, c].  Here the same operator is
one memory-bound kernel each way (lsurge_causal_conv1d / lsurge_causal_conv1d_bwd): x read once, y written once,
products accumulated in f32 with one rounding.

  applies(...)                 the reference's eligibility test (fast_conv.py:17-22)
  causal_conv1d(inputs, kernel) differentiable op: inputs [B, T, C] bf16, kernel [K, 1, C] (or [K, C]) bf16

Serving keeps each sequence's last K - 1 inputs between calls and takes new ones after them (the reference leaves decoding to
MaxText, third-party and not vendored):

  alloc_conv_state(slots, taps, channels, dtype, device)  empty states [slots, K - 1, C]
  causal_conv1d_update(inputs, kernel, state, state_slots=None, cu_seqlens=None, activation=None)
      the convolution of packed new rows, one of each sequence or any number, the states updated in place (inference only)
"""
from __future__ import annotations

import torch

import _calls as calls
import _lib as L


def applies(kernel_size, feature_group_count, in_features, out_features, padding, ndim, has_bias=False,
            dilation=1, strides=1):
    """Shapes the reference's fast path takes (modal/fast_conv.py:17-22); the others go to the original Conv."""
    k = kernel_size if isinstance(kernel_size, (tuple, list)) else (kernel_size,)
    depthwise = feature_group_count == in_features == out_features
    return (len(k) == 1 and depthwise and padding == "CAUSAL" and ndim == 3 and not has_bias
            and dilation in (1, (1,), None) and strides in (1, (1,), None))


def _check(x, w):
    if x.dim() != 3 or x.dtype != torch.bfloat16 or not x.is_cuda:
        raise ValueError("causal_conv1d: inputs must be a [B, T, C] bf16 ROCm tensor")
    if w.dim() == 3:
        w = w.reshape(w.shape[0], w.shape[2])
    if w.dim() != 2 or w.shape[1] != x.shape[2]:
        raise ValueError("causal_conv1d: kernel must be [K, 1, C] or [K, C] with C = inputs.shape[-1]")
    return L.contig(x), L.contig(w.to(torch.bfloat16))


class _ConvFn(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, w):
        B, T, C = x.shape
        y = torch.empty_like(x)
        L.check(L.lib().lsurge_causal_conv1d(L.ptr(x), L.ptr(w), B, T, C, w.shape[0], L.ptr(y), L.stream(x.device)),
                "causal_conv1d")
        ctx.save_for_backward(x, w)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, w = ctx.saved_tensors
        B, T, C = x.shape
        K = w.shape[0]
        dy = L.contig(dy.to(torch.bfloat16))
        dx = torch.empty_like(x)
        dw = torch.empty((K, C), dtype=torch.float32, device=x.device)
        lib = L.lib()
        ws = L.workspace(lib.lsurge_causal_conv1d_bwd_workspace_bytes(B, T, C, K), x.device)
        L.check(lib.lsurge_causal_conv1d_bwd(L.ptr(x), L.ptr(w), L.ptr(dy), B, T, C, K, L.ptr(dx), L.ptr(dw),
                                             L.ptr(ws), ws.numel(), L.stream(x.device)), "causal_conv1d_bwd")
        return dx, dw.to(w.dtype)


def causal_conv1d(inputs, kernel):
    """y = causal depthwise conv of inputs [B, T, C] with kernel [K, 1, C] (modal/fast_conv.py:24-31)."""
    x, w = _check(inputs, kernel)
    y = _ConvFn.apply(x, w)
    return y


def alloc_conv_state(slots, taps, channels, dtype=torch.bfloat16, device="cuda"):
    """The kept inputs of sequences that have no row yet, zeros [slots, taps - 1, channels].  A slot that passes on to a new
    sequence is cleared by the caller."""
    return torch.zeros((slots, taps - 1, channels), dtype=dtype, device=device)


_ACTIVATIONS = {None: 0, "silu": 1}


def causal_conv1d_update(inputs, kernel, state, state_slots=None, cu_seqlens=None, activation=None):
    """causal_conv1d of new rows of sequences whose last inputs are kept.  inputs [rows, C] and kernel [K, 1, C] or [K, C],
    2 <= K <= 8, all bfloat16 or all float16, C a multiple of 8.  Row b is the one new row of sequence b, or with cu_seqlens
    (int32 [sequences + 1] on the device, ascending from 0) sequence b has the rows cu_seqlens[b] .. cu_seqlens[b + 1].  state
    [slots, K - 1, C] (alloc_conv_state), oldest first, of the same dtype: sequence b's last K - 1 inputs before its new rows are
    in slot state_slots[b] (int32 on the device; None: b), and its last K - 1 with all of them replace them, in place (who may
    take drafted rows back keeps a copy of the slots).  activation: None, or "silu", y = s / (1 + exp(-s)) of the float32 sum s.
    Returns y [rows, C].

    A sequence without rows keeps its state.  One whose slot is outside [0, slots), such as -1 for a place of the batch that is
    not in use, and rows behind the last sequence give zeros and change no state.  No two sequences with rows may name one slot.
    inputs may be a view with rows of any stride.  No gradient."""
    what = "causal_conv1d_update"
    K, *one, channels = kernel.shape if kernel.dim() in (2, 3) else (0, 0, 0)
    if inputs.dim() != 2 or one not in ([], [1]) or inputs.shape[1] != channels:
        raise ValueError(f"{what}: inputs must be [rows, C], kernel [K, 1, C] or [K, C] (got {tuple(inputs.shape)}, "
                         f"{tuple(kernel.shape)})")
    if not 2 <= K <= 8 or channels < 8 or channels % 8:
        raise ValueError(f"{what}: 2 to 8 taps and a multiple of 8 channels (got {K}, {channels})")
    if state.dim() != 3 or state.shape[1:] != (K - 1, channels):
        raise ValueError(f"{what}: state must be [slots, {K - 1}, {channels}] (got {tuple(state.shape)})")
    if activation not in _ACTIVATIONS:
        raise ValueError(f"{what}: activation must be None or 'silu' (got {activation!r})")
    calls.check_device(what, inputs, kernel, state, state_slots, cu_seqlens)
    calls.check_dtype(what, inputs, kernel, state)
    calls.check_no_grad(what, inputs, kernel, state)
    return calls.step(_update, inputs, kernel, K, state, state_slots, cu_seqlens, activation)


def _update(x, w, taps, state, state_slots, cu_seqlens, activation):
    what = "causal_conv1d_update"
    rows, channels = x.shape
    nseq, cu, slots = calls.packed(what, rows, cu_seqlens, state, state_slots)
    stride = calls.slot_stride(what, state, 8)
    if x.stride(1) != 1 or x.stride(0) % 8 or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
    w = calls.aligned(L.contig(w))
    y = x.new_empty((rows, channels))
    arg = L.ConvUpdate(x.data_ptr(), w.data_ptr(), state.data_ptr(), y.data_ptr(), calls.ptr(slots), calls.ptr(cu), rows, nseq,
                       channels, taps, x.stride(0), state.shape[0], stride, L.dt(x), _ACTIVATIONS[activation])
    calls.call(what, x.device, L.lib().lsurge_causal_conv1d_update, arg)
    torch.autograd.graph.increment_version(state)
    return y
