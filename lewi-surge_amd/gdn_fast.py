"""Chunked gated delta rule of the Gated DeltaNet block on the HIP library (mirrors modal/gdn_fast.py).

The reference swaps MaxText's `jax_chunk_gated_delta_rule` for `fast_chunk_gated_delta_rule` (gdn_fast.py:37-113) and
trains through it with XLA autodiff, which keeps the forward's residuals for the backward.  Here, when a gradient is
needed, the forward is lsurge_gdn_chunked_fwd_save (the chunk products and the state entering every chunk kept, about
2.25 KiB per token and head) and the backward lsurge_gdn_chunked_bwd_saved.  With SAVE_RESIDUALS = False the forward
keeps only its inputs and the backward lsurge_gdn_chunked_bwd recomputes the rest (less memory, one more forward's
work); the results are bitwise the same.  Without gradients the forward is lsurge_gdn_chunked_fwd.

  fast_chunk_gated_delta_rule(query, key, value, g, beta, chunk_size=64, initial_state=None, ...)
      differentiable op with the reference's signature: query, key [B, T, H, 128], value [B, T, H, 128], g [B, T, H]
      (log decay, float32), beta [B, T, H]; returns (o [B, T, H, 128] in query's dtype, the final state in the compute
      dtype when initial_state is given, else None)
  install(prec, inv, unroll)   the reference's switches (gdn_fast.py:116-125): recorded, the kernels always compute in
      f32 with the exact inverse
With use_qk_norm_in_gdn the query and key heads are l2-normalised first (gdn_fast.py:43-46) by lsurge_l2norm_rows,
whose backward is lsurge_l2norm_rows_bwd.

Serving keeps each sequence's state between calls, in float32, and takes new tokens through it:

  alloc_delta_state(slots, heads, device="cuda")
      empty states [slots, heads, 128, 128]
  recurrent_gated_delta_rule(query, key, value, g, beta, state, state_slots=None, cu_seqlens=None, use_qk_norm_in_gdn=False)
      the rule over packed new tokens, one of each sequence or any number, the states updated in place (inference only)
The reference leaves decoding to MaxText (third-party, not vendored), so these names are this package's own.
"""
from __future__ import annotations

import torch

import _calls as calls
import _lib as L

SAVE_RESIDUALS = True
PREC = "highest"
INV = "solve"
UNROLL = 1
D = 128


class _GdnFn(torch.autograd.Function):

    @staticmethod
    def forward(ctx, q, k, v, g, beta, h0, want_state):
        B, T, H, _ = q.shape
        o = torch.empty_like(v)
        h_out = torch.empty((B, H, D, D), dtype=torch.float32, device=q.device) if want_state else None
        lib = L.lib()
        ctx.saved = None
        if SAVE_RESIDUALS and any(ctx.needs_input_grad[:6]):
            ctx.saved = L.workspace(lib.lsurge_gdn_chunked_saved_bytes(B, T, H, D, D), q.device)
            L.check(lib.lsurge_gdn_chunked_fwd_save(L.ptr(q), L.ptr(k), L.ptr(v), L.ptr(g), L.ptr(beta), B, T, H, D,
                                                    D, L.ptr(h0), L.ptr(o), L.ptr(h_out), L.ptr(ctx.saved),
                                                    ctx.saved.numel(), L.stream(q.device)), "gdn_chunked_fwd_save")
        else:
            ws = L.workspace(lib.lsurge_gdn_chunked_workspace_bytes(B, T, H, D, D), q.device)
            L.check(lib.lsurge_gdn_chunked_fwd(L.ptr(q), L.ptr(k), L.ptr(v), L.ptr(g), L.ptr(beta), B, T, H, D, D,
                                               L.ptr(h0), L.ptr(o), L.ptr(h_out), L.ptr(ws), ws.numel(),
                                               L.stream(q.device)), "gdn_chunked_fwd")
        ctx.save_for_backward(q, k, v, g, beta, h0)
        ctx.has_h0 = h0 is not None
        return (o, h_out) if want_state else (o,)

    @staticmethod
    def backward(ctx, do, dh_final=None):
        q, k, v, g, beta, h0 = ctx.saved_tensors
        B, T, H, _ = q.shape
        do = L.contig(do.to(torch.bfloat16))
        dhf = None if dh_final is None else L.contig(dh_final.to(torch.float32))
        dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
        dg = torch.empty((B, T, H), dtype=torch.float32, device=q.device)
        db = torch.empty_like(dg)
        dh0 = torch.empty((B, H, D, D), dtype=torch.float32, device=q.device) if ctx.has_h0 else None
        lib = L.lib()
        if ctx.saved is not None:
            ws = L.workspace(lib.lsurge_gdn_chunked_bwd_saved_workspace_bytes(B, T, H, D, D), q.device)
            L.check(lib.lsurge_gdn_chunked_bwd_saved(L.ptr(q), L.ptr(k), L.ptr(v), L.ptr(beta), B, T, H, D, D,
                                                     L.ptr(do), L.ptr(dhf), L.ptr(dq), L.ptr(dk), L.ptr(dv), L.ptr(dg),
                                                     L.ptr(db), L.ptr(dh0), L.ptr(ctx.saved), ctx.saved.numel(),
                                                     L.ptr(ws), ws.numel(), L.stream(q.device)), "gdn_chunked_bwd_saved")
            ctx.saved = None
        else:
            ws = L.workspace(lib.lsurge_gdn_chunked_bwd_workspace_bytes(B, T, H, D, D), q.device)
            L.check(lib.lsurge_gdn_chunked_bwd(L.ptr(q), L.ptr(k), L.ptr(v), L.ptr(g), L.ptr(beta), B, T, H, D, D,
                                               L.ptr(h0), L.ptr(do), L.ptr(dhf), L.ptr(dq), L.ptr(dk), L.ptr(dv),
                                               L.ptr(dg), L.ptr(db), L.ptr(dh0), L.ptr(ws), ws.numel(),
                                               L.stream(q.device)), "gdn_chunked_bwd")
        return dq, dk, dv, dg, db, dh0, None


class _L2NormFn(torch.autograd.Function):
    """Row-wise l2 normalisation over the last axis (MaxText l2norm, eps as given), bf16 in and out."""

    @staticmethod
    def forward(ctx, x, eps):
        rows = x.numel() // x.shape[-1]
        y = torch.empty_like(x)
        r = torch.empty(rows, dtype=torch.float32, device=x.device)
        L.check(L.lib().lsurge_l2norm_rows(L.ptr(x), rows, x.shape[-1], float(eps), L.ptr(y), L.ptr(r),
                                           L.stream(x.device)), "l2norm_rows")
        ctx.save_for_backward(x, r)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, r = ctx.saved_tensors
        dy = L.contig(dy.to(torch.bfloat16))
        dx = torch.empty_like(x)
        L.check(L.lib().lsurge_l2norm_rows_bwd(L.ptr(x), L.ptr(dy), L.ptr(r), r.numel(), x.shape[-1], L.ptr(dx),
                                               L.stream(x.device)), "l2norm_rows_bwd")
        return dx, None


def fast_chunk_gated_delta_rule(query, key, value, g, beta, chunk_size=64, initial_state=None,
                                use_qk_norm_in_gdn=False, cp_axis=None, compute_dtype=torch.bfloat16):
    """modal/gdn_fast.py:37-113.  The kernels take chunks of 64, head dims of 128 and the bf16 compute dtype.  With
    use_qk_norm_in_gdn, query and key are l2-normalised over the head dim first (43-46).  The reference normalises in
    the input dtype and casts afterwards; the l2-norm kernel takes bf16, so qk-norm requires bf16 query and key (for
    them the two orders agree) and other dtypes raise ValueError rather than round twice.  The context-parallel
    branch (39-42) is not built and raises NotImplementedError."""
    if cp_axis is not None:
        raise NotImplementedError("fast_chunk_gated_delta_rule: context parallelism (cp_axis) is not built")
    if use_qk_norm_in_gdn and (query.dtype != torch.bfloat16 or key.dtype != torch.bfloat16):
        raise ValueError("fast_chunk_gated_delta_rule: use_qk_norm_in_gdn takes bf16 query and key (got "
                         f"{query.dtype}, {key.dtype}); the reference normalises before its cast, which the bf16 "
                         "l2-norm kernel reproduces only for bf16 inputs")
    if chunk_size != 64 or compute_dtype != torch.bfloat16:
        raise ValueError("fast_chunk_gated_delta_rule: the kernels take chunk_size=64 and a bf16 compute dtype")
    if query.shape[-1] != D or value.shape[-1] != D or key.shape != query.shape:
        raise ValueError(f"fast_chunk_gated_delta_rule: head dims must be {D} (query {tuple(query.shape)}, "
                         f"value {tuple(value.shape)})")
    L.require_cuda(query, key, value, g, beta, initial_state)
    out_dtype = query.dtype
    q, k, v = (L.contig(t.to(torch.bfloat16)) for t in (query, key, value))
    if use_qk_norm_in_gdn:
        q, k = _L2NormFn.apply(q, 1e-6), _L2NormFn.apply(k, 1e-6)
    bt = L.contig(beta.to(torch.bfloat16))
    gf = L.contig(g.to(torch.float32))
    h0 = None if initial_state is None else L.contig(initial_state.to(torch.float32))
    res = _GdnFn.apply(q, k, v, gf, bt, h0, initial_state is not None)
    o = res[0].to(out_dtype)
    return o, (res[1].to(compute_dtype) if initial_state is not None else None)


def alloc_delta_state(slots, heads, device="cuda"):
    """States of sequences that have no token yet, zeros [slots, heads, 128, 128] float32.  A slot that passes on to a new
    sequence is cleared by the caller."""
    return torch.zeros((slots, heads, D, D), dtype=torch.float32, device=device)


def recurrent_gated_delta_rule(query, key, value, g, beta, state, state_slots=None, cu_seqlens=None,
                               use_qk_norm_in_gdn=False):
    """The gated delta rule over new tokens of sequences whose states are kept: per sequence and value head
    S <- e^g S, d = beta (v - S^T k), S <- S + k d^T, o = S^T q / sqrt(128).

    query, key [rows, Hk, 128] and value [rows, H, 128], bfloat16 or float16, head h reading query and key head
    h // (H // Hk); g [rows, H] float32, the log decay; beta [rows, H] float32 or the others' dtype.  Row b is the one new
    token of sequence b, or with cu_seqlens (int32 [sequences + 1] on the device, ascending from 0) sequence b has the rows
    cu_seqlens[b] .. cu_seqlens[b + 1].  state [slots, H, 128, 128] float32 (alloc_delta_state, or what
    fast_chunk_gated_delta_rule ends with, as float32) is updated in place: sequence b's in slot state_slots[b] (int32 on the
    device; None: b), by all of its rows: who may take drafted tokens back keeps a copy of the slots.  Returns o [rows, H, 128]
    in value's dtype.

    A sequence without rows keeps its state.  One whose slot is outside [0, slots), such as -1 for a place of the batch that
    is not in use, and rows behind the last sequence give zeros and change no state.  No two sequences with rows may name one
    slot.  use_qk_norm_in_gdn: query and key heads are l2-normalised first (eps 1e-6), without the rounding of the normalised
    heads that fast_chunk_gated_delta_rule makes.  States and o are held to float32 until o's one rounding, where the chunked form
    rounds as the reference does; their last bits depend on how a sequence is cut into calls, not on what else is in a call with
    cu_seqlens.  From four rows on a sequence goes in chunks of 32: beside float16 rows the state and what is added to it enter
    products with 23 bits, one less than float32's, and a value that is not finite, or a head whose squares' sum is
    not, reaches all rows of its chunk.  Strides are free: views of one projection are read in place.  No gradient."""
    what = "recurrent_gated_delta_rule"
    shape, vshape = query.shape, value.shape
    if len(shape) != 3 or key.shape != shape or len(vshape) != 3 or vshape[0] != shape[0] or shape[2] != D or vshape[2] != D:
        raise ValueError(f"{what}: query and key must be [rows, key heads, {D}], value [rows, heads, {D}] (got "
                         f"{tuple(query.shape)}, {tuple(key.shape)}, {tuple(value.shape)})")
    rows, hk, hv = shape[0], shape[1], vshape[1]
    if hk < 1 or hv < 1 or hv % hk:
        raise ValueError(f"{what}: {hv} value heads are no multiple of {hk} key heads")
    if g.shape != (rows, hv) or beta.shape != (rows, hv):
        raise ValueError(f"{what}: g and beta must be [{rows}, {hv}] (got {tuple(g.shape)}, {tuple(beta.shape)})")
    if state.dim() != 4 or state.shape[1:] != (hv, D, D):
        raise ValueError(f"{what}: state must be [slots, {hv}, {D}, {D}] (got {tuple(state.shape)})")
    calls.check_device(what, query, key, value, g, beta, state, state_slots, cu_seqlens)
    calls.check_dtype(what, query, key, value)
    if g.dtype is not torch.float32 or state.dtype is not torch.float32 or beta.dtype not in (torch.float32, query.dtype):
        raise TypeError(f"{what}: g and state must be float32, beta float32 or {query.dtype} (got {g.dtype}, {state.dtype}, "
                        f"{beta.dtype})")
    calls.check_no_grad(what, query, key, value, g, beta, state)
    return calls.step(_recurrent, query, key, value, g, beta, state, state_slots, cu_seqlens, use_qk_norm_in_gdn)


def _recurrent(query, key, value, g, beta, state, state_slots, cu_seqlens, norm):
    what = "recurrent_gated_delta_rule"
    rows, hv, _ = value.shape
    nseq, cu, slots = calls.packed(what, rows, cu_seqlens, state, state_slots)
    stride = calls.slot_stride(what, state, 4)
    q, k, v = (calls.row_args(t, D, 1 << 22) for t in (query, key, value))
    if not g.is_contiguous() and not (g.stride(1) == 1 and hv <= g.stride(0) < 1 << 22):
        g = g.contiguous()
    if not beta.is_contiguous() and not (beta.stride(1) == 1 and hv <= beta.stride(0) < 1 << 22):
        beta = beta.contiguous()
    o = value.new_empty((rows, hv, D))
    arg = L.GdnTokens(*q[1:], *k[1:], *v[1:], g.data_ptr(), beta.data_ptr(), state.data_ptr(), o.data_ptr(), calls.ptr(slots),
                      calls.ptr(cu), rows, nseq, key.shape[1], hv, hv if g.is_contiguous() else g.stride(0),
                      hv if beta.is_contiguous() else beta.stride(0), state.shape[0], stride, 1e-6 if norm else -1.0, L.dt(o),
                      L.dt(beta))
    calls.call("gdn_recurrent", o.device, L.lib().lsurge_gdn_recurrent, arg)
    torch.autograd.graph.increment_version(state)
    return o


def install(prec="high", inv="neumann", unroll=1):
    """Record the reference's switches (gdn_fast.py:116-125).  The reference then rebinds MaxText's
    qwen3.jax_chunk_gated_delta_rule; MaxText is a JAX package and absent here, so JAX callers bind the C ABI through
    XLA FFI instead."""
    global PREC, INV, UNROLL
    PREC, INV, UNROLL = prec, inv, int(unroll)
    print(f"[gdn_fast] chunked gated delta rule -> gfx950 kernels (precision={prec} and inverse={inv} recorded; "
          "f32 arithmetic, exact inverse)", flush=True)
