"""Softmax attention of the hybrid model's full-attention layers on the HIP library: whole prompts and training, and one
new token per sequence over a paged key-value cache; and the rotation of its queries and keys by their positions.

The Gated DeltaNet block (fast_conv, gdn_fast) mixes a sequence in the model's linear layers; these operators do it in the
others.  The reference leaves them to MaxText (third-party, not vendored), so the names are this package's own.

  causal_attention(q, k, v, cu_seqlens_q=None, cu_seqlens_k=None, scale=None, return_lse=False)
      differentiable; dense [B, T, H, D] or packed [T, H, D] with the sequences' ends in cu_seqlens
  alloc_kv_cache(num_pages, page_size, kv_heads, head_dim, dtype, device)
      an empty key and value cache [num_pages, page_size, kv_heads, head_dim]
  append_kv(k_cache, v_cache, page_table, seq_lens, k, v, cu_seqlens=None)
      new tokens' keys and values written to their pages, in place
  rotary_inv_freq(rotary_dim, theta=10000.0, device="cuda")
      the rotation's angles a position, float64 [rotary_dim / 2]
  rotary(q, k, inv_freq, positions=None, cu_seqlens=None, interleaved=False)
      differentiable; queries and keys of prompts and training turned by their positions, dense or packed
  rotary_append_kv(q, k, v, k_cache, v_cache, page_table, seq_lens, inv_freq, cu_seqlens=None, positions=None,
                   interleaved=False, return_k=False)
      append_kv with q and k turned on the way (inference only); returns the turned q
  paged_attention(q, k_cache, v_cache, page_table, seq_lens, scale=None, return_lse=False)
      one query token per sequence over its cached tokens (inference only)

Query head h reads key head h // (H // Hkv).  Types: bf16 and f16, head dims 64, 128 and 256; scores and sums are f32, and
every output is rounded once.  Sequence ends, lengths and page tables stay on the device: no call waits for the GPU, and
all of them can be captured in a graph.  What the device holds is not checked on the host; entries outside their range are
held to it, so that nothing outside the tensors is read or written; like any input it has to stay as it is until a call's
kernels have run.
"""
from __future__ import annotations

import ctypes
import math

import torch

import _lib as L
from _calls import aligned as _aligned, call as _call, check_device as _check_device, check_dtype as _check_dtype
from _calls import check_index as _check_index, check_no_grad as _check_no_grad, ptr as _ptr, rows as _rows
from _calls import row_args as _row_args, rows_arg as _rows_arg, step as _step

HEAD_DIMS = (64, 128, 256)


def _check_heads(what, q_heads, kv_heads, d, *ts):
    _check_device(what, *ts)
    if d not in HEAD_DIMS:
        raise ValueError(f"{what}: head dim must be one of {HEAD_DIMS} (got {d})")
    if kv_heads < 1 or q_heads < 1 or q_heads % kv_heads:
        raise ValueError(f"{what}: {q_heads} query heads are no multiple of {kv_heads} key heads")


def _scale(what, scale, d):
    scale = float(d) ** -0.5 if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"{what}: scale must be positive and finite (got {scale})")
    return scale


def _forward(q, k, v, cu_q, cu_k, nseq, scale, want_lse, training):
    """o, lse (or None) of packed rows, and what the backward needs: the rows as read, what o's rounding left over, the
    shape."""
    tq, hq, d = q.shape
    tk, hk, _ = k.shape
    q, k, v = _rows(q, d), _rows(k, d), _rows(v, d)
    shape = L.AttnShape(nseq, tq, tk, hq, hk, d, L.dt(q))
    o = torch.empty((tq, hq, d), dtype=q.dtype, device=q.device)
    lse = torch.empty((hq, tq), dtype=torch.float32, device=q.device) if want_lse else None
    o_lo = torch.empty((tq, hq, d), dtype=torch.uint8, device=q.device) if training else None
    lib, arg = L.lib(), ctypes.byref(shape)
    nbytes = lib.lsurge_attn_fwd_workspace_bytes(arg)
    ws = L.workspace(nbytes, q.device) if nbytes else None
    _call("attn_fwd", q.device, lib.lsurge_attn_fwd, arg, _rows_arg(q), _rows_arg(k), _rows_arg(v), _ptr(cu_q), _ptr(cu_k),
          scale, _ptr(o), _ptr(o_lo), _ptr(lse), _ptr(ws), nbytes)
    return o, lse, (q, k, v, o_lo), shape


class _AttnFn(torch.autograd.Function):
    """Every call goes through here, with or without gradients, so that whatever records or differentiates functions sees
    it: forward-mode tangents raise instead of being dropped, and a trace holds the call instead of an empty tensor."""

    @staticmethod
    def forward(ctx, q, k, v, cu_q, cu_k, nseq, scale, want_lse, training):
        if training is None:
            training = any(ctx.needs_input_grad[:3])
        o, lse, rows, shape = _forward(q, k, v, cu_q, cu_k, nseq, scale, want_lse or training, training)
        if training:
            ctx.save_for_backward(*rows, cu_q, cu_k, o, lse)
            ctx.shape, ctx.scale = shape, scale
            ctx.set_materialize_grads(False)
        return o, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do, dlse):
        q, k, v, o_lo, cu_q, cu_k, o, lse = ctx.saved_tensors
        if do is None:
            do = torch.zeros_like(o)
        do = _aligned(L.contig(do.to(o.dtype)))
        dlse = None if dlse is None else L.contig(dlse.to(torch.float32))
        dq = torch.empty_like(o)
        dk, dv = (torch.empty(k.shape, dtype=k.dtype, device=k.device) for _ in range(2))
        lib = L.lib()
        shape = ctypes.byref(ctx.shape)
        ws = L.workspace(lib.lsurge_attn_bwd_workspace_bytes(shape), q.device)
        _call("attn_bwd", q.device, lib.lsurge_attn_bwd, shape, _rows_arg(q), _rows_arg(k), _rows_arg(v), _ptr(cu_q),
              _ptr(cu_k), ctx.scale, _ptr(o), _ptr(o_lo), _ptr(lse), _ptr(do), _ptr(dlse), _ptr(dq), _ptr(dk),
              _ptr(dv), _ptr(ws), ws.numel())
        return dq, dk, dv, None, None, None, None, None, None


def causal_attention(q, k, v, cu_seqlens_q=None, cu_seqlens_k=None, scale=None, return_lse=False):
    """Causal attention of grouped heads.  q [B, Tq, H, D] with k, v [B, Tk, Hkv, D], or packed: q [Tq, H, D] with k, v
    [Tk, Hkv, D], sequence s holding the query rows cu_seqlens_q[s] .. cu_seqlens_q[s + 1] and the key rows given by
    cu_seqlens_k alike (None: cu_seqlens_q; int32 [sequences + 1] on the device, ascending from 0).  A sequence's queries
    are its last positions: query i of nq sees the keys j <= i + nk - nq, so that k and v may hold a cached prefix; a query
    that sees no key gives zeros.  scale (default D ** -0.5) multiplies the scores.

    Returns o in q's shape and dtype, and with return_lse also the natural logarithm of each row's sum of exponentials, f32
    [B, Tq, H] or [Tq, H] (-inf for a row without keys, whose upstream gradient counts for nothing).  Both are differentiable
    (once, in backward mode); rows of packed tensors behind the last sequence give zeros and get zero gradients.  Where a
    gradient will be taken, o is divided by the sum of the weights as they were rounded, which is a little more exact: its
    last bits differ from those of a call without gradients, so reentrant activation checkpointing, which makes both, passes
    on another o than it recomputes.  A masked key never counts, whatever k holds there; a value of v that is
    not finite may also reach queries up to 62 before the first that sees it (its weight there is 0, and 0 x inf is NaN), and
    in the backward any input that is not finite gradients of rows up to 95 away, of its own sequence.  Strides are free;
    q, k and v that are views of one projection's output are read in place, and copied are tensors whose last axis is not
    contiguous, whose rows or heads do not start on 16 bytes, overlap or lie 2^22 elements apart, or, dense, whose sequences do
    not follow each other at the rows' stride ([B, H, T, D] transposed).  While a training step is captured in a graph no eager
    autograd graph of the same leaves may live (torch's accumulators of those leaves belong to the other stream)."""
    what = "causal_attention"
    if q.dim() not in (3, 4) or k.dim() != q.dim() or v.shape != k.shape or k.shape[-1] != q.shape[-1]:
        raise ValueError(f"{what}: q [B, Tq, H, D] or [Tq, H, D], k and v alike with their own rows and heads (got "
                         f"{tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)})")
    d = q.shape[-1]
    _check_heads(what, q.shape[-2], k.shape[-2], d, q, k, v, cu_seqlens_q, cu_seqlens_k)
    _check_dtype(what, q, k, v)
    scale = _scale(what, scale, d)
    if q.dim() == 4:
        if cu_seqlens_q is not None or cu_seqlens_k is not None:
            raise ValueError(f"{what}: cu_seqlens go with packed [T, H, D] tensors")
        if k.shape[0] != q.shape[0]:
            raise ValueError(f"{what}: {q.shape[0]} sequences of queries, {k.shape[0]} of keys")
        nseq, cu_q, cu_k = q.shape[0], None, None
    else:
        if cu_seqlens_q is None:
            raise ValueError(f"{what}: packed tensors need cu_seqlens_q")
        nseq = max(cu_seqlens_q.numel() - 1, 0)
        cu_q = _check_index(what, "cu_seqlens_q", cu_seqlens_q, (nseq + 1,))
        if cu_seqlens_k is None and k.shape[0] != q.shape[0]:
            raise ValueError(f"{what}: {q.shape[0]} query rows and {k.shape[0]} key rows need cu_seqlens_k")
        cu_k = cu_q if cu_seqlens_k is None else _check_index(what, "cu_seqlens_k", cu_seqlens_k, (nseq + 1,))
    shape = q.shape
    if q.dim() == 4:
        q, k, v = q.flatten(0, 1), k.flatten(0, 1), v.flatten(0, 1)
    # a trace does not hold what it was recorded for: a replay goes by its own inputs
    training = None if torch.jit.is_tracing() else \
        torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    o, lse = _AttnFn.apply(q, k, v, cu_q, cu_k, nseq, scale, return_lse, training)
    o = o.view(shape)
    return (o, lse.t().reshape(shape[:-1])) if return_lse else o


def alloc_kv_cache(num_pages, page_size, kv_heads, head_dim, dtype=torch.bfloat16, device="cuda"):
    """An empty key and value cache, each [num_pages, page_size, kv_heads, head_dim], with the tokens of one head and page
    consecutive in memory."""
    shape = (num_pages, kv_heads, page_size, head_dim)
    return tuple(torch.empty(shape, dtype=dtype, device=device).transpose(1, 2) for _ in range(2))


def _cache_strides(what, t, shape):
    page, slot, head, one = t.stride()
    if 1 in shape:  # the stride of an axis of one means nothing
        page, slot, head = (0 if n == 1 else s for n, s in zip(shape, (page, slot, head)))
    p = t.data_ptr()
    if one != 1 or (page | slot | head) % 8 or p % 16:
        raise ValueError(f"{what}: a token's values in a cache must be contiguous and 16-byte aligned (strides {t.stride()})")
    return p, page, slot, head


def _cache_arg(what, k_cache, v_cache, page_table, seq_lens):
    shape, tshape = k_cache.shape, page_table.shape
    if len(shape) != 4 or v_cache.shape != shape:
        raise ValueError(f"{what}: caches must be [num_pages, page_size, kv_heads, head_dim] (got {tuple(k_cache.shape)}, "
                         f"{tuple(v_cache.shape)})")
    pages, size, heads, d = shape
    if pages < 1 or size < 8 or size > 4096 or size & (size - 1):
        raise ValueError(f"{what}: at least one page, of a power of two from 8 to 4096 tokens (got {pages} of {size})")
    if len(tshape) != 2 or tshape[1] < 1:
        raise ValueError(f"{what}: page_table must be [sequences, pages] (got {tuple(tshape)})")
    nseq, most = tshape
    table = _check_index(what, "page_table", page_table, tshape)
    lens = _check_index(what, "seq_lens", seq_lens, (nseq,))
    k, *k_strides = _cache_strides(what, k_cache, shape)
    v, *v_strides = _cache_strides(what, v_cache, shape)
    arg = L.KvCache(k, v, *k_strides, *v_strides, table.data_ptr(), most, lens.data_ptr(), pages, size, most, heads, d,
                    L.dt(k_cache))
    return arg, (table, lens)


def append_kv(k_cache, v_cache, page_table, seq_lens, k, v, cu_seqlens=None):
    """Write new tokens into a paged cache, in place.  k, v [rows, Hkv, D]: one token for each sequence, or with cu_seqlens
    (int32 [sequences + 1]) the rows cu_seqlens[b] .. cu_seqlens[b + 1] of sequence b.  They become the last of its
    seq_lens[b] tokens (int32, the new ones counted); token t goes to page page_table[b, t // page_size], slot
    t % page_size.  Nothing is written for a sequence of length 0 without cu_seqlens, for rows behind the last sequence, or
    where the table names no page.  Two sequences that share a page must not write to the same place of it.  No gradient
    passes through a cache; a backward that saved it before the call raises, as after any write in place."""
    what = "append_kv"
    if k.dim() != 3 or v.shape != k.shape or k_cache.dim() != 4 or k.shape[1:] != k_cache.shape[2:]:
        raise ValueError(f"{what}: k and v must be [rows, kv_heads, head_dim] of the caches (got {tuple(k.shape)}, "
                         f"{tuple(v.shape)}, caches {tuple(k_cache.shape)})")
    _check_heads(what, k.shape[1], k.shape[1], k.shape[2], k, v, k_cache, v_cache, page_table, seq_lens, cu_seqlens)
    _check_dtype(what, k, v, k_cache, v_cache)
    _check_no_grad(what, k, v, k_cache, v_cache)
    _step(_append, k_cache, v_cache, page_table, seq_lens, k, v, cu_seqlens)


def _append(k_cache, v_cache, page_table, seq_lens, k, v, cu_seqlens):
    what = "append_kv"
    arg, keep = _cache_arg(what, k_cache, v_cache, page_table, seq_lens)
    nseq = page_table.shape[0]
    if cu_seqlens is not None:
        cu_seqlens = _check_index(what, "cu_seqlens", cu_seqlens, (nseq + 1,))
    elif k.shape[0] != nseq:
        raise ValueError(f"{what}: {k.shape[0]} tokens for {nseq} sequences need cu_seqlens")
    k, v = _rows(k), _rows(v)
    _call("kv_append", k.device, L.lib().lsurge_kv_append, arg, _rows_arg(k), _rows_arg(v), k.shape[0], nseq,
          _ptr(cu_seqlens))
    torch.autograd.graph.increment_version((k_cache, v_cache))
    del keep


def paged_attention(q, k_cache, v_cache, page_table, seq_lens, scale=None, return_lse=False):
    """Attention of one new token per sequence, q [sequences, H, D], over its seq_lens[b] cached tokens (the new one among
    them, see append_kv).  Returns o [sequences, H, D] in q's dtype, and with return_lse also f32 [sequences, H].  Length 0
    gives zeros (lse -inf); tokens whose page_table entry names no page are left out.  Slots behind a sequence's last token are
    never used, whatever they hold.  Results repeat bit for bit for the same lengths; a sequence's last bits depend on the
    lengths of the others, which decide where its tokens are cut into parts.  No gradient."""
    what = "paged_attention"
    if q.dim() != 3 or k_cache.dim() != 4 or q.shape[2] != k_cache.shape[3] or q.shape[0] != page_table.shape[0]:
        raise ValueError(f"{what}: q must be [sequences, heads, head_dim] (got {tuple(q.shape)}, caches "
                         f"{tuple(k_cache.shape)}, page_table {tuple(page_table.shape)})")
    _check_no_grad(what, q, k_cache, v_cache)
    n, hq, d = q.shape
    _check_heads(what, hq, k_cache.shape[2], d, q, k_cache, v_cache, page_table, seq_lens)
    _check_dtype(what, q, k_cache, v_cache)
    o, lse = _step(_paged, q, k_cache, v_cache, page_table, seq_lens, _scale(what, scale, d), return_lse)
    return (o, lse) if return_lse else o


def _paged(q, k_cache, v_cache, page_table, seq_lens, scale, return_lse):
    n, hq, d = q.shape
    arg, keep = _cache_arg("paged_attention", k_cache, v_cache, page_table, seq_lens)
    q = _rows(q)
    o = torch.empty((n, hq, d), dtype=q.dtype, device=q.device)
    lse = torch.empty((n, hq), dtype=torch.float32, device=q.device) if return_lse else None
    lib = L.lib()
    ws = L.workspace(lib.lsurge_paged_attn_workspace_bytes(n, hq, d), q.device)
    _call("paged_attn", q.device, lib.lsurge_paged_attn, arg, _rows_arg(q), n, hq, scale, _ptr(o), _ptr(lse), _ptr(ws),
          ws.numel())
    del keep
    return o, lse


def rotary_inv_freq(rotary_dim, theta=10000.0, device="cuda"):
    """theta ** (-2 i / rotary_dim) for pair i: the angle that each position adds, float64 [rotary_dim / 2].  Scaled variants
    are the caller's own tensors of that form."""
    i = torch.arange(rotary_dim // 2, dtype=torch.float64, device=device)
    return torch.pow(torch.full_like(i, float(theta)), -2 * i / rotary_dim)


def _rotary_arg(what, d, rows, like, inv_freq, positions, interleaved, inverse=False):
    """The C call's lsurge_rotary, and what it points at."""
    if inv_freq.dim() != 1 or inv_freq.dtype is not torch.float64:
        raise ValueError(f"{what}: inv_freq must be float64 [rotary_dim / 2], since float32 loses the angles of far positions "
                         f"(got {inv_freq.dtype}, {tuple(inv_freq.shape)})")
    rot = 2 * inv_freq.shape[0]
    if not 16 <= rot <= d or rot % 16:
        raise ValueError(f"{what}: rotary_dim must be a multiple of 16 from 16 to the head dim {d} (got {rot})")
    inv_freq = L.contig(inv_freq)
    if positions is not None:
        positions = _check_index(what, "positions", positions, rows).view(-1)
    arg = L.Rotary(inv_freq.data_ptr(), _ptr(positions), rot, bool(interleaved), inverse, L.dt(like))
    return arg, (inv_freq, positions)


def _rotate(q, k, inv_freq, positions, cu, interleaved, inverse, nseq):
    """Dense or packed q and k (either may be None) turned, or by `inverse` turned back."""
    like = k if q is None else q
    arg, keep = _rotary_arg("rotary", like.shape[-1], like.shape[:-2], like, inv_freq, positions, interleaved, inverse)
    outs, args, rows = [], [], 0
    for t in (q, k):
        if t is None:
            outs.append(None)
            args += (None, 0)
        else:
            outs.append(t.new_empty(t.shape))
            t, *where = _row_args(t if t.dim() == 3 else t.flatten(0, 1))
            keep += (t,)
            rows, heads, _ = t.shape
            args += (L.AttnRows(*where), heads)
    _call("rotary", like.device, L.lib().lsurge_rotary_rows, arg, *args, like.shape[-1], rows, nseq, _ptr(cu), _ptr(outs[0]),
          _ptr(outs[1]))
    del keep
    return outs


class _RotaryFn(torch.autograd.Function):
    """Always called through here, as _AttnFn is.  The backward turns the gradients back."""

    @staticmethod
    def forward(ctx, q, k, inv_freq, positions, cu, interleaved, nseq):
        ctx.save_for_backward(inv_freq, positions, cu)
        ctx.rest = interleaved, nseq, q.dtype
        ctx.set_materialize_grads(False)
        out = _rotate(q, k, inv_freq, positions, cu, interleaved, False, nseq)
        want = ctx.needs_input_grad[:2]
        if want[0] != want[1]:  # the other's result needs no gradient either, so that a cache takes it
            ctx.mark_non_differentiable(out[want[0]])
        return tuple(out)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk):
        interleaved, nseq, dtype = ctx.rest
        want_q, want_k = ctx.needs_input_grad[:2]
        dq = dq.to(dtype) if want_q and dq is not None else None
        dk = dk.to(dtype) if want_k and dk is not None else None
        if dq is not None or dk is not None:
            dq, dk = _rotate(dq, dk, *ctx.saved_tensors, interleaved, True, nseq)
        return dq, dk, None, None, None, None, None


def rotary(q, k, inv_freq, positions=None, cu_seqlens=None, interleaved=False):
    """q and k with the first rotary_dim = 2 len(inv_freq) values of every head turned pair by pair by their token's position p:
    (a, b) -> (a cos p f_i - b sin p f_i, b cos p f_i + a sin p f_i), where pair i is the values i and i + rotary_dim / 2, or
    with interleaved 2 i and 2 i + 1.  Dense q [B, T, H, D], k [B, T, Hkv, D], or packed q [T, H, D], k [T, Hkv, D] with
    cu_seqlens (int32 [sequences + 1] on the device) or positions.  positions: int32 of q.shape[:-2]; without them a token's is
    its place in its sequence.  inv_freq: float64 [rotary_dim / 2] (rotary_inv_freq), a constant; angles are formed in 64 bits,
    the rotation in 32, the outputs rounded once.

    Returns new tensors (q, k), differentiable once, in backward mode: the gradients are turned back.  Rows behind the last
    sequence give zeros and get zero gradients.  Strides are free, as in causal_attention, which takes the result."""
    what = "rotary"
    if q.dim() not in (3, 4) or k.dim() != q.dim() or k.shape[:-2] != q.shape[:-2] or k.shape[-1] != q.shape[-1]:
        raise ValueError(f"{what}: q [B, T, H, D] or [T, H, D] and k alike with its own heads (got {tuple(q.shape)}, "
                         f"{tuple(k.shape)})")
    _check_heads(what, q.shape[-2], q.shape[-2], q.shape[-1], q, k, inv_freq, positions, cu_seqlens)
    _check_dtype(what, q, k)
    if inv_freq.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what}: inv_freq has no gradient; detach it")
    if q.dim() == 4:
        if cu_seqlens is not None:
            raise ValueError(f"{what}: cu_seqlens go with packed [T, H, D] tensors")
        nseq = q.shape[0]
    elif cu_seqlens is None:
        if positions is None:
            raise ValueError(f"{what}: packed tensors need cu_seqlens or positions")
        nseq = 0
    else:
        nseq = max(cu_seqlens.numel() - 1, 0)
        cu_seqlens = _check_index(what, "cu_seqlens", cu_seqlens, (nseq + 1,))
    return _RotaryFn.apply(q, k, inv_freq, positions, cu_seqlens, interleaved, nseq)


def rotary_append_kv(q, k, v, k_cache, v_cache, page_table, seq_lens, inv_freq, cu_seqlens=None, positions=None,
                     interleaved=False, return_k=False):
    """append_kv of new tokens whose queries and keys are turned first, as rotary turns them: q [rows, H, D], k, v
    [rows, Hkv, D], everything else as append_kv takes it.  A token's position is its place in its sequence, seq_lens counted
    back from, or positions[row] (int32 [rows]).  The turned k goes to the cache, v as it is.

    Returns the turned q [rows, H, D] for paged_attention (one token a sequence) or, with the turned k [rows, Hkv, D] that
    return_k adds, for causal_attention (prompts).  Rows that hold no token give zeros; a token whose page the table does not
    name is turned and not written.  No gradient."""
    what = "rotary_append_kv"
    n, kv, d = k.shape if k.dim() == 3 else (-1, -1, -1)
    if v.shape != k.shape or k_cache.dim() != 4 or k_cache.shape[2:] != (kv, d) or q.dim() != 3 or q.shape[0] != n or \
            q.shape[2] != d:
        raise ValueError(f"{what}: q must be [rows, heads, head_dim], k and v [rows, kv_heads, head_dim] of the caches (got "
                         f"{tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}, caches {tuple(k_cache.shape)})")
    _check_heads(what, q.shape[1], kv, d, q, k, v, k_cache, v_cache, page_table, seq_lens, inv_freq, cu_seqlens,
                 positions)
    _check_dtype(what, q, k, v, k_cache, v_cache)
    _check_no_grad(what, q, k, v, k_cache, v_cache, inv_freq)
    q, k = _step(_rotary_append, q, k, v, k_cache, v_cache, page_table, seq_lens, inv_freq, cu_seqlens, positions, interleaved,
                 return_k)
    return (q, k) if return_k else q


def _rotary_append(q, k, v, k_cache, v_cache, page_table, seq_lens, inv_freq, cu_seqlens, positions, interleaved, return_k):
    what = "rotary_append_kv"
    n, hq, d = q.shape
    cache, keep = _cache_arg(what, k_cache, v_cache, page_table, seq_lens)
    nseq = page_table.shape[0]
    if cu_seqlens is not None:
        cu_seqlens = _check_index(what, "cu_seqlens", cu_seqlens, (nseq + 1,))
    elif n != nseq:
        raise ValueError(f"{what}: {n} tokens for {nseq} sequences need cu_seqlens")
    rotation, more = _rotary_arg(what, d, (n,), q, inv_freq, positions, interleaved)
    q_out = q.new_empty((n, hq, d))
    k_out = k.new_empty(k.shape) if return_k else None
    if nseq == 0:  # no sequence: every row is behind the last
        q_out.zero_()
        return q_out, k_out.zero_() if return_k else None
    q, k, v = _row_args(q), _row_args(k), _row_args(v)
    _call("rotary_append", q_out.device, L.lib().lsurge_rotary_append, cache, rotation, L.AttnRows(*q[1:]), hq,
          L.AttnRows(*k[1:]), L.AttnRows(*v[1:]), n, nseq, _ptr(cu_seqlens), q_out.data_ptr(), _ptr(k_out))
    torch.autograd.graph.increment_version((k_cache, v_cache))
    del keep, more
    return q_out, k_out
