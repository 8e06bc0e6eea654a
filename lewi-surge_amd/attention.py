"""Softmax attention of the hybrid model's full-attention layers on the HIP library: whole prompts and training, and one
new token per sequence over a paged key-value cache.

The Gated DeltaNet block (fast_conv, gdn_fast) mixes a sequence in the model's linear layers; these operators do it in the
others.  The reference leaves them to MaxText (third-party, not vendored), so the names are this package's own.

  causal_attention(q, k, v, cu_seqlens_q=None, cu_seqlens_k=None, scale=None, return_lse=False)
      differentiable; dense [B, T, H, D] or packed [T, H, D] with the sequences' ends in cu_seqlens
  alloc_kv_cache(num_pages, page_size, kv_heads, head_dim, dtype, device)
      an empty key and value cache [num_pages, page_size, kv_heads, head_dim]
  append_kv(k_cache, v_cache, page_table, seq_lens, k, v, cu_seqlens=None)
      new tokens' keys and values written to their pages, in place
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
from torch.autograd import forward_ad

import _lib as L

HEAD_DIMS = (64, 128, 256)


def _check_heads(what, q_heads, kv_heads, d, *ts):
    L.require_cuda(*ts)
    device = ts[0].device
    for t in ts:
        if t is not None and t.device != device:
            raise ValueError(f"{what}: all tensors must be on one device (got {device} and {t.device})")
    if d not in HEAD_DIMS:
        raise ValueError(f"{what}: head dim must be one of {HEAD_DIMS} (got {d})")
    if kv_heads < 1 or q_heads < 1 or q_heads % kv_heads:
        raise ValueError(f"{what}: {q_heads} query heads are no multiple of {kv_heads} key heads")


def _check_dtype(what, *ts):
    dt = ts[0].dtype
    for t in ts:
        if t.dtype is not dt or dt is not torch.bfloat16 and dt is not torch.float16:
            raise TypeError(f"{what}: tensors must all be bfloat16 or all float16 (got {[str(t.dtype) for t in ts]})")


def _check_no_grad(what, *ts):
    if torch.is_grad_enabled() and any(t.requires_grad for t in ts):
        raise ValueError(f"{what}: no gradient; call it under torch.no_grad() or on detached tensors")
    # no level is open outside of forward-mode code (unpack_dual would say so too, 0.3 us a tensor)
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in ts):
        raise ValueError(f"{what}: no gradient, of the forward mode neither; call it on detached tensors")


def _check_index(what, name, t, shape):
    if t.dtype is not torch.int32 or t.shape != shape:
        raise ValueError(f"{what}: {name} must be int32 of shape {shape} (got {t.dtype}, {tuple(t.shape)})")
    return L.contig(t)


def _call(what, device, fn, *args):
    """fn(*args, the current stream of `device`), with `device` current while its kernels are launched.  The stream's bare
    handle: a Stream object around it costs 2 us, as much as a short call's launch."""
    stream = torch._C._cuda_getCurrentRawStream(device.index)
    if device.index == torch.cuda.current_device():
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, stream)
    L.check(rc, what)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _scale(what, scale, d):
    scale = float(d) ** -0.5 if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"{what}: scale must be positive and finite (got {scale})")
    return scale


def _rows(t, min_row=None):
    """t [rows, heads, D] as the kernels read it, by strides: a copy only where its last axis is not contiguous, a row or
    head does not start on 16 bytes, or (min_row) rows overlap or lie too far apart."""
    if t.is_contiguous():
        return _aligned(t)
    ok = t.stride(2) == 1 and t.data_ptr() % 16 == 0 and t.stride(0) % 8 == 0 and t.stride(1) % 8 == 0
    if min_row is not None:
        ok = ok and min_row <= t.stride(0) < 1 << 22
    return t if ok else t.contiguous()


def _aligned(t):
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _rows_arg(t):
    row, head = (t.shape[1] * t.shape[2], t.shape[2]) if t.is_contiguous() else t.stride()[:2]
    return L.AttnRows(t.data_ptr(), row, head)


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


def _cache_strides(what, t):
    st = t.stride()
    if 1 in t.shape:  # the stride of an axis of one means nothing
        st = [0 if n == 1 else s for n, s in zip(t.shape, st)]
    if t.stride(3) != 1 or (st[0] | st[1] | st[2]) % 8 or t.data_ptr() % 16:
        raise ValueError(f"{what}: a token's values in a cache must be contiguous and 16-byte aligned (strides {t.stride()})")
    return st[:3]


def _cache_arg(what, k_cache, v_cache, page_table, seq_lens):
    if k_cache.dim() != 4 or v_cache.shape != k_cache.shape:
        raise ValueError(f"{what}: caches must be [num_pages, page_size, kv_heads, head_dim] (got {tuple(k_cache.shape)}, "
                         f"{tuple(v_cache.shape)})")
    pages, size, heads, d = k_cache.shape
    if pages < 1 or size < 8 or size > 4096 or size & (size - 1):
        raise ValueError(f"{what}: at least one page, of a power of two from 8 to 4096 tokens (got {pages} of {size})")
    if page_table.dim() != 2 or page_table.shape[1] < 1:
        raise ValueError(f"{what}: page_table must be [sequences, pages] (got {tuple(page_table.shape)})")
    nseq, most = page_table.shape
    table = _check_index(what, "page_table", page_table, (nseq, most))
    lens = _check_index(what, "seq_lens", seq_lens, (nseq,))
    arg = L.KvCache(k_cache.data_ptr(), v_cache.data_ptr(), *_cache_strides(what, k_cache), *_cache_strides(what, v_cache),
                    table.data_ptr(), most, lens.data_ptr(), pages, size, most, heads, d, L.dt(k_cache))
    return arg, (table, lens)


class _Step(torch.autograd.Function):
    """fn(*args) as one step of a trace."""

    @staticmethod
    def forward(ctx, fn, *args):
        return fn(*args)


def _step(fn, *args):
    """fn(*args), which has no gradient: plainly, 3 us less than an autograd function takes, but as one where torch.jit
    traces, which would otherwise record the empty output and not the call that fills it."""
    return _Step.apply(fn, *args) if torch.jit.is_tracing() else fn(*args)


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
