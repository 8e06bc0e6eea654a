"""CPU oracle of the softmax attention operators (numpy, float64), with first-order error bounds of 16-bit kernels.

TEST INFRASTRUCTURE ONLY: only `tests/` may import this module.  No product code calls it.

One sequence: q [nq, Hq, D], k, v [nk, Hk, D]; query i sees the keys j <= i + nk - nq, head h reads key head
h // (Hq // Hk).  s = scale q k^T, w = softmax(s) over the visible keys (all zero for a row that sees none), o = w v,
lse = log sum exp s.  The backward is the chain rule: ds = w (do v^T - (do . o) + dlse).  Pinned in
tests/test_attention.py by a loop over single elements and by central finite differences.

Bounds.  u is half a step of the 16-bit type (2^-8 bf16, 2^-11 f16), x = 2^-24 that of f32.  A kernel that keeps scores,
sums and accumulators in f32 and rounds the weights and score gradients to the type for its products, and each output
once, is within (to first order, each term a count of roundings)
  score           es = (D + 4) x scale |q| . |k|           (D products summed, the scale, the base change)
  weight          ew = u + 2 max_j es + (nk + 8) x          (relative; its rounding, its exponent, the row's sum, exp2)
  o               ew (A + |o|) + u |o| + tiny,   A = w |v|   (divided by the sum of the weights as rounded, w (1 + e), |e| <= ew:
                  sum w (1 + e) v / sum w (1 + e) - o = sum w e (v - o) / (1 + sum w e), at most ew (A + |o|) to first order; by
                  the sum of the unrounded ones: ew A)
  do . v          ep = (D + 2) x |do| . |v|
  delta           ed = |do| . (error of o) + (D + 2) x |do| . |o|
  ds              eds = ew |ds| + w (ep + ed)               (one more u inside ew stands for its own rounding)
  dq              scale eds |k| + u |dq|, dk = scale eds^T |q| + u |dk|, dv = (ew w)^T |do| + u |dv|
f16 has few exponent bits: a weight or score gradient below 2^-14 of its scaled range is off by up to 2^-25 of it, which
`tiny` adds for every key.
"""
from __future__ import annotations

import numpy as np

X = 2.0 ** -24


def visible(nq, nk):
    return np.arange(nk)[None, :] <= np.arange(nq)[:, None] + nk - nq


def _heads(t, group):
    """[n, Hk, D] -> [Hq, n, D]"""
    return np.repeat(np.asarray(t, np.float64).transpose(1, 0, 2), group, axis=0)


def _weights(q, k, scale, mask=None):
    group = q.shape[1] // k.shape[1]
    qh, kh = np.asarray(q, np.float64).transpose(1, 0, 2), _heads(k, group)
    s = scale * (qh @ kh.transpose(0, 2, 1))
    mask = visible(q.shape[0], k.shape[0]) if mask is None else mask
    s = np.where(mask, s, -np.inf)
    if k.shape[0] == 0:
        return s, s, np.full(s.shape[:2], -np.inf)
    m = s.max(-1, keepdims=True)
    m = np.where(np.isfinite(m), m, 0.0)
    e = np.exp(s - m)
    l = e.sum(-1, keepdims=True)
    with np.errstate(divide="ignore"):
        lse = (m + np.log(l))[..., 0]
    return s, e / np.where(l == 0, 1.0, l), lse


def attention(q, k, v, scale, mask=None):
    """o [nq, Hq, D] and lse [nq, Hq]."""
    _, w, lse = _weights(q, k, scale, mask)
    o = w @ _heads(v, q.shape[1] // k.shape[1])
    return o.transpose(1, 0, 2), lse.T


def attention_bwd(q, k, v, do, scale, dlse=None):
    """dq, dk, dv for upstream do [nq, Hq, D] and dlse [nq, Hq]."""
    group, hk = q.shape[1] // k.shape[1], k.shape[1]
    _, w, _ = _weights(q, k, scale)
    qh, g = (np.asarray(t, np.float64).transpose(1, 0, 2) for t in (q, do))
    kh, vh = _heads(k, group), _heads(v, group)
    delta = (g * (w @ vh)).sum(-1, keepdims=True)
    if dlse is not None:
        delta = delta - np.asarray(dlse, np.float64).T[..., None]
    ds = w * (g @ vh.transpose(0, 2, 1) - delta)
    dq = scale * (ds @ kh)
    dk, dv = scale * (ds.transpose(0, 2, 1) @ qh), w.transpose(0, 2, 1) @ g
    fold = lambda t: t.reshape(hk, group, *t.shape[1:]).sum(1).transpose(1, 0, 2)  # noqa: E731
    return dq.transpose(1, 0, 2), fold(dk), fold(dv)


def bounds(q, k, v, scale, u, do=None, dlse=None, mask=None):
    """Elementwise bounds of o, lse (and dq, dk, dv) as derived above."""
    nk, D = k.shape[0], k.shape[2]
    group, hk = q.shape[1] // k.shape[1], k.shape[1]
    _, w, lse = _weights(q, k, scale, mask)
    aq = np.abs(np.asarray(q, np.float64)).transpose(1, 0, 2)
    ak, av = np.abs(_heads(k, group)), np.abs(_heads(v, group))
    es = (D + 4) * X * scale * (aq @ ak.transpose(0, 2, 1)) if nk else np.zeros(w.shape)
    es = np.where(w > 0, es, 0.0).max(-1, keepdims=True) if nk else np.zeros(w.shape[:2] + (1,))
    ew = u + 2 * es + (nk + 8) * X
    tiny = 2.0 ** -25 if u == 2.0 ** -11 else 0.0
    vsum = av.sum(1, keepdims=True)
    o = w @ _heads(v, group)
    eo = 1.05 * (ew * (w @ av + np.abs(o)) + u * np.abs(o) + tiny * (vsum + 1))
    el = np.where(np.isfinite(lse), es[..., 0] + (nk + 8) * X + 4 * X * np.abs(np.where(np.isfinite(lse), lse, 0)), 0.0)
    out = [eo.transpose(1, 0, 2), el.T]
    if do is None:
        return out
    g = np.asarray(do, np.float64).transpose(1, 0, 2)
    ag, vh = np.abs(g), _heads(v, group)
    delta = (g * o).sum(-1, keepdims=True)
    if dlse is not None:
        delta = delta - np.asarray(dlse, np.float64).T[..., None]
    ds = np.abs(w * (g @ vh.transpose(0, 2, 1) - delta))
    ed = (ag * eo).sum(-1, keepdims=True) + (D + 2) * X * (ag * np.abs(o)).sum(-1, keepdims=True)
    ep = (D + 2) * X * (ag @ av.transpose(0, 2, 1))
    eds = (ew + u) * ds + w * (ep + ed)
    # half a subnormal step of the score gradients at their scale: 2^-35 of the largest upstream gradient, or 2^-25 of the
    # row's (key's) largest score gradient, which the second u of eds, unused since ds is formed of unrounded weights, covers
    # for up to 2^14 keys (rows); of the weights, scaled by 2^10: 2^-35
    if tiny:
        eds = eds + 2.0 ** -29 * ag.max(initial=0)
    ewt = ew * w + tiny * 2.0 ** -10 * (w > 0)
    dq, dk, dv = attention_bwd(q, k, v, do, scale, dlse)
    fold = lambda t: t.reshape(hk, group, *t.shape[1:]).sum(1).transpose(1, 0, 2)  # noqa: E731
    edq = scale * (eds @ ak) + tiny
    edk, edv = scale * (eds.transpose(0, 2, 1) @ aq) + tiny, ewt.transpose(0, 2, 1) @ ag + tiny
    return out + [1.05 * (edq.transpose(1, 0, 2) + u * np.abs(dq)), 1.05 * (fold(edk) + u * np.abs(dk)),
                  1.05 * (fold(edv) + u * np.abs(dv))]
