"""CPU oracle of the operators that carry a hybrid model's sequences from token to token, in float64: the gated delta rule and
the causal convolution from kept states, and the rotation of heads by their positions.

TEST INFRASTRUCTURE ONLY: only `tests/` may import this module.  No product code calls it.

The rule and the convolution are those of modal/gdn_fast.py and modal/fast_conv.py token by token; carrying their state between
calls and the rotation have no counterpart in the reference.  Each function also returns how far a float32 computation with one
last rounding of relative size u (half a step of the output's type) may be from its result.  `tiny` is half the spacing of the
type's smallest values.

Pinned by tests/test_serving.py: the recurrence against gdn_oracle.gated_delta_recurrence, cut into calls at any token; the
convolution against fast_conv's shift-add over the whole sequence; the rotation against complex multiplication, its inverse and
the dot product's dependence on the distance alone; the bounds against a float32 computation and against planted errors.
"""
from __future__ import annotations

import numpy as np

EPS = 2.0 ** -24  # a float32 rounding
HALF_STEP = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}
TINY = {"bf16": 2.0 ** -134, "f16": 2.0 ** -25}


def delta_rule(q, k, v, g, beta, S, norm, terms=32):
    """One sequence's tokens: q, k [T, Hk, D], v [T, H, Dv], g, beta [T, H], S [H, D, Dv].

    Returns o [T, H, Dv], the state, and bounds of the errors' 2-norms before o's last rounding: of o [T, H] and of the state
    [H].  One step is S' = a (I - beta k k^T) S + beta k v^T, and its factor has a 2-norm of a max(1, |1 - beta k.k|), so what
    the state was off goes on no larger than that.  A step adds: its sums of D products, formed in at most `terms` additions
    one after the other (each product and addition rounded), hold to (terms + 2) EPS |k| |S|; the factors of decay, norms and
    beta round a few times each (8 EPS of what they multiply, 2 of them for what two f16 terms leave over of a float32 operand);
    the update rounds twice each of its parts.  Steps taken together
    in chunks round no more of each part, in another order, and are held to the same."""
    q, k, v, g, beta, S = (np.array(x, np.float64) for x in (q, k, v, g, beta, S))
    T, H, D = v.shape[0], v.shape[1], k.shape[2]
    group = H // k.shape[1]
    q, k = (np.repeat(x, group, axis=1) for x in (q, k))
    if norm:
        q, k = (x / np.sqrt((x * x).sum(-1, keepdims=True) + 1e-6) for x in (q, k))
    o, bo, bs = np.zeros(v.shape), np.zeros((T, H)), np.zeros(H)
    c = (terms + 2 + 8) * EPS
    n2 = lambda x, ax=-1: np.sqrt((x * x).sum(ax))  # noqa: E731
    for t in range(T):
        a, b = np.exp(g[t]), np.abs(beta[t])
        nk, nq, nv, ns = n2(k[t]), n2(q[t]), n2(v[t]), n2(S, (1, 2))
        pred = a[:, None] * np.einsum("hk,hkv->hv", k[t], S)
        d = beta[t][:, None] * (v[t] - pred)
        off = b * (a * nk * (bs + c * ns) + 8 * EPS * nv)  # of d, what the state was off counted
        S = a[:, None, None] * S + k[t][:, :, None] * d[:, None, :]
        o[t] = np.einsum("hk,hkv->hv", q[t], S) / np.sqrt(D)
        bo[t] = nq / np.sqrt(D) * (a * (bs + c * ns) + nk * (off + c * n2(d)))
        bs = a * np.maximum(1, np.abs(1 - beta[t] * nk * nk)) * bs \
            + nk * (b * (a * nk * c * ns + 8 * EPS * nv) + 8 * EPS * n2(d)) + 8 * EPS * a * ns
    return o, S, bo, bs


def conv(x, w, state, silu, u, tiny):
    """One sequence's rows x [T, C] after the kept inputs state [K - 1, C], w [K, C].  Returns y, the state, and y's bound:
    K products and sums in float32, SiLU's slope (at most 1.1) and its exponential and quotient (8 EPS), one rounding."""
    x, w, state = (np.asarray(a, np.float64) for a in (x, w, state))
    K, T = w.shape[0], x.shape[0]
    seen = np.concatenate([state, x])
    s = sum(seen[j:j + T] * w[j] for j in range(K))
    off = (K + 1) * EPS * sum(np.abs(seen[j:j + T] * w[j]) for j in range(K))
    y = s
    if silu:
        # s / (1 + e^-s); e^-s is off by up to |s| EPS besides, which reaches y multiplied by s e^-s / (1 + e^-s)^2 < |s| / 4
        y = s * 0.5 * (1 + np.tanh(s / 2))
        off = 1.1 * off + 16 * EPS * (np.abs(y) + np.minimum(s * s, 4))
    return y, seen[T:], off + u * (np.abs(y) + off) + tiny


def rotate(x, pos, inv_freq, interleaved, u, tiny, sign=1.0):
    """x [T, H, D] with its first 2 len(inv_freq) values turned by pos [T] times inv_freq.  Returns the result and its bound:
    the angle's fraction of a turn is rounded to float32 (2^-25 of a turn at most, 2^-22 of an angle), the reduced angle and
    the series a few EPS more, the products and the sum three."""
    x = np.asarray(x, np.float64)
    half = len(inv_freq)
    rot = 2 * half
    ang = sign * np.asarray(pos, np.float64)[:, None] * np.asarray(inv_freq, np.float64)
    c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
    y, off = x.copy(), np.zeros(x.shape)
    ia, ib = (np.arange(0, rot, 2), np.arange(1, rot, 2)) if interleaved else (np.arange(half), np.arange(half, rot))
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    off[..., ia] = off[..., ib] = (np.abs(a) + np.abs(b)) * (2.0 ** -22 + 8 * EPS)
    return y, np.where(off > 0, off + u * (np.abs(y) + off) + tiny, 0.0)
