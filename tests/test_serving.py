"""The operators that carry a hybrid model's sequences from token to token, without a GPU: their oracle against independent
forms, its bounds against rounded arithmetic and planted errors, and every refusal of the Python surfaces and of the C ABI
before anything is launched."""
import ctypes

import numpy as np
import pytest
import torch

import _lib as L
import attention as A
import fast_conv as FC
import gdn_fast as G
from oracle import gdn_oracle as go
from oracle import serving_oracle as so

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U, TINY = so.HALF_STEP["bf16"], so.TINY["bf16"]


def _rule(rng, T, hk, hv, D=16):
    q, k, v = rng.standard_normal((T, hk, D)), rng.standard_normal((T, hk, D)), rng.standard_normal((T, hv, D))
    g, beta = -np.abs(rng.standard_normal((T, hv))) * 0.1, 1 / (1 + np.exp(-rng.standard_normal((T, hv))))
    return q, k, v, g, beta, rng.standard_normal((hv, D, D)) * 0.2


@pytest.mark.parametrize("hk,hv", [(2, 2), (1, 3), (2, 4)])
def test_oracle_delta_rule_is_the_recurrence(hk, hv):
    rng = np.random.default_rng(hv)
    q, k, v, g, beta, S = _rule(rng, 9, hk, hv)
    k /= np.linalg.norm(k, axis=-1, keepdims=True)
    o, h, _, _ = so.delta_rule(q, k, v, g, beta, S, False)
    rep = lambda x: np.repeat(x, hv // hk, 1)[None]  # noqa: E731
    wo, wh = go.gated_delta_recurrence(rep(q), rep(k), v[None], g[None], beta[None], h0=S[None])
    np.testing.assert_allclose(o, wo[0], atol=1e-12)
    np.testing.assert_allclose(h, wh[0], atol=1e-12)
    a = so.delta_rule(q[:4], k[:4], v[:4], g[:4], beta[:4], S, False)
    b = so.delta_rule(q[4:], k[4:], v[4:], g[4:], beta[4:], a[1], False)
    np.testing.assert_allclose(np.concatenate([a[0], b[0]]), o, atol=1e-13)
    np.testing.assert_allclose(b[1], h, atol=1e-13)


def test_oracle_delta_rule_norm():
    rng = np.random.default_rng(5)
    q, k, v, g, beta, S = _rule(rng, 6, 2, 2)
    unit = lambda x: x / np.sqrt((x ** 2).sum(-1, keepdims=True) + 1e-6)  # noqa: E731
    for x, y in zip(so.delta_rule(q, k, v, g, beta, S, True), so.delta_rule(unit(q), unit(k), v, g, beta, S, False)):
        np.testing.assert_allclose(x, y, atol=1e-12)


def _rule_f32(q, k, v, g, beta, S):
    f = np.float32
    q, k, v, g, beta, S = (np.asarray(x, f) for x in (q, k, v, g, beta, S))
    o = np.zeros(v.shape, f)
    for t in range(len(v)):
        S = S * np.exp(g[t])[:, None, None]
        d = beta[t][:, None] * (v[t] - np.einsum("hk,hkv->hv", k[t], S))
        S = S + k[t][:, :, None] * d[:, None, :]
        o[t] = np.einsum("hk,hkv->hv", q[t], S) * f(q.shape[2] ** -0.5)
    return o, S


def test_delta_rule_bounds_hold_for_float32_and_show_errors():
    rng = np.random.default_rng(6)
    q, k, v, g, beta, S = (x.astype(np.float32) for x in _rule(rng, 200, 2, 2))
    k /= np.linalg.norm(k, axis=-1, keepdims=True)
    o, h, bo, bs = so.delta_rule(q, k, v, g, beta, S, False)
    fo, fh = _rule_f32(q, k, v, g, beta, S)
    assert (np.linalg.norm(fo - o, axis=-1) <= bo).all() and (np.linalg.norm(fh - h, axis=(1, 2)) <= bs).all()
    assert (bs < 1e-3 * np.linalg.norm(h, axis=(1, 2))).all()  # not idle
    late = beta.copy()
    late[150, 0] *= 1.02  # one token's beta 2% off
    fo, fh = _rule_f32(q, k, v, g, late, S)
    assert np.linalg.norm(fo[150, 0] - o[150, 0]) > bo[150, 0]
    kept = _rule_f32(q, k, v, np.where(np.arange(200)[:, None] == 150, 0, g), beta, S)  # one decay left out
    assert np.linalg.norm(kept[0][150:] - o[150:]) > np.linalg.norm(bo[150:])


def test_terms_of_a_float32_operand():
    """Three bf16 terms hold a float32 value; two f16 ones leave up to 2^-23 of it over, in a quarter of all values."""
    x = torch.from_numpy(np.random.default_rng(7).uniform(256, 32768, 1 << 16).astype(np.float32))
    x = torch.cat([x, -x, 4096 + 2049 * 2.0 ** -11 * torch.ones(1)])

    def left(t, dt, n):
        for _ in range(n):
            t = t - t.to(dt).float()  # exact
        return t

    assert not left(x, BF16, 3).any()
    rest = (left(x, F16, 2) / x).abs()
    assert rest.max() <= 2.0 ** -23 and rest.max() > 2.0 ** -23 * 0.99 and 0.2 < (rest > 0).float().mean() < 0.3
    assert (left(x, F16, 3) / x).abs().max() < 2.0 ** -33


@pytest.mark.parametrize("K", [2, 4, 8])
def test_oracle_conv(K):
    rng = np.random.default_rng(K)
    x, w, before = rng.standard_normal((11, 3)), rng.standard_normal((K, 3)), rng.standard_normal((K - 1, 3))
    y, state, _ = so.conv(x, w, before, False, U, TINY)
    whole = np.concatenate([before, x])
    for t in range(11):
        np.testing.assert_allclose(y[t], sum(w[j] * whole[t + j] for j in range(K)), atol=1e-13)
    np.testing.assert_array_equal(state, whole[-(K - 1):])
    a = so.conv(x[:1], w, before, True, U, TINY)
    b = so.conv(x[1:], w, a[1], True, U, TINY)
    ys = so.conv(x, w, before, True, U, TINY)[0]
    np.testing.assert_allclose(np.concatenate([a[0], b[0]]), ys, atol=1e-13)
    np.testing.assert_allclose(ys, y / (1 + np.exp(-y)), atol=1e-13)
    assert (np.abs(y.astype(np.float32) - y) <= so.conv(x, w, before, False, U, TINY)[2]).all()


@pytest.mark.parametrize("inter", [False, True])
def test_oracle_rotation(inter):
    rng = np.random.default_rng(1)
    x, f = rng.standard_normal((5, 2, 24)), 0.3 ** np.arange(8)
    pos = np.array([0, 1, 7, 1000, -3])
    y, _ = so.rotate(x, pos, f, inter, U, TINY)
    pairs = (lambda z: z[..., 0:16:2] + 1j * z[..., 1:16:2]) if inter else (lambda z: z[..., :8] + 1j * z[..., 8:16])
    np.testing.assert_allclose(pairs(y), pairs(x) * np.exp(1j * pos[:, None, None] * f), atol=1e-11)
    np.testing.assert_array_equal(y[..., 16:], x[..., 16:])
    np.testing.assert_array_equal(y[0], x[0])
    back, _ = so.rotate(y, pos, f, inter, U, TINY, -1.0)
    np.testing.assert_allclose(back, x, atol=1e-12)
    a, b = x[:1], x[1:2]  # scores depend on the distance alone
    dots = [(so.rotate(a, [p], f, inter, U, TINY)[0] * so.rotate(b, [p + 9], f, inter, U, TINY)[0]).sum() for p in (0, 3, 500)]
    np.testing.assert_allclose(dots, dots[0], atol=1e-11)


def test_rotation_bound_shows_float32_angles():
    """Angles formed in float32 are outside of the bound at far positions, inside near 0."""
    x, f = np.random.default_rng(2).standard_normal((1, 4, 64)), 10000.0 ** (-np.arange(32) / 32)
    for p, inside in ((3, True), (1000000, False)):
        ang = (np.float32(p) * f.astype(np.float32)).astype(np.float64)
        c, s = np.cos(ang), np.sin(ang)
        got = np.concatenate([x[..., :32] * c - x[..., 32:] * s, x[..., 32:] * c + x[..., :32] * s], -1)
        y, bound = so.rotate(x, [p], f, False, 2.0 ** -11, 2.0 ** -25)
        assert (np.abs(got - y) <= bound).all() == inside


# ----------------------------------------------------------------------------------------------- refusals


def _fake(monkeypatch):
    """The surfaces' argument checks on CPU tensors, with the library out of reach."""
    monkeypatch.setattr(L, "require_cuda", lambda *_: None)
    monkeypatch.setattr(L, "lib", lambda: pytest.fail("the library was called"))


def _t(*shape, dt=BF16):
    return torch.zeros(shape, dtype=dt)


def _i(*v):
    return torch.tensor(v, dtype=torch.int32)


def _gdn(n=4, hk=1, hv=2, slots=4, **kw):
    a = dict(query=_t(n, hk, 128), key=_t(n, hk, 128), value=_t(n, hv, 128), g=_t(n, hv, dt=F32), beta=_t(n, hv),
             state=_t(slots, hv, 128, 128, dt=F32))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,err,match", [
    (dict(query=_t(4, 1, 64), key=_t(4, 1, 64)), ValueError, "query and key must be"),
    (dict(key=_t(4, 2, 128)), ValueError, "query and key must be"),
    (dict(value=_t(3, 2, 128)), ValueError, "query and key must be"),
    (dict(query=_t(4, 3, 128), key=_t(4, 3, 128)), ValueError, "no multiple of 3"),
    (dict(g=_t(4, 1, dt=F32)), ValueError, "g and beta must be"),
    (dict(beta=_t(4)), ValueError, "g and beta must be"),
    (dict(state=_t(4, 1, 128, 128, dt=F32)), ValueError, "state must be"),
    (dict(state=_t(3, 2, 128, 128, dt=F32)), ValueError, "need state_slots"),
    (dict(state=_t(4, 2, 128, 128)), TypeError, "g and state must be float32"),
    (dict(g=_t(4, 2)), TypeError, "g and state must be float32"),
    (dict(beta=_t(4, 2, dt=F16)), TypeError, "beta float32 or"),
    (dict(query=_t(4, 1, 128, dt=F32), key=_t(4, 1, 128, dt=F32), value=_t(4, 2, 128, dt=F32)), TypeError, "all be bfloat16"),
    (dict(key=_t(4, 1, 128, dt=F16)), TypeError, "all be bfloat16"),
    (dict(state_slots=_i(0, 1)), ValueError, "state_slots must be int32"),
    (dict(state_slots=_i(0, 1, 2, 3).long()), ValueError, "state_slots must be int32"),
    (dict(cu_seqlens=_i(0, 4).float()), ValueError, "cu_seqlens must be int32"),
    (dict(cu_seqlens=_i()), ValueError, "sequences' ends"),
    (dict(state=_t(4, 2, 128, 128, dt=F32).transpose(2, 3)), ValueError, "contiguous, 16-byte aligned and apart"),
    (dict(state=_t(1, 2, 128, 128, dt=F32).expand(4, -1, -1, -1)), ValueError, "apart from the others"),
    (dict(state=_t(4 * 32768 + 1, dt=F32)[1:].view(4, 2, 128, 128)), ValueError, "16-byte aligned"),
    (dict(query=_t(4, 1, 128).requires_grad_()), ValueError, "no gradient"),
    (dict(state=_t(4, 2, 128, 128, dt=F32).requires_grad_()), ValueError, "no gradient"),
])
def test_recurrent_refusals(kw, err, match, monkeypatch):
    _fake(monkeypatch)
    with pytest.raises(err, match=match):
        G.recurrent_gated_delta_rule(**_gdn(**kw))


@pytest.mark.parametrize("kw,err,match", [
    (dict(inputs=_t(4, 2, 16)), ValueError, "inputs must be"),
    (dict(kernel=_t(4, 8)), ValueError, "inputs must be"),
    (dict(kernel=_t(1, 16), state=_t(4, 0, 16)), ValueError, "2 to 8 taps"),
    (dict(kernel=_t(9, 16), state=_t(4, 8, 16)), ValueError, "2 to 8 taps"),
    (dict(inputs=_t(4, 12), kernel=_t(4, 12), state=_t(4, 3, 12)), ValueError, "multiple of 8 channels"),
    (dict(state=_t(4, 4, 16)), ValueError, "state must be"),
    (dict(state=_t(3, 3, 16)), ValueError, "need state_slots"),
    (dict(activation="relu"), ValueError, "activation must be"),
    (dict(kernel=_t(4, 1, 16, dt=F16)), TypeError, "all be bfloat16"),
    (dict(inputs=_t(4, 16, dt=F32), kernel=_t(4, 16, dt=F32), state=_t(4, 3, 16, dt=F32)), TypeError, "all be bfloat16"),
    (dict(state=_t(4, 16, 3).transpose(1, 2)), ValueError, "contiguous, 16-byte aligned and apart"),
    (dict(state=_t(4 * 52)[:208].view(4, 52)[:, :48].unflatten(1, (3, 16))), ValueError, "16-byte aligned"),
    (dict(state_slots=_i(0, 1, 2)), ValueError, "state_slots must be int32"),
    (dict(cu_seqlens=_i(0, 2, 4), state_slots=_i(0, 1, 2, 3)), ValueError, "state_slots must be int32"),
    (dict(kernel=_t(4, 1, 16).requires_grad_()), ValueError, "no gradient"),
])
def test_conv_update_refusals(kw, err, match, monkeypatch):
    _fake(monkeypatch)
    a = dict(inputs=_t(4, 16), kernel=_t(4, 1, 16), state=_t(4, 3, 16))
    a.update(kw)
    with pytest.raises(err, match=match):
        FC.causal_conv1d_update(**a)


FREQ = torch.ones(32, dtype=torch.float64)


@pytest.mark.parametrize("kw,err,match", [
    (dict(q=_t(4, 64)), ValueError, "k alike"),
    (dict(k=_t(3, 1, 64)), ValueError, "k alike"),
    (dict(k=_t(4, 1, 128)), ValueError, "k alike"),
    (dict(q=_t(4, 2, 96), k=_t(4, 1, 96)), ValueError, "head dim must be one of"),
    (dict(cu_seqlens=None), ValueError, "need cu_seqlens or positions"),
    (dict(q=_t(1, 4, 2, 64), k=_t(1, 4, 1, 64)), ValueError, "go with packed"),
    (dict(cu_seqlens=_i(0, 4).long()), ValueError, "must be int32"),
    (dict(positions=_i(0, 1, 2)), ValueError, "positions must be int32"),
    (dict(inv_freq=FREQ.float()), ValueError, "must be float64"),
    (dict(inv_freq=FREQ[:, None]), ValueError, "must be float64"),
    (dict(inv_freq=torch.ones(40, dtype=torch.float64)), ValueError, "rotary_dim must be"),
    (dict(inv_freq=FREQ[:12]), ValueError, "rotary_dim must be"),
    (dict(inv_freq=FREQ[:0]), ValueError, "rotary_dim must be"),
    (dict(inv_freq=FREQ.clone().requires_grad_()), ValueError, "inv_freq has no gradient"),
    (dict(k=_t(4, 1, 64, dt=F16)), TypeError, "all be bfloat16"),
    (dict(q=_t(4, 2, 64, dt=F32), k=_t(4, 1, 64, dt=F32)), TypeError, "all be bfloat16"),
])
def test_rotary_refusals(kw, err, match, monkeypatch):
    _fake(monkeypatch)
    a = dict(q=_t(4, 2, 64), k=_t(4, 1, 64), inv_freq=FREQ, cu_seqlens=_i(0, 4))
    a.update(kw)
    with pytest.raises(err, match=match):
        A.rotary(**a)


@pytest.mark.parametrize("kw,err,match", [
    (dict(q=_t(3, 2, 64)), ValueError, "q must be"),
    (dict(q=_t(4, 2, 128)), ValueError, "q must be"),
    (dict(v=_t(4, 2, 64)), ValueError, "q must be"),
    (dict(k=_t(4, 2, 64), v=_t(4, 2, 64)), ValueError, "q must be"),
    (dict(q=_t(4, 2, 64, dt=F16)), TypeError, "all be bfloat16"),
    (dict(page_table=_i(0, 1).view(2, 1), seq_lens=_i(1, 1)), ValueError, "need cu_seqlens"),
    (dict(page_table=_i(0, 1)), ValueError, "page_table must be"),
    (dict(seq_lens=_i(1)), ValueError, "seq_lens must be int32"),
    (dict(inv_freq=FREQ.float()), ValueError, "must be float64"),
    (dict(positions=_i(1)), ValueError, "positions must be int32"),
    (dict(cu_seqlens=_i(0, 4)), ValueError, "cu_seqlens must be int32"),
    (dict(k=_t(4, 1, 64).requires_grad_()), ValueError, "no gradient"),
    (dict(k_cache=_t(2, 12, 1, 64), v_cache=_t(2, 12, 1, 64)), ValueError, "a power of two"),
])
def test_rotary_append_refusals(kw, err, match, monkeypatch):
    _fake(monkeypatch)
    a = dict(q=_t(4, 2, 64), k=_t(4, 1, 64), v=_t(4, 1, 64), k_cache=_t(2, 8, 1, 64), v_cache=_t(2, 8, 1, 64),
             page_table=_i(0, 1, 0, 1).view(4, 1), seq_lens=_i(1, 1, 2, 2), inv_freq=FREQ)
    a.update(kw)
    with pytest.raises(err, match=match):
        A.rotary_append_kv(**a)


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError, match="ROCm device"):
        G.recurrent_gated_delta_rule(**_gdn())
    with pytest.raises(ValueError, match="ROCm device"):
        FC.causal_conv1d_update(_t(4, 16), _t(4, 1, 16), _t(4, 3, 16))
    with pytest.raises(ValueError, match="ROCm device"):
        A.rotary(_t(4, 2, 64), _t(4, 1, 64), FREQ, cu_seqlens=_i(0, 4))


def test_empty_states_and_frequencies():
    assert not G.alloc_delta_state(3, 2, "cpu").any() and G.alloc_delta_state(3, 2, "cpu").shape == (3, 2, 128, 128)
    s = FC.alloc_conv_state(5, 4, 16, F16, "cpu")
    assert s.shape == (5, 3, 16) and s.dtype is F16 and not s.any()
    f = A.rotary_inv_freq(64, 1e6, "cpu")
    assert f.dtype is torch.float64
    np.testing.assert_allclose(f.numpy(), 1e6 ** (-np.arange(32) / 32), rtol=1e-14)


FAKE = 256  # aligned, never read: the checks return first


def _rows(stride=128, head=128, data=FAKE):
    return L.AttnRows(data, stride, head)


def _tokens(**kw):
    a = dict(g=FAKE, beta=FAKE, state=FAKE, o=FAKE, rows=4, nseq=4, hk=1, hv=2, g_stride=2,
             beta_stride=2, num_slots=4, slot_stride=32768, l2_eps=-1.0, dtype=L.BF16, beta_dtype=L.BF16)
    a.update(kw)
    for n in "qkv":
        r = a.pop(n, _rows())
        a.update({n + f: getattr(r, f) for f, _ in L.AttnRows._fields_})
    return L.GdnTokens(**a)


@pytest.mark.parametrize("kw,msg", [
    (dict(rows=5), b"5 rows of 4"), (dict(rows=-1, cu=FAKE), b"-1 rows"), (dict(hv=3, hk=2), b"3 value heads over 2"),
    (dict(hk=0), b"value heads over 0"), (dict(dtype=L.F32), b"bf16 or f16"), (dict(beta_dtype=L.F16), b"beta alike"),
    (dict(q=_rows(stride=132)), b"multiples of 8"), (dict(k=_rows(stride=120)), b"multiples of 8"),
    (dict(v=_rows(stride=1 << 22)), b"multiples of 8"),
    (dict(g_stride=1), b"strides"), (dict(beta_stride=1 << 22), b"strides"), (dict(k=_rows(data=264)), b"misaligned rows"), (dict(v=_rows(data=0)), b"null"),
    (dict(o=0), b"null pointer"), (dict(state=0), b"null pointer"), (dict(state=264), b"misaligned"),
    (dict(slot_stride=32770), b"strides"), (dict(slot_stride=32764), b"strides"),
    (dict(num_slots=-1), b"slots"), (dict(rows=1 << 30, nseq=1 << 30), b"rows of"),
    (dict(rows=1 << 21, nseq=1 << 21), b"sequences of 2 heads"),
])
def test_recurrent_abi_refusals(kw, msg):
    lib, t = L.lib(), _tokens(**kw)
    assert lib.lsurge_gdn_recurrent(ctypes.byref(t), None) != 0
    assert msg in lib.lsurge_last_error(), lib.lsurge_last_error()


def test_recurrent_abi_empty():
    lib, t = L.lib(), _tokens(rows=0, nseq=0)
    assert lib.lsurge_gdn_recurrent(ctypes.byref(t), None) == 0
    assert lib.lsurge_gdn_recurrent(None, None) != 0


def _update(**kw):
    a = dict(x=FAKE, w=FAKE, state=FAKE, y=FAKE, rows=4, nseq=4, channels=16, taps=4, x_stride=16, num_slots=4, slot_stride=48,
             dtype=L.BF16, activation=0)
    a.update(kw)
    return L.ConvUpdate(**a)


@pytest.mark.parametrize("kw,msg", [
    (dict(channels=12), b"12 channels"), (dict(taps=1), b"1 taps"), (dict(taps=9), b"9 taps"), (dict(rows=3), b"3 rows of 4"),
    (dict(dtype=L.F32), b"bf16 or f16"), (dict(activation=2), b"activation 2"),
    (dict(slot_stride=44), b"strides"), (dict(slot_stride=40), b"strides"), (dict(x_stride=17), b"strides"), (dict(x=0), b"null pointer"), (dict(state=0), b"null pointer"), (dict(y=264), b"aligned"),
])
def test_conv_update_abi_refusals(kw, msg):
    lib, u = L.lib(), _update(**kw)
    assert lib.lsurge_causal_conv1d_update(ctypes.byref(u), None) != 0
    assert msg in lib.lsurge_last_error(), lib.lsurge_last_error()
    assert lib.lsurge_causal_conv1d_update(ctypes.byref(_update(rows=0, nseq=0)), None) == 0


def _rotary(**kw):
    a = dict(inv_freq=FAKE, rotary_dim=64, dtype=L.BF16)
    a.update(kw)
    return L.Rotary(**a)


@pytest.mark.parametrize("kw,call,msg", [
    (dict(rotary_dim=80), {}, b"rotary_dim 80"), (dict(rotary_dim=24), {}, b"rotary_dim 24"), (dict(rotary_dim=0), {}, b"rotary_dim 0"),
    (dict(inv_freq=0), {}, b"frequencies"), (dict(inv_freq=260), {}, b"frequencies"), (dict(dtype=L.F32), {}, b"bf16 or f16"),
    ({}, dict(d=96), b"head_dim 96"), ({}, dict(hq=70000), b"heads"), ({}, dict(rows=5, nseq=2), b"dense"),
    ({}, dict(q=_rows(stride=100)), b"multiples of 8"), ({}, dict(q_out=264), b"q_out"), ({}, dict(k_out=0), b"k_out"),
])
def test_rotary_abi_refusals(kw, call, msg):
    lib = L.lib()
    a = dict(r=_rotary(**kw), q=_rows(), hq=2, k=_rows(), hk=1, d=64, rows=4, nseq=1, cu=None, q_out=FAKE, k_out=FAKE)
    a.update(call)
    assert lib.lsurge_rotary_rows(*a.values(), None) != 0
    assert msg in lib.lsurge_last_error(), lib.lsurge_last_error()


def test_rotary_append_abi_refusals():
    lib = L.lib()
    cache = dict(k=FAKE, v=FAKE, k_page_stride=512, k_slot_stride=64, k_head_stride=64, v_page_stride=512, v_slot_stride=64,
                 v_head_stride=64, page_table=FAKE, table_stride=4, seq_lens=FAKE, num_pages=4, page_size=8, max_pages=4, heads=1,
                 d=64, dtype=L.BF16)
    for c, r, kw, msg in (({}, {}, dict(rows=3), b"3 rows for 4"), (dict(page_size=12), {}, {}, b"page_size"),
                          ({}, dict(dtype=L.F16), {}, b"dtype"), ({}, {}, dict(q_out=0), b"q_out"),
                          ({}, {}, dict(k_out=264), b"k_out"), ({}, dict(rotary_dim=128), {}, b"rotary_dim")):
        a = dict(q=_rows(), hq=2, k=_rows(), v=_rows(), rows=4, nseq=4, cu=None, q_out=FAKE, k_out=None)
        a.update(kw)
        assert lib.lsurge_rotary_append(L.KvCache(**dict(cache, **c)), _rotary(**r), *a.values(), None) != 0
        assert msg in lib.lsurge_last_error(), lib.lsurge_last_error()
