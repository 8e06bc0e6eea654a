"""Softmax attention without a GPU: the oracle against single-element loops and finite differences, and every refusal of
the Python surface and of the C ABI before anything is launched."""
import ctypes
import math

import numpy as np
import pytest
import torch

import _lib as L
import attention as A
from oracle import attention_oracle as ao


def _loop(q, k, v, scale):
    nq, hq, d = q.shape
    nk, hk, _ = k.shape
    o, lse = np.zeros((nq, hq, d)), np.full((nq, hq), -np.inf)
    for i in range(nq):
        for h in range(hq):
            kh = h // (hq // hk)
            js = [j for j in range(nk) if j <= i + nk - nq]
            if js:
                e = [math.exp(scale * float(np.dot(q[i, h], k[j, kh]))) for j in js]
                lse[i, h] = math.log(sum(e))
                o[i, h] = sum(x * v[j, kh] for x, j in zip(e, js)) / sum(e)
    return o, lse


@pytest.mark.parametrize("nq,nk,hq,hk", [(1, 1, 1, 1), (5, 5, 4, 2), (3, 7, 2, 1), (6, 2, 3, 3), (2, 0, 2, 1)])
def test_oracle_forward(nq, nk, hq, hk):
    rng = np.random.default_rng(nq + nk)
    q, k, v = rng.standard_normal((nq, hq, 4)), rng.standard_normal((nk, hk, 4)), rng.standard_normal((nk, hk, 4))
    o, lse = ao.attention(q, k, v, 0.7)
    wo, wl = _loop(q, k, v, 0.7)
    np.testing.assert_allclose(o, wo, atol=1e-13)
    np.testing.assert_allclose(lse, wl, atol=1e-13)


@pytest.mark.parametrize("nq,nk,hq,hk", [(4, 4, 2, 1), (3, 6, 2, 2), (5, 3, 4, 2)])
def test_oracle_backward_against_differences(nq, nk, hq, hk):
    rng = np.random.default_rng(7)
    q, k, v = rng.standard_normal((nq, hq, 3)), rng.standard_normal((nk, hk, 3)), rng.standard_normal((nk, hk, 3))
    do, dl = rng.standard_normal((nq, hq, 3)), rng.standard_normal((nq, hq))

    def loss():
        o, lse = ao.attention(q, k, v, 0.6)
        return (o * do).sum() + (np.where(np.isfinite(lse), lse, 0) * dl).sum()

    seen = np.isfinite(ao.attention(q, k, v, 0.6)[1])
    got = ao.attention_bwd(q, k, v, do, 0.6, np.where(seen, dl, 0))
    for t, g in zip((q, k, v), got):
        for i in np.ndindex(*t.shape):
            keep = t[i]
            t[i] = keep + 1e-6
            up = loss()
            t[i] = keep - 1e-6
            down = loss()
            t[i] = keep
            assert abs((up - down) / 2e-6 - g[i]) < 1e-7


def test_bounds_hold_for_rounded_arithmetic():
    """The bounds cover a float32 computation with weights and outputs rounded to the type, and are not idle: an error of
    five times the type's half step in the weights is outside."""
    rng = np.random.default_rng(3)
    for dt, u in ((torch.bfloat16, 2.0 ** -8), (torch.float16, 2.0 ** -11)):
        q, k, v = (torch.from_numpy(rng.standard_normal((40, 2, 64))).to(dt) for _ in range(3))
        q, k, v = (t.double().numpy() for t in (q, k, v))
        o, _ = ao.attention(q, k, v, 0.125)
        _, w, _ = ao._weights(q, k, 0.125)
        wr = torch.from_numpy(w).float().to(dt).double().numpy()
        got = torch.from_numpy((wr @ v.transpose(1, 0, 2)).transpose(1, 0, 2)).float().to(dt).double().numpy()
        bo = ao.bounds(q, k, v, 0.125, u)[0]
        assert (np.abs(got - o) <= bo).all()
        bad = ((w * (1 + 5 * u)) @ np.abs(v.transpose(1, 0, 2))).transpose(1, 0, 2)
        good = (w @ np.abs(v.transpose(1, 0, 2))).transpose(1, 0, 2)
        assert (np.abs(bad - good) > ao.bounds(q, k, np.abs(v), 0.125, u)[0]).any()


def _fake(monkeypatch):
    """The surface's argument checks on CPU tensors, with the library out of reach."""
    monkeypatch.setattr(A.L, "require_cuda", lambda *_: None)
    monkeypatch.setattr(A.L, "lib", lambda: pytest.fail("the library was called"))


def _t(*shape, dt=torch.bfloat16):
    return torch.zeros(shape, dtype=dt)


CU = torch.tensor([0, 4], dtype=torch.int32)


@pytest.mark.parametrize("args,kw,err", [
    ((_t(4, 2, 64), _t(4, 2, 64), _t(4, 2, 64)), {}, "packed tensors need cu_seqlens_q"),
    ((_t(1, 4, 2, 64), _t(1, 4, 2, 64), _t(1, 4, 2, 64), CU), {}, "go with packed"),
    ((_t(1, 4, 2, 64), _t(2, 4, 2, 64), _t(2, 4, 2, 64)), {}, "1 sequences of queries, 2 of keys"),
    ((_t(4, 2, 80), _t(4, 2, 80), _t(4, 2, 80), CU), {}, "head dim must be one of"),
    ((_t(4, 3, 64), _t(4, 2, 64), _t(4, 2, 64), CU), {}, "no multiple of 2 key heads"),
    ((_t(4, 2, 64), _t(4, 2, 64), _t(4, 1, 64), CU), {}, "k and v alike"),
    ((_t(4, 64), _t(4, 64), _t(4, 64), CU), {}, "k and v alike"),
    ((_t(4, 2, 64), _t(5, 2, 64), _t(5, 2, 64), CU), {}, "need cu_seqlens_k"),
    ((_t(4, 2, 64), _t(4, 2, 64), _t(4, 2, 64), CU.long()), {}, "must be int32"),
    ((_t(4, 2, 64), _t(4, 2, 64), _t(4, 2, 64), CU, torch.tensor([0, 2, 4], dtype=torch.int32)), {}, "must be int32 of shape"),
    ((_t(4, 2, 64), _t(4, 2, 64), _t(4, 2, 64), CU), dict(scale=0.0), "positive and finite"),
    ((_t(4, 2, 64), _t(4, 2, 64), _t(4, 2, 64), CU), dict(scale=math.inf), "positive and finite"),
])
def test_causal_attention_refusals(args, kw, err, monkeypatch):
    _fake(monkeypatch)
    with pytest.raises(ValueError, match=err):
        A.causal_attention(*args, **kw)


def test_types_are_refused(monkeypatch):
    with pytest.raises(ValueError, match="ROCm device"):
        A.causal_attention(_t(4, 2, 64), _t(4, 2, 64), _t(4, 2, 64), CU)
    _fake(monkeypatch)
    for q, k in ((torch.float32, torch.float32), (torch.bfloat16, torch.float16)):
        with pytest.raises(TypeError, match="bfloat16 or all float16"):
            A.causal_attention(_t(4, 2, 64, dt=q), _t(4, 2, 64, dt=k), _t(4, 2, 64, dt=k), CU)


def _cache(pages=3, size=16, heads=2, d=64, n=2, most=2, dt=torch.bfloat16):
    kc, vc = A.alloc_kv_cache(pages, size, heads, d, dtype=dt, device="cpu")
    return kc, vc, torch.zeros((n, most), dtype=torch.int32), torch.zeros(n, dtype=torch.int32)


def test_cache_layout():
    kc, vc, _, _ = _cache()
    assert kc.shape == vc.shape == (3, 16, 2, 64) and kc.stride() == (2 * 16 * 64, 64, 16 * 64, 1)


@pytest.mark.parametrize("change,err", [
    (dict(size=12), "power of two"), (dict(size=4), "power of two"), (dict(size=8192), "power of two"),
    (dict(pages=0), "at least one page"), (dict(d=96), "head dim must be one of"), (dict(most=0), "page_table must be"),
])
def test_cache_refusals(change, err, monkeypatch):
    _fake(monkeypatch)
    kc, vc, table, lens = _cache(**change)
    q = _t(2, 4, kc.shape[3])
    with pytest.raises(ValueError, match=err):
        A.paged_attention(q, kc, vc, table, lens)
    with pytest.raises(ValueError, match=err):
        A.append_kv(kc, vc, table, lens, _t(2, 2, kc.shape[3]), _t(2, 2, kc.shape[3]))


def test_more_cache_refusals(monkeypatch):
    _fake(monkeypatch)
    kc, vc, table, lens = _cache()
    q, k = _t(2, 4, 64), _t(2, 2, 64)
    for call in (lambda: A.paged_attention(_t(3, 4, 64), kc, vc, table, lens), lambda: A.paged_attention(_t(2, 3, 64), kc, vc, table, lens),
                 lambda: A.paged_attention(q, kc, vc, table.long(), lens), lambda: A.paged_attention(q, kc, vc, table, lens[:1]),
                 lambda: A.paged_attention(q, kc[..., :32], vc[..., :32], table, lens),
                 lambda: A.paged_attention(q, kc[:, ::2][:, :8].transpose(1, 3).transpose(1, 3), vc, table, lens),
                 lambda: A.paged_attention(q, kc, vc, table, lens, scale=-1.0),
                 lambda: A.paged_attention(q.requires_grad_(True), kc, vc, table, lens),
                 lambda: A.append_kv(kc, vc, table, lens, _t(3, 2, 64), _t(3, 2, 64)),
                 lambda: A.append_kv(kc, vc, table, lens, k, _t(2, 1, 64)),
                 lambda: A.append_kv(kc, vc, table, lens, _t(2, 1, 64), _t(2, 1, 64)),
                 lambda: A.append_kv(kc, vc, table, lens, k, k, cu_seqlens=CU)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        A.append_kv(kc, vc, table, lens, k.half(), k.half())


FAKE = ctypes.c_void_p(256)


def _shape(**kw):
    d = dict(nseq=1, total_q=8, total_k=8, hq=4, hk=2, d=64, dtype=L.BF16)
    d.update(kw)
    return L.AttnShape(*(d[n] for n in ("nseq", "total_q", "total_k", "hq", "hk", "d", "dtype")))


def _fwd(shape, rows=None, cu=(None, None), scale=1.0, o=FAKE, ws=FAKE, nbytes=1 << 40):
    r = [ctypes.byref(x) for x in (rows or [L.AttnRows(256, 512, 64)] * 3)]
    return L.lib().lsurge_attn_fwd(ctypes.byref(shape), *r, *cu, scale, o, None, None, ws, nbytes, None)


def test_c_abi_forward_refusals():
    lib = L.lib()
    for kw, msg in ((dict(d=80), b"head_dim"), (dict(hq=3), b"query heads"), (dict(hk=0), b"query heads"), (dict(nseq=-1), b"nseq"),
                    (dict(total_q=1 << 30), b"total_q"), (dict(nseq=3), b"whole number"), (dict(nseq=0), b"whole number")):
        assert _fwd(_shape(**kw)) == -1 and msg in lib.lsurge_last_error(), lib.lsurge_last_error()
    assert _fwd(_shape(dtype=L.F32)) == -2
    assert _fwd(_shape(), scale=float("nan")) == -1 and b"scale" in lib.lsurge_last_error()
    assert _fwd(_shape(), cu=(FAKE, None)) == -1 and b"go together" in lib.lsurge_last_error()
    assert _fwd(_shape(), o=None) == -1
    good = L.AttnRows(256, 512, 64)
    for bad, msg in ((L.AttnRows(None, 512, 64), b"null"), (L.AttnRows(264, 512, 64), b"aligned"), (L.AttnRows(256, 510, 64), b"aligned"),
                     (L.AttnRows(256, 512, 4), b"aligned"), (L.AttnRows(256, 56, 64), b"row stride"), (L.AttnRows(256, 1 << 22, 64), b"row stride")):
        for i in range(3):
            rows = [good] * 3
            rows[i] = bad
            assert _fwd(_shape(), rows) == -1 and msg in lib.lsurge_last_error()
    assert _fwd(_shape(nseq=0, total_q=0, total_k=0)) == 0  # nothing to do
    few = _shape(total_q=16, total_k=16384)  # few rows over many keys: split, and the parts need room
    need = lib.lsurge_attn_fwd_workspace_bytes(ctypes.byref(few))
    assert need > 2 * 16 * 4 * 66 * 4 and lib.lsurge_attn_fwd_workspace_bytes(ctypes.byref(_shape())) == 0
    assert _fwd(few, nbytes=need - 1) == -4 and b"workspace" in lib.lsurge_last_error()
    assert _fwd(few, ws=None, nbytes=need) == -1 and _fwd(few, ws=ctypes.c_void_p(264), nbytes=need) == -1


def test_c_abi_backward_refusals():
    lib = L.lib()
    s, r = _shape(), ctypes.byref(L.AttnRows(256, 512, 64))
    need = lib.lsurge_attn_bwd_workspace_bytes(ctypes.byref(s))
    assert need >= 2 * 4 * 8 * 4
    assert lib.lsurge_attn_bwd_workspace_bytes(ctypes.byref(_shape(dtype=L.F16))) > need
    call = lambda o=FAKE, g=FAKE, dk=FAKE, ws=FAKE, n=need: lib.lsurge_attn_bwd(  # noqa: E731
        ctypes.byref(s), r, r, r, None, None, 1.0, o, None, FAKE, g, None, FAKE, dk, FAKE, ws, n, None)
    assert call(n=need - 1) == -4 and b"workspace" in lib.lsurge_last_error()
    assert call(ws=None) == -1 and call(o=None) == -1 and call(dk=None) == -1
    assert call(g=ctypes.c_void_p(264)) == -1 and b"aligned" in lib.lsurge_last_error()


def _kv(**kw):
    d = dict(k=256, v=256, k_page_stride=2048, k_slot_stride=64, k_head_stride=1024, v_page_stride=2048, v_slot_stride=64,
             v_head_stride=1024, page_table=256, table_stride=2, seq_lens=256, num_pages=3, page_size=16, max_pages=2, heads=2,
             d=64, dtype=L.BF16)
    d.update(kw)
    return L.KvCache(**d)


def test_c_abi_cache_refusals():
    lib = L.lib()
    r = ctypes.byref(L.AttnRows(256, 512, 64))
    ws = lib.lsurge_paged_attn_workspace_bytes(2, 4, 64)
    attn = lambda c, n=2, hq=4, scale=1.0, o=FAKE, nb=ws: lib.lsurge_paged_attn(  # noqa: E731
        ctypes.byref(c), r, n, hq, scale, o, None, FAKE, nb, None)
    put = lambda c, rows=2, n=2, cu=None, k=r: lib.lsurge_kv_append(ctypes.byref(c), k, r, rows, n, cu, None)  # noqa: E731
    for kw, msg in ((dict(d=32), b"head_dim"), (dict(heads=0), b"key heads"), (dict(num_pages=0), b"num_pages"),
                    (dict(max_pages=0), b"max_pages"), (dict(table_stride=1), b"table_stride"), (dict(page_size=24), b"page_size"),
                    (dict(page_size=4), b"page_size"), (dict(page_size=8192), b"page_size"), (dict(k=None), b"null"),
                    (dict(seq_lens=None), b"null"), (dict(v=264), b"aligned"), (dict(k_slot_stride=60), b"stride"),
                    (dict(v_page_stride=-8), b"stride")):
        for call in (attn, put):
            assert call(_kv(**kw)) == -1 and msg in lib.lsurge_last_error(), (kw, lib.lsurge_last_error())
    assert attn(_kv(dtype=L.F32)) == -2 and put(_kv(dtype=L.F32)) == -2
    assert attn(_kv(), hq=3) == -1 and attn(_kv(), scale=0.0) == -1 and attn(_kv(), o=None) == -1
    assert attn(_kv(), nb=ws - 1) == -4
    assert attn(_kv(max_pages=1 << 28, table_stride=1 << 28)) == -1
    assert put(_kv(), rows=3) == -1 and put(_kv(), k=None) == -1
    assert attn(_kv(), n=0) == 0 and put(_kv(), rows=0, n=0) == 0


def test_c_abi_refuses_grids_past_the_launch_limit():
    """Workgroups of 256 threads, less than 2^32 threads a launch: 2^24 tiles times heads are refused before anything runs."""
    lib = L.lib()
    for kw in (dict(hq=64), dict(hq=4, nseq=1 << 22)):
        s = _shape(total_q=1 << 29, total_k=1 << 29, **kw)
        assert _fwd(s) == -1 and b"tiles" in lib.lsurge_last_error()
        r = ctypes.byref(L.AttnRows(256, 512, 64))
        assert lib.lsurge_attn_bwd(ctypes.byref(s), r, r, r, None, None, 1.0, FAKE, None, FAKE, FAKE, None, FAKE, FAKE, FAKE,
                                   FAKE, 1 << 50, None) == -1 and b"tiles" in lib.lsurge_last_error()
    c = _kv()
    assert lib.lsurge_paged_attn(ctypes.byref(c), ctypes.byref(L.AttnRows(256, 512, 64)), 1 << 22, 4, 1.0, FAKE, None, FAKE,
                                 1 << 50, None) == -1 and b"sequences" in lib.lsurge_last_error()


def test_gradients_are_refused_at_the_cache(monkeypatch):
    _fake(monkeypatch)
    kc, vc, table, lens = _cache()
    k = _t(2, 2, 64)
    for args in ((kc, vc, k.clone().requires_grad_(True), k), (kc, vc, k, k.clone().requires_grad_(True)),
                 (kc.detach().requires_grad_(True), vc, k, k), (kc, vc.detach().requires_grad_(True), k, k)):
        with pytest.raises(ValueError, match="no gradient"):
            A.append_kv(args[0], args[1], table, lens, *args[2:])


class _Stub:
    """The library with calls that are noted instead of made."""

    def __init__(self, monkeypatch):
        self.calls = []
        monkeypatch.setattr(A.L, "require_cuda", lambda *_: None)
        monkeypatch.setattr(A.L, "lib", lambda: self)
        monkeypatch.setattr(A, "_call", lambda what, device, fn, *args: fn(*args))

    def __getattr__(self, name):
        return (lambda *_: 0) if name.endswith("_bytes") else lambda *_: self.calls.append(name)


def test_forward_mode_tangents_are_not_dropped(monkeypatch):
    stub = _Stub(monkeypatch)
    kc, vc, table, lens = _cache()
    q, k = _t(4, 2, 64), _t(2, 2, 64)
    with torch.autograd.forward_ad.dual_level():
        dual = lambda t: torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for i in range(3):
            args = [q, q, q]
            args[i] = dual(q)
            with pytest.raises(NotImplementedError, match="jvp"):
                A.causal_attention(*args, CU)
        stub.calls.clear()
        for i in range(3):
            args = [k, kc, vc]
            args[i] = dual(args[i])
            with pytest.raises(ValueError, match="no gradient"):
                A.paged_attention(*args, table, lens)
        for i in range(4):
            args = [kc, vc, table, lens, k, k]
            args[(0, 1, 4, 5)[i]] = dual(args[(0, 1, 4, 5)[i]])
            with pytest.raises(ValueError, match="no gradient"):
                A.append_kv(*args)
        assert not stub.calls  # nothing was written
        A.append_kv(kc, vc, table, lens, k, k)
        assert stub.calls == ["lsurge_kv_append"]


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning", "ignore::DeprecationWarning")
def test_a_trace_holds_the_calls(monkeypatch):
    """What torch.jit.trace records calls the kernels again, and returns their outputs instead of an empty tensor."""
    stub = _Stub(monkeypatch)
    kc, vc, table, lens = _cache()
    q, k = _t(4, 2, 64), _t(2, 2, 64)

    def step(k, v, q, table, lens):
        A.append_kv(kc, vc, table, lens, k, v)
        return A.paged_attention(q, kc, vc, table, lens)

    for f, args, names in ((lambda q, k, v, cu: A.causal_attention(q, k, v, cu), (q, q, q, CU), ["lsurge_attn_fwd"]),
                           (lambda q, k, v, cu: A.causal_attention(q, k, v, cu, return_lse=True), (q, q, q, CU), ["lsurge_attn_fwd"]),
                           (step, (k, k, k, table, lens), ["lsurge_kv_append", "lsurge_paged_attn"])):
        with torch.no_grad():
            traced = torch.jit.trace(f, args, check_trace=False)
        stub.calls.clear()
        traced(*args)
        assert stub.calls == names


def test_backward_workspace_is_bounded():
    """lse2 and delta of every query and head, the tiles' maxima in f16, and f32 sums of parts: up to 512 MiB, or 4 times dk
    and dv where that is more."""
    lib = L.lib()
    for nseq in (1, 4):
        for n in (1, 300, 4096, 32768, 131072, 1 << 20):
            for hq, hk in ((1, 1), (8, 8), (16, 2), (64, 8), (32, 32)):
                for d in (64, 128, 256):
                    s = _shape(nseq=nseq, total_q=nseq * n, total_k=nseq * n, hq=hq, hk=hk, d=d)
                    prep = 8 * nseq * n * hq
                    dkv = 2 * 2 * nseq * n * hk * d
                    assert lib.lsurge_attn_bwd_workspace_bytes(ctypes.byref(s)) <= prep + 512 + max(512 << 20, 4 * dkv)
