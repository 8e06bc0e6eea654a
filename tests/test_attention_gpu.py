"""Softmax attention on the GPU against the float64 oracle, every output element within the bound that the oracle derives
from the number of roundings (oracle/attention_oracle.py): prompts and training, and single tokens over a paged cache."""
import numpy as np
import pytest
import torch

import attention as A
from oracle import attention_oracle as ao

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
BF16, F16 = torch.bfloat16, torch.float16


def _np(t):
    return t.detach().double().cpu().numpy()


def _randn(gen, shape, dt, dev, std=1.0):
    return (torch.randn(shape, generator=gen, dtype=torch.float32) * std).to(dt).to(dev)


def _ends(lens, dev):
    return torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device=dev)


def _within(got, want, bound, what):
    got = _np(got) if torch.is_tensor(got) else got
    inf = ~np.isfinite(want)
    assert np.array_equal(got[inf], want[inf]), what
    err = np.abs(np.where(inf, 0, got) - np.where(inf, 0, want))
    assert np.isfinite(err).all(), what
    over = err - bound
    assert (over <= 0).all(), f"{what}: {(over > 0).sum()} elements out of bound, the worst {err.flat[over.argmax()]:.3e} " \
                              f"against {np.asarray(bound).flat[over.argmax()]:.3e}"


def check(q, k, v, lens_q, lens_k, scale, do=None, dlse=None, cu=True, tail=0):
    """One packed or dense call and its backward against the oracle, sequence by sequence."""
    dt, dev = q.dtype, q.device
    leaves = [t.detach().requires_grad_(do is not None) for t in (q, k, v)]
    ends = (_ends(lens_q, dev), _ends(lens_k, dev)) if cu else ()
    o, lse = A.causal_attention(*leaves, *ends, scale=scale, return_lse=True)
    assert o.dtype == dt and o.shape == q.shape and lse.shape == q.shape[:-1] and lse.dtype == torch.float32
    got = [o, lse]
    if do is not None:
        up = [(o, do)] + ([(lse, dlse)] if dlse is not None else [])
        got += torch.autograd.grad([a for a, _ in up], leaves, [b for _, b in up])
    torch.cuda.synchronize()
    flat = lambda t: t if t is None or cu else t.reshape(-1, *t.shape[2:])  # noqa: E731
    got = [_np(flat(t)) for t in got]
    q, k, v, do, dlse = (None if t is None else _np(flat(t)) for t in (q, k, v, do, dlse))
    a = e = 0
    for m, n in zip(lens_q, lens_k):
        qs, ks = slice(a, a + m), slice(e, e + n)
        one = [q[qs], k[ks], v[ks]]
        g = None if do is None else do[qs]
        want = list(ao.attention(*one, scale))
        dl = None
        if dlse is not None:
            dl = np.where(np.isfinite(want[1]), dlse[qs], 0)
        bound = ao.bounds(*one, scale, HALF_STEP[dt], do=g, dlse=dl)
        if do is not None:
            want += ao.attention_bwd(*one, g, scale, dl)
        for name, x, y, b, rows in zip(("o", "lse", "dq", "dk", "dv"), got, want, bound, (qs, qs, qs, ks, ks)):
            _within(x[rows], y, b, f"{name} of {m} queries over {n} keys")
        a, e = a + m, e + n
    if tail:
        assert not got[0][a:].any() and np.isneginf(got[1][a:]).all()
        for g in got[2:]:
            assert not g[e if g.shape[1] == k.shape[1] and g.shape[0] == k.shape[0] else a:].any()


def run(dt, D, hq, hk, lens_q, lens_k, dev, seed=0, backward=True, dlse=False, scale=None, tail=0):
    gen = torch.Generator().manual_seed(seed)
    tq, tk = sum(lens_q) + tail, sum(lens_k) + tail
    q, k, v = (_randn(gen, (n, h, D), dt, dev, s) for n, h, s in ((tq, hq, 1.5), (tk, hk, 1.5), (tk, hk, 1.0)))
    do = _randn(gen, (tq, hq, D), dt, dev) if backward else None
    dl = torch.randn((tq, hq), generator=gen).to(dev) if dlse else None
    if tail:  # rows behind the last sequence are not read
        for t in (q, k, v):
            t[-tail:] = float("nan")
        do[-tail:] = 0
    check(q, k, v, lens_q, lens_k, D ** -0.5 if scale is None else scale, do, dl, tail=tail)


EDGES = [1, 2, 31, 32, 33, 63, 64, 65, 127, 129, 255, 256, 257, 300]


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_lengths_around_every_tile(dt, D, dev):
    run(dt, D, 2, 1, EDGES, EDGES, dev, seed=D)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("lens", [([5, 64, 1, 130], [5 + 300, 64 + 1, 1 + 511, 130 + 62]), ([40, 3, 7], [8, 0, 7]), ([0, 9, 0], [5, 9, 0])])
def test_keys_of_other_lengths(D, lens, dev):
    """Prefixes of cached keys, rows that see no key, sequences without queries or keys."""
    run(BF16, D, 4, 2, *lens, dev, seed=D + lens[0][0], dlse=True)
    run(F16, D, 2, 2, *lens, dev, seed=D)


@pytest.mark.parametrize("hq,hk", [(1, 1), (8, 8), (16, 2), (5, 1), (6, 2), (7, 7), (24, 3)])
def test_heads(hq, hk, dev):
    run(BF16, 64, hq, hk, [70, 1, 133], [70, 1, 133], dev, seed=hq)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_rows_behind_the_last_sequence(D, dev):
    run(BF16, D, 4, 2, [37, 200], [37, 200], dev, tail=517, seed=1)


def test_no_sequence_at_all(dev):
    q, k = torch.full((300, 2, 64), float("nan"), dtype=BF16, device=dev), torch.zeros((300, 1, 64), dtype=BF16, device=dev)
    o = A.causal_attention(q, k, k, torch.zeros(1, dtype=torch.int32, device=dev))
    assert not o.any()
    e = torch.zeros((0, 2, 64), dtype=BF16, device=dev, requires_grad=True)
    o = A.causal_attention(e, e, e, torch.zeros(1, dtype=torch.int32, device=dev))
    assert o.shape == e.shape and torch.autograd.grad(o.sum(), e)[0].shape == e.shape


@pytest.mark.parametrize("D", [64, 128, 256])
def test_many_sequences(D, dev):
    rng = np.random.default_rng(D)
    lens = [int(n) for n in rng.integers(0, 40, 700)]
    run(BF16, D, 1, 1, lens, lens, dev, seed=2, backward=D == 64)


@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64), (BF16, 256)])
def test_dense(dt, D, dev):
    gen = torch.Generator().manual_seed(5)
    q, k, v = (_randn(gen, (3, 150, h, D), dt, dev) for h in (4, 2, 2))
    do = _randn(gen, (3, 150, 4, D), dt, dev)
    check(q, k, v, [150] * 3, [150] * 3, D ** -0.5, do, cu=False)
    check(q[:, :70], k, v, [70] * 3, [150] * 3, 0.3, do[:, :70], cu=False)  # strided over the sequences: copied


@pytest.mark.parametrize("D", [64, 128, 256])
def test_strides(D, dev):
    """Views of one projection, heads before rows, and tensors that have to be copied (misaligned, expanded)."""
    gen = torch.Generator().manual_seed(6)
    n, lens = 210, [100, 110]
    rows = _randn(gen, (n, 8, D), BF16, dev)
    do = _randn(gen, (n, 4, D), BF16, dev)
    check(rows[:, :4], rows[:, 4:6], rows[:, 6:], lens, lens, D ** -0.5, do)
    heads = _randn(gen, (8, n, D), BF16, dev).transpose(0, 1)
    check(heads[:, :4], heads[:, 4:6], heads[:, 6:], lens, lens, D ** -0.5, do)
    flat = _randn(gen, (n * 8 * D + 1,), BF16, dev)[1:].view(n, 8, D)
    one = _randn(gen, (1, 2, D), BF16, dev).expand(n, 2, D)
    check(flat[:, :4], one, flat[:, 6:], lens, lens, D ** -0.5, do)


def test_long_rows(dev):
    """Many key stages, peaked and flat rows: large score jumps between stages (both directions)."""
    gen = torch.Generator().manual_seed(8)
    for dt, D in ((BF16, 128), (F16, 64), (BF16, 256)):
        q, k, v = (_randn(gen, (1, 1500, h, D), dt, dev) for h in (2, 1, 1))
        ramp = torch.linspace(-1, 1, 1500).view(1, -1, 1, 1).to(dev)
        do = _randn(gen, (1, 1500, 2, D), dt, dev)
        for kk in (k, (k * (4 + 3 * ramp)).to(dt), (k * (4 - 3 * ramp)).to(dt)):
            check(q, kk, v, [1500], [1500], D ** -0.5, do, cu=False)


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_few_rows_over_many_keys(dt, D, dev):
    """The keys cut into parts that are joined, forward and backward: chunks of new tokens over long prefixes, a sequence
    without queries, rows that see no key, rows behind the last sequence; and one dense sequence."""
    run(dt, D, 2, 1, [40, 0, 1, 130, 5], [2500, 700, 3000, 130 + 2200, 3], dev, seed=D, dlse=True, tail=70)
    gen = torch.Generator().manual_seed(D)
    q, k, v, do = (_randn(gen, (1, 2400, 1, D), dt, dev) for _ in range(4))
    check(q, k, v, [2400], [2400], D ** -0.5, do, cu=False)


def test_small_gradients_in_f16(dev):
    """Upstream gradients near the bottom of f16's normal range, rows of very different sizes, long flat rows."""
    gen = torch.Generator().manual_seed(9)
    q, k, v = (_randn(gen, (1, 2000, 1, 64), F16, dev, 0.1) for _ in range(3))
    do = _randn(gen, (1, 2000, 1, 64), F16, dev) * 2.0 ** -8
    do[:, ::3] *= 2.0 ** -4
    check(q, k, v * 10, [2000], [2000], 0.125, do, cu=False)
    check(q * 20, k, v * 1000, [2000], [2000], 0.125, do * 256, cu=False)  # and values in the hundreds, peaked rows


def test_extreme_scores(dev):
    """Scores of +-1e4 and weights that underflow; a key of infinite score gives NaN, a masked one changes nothing."""
    gen = torch.Generator().manual_seed(10)
    q, k, v = (_randn(gen, (1, 200, 1, 64), BF16, dev) for _ in range(3))
    check(q * 100, k * 8, v, [200], [200], 1.0, cu=False)
    base = A.causal_attention(q, k, v)
    k2 = k.clone()
    k2[:, 150] = float("nan")
    o = A.causal_attention(q, k2, v)
    assert torch.equal(o[:, :150], base[:, :150]) and o[:, 150:].isnan().all()


@pytest.mark.parametrize("dt,D", [(BF16, 64), (F16, 64), (F16, 128), (BF16, 256)])
def test_other_sequences_never_reach(dt, D, dev):
    """NaN and infinities everywhere in one sequence and behind the last leave the others' bits alone, gradients too."""
    gen = torch.Generator().manual_seed(13)
    lens, tail = [70, 150, 33, 1, 64], 50
    a, b = sum(lens[:1]), sum(lens[:2])
    t = [_randn(gen, (sum(lens) + tail, h, D), dt, dev) for h in (4, 2, 2, 4)]  # q, k, v, do
    bad = [x.clone() for x in t]
    for i, x in enumerate(bad):
        x[a:b] = float("nan") if i % 2 else float("inf")
        x[sum(lens):] = float("nan")
    out = []
    for q, k, v, do in (t, bad):
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
        o, lse = A.causal_attention(*leaves, _ends(lens, dev), return_lse=True)
        out.append([o.detach(), lse.detach(), *torch.autograd.grad(o, leaves, do)])
    for name, x, y in zip(("o", "lse", "dq", "dk", "dv"), *out):
        assert torch.equal(x[:a], y[:a]) and torch.equal(x[b:], y[b:]), name
        assert name == "lse" or not y[sum(lens):].any(), name


def test_rows_past_32_bits(dev):
    """Query rows, outputs and gradients of more than 2^31 elements: the last sequences are as if they were alone."""
    lens = [512] * 2049 + [300, 77]
    n, last, D = sum(lens), 377, 128
    q, do = (torch.zeros((n, 16, D), dtype=BF16, device=dev) for _ in range(2))
    k, v = (torch.zeros((n, 1, D), dtype=BF16, device=dev) for _ in range(2))
    gen = torch.Generator().manual_seed(14)
    part = [_randn(gen, (last, h, D), BF16, dev) for h in (16, 1, 1, 16)]
    for big, small in zip((q, k, v, do), part):
        big[-last:] = small
    assert q.numel() > 2 ** 31
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    o = A.causal_attention(*leaves, _ends(lens, dev))
    got = [o.detach(), *torch.autograd.grad(o, leaves, do)]
    a = 0
    for m in lens[-2:]:
        one = [_np(x[a:a + m]) for x in part]
        want = [ao.attention(*one[:3], D ** -0.5)[0], *ao.attention_bwd(*one, D ** -0.5)]
        bound = ao.bounds(*one[:3], D ** -0.5, HALF_STEP[BF16], do=one[3])
        for name, x, y, e in zip(("o", "dq", "dk", "dv"), got, want, [bound[0], *bound[2:]]):
            _within(x[x.shape[0] - last + a:][:m], y, e, name)
        a += m


def test_repeats_bitwise_on_another_stream(dev):
    gen = torch.Generator().manual_seed(11)
    lens = [513, 77, 1024]
    q, k, v = (_randn(gen, (sum(lens), h, 128), BF16, dev) for h in (4, 2, 2))
    do = _randn(gen, (sum(lens), 4, 128), BF16, dev)
    cu = _ends(lens, dev)

    def step():
        t = [x.detach().requires_grad_(True) for x in (q, k, v)]
        o = A.causal_attention(*t, cu)
        return [o.detach(), *torch.autograd.grad(o, t, do)]

    first = step()
    torch.cuda.synchronize()
    s = torch.cuda.Stream(dev)
    with torch.cuda.stream(s):
        again = step()
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_training_step_captured(dev):
    """A captured forward and backward, replayed on new inputs between eager work, equals the eager step."""
    gen = torch.Generator().manual_seed(12)
    lens = [130, 300]
    q, k, v = (_randn(gen, (430, h, 64), F16, dev).requires_grad_(True) for h in (4, 2, 2))
    do, cu = _randn(gen, (430, 4, 64), F16, dev), _ends(lens, dev)

    def step():
        o = A.causal_attention(q, k, v, cu)
        return [o.detach(), *torch.autograd.grad(o, (q, k, v), do)]

    s = torch.cuda.Stream(dev)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for i in range(4):
        with torch.no_grad():
            for t in (q, k, v, do):
                t.copy_(_randn(gen, t.shape, F16, dev))
            n = 100 + 50 * i
            cu.copy_(torch.tensor([0, n, 430], dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i


def test_ends_out_of_range_stay_inside(dev):
    """Sequence ends outside the rows or out of order are held to them: nothing outside the tensors is touched."""
    big = torch.full((1000, 2, 64), 3.0, dtype=BF16, device=dev)
    q = big[300:600]
    for cu in ([0, 200, 5000], [0, 250, 100, 300], [0, -5, 300], [100, 50, 20]):
        c = torch.tensor(cu, dtype=torch.int32, device=dev)
        t = [q.detach().requires_grad_(True) for _ in range(3)]
        o = A.causal_attention(*t, c)
        torch.autograd.grad(o, t, torch.ones_like(o))
    torch.cuda.synchronize()
    assert (big == 3).all()


# ------------------------------------------------------------------------------------ paged cache


def make_cache(gen, lens, size, hk, D, dt, dev, token_major=False, spare=2, most=None):
    """Scattered pages holding random tokens of the given lengths; every slot without a token holds NaN."""
    need = [-(-n // size) for n in lens]
    pages = sum(need) + spare
    if token_major:
        kc, vc = (torch.empty((pages, size, hk, D), dtype=dt, device=dev) for _ in range(2))
    else:
        kc, vc = A.alloc_kv_cache(pages, size, hk, D, dt, dev)
    kc.fill_(float("nan"))
    vc.fill_(float("nan"))
    perm = torch.randperm(pages, generator=gen)
    table = torch.full((len(lens), most or max([1] + need)), -1, dtype=torch.int32)
    ks, vs, at = [], [], 0
    for b, n in enumerate(lens):
        ids = perm[at:at + need[b]]
        at += need[b]
        table[b, :need[b]] = ids
        k, v = _randn(gen, (n, hk, D), dt, dev, 1.5), _randn(gen, (n, hk, D), dt, dev)
        if n:
            where = (ids[torch.arange(n) // size].to(dev), (torch.arange(n) % size).to(dev))
            kc[where], vc[where] = k, v
        ks.append(k)
        vs.append(v)
    return kc, vc, table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), ks, vs


def check_decode(dt, D, hq, hk, lens, size, dev, seed=0, lost=(), **kw):
    gen = torch.Generator().manual_seed(seed)
    kc, vc, table, sl, ks, vs = make_cache(gen, lens, size, hk, D, dt, dev, **kw)
    masks = [np.ones((1, n), bool) for n in lens]
    for b, i, bad in lost:
        table[b, i] = bad
        masks[b][0, i * size:(i + 1) * size] = False
    q = _randn(gen, (len(lens), hq, D), dt, dev, 1.5)
    o, lse = A.paged_attention(q, kc, vc, table, sl, return_lse=True)
    only = A.paged_attention(q, kc, vc, table, sl)
    torch.cuda.synchronize()
    assert torch.equal(o, only) and o.dtype == dt and lse.dtype == torch.float32
    o, lse = _np(o), _np(lse)
    for b, n in enumerate(lens):
        one = (_np(q[b:b + 1]), _np(ks[b]), _np(vs[b]), D ** -0.5)
        wo, wl = ao.attention(*one, mask=masks[b])
        bo, bl = ao.bounds(*one, HALF_STEP[dt], mask=masks[b])
        _within(o[b:b + 1], wo, bo, f"o of length {n}")
        _within(lse[b:b + 1], wl, bl, f"lse of length {n}")


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("size", [8, 32, 256])
def test_decode_lengths(dt, D, size, dev):
    check_decode(dt, D, 8, 2, [0, 1, 7, 8, 9, 31, 32, 33, 127, 128, 129, 0, 255, 257, 700], size, dev, seed=size)


@pytest.mark.parametrize("hq,hk", [(1, 1), (16, 16), (5, 1), (16, 1), (20, 1), (40, 2), (6, 3), (17, 17)])
def test_decode_heads(hq, hk, dev):
    check_decode(BF16, 128, hq, hk, [300, 5, 64], 16, dev, seed=hq)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_decode_one_long_sequence(D, dev):
    """Split over the whole GPU and joined, also where a share holds the ends of several sequences."""
    check_decode(BF16, D, 4, 1, [70001], 64, dev, seed=1)
    check_decode(F16, D, 2, 2, [9000, 1, 0, 20000, 130], 16, dev, seed=2)


def test_decode_many_sequences(dev):
    rng = np.random.default_rng(4)
    check_decode(BF16, 64, 2, 1, [int(n) for n in rng.integers(0, 300, 900)], 16, dev, seed=3)


def test_decode_token_major_cache_and_wide_table(dev):
    check_decode(BF16, 128, 8, 2, [100, 33, 0], 16, dev, seed=5, token_major=True, most=4096)


def test_decode_entries_that_name_no_page(dev):
    check_decode(BF16, 64, 4, 2, [100, 40, 20, 300], 16, dev, seed=6,
                 lost=[(0, 2, -1), (0, 6, 1 << 30), (1, 0, 99), (2, 0, -7), (2, 1, -1), (3, 5, -2 ** 31)])


def test_decode_lengths_past_the_table(dev):
    """Lengths outside [0, max_pages * page_size] are held to it."""
    gen = torch.Generator().manual_seed(7)
    kc, vc, table, sl, _, _ = make_cache(gen, [64, 64, 64], 16, 1, 64, BF16, dev)
    q = _randn(gen, (3, 2, 64), BF16, dev)
    want = A.paged_attention(q, kc, vc, table, sl)
    got = A.paged_attention(q, kc, vc, table, torch.tensor([64, 2 ** 31 - 1, -3], dtype=torch.int32, device=dev))
    torch.cuda.synchronize()
    assert torch.equal(got[:2], want[:2]) and not got[2].any()


def test_decode_values_behind_a_masked_key(dev):
    """A row's own infinite value reaches it; dead slots (NaN everywhere in these tests) never do."""
    gen = torch.Generator().manual_seed(8)
    kc, vc, table, sl, _, _ = make_cache(gen, [40], 16, 1, 64, BF16, dev)
    vc[table[0, 1].item(), 3] = float("inf")
    o = A.paged_attention(_randn(gen, (1, 1, 64), BF16, dev), kc, vc, table, sl)
    assert (o == float("inf")).all()


def test_decode_shared_pages(dev):
    """Sequences that share their first pages, and one that names a page twice, read what each of their entries names."""
    gen = torch.Generator().manual_seed(15)
    kc, vc = (_randn(gen, (6, 2, 32, 128), BF16, dev).transpose(1, 2) for _ in range(2))
    table = torch.tensor([[0, 1, 2], [0, 1, 3], [4, 4, 4]], dtype=torch.int32, device=dev)
    lens = [90, 70, 96]
    q = _randn(gen, (3, 8, 128), BF16, dev)
    o, lse = A.paged_attention(q, kc, vc, table, torch.tensor(lens, dtype=torch.int32, device=dev), return_lse=True)
    for b, n in enumerate(lens):
        k, v = (_np(torch.cat([c[i] for i in table[b].tolist()])[:n]) for c in (kc, vc))
        one, m = (_np(q[b:b + 1]), k, v, 128 ** -0.5), np.ones((1, n), bool)
        for name, x, y, e in zip(("o", "lse"), (o[b:b + 1], lse[b:b + 1]), ao.attention(*one, mask=m),
                                 ao.bounds(*one, 2.0 ** -8, mask=m)):
            _within(x, y, e, f"{name} {b}")


def test_offsets_past_32_bits(dev):
    """Pages more than 2^31 elements into the cache."""
    gen = torch.Generator().manual_seed(9)
    pages, size, D = 70000, 256, 128  # 2.29e9 elements: 4.6 GB for one cache, shared by keys and values
    c = torch.zeros((pages, 1, size, D), dtype=BF16, device=dev).transpose(1, 2)
    table = torch.tensor([[69999, 3, 69000]], dtype=torch.int32, device=dev)
    k = _randn(gen, (600, 1, D), BF16, dev)
    n = torch.tensor([600], dtype=torch.int32, device=dev)
    A.append_kv(c, c, table, n, k, k, cu_seqlens=torch.tensor([0, 600], dtype=torch.int32, device=dev))
    assert torch.equal(c[69000, :88], k[512:]) and torch.equal(c[69999], k[:256])
    q = _randn(gen, (1, 1, D), BF16, dev)
    o = _np(A.paged_attention(q, c, c, table, n))
    one = (_np(q), _np(k), _np(k), D ** -0.5)
    m = np.ones((1, 600), bool)
    _within(o, ao.attention(*one, mask=m)[0], ao.bounds(*one, 2.0 ** -8, mask=m)[0], "o")


@pytest.mark.parametrize("dt,D,size", [(BF16, 64, 8), (F16, 128, 16), (BF16, 256, 64)])
def test_append(dt, D, size, dev):
    gen = torch.Generator().manual_seed(D)
    old, new = [0, 5, 8, 100, 0, 63], [3, 1, 0, 40, 0, 130]
    lens = [a + b for a, b in zip(old, new)]
    kc, vc, table, _, _, _ = make_cache(gen, lens, size, 3, D, dt, dev)
    table[3, (120 // size)] = -1
    sl = torch.tensor(lens, dtype=torch.int32, device=dev)
    rows = sum(new) + 9  # and rows behind the last sequence
    qkv = _randn(gen, (rows, 8, D), dt, dev)
    k, v = qkv[:, 1:4], qkv[:, 4:7]
    wk, wv, at = kc.clone(), vc.clone(), 0
    for b, (m, n) in enumerate(zip(old, new)):
        for t in range(m, m + n):
            p = table[b, t // size].item()
            if p >= 0:
                wk[p, t % size], wv[p, t % size] = k[at], v[at]
            at += 1
    A.append_kv(kc, vc, table, sl, k, v, cu_seqlens=_ends(new, dev))
    torch.cuda.synchronize()
    assert torch.equal(kc.nan_to_num(7), wk.nan_to_num(7)) and torch.equal(vc.nan_to_num(7), wv.nan_to_num(7))


def test_append_one_token_each(dev):
    gen = torch.Generator().manual_seed(20)
    kc, vc, table, sl, _, _ = make_cache(gen, [1, 17, 0, 32], 16, 2, 64, BF16, dev)
    k, v = _randn(gen, (4, 2, 64), BF16, dev), _randn(gen, (4, 2, 64), BF16, dev)
    wk, wv = kc.clone(), vc.clone()
    for b, n in enumerate((1, 17, 0, 32)):
        if n:
            wk[table[b, (n - 1) // 16], (n - 1) % 16], wv[table[b, (n - 1) // 16], (n - 1) % 16] = k[b], v[b]
    A.append_kv(kc, vc, table, sl, k, v)
    assert torch.equal(kc.nan_to_num(7), wk.nan_to_num(7)) and torch.equal(vc.nan_to_num(7), wv.nan_to_num(7))


def test_append_is_a_write_in_place(dev):
    """A backward that saved the cache before a token was appended raises instead of using the new values."""
    gen = torch.Generator().manual_seed(16)
    kc, vc, table, sl, _, _ = make_cache(gen, [20], 16, 1, 64, BF16, dev)
    w = torch.ones(64, dtype=BF16, device=dev, requires_grad=True)
    y = (kc * w).sum()
    k = _randn(gen, (1, 1, 64), BF16, dev)
    A.append_kv(kc, vc, table, sl, k, k)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_prompt_then_tokens(dev):
    """The operators as a serving program runs them: packed prompts through causal_attention and into the cache, then
    tokens one by one, each step captured once and replayed; every token's output equals whole-sequence attention."""
    gen = torch.Generator().manual_seed(21)
    hq, hk, D, size, steps = 4, 2, 128, 16, 5
    lens = [37, 1, 130]
    full = [n + steps for n in lens]
    qkv = [_randn(gen, (n, hq + 2 * hk, D), BF16, dev, 1.2) for n in full]
    prompt = torch.cat([t[:n] for t, n in zip(qkv, lens)])
    kc, vc = A.alloc_kv_cache(40, size, hk, D, BF16, dev)
    table = torch.randperm(40, generator=gen)[:30].view(3, 10).to(torch.int32).to(dev)
    sl, cu = torch.tensor(lens, dtype=torch.int32, device=dev), _ends(lens, dev)
    with torch.no_grad():
        o = A.causal_attention(prompt[:, :hq], prompt[:, hq:hq + hk], prompt[:, hq + hk:], cu)
        A.append_kv(kc, vc, table, sl, prompt[:, hq:hq + hk], prompt[:, hq + hk:], cu_seqlens=cu)
        got = [[o[cu[b]:cu[b + 1]]] for b in range(3)]
        tok = torch.empty((3, hq + 2 * hk, D), dtype=BF16, device=dev)

        def step():
            A.append_kv(kc, vc, table, sl, tok[:, hq:hq + hk], tok[:, hq + hk:])
            return A.paged_attention(tok[:, :hq], kc, vc, table, sl)

        tok.copy_(torch.stack([t[n] for t, n in zip(qkv, lens)]))
        sl += 1
        s = torch.cuda.Stream(dev)
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step()
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        for i in range(steps):
            tok.copy_(torch.stack([t[n + i] for t, n in zip(qkv, lens)]))
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, A.paged_attention(tok[:, :hq], kc, vc, table, sl))
            for b in range(3):
                got[b].append(out[b:b + 1].clone())
            sl += 1
    for b, t in enumerate(qkv):
        one = (_np(t[:, :hq]), _np(t[:, hq:hq + hk]), _np(t[:, hq + hk:]), D ** -0.5)
        _within(_np(torch.cat(got[b])), ao.attention(*one)[0], ao.bounds(*one, 2.0 ** -8)[0], f"sequence {b}")


def shared_cache(k, v, size, rows, dt, dev):
    """One sequence's tokens k, v [n, Hkv, D] in a cache whose table gives its pages to every one of `rows` sequences."""
    n, hk, D = k.shape
    pages = -(-n // size)
    kc, vc = A.alloc_kv_cache(pages + 1, size, hk, D, dt, dev)
    perm = torch.randperm(pages + 1, generator=torch.Generator().manual_seed(n))[:pages]
    where = (perm.to(dev)[torch.arange(n, device=dev) // size], torch.arange(n, device=dev) % size)
    kc[where], vc[where] = k.to(dev), v.to(dev)
    return kc, vc, perm.to(torch.int32).to(dev).expand(rows, pages)


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_decode_equal_scores_over_many_units(dt, D, dev):
    """Every weight of a row is the same, whatever part of the sequence it comes from: keys all alike, values 1 in the first
    half and -1 in the second, hundreds of units of one sequence in a share.  Then o = 0 and lse = s + log n but for the f32
    sums: a share adds up 512 units of 8 keys a lane and joins 16 lanes' and 4 waves' sums, 540 roundings of 2^-24 at most,
    each relative to at most the whole; s = 3.4 (D = 64) to 6.8 times a power of two is exact, and its product with the
    scale and log2 e, the sum of logarithms, its factor log 2 are rounded to half of 2^-23 |lse|, four times."""
    n, rows = 65536, 768
    k = torch.full((n, 1, D), 1.6875).to(dt)
    v = torch.ones((n, 1, D)).to(dt)
    v[n // 2:] = -1
    kc, vc, table = shared_cache(k, v, 64, rows, dt, dev)
    level = torch.tensor([0.34375, 2.203125, 5.40625, -3.3125])  # scores of some tens of nats, both signs
    q = level.repeat(rows // 4).view(-1, 1, 1).expand(rows, 1, D).to(dt).to(dev)
    o, lse = A.paged_attention(q, kc, vc, table, torch.full((rows,), n, dtype=torch.int32, device=dev), scale=0.125,
                               return_lse=True)
    s = 0.125 * D * 1.6875 * level.double().numpy()
    want = np.tile(s + np.log(n), rows // 4)[:, None]
    _within(lse, want, 540 * 2.0 ** -24 + 4 * 2.0 ** -24 * np.abs(want), "lse")
    _within(o, np.zeros(o.shape), np.full(o.shape, 540 * 2.0 ** -24), "o")


def grads(q, k, v, do, lens, dlse=None, scale=None):
    """o, lse, dq, dk, dv of packed sequences, lens (queries, keys) of each."""
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    ends = [_ends([n[i] for n in lens], q.device) for i in (0, 1)]
    o, lse = A.causal_attention(*leaves, *ends, scale=scale, return_lse=True)
    up = [(a, b) for a, b in ((o, do), (lse, dlse)) if b is not None]
    return [o.detach(), lse.detach(), *torch.autograd.grad([a for a, _ in up], leaves, [b for _, b in up])]


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("others", [2.0 ** 14, float("inf")])
def test_f16_gradients_do_not_depend_on_other_documents(D, others, dev):
    """A document's gradients are the same bits beside a document whose upstream gradients are 2^20 times larger, or
    infinite, and within the bounds that its own sizes give."""
    gen = torch.Generator().manual_seed(D)
    lens = [(300, 300), (257, 257), (500, 500)]
    n, a, b = 1057, 300, 557
    q, k, v, do = (_randn(gen, (n, h, D), F16, dev) for h in (4, 2, 2, 4))
    do *= 2.0 ** -6
    alone = grads(q, k, v, do, lens)
    loud = do.clone()
    loud[a:b] *= others
    got = grads(q, k, v, loud, lens)
    for name, x, y in zip(("o", "lse", "dq", "dk", "dv"), alone, got):
        assert torch.equal(x[:a], y[:a]) and torch.equal(x[b:], y[b:]), name
    check(*(t[b:] for t in (q, k, v)), [500], [500], D ** -0.5, do[b:])
    if others < 65504:
        check(*(t[:, :] for t in (q, k, v)), *([m for m, _ in lens],) * 2, D ** -0.5, loud)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("size", [2.0 ** -10, 2.0 ** 5, 2.0 ** 11])
def test_f16_values_of_every_size(D, size, dev):
    """Score gradients p (do . v - delta) that are much larger or smaller than do: values of thousands and of thousandths,
    peaked and flat rows, chunks whose keys are cut into parts."""
    gen = torch.Generator().manual_seed(D)
    for std, lens in ((2.0, [200, 77, 1]), (0.3, [700])):
        n = sum(lens)
        q, k, v, do = (_randn(gen, (n, h, D), F16, dev, s) for h, s in ((4, std), (2, std), (2, size), (4, 1 / size)))
        check(q, k, v, lens, lens, D ** -0.5, do)
    q, k, v, do = (_randn(gen, (m, 2, D), F16, dev, s) for m, s in ((40, 1.0), (2500, 1.0), (2500, size), (40, 0.25 / size)))
    check(q, k, v, [40], [2500], D ** -0.5, do)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_f16_gradients_of_lse(D, dev):
    """Score gradients that come from lse alone, or that lse's upstream gradient makes larger than do by far."""
    gen = torch.Generator().manual_seed(D)
    q, k, v = (_randn(gen, (270, h, D), F16, dev, 1.5) for h in (4, 2, 2))
    do = _randn(gen, (270, 4, D), F16, dev)
    dl = torch.randn((270, 4), generator=gen).to(dev)
    lens = [200, 70]
    for a, b in ((0.0, 1.0), (0.0, 2000.0), (2.0 ** -7, 300.0)):
        check(q, k, v, lens, lens, D ** -0.5, do * a, dl * b)
    got = grads(q, k, v, None, [(200, 200), (70, 70)], dl)
    assert all(torch.equal(x, y) for x, y in zip(got, grads(q, k, v, do * 0, [(200, 200), (70, 70)], dl)))


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_lse_gradient_of_rows_without_keys(dt, D, dev):
    """lse is the constant -inf where a row sees no key, so its upstream gradient there counts for nothing, whatever it is:
    one taken through a join of two such parts is NaN."""
    gen = torch.Generator().manual_seed(D)
    lens = [(45, 8), (70, 70), (9, 0)]  # 37 rows without a key: some share a stage of 32 with rows that have some
    q, k, v, do = (_randn(gen, (m, h, D), dt, dev) for m, h in ((124, 4), (78, 2), (78, 2), (124, 4)))
    dl = torch.randn((124, 4), generator=gen).to(dev)
    dl[:37] = dl[115:] = 0
    want = grads(q, k, v, do, lens, dl)
    assert torch.isneginf(want[1][:37]).all() and torch.isneginf(want[1][115:]).all()
    for bad in (float("nan"), float("inf"), 7.0):
        dl[:37] = dl[115:] = bad
        for name, x, y in zip(("o", "lse", "dq", "dk", "dv"), want, grads(q, k, v, do, lens, dl)):
            assert torch.equal(x, y), (bad, name)


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning", "ignore::DeprecationWarning")
def test_traced_serving_step(dev):
    """A prompt's attention and a token's, traced, compute on new inputs what the calls themselves do."""
    gen = torch.Generator().manual_seed(23)
    kc, vc, table, sl, _, _ = make_cache(gen, [20, 33], 16, 2, 64, BF16, dev)
    cu = _ends([20, 33], dev)

    def prompt(q, k, v):
        return A.causal_attention(q, k, v, cu, return_lse=True)

    def token(q, k, v):
        A.append_kv(kc, vc, table, sl, k, v)
        return A.paged_attention(q, kc, vc, table, sl)

    draw = lambda n: [_randn(gen, (n, h, 64), BF16, dev) for h in (4, 2, 2)]  # noqa: E731
    with torch.no_grad():
        p, t = (torch.jit.trace(f, tuple(draw(n)), check_trace=False) for f, n in ((prompt, 53), (token, 2)))
        for _ in range(2):
            x, y = draw(53), draw(2)
            assert all(torch.equal(a, b) for a, b in zip(p(*x), prompt(*x)))
            got, rows = t(*y), kc.clone()
            assert torch.equal(got, token(*y)) and torch.equal(rows.nan_to_num(7), kc.nan_to_num(7))


# One key holds nearly all of a row's weight; 65535 others of value 1 hold 2^-25.5 of it each, less than half of f16's least
# subnormal, and W = 1/720 of it together.
FLAT_KEYS, FLAT = 65536, 65535 * 2.0 ** -25.5


def flat_rows(D, value):
    """Keys, values and the scale that with queries of ones makes the scores; `value` is that of the one."""
    k, v = torch.zeros((FLAT_KEYS, 1, D), dtype=F16), torch.ones((FLAT_KEYS, 1, D), dtype=F16)
    k[FLAT_KEYS // 3], v[FLAT_KEYS // 3] = 1.0, value
    return k, v, 25.5 * np.log(2) / D


@pytest.mark.parametrize("D", [64, 128, 256])
def test_f16_decode_weights_far_below_the_largest(D, dev):
    """Value 0 for the one: o = W / (1 + W).  The others' weights are held as 2^-10.5, within 2^-11 of themselves, o is
    rounded to 2^-11, and 2^-12 is for f32's sums and exponents."""
    k, v, scale = flat_rows(D, 0.0)
    rows = 768
    kc, vc, table = shared_cache(k, v, 64, rows, F16, dev)
    q = torch.ones((rows, 1, D), dtype=F16, device=dev)
    o = A.paged_attention(q, kc, vc, table, torch.full((rows,), FLAT_KEYS, dtype=torch.int32, device=dev), scale=scale)
    want = np.full(o.shape, FLAT / (1 + FLAT))
    _within(o, want, want * (2 * 2.0 ** -11 + 2.0 ** -12), "o")


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_f16_forward_weights_far_below_the_largest(D, grad, dev):
    """Value -1 for the one: o = (W - 1) / (W + 1), -0.997.  The others' weights are held as 2^-21.5 at least (the base may
    lag behind the largest score by 2^8), within half a subnormal step, 2^-25, or 2^-3.5 of themselves, which counts twice
    in o; o's own rounding is 2^-12 of less than 1, but 2^-11 is allowed, and 2^-20 for f32.  128 rows of 768 heads leave the
    keys in one part; the last rows see up to 127 keys more, of weight e^-1060."""
    k, v, scale = (x.to(dev) if torch.is_tensor(x) else x for x in flat_rows(D, -1.0))
    k = torch.cat([k, torch.full((127, 1, D), -60.0, dtype=F16, device=dev)])
    v = torch.cat([v, torch.ones((127, 1, D), dtype=F16, device=dev)])
    q = torch.ones((1, 128, 768, D), dtype=F16, device=dev)
    o = A.causal_attention(q, *(x[None].detach().requires_grad_(grad) for x in (k, v)), scale=scale).detach()
    assert o.shape == q.shape and (o == o[:, :, :1, :1]).all()
    o = o[0, :, 0, :1]
    _within(o, np.full(o.shape, (FLAT - 1) / (FLAT + 1)), np.full(o.shape, 2 * FLAT * 2.0 ** -3.5 + 2.0 ** -11 + 2.0 ** -20), "o")


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_decode_many_units_of_a_sequence_in_a_share(dt, D, dev):
    """Shares of 5 and more units of 128 keys of one sequence and head (odd and even numbers of them), borders of sequences
    inside a share, lengths that end inside a tile: 300 sequences of 1 to 2300 tokens, 2 key heads."""
    gen = torch.Generator().manual_seed(D)
    n, rows = 2300, 300
    k, v = _randn(gen, (n, 2, D), dt, "cpu", 1.5), _randn(gen, (n, 2, D), dt, "cpu")
    kc, vc, table = shared_cache(k, v, 16, rows, dt, dev)
    lens = [2300, 1, 0, 640, 641, 767, 768, 769, 1024] + [int(x) for x in np.random.default_rng(D).integers(900, n, rows - 9)]
    q = _randn(gen, (rows, 4, D), dt, dev, 1.5)
    o, lse = A.paged_attention(q, kc, vc, table, torch.tensor(lens, dtype=torch.int32, device=dev), return_lse=True)
    o, lse = _np(o), _np(lse)
    for b, m in enumerate(lens):
        if b > 40 and b % 8:
            continue
        one = (_np(q[b:b + 1]), _np(k[:m]), _np(v[:m]), D ** -0.5)
        mask = np.ones((1, m), bool)
        for name, x, y, e in zip(("o", "lse"), (o[b:b + 1], lse[b:b + 1]), ao.attention(*one, mask=mask),
                                 ao.bounds(*one, HALF_STEP[dt], mask=mask)):
            _within(x, y, e, f"{name} of length {m}")


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_lengths_around_every_tile_without_gradients(dt, D, dev):
    """The serving forward, which is compiled apart from the one that keeps what a backward needs."""
    run(dt, D, 2, 1, EDGES, EDGES, dev, seed=D, backward=False)
    run(dt, D, 4, 2, [5, 64, 1, 130], [5 + 300, 64 + 1, 1 + 511, 130 + 62], dev, seed=D, backward=False)
    run(dt, D, 4, 2, [40, 3, 7, 0, 9], [8, 0, 7, 5, 9], dev, seed=D, backward=False)


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_few_rows_over_many_keys_without_gradients(dt, D, dev):
    run(dt, D, 2, 1, [40, 0, 1, 130, 5], [2500, 700, 3000, 130 + 2200, 3], dev, seed=D, backward=False)
    gen = torch.Generator().manual_seed(D)
    q, k, v = (_randn(gen, (1, 2400, 1, D), dt, dev) for _ in range(3))
    check(q, k, v, [2400], [2400], D ** -0.5, cu=False)


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_long_rows_without_gradients(dt, D, dev):
    """Many turns of the stages' ring in one part: 8 heads of 12 dense sequences leave the keys whole.  Rising and falling
    scores move the base of the weights."""
    gen = torch.Generator().manual_seed(8)
    n, b, h = 1100, 12, 8
    ramp = torch.linspace(-1, 1, n).view(1, -1, 1, 1).to(dev)
    q, k, v = (_randn(gen, (b, n, x, D), dt, dev) for x in (h, 2, 2))
    for kk in (k, (k * (4 + 3 * ramp)).to(dt), (k * (4 - 3 * ramp)).to(dt)):
        o, lse = A.causal_attention(q, kk, v, return_lse=True)
        for i in (0, b - 1):
            one = [_np(t[i]) for t in (q, kk, v)]
            for name, x, y, e in zip(("o", "lse"), (o[i], lse[i]), ao.attention(*one, D ** -0.5),
                                     ao.bounds(*one, D ** -0.5, HALF_STEP[dt])):
                _within(x, y, e, name)


@pytest.mark.parametrize("dt,D", [(BF16, 64), (F16, 64), (BF16, 128), (F16, 256)])
def test_c_abi_backward_without_the_left_over(dt, D, dev):
    """o_lo may be NULL for the backward: o is then taken as it was rounded, for which delta is off by u |do| |o| more."""
    import _lib as L
    gen = torch.Generator().manual_seed(D)
    n, hq, hk, u, scale = 333, 4, 2, HALF_STEP[dt], D ** -0.5
    q, k, v, do = (_randn(gen, (n, h, D), dt, dev) for h in (hq, hk, hk, hq))
    o, lse = A.causal_attention(q, k, v, _ends([n], dev), return_lse=True)
    shape = L.AttnShape(1, n, n, hq, hk, D, L.dt(q))
    lse_t, grads_ = lse.t().contiguous(), [torch.empty_like(t) for t in (q, k, v)]
    ws = L.workspace(L.lib().lsurge_attn_bwd_workspace_bytes(shape), dev)
    rows = [L.AttnRows(t.data_ptr(), t.stride(0), t.stride(1)) for t in (q, k, v)]
    L.check(L.lib().lsurge_attn_bwd(shape, *rows, None, None, scale, L.ptr(o), None, L.ptr(lse_t), L.ptr(do), None,
                                    *(L.ptr(t) for t in grads_), L.ptr(ws), ws.numel(), L.stream(dev)), "attn_bwd")
    one, g = [_np(t) for t in (q, k, v)], _np(do)
    bound = ao.bounds(*one, scale, u, do=g)[2:]
    _, w, _ = ao._weights(*one[:2], scale)
    ed = w * (np.abs(g) * u * np.abs(_np(o))).sum(-1).T[..., None]  # of ds
    more = (scale * (ed @ np.abs(ao._heads(one[1], 2))).transpose(1, 0, 2),
            scale * (ed.transpose(0, 2, 1) @ np.abs(one[0].transpose(1, 0, 2))).reshape(hk, 2, n, D).sum(1).transpose(1, 0, 2), 0.0)
    for name, x, y, b, m in zip(("dq", "dk", "dv"), grads_, ao.attention_bwd(*one, g, scale), bound, more):
        _within(x, y, b + m, name)


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning", "ignore::DeprecationWarning")
def test_traced_without_gradients_then_trained(dev):
    gen = torch.Generator().manual_seed(24)
    cu = _ends([20, 33], dev)
    draw = lambda: [_randn(gen, (53, h, 64), BF16, dev) for h in (4, 2, 2)]  # noqa: E731
    call = lambda q, k, v: A.causal_attention(q, k, v, cu, return_lse=True)  # noqa: E731
    with torch.no_grad():
        traced = torch.jit.trace(call, tuple(draw()), check_trace=False)
    do, dl = _randn(gen, (53, 4, 64), BF16, dev), torch.randn((53, 4), generator=gen).to(dev)
    for _ in range(3):
        x = [t.requires_grad_(True) for t in draw()]
        got, want = traced(*x), call(*x)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(got, x, (do, dl)), torch.autograd.grad(want, x, (do, dl))))


@pytest.mark.parametrize("D", [64, 128, 256])
def test_f16_scores_past_the_roundings_of_their_base(D, dev):
    """Scores of 2^24 to 2^25.5, in base 2 up to 2^26, where an f32 step is 4.  The scores are exact here (17 bits and the 4 of
    a sum over D / 16), so each row is the mean of the values at its largest ones, whose weights are alike, rounded to 2^-11 of
    themselves, and o to 2^-11.  lse has six roundings in f32: log2 e, its product with the score, the room below it, the
    logarithm of the sum added, log 2, its product."""
    gen = torch.Generator().manual_seed(D)
    n, scale = 300, 8 / D
    k, v = torch.full((n, 1, D), 2048.0, dtype=F16), _randn(gen, (n, 1, D), F16, "cpu")
    k[7] = k[200] = 3008.0
    q = (1025.0 + 3 * torch.arange(n)).view(n, 1, 1).repeat(1, 2, D).to(F16)
    q[:, 1] *= -1  # the largest scores are the small keys'
    want, want_lse = ao.attention(_np(q), _np(k), _np(v), scale)
    off = 2.1 * 2.0 ** -11 * ao.attention(_np(q), _np(k), np.abs(_np(v)), scale)[0]
    step = 6 * 2.0 ** -24 * np.abs(want_lse)
    for grad in (False, True):
        o, lse = A.causal_attention(q[None].to(dev), *(t[None].to(dev).requires_grad_(grad) for t in (k, v)), scale=scale,
                                    return_lse=True)
        _within(lse[0], want_lse, step, "lse")
        _within(o[0], want, off, "o")
    kc, vc, table = shared_cache(k, v, 16, n, F16, dev)
    lens = torch.arange(1, n + 1, dtype=torch.int32, device=dev)
    o, lse = A.paged_attention(q.to(dev), kc, vc, table, lens, scale=scale, return_lse=True)
    _within(lse, want_lse, step, "lse, decode")
    _within(o, want, off, "o, decode")
