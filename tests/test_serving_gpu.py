"""The operators that carry a hybrid model's sequences from token to token, on the GPU: every output within the bounds that the
float64 oracle derives from the roundings (oracle/serving_oracle.py); what has to stay as it was compared bit for bit."""
import ctypes

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

import _lib as L
import attention as A
import fast_conv as FC
import gdn_fast as G
from oracle import serving_oracle as so

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
NAME = {BF16: "bf16", F16: "f16"}


def _np(t):
    return t.detach().double().cpu().numpy()


def _randn(gen, shape, dt, dev, std=1.0):
    return (torch.randn(shape, generator=gen) * std).to(dt).to(dev)


def _ends(lens, dev):
    return torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device=dev)


def _i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def _starts(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(int)


# ----------------------------------------------------------------------------------------------- gated delta rule


class Rule:
    """Inputs of packed sequences: q, k, v views of one projection's rows, scattered slots, `tail` rows behind the last."""

    def __init__(self, dt, hk, hv, lens, dev, seed=0, norm=True, beta32=False, tail=0, extra=3, decay=0.05, unit=None):
        gen = torch.Generator().manual_seed(seed)
        n = sum(lens) + tail
        rows = _randn(gen, (n, 2 * hk + hv, 128), dt, dev)
        self.q, self.k, self.v = rows[:, :hk], rows[:, hk:2 * hk], rows[:, 2 * hk:]
        if not norm if unit is None else unit:
            self.k.copy_((self.k.float() / self.k.float().norm(dim=-1, keepdim=True)).to(dt))
        self.g = (-decay * torch.exp(torch.randn((n, hv), generator=gen))).to(dev)
        self.beta = torch.sigmoid(torch.randn((n, hv), generator=gen)).to(F32 if beta32 else dt).to(dev)
        self.state = (torch.randn((len(lens) + extra, hv, 128, 128), generator=gen) * 0.1).to(dev)
        self.slots = [int(s) for s in torch.randperm(len(lens) + extra, generator=gen)[:len(lens)]]
        self.lens, self.norm, self.tail, self.dt, self.dev = lens, norm, tail, dt, dev
        if tail:
            for t in (self.q, self.k, self.v, self.g, self.beta):
                t[-tail:] = float("nan")

    def call(self, cu=True, slots=None, state=None):
        slots = self.slots if slots is None else slots
        return G.recurrent_gated_delta_rule(
            self.q, self.k, self.v, self.g, self.beta, self.state if state is None else state,
            state_slots=_i32(slots, self.dev), cu_seqlens=_ends(self.lens, self.dev) if cu else None,
            use_qk_norm_in_gdn=self.norm)

    def check(self, o, before, after, terms=32):
        """o and the states within their bounds, sequence by sequence; slots of no sequence as they were."""
        assert o.dtype == self.dt and o.shape == self.v.shape
        o, q, k, v, g, beta, new = (_np(t) for t in (o, self.q, self.k, self.v, self.g, self.beta, after))
        u, tiny = so.HALF_STEP[NAME[self.dt]], so.TINY[NAME[self.dt]]
        at = _starts(self.lens)
        for b, (a, n) in enumerate(zip(at, self.lens)):
            if n == 0:
                continue
            r = slice(a, a + n)
            S0 = _np(before[self.slots[b]])
            wo, wS, bo, bS = so.delta_rule(q[r], k[r], v[r], g[r], beta[r], S0, self.norm, terms)
            off = np.linalg.norm(new[self.slots[b]] - wS, axis=(1, 2))
            assert (off <= bS).all(), f"state of sequence {b} ({n} rows): {off.max():.2e} against {bS[off.argmax()]:.2e}"
            off = np.linalg.norm(o[r] - wo, axis=-1)
            bound = bo + u * (np.linalg.norm(wo, axis=-1) + bo) + 128 ** 0.5 * tiny
            assert (off <= bound).all(), f"o of sequence {b} ({n} rows): {(off - bound).max():.2e} over"
        assert not o[at[-1]:].any()
        kept = [s for s in range(before.shape[0]) if s not in [x for x, n in zip(self.slots, self.lens) if n]]
        assert torch.equal(before[kept], after[kept])


def run_rule(*args, cu=True, **kw):
    r = Rule(*args, **kw)
    before = r.state.clone()
    o = r.call(cu)
    torch.cuda.synchronize()
    r.check(o, before, r.state)


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("hk,hv", [(1, 1), (4, 8), (2, 8), (3, 3), (1, 5)])
def test_rule_one_token_each(dt, hk, hv, dev):
    for n in (1, 2, 37):
        run_rule(dt, hk, hv, [1] * n, dev, seed=n, cu=False, norm=n != 2, beta32=n == 1)


@pytest.mark.parametrize("hv", [1, 8, 40])
def test_rule_batches_of_every_column_rule(hv, dev):
    """Batches on both sides of the numbers at which a wave takes more columns."""
    for n in (300, 30) if hv == 40 else (300,):
        run_rule(BF16, hv, hv, [1] * n, dev, seed=hv, cu=False)


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("beta32", [False, True])
@pytest.mark.parametrize("hv,n", [(1, 255), (1, 256), (1, 257), (5, 51), (5, 52), (8, 31), (8, 32), (8, 33)])
def test_rule_one_token_each_around_the_column_rule(dt, beta32, hv, n, dev):
    """255 to 264 (sequence, head) pairs: the last with 8 columns a wave and the first with 32, in both types of beta."""
    run_rule(dt, hv, hv, [1] * n, dev, seed=n, cu=False, norm=n % 2 == 0, beta32=beta32)


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("norm", [False, True])
def test_rule_runs_of_any_length(dt, norm, dev):
    run_rule(dt, 2, 4, [1, 5, 0, 2, 31, 17, 0, 8, 3], dev, norm=norm, beta32=norm, tail=11)


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("norm,decay", [(True, 0.05), (False, 0.05), (True, 0.001), (True, 3.0)])
def test_rule_long_runs(dt, norm, decay, dev):
    run_rule(dt, 1, 2, [63, 64, 65, 127, 128, 129, 1, 200, 333, 0, 32, 31, 33], dev, norm=norm, decay=decay, tail=5, seed=7)


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("hk,hv", [(2, 8), (5, 5), (1, 13)])
def test_rule_runs_of_many_heads(dt, hk, hv, dev):
    """More (sequence, head) pairs than get two taking waves a workgroup."""
    run_rule(dt, hk, hv, [1, 5, 0, 2, 31, 17, 0, 8, 3, 150, 4, 64, 33, 32], dev, beta32=hv == 8, tail=3, seed=hv)


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("hv,lens", [(6, [63, 64, 65, 127, 128, 129, 1, 200, 333, 0, 32, 31, 33]), (7, [1000, 2, 96, 4, 0, 160, 161, 3, 7, 5]),
                                     (32, [700, 1, 40, 500, 290])])
def test_rule_long_runs_of_many_heads(dt, hv, lens, dev):
    """So long on average that two pairs of waves prepare: odd and even numbers of chunks, and sequences of one."""
    run_rule(dt, 1, hv, lens, dev, beta32=hv == 7, seed=hv, tail=2)


@pytest.mark.parametrize("dt", [BF16, F16])
def test_rule_has_the_same_bits_in_any_batch(dt, dev):
    """One sequence alone, among few and among many."""
    r = Rule(dt, 2, 4, [77], dev, seed=3, extra=2)
    before = r.state.clone()
    o, whole = r.call(), r.state.clone()
    for n, size in ((3, 5), (40, 5), (20, 100)):
        many = Rule(dt, 2, 4, [size] * n + [77, 1, 0, 200], dev, seed=n)
        at = size * n
        for t in "qkvg":
            getattr(many, t)[at:at + 77] = getattr(r, t)
        many.beta[at:at + 77] = r.beta
        many.state[many.slots[n]] = before[r.slots[0]]
        assert torch.equal(many.call()[at:at + 77], o) and torch.equal(many.state[many.slots[n]], whole[r.slots[0]])


def _rule_by_abi(r, cu, l2_eps):
    o = torch.full(r.v.shape, 7.0, dtype=r.dt, device=r.dev)
    slots, cu = _i32(r.slots, r.dev), _ends(r.lens, r.dev) if cu else None
    arg = L.GdnTokens(*(x for t in (r.q, r.k, r.v) for x in (t.data_ptr(), *t.stride()[:2])), r.g.data_ptr(), r.beta.data_ptr(),
                      r.state.data_ptr(), o.data_ptr(), slots.data_ptr(), None if cu is None else cu.data_ptr(), r.v.shape[0],
                      len(r.lens), r.k.shape[1], r.v.shape[1], r.g.stride(0), r.beta.stride(0), r.state.shape[0],
                      r.state.stride(0), l2_eps, L.dt(o), L.dt(r.beta))
    L.check(L.lib().lsurge_gdn_recurrent(ctypes.byref(arg), torch.cuda.current_stream().cuda_stream), "gdn_recurrent")
    torch.cuda.synchronize()
    return o


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("lens,cu", [([1, 1, 1], False), ([3, 5, 31, 32, 33, 0, 71, 2], True), ([5, 31, 33] * 14, True),
                                     ([71, 95] * 17, True)])
def test_rule_norm_without_an_eps(dt, lens, cu, dev):
    """l2_eps 0 of the C entry at lengths that end inside a chunk, in every kernel: rows behind a sequence's end count for
    nothing, and heads of zeros and of values whose squares are below float32's smallest normal number are as good as any."""
    r = Rule(dt, 1, 2, lens, dev, norm=False, unit=False, seed=len(lens), tail=2 if cu else 0)
    at = _starts(lens)
    r.k[at[1]], r.q[at[1]] = 0, 0
    if cu:
        r.k[at[1] + 1], r.q[at[2] + 1] = 0, 0
        if dt is BF16:
            r.k[at[3] + 3] *= 2.0 ** -70
    before = r.state.clone()
    o = _rule_by_abi(r, cu, 0.0)
    unit = [_np(x) / np.maximum(np.linalg.norm(_np(x), axis=-1, keepdims=True), 1e-300) for x in (r.q, r.k)]
    v, g, beta = (_np(x) for x in (r.v, r.g, r.beta))
    u, tiny = so.HALF_STEP[NAME[dt]], so.TINY[NAME[dt]]
    for b, (a, n) in enumerate(zip(at, lens)):
        rows = slice(a, a + n)
        wo, wS, bo, bS = so.delta_rule(unit[0][rows], unit[1][rows], v[rows], g[rows], beta[rows], _np(before[r.slots[b]]), False)
        if n == 0:
            continue
        off = np.linalg.norm(_np(r.state[r.slots[b]]) - wS, axis=(1, 2))
        assert (off <= bS).all(), (b, n, off, bS)
        off = np.linalg.norm(_np(o[rows]) - wo, axis=-1)
        assert (off <= bo + u * (np.linalg.norm(wo, axis=-1) + bo) + 128 ** 0.5 * tiny).all(), (b, n)
    assert not o[at[-1]:].any()


def test_rule_keys_without_a_norm(dev):
    """Keys twice as long as unit ones with beta near 1: a step's factor is larger than one, and the state grows."""
    r = Rule(BF16, 1, 2, [40, 9], dev, norm=False, unit=True, decay=0.5)
    r.k.mul_(1.5)
    before = r.state.clone()
    o = r.call()
    r.check(o, before, r.state)


def test_rule_repeated_keys(dev):
    """One key for all tokens of a sequence, beta 1 and no decay: the state holds the last value alone."""
    r = Rule(BF16, 1, 1, [150, 70], dev, norm=True, beta32=True)
    r.k[:150], r.k[150:] = r.k[0].clone(), r.k[150].clone()
    r.beta.fill_(1.0), r.g.zero_()
    r.state.zero_()
    before = r.state.clone()
    o = r.call()
    r.check(o, before, r.state)


def test_rule_decay_of_nothing_and_of_everything(dev):
    r = Rule(BF16, 1, 2, [70, 3, 1], dev, norm=True)
    r.g.zero_()
    r.g[40], r.g[71], r.g[73] = -float("inf"), -200.0, -float("inf")
    before = r.state.clone()
    o = r.call()
    torch.cuda.synchronize()
    assert torch.isfinite(r.state).all()
    r.g[r.g < -100] = -745.0  # the oracle's exp of it is 0 in float32
    r.check(o, before, r.state)


@pytest.mark.parametrize("lens,cu", [([1] * 5, False), ([1] * 140, False), ([1, 2, 3, 4, 40], True)])
def test_rule_values_far_from_what_the_decay_leaves(lens, cu, dev):
    """Values of 10^27 after decays of e^-27 and more, and small ones beside a state that grows: both the values and what is left
    are float32 numbers, their quotients are not."""
    for size, g in ((1e27, -27.0), (1e27, -60.0), (1e-30, 26.0), (1e30, -0.5)):
        r = Rule(BF16, 1, 2, lens, dev, norm=True, seed=3)
        if g > 0:
            r.state.zero_()  # three steps of it at most
            r.lens = [min(n, 3) for n in lens]
            for t in (r.q, r.k, r.v, r.g, r.beta):
                t[sum(r.lens):] = float("nan")
        r.v.mul_(size), r.g.fill_(g)
        before = r.state.clone()
        o = r.call(cu)
        torch.cuda.synchronize()
        assert torch.isfinite(r.state).all()
        r.check(o, before, r.state)


def test_rule_places_without_a_slot(dev):
    """-1 and slots behind the pool give zeros, change nothing, and leave the other sequences' bits alone."""
    r = Rule(BF16, 2, 4, [1] * 9, dev)
    before = r.state.clone()
    want = r.call(cu=False)
    full = r.state.clone()
    r.state.copy_(before)
    slots = list(r.slots)
    slots[2], slots[5], slots[8] = -1, r.state.shape[0], 2 ** 31 - 1
    o = r.call(cu=False, slots=slots)
    torch.cuda.synchronize()
    live = [b for b in range(9) if b not in (2, 5, 8)]
    assert not o[[2, 5, 8]].any() and torch.equal(o[live], want[live])
    for b in range(9):
        assert torch.equal(r.state[r.slots[b]], (full if b in live else before)[r.slots[b]])
    r = Rule(F16, 1, 2, [3, 70, 2], dev)
    before = r.state.clone()
    o = r.call(slots=[-1, -5, r.slots[2]])
    assert not o[:73].any() and o[73:].any() and torch.equal(before[r.slots[1]], r.state[r.slots[1]])


def test_rule_without_sequences_and_without_rows(dev):
    r = Rule(BF16, 1, 2, [5], dev)
    before = r.state.clone()
    o = G.recurrent_gated_delta_rule(r.q, r.k, r.v, r.g, r.beta, r.state, cu_seqlens=_i32([0], dev))
    assert not o.any() and torch.equal(before, r.state)
    o = G.recurrent_gated_delta_rule(r.q[:0], r.k[:0], r.v[:0], r.g[:0], r.beta[:0], r.state)
    assert o.shape == (0, 2, 128) and torch.equal(before, r.state)
    o = G.recurrent_gated_delta_rule(r.q, r.k, r.v, r.g, r.beta, r.state[:0], state_slots=_i32([0] * 5, dev))
    assert not o.any()


@pytest.mark.parametrize("cu", [[0, 7, 3, 12], [-5, 4, 10 ** 9, 2], [3, 6, 9, 12], [12, 0, 12, 12]])
def test_rule_ends_out_of_range_stay_inside(cu, dev):
    """Ends that ascend from 0 only in part: nothing outside of the rows is read, nor a slot of no sequence changed."""
    r = Rule(BF16, 1, 2, [4, 4, 4], dev)
    before = r.state.clone()
    o = G.recurrent_gated_delta_rule(r.q, r.k, r.v, r.g, r.beta, r.state, state_slots=_i32(r.slots, dev), cu_seqlens=_i32(cu, dev))
    torch.cuda.synchronize()
    kept = [s for s in range(before.shape[0]) if s not in r.slots]
    assert torch.equal(before[kept], r.state[kept]) and o.shape == r.v.shape


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("lens", [[2, 1, 3], [5, 40, 1], [33] * 40, [70, 100] * 17])
def test_rows_before_the_first_sequence_give_zeros(dt, lens, dev):
    """Ends that start behind 0: the rows before are rows of no sequence, in all operators of packed rows, and the others have
    the bits of a call without them."""
    skip = 3
    r, c = Rule(dt, 1, 2, lens, dev, tail=2), Conv(dt, 4, 64, lens, dev, tail=2)
    before, kept = r.state.clone(), c.state.clone()
    want, after = (r.call(), c.call()), (r.state.clone(), c.state.clone())
    f = A.rotary_inv_freq(64, 1e4, dev)
    turned = A.rotary(r.q, r.k, f, cu_seqlens=_ends(lens, dev))
    nan = lambda t: torch.cat([torch.full_like(t[:skip], float("nan")), t])  # noqa: E731
    r.q, r.k, r.v, r.g, r.beta, c.x = (nan(t) for t in (r.q, r.k, r.v, r.g, r.beta, c.x))
    r.state.copy_(before), c.state.copy_(kept)
    cu = _ends(lens, dev) + skip
    for shape, call in ((r.v.shape, lambda: G.recurrent_gated_delta_rule(r.q, r.k, r.v, r.g, r.beta, r.state, _i32(r.slots, dev),
                                                                         cu, use_qk_norm_in_gdn=True)),
                        (c.x.shape, lambda: FC.causal_conv1d_update(c.x, c.w, c.state, _i32(c.slots, dev), cu, "silu"))):
        torch.full(shape, 7.0, dtype=dt, device=dev)  # freed: where an output of its size goes
        got, w = call(), want[len(shape) == 2]
        assert not got[:skip].any() and torch.equal(got[skip:], w)
    assert torch.equal(r.state, after[0]) and torch.equal(c.state, after[1])
    for got, w in zip(A.rotary(r.q, r.k, f, cu_seqlens=cu), turned):
        assert not got[:skip].any() and torch.equal(got[skip:], w)


def test_rule_split_into_calls(dev):
    """A sequence taken in calls of any size ends in the state of one call; alone or among others it has the same bits."""
    r = Rule(BF16, 2, 4, [77], dev, seed=3, extra=2)
    before = r.state.clone()
    o = r.call()
    r.check(o, before, r.state)
    whole = r.state.clone()
    r.state.copy_(before)
    got, a = [], 0
    for n in (1, 1, 5, 40, 1, 29):
        s = slice(a, a + n)
        got.append(G.recurrent_gated_delta_rule(r.q[s], r.k[s], r.v[s], r.g[s], r.beta[s], r.state, _i32(r.slots, dev),
                                                _i32([0, n], dev), use_qk_norm_in_gdn=True))
        a += n
    r.check(torch.cat(got), before, r.state)
    many = Rule(BF16, 2, 4, [3, 77, 1, 200], dev, seed=9)
    many.q[3:80], many.k[3:80], many.v[3:80], many.g[3:80], many.beta[3:80] = r.q, r.k, r.v, r.g, r.beta
    many.state[many.slots[1]] = before[r.slots[0]]
    mo = many.call()
    assert torch.equal(mo[3:80], o) and torch.equal(many.state[many.slots[1]], whole[r.slots[0]])


def test_rule_follows_the_chunked_form(dev):
    """A prompt by the chunked form, the next tokens by the recurrent one from its state, against the whole by the recurrent
    form; the chunked form rounds to bf16 on the way (2e-2 of its own tests)."""
    gen = torch.Generator().manual_seed(1)
    T, P = 150, 130
    q, k, v = (_randn(gen, (1, T, 2, 128), BF16, dev) for _ in range(3))
    g, beta = (-0.05 * torch.rand((1, T, 2), generator=gen)).to(dev), torch.rand((1, T, 2), generator=gen).to(BF16).to(dev)
    h0 = torch.zeros((1, 2, 128, 128), device=dev)
    o, h = G.fast_chunk_gated_delta_rule(q[:, :P], k[:, :P], v[:, :P], g[:, :P], beta[:, :P], initial_state=h0,
                                         use_qk_norm_in_gdn=True)
    state = h.float()
    rest = G.recurrent_gated_delta_rule(q[0, P:], k[0, P:], v[0, P:], g[0, P:], beta[0, P:], state, cu_seqlens=_i32([0, T - P], dev),
                                        use_qk_norm_in_gdn=True)
    one = G.alloc_delta_state(1, 2, dev)
    want = G.recurrent_gated_delta_rule(q[0], k[0], v[0], g[0], beta[0], one, cu_seqlens=_i32([0, T], dev), use_qk_norm_in_gdn=True)
    for x, y in ((o[0], want[:P]), (rest, want[P:]), (state, one)):
        assert (x.float() - y.float()).norm() < 2e-2 * y.float().norm()


def test_rule_strides(dev):
    """Rows of other strides than the tested ones, a pool inside a larger one, g and beta as columns of a projection."""
    r = Rule(BF16, 2, 4, [1, 40, 66], dev, beta32=True)
    before = r.state.clone()
    want = r.call()
    after = r.state.clone()
    pool = torch.full((3, *before.shape), 7.0, device=dev).transpose(0, 1).contiguous()
    pool[:, 1] = before
    gb = torch.cat([r.g, r.beta, r.g], 1)
    r.g, r.beta, r.state = gb[:, :4], gb[:, 4:8], pool[:, 1]
    r.q, r.k = r.q.transpose(0, 1).contiguous().transpose(0, 1), r.k.transpose(1, 2).contiguous().transpose(1, 2)
    o = r.call()
    assert torch.equal(o, want) and torch.equal(pool[:, 1], after)
    assert (pool[:, 0] == 7).all() and (pool[:, 2] == 7).all()


def test_rule_values_that_are_not_finite_stay_in_their_sequence(dev):
    for lens in ([1, 1, 1, 1], [3, 70, 100, 2]):
        r = Rule(BF16, 1, 2, lens, dev)
        before = r.state.clone()
        want, at = r.call(), _starts(lens)
        after = r.state.clone()
        r.state.copy_(before)
        r.v[at[1]:at[2]], r.g[at[1]], r.k[at[1]] = float("nan"), float("inf"), float("inf")
        o = r.call()
        for b in (0, 2, 3):
            assert torch.equal(o[at[b]:at[b + 1]], want[at[b]:at[b + 1]]) and torch.equal(r.state[r.slots[b]], after[r.slots[b]])


def test_rule_states_of_any_size(dev):
    """Columns of sizes from 2^-50 to 2^60 side by side; the rule takes columns apart, so each group of one size is held to its
    own bounds.  f16's range is short: a column's state is scaled there.  Without values and queries, the states alone.

    The decays take some columns below what any type holds.  float32 loses up to 2^-126 a value there.  f16 scales by 2^60 at
    most, and two terms leave up to 2^-25 of a scaled value over, so 2^-85: k, a unit vector of 128 values, sums that to
    sqrt(128) 2^-85 a column, 4 sqrt(128) 2^-85 in the 2-norm over 16 columns, which d and, times k, the state take over, and
    the update's own terms as much again, at each of the n tokens, with factors of at most 1 afterwards."""
    scale = torch.tensor([2.0 ** e for e in (-50, -30, -14, 0, 10, 30, 50, 60)], device=dev).repeat_interleave(16)
    for dt, decay in ((F16, 0.05), (F16, 2.0), (BF16, 0.05)):
        r = Rule(dt, 1, 2, [70, 5, 2], dev, decay=decay)
        r.q.zero_(), r.v.zero_(), r.state.mul_(scale)
        before = r.state.clone()
        assert not r.call().any()
        at = _starts(r.lens)
        for b, n in enumerate(r.lens):
            rows = slice(at[b], at[b] + n)
            for c in range(0, 128, 16):
                _, want, _, bound = so.delta_rule(*(_np(t[rows]) for t in (r.q, r.k)), np.zeros((n, 2, 16)), _np(r.g[rows]),
                                                  _np(r.beta[rows]), _np(before[r.slots[b]][..., c:c + 16]), True)
                off = np.linalg.norm(_np(r.state[r.slots[b]][..., c:c + 16]) - want, axis=(1, 2))
                least = 2 * n * 4 * 128 ** 0.5 * 2.0 ** (-85 if dt is F16 else -126)
                assert (off <= bound + least).all(), (dt, decay, n, c, off, bound)


@pytest.mark.parametrize("dt", [BF16, F16])
def test_rule_reads_what_was_erased(dt, dev):
    """Queries equal to their keys, beta 1, no decay and no values: each token erases what it reads, and o is 0 but for what the
    chunks' parts of o are held to.  These are q_i.S0 and (q_i.k_j) d_j, |d_j| <= |S0|, each with 2^-18 of either factor left
    out and 2^-18 of both together, 2^-16 at most; the state's own bound besides."""
    r = Rule(dt, 1, 2, [32], dev, norm=True, beta32=True)
    r.q.copy_(r.k), r.v.zero_(), r.g.zero_(), r.beta.fill_(1)
    before = r.state.clone()
    o = _np(r.call())
    k = _np(r.k)[:, 0]
    k /= np.sqrt((k * k).sum(-1, keepdims=True) + 1e-6)
    wo, wS, bo, bS = so.delta_rule(*(_np(t) for t in (r.q, r.k, r.v, r.g, r.beta)), _np(before[r.slots[0]]), True)
    size = np.linalg.norm(_np(before[r.slots[0]]), axis=(1, 2))
    parts = (1 + np.tril(np.abs(k @ k.T)).sum(1))[:, None] * size / 128 ** 0.5
    assert (np.linalg.norm(o - wo, axis=-1) <= bo + 2.0 ** -16 * parts * (1 + so.HALF_STEP[NAME[dt]])).all()
    assert (np.linalg.norm(_np(r.state[r.slots[0]]) - wS, axis=(1, 2)) <= bS).all()


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("n,length", [(1, 32), (2, 150), (40, 32), (33, 64)])
def test_rule_reads_what_was_erased_by_every_kernel(dt, n, length, dev):
    """Queries equal to their keys, beta 1 and no decay in workgroups of two and of four taking waves, with one and two pairs
    that prepare; o within the bound of any other input, without values and beside states a thousand times as large."""
    for size in (0.0, 1.0):
        r = Rule(dt, 1, 2, [length] * n, dev, norm=True, beta32=True, seed=n)
        r.q.copy_(r.k), r.g.zero_(), r.beta.fill_(1), r.v.mul_(size), r.state.mul_(1000)
        before = r.state.clone()
        r.check(r.call(), before, r.state)


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("lag", [0, 1, 5, 17])
@pytest.mark.parametrize("lens", [[4, 5, 31, 1, 3, 128, 2], [32] * 40, [64] * 33 + [127], [20, 1, 8, 4] * 20])
def test_rule_o_is_float32_beside_large_states(dt, lens, lag, dev):
    """Every token has an axis of its own as its key, beta 1, and reads that axis or the one of `lag` tokens before: o is that
    token's value / sqrt(128), whatever the state held there, 2^13 times as large here.  With one value that is not 0 to a
    product, what remains are single roundings of EPS times p, the state's decayed value: of the right side, of the sums of
    three terms (the state against k 2 and q 2, two solutions 6, the weight times what was solved for 6 and the terms left out 1)
    and of the factors of o (2): 20.  A value read from a state was rounded on the way in instead, 12 times.  Without decays
    where another token is read, since the exponentials of two tokens are rounded apart."""
    r = Rule(dt, 1, 2, lens, dev, norm=False, beta32=True, seed=len(lens), decay=0.01)
    gen = torch.Generator().manual_seed(lag)
    at = _starts(lens)
    axis = torch.cat([torch.randperm(128, generator=gen)[:n] for n in lens])
    read = torch.cat([torch.arange(a, a + n).sub(lag).clamp(min=a) if lag else torch.arange(a, a + n) for a, n in zip(at, lens)])
    if lag:  # the first ones read themselves
        first = torch.cat([torch.arange(n) < lag for n in lens])
        read[first] = torch.arange(len(read))[first]
        r.g.zero_()
    eye = torch.eye(128, dtype=dt)
    r.k.copy_(eye[axis][:, None]), r.q.copy_(eye[axis[read]][:, None]), r.beta.fill_(1), r.state.mul_(10 * 2.0 ** 13)
    held = _np(r.state[r.slots])
    o, v = _np(r.call()), _np(r.v)
    u, tiny = so.HALF_STEP[NAME[dt]], so.TINY[NAME[dt]]
    for b, (a, n) in enumerate(zip(at, lens)):
        rows = read[a:a + n].numpy()
        want = v[rows] / 128 ** 0.5
        p = np.abs(held[b][:, axis[rows].numpy()]).transpose(1, 0, 2) / 128 ** 0.5  # decays are at most 1
        off = 20 * so.EPS * p
        err = np.abs(o[a:a + n] - want) - (off + u * (np.abs(want) + off) + tiny)
        assert (err <= 0).all(), f"sequence {b} ({n} rows): {err.max():.2e} over"


def test_rule_columns_of_any_size(dev):
    """Values from f16's smallest to its largest in one head: each group of columns of one size within its own bounds."""
    scale = torch.tensor([2.0 ** e for e in (-22, -14, -8, -2, 0, 4, 8, 12)], device=dev).repeat_interleave(16)
    r = Rule(F16, 1, 2, [100, 6], dev)
    r.v.copy_((r.v.float() * scale).half()), r.state.mul_(scale)
    before = r.state.clone()
    o, at = r.call(), _starts(r.lens)
    for b, n in enumerate(r.lens):
        rows = slice(at[b], at[b] + n)
        for c in range(0, 128, 16):
            wo, want, bo, bound = so.delta_rule(*(_np(t[rows]) for t in (r.q, r.k)), _np(r.v[rows][..., c:c + 16]), _np(r.g[rows]),
                                                _np(r.beta[rows]), _np(before[r.slots[b]][..., c:c + 16]), True)
            off = np.linalg.norm(_np(r.state[r.slots[b]][..., c:c + 16]) - want, axis=(1, 2))
            assert (off <= bound).all(), (n, c, off, bound)
            off = np.linalg.norm(_np(o[rows][..., c:c + 16]) - wo, axis=-1)
            assert (off <= bo + so.HALF_STEP["f16"] * (np.linalg.norm(wo, axis=-1) + bo) + 4 * so.TINY["f16"]).all(), (n, c)


def test_rule_far_slots(dev):
    """A pool of more than 2^31 elements."""
    hv = 8
    state = torch.zeros((16500, hv, 128, 128), device=dev)
    r = Rule(BF16, 4, hv, [1, 1, 3], dev)
    small = r.state[r.slots].clone()
    r.state, r.slots = state, [16499, 16384, 7]
    state[r.slots] = small
    o = r.call()
    torch.cuda.synchronize()
    wide = dict(zip(r.slots, range(3)))
    got, r.slots = state[r.slots].clone(), [wide[s] for s in r.slots]
    r.check(o, small, got)
    state[[16499, 16384, 7]] = 0
    assert not state.any()


# ----------------------------------------------------------------------------------------------- convolution


class Conv:

    def __init__(self, dt, K, C, lens, dev, seed=0, silu=True, tail=0, extra=3):
        gen = torch.Generator().manual_seed(seed)
        self.x = _randn(gen, (sum(lens) + tail, C), dt, dev)
        self.w = _randn(gen, (K, 1, C), dt, dev, 0.5)
        self.state = _randn(gen, (len(lens) + extra, K - 1, C), dt, dev)
        self.slots = [int(s) for s in torch.randperm(len(lens) + extra, generator=gen)[:len(lens)]]
        self.lens, self.silu, self.dt, self.dev, self.tail = lens, silu, dt, dev, tail
        if tail:
            self.x[-tail:] = float("nan")

    def call(self, cu=True, slots=None):
        return FC.causal_conv1d_update(self.x, self.w, self.state, state_slots=_i32(self.slots if slots is None else slots, self.dev),
                                       cu_seqlens=_ends(self.lens, self.dev) if cu else None,
                                       activation="silu" if self.silu else None)

    def check(self, y, before, after):
        u, tiny = so.HALF_STEP[NAME[self.dt]], so.TINY[NAME[self.dt]]
        got, x, w = _np(y), _np(self.x), _np(self.w)[:, 0]
        at = _starts(self.lens)
        for b, (a, n) in enumerate(zip(at, self.lens)):
            wy, ws, bound = so.conv(x[a:a + n], w, _np(before[self.slots[b]]), self.silu, u, tiny)
            assert (np.abs(got[a:a + n] - wy) <= bound).all(), (b, n)
            assert np.array_equal(_np(after[self.slots[b]]), ws), (b, n)
        assert not got[at[-1]:].any()
        kept = [s for s in range(before.shape[0]) if s not in self.slots]
        assert torch.equal(before[kept], after[kept])


def run_conv(*args, cu=True, **kw):
    c = Conv(*args, **kw)
    before = c.state.clone()
    c.check(c.call(cu), before, c.state)


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("K", [2, 3, 4, 5, 6, 7, 8])
def test_conv_runs_of_any_length(dt, K, dev):
    run_conv(dt, K, 40, [1, 0, 5, 2, 3, 0, 8, 17, 1, 1, 64], dev, silu=K % 2 == 0, tail=9, seed=K)


@pytest.mark.parametrize("n,C", [(1, 8), (1, 2048), (64, 2048), (300, 264)])
def test_conv_one_row_each(n, C, dev):
    run_conv(BF16, 4, C, [1] * n, dev, cu=False)
    run_conv(F16, 4, C, [1] * n, dev, cu=False, silu=False)


@pytest.mark.parametrize("K", [2, 4, 8])
def test_conv_tiles_of_every_size(K, dev):
    """So many rows that a thread walks 4 to 16 of them: sequences that begin at and around the tiles' ends, and many of fewer
    rows than taps."""
    rng = np.random.default_rng(K)
    for C, lens in ((8192, [31, 1, 33, 32, 2, 64, 7, 130, 600, 30, 1, 1, 2, 95]),
                    (4096, [int(n) for n in rng.integers(0, 12, 700)]), (2048, [4000, 63, 1, 65, 31, 3, 2500])):
        run_conv(BF16, K, C, lens, dev, tail=70)


def test_conv_thousands_of_sequences(dev):
    """More than 64 and more than 64^2 ends to find a row's sequence among, many of them without rows."""
    rng = np.random.default_rng(1)
    for n, most in ((65, 4), (4097, 3), (9000, 2)):
        run_conv(BF16, 4, 8, [int(i) for i in rng.integers(0, most, n)], dev, tail=3)
    run_conv(BF16, 4, 16, [0] * 5000 + [7] + [0] * 5000, dev)


def test_conv_far_rows(dev):
    """Inputs and outputs of more than 2^31 values: the last rows against a call of their own after the rows before them."""
    rows, C = 270000, 8192
    x = torch.zeros((rows, C), dtype=BF16, device=dev)
    gen = torch.Generator().manual_seed(21)
    x[-40:] = _randn(gen, (40, C), BF16, dev)
    w = _randn(gen, (4, C), BF16, dev)
    state = FC.alloc_conv_state(2, 4, C, BF16, dev)
    y = FC.causal_conv1d_update(x, w, state, cu_seqlens=_i32([0, 100000, rows], dev), activation="silu")
    own = FC.alloc_conv_state(1, 4, C, BF16, dev)
    want = FC.causal_conv1d_update(x[-40:], w, own, cu_seqlens=_i32([0, 40], dev), activation="silu")
    assert torch.equal(y[-40:], want) and torch.equal(state[1], own[0])
    assert not y[:-40].any() and not state[0].any()


def test_conv_places_without_a_slot(dev):
    c = Conv(BF16, 4, 64, [1, 6, 2, 70, 0, 4], dev)
    before = c.state.clone()
    want = c.call()
    after = c.state.clone()
    c.state.copy_(before)
    slots = list(c.slots)
    slots[1], slots[3] = -1, c.state.shape[0]
    y = c.call(slots=slots)
    at = _starts(c.lens)
    for b in range(6):
        r = slice(at[b], at[b + 1])
        assert torch.equal(y[r], torch.zeros_like(y[r]) if b in (1, 3) else want[r])
        assert torch.equal(c.state[c.slots[b]], (before if b in (1, 3) else after)[c.slots[b]])


def test_conv_split_into_calls_is_the_training_form(dev):
    """Rows one by one, in parts and at once have the bits of causal_conv1d over the whole sequence."""
    c = Conv(BF16, 4, 128, [50], dev, silu=False, extra=0)
    c.state.zero_()
    want = FC.causal_conv1d(c.x[None], c.w)[0]
    assert torch.equal(c.call(), want)
    end = c.state.clone()
    for parts in ([1] * 50, [2, 1, 40, 3, 4]):
        state, got, a = FC.alloc_conv_state(1, 4, 128, BF16, dev), [], 0
        for n in parts:
            got.append(FC.causal_conv1d_update(c.x[a:a + n], c.w[:, 0], state, cu_seqlens=_i32([0, n], dev)))
            a += n
        assert torch.equal(torch.cat(got), want) and torch.equal(state, end)


def test_conv_strides_ends_and_nothing(dev):
    c = Conv(BF16, 4, 64, [3, 9], dev)
    before = c.state.clone()
    want = c.call()
    wide = torch.full((12, 200), float("nan"), dtype=BF16, device=dev)
    wide[:, 64:128] = c.x
    for x in (wide[:, 64:128], c.x.t().contiguous().t()):
        c.x = x
        c.state.copy_(before)
        assert torch.equal(c.call(), want)
    c.x = wide[:, 64:128]
    for cu in ([0, 7, 3], [-5, 4, 10 ** 9], [3, 6, 12]):
        c.state.copy_(before)
        FC.causal_conv1d_update(c.x, c.w, c.state, _i32(c.slots, dev), _i32(cu, dev))
        kept = [s for s in range(5) if s not in c.slots]
        assert torch.equal(before[kept], c.state[kept])
    y = FC.causal_conv1d_update(c.x, c.w, c.state, cu_seqlens=_i32([0], dev))
    assert not y.any()
    assert FC.causal_conv1d_update(c.x[:0], c.w, c.state).shape == (0, 64)


def test_conv_silu_of_large_values(dev):
    x = torch.tensor([[0.0, 1e-3, -1e-3, 30.0, -30.0, 100.0, -100.0, 1e30]], device=dev).to(BF16)
    w = torch.zeros((2, 8), dtype=BF16, device=dev)
    w[1] = 1
    y = FC.causal_conv1d_update(x, w, FC.alloc_conv_state(1, 2, 8, BF16, dev), activation="silu")
    want, _, bound = so.conv(_np(x), _np(w), np.zeros((1, 8)), True, so.HALF_STEP["bf16"], so.TINY["bf16"])
    assert (np.abs(_np(y) - want) <= bound).all()


# ----------------------------------------------------------------------------------------------- rotation


def _within(got, want, bound, what=""):
    err = np.abs(_np(got) - want)
    assert (err <= bound).all(), f"{what}: {np.nanmax(err - bound):.2e} over the bound"


def _pos(lens):
    return np.concatenate([np.arange(n) for n in lens] + [[]]).astype(int)


def check_rotary(q, k, f, pos, inter, live, back=True, **kw):
    """rotary and its gradients; rows from `live` on give zeros."""
    u, tiny = so.HALF_STEP[NAME[q.dtype]], so.TINY[NAME[q.dtype]]
    lq, lk = q.detach().requires_grad_(back), k.detach().requires_grad_(back)
    out = A.rotary(lq, lk, f, interleaved=inter, **kw)
    ups = [torch.randn(t.shape, generator=torch.Generator().manual_seed(2)).to(t.dtype).to(t.device) for t in out]
    grads = torch.autograd.grad(out, (lq, lk), ups) if back else ()
    for got, x, sign in [(out[0], q, 1), (out[1], k, 1)] + ([(grads[0], ups[0], -1), (grads[1], ups[1], -1)] if back else []):
        assert got.shape == x.shape and got.dtype == x.dtype
        x, got = x.flatten(0, -3), got.flatten(0, -3)
        _within(got[:live], *so.rotate(_np(x[:live]), pos, _np(f), inter, u, tiny, sign))
        assert not got[live:].any()


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("D,rot", [(64, 64), (64, 16), (64, 48), (128, 128), (128, 32), (256, 256), (256, 64), (256, 240)])
@pytest.mark.parametrize("inter", [False, True])
def test_rotary_packed(dt, D, rot, inter, dev):
    gen = torch.Generator().manual_seed(rot)
    lens = [1, 0, 33, 7, 2, 90]
    rows = _randn(gen, (sum(lens) + 6, 5 + 2, D), dt, dev)
    rows[-6:] = float("nan")
    check_rotary(rows[:, :5], rows[:, 5:7], A.rotary_inv_freq(rot, 1e4, dev), _pos(lens), inter, sum(lens),
                 cu_seqlens=_ends(lens, dev))


@pytest.mark.parametrize("hq,hk", [(1, 1), (16, 2), (7, 7), (12, 3), (40, 1)])
def test_rotary_heads_dense(hq, hk, dev):
    gen = torch.Generator().manual_seed(hq)
    q, k = _randn(gen, (3, 50, hq, 64), BF16, dev), _randn(gen, (3, 50, hk, 64), BF16, dev)
    f = A.rotary_inv_freq(64, 1e4, dev)
    check_rotary(q, k, f, _pos([50] * 3), False, 150)
    check_rotary(q.transpose(1, 2).contiguous().transpose(1, 2), k[:, :, :1].expand(-1, -1, hk, -1), f, _pos([50] * 3), True, 150)


@pytest.mark.parametrize("rows,heads", [(4000, 8), (16000, 8), (30000, 12)])
def test_rotary_heads_a_thread(rows, heads, dev):
    """So many rows that a thread turns 2 and 4 heads, in numbers that they do and do not divide."""
    gen = torch.Generator().manual_seed(rows)
    q, k = _randn(gen, (rows, heads - 3, 128), BF16, dev), _randn(gen, (rows, 2, 128), BF16, dev)
    check_rotary(q, k, A.rotary_inv_freq(128, 1e6, dev), _pos([rows]), False, rows, cu_seqlens=_ends([rows], dev))


def test_rotary_thousands_of_sequences(dev):
    rng = np.random.default_rng(2)
    gen = torch.Generator().manual_seed(2)
    f = A.rotary_inv_freq(16, 1e4, dev)
    for n, most in ((65, 40), (4097, 3), (9000, 2)):
        lens = [int(i) for i in rng.integers(0, most, n)]
        rows = _randn(gen, (sum(lens) + 4, 2, 64), F16, dev)
        check_rotary(rows[:, :1], rows[:, 1:], f, _pos(lens), False, sum(lens), cu_seqlens=_ends(lens, dev))


def test_rotary_far_positions(dev):
    """Positions up to 2^31 - 1 and negative ones, given by themselves."""
    pos = [0, 1, -1, 100003, 10 ** 6, 2 ** 24 + 1, 2 ** 31 - 1, -2 ** 31]
    gen = torch.Generator().manual_seed(3)
    q, k = _randn(gen, (8, 3, 128), F16, dev), _randn(gen, (8, 1, 128), F16, dev)
    for theta in (1e4, 1e6):
        check_rotary(q, k, A.rotary_inv_freq(128, theta, dev), pos, False, 8, positions=_i32(pos, dev))
    check_rotary(q.view(2, 4, 3, 128), k.view(2, 4, 1, 128), A.rotary_inv_freq(128, 1e4, dev), pos, True, 8,
                 positions=_i32(pos, dev).view(2, 4))


def test_rotary_gradient_against_differences(dev):
    """The gradient against central differences of the forward on float-valued inputs: steps of 1 in f16 values are exact, the
    map is linear, so a difference is the column of the Jacobian within two output roundings."""
    gen = torch.Generator().manual_seed(4)
    q, k = _randn(gen, (3, 1, 64), F16, dev), _randn(gen, (3, 1, 64), F16, dev)
    f, cu = A.rotary_inv_freq(32, 1e4, dev), _i32([0, 3], dev)
    up = _randn(gen, (3, 1, 64), F16, dev)
    lq = q.clone().requires_grad_()
    got = torch.autograd.grad(A.rotary(lq, k, f, cu_seqlens=cu)[0], lq, up)[0]
    zero = torch.zeros_like(q)
    for t, d in ((0, 3), (1, 0), (2, 17), (2, 31), (1, 40)):
        e = zero.clone()
        e[t, 0, d] = 1
        diff = (A.rotary(e, k, f, cu_seqlens=cu)[0].double() - A.rotary(-e, k, f, cu_seqlens=cu)[0].double()) / 2
        col = (diff * up.double()).sum()
        # two values of the column, each off by half a step of 1 at most, and the gradient's own rounding
        assert abs(col - got[t, 0, d].double()) <= 2 ** -11 * (up[t].double().abs().sum() * 2 ** -1 + got[t, 0, d].double().abs()) + 2 ** -20


def test_rotary_one_gradient_and_empty(dev):
    gen = torch.Generator().manual_seed(5)
    q, k = _randn(gen, (9, 2, 64), BF16, dev), _randn(gen, (9, 1, 64), BF16, dev)
    f, cu = A.rotary_inv_freq(64, 1e4, dev), _i32([0, 9], dev)
    lq, lk = q.clone().requires_grad_(), k.clone().requires_grad_()
    both = torch.autograd.grad(A.rotary(lq, lk, f, cu_seqlens=cu), (lq, lk), (q, k))
    out = A.rotary(lq, lk, f, cu_seqlens=cu)
    assert torch.equal(torch.autograd.grad(out[0], lq, q)[0], both[0])
    out = A.rotary(lq, lk, f, cu_seqlens=cu)
    dq, dk = torch.autograd.grad(out[1], (lq, lk), k, allow_unused=True)
    assert torch.equal(dk, both[1]) and (dq is None or not dq.any())
    assert torch.equal(torch.autograd.grad(A.rotary(lq, k, f, cu_seqlens=cu)[0], lq, q)[0], both[0])
    o, p = A.rotary(q[:0], k[:0], f, cu_seqlens=_i32([0], dev))
    assert o.shape == (0, 2, 64) and p.shape == (0, 1, 64)
    o, p = A.rotary(q, k, f, cu_seqlens=_i32([0], dev))  # no sequence: every row is behind the last
    assert not o.any() and not p.any()


def test_rotary_results_without_a_gradient(dev):
    """What comes of a tensor that needs no gradient needs none: a turned k goes into a cache beside a q that trains."""
    gen = torch.Generator().manual_seed(8)
    q, k = _randn(gen, (9, 2, 64), BF16, dev).requires_grad_(), _randn(gen, (9, 1, 64), BF16, dev)
    f, cu = A.rotary_inv_freq(64, 1e4, dev), _i32([0, 9], dev)
    oq, ok = A.rotary(q, k, f, cu_seqlens=cu)
    assert oq.requires_grad and not ok.requires_grad
    c = Cache(BF16, 1, 64, 16, [9], dev)
    A.append_kv(c.k, c.v, c.table, c.lens, ok, k, cu_seqlens=cu)
    grad, = torch.autograd.grad(oq, q, q)
    ok, oq = A.rotary(k, q[:, :1], f, cu_seqlens=cu)
    assert oq.requires_grad and not ok.requires_grad
    assert torch.equal(torch.autograd.grad(oq, q, q[:, :1])[0][:, :1], grad[:, :1])
    with torch.no_grad():
        assert not any(t.requires_grad for t in A.rotary(q, k, f, cu_seqlens=cu))


def test_rotary_refuses_what_its_gradient_cannot_give(dev):
    gen = torch.Generator().manual_seed(9)
    q, k = _randn(gen, (9, 2, 64), BF16, dev).requires_grad_(), _randn(gen, (9, 1, 64), BF16, dev)
    f, cu, pos = A.rotary_inv_freq(64, 1e4, dev), _i32([0, 9], dev), _i32(range(9), dev)
    for kw in (dict(positions=pos), dict(cu_seqlens=cu), dict(cu_seqlens=cu, positions=pos)):
        for t in kw.values():
            out = A.rotary(q, k, f, **kw)[0].sum()
            t.add_(0)
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                out.backward()
    dq, = torch.autograd.grad(A.rotary(q, k, f, cu_seqlens=cu)[0].square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dq.sum().backward()
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(q.detach(), torch.ones_like(q))
        with pytest.raises((RuntimeError, NotImplementedError)):
            A.rotary(dual, k, f, cu_seqlens=cu)
        with pytest.raises((RuntimeError, NotImplementedError)):
            A.rotary(k, k, forward_ad.make_dual(f, torch.ones_like(f)), cu_seqlens=cu)
        r, c = Rule(BF16, 1, 2, [1], dev), Conv(BF16, 4, 16, [1], dev)
        r.v = forward_ad.make_dual(r.v, torch.ones_like(r.v))
        c.x = forward_ad.make_dual(c.x, torch.ones_like(c.x))
        for call in (r.call, c.call):
            with pytest.raises(ValueError, match="of the forward mode neither"):
                call()


def test_rotary_then_attention_trains(dev):
    """Rotated queries and keys through causal_attention: gradients of q and k are those of the attention turned back."""
    gen = torch.Generator().manual_seed(6)
    lens = [40, 3, 70]
    q, k, v = (_randn(gen, (113, h, 64), BF16, dev) for h in (4, 2, 2))
    cu, f, do = _ends(lens, dev), A.rotary_inv_freq(64, 1e4, dev), _randn(gen, (113, 4, 64), BF16, dev)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    o = A.causal_attention(*A.rotary(*leaves[:2], f, cu_seqlens=cu), leaves[2], cu)
    got = torch.autograd.grad(o, leaves, do)
    rq, rk = (t.detach().requires_grad_() for t in A.rotary(q, k, f, cu_seqlens=cu))
    lv = v.clone().requires_grad_()
    o2 = A.causal_attention(rq, rk, lv, cu)
    mid = torch.autograd.grad(o2, (rq, rk, lv), do)
    back = A.rotary(mid[0], mid[1], f, positions=_i32(-_pos(lens), dev))
    assert torch.equal(o, o2) and torch.equal(got[2], mid[2])
    assert torch.equal(got[0], back[0]) and torch.equal(got[1], back[1])


# ----------------------------------------------------------------------------------------------- rotated appends


class Cache:

    def __init__(self, dt, hk, D, page, keys, dev, seed=0, hole=None):
        gen = torch.Generator().manual_seed(seed)
        need = [max(1, -(-n // page)) for n in keys]
        total = sum(need) + 2
        self.k, self.v = A.alloc_kv_cache(total, page, hk, D, dt, dev)
        self.k.copy_(_randn(gen, self.k.shape, dt, dev)), self.v.copy_(_randn(gen, self.v.shape, dt, dev))
        perm = torch.randperm(total, generator=gen).to(torch.int32)
        self.table = torch.full((len(keys), max(need) if need else 1), -1, dtype=torch.int32)
        for b, (m, a) in enumerate(zip(need, _starts(need))):
            self.table[b, :m] = perm[a:a + m]
        if hole is not None:
            self.table[hole] = total + 5
        self.table = self.table.to(dev)
        self.lens = _i32(keys, dev)


def check_append(dt, hq, hk, D, rot, page, new, keys, dev, inter=False, cu=True, tail=0, hole=None, positions=None, seed=0):
    """rotary_append_kv against rotary (bit for bit) and append_kv of its k (bit for bit), and against the oracle."""
    gen = torch.Generator().manual_seed(seed)
    n = sum(new) + tail
    rows = _randn(gen, (n, hq + 2 * hk, D), dt, dev)
    if tail:
        rows[-tail:] = float("nan")
    q, k, v = rows[:, :hq], rows[:, hq:hq + hk], rows[:, hq + hk:]
    f = A.rotary_inv_freq(rot, 1e6, dev)
    ends = _ends(new, dev) if cu else None
    c = Cache(dt, hk, D, page, keys, dev, seed, hole)
    kc, vc = c.k.clone(), c.v.clone()
    qo, ko = A.rotary_append_kv(q, k, v, c.k, c.v, c.table, c.lens, f, cu_seqlens=ends, interleaved=inter, return_k=True,
                                positions=None if positions is None else _i32(positions, dev))
    place = np.concatenate([np.arange(b - a, b) for a, b in zip(new, keys)] + [[]]).astype(int)
    pos = place if positions is None else np.asarray(positions)
    live = sum(new)
    u, tiny = so.HALF_STEP[NAME[dt]], so.TINY[NAME[dt]]
    for got, x in ((qo, q), (ko, k)):
        ok = place >= 0
        _within(got[:live][ok], *so.rotate(_np(x[:live])[ok], pos[:live][ok], _np(f), inter, u, tiny))
        assert not got[:live][~ok].any() and not got[live:].any()
    A.append_kv(kc, vc, c.table, c.lens, ko, v, cu_seqlens=ends)
    assert torch.equal(c.k, kc) and torch.equal(c.v, vc)
    other = Cache(dt, hk, D, page, keys, dev, seed, hole)
    alone = A.rotary_append_kv(q, k, v, other.k, other.v, c.table, c.lens, f, cu_seqlens=ends, interleaved=inter,
                               positions=None if positions is None else _i32(positions, dev))
    assert torch.equal(alone, qo) and torch.equal(other.k, kc) and torch.equal(other.v, vc)


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("D,rot,inter", [(64, 64, False), (128, 64, True), (256, 256, False)])
def test_append_one_token_each(dt, D, rot, inter, dev):
    check_append(dt, 4, 2, D, rot, 16, [1] * 6, [1, 16, 17, 100, 33, 5000], dev, inter=inter, cu=False)


def test_append_unused_places(dev):
    """Sequences of length 0 in a step: their q gives zeros, nothing is written."""
    check_append(BF16, 4, 1, 64, 64, 8, [1] * 5, [1, 0, 9, 0, 3], dev, cu=False)


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("hq,hk,page", [(8, 2, 8), (5, 1, 64), (7, 7, 16)])
def test_append_prompts(dt, hq, hk, page, dev):
    check_append(dt, hq, hk, 128, 128, page, [1, 0, 70, 9, 300], [1, 5, 70, 200, 1000], dev, tail=13)


def test_append_lengths_shorter_than_the_rows_and_pages_missing(dev):
    check_append(BF16, 2, 1, 64, 32, 8, [4, 9], [2, 30], dev)  # two rows of the first before its position 0
    check_append(BF16, 2, 1, 64, 32, 8, [4, 20], [4, 30], dev, hole=(1, 2))


def test_append_positions(dev):
    check_append(F16, 2, 1, 128, 128, 16, [3, 5], [3, 40], dev, positions=[5, 6, 7, 10 ** 6, -4, 0, 2 ** 31 - 1, 12])


def test_append_thousands_of_sequences(dev):
    rng = np.random.default_rng(3)
    new = [int(i) for i in rng.integers(0, 3, 4200)]
    check_append(BF16, 2, 1, 64, 64, 8, new, [n + int(i) for n, i in zip(new, rng.integers(0, 9, 4200))], dev, tail=2)


def test_append_far_pages(dev):
    """Caches of more than 2^31 values, pages at both ends."""
    pages, D = 140000, 256
    gen = torch.Generator().manual_seed(22)
    kc, vc = (torch.zeros((pages, 64, 1, D), dtype=BF16, device=dev) for _ in range(2))
    q, k, v = _randn(gen, (70, 2, D), BF16, dev), _randn(gen, (70, 1, D), BF16, dev), _randn(gen, (70, 1, D), BF16, dev)
    table, f = _i32([[pages - 1, 0]], dev), A.rotary_inv_freq(64, 1e4, dev)
    _, kt = A.rotary_append_kv(q, k, v, kc, vc, table, _i32([70], dev), f, cu_seqlens=_i32([0, 70], dev), return_k=True)
    _within(kt, *so.rotate(_np(k), np.arange(70), _np(f), False, so.HALF_STEP["bf16"], so.TINY["bf16"]))
    for c, t in ((kc, kt), (vc, v)):
        assert torch.equal(c[pages - 1], t[:64]) and torch.equal(c[0, :6], t[64:])
        assert not c[1:pages - 1].any() and not c[0, 6:].any()


def test_append_no_sequence(dev):
    gen = torch.Generator().manual_seed(0)
    q, k = _randn(gen, (4, 2, 64), BF16, dev), _randn(gen, (4, 1, 64), BF16, dev)
    c = Cache(BF16, 1, 64, 8, [3], dev)
    kc = c.k.clone()
    qo, ko = A.rotary_append_kv(q, k, k, c.k, c.v, c.table[:0], c.lens[:0], A.rotary_inv_freq(64, 1e4, dev),
                                cu_seqlens=_i32([0], dev), return_k=True)
    assert not qo.any() and not ko.any() and torch.equal(kc, c.k)
    qo = A.rotary_append_kv(q[:0], k[:0], k[:0], c.k, c.v, c.table, c.lens, A.rotary_inv_freq(64, 1e4, dev), cu_seqlens=_i32([0, 0], dev))
    assert qo.shape == (0, 2, 64) and torch.equal(kc, c.k)


# ----------------------------------------------------------------------------------------------- together


def _layer(gen, dev, hk=2, hv=4, hq=4, hkv=2, D=64):
    C = (2 * hk + hv) * 128
    return dict(conv=_randn(gen, (4, 1, C), BF16, dev, 0.5), hk=hk, hv=hv, C=C, freq=A.rotary_inv_freq(32, 1e4, dev), hq=hq,
                hkv=hkv, D=D)


def _mix(p, x, gb, qkv, conv_state, delta_state, slots, cu, cache, table, lens, prompt):
    """One linear and one softmax layer's mixing of new rows."""
    hk, hv = p["hk"], p["hv"]
    y = FC.causal_conv1d_update(x, p["conv"], conv_state, slots, cu, activation="silu")
    heads = y.view(-1, 2 * hk + hv, 128)
    o = G.recurrent_gated_delta_rule(heads[:, :hk], heads[:, hk:2 * hk], heads[:, 2 * hk:], gb[0], gb[1], delta_state, slots, cu,
                                     use_qk_norm_in_gdn=True)
    q, k, v = qkv.split((p["hq"], p["hkv"], p["hkv"]), 1)
    if prompt:
        q, k = A.rotary_append_kv(q, k, v, *cache, table, lens, p["freq"], cu_seqlens=cu, return_k=True)
        return o, A.causal_attention(q, k, v, cu)
    q = A.rotary_append_kv(q, k, v, *cache, table, lens, p["freq"])
    return o, A.paged_attention(q, *cache, table, lens)


def test_a_models_life(dev):
    """Prompts, then tokens one by one, against all tokens at once as prompts: conv, delta rule, rotation, cache and attention
    as a model calls them.  Both ways differ by float32 sums in another order and bf16 outputs rounded from them."""
    gen = torch.Generator().manual_seed(11)
    p = _layer(gen, dev)
    lens, more = [5, 70, 1, 33], 6
    n = len(lens)
    full = [a + more for a in lens]
    rows = sum(full)
    x, qkv = _randn(gen, (rows, p["C"]), BF16, dev), _randn(gen, (rows, p["hq"] + 2 * p["hkv"], p["D"]), BF16, dev)
    g = (-0.1 * torch.rand((rows, p["hv"]), generator=gen)).to(dev)
    beta = torch.rand((rows, p["hv"]), generator=gen).to(BF16).to(dev)
    slots = _i32([4, 0, 2, 5], dev)

    def fresh():
        c = Cache(BF16, p["hkv"], p["D"], 16, full, dev)
        return (FC.alloc_conv_state(6, 4, p["C"], BF16, dev), G.alloc_delta_state(6, p["hv"], dev)), (c.k, c.v), c.table

    states, cache, table = fresh()
    want = _mix(p, x, (g, beta), qkv, *states, slots, _ends(full, dev), cache, table, _i32(full, dev), True)
    at = _starts(full)
    states2, cache2, table2 = fresh()
    first = torch.cat([torch.arange(a, a + m) for a, m in zip(at, lens)]).to(dev)
    o = _mix(p, x[first], (g[first], beta[first]), qkv[first], *states2, slots, _ends(lens, dev), cache2, table2, _i32(lens, dev), True)
    got = [[t.clone()] for t in o]
    rows_of = [first]
    for i in range(more):
        r = torch.tensor([a + m + i for a, m in zip(at, lens)], device=dev)
        o = _mix(p, x[r], (g[r], beta[r]), qkv[r], *states2, slots, None, cache2, table2, _i32([m + i + 1 for m in lens], dev), False)
        for a, t in zip(got, o):
            a.append(t)
        rows_of.append(r)
    rows_of = torch.cat(rows_of)
    assert torch.equal(states[0], states2[0])  # the convolution's inputs are copies
    err = (states[1] - states2[1]).norm() / states[1].norm()
    assert err < 1e-5, err
    # both round o once to bf16 (2^-8 of a value at most), the attention its weights too
    for a, w, tol in zip(got, want, (2 ** -8, 2 ** -7)):
        a, w = torch.cat(a).float(), w[rows_of].float()
        assert (a - w).norm() <= 2 * tol * w.norm()
    assert torch.equal(table, table2)
    place = torch.zeros(cache[0].shape[:2], dtype=torch.bool, device=dev)
    for b, m in enumerate(full):
        t = torch.arange(m, device=dev)
        place[table[b, t // 16].long(), t % 16] = True
    for a, b in zip(cache, cache2):
        assert torch.equal(a[place], b[place])


@pytest.mark.parametrize("dt", [BF16, F16])
def test_drafts_taken_back(dt, dev):
    """Drafted tokens of several sequences, of which some are accepted: with the slots' copies written back and the accepted
    rows run again, outputs and states are those of a program that never saw the others."""
    drafts, accepted = [5, 4, 1, 7], [2, 4, 1, 5]
    r, c = Rule(dt, 1, 2, drafts, dev, seed=4), Conv(dt, 4, 64, drafts, dev, seed=4)
    states = r.state, c.state
    slots = [torch.tensor(x.slots, device=dev) for x in (r, c)]
    fresh = [t.clone() for t in states]
    keep = [t[s] for t, s in zip(states, slots)]
    r.call(), c.call()
    for t, s, k in zip(states, slots, keep):
        t[s] = k
    rows = torch.cat([torch.arange(a, a + n) for a, n in zip(_starts(drafts), accepted)]).to(dev)
    r.q, r.k, r.v, r.g, r.beta, c.x = (t[rows] for t in (r.q, r.k, r.v, r.g, r.beta, c.x))
    r.lens = c.lens = accepted
    o, y = r.call(), c.call()
    ends = [t.clone() for t in states]
    r.state, c.state = fresh
    assert torch.equal(r.call(), o) and torch.equal(c.call(), y)
    assert torch.equal(r.state, ends[0]) and torch.equal(c.state, ends[1])
    r.check(o, states[0].index_copy(0, slots[0], keep[0]), ends[0])


def test_captured_step_replays(dev):
    """A decode step in a graph, replayed with other inputs, lengths and slots between eager calls, bit for bit."""
    gen = torch.Generator().manual_seed(12)
    p = _layer(gen, dev)
    n, hv = 5, p["hv"]
    x, qkv = _randn(gen, (n, p["C"]), BF16, dev), _randn(gen, (n, p["hq"] + 2 * p["hkv"], p["D"]), BF16, dev)
    g, beta = torch.zeros((n, hv), device=dev), torch.ones((n, hv), dtype=BF16, device=dev)
    slots, lens = _i32([0, 1, 2, 3, 4], dev), _i32([1] * n, dev)
    c = Cache(BF16, p["hkv"], p["D"], 8, [90] * n, dev)
    states = FC.alloc_conv_state(7, 4, p["C"], BF16, dev), G.alloc_delta_state(7, hv, dev)
    keep = [t for t in (*states, c.k, c.v)]
    args = (p, x, (g, beta), qkv, *states, slots, None, (c.k, c.v), c.table, lens, False)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _mix(*args)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _mix(*args)
    for i in range(4):
        x.copy_(_randn(gen, x.shape, BF16, dev)), qkv.copy_(_randn(gen, qkv.shape, BF16, dev))
        g.copy_(-0.1 * torch.rand(g.shape, generator=gen)), beta.copy_(torch.rand(beta.shape, generator=gen))
        slots.copy_(_i32([5, -1, 0, 6, 1] if i % 2 else [3, 2, -1, 0, 6], dev))
        lens.copy_(_i32([1 + i, 8 * i, 0, 40 + i, 80 + i], dev))
        before = [t.clone() for t in keep]
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in (*out, *keep)]
        for t, b in zip(keep, before):
            t.copy_(b)
        eager = _mix(*args)
        torch.cuda.synchronize()
        for a, b in zip(replayed, (*eager, *keep)):
            assert torch.equal(a, b)


def test_captured_rotary_training_step(dev):
    gen = torch.Generator().manual_seed(13)
    q, k = _randn(gen, (40, 4, 64), BF16, dev).requires_grad_(), _randn(gen, (40, 2, 64), BF16, dev).requires_grad_()
    ups = [_randn(gen, t.shape, BF16, dev) for t in (q, k)]
    f, cu = A.rotary_inv_freq(64, 1e4, dev), _i32([0, 9, 40], dev)

    def step():
        out = A.rotary(q, k, f, cu_seqlens=cu)
        return [*(t.detach() for t in out), *torch.autograd.grad(out, (q, k), ups)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        with torch.no_grad():
            q.copy_(_randn(gen, q.shape, BF16, dev)), k.copy_(_randn(gen, k.shape, BF16, dev))
        cu.copy_(_i32([0, 3 * i + 1, 40 - i], dev))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_other_streams(dev):
    """Calls on a stream of their own, beside others on the current one."""
    r, c = Rule(BF16, 2, 4, [1] * 20, dev), Conv(BF16, 4, 256, [1] * 20, dev)
    before, kept = r.state.clone(), c.state.clone()
    o, y = r.call(cu=False), c.call(cu=False)
    after = r.state.clone(), c.state.clone()
    r.state.copy_(before), c.state.copy_(kept)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        o2, y2 = r.call(cu=False), c.call(cu=False)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(o, o2) and torch.equal(y, y2) and torch.equal(r.state, after[0]) and torch.equal(c.state, after[1])


def test_a_backward_that_saved_a_state_raises(dev):
    """The states count as written in place."""
    r, c = Rule(BF16, 1, 2, [1], dev), Conv(BF16, 4, 16, [1], dev)
    for t, call in ((r.state, r.call), (c.state, c.call)):
        w = torch.ones_like(t, requires_grad=True)
        loss = (w * t).sum()
        with torch.no_grad():
            call()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


def test_traces_hold_the_calls(dev):
    r = Rule(BF16, 1, 2, [1, 1], dev, extra=0)
    slots = _i32([0, 1], dev)

    def fn(q, k, v, g, beta, state):
        return G.recurrent_gated_delta_rule(q, k, v, g, beta, state, slots)

    args = (r.q.contiguous(), r.k.contiguous(), r.v.contiguous(), r.g, r.beta)
    want = fn(*args, r.state.clone())
    traced = torch.jit.trace(fn, (*args, r.state.clone()), check_trace=False)
    assert torch.equal(traced(*args, r.state.clone()), want)

    w, f = torch.ones((4, 16), dtype=BF16, device=dev), A.rotary_inv_freq(64, 1e4, dev)
    gen = torch.Generator().manual_seed(14)
    x, states = _randn(gen, (2, 16), BF16, dev), FC.alloc_conv_state(2, 4, 16, BF16, dev)

    def conv(x, state):
        return FC.causal_conv1d_update(x, w, state)

    traced = torch.jit.trace(conv, (x, states.clone()), check_trace=False)
    y, kept, kept2 = 2 * x, states.clone(), states.clone()
    assert torch.equal(traced(y, kept), conv(y, kept2)) and torch.equal(kept, kept2)

    rows = _randn(gen, (2, 4, 64), BF16, dev)
    table, lens = _i32([[0], [1]], dev), _i32([3, 8], dev)

    def append(rows, kc, vc):
        return A.rotary_append_kv(rows[:, :2], rows[:, 2:3], rows[:, 3:], kc, vc, table, lens, f)

    caches = [[torch.zeros_like(t) for t in A.alloc_kv_cache(2, 8, 1, 64, BF16, dev)] for _ in range(3)]
    traced = torch.jit.trace(append, (rows, *caches[0]), check_trace=False)
    rows = 2 * rows
    assert torch.equal(traced(rows, *caches[1]), append(rows, *caches[2]))
    assert torch.equal(caches[1][0], caches[2][0]) and torch.equal(caches[1][1], caches[2][1])
    assert caches[1][0].any() and caches[1][1].any()

    def turn(rows):
        return A.rotary(rows[:, :3], rows[:, 3:], f, positions=lens)

    traced = torch.jit.trace(turn, (rows,), check_trace=False)
    assert all(torch.equal(a, b) for a, b in zip(traced(2 * rows), turn(2 * rows)))


def test_captured_runs_replay(dev):
    """Prompts and single tokens in a graph whose sequences' ends, slots and lengths change between replays, the last of them
    without rows; padding rows of NaN behind them."""
    gen = torch.Generator().manual_seed(15)
    p = _layer(gen, dev)
    n, rows, hv = 4, 90, p["hv"]
    x, qkv = _randn(gen, (rows, p["C"]), BF16, dev), _randn(gen, (rows, p["hq"] + 2 * p["hkv"], p["D"]), BF16, dev)
    g, beta = -0.1 * torch.rand((rows, hv), device=dev), torch.ones((rows, hv), dtype=BF16, device=dev)
    slots, lens, cu = _i32([0, 1, 2, 3], dev), _i32([1, 40, 2, 5], dev), _i32([0, 1, 41, 43, 48], dev)
    c = Cache(BF16, p["hkv"], p["D"], 8, [90] * n, dev)
    states = FC.alloc_conv_state(6, 4, p["C"], BF16, dev), G.alloc_delta_state(6, hv, dev)
    keep = [*states, c.k, c.v]

    def step():
        y = FC.causal_conv1d_update(x, p["conv"], states[0], slots, cu, activation="silu")
        q, k, v = y.view(rows, -1, 128).split((p["hk"], p["hk"], hv), 1)
        o = G.recurrent_gated_delta_rule(q, k, v, g, beta, states[1], slots, cu, use_qk_norm_in_gdn=True)
        q, k, v = qkv.split((p["hq"], p["hkv"], p["hkv"]), 1)
        return [y, o, *A.rotary_append_kv(q, k, v, c.k, c.v, c.table, lens, p["freq"], cu_seqlens=cu, return_k=True)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i, ends in enumerate(([1, 2, 3, 4], [33, 34, 34, 90], [0, 0, 0, 0], [70, 75, 77, 80], [1, 41, 43, 48])):
        x.copy_(_randn(gen, x.shape, BF16, dev)), qkv.copy_(_randn(gen, qkv.shape, BF16, dev))
        x[ends[-1]:], qkv[ends[-1]:] = float("nan"), float("nan")
        cu.copy_(_i32([0] + ends, dev))
        slots.copy_(_i32([5, -1, 0, 1] if i % 2 else [3, 2, 4, -1], dev))
        lens.copy_(_i32([max(b - a, 0) + i for a, b in zip([0] + ends, ends)], dev))
        before = [t.clone() for t in keep]
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in (*out, *keep)]
        for t, b in zip(keep, before):
            t.copy_(b)
        eager = step()
        torch.cuda.synchronize()
        for a, b in zip(replayed, (*eager, *keep)):
            assert torch.equal(a, b)


def test_two_streams_at_once(dev):
    """Two streams' calls on slots of their own of the same pools, in flight together, give what they give in turn."""
    calls, before, want = [], [], []
    for seed in range(2):
        r, c = Rule(BF16, 2, 8, [200, 1, 33, 5], dev, seed=seed), Conv(BF16, 4, 1024, [200, 1, 33, 5], dev, seed=seed)
        if calls:  # one pool for both
            pool, conv = calls[0][0].state, calls[0][1].state
            pool[7:], conv[7:] = r.state, c.state
            r.state, c.state = pool, conv
            r.slots, c.slots = [s + 7 for s in r.slots], [s + 7 for s in c.slots]
        else:
            r.state, c.state = torch.cat([r.state, r.state]), torch.cat([c.state, c.state])
        calls.append((r, c))
    pools = calls[0][0].state, calls[0][1].state
    before = [t.clone() for t in pools]
    want = [(r.call(), c.call()) for r, c in calls]
    after = [t.clone() for t in pools]
    for t, b in zip(pools, before):
        t.copy_(b)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in calls], []
    for s, (r, c) in zip(streams, calls):
        with torch.cuda.stream(s):
            got.append((r.call(), c.call()))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert torch.equal(pools[0], after[0]) and torch.equal(pools[1], after[1])
