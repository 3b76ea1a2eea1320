"""Sequence operators on the GPU through their plans, against the formulas in float64
(oracle/sequences.py) at small sizes where they can go wrong.

Tolerances.  With u = 2^-24 (float32's half step) a float32 evaluation of a sum of products is off by at
most (roundings along the longest chain) * u times the same sum over absolute values, which the oracle
computes (``magnitude=True``).  The chains:

* convolution: taps products and additions, the bias: taps + 2; its silu: an exponential of relative error
  (2 + 1.2 |v|) * 2u whose effect on v sigmoid(v) is at most 1.2 u |v| (2 + 1.2 |v|) e^-|v| ... < 8 u, a
  division (4 u) and two products: 16 more.
* scan: a row's factor exp(s A) carries 4 u (the exponential's two units in the last place, 2^-22) plus
  |s A| times the relative error of its argument: two products (2 u), log2 e (u) and s itself, whose
  softplus is log1p of an exponential (2 + 1.2 |v|) * 2 u <= 24 u for |v| <= 8, log1p 2 u: 30 u in all.
  Two more for the multiply-add: a row adds (6 + 30 |s A|) u to what passes through it, so T rows
  T (6 + 30 max |s A|); the rest of the chain (s x B, the sums over at most 128 states and over the
  channels of a group, gate, products of gradients) stays under 200 + channels + rows.
* norms: sums over the channels are split over the lanes of a block, 32 additions in a thread at most and
  10 levels of a tree: under 64 roundings, twice (two norms), and the square root's argument is a sum of
  squares, whose relative error halves; sums over rows in order: rows.

A value is then rounded to its type once: half a step, eps/2 relative (for a result below the smallest
normal number half its step, tiny * eps / 2 ... the ``+ tiny`` below)."""

import ctypes

import numpy as np
import pytest

from nengo_ocl_b200 import cura_sequence as seq
from nengo_ocl_b200.curaggedarray import CUDARaggedArray
from nengo_ocl_b200.plan import Plans
from nengo_ocl_b200.raggedarray import RaggedArray
from nengo_ocl_b200.runtime import CommandQueue, DeviceArray, to_device
from nengo_ocl_b200.utils import as_dtype, bfloat16, from_bfloat16
from oracle import sequences as S

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_STEP = {np.dtype(np.float32): 2.0 ** -24, np.dtype(np.float16): 2.0 ** -11, bfloat16: 2.0 ** -8}
TINY = {np.dtype(np.float32): 2.0 ** -126, np.dtype(np.float16): 2.0 ** -24, bfloat16: 2.0 ** -126}
F32, F16, BF16 = np.dtype(np.float32), np.dtype(np.float16), bfloat16
DTYPES = pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])


def widen(a):
    return (from_bfloat16(a) if a.dtype == bfloat16 else np.asarray(a)).astype(np.float64)


class Rows:
    """A sequence array on the device: items inside a wider buffer (``pad`` columns around, ``lead``
    elements in front), everything else filled with a guard value."""

    def __init__(self, queue, items, dtype, pad=0, lead=0, empty=False, columns=None):
        self.dtype = np.dtype(dtype)
        items = [np.asarray(v) for v in items]
        columns = columns or items[0].shape[1]
        pitch = columns + pad
        n = np.array([len(v) for v in items])
        self.starts = lead + (np.cumsum(n) - n) * pitch
        self.guard = as_dtype(np.float32(-7.5), self.dtype)
        buf = np.empty(lead + int(n.sum()) * pitch + 19, self.dtype)
        buf[:] = self.guard
        self.covered = np.zeros(len(buf), bool)
        self.values = []
        self.place = [(int(s), len(v), columns, pitch) for s, v in zip(self.starts, items)]
        for (s, r, c, p), v in zip(self.place, items):
            at = s + np.arange(r)[:, None] * p + np.arange(c)
            self.covered[at] = True
            if not empty:
                buf[at] = as_dtype(v, self.dtype)
            self.values.append(widen(buf[at]))
        self.buf = to_device(queue, buf)
        k = len(n)
        self.ra = CUDARaggedArray.from_buffer(queue, self.buf, self.starts, n, [columns] * k, [pitch] * k, [1] * k)

    def get(self):
        buf = self.buf.get()
        outside = buf[~self.covered]
        assert np.array_equal(outside, np.full(outside.shape, self.guard, self.dtype)), "written outside the items"
        return [widen(buf[s + np.arange(r)[:, None] * p + np.arange(c)]) for s, r, c, p in self.place]


def close(got, want, magnitude, chain, dtype, what=""):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape, what
    tol = chain * U * np.asarray(magnitude) * (1 + HALF_STEP[dtype]) + HALF_STEP[dtype] * np.abs(want) + TINY[dtype]
    over = np.abs(got - want) > tol
    assert not over.any() and np.isfinite(got).all(), "%s: %d of %d off, worst %.3g times the tolerance" % (
        what, over.sum(), over.size, np.max(np.abs(got - want) / tol))


def vec(queue, v):
    return to_device(queue, np.asarray(v, np.float32))


def normal(rng, *shape):
    return rng.normal(size=shape).astype(np.float32)


LENGTHS = [[1], [0, 1, 2, 3, 5], [65, 1, 0, 40], [130]]


# ---- short causal convolution --------------------------------------------------------------------
@DTYPES
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
@pytest.mark.parametrize("chan,taps,pad,lead,silu,bias,state", [
    (1, 4, 0, 0, True, True, True), (7, 1, 3, 1, False, True, True), (64, 2, 0, 0, True, False, True),
    (136, 4, 8, 16, True, True, True), (136, 4, 1, 3, True, True, False), (520, 8, 0, 8, False, True, True),
    (24, 3, 40, 0, True, True, True), (1032, 5, 0, 0, True, True, True)])
def test_causal_conv(queue, rng, dtype, lengths, chan, taps, pad, lead, silu, bias, state):
    x = Rows(queue, [normal(rng, n, chan) for n in lengths], dtype, pad, lead)
    y = Rows(queue, x.values, dtype, pad + 8, lead, empty=True)
    w, b = normal(rng, chan, taps), normal(rng, chan) if bias else None
    old = Rows(queue, [normal(rng, taps - 1, chan) for _ in lengths], dtype, columns=chan) if state else None
    new = Rows(queue, [np.zeros((taps - 1, chan)) for _ in lengths], dtype, empty=True, columns=chan)
    plan = seq.plan_causal_conv(queue, x.ra, vec(queue, w), y.ra, bias=vec(queue, b) if bias else None,
                                state=old.ra if state else None, new_state=new.ra, activation="silu" if silu else None)
    plan()
    for k, (got, end) in enumerate(zip(y.get(), new.get())):
        s = old.values[k] if state else None
        want, want_end = S.causal_conv(x.values[k], w, b, s, silu)
        size, _ = S.causal_conv(x.values[k], w, b, s, silu, magnitude=True)
        close(got, want, size, taps + 18, dtype, "y")
        assert np.array_equal(end, want_end)
    if state:  # in place, from the same start
        again = Rows(queue, x.values, dtype, empty=True, columns=chan)
        seq.plan_causal_conv(queue, x.ra, vec(queue, w), again.ra, bias=vec(queue, b) if bias else None, state=old.ra,
                             new_state=old.ra, activation="silu" if silu else None)()
        for a, b_, c, d in zip(again.get(), y.get(), old.get(), new.get()):
            assert np.array_equal(a, b_) and np.array_equal(c, d)


@DTYPES
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
@pytest.mark.parametrize("chan,taps,pad,lead,silu,bias,state,ends", [
    (1, 4, 0, 0, True, True, True, True), (7, 1, 3, 1, False, True, False, False),
    (64, 2, 0, 0, True, False, True, True), (136, 4, 8, 16, True, True, True, True),
    (136, 4, 1, 3, True, True, True, False), (520, 8, 0, 8, True, True, False, True), (24, 3, 0, 0, False, True, True, True)])
def test_causal_conv_grad(queue, rng, dtype, lengths, chan, taps, pad, lead, silu, bias, state, ends):
    x = Rows(queue, [normal(rng, n, chan) for n in lengths], dtype, pad, lead)
    y, dx = (Rows(queue, x.values, dtype, pad, lead, empty=True) for _ in range(2))
    dy = Rows(queue, [normal(rng, n, chan) for n in lengths], dtype, pad, lead)
    w, b = normal(rng, chan, taps), normal(rng, chan) if bias else None
    tails = lambda empty=False: Rows(queue, [normal(rng, taps - 1, chan) for _ in lengths], dtype, empty=empty, columns=chan)
    old, dold, dnew = tails() if state else None, tails(True) if state else None, tails() if ends else None
    fwd = seq.plan_causal_conv(queue, x.ra, vec(queue, w), y.ra, bias=vec(queue, b) if bias else None,
                               state=old.ra if state else None, activation="silu" if silu else None)
    dw, db = vec(queue, np.full((chan, taps), 9)), vec(queue, np.full(chan, 9))
    bwd = seq.plan_causal_conv_grad(queue, fwd, dy.ra, dx.ra, dw, dbias=db if bias else None,
                                    dstate=dold.ra if state else None, dnew_state=dnew.ra if ends else None)
    bwd()
    first = dw.get()
    sums = {"dw": 0, "dbias": 0}
    sizes = {"dw": 0, "dbias": 0}
    for k, got in enumerate(dx.get()):
        args = dict(x=x.values[k], w=w, dy=dy.values[k], bias=b, state=old.values[k] if state else None,
                    dnew_state=dnew.values[k] if ends else None, silu_=silu)
        want, size = S.causal_conv_grad(**args), S.causal_conv_grad(**args, magnitude=True)
        # the slope of silu carries the sum's error (taps + 2) and its own (an exponential, a division: 24)
        chain = 3 * taps + 40
        # (the slope's error in `pre`: its magnitude, at most sum |w x|, bounds |silu''| <= 1/2 times the error)
        pre = S.causal_conv(x.values[k], w, b, args["state"], False, magnitude=True)[0]
        extra = 1 + (pre.max() if pre.size else 0)
        close(got, want["dx"], size["dx"] * extra, chain, dtype, "dx")
        if state:
            close(dold.get()[k], want["dstate"], size["dstate"] * extra, chain, dtype, "dstate")
        for name in sums:
            sums[name], sizes[name] = sums[name] + want[name], sizes[name] + size[name] * extra
    rows = sum(lengths)
    close(dw.get(), sums["dw"], sizes["dw"], 3 * taps + 40 + rows, F32, "dw")
    if bias:
        close(db.get(), sums["dbias"], sizes["dbias"], 3 * taps + 40 + rows, F32, "dbias")
    bwd()
    assert np.array_equal(dw.get(), first)


UNIT_LENGTHS = [[17, 0, 64, 65, 130, 9], [8, 9, 16, 1, 33]]


@DTYPES
@pytest.mark.parametrize("lengths", UNIT_LENGTHS, ids=str)
@pytest.mark.parametrize("unit_rows", [9, 17, 64])
@pytest.mark.parametrize("chan,taps,pad,lead,silu", [(136, 4, 8, 16, True), (520, 8, 0, 8, False), (24, 2, 0, 0, True),
                                                     (33, 3, 1, 1, True)])
def test_causal_conv_in_long_units(queue, rng, monkeypatch, dtype, lengths, unit_rows, chan, taps, pad, lead, silu):
    """Units of more rows than a group, as large batches have them: rows copied ahead, several groups to a unit."""
    monkeypatch.setattr(seq, "_unit_rows", lambda *a: unit_rows)
    plans = _recorded(monkeypatch, "plan_causal_conv")
    test_causal_conv(queue, rng, dtype, lengths, chan, taps, pad, lead, silu, True, True)
    assert plans and all(p.full_args[0].unit_rows == unit_rows for p in plans)
    assert all(p.full_args[0].vec == (chan != 33) for p in plans[:1])


@DTYPES
@pytest.mark.parametrize("unit_rows", [9, 17, 64])
@pytest.mark.parametrize("chan,taps,pad,lead,silu", [(136, 4, 8, 16, True), (520, 8, 0, 8, False), (33, 3, 1, 1, True)])
def test_causal_conv_grad_in_long_units(queue, rng, monkeypatch, dtype, unit_rows, chan, taps, pad, lead, silu):
    monkeypatch.setattr(seq, "_unit_rows", lambda *a: unit_rows)
    plans = _recorded(monkeypatch, "plan_causal_conv_grad")
    test_causal_conv_grad(queue, rng, dtype, UNIT_LENGTHS[0], chan, taps, pad, lead, silu, True, True, True)
    assert plans and all(p.full_args[0].unit_rows == unit_rows for p in plans)


def _recorded(monkeypatch, name):
    """The plans that ``seq.<name>`` makes from here on."""
    plans, make = [], getattr(seq, name)
    monkeypatch.setattr(seq, name, lambda *a, **k: plans.append(make(*a, **k)) or plans[-1])
    return plans


def _float32_sum(values):
    total = np.float32(0)
    for v in values:
        total = np.float32(total + v)
    return total


@pytest.mark.parametrize("rows", [64, 1000, 40003])
def test_order_of_the_sums_over_rows(queue, rng, rows):
    """dbias (and dw where x is one) without an activation is a plain sum: four rows apart, then a unit's groups
    of them, every eighth unit in runs of 16, the eight shares.  The float32 additions in that order, to the bit."""
    chan, taps = 4, 2
    x, dy = Rows(queue, [np.ones((rows, chan))], F32), Rows(queue, [normal(rng, rows, chan) + 1], F32)
    y, dx = (Rows(queue, x.values, F32, empty=True) for _ in range(2))
    dw, db = vec(queue, np.zeros((chan, taps))), vec(queue, np.zeros(chan))
    fwd = seq.plan_causal_conv(queue, x.ra, vec(queue, np.ones((chan, taps))), y.ra, bias=vec(queue, np.zeros(chan)))
    bwd = seq.plan_causal_conv_grad(queue, fwd, dy.ra, dx.ra, dw, dbias=db)
    bwd()
    unit = bwd.full_args[0].unit_rows
    assert unit % 4 == 0 and (rows < 40000 or bwd.full_args[0].n_units > 128)
    for c in range(chan):
        v = dy.values[0][:, c].astype(np.float32)
        units = [_float32_sum(_float32_sum(v[i:min(i + 4, t + unit)]) for i in range(t, min(t + unit, rows), 4))
                 for t in range(0, rows, unit)]
        shares = [_float32_sum(_float32_sum(units[w::8][i:i + 16]) for i in range(0, len(units[w::8]), 16)) for w in range(8)]
        assert db.get()[c] == dw.get()[c, 1] == _float32_sum(shares)


# ---- selective scan ------------------------------------------------------------------------------
class Scan:
    """Arguments of a scan at the usual scales, on the device and for the oracle."""

    def __init__(self, queue, rng, lengths, chan, n, groups, dtype, pad=0, lead=0, D=True, gate=True, bias=True,
                 softplus=True, state=True):
        rows = lambda c=chan, scale=1.0: Rows(queue, [scale * normal(rng, k, c) for k in lengths], dtype, pad, lead, columns=c)
        self.queue, self.lengths, self.chan, self.n, self.dtype = queue, lengths, chan, n, dtype
        self.x, self.B, self.C = rows(), rows(groups * n), rows(groups * n, n ** -0.5)
        if softplus:
            self.dt = rows()
        else:
            self.dt = Rows(queue, [rng.uniform(0.01, 0.3, size=(k, chan)) for k in lengths], dtype, pad, lead, columns=chan)
        self.z = rows() if gate else None
        self.A = -rng.uniform(0.5, 4, size=(chan, n)).astype(np.float32)
        self.D = normal(rng, chan) if D else None
        self.bias = (rng.uniform(-4, -1, size=chan) if softplus else rng.uniform(0, 0.1, size=chan)).astype(np.float32) \
            if bias else None
        self.softplus = softplus
        self.state = Rows(queue, [normal(rng, chan, n) for _ in lengths], F32) if state else None
        self.y = Rows(queue, self.x.values, dtype, pad, lead, empty=True, columns=chan)
        self.new = Rows(queue, [np.zeros((chan, n)) for _ in lengths], F32, empty=True)
        self.params = {k: vec(queue, v) for k, v in (("A", self.A), ("D", self.D), ("dt_bias", self.bias)) if v is not None}

    def plan(self, **more):
        args = dict(new_state=self.new.ra, keep=False)
        args.update(more)
        return seq.plan_selective_scan(
            self.queue, self.x.ra, self.dt.ra, self.params["A"], self.B.ra, self.C.ra, self.y.ra, D=self.params.get("D"),
            Z=self.z.ra if self.z else None, dt_bias=self.params.get("dt_bias"), softplus=self.softplus,
            **dict(dict(state=self.state.ra if self.state else None), **args))

    def of(self, k):
        return dict(x=self.x.values[k], dt=self.dt.values[k], A=self.A, B=self.B.values[k], C=self.C.values[k], D=self.D,
                    z=self.z.values[k] if self.z else None, dt_bias=self.bias, softplus=self.softplus,
                    state=self.state.values[k] if self.state else None)

    def chain(self, k, more=0):
        _, s = S.scan_steps(self.dt.values[k], self.bias, self.softplus)
        top = float((s.max() if s.size else 0) * np.abs(self.A).max())
        return self.lengths[k] * (6 + 30 * top) + 200 + more

    def check(self):
        for k, (got, end) in enumerate(zip(self.y.get(), self.new.get())):
            want, want_end = S.selective_scan(**self.of(k))
            size, size_end = S.selective_scan(**self.of(k), magnitude=True)
            close(got, want, size, self.chain(k), self.dtype, "y")
            close(end, want_end, size_end, self.chain(k), F32, "new_state")


SCANS = [  # chan, n, groups, pad, lead, options
    (1, 1, 1, 0, 0, {}), (40, 3, 2, 1, 3, dict(gate=False)), (33, 4, 1, 0, 0, dict(D=False)), (48, 8, 3, 8, 8, {}),
    (130, 12, 2, 4, 4, dict(state=False)), (72, 16, 1, 0, 0, {}), (70, 16, 2, 8, 16, dict(bias=False)),
    (10, 17, 1, 0, 0, dict(softplus=False)), (9, 33, 1, 3, 0, {}), (12, 64, 2, 0, 0, {}),
    (5, 128, 1, 0, 0, dict(softplus=False, bias=False)), (3, 127, 1, 1, 1, {})]


@DTYPES
@pytest.mark.parametrize("lengths", LENGTHS + [[210, 0, 33]], ids=str)
@pytest.mark.parametrize("chan,n,groups,pad,lead,options", SCANS)
def test_selective_scan(queue, rng, dtype, lengths, chan, n, groups, pad, lead, options):
    s = Scan(queue, rng, lengths, chan, n, groups, dtype, pad, lead, **options)
    s.plan()()
    s.check()
    first = s.y.buf.get(), s.new.buf.get()
    s.plan(keep=True)()  # (few rows: another kernel, which adds the states in another order)
    s.check()
    if s.state:  # in place
        s.plan(new_state=s.state.ra)()
        assert np.array_equal(s.y.buf.get(), first[0])
        for a, b in zip(s.state.buf.get(), first[1]):
            assert np.array_equal(a, b)


@DTYPES
@pytest.mark.parametrize("lengths", LENGTHS + [[210, 0, 33]], ids=str)
@pytest.mark.parametrize("chan,n,groups,pad,lead,options", SCANS)
def test_selective_scan_grad(queue, rng, dtype, lengths, chan, n, groups, pad, lead, options):
    s = Scan(queue, rng, lengths, chan, n, groups, dtype, pad, lead, **options)
    like = lambda r: Rows(queue, r.values, r.dtype, pad if r.dtype != F32 or dtype == F32 else 0, lead, empty=True,
                          columns=r.place[0][2])
    dy = Rows(queue, [normal(rng, k, chan) for k in lengths], dtype, pad, lead, columns=chan)
    dx, ddt, dB, dC = like(s.x), like(s.dt), like(s.B), like(s.C)
    dz = like(s.z) if s.z else None
    dstate = Rows(queue, [np.zeros((chan, n)) for _ in lengths], F32, empty=True) if s.state else None
    dnew = Rows(queue, [normal(rng, chan, n) for _ in lengths], F32) if s.state else None
    grads = {"d" + k: vec(queue, np.full(v.shape, 9.0)) for k, v in s.params.items()}
    fwd = s.plan(keep=True)
    bwd = seq.plan_selective_scan_grad(
        queue, fwd, dy.ra, dx.ra, ddt.ra, grads["dA"], dB.ra, dC.ra, dD=grads.get("dD"), dZ=dz.ra if dz else None,
        ddt_bias=grads.get("ddt_bias"), dstate=dstate.ra if dstate else None, dnew_state=dnew.ra if dnew else None)
    fwd()
    bwd()
    rows_of = dict(dx=dx, ddt=ddt, dB=dB, dC=dC, dz=dz, dstate=dstate)
    sums = {k: [0, 0, 0] for k in ("dA", "dD", "ddt_bias")}
    for k in range(len(lengths)):
        args = dict(s.of(k), dy=dy.values[k], dnew_state=dnew.values[k] if dnew else None)
        want, size = S.selective_scan_grad(**args), S.selective_scan_grad(**args, magnitude=True)
        chain = 2 * s.chain(k, chan + sum(lengths))
        for name, r in rows_of.items():
            if r is not None:
                close(r.get()[k], want[name], size[name], chain, r.dtype, name)
        for name, v in sums.items():
            v[0], v[1], v[2] = v[0] + want[name], v[1] + size[name], max(v[2], chain)
    for name, (want, size, chain) in sums.items():
        if name in grads:
            close(grads[name].get(), want, size, chain, F32, name)
    before = {k: v.get() for k, v in grads.items()}, dB.buf.get(), ddt.buf.get()
    bwd()
    assert all(np.array_equal(before[0][k], v.get()) for k, v in grads.items())
    assert np.array_equal(before[1], dB.buf.get()) and np.array_equal(before[2], ddt.buf.get())


@DTYPES
@pytest.mark.parametrize("n_seq,chan,n,groups,each", [
    (131, 1024, 4, 1024, 64),  # (the most sequences of a block, and a last block with the rest)
    (301, 512, 16, 2, 2), (100, 1000, 128, 1, 6), (40, 1010, 128, 2, 3), (37, 2370, 3, 790, 19)])  # (2368 // 790 tiles: two blocks to a tile)
@pytest.mark.parametrize("longest", [1, 2])
def test_tokens_of_many_sequences(queue, rng, dtype, n_seq, chan, n, groups, each, longest):
    """A block takes several sequences one after the other, the next one's state on its way: 0, 1 or 2 rows each, states
    in place, in the order of a pool's slots."""
    lengths = list(rng.randint(0, longest + 1, size=n_seq))
    lengths[:2] = [longest, 0]
    s = Scan(queue, rng, lengths, chan, n, groups, dtype)
    start = s.state.buf.get()
    plan = s.plan()
    args = plan.full_args[0]
    # 16 blocks to each of the 148 multiprocessors; a block takes as many channels as the walk's
    tiles = groups * -(-(chan // groups) // seq.scan_tile(n))
    blocks = max(1, min(n_seq, 16 * 148 // tiles))
    assert args.tokens == 1 and min(-(-n_seq // blocks), 64) == each
    plan()
    s.check()
    y, new = s.y.buf.get(), s.new.buf.get()
    in_place = s.plan(new_state=s.state.ra)
    in_place()
    assert np.array_equal(s.y.buf.get(), y) and np.array_equal(s.state.buf.get(), new)
    # one sequence by itself: the same additions
    s.state.buf.set(start)
    k = int(np.argmax(lengths[5:])) + 5
    one = lambda r: r.ra[[k]]
    alone = Rows(queue, [np.zeros((lengths[k], chan))], dtype, empty=True, columns=chan)
    seq.plan_selective_scan(queue, one(s.x), one(s.dt), s.params["A"], one(s.B), one(s.C), alone.ra, D=s.params["D"],
                            Z=one(s.z), dt_bias=s.params["dt_bias"], softplus=True, state=one(s.state))()
    assert np.array_equal(alone.get()[0], s.y.get()[k])
    # slots of a pool, in another order, in place
    slots = rng.permutation(n_seq)
    s.plan(state=s.state.ra[slots], new_state=s.state.ra[slots])()
    s.state.values = [s.state.values[i] for i in slots]
    s.new.get = lambda have=s.state.get(): [have[i] for i in slots]
    s.check()


def test_several_sequences_start_from_one_state(queue, rng):
    s = Scan(queue, rng, [4, 7, 0], 12, 16, 1, F32)
    s.plan(state=s.state.ra[[1, 1, 1]])()
    s.state.values = [s.state.values[1]] * 3
    s.check()


def test_sequences_do_not_mix(queue, rng):
    """NaN and infinities of one sequence, and of a sequence's later rows, reach nothing else."""
    lengths = [40, 33, 20]
    clean = Scan(queue, rng, lengths, 24, 16, 1, F32)
    clean.plan()()
    want = clean.y.get(), clean.new.get()
    for array in (clean.x, clean.dt, clean.B, clean.C, clean.z):
        items = [v.copy() for v in array.values]
        items[1][:] = np.nan
        items[2][10:] = np.inf
        saved, array.ra = array.ra, Rows(queue, items, F32).ra
        clean.plan()()
        array.ra = saved
        got = clean.y.get(), clean.new.get()
        assert np.array_equal(got[0][0], want[0][0]) and np.array_equal(got[1][0], want[1][0])
        assert np.array_equal(got[0][2][:10], want[0][2][:10])
    # the convolution's rows before a NaN, and the other sequences
    x = [normal(rng, n, 24) for n in lengths]
    w = vec(queue, normal(rng, 24, 4))
    outs = []
    for poison in (False, True):
        if poison:
            x[1][5:] = np.nan
        y = Rows(queue, x, F32, empty=True)
        seq.plan_causal_conv(queue, Rows(queue, x, F32).ra, w, y.ra)()
        outs.append(y.get())
    assert np.array_equal(outs[0][0], outs[1][0]) and np.array_equal(outs[0][2], outs[1][2])
    assert np.array_equal(outs[0][1][:5], outs[1][1][:5]) and np.isnan(outs[1][1][5:]).all()


def test_scan_forgets_at_infinite_decay(queue, rng):
    """A = -inf: every row's state is its own input alone, and an empty sequence's state stays."""
    s = Scan(queue, rng, [6, 0, 35], 8, 4, 1, F32, bias=False, softplus=False)
    s.A[:] = -np.inf
    s.params["A"] = vec(queue, s.A)
    s.plan()()
    for k, (y, end) in enumerate(zip(s.y.get(), s.new.get())):
        own = (s.dt.values[k] * s.x.values[k])[:, :, None] * s.B.values[k][:, None, :]
        if not len(own):
            assert np.array_equal(end, s.state.values[k])
            continue
        p = (own * s.C.values[k][:, None, :]).sum(-1) + s.D * s.x.values[k]
        size = np.abs(own * s.C.values[k][:, None, :]).sum(-1) + np.abs(s.D * s.x.values[k])
        gate = S.silu(s.z.values[k])
        close(y, p * gate, size * np.abs(gate), 40, F32, "y")
        close(end, own[-1], np.abs(own[-1]), 4, F32, "new_state")


@pytest.mark.parametrize("lengths,split", [([210, 0, 33], True), ([1, 2, 0, 1], False), ([40, 90], False)], ids=str)
def test_zero_steps_at_infinite_decay(queue, rng, lengths, split):
    """A = -inf and masked rows (a step of zero) among others: such a row leaves the state as it is, wherever the
    sequence is split and whichever kernel takes it.  The oracle's A is -1e30, which decays as completely."""
    s = Scan(queue, rng, lengths, 8, 4, 1, F32, bias=False, softplus=False)
    for k, n in enumerate(lengths):
        s.dt.values[k][(2 * n) // 10:(8 * n + 9) // 10] = 0
    s.dt = Rows(queue, s.dt.values, F32, columns=8)
    s.A[:] = -np.inf
    s.params["A"] = vec(queue, s.A)
    plan = s.plan()
    assert (plan.full_args[0].n_units > len(lengths)) == split and bool(plan.full_args[0].tokens) == (max(lengths) < 3)
    dy = Rows(queue, [normal(rng, n, 8) for n in lengths], F32, columns=8)
    outs = {name: Rows(queue, r.values, F32, empty=True, columns=r.place[0][2])
            for name, r in (("dx", s.x), ("ddt", s.dt), ("dB", s.B), ("dC", s.C))}
    dstate, dnew = Rows(queue, s.state.values, F32, empty=True), Rows(queue, [normal(rng, 8, 4) for _ in lengths], F32)
    dA = vec(queue, np.full((8, 4), 9.0))
    plan()
    y, new = s.y.get(), s.new.get()
    fwd = s.plan(keep=True)
    bwd = seq.plan_selective_scan_grad(queue, fwd, dy.ra, outs["dx"].ra, outs["ddt"].ra, dA, outs["dB"].ra, outs["dC"].ra,
                                       dstate=dstate.ra, dnew_state=dnew.ra)
    assert (bwd.full_args[0].n_units > len(lengths)) == split
    fwd()
    bwd()
    assert (dA.get() == 0).all()
    for k in range(len(lengths)):
        args = dict(s.of(k), A=np.full((8, 4), -1e30))
        want, size = S.selective_scan(**args), S.selective_scan(**args, magnitude=True)
        for got in ((y[k], new[k]), (s.y.get()[k], s.new.get()[k])):
            for g, w, m, what in zip(got, want, size, ("y", "new_state")):
                close(g, w, m, lengths[k] * 6 + 200, F32, what)
        grads = dict(args, dy=dy.values[k], dnew_state=dnew.values[k])
        want, size = S.selective_scan_grad(**grads), S.selective_scan_grad(**grads, magnitude=True)
        for name, r in dict(outs, dstate=dstate).items():
            if name != "ddt":  # (q A of a state that stays: infinite)
                close(r.get()[k], want[name], size[name], 2 * (lengths[k] * 6 + 300), F32, name)


def test_growing_states_over_split_sequences(queue, rng):
    """A > 0 (and steps of both signs): over a unit of 32 rows the growth passes float32's range, the states do
    not.  A zero state stays zero, a small one grows to what it is row by row."""
    lengths = [224, 224]
    s = Scan(queue, rng, lengths, 8, 4, 1, F32, bias=False, softplus=False, D=False, gate=False)
    sign = np.where(np.arange(224) // 32 % 2, -1.0, 1.0)[:, None]
    s.dt = Rows(queue, [np.broadcast_to(sign, (224, 8))] * 2, F32)
    x = np.zeros((224, 8), np.float32)
    x[200:] = normal(rng, 24, 8) * 1e-20  # (rows that grow, for less than a unit)
    s.x = Rows(queue, [x, x], F32)
    s.A = np.full((8, 4), 4.0, np.float32)  # 32 rows: e^128
    s.params["A"] = vec(queue, s.A)
    state = np.full((8, 4), 1e-30, np.float32)
    s.state = Rows(queue, [np.zeros((8, 4)), state], F32)
    dy = Rows(queue, [np.where(np.arange(224)[:, None] < 20, 1e-20, 0) * normal(rng, 224, 8) for _ in lengths], F32)
    outs = [Rows(queue, r.values, F32, empty=True) for r in (s.x, s.dt, s.B, s.C)]
    dnew = Rows(queue, [np.zeros((8, 4)), state], F32)
    dstate, dA = Rows(queue, [state] * 2, F32, empty=True), vec(queue, np.zeros((8, 4)))
    fwd = s.plan(keep=True)
    bwd = seq.plan_selective_scan_grad(queue, fwd, dy.ra, outs[0].ra, outs[1].ra, dA, outs[2].ra, outs[3].ra,
                                       dstate=dstate.ra, dnew_state=dnew.ra)
    assert fwd.full_args[0].unit_rows == bwd.full_args[0].unit_rows == 32
    fwd()
    bwd()
    s.check()
    for k in range(2):
        args = dict(s.of(k), dy=dy.values[k], dnew_state=dnew.values[k])
        want, size = S.selective_scan_grad(**args), S.selective_scan_grad(**args, magnitude=True)
        close(dstate.get()[k], want["dstate"], size["dstate"], 2 * s.chain(k, 300), F32, "dstate")


@pytest.mark.parametrize("chan,groups,n", [(40, 1, 16), (66, 2, 12), (9, 1, 64), (130, 1, 4), (3, 3, 128)])
@pytest.mark.parametrize("which", ["B", "C"])
def test_infinite_weights_of_a_partial_tile(queue, rng, which, chan, groups, n):
    """One infinite value of B (or C): with positive inputs dC of its row and the later ones (dB of its row and
    the earlier ones) is infinite in that state, nothing is NaN, and the rest is what it is without it.  The blocks'
    channels do not fill them, and what the idle lanes hold must not get into the sums over channels."""
    rows, at, state = 21, 9, n // 2
    s = Scan(queue, rng, [rows], chan, n, groups, F32, bias=False, softplus=False, gate=False, state=False)
    s.x = Rows(queue, [rng.uniform(0.5, 1, size=(rows, chan))], F32)
    dy = Rows(queue, [rng.uniform(0.5, 1, size=(rows, chan))], F32)
    dB, dC = (Rows(queue, [np.zeros((rows, groups * n))], F32, empty=True) for _ in range(2))
    want, size = (S.selective_scan_grad(**s.of(0), dy=dy.values[0], magnitude=m) for m in (False, True))
    items = getattr(s, which).values[0].copy()
    items[at, state] = np.inf
    setattr(s, which, Rows(queue, [items], F32))
    dx, ddt = (Rows(queue, [np.zeros((rows, chan))], F32, empty=True) for _ in range(2))
    fwd = s.plan(keep=True)
    bwd = seq.plan_selective_scan_grad(queue, fwd, dy.ra, dx.ra, ddt.ra, vec(queue, np.zeros((chan, n))), dB.ra, dC.ra)
    fwd()
    bwd()
    for name, r in (("dB", dB), ("dC", dC)):
        got = r.get()[0]
        infinite = np.zeros(got.shape, bool)
        if name == "dC" and which == "B":
            infinite[at:, state] = True
        if name == "dB" and which == "C":
            infinite[:at + 1, state] = True
        assert (got[infinite] == np.inf).all()
        close(got[~infinite], want[name][~infinite], size[name][~infinite], 2 * s.chain(0, chan + rows), F32, name)


@pytest.mark.parametrize("rows", [1, 7, 21, 16])
def test_a_state_that_overflows_in_the_last_row(queue, rng, rows):
    """The last state stands before no row, so dA does not see it, wherever in a tile the sequence ends."""
    chan, n = 40, 12
    s = Scan(queue, rng, [rows], chan, n, 1, F32)
    dy = Rows(queue, [normal(rng, rows, chan)], F32)
    want, size = (S.selective_scan_grad(**s.of(0), dy=dy.values[0], magnitude=m) for m in (False, True))
    B = s.B.values[0].copy()
    B[-1, 5] = np.inf
    s.B = Rows(queue, [B], F32)
    dA = vec(queue, np.full((chan, n), 9.0))
    outs = [Rows(queue, r.values, F32, empty=True) for r in (s.x, s.dt, s.B, s.C)]
    fwd = s.plan(keep=True)
    bwd = seq.plan_selective_scan_grad(queue, fwd, dy.ra, outs[0].ra, outs[1].ra, dA, outs[2].ra, outs[3].ra)
    fwd()
    bwd()
    assert np.isinf(s.new.get()[0][:, 5]).all()
    close(dA.get(), want["dA"], size["dA"], 2 * s.chain(0, chan + rows), F32, "dA")


def test_sums_over_rows_are_summed_by_tiles(queue, rng, monkeypatch):
    """dD of a unit of 1008 rows.  Sixteen rows to a tile, 63 tiles, and three more additions: under 90 roundings
    on the longest chain.  Row after row the same value, 1 + 255 * 2^-23, loses almost half a step with each of the
    last 496 additions: 250 half steps of the sum."""
    monkeypatch.setattr(seq, "SCAN_WHOLE_ROWS", 4096)
    rows, chan, value = 1008, 5, 1 + 255 * 2.0 ** -23
    s = Scan(queue, rng, [rows], chan, 4, 1, F32, gate=False)
    s.x = Rows(queue, [np.ones((rows, chan))], F32)
    dy = Rows(queue, [np.full((rows, chan), value)], F32)
    outs = [Rows(queue, r.values, F32, empty=True) for r in (s.x, s.dt, s.B, s.C)]
    dD = vec(queue, np.zeros(chan))
    fwd = s.plan(keep=True)
    bwd = seq.plan_selective_scan_grad(queue, fwd, dy.ra, outs[0].ra, outs[1].ra, vec(queue, s.A), outs[2].ra, outs[3].ra, dD=dD)
    assert bwd.full_args[0].n_units == 1
    fwd()
    bwd()
    close(dD.get(), np.full(chan, rows * value), rows * value, 90, F32, "dD")


def test_decays_are_right_on_average(queue, rng, monkeypatch):
    """A state that only decays, over 2048 rows of exponents between -0.04 and -0.02: the decays' mean error counts
    2048 times.  A mean of at most 0.2 half steps, and 0.7 of them at random (the exponential 0.53, the product's
    rounding 0.29, the exponent's less) six times sqrt(2048): 600.  Off by 0.45 on average it would be 900."""
    monkeypatch.setattr(seq, "SCAN_WHOLE_ROWS", 4096)
    rows, chan, n = 2048, 16, 4
    s = Scan(queue, rng, [rows], chan, n, 1, F32, bias=False, softplus=False, gate=False)
    s.A = -np.ones((chan, n), np.float32)
    s.params["A"] = vec(queue, s.A)
    s.dt = Rows(queue, [np.log(2) * rng.uniform(0.02, 0.04, size=(rows, chan))], F32)
    s.x = Rows(queue, [np.zeros((rows, chan))], F32)
    dy, dnew = Rows(queue, [np.zeros((rows, chan))], F32), Rows(queue, [normal(rng, chan, n)], F32)
    outs = [Rows(queue, r.values, F32, empty=True) for r in (s.x, s.dt, s.B, s.C)]
    dstate = Rows(queue, [np.zeros((chan, n))], F32, empty=True)
    fwd = s.plan(keep=True)
    bwd = seq.plan_selective_scan_grad(queue, fwd, dy.ra, outs[0].ra, outs[1].ra, vec(queue, s.A), outs[2].ra, outs[3].ra,
                                       dstate=dstate.ra, dnew_state=dnew.ra)
    assert fwd.full_args[0].n_units == bwd.full_args[0].n_units == 1
    fwd()
    bwd()
    decay = np.exp(-s.dt.values[0].sum(0))[:, None]
    for got, start in ((s.new, s.state), (dstate, dnew)):
        close(got.get()[0], decay * start.values[0], np.abs(decay * start.values[0]), 600, F32, "decayed")


# ---- norms ---------------------------------------------------------------------------------------
NORMS = [  # chan, groups, pad, lead, gate, gate_first, residual, weight, scale, norm_weight, Y, H
    (1, 1, 0, 0, True, True, True, True, True, True, True, True),
    (7, 7, 2, 1, True, False, True, True, True, True, True, True),
    (64, 8, 0, 0, True, True, True, True, True, True, True, True),
    (200, 1, 8, 8, False, True, False, False, 1.0, True, False, True),
    (1000, 5, 0, 0, True, False, True, True, 0.5, False, True, True),
    (1030, 2, 0, 3, True, True, False, True, True, True, True, False),
    (2048, 16, 0, 0, True, True, True, True, True, True, True, True),
    (4096, 1, 8, 0, False, True, True, False, True, True, True, True),
    (9001, 1, 0, 0, True, True, True, True, True, True, True, True),
    (20000, 4, 0, 0, True, False, True, True, True, True, True, True),
    (32768, 1, 0, 0, True, True, True, True, True, True, True, True),
    (32767, 1, 0, 0, True, True, True, True, True, True, False, True),
    (32766, 10922, 0, 0, True, False, True, True, True, True, True, True),
    (1280, 5, 0, 0, True, True, True, True, True, True, True, True),
    (3200, 100, 0, 0, False, True, True, True, 2.0, True, True, False)]


@DTYPES
@pytest.mark.parametrize("lengths", [[1], [3, 0, 2]], ids=str)
@pytest.mark.parametrize("chan,groups,pad,lead,gate,gate_first,residual,weight,scale,norm_weight,Y,H", NORMS)
def test_residual_norm(queue, rng, dtype, lengths, chan, groups, pad, lead, gate, gate_first, residual, weight, scale,
                       norm_weight, Y, H):
    rows = lambda empty=False: Rows(queue, [normal(rng, n, chan) for n in lengths], dtype, pad, lead, empty, chan)
    par = lambda: rng.uniform(0.5, 1.5, size=chan).astype(np.float32)
    x, g, r = rows(), rows() if gate else None, rows() if residual else None
    y, h = rows(True) if Y else None, rows(True) if H else None
    w, nw = par() if weight else None, par() if norm_weight and H else None
    sc = par() if scale is True else scale
    ra = lambda v: v.ra if v else None
    dev = lambda v: None if v is None else vec(queue, v)
    fwd = seq.plan_residual_norm(queue, x.ra, Y=ra(y), H=ra(h), gate=ra(g), gate_first=gate_first, residual=ra(r),
                                 weight=dev(w), scale=dev(sc) if scale is True else scale, norm_weight=dev(nw), groups=groups)
    fwd()
    of = lambda k: dict(x=x.values[k], gate=g.values[k] if g else None, gate_first=gate_first,
                        residual=r.values[k] if r else None, weight=w, scale=sc, norm_weight=nw, groups=groups)
    chain = 300
    for k in range(len(lengths)):
        want_y, want_h, (sg, u, inv, hat, o, rinv) = S.residual_norm(**of(k), parts=True)
        size = np.abs(sc * o) + (np.abs(r.values[k]) if r else 0)
        if Y:
            close(y.get()[k], want_y, size, chain, dtype, "y")
        if H:
            # (the norm of y: relative to it, and to its own row's error)
            top = np.sqrt((size ** 2).mean(-1, keepdims=True)) * rinv
            close(h.get()[k], want_h, (size * rinv + np.abs(want_y) * rinv * top) * (1 if nw is None else nw), chain, dtype, "h")
    # backward, from whichever outputs there are
    dy, dh = rows() if Y else None, rows() if H else None
    dx, dg, dr = rows(True), rows(True) if gate else None, rows(True) if residual else None
    grads = dict(dweight=w, dscale=sc if scale is True else None, dnorm_weight=nw)
    grads = {k: None if v is None else vec(queue, np.full(chan, 9.0)) for k, v in grads.items()}
    bwd = seq.plan_residual_norm_grad(queue, fwd, dx.ra, dY=ra(dy), dH=ra(dh), dgate=ra(dg), dresidual=ra(dr), **grads)
    bwd()
    sums = {k: [np.zeros(chan), np.zeros(chan)] for k in grads}
    for k in range(len(lengths)):
        args = dict(of(k), dy=dy.values[k] if dy else None, dh=dh.values[k] if dh else None)
        want = S.residual_norm_grad(**args)
        _, _, (sg, u, inv, hat, o, rinv) = S.residual_norm(**of(k), parts=True)
        # magnitudes: every term of the formulas in absolute value, a row's mean of products by its size
        a = np.abs
        yv = S.residual_norm(**of(k))[0]
        size_y = a(sc * o) + (a(r.values[k]) if r else 0)
        yhat = a(size_y * rinv)
        e = a(dh.values[k]) * (1 if nw is None else nw) if dh else 0 * yv
        size_r = (a(dy.values[k]) if dy else 0) + a(rinv) * (e * (1 + yhat.max(-1, keepdims=True)) + yhat * ((e * yhat).mean(
            -1, keepdims=True) + 1e-30) * (1 + yhat.max(-1, keepdims=True))) + 0 * yv
        gate_size = a(sg) if gate else 1.0
        do = size_r * a(sc)
        dv = do if gate_first else do * gate_size
        wv = 1 if w is None else w
        if w is not None:
            e3 = (dv * wv).reshape(len(dv), groups, chan // groups)
            h3 = a(hat).reshape(len(dv), groups, chan // groups)
            du = a(inv) * (e3 + h3 * (e3 * h3).mean(-1, keepdims=True)).reshape(dv.shape)
        else:
            du = dv
        sizes = dict(dx=du * gate_size if gate_first else du, dresidual=size_r, dweight=(dv * a(hat)).sum(0),
                     dscale=(size_r * a(o)).sum(0))
        if dh:
            sizes["dnorm_weight"] = (a(dh.values[k]) * yhat * (1 + yhat.max(-1, keepdims=True))).sum(0)
        close(dx.get()[k], want["dx"], sizes["dx"], 2 * chain, dtype, "dx")
        if residual:
            close(dr.get()[k], want["dresidual"], sizes["dresidual"], 2 * chain, dtype, "dresidual")
        if gate:
            slope = S.silu_slope(g.values[k], True)
            close(dg.get()[k], want["dgate"], (du * a(x.values[k]) if gate_first else do * a(hat) * wv) * slope, 2 * chain,
                  dtype, "dgate")
        for name in sums:
            if name in want:
                sums[name][0] += want[name]
                sums[name][1] += sizes[name]
    for name, dev_ in grads.items():
        if dev_ is not None:
            close(dev_.get(), sums[name][0], sums[name][1], 2 * chain + sum(lengths), F32, name)


@DTYPES
@pytest.mark.parametrize("eps", [0.0, 1e-42, 0.1])
@pytest.mark.parametrize("gate_first", [True, False])
@pytest.mark.parametrize("chan,groups", [(1000, 5), (1000, 1), (80, 5), (160, 5), (40, 1), (35, 7), (35, 1), (1280, 5),
                                         (8200, 5), (8200, 1)])
def test_norm_eps(queue, rng, monkeypatch, dtype, eps, gate_first, chan, groups):
    """Other eps than the usual one, zero among them (1e-42 is below float32's normal numbers), with rows that
    do not fill their block of threads: the threads past the end add nothing."""
    for f in (seq.plan_residual_norm, S.residual_norm, S.residual_norm_grad):
        monkeypatch.setattr(f, "__defaults__", tuple(eps if d == 1e-5 else d for d in f.__defaults__))
    test_residual_norm(queue, rng, dtype, [3, 0, 2], chan, groups, 0, 0, True, gate_first, True, True, True, True, True, True)


@DTYPES
@pytest.mark.parametrize("chan,groups,pad,lead,gate,gate_first,Y,H", [
    (64, 8, 0, 0, True, True, True, True), (80, 5, 0, 0, True, False, True, True), (136, 1, 8, 8, True, True, True, True),
    (1280, 5, 0, 0, True, True, True, True), (1280, 5, 0, 0, False, True, True, False), (1000, 5, 0, 0, True, False, True, True),
    (1000, 5, 0, 0, True, True, True, False), (1000, 1, 0, 0, True, True, True, False), (33, 3, 1, 1, True, True, False, True),
    (201, 67, 0, 0, True, False, True, True), (201, 67, 0, 0, True, False, True, False)])
def test_norm_of_many_rows(queue, rng, monkeypatch, dtype, chan, groups, pad, lead, gate, gate_first, Y, H):
    """Several rows to a block, as large batches have them: rows on their way in a ring, sums' buffers in turn, gradients
    summed over the block's rows."""
    recorded = [_recorded(monkeypatch, "plan_residual_norm"), _recorded(monkeypatch, "plan_residual_norm_grad")]
    test_residual_norm(queue, rng, dtype, [1301, 0, 300], chan, groups, pad, lead, gate, gate_first, True, True, True, True, Y, H)
    assert [p[0].full_args[0].unit_rows for p in recorded] == [6, 11]


@DTYPES
@pytest.mark.parametrize("chan,groups,gate_first", [(3000, 5, True), (6000, 1, False), (9001, 1, True), (12000, 125, False),
                                                    (20000, 4, True), (32768, 1, True)])
def test_wide_norm_of_many_rows(queue, rng, monkeypatch, dtype, chan, groups, gate_first):
    """The same with several vectors to a thread; above 16384 channels (16 bits: 8192) the gradients are summed in memory."""
    recorded = [_recorded(monkeypatch, "plan_residual_norm"), _recorded(monkeypatch, "plan_residual_norm_grad")]
    test_residual_norm(queue, rng, dtype, [150, 0, 147], chan, groups, 0, 0, True, gate_first, True, True, True, True, True, True)
    assert [p[0].full_args[0].unit_rows for p in recorded] == [2, 3]


def test_norm_infinite_weight_stays_in_its_channel(queue, rng):
    """The last channel's infinite weight: the row's norm is infinite, so every other h is zero, none is NaN."""
    chan = 1000
    x, h = Rows(queue, [normal(rng, 2, chan)], F32), Rows(queue, [np.zeros((2, chan))], F32, empty=True)
    w = np.ones(chan, np.float32)
    w[-1] = np.inf
    seq.plan_residual_norm(queue, x.ra, H=h.ra, weight=vec(queue, w), groups=5)()
    got = h.get()[0]
    assert (got[:, :-1] == 0).all() and np.isnan(got[:, -1]).all()


def test_norm_of_zero_rows_and_infinities(queue, rng):
    x = np.zeros((3, 40), np.float32)
    x[1, 3] = np.inf
    x[2] = normal(rng, 40)
    X, H = Rows(queue, [x], F32), Rows(queue, [x], F32, empty=True)
    seq.plan_residual_norm(queue, X.ra, H=H.ra)()
    got = H.buf.get()[:120].reshape(3, 40)
    assert (got[0] == 0).all() and np.isnan(got[1, 3]) and (got[1, :3] == 0).all()
    close(got[2:], S.residual_norm(x[2:].astype(float))[1], np.abs(x[2:]) * 2, 64, F32)


# ---- placement, streams, graphs ------------------------------------------------------------------
def test_offsets_past_32_bits(queue, rng):
    """Rows 2^30 elements apart in a 2^31-element buffer: byte and element offsets pass 2^31 and 2^32."""
    chan, rows, pitch = 24, 3, 2 ** 30 + 8
    size = 2 * pitch + chan
    x, y = DeviceArray(queue, (size,), BF16), DeviceArray(queue, (size,), BF16)
    ra = lambda buf: CUDARaggedArray.from_buffer(queue, buf, [0], [rows], [chan], [pitch], [1])
    values = as_dtype(normal(rng, rows, chan), BF16)
    for r in range(rows):
        x.write_region(r * pitch, values[r])
    w = normal(rng, chan, 2)
    seq.plan_causal_conv(queue, ra(x), vec(queue, w), ra(y))()
    want, _ = S.causal_conv(widen(values), w)
    mag, _ = S.causal_conv(widen(values), w, magnitude=True)
    close([widen(y.read_region(r * pitch, chan)) for r in range(rows)], want, mag, 4, BF16)
    seq.plan_residual_norm(queue, ra(x), H=ra(y))()
    want = S.residual_norm(widen(values))[1]
    close([widen(y.read_region(r * pitch, chan)) for r in range(rows)], want, 2 * np.abs(want), 64, BF16)
    short = Rows(queue, [normal(rng, rows, 8)], BF16)
    A = -np.ones((chan, 8), np.float32)
    dt = Rows(queue, [np.full((rows, chan), 0.25)], BF16)
    seq.plan_selective_scan(queue, ra(x), dt.ra, vec(queue, A), short.ra, short.ra, ra(y))()
    args = (widen(values), dt.values[0], A, short.values[0], short.values[0])
    want, mag = S.selective_scan(*args)[0], S.selective_scan(*args, magnitude=True)[0]
    close([widen(y.read_region(r * pitch, chan)) for r in range(rows)], want, mag, 60, BF16)


def test_starts_past_32_bits(queue, rng):
    """Items that begin 2^32 + 64 elements into their buffer, inputs and outputs, beside one at the front."""
    chan, rows, far = 24, 5, 2 ** 32 + 64
    starts = np.array([64, far])
    x, y = (DeviceArray(queue, (far + 4096,), BF16) for _ in range(2))
    ra = lambda buf, n=rows, c=chan, at=starts: CUDARaggedArray.from_buffer(queue, buf, at, [n] * 2, [c] * 2, [c] * 2, [1] * 2)
    data = [as_dtype(normal(rng, rows, chan), BF16) for _ in starts]
    for v, s in zip(data, starts):
        x.write_region(s, v.ravel())
    got = lambda: [widen(y.read_region(s, rows * chan).reshape(rows, chan)) for s in starts]
    w = normal(rng, chan, 4)
    seq.plan_causal_conv(queue, ra(x), vec(queue, w), ra(y))()
    for v, g in zip(data, got()):
        mag = S.causal_conv(widen(v), w, magnitude=True)[0]
        close(g, S.causal_conv(widen(v), w)[0], mag, 6, BF16, "convolution")
    seq.plan_residual_norm(queue, ra(x), H=ra(y))()
    for v, g in zip(data, got()):
        want = S.residual_norm(widen(v))[1]
        close(g, want, 2 * np.abs(want), 64, BF16, "norm")
    n, A = 8, -np.ones((chan, 8), np.float32)
    pool = DeviceArray(queue, (far + 4096,), F32)
    states = [normal(rng, chan, n) for _ in starts]
    at = starts[::-1]  # (the first sequence's state far away)
    for v, s in zip(states, at):
        pool.write_region(s, v.ravel())
    both = ra(pool, chan, n, at)
    dt, short = Rows(queue, [np.full((rows, chan), 0.25)] * 2, BF16), Rows(queue, [normal(rng, rows, n)] * 2, BF16)
    seq.plan_selective_scan(queue, ra(x), dt.ra, vec(queue, A), short.ra, short.ra, ra(y), state=both, new_state=both)()
    for k, g in enumerate(got()):
        args = (widen(data[k]), dt.values[k], A, short.values[k], short.values[k])
        want, end = S.selective_scan(*args, state=states[k])
        mag, mag_end = S.selective_scan(*args, state=states[k], magnitude=True)
        close(g, want, mag, 100, BF16, "scan")
        close(pool.read_region(at[k], chan * n).reshape(chan, n), end, mag_end, 100, F32, "state")


class Block:
    """norm -> convolution -> scan -> gate, norm and residual, as one would run them."""

    def __init__(self, queue, rng, chan=48, n=16, taps=4):
        self.queue, self.chan, self.n, self.taps = queue, chan, n, taps
        p = lambda *s: vec(queue, normal(rng, *s))
        self.pre, self.post, self.scale = p(chan), p(chan), p(chan)
        self.w, self.bias, self.D, self.dt_bias = p(chan, taps), p(chan), p(chan), vec(queue, np.full(chan, -2.0))
        self.A = vec(queue, -rng.uniform(0.5, 4, size=(chan, n)))

    def plans(self, stream, gate, dt, B, C, out, conv_state, scan_state):
        q = self.queue
        rows = [np.zeros((k, self.chan)) for k in stream.ra.shape0s]
        tmp = [Rows(q, rows, F32, empty=True, columns=self.chan) for _ in range(3)]
        return [seq.plan_residual_norm(q, stream.ra, H=tmp[0].ra, norm_weight=self.pre),
                seq.plan_causal_conv(q, tmp[0].ra, self.w, tmp[1].ra, bias=self.bias, state=conv_state.ra,
                                     new_state=conv_state.ra, activation="silu"),
                seq.plan_selective_scan(q, tmp[1].ra, dt.ra, self.A, B.ra, C.ra, tmp[2].ra, D=self.D, dt_bias=self.dt_bias,
                                        softplus=True, state=scan_state.ra, new_state=scan_state.ra),
                seq.plan_residual_norm(q, tmp[2].ra, Y=out.ra, gate=gate.ra, residual=stream.ra, weight=self.post,
                                       scale=self.scale)]


@pytest.mark.parametrize("graph", [False, True])
def test_prompt_then_tokens_equals_one_pass(queue, rng, graph):
    """A whole pass over the sequences against a prompt followed by single tokens with the carried states,
    launched one by one or replayed from a captured graph."""
    block, lengths, head = Block(queue, rng), [37, 41], [30, 34]
    chan, n = block.chan, block.n
    data = {k: [normal(rng, m, c) for m in lengths] for k, c in
            dict(stream=chan, gate=chan, dt=chan, B=n, C=n).items()}
    states = lambda: (Rows(queue, [np.zeros((block.taps - 1, chan))] * 2, F32), Rows(queue, [np.zeros((chan, n))] * 2, F32))

    def run(pieces, out, st, repeat=1):
        plans = block.plans(*[Rows(queue, v, F32) for v in pieces], out, *st)
        if graph:
            Plans(plans, False).call_n_times(repeat)
        else:
            for p in plans * repeat:
                p.enqueue()
            queue.finish()

    part = lambda lo, hi: [[v[a:b] for v, a, b in zip(data[k], lo, hi)] for k in ("stream", "gate", "dt", "B", "C")]
    whole = Rows(queue, data["stream"], F32, empty=True)
    end = states()
    run(part([0, 0], lengths), whole, end)
    st = states()
    first = Rows(queue, [np.zeros((h, chan)) for h in head], F32, empty=True)
    run(part([0, 0], head), first, st)
    got = [[v] for v in first.get()]
    for t in range(7):
        lo = [h + t for h in head]
        out = Rows(queue, [np.zeros((1, chan))] * 2, F32, empty=True)
        run(part(lo, [v + 1 for v in lo]), out, st)
        for g, v in zip(got, out.get()):
            g.append(v)
    # the same arithmetic row by row, in a different grouping of the rows: as far apart as two roundings
    # of each step can be, 41 rows of a decaying state
    for a, b in zip(whole.get(), got):
        b = np.concatenate(b)
        assert np.allclose(a, b, rtol=2e-5, atol=2e-5 * np.abs(a).max())
    for a, b in zip(end[1].get(), st[1].get()):
        assert np.allclose(a, b, rtol=2e-5, atol=2e-5 * np.abs(a).max())
    for a, b in zip(end[0].get(), st[0].get()):
        assert np.allclose(a, b, rtol=1e-5, atol=1e-5)


def test_graph_replay_steps_the_state(queue, rng):
    """n replays of a captured single-token plan are n launches of it."""
    s = Scan(queue, rng, [1, 1], 40, 16, 1, F32)
    start = s.state.buf.get()
    plan = s.plan(new_state=s.state.ra)
    for _ in range(5):
        plan()
    want = s.state.buf.get(), s.y.buf.get()
    s.state.buf.set(start)
    Plans([plan], False, unroll=2).call_n_times(5)
    assert np.array_equal(s.state.buf.get(), want[0]) and np.array_equal(s.y.buf.get(), want[1])


@pytest.mark.parametrize("lengths", [[300, 1, 0, 1, 40], [200, 180]], ids=str)
def test_split_sequences_in_place_replayed(queue, rng, lengths):
    """A prompt among single tokens, split over time, states in place: replays of a captured graph are launches of it."""
    s = Scan(queue, rng, lengths, 40, 16, 1, BF16)
    start = s.state.buf.get()
    plan = s.plan(new_state=s.state.ra)
    assert plan.full_args[0].n_units > len(lengths) and not plan.full_args[0].tokens
    plan()
    for k, end in enumerate(s.state.get()):
        close(end, S.selective_scan(**s.of(k))[1], S.selective_scan(**s.of(k), magnitude=True)[1], s.chain(k), F32, "state")
    for _ in range(3):
        plan()
    end = s.state.buf.get(), s.y.buf.get()
    s.state.buf.set(start)
    Plans([plan], False, unroll=2).call_n_times(4)
    assert np.array_equal(s.state.buf.get(), end[0]) and np.array_equal(s.y.buf.get(), end[1])


def test_training_pass_in_a_torch_graph(ctx, queue, rng):
    """Forward and backward plans of all three operators captured by torch on its own stream, replayed twice while the
    same plans also ran outside of it."""
    torch = pytest.importorskip("torch")
    side = torch.cuda.Stream()
    q = CommandQueue(ctx, stream=side.cuda_stream)
    lengths, chan = [70, 0, 33], 48
    s = Scan(q, rng, lengths, chan, 16, 2, F32)
    rows = lambda: Rows(q, [normal(rng, k, chan) for k in lengths], F32, columns=chan)
    dy, outs = rows(), [Rows(q, v.values, F32, empty=True, columns=v.place[0][2]) for v in (s.x, s.dt, s.B, s.C)]
    par = lambda *shape: vec(q, np.zeros(shape))
    fwd = s.plan(keep=True)
    plans = [fwd, seq.plan_selective_scan_grad(q, fwd, dy.ra, outs[0].ra, outs[1].ra, par(chan, 16), outs[2].ra, outs[3].ra)]
    conv = seq.plan_causal_conv(q, s.x.ra, vec(q, normal(rng, chan, 4)), rows().ra, activation="silu")
    cdx, cdw = rows(), par(chan, 4)
    plans += [conv, seq.plan_causal_conv_grad(q, conv, dy.ra, cdx.ra, cdw)]
    norm = seq.plan_residual_norm(q, s.x.ra, H=rows().ra, gate=s.z.ra, weight=vec(q, np.ones(chan)), groups=3)
    ndx, ndw = rows(), par(chan)
    plans += [norm, seq.plan_residual_norm_grad(q, norm, ndx.ra, dH=dy.ra, dweight=ndw)]
    results = lambda: [r.buf.get() for r in outs + [s.y, cdx, ndx]] + [cdw.get(), ndw.get()]
    for p in plans:
        p.enqueue()
    want = results()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        for p in plans:
            p.enqueue()
    for r in outs + [s.y, cdx, ndx]:
        r.buf.set(np.full(r.buf.size, -7.5, np.float32))
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert all(np.array_equal(a, b) for a, b in zip(results(), want))
        for p in plans:
            p.enqueue()
        assert all(np.array_equal(a, b) for a, b in zip(results(), want))


def test_training_pass_replayed_and_on_another_stream(ctx, queue, rng):
    s = Scan(queue, rng, [70, 33], 40, 16, 2, F32)
    dy = Rows(queue, [normal(rng, k, 40) for k in s.lengths], F32)
    outs = [Rows(queue, v.values, F32, empty=True) for v in (s.x, s.dt, s.B, s.C)]
    dA = vec(queue, np.zeros(s.A.shape))
    results = []
    torch = pytest.importorskip("torch")
    stream = torch.cuda.Stream()
    for mode in ("enqueue", "graph", "torch"):
        q = CommandQueue(ctx, stream=stream.cuda_stream) if mode == "torch" else queue
        s.queue = q
        fwd = s.plan(keep=True)
        bwd = seq.plan_selective_scan_grad(q, fwd, dy.ra, outs[0].ra, outs[1].ra, dA, outs[2].ra, outs[3].ra)
        if mode == "graph":
            Plans([fwd, bwd], False).call_n_times(2)
        else:
            fwd.enqueue()
            bwd.enqueue()
            q.finish()
        results.append([o.buf.get() for o in outs] + [dA.get()])
        for o in outs:
            o.buf.set(np.full(o.buf.size, -7.5, np.float32))
    for r in results[1:]:
        assert all(np.array_equal(a, b) for a, b in zip(results[0], r))


def test_torch_memory_is_used_in_place(ctx, rng):
    torch = pytest.importorskip("torch")
    q = CommandQueue(ctx, stream=torch.cuda.current_stream().cuda_stream)
    x = torch.randn(6, 40, device="cuda", dtype=torch.bfloat16)
    h = torch.empty_like(x)
    ra = lambda t: CUDARaggedArray.from_buffer(q, DeviceArray(q, t.shape, BF16, data=t.data_ptr(), base=t), [0], [6], [40],
                                               [40], [1])
    seq.plan_residual_norm(q, ra(x), H=ra(h)).enqueue()
    want = S.residual_norm(x.double().cpu().numpy())[1]
    close(h.double().cpu().numpy(), want, 2 * np.abs(want), 64, BF16)


def test_host_memory_is_refused_unless_the_device_reaches_it(ctx, queue, rng):
    torch = pytest.importorskip("torch")
    x = Rows(queue, [normal(rng, 6, 40)], F32)
    host = np.zeros(240, np.float32)
    ra = lambda address, base: CUDARaggedArray.from_buffer(queue, DeviceArray(queue, (240,), F32, data=address, base=base),
                                                           [0], [6], [40], [40], [1])
    with pytest.raises(ValueError, match="host memory"):  # (refused when the plan is built: nothing is launched)
        seq.plan_residual_norm(queue, x.ra, H=ra(host.ctypes.data, host))
    pinned = torch.zeros(240).pin_memory()
    seq.plan_residual_norm(queue, x.ra, H=ra(pinned.data_ptr(), pinned))()
    want = S.residual_norm(x.values[0])[1]
    close(pinned.numpy().reshape(6, 40), want, 2 * np.abs(want), 64, F32)
    with torch.cuda.device(0):
        mine = torch.zeros(240, device="cuda")
    seq.plan_residual_norm(queue, x.ra, H=ra(mine.data_ptr(), mine))()
    assert np.array_equal(mine.cpu().numpy(), pinned.numpy())


def test_the_plans_device_must_be_current(queue, rng):
    """A launch whose plan names another device than the current one is refused, not run."""
    from nengo_ocl_b200 import _capi

    s = Scan(queue, rng, [3], 8, 4, 1, F32)
    plan = s.plan()
    args = plan.full_args[0]
    args.device = 1
    with pytest.raises(_capi.NB2Error, match="current CUDA device"):
        plan()
    args.device = 0
    plan()
    s.check()
    assert ctypes.sizeof(args) > 0


# ---- in a simulated model ------------------------------------------------------------------------
def test_simulated_block_matches_the_oracle(ctx):
    from nengo_ocl_b200 import synth
    from nengo_ocl_b200.simulator import Simulator
    from oracle.simulator import OracleSimulator

    mdl = synth.state_space_model()
    ora = OracleSimulator(mdl)
    ora.run_steps(40)
    with Simulator(None, model=mdl, context=ctx) as sim:
        first = None
        for _ in range(2):  # again after a reset: the states start over
            sim.run_steps(40)
            for p in mdl.info["probes"]:
                want = np.array(ora.probe_data[p])
                # values of order one; float32 products over 48 channels and 40 rows of a decaying state
                assert np.allclose(sim.data[p], want, rtol=1e-4, atol=1e-4)
            for pair in mdl.info["states"]:
                for s in pair:
                    assert np.allclose(sim.signals[s], ora[s], rtol=1e-4, atol=1e-4)
            data = [np.array(sim.data[p]) for p in mdl.info["probes"]]
            assert first is None or all(np.array_equal(a, b) for a, b in zip(first, data))
            first = data
            sim.reset()


def test_simulated_scans_of_other_widths(ctx):
    from nengo_ocl_b200.simulator import Simulator
    from oracle.simulator import OracleSimulator
    from test_sequence import two_widths_model

    mdl = two_widths_model()
    ora = OracleSimulator(mdl)
    ora.run_steps(9)
    with Simulator(None, model=mdl, context=ctx) as sim:
        sim.run_steps(9)
        for s in mdl.info["outs"]:
            # (nine rows of a decaying state of order one: 9 (6 + 30 * 4 * 2) + 200 half steps)
            assert np.allclose(sim.signals[s].ravel(), ora[s].ravel(), rtol=2e-4, atol=2e-4)
