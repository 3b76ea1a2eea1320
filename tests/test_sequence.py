"""Sequence operators without a GPU: the 64-bit formulas against differences, bfloat16 storage, and what
the plan functions refuse (with a host-memory stand-in for the library)."""

import ctypes

import numpy as np
import pytest

import fake_library
from nengo_ocl_b200 import _capi
from nengo_ocl_b200 import cura_sequence as seq
from nengo_ocl_b200.curaggedarray import CUDARaggedArray
from nengo_ocl_b200.raggedarray import RaggedArray
from nengo_ocl_b200.runtime import CommandQueue, Context, DeviceArray, to_device
from nengo_ocl_b200.utils import bfloat16, from_bfloat16, to_bfloat16
from oracle import sequences as S


# ---- the formulas' gradients against differences ----------------------------------------------
def _differences(f, args, names, grads, rng, eps=1e-5):
    """Directional derivative of every named argument, central differences."""
    for name in names:
        v = rng.normal(size=np.shape(args[name]))
        up, down = (f(**dict(args, **{name: args[name] + sign * eps * v})) for sign in (1, -1))
        want = (up - down) / (2 * eps)
        got = float((grads["d" + name] * v).sum())
        # central differences: eps^2 times third derivatives (order 10) and rounding of f, 1e-16 |f| / eps
        assert abs(got - want) <= 1e-7 * (1 + abs(want)), name


@pytest.mark.parametrize("silu_", [False, True])
@pytest.mark.parametrize("rows", [0, 1, 2, 9])
def test_conv_gradient_formula(rng, silu_, rows):
    chan, taps = 3, 4
    args = dict(x=rng.normal(size=(rows, chan)), w=rng.normal(size=(chan, taps)), bias=rng.normal(size=chan),
                state=rng.normal(size=(taps - 1, chan)))
    dy, dn = rng.normal(size=(rows, chan)), rng.normal(size=(taps - 1, chan))

    def f(**a):
        y, new = S.causal_conv(silu_=silu_, **a)
        return (y * dy).sum() + (new * dn).sum()

    _differences(f, args, args, S.causal_conv_grad(dy=dy, dnew_state=dn, silu_=silu_, **args), rng)


@pytest.mark.parametrize("softplus", [False, True])
@pytest.mark.parametrize("groups", [1, 2])
def test_scan_gradient_formula(rng, softplus, groups):
    rows, chan, n = 6, 4, 3
    args = dict(x=rng.normal(size=(rows, chan)), dt=rng.uniform(0.1, 0.5, size=(rows, chan)),
                A=-rng.uniform(0.5, 2, size=(chan, n)), B=rng.normal(size=(rows, groups * n)),
                C=rng.normal(size=(rows, groups * n)), D=rng.normal(size=chan), z=rng.normal(size=(rows, chan)),
                dt_bias=rng.uniform(0, 0.2, size=chan), state=rng.normal(size=(chan, n)))
    dy, dn = rng.normal(size=(rows, chan)), rng.normal(size=(chan, n))

    def f(**a):
        y, new = S.selective_scan(softplus=softplus, **a)
        return (y * dy).sum() + (new * dn).sum()

    _differences(f, args, args, S.selective_scan_grad(dy=dy, dnew_state=dn, softplus=softplus, **args), rng)


@pytest.mark.parametrize("gate_first", [False, True])
@pytest.mark.parametrize("groups", [1, 3])
def test_norm_gradient_formula(rng, gate_first, groups):
    rows, chan = 4, 6
    args = dict(x=rng.normal(size=(rows, chan)), gate=rng.normal(size=(rows, chan)),
                residual=rng.normal(size=(rows, chan)), weight=rng.normal(size=chan), scale=rng.normal(size=chan),
                norm_weight=rng.normal(size=chan))
    dy, dh = rng.normal(size=(rows, chan)), rng.normal(size=(rows, chan))

    def f(**a):
        y, h = S.residual_norm(gate_first=gate_first, groups=groups, **a)
        return (y * dy).sum() + (h * dh).sum()

    _differences(f, args, args, S.residual_norm_grad(dy=dy, dh=dh, gate_first=gate_first, groups=groups, **args), rng)


# ---- bfloat16 ----------------------------------------------------------------------------------
def test_bfloat16_round_to_nearest_even(rng):
    torch = pytest.importorskip("torch")
    v = np.concatenate([rng.normal(size=1000) * 10.0 ** rng.randint(-38, 38, size=1000),
                        [0.0, -0.0, np.inf, -np.inf, 1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8, 3.4e38]]).astype(np.float32)
    want = torch.from_numpy(v).to(torch.bfloat16)
    got = to_bfloat16(v)
    assert np.array_equal(got.view(np.uint16), want.view(torch.uint16).numpy())
    assert np.array_equal(from_bfloat16(got), want.float().numpy())
    assert np.isnan(from_bfloat16(to_bfloat16(np.float32([np.nan, -np.nan])))).all()
    assert np.array_equal(to_bfloat16(got), got) and from_bfloat16(got.reshape(-1, 1)).shape == (len(v), 1)


def test_ragged_arrays_of_16_bit_types(rng, fake_queue):
    values = [rng.normal(size=(3, 4)), rng.normal(size=(2, 5))]
    for dtype in (np.float16, bfloat16):
        ra = RaggedArray(values, dtype=dtype)
        clra = CUDARaggedArray(fake_queue, ra)
        assert clra.dtype == dtype and clra.ctype == ("half" if dtype == np.float16 else "bfloat16")
        for i, v in enumerate(values):
            want = to_bfloat16(v) if dtype == bfloat16 else v.astype(dtype)
            assert np.array_equal(ra[i], want) and np.array_equal(clra[i], want)
        clra[1] = 2.0
        clra[0] = values[0][::-1]
        two = to_bfloat16(np.float32(2)) if dtype == bfloat16 else np.float16(2)
        assert (clra[1] == two).all() and np.array_equal(clra[0], ra[0][::-1])
    with pytest.raises(AssertionError):
        RaggedArray(values, dtype=np.float64)


def test_values_cross_between_bfloat16_and_other_types(rng, fake_queue):
    """Host values go into an array of another type as values, not as the integers that bfloat16 is stored as."""
    v = rng.normal(size=(3, 4)).astype(np.float32)
    short = to_bfloat16(v)
    into = {np.dtype(np.float32): from_bfloat16(short), np.dtype(np.float16): from_bfloat16(short).astype(np.float16),
            bfloat16: short}
    for dtype, want in into.items():
        two = to_bfloat16(np.float32(2)) if dtype == bfloat16 else dtype.type(2)
        for source in (v, v.astype(np.float64)) if dtype == bfloat16 else (short,):
            d = DeviceArray(fake_queue, (3, 4), dtype)
            d.set(source)
            assert np.array_equal(d.get(), want)
            d.fill(2.0)
            assert (d.get() == two).all()
            d.write_region(4, source[0])
            assert np.array_equal(d.get()[1], want[0]) and (d.get()[0] == two).all()
            ra = RaggedArray([source, source[:2]], dtype=dtype)
            assert np.array_equal(ra[0], want) and np.array_equal(ra[1], want[:2])
            ra[1] = 2.0
            assert (ra[1] == two).all()
            ra[1] = source[1:]
            assert np.array_equal(ra[1], want[1:])
            clra = CUDARaggedArray(fake_queue, ra)
            clra[1] = 2.0
            assert (clra[1] == two).all()
            clra[1] = source[:2]
            assert np.array_equal(clra[1], want[:2])
            turned = CUDARaggedArray.from_buffer(fake_queue, clra.cl_buf, [0], [2], [3], [4], [1])
            turned[0] = source[:2, :3]
            assert np.array_equal(turned[0], want[:2, :3])
        d.fill(to_bfloat16(np.float32(2)))
        assert (d.get() == two).all()
        d.fill(to_bfloat16(np.float32(0)))
        assert not d.get().view(np.uint8).any()


# ---- which rows share memory -------------------------------------------------------------------
def test_shared_bytes_against_enumeration(rng):
    def cells(low, rows, pitch, width):
        return {low + r * pitch + b for r in range(rows) for b in range(width)}

    def memory(entries):
        return seq._Memory("m", *(np.array(v, np.int64) for v in zip(*entries)), True)

    seen = [0, 0]
    for _ in range(3000):
        pitch = int(rng.randint(1, 9))
        a, b = ((int(rng.randint(0, 40)), int(rng.randint(0, 5)), pitch if rng.rand() < 0.9 else int(rng.randint(0, 9)),
                 int(rng.randint(0, 9))) for _ in range(2))
        want = bool(cells(*a) & cells(*b))
        got = len(memory([a]).pairs(memory([b]))) > 0
        exact = a[2] == b[2] and a[2] > 0 or a[1] == 1 and b[2] > 0 or b[1] == 1 and a[2] > 0
        assert got == want if exact else got >= want, (a, b)
        seen[want] += 1
        both = memory([a, b]).repeats()
        if want or any(v[1] > 1 and v[2] < v[3] for v in (a, b)):
            assert both or not (a[1] and a[3] and b[1] and b[3])
    assert min(seen) > 300


# ---- refusals ----------------------------------------------------------------------------------
@pytest.fixture
def fake_queue(monkeypatch):
    fake_library.install(monkeypatch)
    return CommandQueue(Context(0))


def _rows(queue, lengths, columns, dtype=np.float32):
    n = np.asarray(lengths)
    buf = DeviceArray(queue, max(1, int(n.sum()) * columns), dtype)
    wide = np.full(len(n), columns)
    return CUDARaggedArray.from_buffer(queue, buf, (np.cumsum(n) - n) * columns, n, wide, wide, np.ones(len(n), int))


def _again(ra, **changes):
    fields = dict(starts=ra.starts, shape0s=ra.shape0s, shape1s=ra.shape1s, stride0s=ra.stride0s, stride1s=ra.stride1s)
    fields.update(changes)
    return CUDARaggedArray.from_buffer(ra.queue, ra.cl_buf, **fields)


class Case:
    """A well-formed set of arguments; tests change one."""

    def __init__(self, q, lengths=(5, 0, 3), chan=8, dtype=np.float32):
        rows = lambda c=chan, d=dtype: _rows(q, lengths, c, d)
        vec = lambda *shape: DeviceArray(q, shape or (chan,), np.float32)
        k = len(lengths)
        self.q = q
        self.conv = dict(X=rows(), W=vec(chan, 4), Y=rows(), bias=vec(), state=_rows(q, [3] * k, chan, dtype),
                         new_state=_rows(q, [3] * k, chan, dtype), activation="silu")
        self.scan = dict(X=rows(), dt=rows(), A=vec(chan, 4), B=rows(8), C=rows(8), Y=rows(), D=vec(), Z=rows(),
                         dt_bias=vec(), softplus=True, state=_rows(q, [chan] * k, 4), new_state=_rows(q, [chan] * k, 4),
                         keep=True)
        self.norm = dict(X=rows(), Y=rows(), H=rows(), gate=rows(), residual=rows(), weight=vec(), scale=vec(),
                         norm_weight=vec(), groups=2)
        self.conv_grad = dict(dY=rows(), dX=rows(), dW=vec(chan, 4), dbias=vec(), dstate=_rows(q, [3] * k, chan, dtype),
                              dnew_state=_rows(q, [3] * k, chan, dtype))
        self.scan_grad = dict(dY=rows(), dX=rows(), ddt=rows(), dA=vec(chan, 4), dB=rows(8), dC=rows(8), dD=vec(),
                              dZ=rows(), ddt_bias=vec(), dstate=_rows(q, [chan] * k, 4),
                              dnew_state=_rows(q, [chan] * k, 4))
        self.norm_grad = dict(dX=rows(), dY=rows(), dH=rows(), dgate=rows(), dresidual=rows(), dweight=vec(),
                              dscale=vec(), dnorm_weight=vec())

    def forward(self, kind, **changes):
        f = dict(conv=seq.plan_causal_conv, scan=seq.plan_selective_scan, norm=seq.plan_residual_norm)[kind]
        return f(self.q, **dict(getattr(self, kind), **changes))

    def backward(self, kind, forward=None, **changes):
        f = dict(conv=seq.plan_causal_conv_grad, scan=seq.plan_selective_scan_grad,
                 norm=seq.plan_residual_norm_grad)[kind]
        return f(self.q, forward or self.forward(kind), **dict(getattr(self, kind + "_grad"), **changes))


@pytest.mark.parametrize("dtype", [np.float32, np.float16, bfloat16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("kind", ["conv", "scan", "norm"])
def test_well_formed_plans_are_built(fake_queue, kind, dtype):
    case = Case(fake_queue, dtype=dtype)
    fwd = case.forward(kind)
    bwd = case.backward(kind, fwd)
    assert fwd.bw_per_call > 0 and fwd.flops_per_call > 0 and bwd.bw_per_call > 0
    fwd.enqueue()
    bwd.enqueue()
    names = [n for n, _ in _capi.lib().calls]
    assert names[-1].endswith("_grad") and names[-1].startswith(names[-2])


@pytest.mark.parametrize("kind", ["conv", "scan", "norm"])
def test_empty_batches_are_planned(fake_queue, kind):
    case = Case(fake_queue, lengths=(0, 0))
    case.backward(kind)


@pytest.mark.parametrize("kind", ["conv", "scan", "norm"])
def test_wrong_sequence_arrays_are_refused(fake_queue, kind):
    q = fake_queue
    case = Case(q)
    for name in [k for k, v in getattr(case, kind).items() if isinstance(v, CUDARaggedArray) and "state" not in k]:
        good = getattr(case, kind)[name]
        cols = int(good.shape1s[0])
        bad = [(ValueError, _rows(q, [5, 3], cols)), (ValueError, _rows(q, [5, 0, 4], cols)),
               (ValueError, _rows(q, [5, 0, 3], cols + 3)), (ValueError, good.cl_buf),
               (ValueError, _again(good, starts=good.starts + 1)),
               (NotImplementedError, _again(good, stride1s=[2, 2, 2], starts=[0, 0, 0])),
               (NotImplementedError, _again(good, stride0s=[-cols] * 3, starts=[4 * cols, 0, 2 * cols]))]
        if name != "X":
            bad.append((ValueError, _rows(q, [5, 0, 3], cols, np.float16)))
        else:
            bad.append(((ValueError, NotImplementedError), _rows(q, [5, 0, 3], cols, np.int32)))
        for error, value in bad:
            with pytest.raises(error):
                case.forward(kind, **{name: value})


@pytest.mark.parametrize("kind", ["conv", "scan", "norm"])
def test_wrong_parameters_are_refused(fake_queue, kind):
    q = fake_queue
    case = Case(q)
    for name in [k for k, v in getattr(case, kind).items() if isinstance(v, DeviceArray)]:
        good = getattr(case, kind)[name]
        slanted = DeviceArray(q, good.shape, np.float32)
        slanted.strides = tuple(4 * s for s in ((1, good.shape[0]) if len(good.shape) == 2 else (2,)))
        for error, value in [(ValueError, DeviceArray(q, tuple(n + 1 for n in good.shape), np.float32)),
                             (ValueError, DeviceArray(q, good.shape, np.float16)),
                             (ValueError, np.zeros(good.shape, np.float32)), (NotImplementedError, slanted)]:
            with pytest.raises(error):
                case.forward(kind, **{name: value})


def test_sizes_out_of_range_are_refused(fake_queue):
    q = fake_queue
    case = Case(q)
    with pytest.raises(NotImplementedError, match="taps"):
        case.forward("conv", W=DeviceArray(q, (8, 9), np.float32))
    with pytest.raises(NotImplementedError, match="activation"):
        case.forward("conv", activation="relu")
    with pytest.raises(NotImplementedError, match="states"):
        case.forward("scan", A=DeviceArray(q, (8, 129), np.float32), B=_rows(q, [5, 0, 3], 129), C=_rows(q, [5, 0, 3], 129))
    with pytest.raises(ValueError, match="multiple"):
        case.forward("scan", B=_rows(q, [5, 0, 3], 6))
    with pytest.raises(ValueError, match="multiple"):
        case.forward("scan", B=_rows(q, [5, 0, 3], 12), C=_rows(q, [5, 0, 3], 12))
    with pytest.raises(ValueError, match="groups"):
        case.forward("norm", groups=3)
    with pytest.raises(ValueError, match="groups"):
        case.forward("norm", weight=None)
    with pytest.raises(ValueError, match="eps"):
        case.forward("norm", eps=-1.0)
    with pytest.raises(ValueError, match="neither"):
        case.forward("norm", Y=None, H=None)
    with pytest.raises(ValueError, match="norm_weight"):
        case.forward("norm", H=None)
    wide = Case(q, lengths=(1,), chan=40000)
    with pytest.raises(NotImplementedError, match="channels"):
        wide.forward("norm")


def test_arrays_without_columns_are_refused(fake_queue):
    q = fake_queue
    case = Case(q)
    with pytest.raises(ValueError, match="multiple"):
        case.forward("scan", B=_rows(q, [5, 0, 3], 0), C=_rows(q, [5, 0, 3], 0))
    empty = Case(q, chan=0)
    for kind in ("conv", "scan", "norm"):
        with pytest.raises(ValueError, match="no channels"):
            empty.forward(kind)


def test_overlapping_outputs_are_refused(fake_queue):
    case = Case(fake_queue)
    for kind, outs in (("conv", ["Y", "new_state"]), ("scan", ["Y", "new_state"]), ("norm", ["Y", "H"])):
        args = getattr(case, kind)
        for out in outs:
            for other, value in args.items():
                if isinstance(value, CUDARaggedArray) and other != out and (value.shape0s == args[out].shape0s).all() \
                        and (out, other) != ("new_state", "state"):
                    with pytest.raises(ValueError, match="overlap"):
                        case.forward(kind, **{out: value})
    # gradients too
    with pytest.raises(ValueError, match="overlap"):
        case.backward("scan", ddt=case.scan_grad["dX"])
    with pytest.raises(ValueError, match="overlap"):
        case.backward("norm", dX=case.norm_grad["dH"])
    with pytest.raises(ValueError, match="overlap"):
        case.backward("conv", dX=case.conv["X"])
    with pytest.raises(ValueError, match="overlap"):
        case.backward("norm", dscale=case.norm_grad["dweight"])
    with pytest.raises(ValueError, match="overlap"):
        case.backward("norm", dweight=case.norm["weight"])


def test_states_in_place_and_repeated_items(fake_queue):
    case = Case(fake_queue)
    for kind in ("conv", "scan"):
        pool = getattr(case, kind)["state"]
        case.forward(kind, state=pool, new_state=pool)                      # in place
        case.forward(kind, state=pool[[2, 0, 1]], new_state=pool[[2, 0, 1]])  # gathered from a pool
        case.forward(kind, state=pool[[1, 1, 1]])                           # all from the same start
        with pytest.raises(ValueError, match="overlap"):
            case.forward(kind, state=pool, new_state=pool[[0, 0, 2]])
        with pytest.raises(ValueError, match="overlap"):
            case.forward(kind, state=pool, new_state=pool[[1, 2, 0]])       # another sequence's old state
        with pytest.raises(ValueError, match="overlap"):
            case.forward(kind, state=pool[[0, 0, 0]], new_state=pool)


def test_column_ranges_of_one_buffer_are_accepted(fake_queue):
    q = fake_queue
    case = Case(q)
    both = _rows(q, [5, 0, 3], 16)
    left = _again(both, shape1s=[8] * 3)
    right = _again(both, shape1s=[8] * 3, starts=both.starts + 8)
    case.forward("norm", Y=left, H=right)
    case.backward("scan", dX=left, ddt=right)
    with pytest.raises(ValueError, match="overlap"):
        case.forward("norm", Y=left, H=_again(both, shape1s=[8] * 3, starts=both.starts + 7))


def test_bytes_of_a_call_count_its_scratch(fake_queue):
    """40 rows of 8 channels x 4 states: 8 float32 vectors, 3 states kept, one channel tile's share of dB and dC."""
    case = Case(fake_queue, lengths=(40,))
    rows, state, params = 4 * 40 * 8, 4 * 8 * 4, 4 * (8 * 4 + 8 + 8)
    fwd = case.forward("scan")
    assert fwd.bw_per_call == 6 * rows + 2 * state + params + 3 * state   # (X, dt, B, C, Y, Z)
    bwd = case.backward("scan", fwd)
    units = 2 * (state + 2 * 4 * 8) * bwd.full_args[0].n_units           # shares of dA, dD and ddt_bias
    assert bwd.full_args[0].n_units == 1
    assert bwd.bw_per_call == 11 * rows + 2 * state + 2 * params + 3 * state + 2 * (4 * 40 * 2 * 8) + units
    fwd = case.forward("conv")
    assert fwd.bw_per_call == 2 * rows + 2 * 4 * 3 * 8 + 4 * 8 * 5
    bwd = case.backward("conv", fwd)
    assert bwd.bw_per_call == 3 * rows + 3 * 4 * 3 * 8 + 2 * 4 * 8 * 5 + 2 * 4 * 8 * 5 * bwd.full_args[0].n_units


def test_gradients_without_their_argument_are_refused(fake_queue):
    case = Case(fake_queue)
    for kind, name, grad in (("conv", "bias", "dbias"), ("conv", "state", "dstate"), ("scan", "D", "dD"),
                             ("scan", "Z", "dZ"), ("scan", "dt_bias", "ddt_bias"), ("scan", "state", "dstate"),
                             ("norm", "gate", "dgate"), ("norm", "residual", "dresidual"),
                             ("norm", "norm_weight", "dnorm_weight")):
        fwd = case.forward(kind, **{name: None})
        with pytest.raises(ValueError, match=grad):
            case.backward(kind, fwd)
        case.backward(kind, fwd, **{grad: None})
    with pytest.raises(ValueError, match="keep"):
        case.backward("scan", case.forward("scan", keep=False))
    with pytest.raises(ValueError, match="dscale"):
        case.backward("norm", case.forward("norm", scale=0.5))
    with pytest.raises(ValueError, match="overwrites"):
        case.backward("conv", case.forward("conv", new_state=case.conv["state"]))
    with pytest.raises(ValueError, match="neither"):
        case.backward("norm", dY=None, dH=None)


def test_c_entries_refuse_bad_arguments():
    """Checked before any CUDA call, so it needs no GPU."""
    lib = _capi.lib()
    for name in ("causal_conv", "causal_conv_grad", "selective_scan", "selective_scan_grad", "residual_norm",
                 "residual_norm_grad"):
        fn, struct = getattr(lib, "nb2_" + name), getattr(_capi, "nb2_%s_args" % name)
        assert fn(None, None) == -2
        assert fn(None, ctypes.byref(struct())) == -2 and b"null pointer" in lib.nb2_last_error()
        args = struct()
        for field, kind in struct._fields_:
            if kind is ctypes.c_void_p:
                setattr(args, field, 256)
        args.dtype = 3
        assert fn(None, ctypes.byref(args)) == -2 and b"dtype" in lib.nb2_last_error()
        args.dtype = 0
        assert fn(None, ctypes.byref(args)) == -2 and b"shape" in lib.nb2_last_error()


def test_limits_agree_with_the_header():
    c = _capi.header_constants("NB2_")
    assert (seq.MAX_TAPS, seq.MAX_STATES, seq.KEEP_ROWS, seq.MAX_NORM_CHANNELS) == (
        c["NB2_CONV_MAX_TAPS"], c["NB2_SCAN_MAX_STATES"], c["NB2_SCAN_KEEP"], c["NB2_NORM_MAX_CHANNELS"])
    assert list(seq._DTYPES.values()) == [c["NB2_F32"], c["NB2_F16"], c["NB2_BF16"]]
    for n in range(1, seq.MAX_STATES + 1):
        for backward in (0, 1):
            assert _capi.lib().nb2_selective_scan_tile(n, backward) == seq.scan_tile(n, bool(backward))
    assert _capi.lib().nb2_selective_scan_tile(0, 0) == -2


def test_queue_over_an_existing_stream(fake_queue):
    q = CommandQueue(fake_queue.context, stream=0)
    assert q.stream == 0
    x = to_device(q, np.arange(4, dtype=np.float32))
    assert np.array_equal(x.get(), np.arange(4))


# ---- in a simulated model ------------------------------------------------------------------------
def test_model_operators_are_planned_once_per_parameter_set(monkeypatch):
    from nengo_ocl_b200 import runtime, synth
    from nengo_ocl_b200 import simulator as sim_mod

    fake_library.install(monkeypatch)
    monkeypatch.setattr(sim_mod.Simulator, "some_context", None)
    monkeypatch.setattr(runtime, "_default_context", None, raising=False)
    sim = sim_mod.Simulator(None, model=synth.state_space_model(n_streams=3))
    names = [p.name for p in sim._plans]
    assert names.count("cura_causal_conv") == names.count("cura_selective_scan") == 1
    assert names.count("cura_residual_norm") == 2  # before and after the block
    ours = ("cura_residual_norm", "cura_causal_conv", "cura_selective_scan")
    order = [n for n in names if n in ours]
    assert order == ["cura_residual_norm", "cura_causal_conv", "cura_selective_scan", "cura_residual_norm"]
    for p in sim._plans:
        if p.name in ours:
            assert len(p.sequence_args["X"]) == 3 and (p.sequence_args["X"].shape0s == 1).all()
            assert p.signal_use is not None
    sim.close()


def two_widths_model(channels=8, n_states=4):
    """Scans that share A, D and dt_bias, with B and C for one group of channels and for two."""
    from nengo_ocl_b200 import model as m

    rng = np.random.RandomState(3)
    mdl = m.Model(dt=0.001)
    const = lambda name, v: m.Signal(v, name=name, readonly=True)
    A, D = const("A", -rng.uniform(0.5, 4, size=(channels, n_states))), const("D", rng.normal(size=channels))
    bias = const("dt_bias", rng.uniform(-2, 0, size=channels))
    outs = []
    for k, groups in enumerate((1, 2, 1)):
        row = lambda name, n: m.Signal(rng.normal(size=n), name="%s%d" % (name, k))
        x, dt, B, C = row("x", channels), row("dt", channels), row("B", groups * n_states), row("C", groups * n_states)
        y, state = m.Signal(np.zeros(channels), name="y%d" % k), m.Signal(np.zeros((channels, n_states)), name="s%d" % k)
        mdl.add_op(m.SimSelectiveScan(x, dt, A, B, C, y, state, D=D, dt_bias=bias))
        outs += [y, state]
    mdl.info = dict(outs=outs)
    return mdl


def test_model_scans_of_other_widths_are_planned_apart(monkeypatch):
    from nengo_ocl_b200 import runtime
    from nengo_ocl_b200 import simulator as sim_mod

    fake_library.install(monkeypatch)
    monkeypatch.setattr(sim_mod.Simulator, "some_context", None)
    monkeypatch.setattr(runtime, "_default_context", None, raising=False)
    sim = sim_mod.Simulator(None, model=two_widths_model())
    plans = [p for p in sim._plans if p.name == "cura_selective_scan"]
    assert sorted(len(p.sequence_args["X"]) for p in plans) == [1, 2]
    assert sorted(p.sequence_args["groups"] for p in plans) == [1, 2]
    sim.close()


def test_oracle_steps_equal_whole_sequences():
    """The operator-list interpreter's step-by-step block against one pass over all rows."""
    from nengo_ocl_b200 import synth
    from oracle.simulator import OracleSimulator

    mdl = synth.state_space_model(n_streams=1)
    ora = OracleSimulator(mdl)
    conv_state, state = mdl.info["states"][0]
    by_name = {s.name: s for op in mdl.operators for s in op.all_signals}
    rows = {n: [] for n in ("normed0", "conv0", "dt0", "B0", "C0", "scanned0")}
    for _ in range(12):
        ora.step()
        for n, v in rows.items():
            v.append(ora[by_name[n]].reshape(-1))
    rows = {n: np.array(v) for n, v in rows.items()}
    get = lambda n: ora[by_name[n]].astype(float)
    y, end = S.causal_conv(rows["normed0"], get("conv_w"), get("conv_b"), None, True)
    assert np.allclose(y, rows["conv0"], rtol=1e-6, atol=1e-6) and np.array_equal(end, ora[conv_state])
    y, end = S.selective_scan(rows["conv0"], rows["dt0"], get("A"), rows["B0"], rows["C0"], get("D"), None, get("dt_bias"), True)
    # (the state is rounded to float32 after every step: 12 half steps)
    assert np.allclose(y, rows["scanned0"], rtol=1e-5, atol=1e-5) and np.allclose(end, ora[state], rtol=1e-5, atol=1e-6)


# ---- places past 2^31 elements -------------------------------------------------------------------
def _table(plan, args=None):
    """The launch's table [fields][sequences] as it was uploaded (the stand-in's memory is the host's)."""
    args = args or plan.full_args[0]
    fields = {"nb2_causal_conv_args": 9, "nb2_residual_norm_args": 11, "nb2_selective_scan_args": 19}[type(args).__name__]
    words = ctypes.cast(args.table, ctypes.POINTER(ctypes.c_int64))
    return np.array([words[i] for i in range(fields * args.n_seq)]).reshape(fields, args.n_seq)


def _far(queue, starts, rows, columns, pitch, size=2 ** 35, address=1 << 40, dtype=np.float32):
    """Items of a buffer that is nowhere (nothing is launched): only its address and size are used."""
    k = len(starts)
    return CUDARaggedArray.from_buffer(queue, DeviceArray(queue, (size,), dtype, data=address), starts, [rows] * k,
                                       [columns] * k, [pitch] * k, [1] * k)


@pytest.mark.parametrize("start", [2 ** 31, 2 ** 31 + 8, 2 ** 32 + 64, 2 ** 33 + 2 ** 31])
@pytest.mark.parametrize("listed", [False, True])
def test_starts_and_strides_past_32_bits_reach_the_launch(fake_queue, start, listed):
    q = fake_queue
    starts = [start, 64]
    x = _far(q, starts if listed else np.array(starts, np.int64), 2, 8, 2 ** 32 + 16)
    y = _far(q, np.array([64, start], np.int64), 2, 8, 2 ** 33 + 16, address=1 << 42)
    pool = _far(q, np.array([start, 2 * start]), 8, 4, 4, address=1 << 43)
    small = _rows(q, [2, 2], 4)
    plan = seq.plan_selective_scan(q, x, _rows(q, [2, 2], 8), DeviceArray(q, (8, 4), np.float32), small, small, y,
                                   state=pool, new_state=pool)
    t = _table(plan)
    assert t[1].tolist() == starts and t[2].tolist() == [2 ** 32 + 16] * 2
    assert t[9].tolist() == [64, start] and t[10].tolist() == [2 ** 33 + 16] * 2
    assert t[13].tolist() == t[15].tolist() == [start, 2 * start]
    assert _table(seq.plan_residual_norm(q, x, H=y))[1].tolist() == starts
    # a selection of items keeps them
    assert _table(seq.plan_residual_norm(q, x[[1, 0]], H=y[[1, 0]]))[1].tolist() == starts[::-1]
    assert len(x) == 2 and x[1:].index64("starts").tolist() == [64]


def test_places_past_32_bits_are_not_handed_to_32_bit_tables(fake_queue):
    """What only takes int32 index tables gets an error, not the place's lower half."""
    x = _far(fake_queue, np.array([2 ** 32 + 64]), 2, 8, 8)
    for name in ("starts", "cl_starts"):
        with pytest.raises(OverflowError, match="starts"):
            getattr(x, name)
    assert x.stride0s.dtype == np.int32 and x.stride0s.tolist() == [8]
    near = _rows(fake_queue, [2], 8)
    again = near[[0]]
    assert again._places("starts") is again._places("starts") and len(again) == 1  # (no copy to look at one item)
    with pytest.raises(ValueError, match="past the end"):
        seq.plan_residual_norm(fake_queue, x, H=_again(_rows(fake_queue, [2], 8), starts=np.array([2 ** 32])))
    with pytest.raises(OverflowError):
        RaggedArray.from_buffer(np.zeros(8, np.float32), np.array([2 ** 32]), [1], [1], [1], [1])
    with pytest.raises(OverflowError):
        RaggedArray.from_buffer(np.zeros(8, np.float32), [2 ** 32], [1], [1], [1], [1])


# ---- memory of another device --------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["conv", "scan", "norm"])
@pytest.mark.parametrize("backward", [False, True])
def test_memory_that_the_device_does_not_reach_is_refused(fake_queue, kind, backward):
    """Borrowed pointers may lie anywhere, whatever their queue says; reading one there would fault."""
    case = Case(fake_queue)
    lib = _capi.lib()
    stray = [0, 0, 0]  # address, kind of memory, device

    def place(address, kind, ordinal):
        if address == stray[0]:
            kind._obj.value, ordinal._obj.value = stray[1:]
        return 0

    lib.nb2_pointer_device = place
    build = case.backward if backward else case.forward
    plan = case.forward(kind)
    args = getattr(case, kind + "_grad" if backward else kind)
    build(kind, *([plan] if backward else []))
    for name, value in args.items():
        if not isinstance(value, (CUDARaggedArray, DeviceArray)):
            continue
        stray[0] = (value.cl_buf if isinstance(value, CUDARaggedArray) else value).data
        for stray[1], stray[2], message in ((2, 1, "on device 1"), (0, 0, "host memory")):
            with pytest.raises(ValueError, match=message):
                build(kind, *([plan] if backward else []))
        for stray[1], stray[2] in ((1, 0), (3, 0), (2, 0)):  # pinned host, managed and the device's own memory
            build(kind, *([plan] if backward else []))


def test_a_workspace_on_another_device_is_refused(fake_queue):
    """The current device is not the queue's while the plan is built: its table would lie on the wrong one."""
    case = Case(fake_queue)
    known = {v.cl_buf.data if isinstance(v, CUDARaggedArray) else v.data for kind in ("conv", "scan", "norm")
             for v in getattr(case, kind).values() if isinstance(v, (CUDARaggedArray, DeviceArray))}

    def place(address, kind, ordinal):
        ordinal._obj.value = 0 if address in known else 1
        return 0

    _capi.lib().nb2_pointer_device = place
    for kind in ("conv", "scan", "norm"):
        with pytest.raises(ValueError, match="workspace.*device 1"):
            case.forward(kind)


def test_memory_kinds_agree_with_the_header():
    c = _capi.header_constants("NB2_MEM_")
    assert (seq.MEM_UNKNOWN, seq.MEM_DEVICE) == (c["NB2_MEM_UNKNOWN"], c["NB2_MEM_DEVICE"])
    assert _capi.lib().nb2_pointer_device(None, None, None) == -2
