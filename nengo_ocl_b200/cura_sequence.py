"""Plans for operators over sequences: the short causal convolution, the selective state space scan
and the norms around a block with its gate and residual, each with its backward pass.

They stand beside ``plan_linearfilter`` (a linear filter with fixed coefficients, stepped once per time
step) and ``plan_conv2d``; the reference has no counterpart.  A *sequence array* is a
``CUDARaggedArray`` with one item of shape (rows, channels) per sequence: rows are time steps (tokens),
lengths may differ and may be zero.  Rows may be any distance apart (an item can be a column range of a
wider buffer), channels lie next to each other.  Element types: float32, float16 and ``bfloat16`` (one
for all sequence arrays of a plan).  Parameters, scan states and their gradients are float32; sums,
states and norms are held in float32 whatever the type, and results are rounded once, when stored.  The
exponentials of gates, steps and decays are the hardware's, for float32 too: a gate's sigmoid is off by up to
(4 + 1.2 |v|) * 2^-23 of its value.  An infinite or NaN input may make NaN of whatever depends on it, and of nothing
else: other sequences, earlier rows (backward: later ones) and the scan's other channels are as without it.

The same plan serves prompts and single tokens: state goes in through ``state`` and comes out through
``new_state``, which may be the same items (updated in place).  Otherwise nothing that a plan writes may
overlap anything else that it reads or writes; this is checked, and ``ValueError`` says what is wrong
with an argument, ``NotImplementedError`` what the kernels do not cover.  Rows that no sequence covers
are left as they were.  A plan owns its workspace: it can be captured and replayed, but not run on two
streams at once.  Memory has to lie on the queue's device, which is the current one while plans are built
and run.
"""

import ctypes

import numpy as np

from nengo_ocl_b200 import _capi
from nengo_ocl_b200.curaggedarray import CUDARaggedArray
from nengo_ocl_b200.plan import Plan
from nengo_ocl_b200.runtime import DeviceArray
from nengo_ocl_b200.utils import bfloat16, is_number

_DTYPES = {np.dtype(np.float32): 0, np.dtype(np.float16): 1, bfloat16: 2}
MAX_TAPS = 8            # NB2_CONV_MAX_TAPS
MAX_STATES = 128        # NB2_SCAN_MAX_STATES
KEEP_ROWS = 16          # NB2_SCAN_KEEP
MAX_NORM_CHANNELS = 32768  # NB2_NORM_MAX_CHANNELS
MEM_UNKNOWN, MEM_DEVICE = 0, 2  # NB2_MEM_*

# Launch shapes, chosen by measurement on a B200 (148 multiprocessors).
# Units a multiprocessor of the convolution (rows of a unit are halved, 64 to 8, until there are so many): 2 / 4 / 8 / 16
# units 42.9 / 43.1 / 40.1 / 43.4 us forward (8192 rows x 4096, bf16), 2 / 4 / 8 53.9 / 57.4 / 57.3 us for both passes
# (4096 x 2048, f32).
CONV_UNITS, CONV_GRAD_UNITS = 8, 2
# Blocks a multiprocessor of the norm: 2 / 4 / 6 / 16 68 / 70 / 76 / 79 us (8192 x 4096 bf16), backward 1 / 2 / 4 129 / 139 /
# 155 us for both passes (4096 x 4096 bf16): every block sums its own share of the parameter gradients.
NORM_UNITS, NORM_GRAD_UNITS = 2, 1
# Sequences of at most this many rows go through the scan's token kernel (all of a plan's, or none: one longer sequence
# sends the tokens beside it through the walk).  4096 channels x 16 states, bf16, token kernel / walk: 1 row 3.7 / 6.0 us (one
# sequence) and 29 / 84 us (128 sequences), 2 rows 5.0 / 6.0 and 43 / 85, 4 rows 7.5 / 6.0 and 72 / 86.
TOKEN_ROWS = 2
# Sequences up to this length are not split; a unit has at least SCAN_LEAST_ROWS rows (512 rows x 1024 channels in units
# of 32 / 64 / 128: 20 / 24 / 38 us), and a split makes about SCAN_BLOCKS blocks (16384 x 1024: 592 / 1184 / 2368 221 / 211 / 209 us).
SCAN_WHOLE_ROWS, SCAN_LEAST_ROWS, SCAN_BLOCKS = 96, 32, 148 * 8


# ---- argument checks -------------------------------------------------------------------------
class _Memory:
    """The strided rows an argument covers, in bytes: one entry per sequence (or one, for a parameter)."""

    def __init__(self, name, low, rows, pitch, width, written):
        self.name, self.written = name, written
        some = (rows > 0) & (width > 0)
        self.index = np.flatnonzero(some)
        self.low, self.rows, self.pitch = low[some], rows[some], pitch[some]
        self.width = width[some]
        self.high = self.low + (self.rows - 1) * self.pitch + self.width

    def pairs(self, other):
        """Pairs of entries (i of self, j of other) whose rows share bytes."""
        if not len(self.low) or not len(other.low):
            return np.zeros((0, 2), int)
        if self.low.min() >= other.high.max() or other.low.min() >= self.high.max():
            return np.zeros((0, 2), int)
        found = []
        order = np.argsort(other.low, kind="stable")
        low, top = other.low[order], np.maximum.accumulate(other.high[order])
        for i in range(len(self.low)):
            a, b = np.searchsorted(top, self.low[i], side="right"), np.searchsorted(low, self.high[i], side="left")
            for j in order[a:b]:
                if self._share(i, other, j):
                    found.append((self.index[i], other.index[j]))
        return np.array(found, int).reshape(-1, 2)

    def _share(self, i, other, j):
        a, b, wa, wb = int(self.low[i]), int(other.low[j]), int(self.width[i]), int(other.width[j])
        na, nb = int(self.rows[i]), int(other.rows[j])
        if a >= int(other.high[j]) or b >= int(self.high[i]):
            return False
        pa, pb = int(self.pitch[i]), int(other.pitch[j])
        if na == 1 and nb == 1:
            return a < b + wb and b < a + wa
        pitch = pb if na == 1 else pa
        if na > 1 and nb > 1 and pa != pb or pitch == 0:
            return True  # (rows of different pitch: not told apart)
        # row m of b minus row m' of a, m - m' = k: they share bytes when -wb < b - a + k pitch < wa
        first, last = (-wb - (b - a)) // pitch + 1, -((b - a - wa) // pitch) - 1
        return max(first, -(na - 1)) <= min(last, nb - 1)

    def repeats(self):
        """Whether two of the entries share bytes, or an entry's rows overlap each other."""
        if ((self.rows > 1) & (self.pitch < self.width)).any():
            return True
        order = np.argsort(self.low, kind="stable")
        top = np.maximum.accumulate(self.high[order])
        if (self.low[order][1:] >= top[:-1]).all():
            return False
        return any(i != j for i, j in self.pairs(self))


class _Arguments:
    """Collects a plan's arrays, checks them and lays out the table of a launch."""

    def __init__(self, queue, X, what="X"):
        self.queue = queue
        self.what = what
        if not isinstance(X, CUDARaggedArray):
            raise ValueError("%s must be a CUDARaggedArray" % what)
        if len(X) == 0:
            raise ValueError("%s has no sequences" % what)
        self.dtype = np.dtype(X.dtype)
        if self.dtype not in _DTYPES:
            raise NotImplementedError("sequences of type %s" % self.dtype)
        self.lengths = X.shape0s.astype(np.int64)
        self.channels = int(X.shape1s[0])
        if self.channels < 1:
            raise ValueError("%s has no channels" % what)
        self.memory = []
        self.fields = []
        self.kept = []
        self.blocks = []
        self.scratched = 0
        self.aligned = True

    def rows(self, name, ra, columns=None, lengths=None, dtype=None, written=False, optional=False, vec=True):
        """One sequence array: adds its (start, stride) fields, returns its buffer's address."""
        if ra is None:
            if not optional:
                raise ValueError("%s is missing" % name)
            self.fields += [np.zeros(len(self.lengths), np.int64)] * 2
            return None
        columns = self.channels if columns is None else columns
        lengths = self.lengths if lengths is None else lengths
        dtype = self.dtype if dtype is None else np.dtype(dtype)
        if not isinstance(ra, CUDARaggedArray):
            raise ValueError("%s must be a CUDARaggedArray" % name)
        if len(ra) != len(self.lengths):
            raise ValueError("%s has %d items, %s has %d" % (name, len(ra), self.what, len(self.lengths)))
        if np.dtype(ra.dtype) != dtype:
            raise ValueError("%s is of type %s, not %s" % (name, np.dtype(ra.dtype), dtype))
        if not np.array_equal(ra.shape0s, lengths):
            raise ValueError("%s: the items' rows differ from those expected" % name)
        if (ra.shape1s != columns).any():
            raise ValueError("%s: %d columns are expected" % (name, columns))
        starts, strides = ra.index64("starts"), ra.index64("stride0s")
        rows, some = lengths, lengths > 0
        strides = np.where(rows > 1, strides, columns)
        if columns > 1 and ((ra.index64("stride1s") != 1) & some).any():
            raise NotImplementedError("%s: channels must lie next to each other (stride1 == 1)" % name)
        if (strides < 0).any():
            raise NotImplementedError("%s: rows in reverse order" % name)
        ends = starts + np.maximum(rows - 1, 0) * strides + columns
        if (some & ((starts < 0) | (ends > ra.cl_buf.size))).any():
            raise ValueError("%s: an item reaches past the end of its buffer" % name)
        self._same_device(name, ra.cl_buf)
        size = dtype.itemsize
        self.memory.append(_Memory(name, ra.cl_buf.data + starts * size, rows, strides * size,
                                   np.full(len(starts), columns * size), written))
        if vec:
            self.aligned = self.aligned and not (ra.cl_buf.data % 16 or (starts[some] * size % 16).any()
                                                 or (strides[rows > 1] * size % 16).any())
        self.fields += [starts, strides]
        self.kept.append(ra.cl_buf)
        return ra.cl_buf.data

    def param(self, name, ary, shape, written=False, optional=False):
        """A contiguous float32 parameter (or its gradient); returns its address."""
        if ary is None:
            if not optional:
                raise ValueError("%s is missing" % name)
            return None
        if not isinstance(ary, DeviceArray):
            raise ValueError("%s must be a DeviceArray" % name)
        if ary.dtype != np.float32:
            raise ValueError("%s must be float32" % name)
        have = tuple(n for n in ary.shape if n != 1)
        if have != tuple(n for n in shape if n != 1):
            raise ValueError("%s has shape %s, not %s" % (name, ary.shape, tuple(shape)))
        strides = getattr(ary, "strides", None)
        if strides is not None:
            want = 4
            for n, s in zip(ary.shape[::-1], strides[::-1]):
                if n > 1 and s != want:
                    raise NotImplementedError("%s must be contiguous" % name)
                want *= n
        if ary.data % 4:
            raise ValueError("%s is not aligned to its elements" % name)
        self._same_device(name, ary)
        one = np.ones(1, np.int64)
        self.memory.append(_Memory(name, one * ary.data, one, one * ary.nbytes, one * ary.nbytes, written))
        self.kept.append(ary)
        return ary.data

    def _same_device(self, name, ary):
        if ary.data % ary.dtype.itemsize:
            raise ValueError("%s is not aligned to its elements" % name)
        if ary.queue.context.ordinal != self.queue.context.ordinal:
            raise ValueError("%s is on device %d, the queue on device %d"
                             % (name, ary.queue.context.ordinal, self.queue.context.ordinal))
        self._reached(name, ary.data)

    def _reached(self, name, address):
        """The address must be memory that the queue's device reaches: a borrowed pointer may lie on another
        one or in ordinary host memory, and what was allocated while another device was current does too."""
        here = self.queue.context.ordinal
        kind, ordinal = ctypes.c_int(MEM_DEVICE), ctypes.c_int(here)
        _capi.call("nb2_pointer_device", address, ctypes.byref(kind), ctypes.byref(ordinal))
        if kind.value == MEM_UNKNOWN:
            raise ValueError("%s lies in host memory that the device does not reach" % name)
        if kind.value == MEM_DEVICE and ordinal.value != here:
            raise ValueError("%s lies on device %d, the queue on device %d" % (name, ordinal.value, here))

    def check_overlaps(self, in_place=()):
        """Nothing written may share memory with anything else; ``in_place``: a (read, written) pair of
        names whose items may be the same one by one."""
        for m in self.memory:
            if m.written and m.repeats():
                raise ValueError("%s: items that are written overlap each other" % m.name)
        for a, m in enumerate(self.memory):
            if not m.written:
                continue
            for b, o in enumerate(self.memory):
                if a == b or (o.written and b < a):
                    continue
                for i, j in m.pairs(o):
                    if (o.name, m.name) == in_place and i == j:
                        at = np.flatnonzero(m.index == i)[0], np.flatnonzero(o.index == j)[0]
                        if m.low[at[0]] == o.low[at[1]] and (m.rows[at[0]] == 1 or m.pitch[at[0]] == o.pitch[at[1]]):
                            continue
                    raise ValueError("%s, which is written, overlaps %s" % (m.name, o.name))

    # A plan's tables and scratch are one allocation and one upload: `table`, `units` and `scratch` note what is
    # needed and return a token, `place` puts the addresses into the launch's arguments.
    def _need(self, nbytes, host=None):
        self.blocks.append((int(nbytes), host))
        return len(self.blocks) - 1

    def table(self, *more):
        host = np.ascontiguousarray(np.stack([self.lengths] + self.fields + list(more)).astype(np.int64))
        return self._need(host.nbytes, host)

    def units(self, rows):
        """(sequence, first row) of every stretch of ``rows`` rows; one for an empty sequence too."""
        n = np.maximum(-(-self.lengths // rows), 1)
        seq = np.repeat(np.arange(len(n)), n)
        first = (np.arange(len(seq)) - np.repeat(np.cumsum(n) - n, n)) * rows
        if first.max() >= 2 ** 31:
            raise NotImplementedError("sequences of 2^31 rows")
        host = np.ascontiguousarray(np.stack([seq, first], axis=1).astype(np.int32))
        return self._need(host.nbytes, host), len(seq)

    def scratch(self, n, passes=2):
        """``n`` floats, read or written ``passes`` times in all."""
        self.scratched += 4 * int(n) * passes
        return self._need(4 * max(int(n), 1))

    def moved(self):
        """Bytes that a call moves: every array's once, and the scratch's."""
        return sum(int((m.rows * m.width).sum()) for m in self.memory) + self.scratched

    def place(self, args, **tokens):
        """Allocates what was asked for and sets the fields ``name=token`` of ``args``."""
        up = lambda n: (n + 255) // 256 * 256
        order = sorted(range(len(self.blocks)), key=lambda i: self.blocks[i][1] is None)  # what is uploaded first
        offsets, total, upload = {}, 0, 0
        for i in order:
            offsets[i] = total
            total += up(self.blocks[i][0])
            upload = total if self.blocks[i][1] is not None else upload
        memory = DeviceArray(self.queue, (total,), np.uint8)
        self._reached("the plan's workspace (allocated on the current device)", memory.data)
        host = np.zeros(upload, np.uint8)
        for i, (nbytes, data) in enumerate(self.blocks):
            if data is not None:
                host[offsets[i]:offsets[i] + nbytes] = data.view(np.uint8).reshape(-1)
        memory.write_region(0, host)
        self.kept.append(memory)
        for name, token in tokens.items():
            if token is not None:
                setattr(args, name, memory.data + offsets[token])

    def common(self):
        return dict(device=self.queue.context.ordinal, dtype=_DTYPES[self.dtype], n_seq=len(self.lengths),
                    channels=self.channels)


def _make_plan(queue, name, entry, args, kept, gsize, n_launches, tag, flops, moved):
    fn, check, ref = getattr(_capi.lib(), entry), _capi.check, ctypes.byref(args)

    def launch(stream):
        check(fn(stream, ref))

    plan = Plan(queue, launch, (max(int(gsize), 1),), n_launches=n_launches, name=name, tag=tag)
    plan.full_args = (args, kept)
    plan.flops_per_call = int(flops)
    plan.bw_per_call = int(moved)
    return plan


def _unit_rows(total, tiles, least, want):
    """Rows to a unit: enough units that every multiprocessor has several, none shorter than ``least``
    (a unit reads a few rows of its neighbours again) and none longer than 64."""
    rows = 64
    while rows > least and -(-total // rows) * tiles < 148 * want:
        rows //= 2
    return max(rows, least)


# ---- short causal convolution ----------------------------------------------------------------
def plan_causal_conv(queue, X, W, Y, bias=None, state=None, new_state=None, activation=None, tag=None):
    """``y[t] = act(bias + sum_j W[:, j] x[t - taps + 1 + j])``, channel by channel.

    ``W``: (channels, taps) float32, 1 <= taps <= 8; ``bias``: (channels,).  ``state`` / ``new_state``:
    (taps - 1, channels) items of X's type, the rows before the first one (zeros if None) and the last
    ones of the sequence; they may be the same items.  ``activation``: None or "silu" (v sigmoid(v))."""
    a = _Arguments(queue, X)
    if not isinstance(W, DeviceArray) or len(W.shape) != 2 or W.shape[0] != a.channels:
        raise ValueError("W must be a (channels, taps) DeviceArray")
    taps = W.shape[1]
    if not 1 <= taps <= MAX_TAPS:
        raise NotImplementedError("%d taps: 1 to %d are supported" % (taps, MAX_TAPS))
    if activation not in (None, "silu"):
        raise NotImplementedError("activation %r" % (activation,))
    back = np.full(len(a.lengths), taps - 1, np.int64)
    args = _capi.nb2_causal_conv_args(
        x=a.rows("X", X), y=a.rows("Y", Y, written=True), w=a.param("W", W, (a.channels, taps)),
        bias=a.param("bias", bias, (a.channels,), optional=True),
        state=a.rows("state", state, lengths=back, optional=True),
        new_state=a.rows("new_state", new_state, lengths=back, written=True, optional=True),
        taps=taps, silu=int(activation == "silu"), **a.common())
    a.check_overlaps(in_place=("state", "new_state"))
    width = 16 // a.dtype.itemsize
    args.vec = int(a.aligned and a.channels % width == 0)
    total = int(a.lengths.sum())
    args.unit_rows = _unit_rows(total, -(-a.channels // (128 * (4 if args.vec else 1))), 8, CONV_UNITS)
    units, args.n_units = a.units(args.unit_rows)
    a.place(args, table=a.table(), units=units)
    plan = _make_plan(queue, "cura_causal_conv", "nb2_causal_conv", args, a.kept, args.n_units * a.channels, 1, tag,
                      total * a.channels * (2 * taps + 4), a.moved())
    plan.sequence_args = dict(X=X, W=W, bias=bias, state=state, new_state=new_state, activation=activation)
    return plan


def plan_causal_conv_grad(queue, plan, dY, dX, dW, dbias=None, dstate=None, dnew_state=None, tag=None):
    """Backward pass of ``plan`` (from ``plan_causal_conv``): sets ``dX``, ``dW``, ``dbias`` and ``dstate``
    from ``dY`` and ``dnew_state`` (zeros if None).  Reads the forward pass's X, W, bias and state again,
    so a plan that updates its state in place has no backward pass."""
    f = plan.sequence_args
    a = _Arguments(queue, f["X"])
    taps = f["W"].shape[1]
    if f["state"] is not None and f["new_state"] is not None:
        probe = _Arguments(queue, f["X"])
        back = np.full(len(a.lengths), taps - 1, np.int64)
        probe.rows("state", f["state"], lengths=back)
        probe.rows("new_state", f["new_state"], lengths=back)
        if len(probe.memory[0].pairs(probe.memory[1])):
            raise ValueError("the forward plan overwrites its state, which the backward pass needs")
    if f["bias"] is None and dbias is not None:
        raise ValueError("dbias: the forward plan has no bias")
    if f["state"] is None and dstate is not None:
        raise ValueError("dstate: the forward plan has no state")
    back = np.full(len(a.lengths), taps - 1, np.int64)
    args = _capi.nb2_causal_conv_grad_args(
        x=a.rows("X", f["X"]), dy=a.rows("dY", dY), dx=a.rows("dX", dX, written=True),
        state=a.rows("state", f["state"], lengths=back, optional=True),
        dstate=a.rows("dstate", dstate, lengths=back, written=True, optional=True),
        dnew_state=a.rows("dnew_state", dnew_state, lengths=back, optional=True),
        w=a.param("W", f["W"], (a.channels, taps)), bias=a.param("bias", f["bias"], (a.channels,), optional=True),
        dw=a.param("dW", dW, (a.channels, taps), written=True),
        dbias=a.param("dbias", dbias, (a.channels,), written=True, optional=True),
        taps=taps, silu=int(f["activation"] == "silu"), **a.common())
    a.check_overlaps()
    width = 16 // a.dtype.itemsize
    args.vec = int(a.aligned and a.channels % width == 0)
    total = int(a.lengths.sum())
    args.unit_rows = _unit_rows(total, -(-a.channels // (128 * (4 if args.vec else 1))), 16, CONV_GRAD_UNITS)
    units, args.n_units = a.units(args.unit_rows)
    a.place(args, table=a.table(), units=units, part=a.scratch(args.n_units * (taps + 1) * a.channels))
    return _make_plan(queue, "cura_causal_conv_grad", "nb2_causal_conv_grad", args, a.kept,
                      args.n_units * a.channels, 2, tag, total * a.channels * (6 * taps + 10), a.moved())


# ---- selective state space scan --------------------------------------------------------------
def scan_tile(n_states, backward=False):
    """Channels that one block of the scan covers (``nb2_selective_scan_tile``): four states of two channels
    (backward: of one) to a lane, as many lanes to a channel as the states need, 128 lanes to a block."""
    lanes = 1
    while 4 * lanes < n_states:
        lanes *= 2
    return 128 // lanes * (1 if backward else 2)


def _scan_units(a, args, tiles, row, work, twice):
    """Splits the sequences into units of rows, or not.  A block walks a unit row after row: unsplit, the longest
    sequence takes ``row`` us a row however few blocks there are, and the whole batch ``work`` us a row and tile of
    channels.  Split, the batch takes ``twice`` that (every row's decay is computed again for the units' ends) and
    three launches.  The cheaper one is taken; measured on a B200, 4096 channels x 16 states, float32, unsplit / split:
    2 x 1024 rows 143 / 117 us, 4 x 1024 174 / 214, 2 x 2048 280 / 216, 8 x 512 138 / 227; backward, 2048
    channels: 2 x 512 rows 153 / 93, 8 x 256 151 / 168.  Returns the sequences' first units and what to place."""
    longest, total = max(int(a.lengths.max()), 1), int(a.lengths.sum())
    args.unit_rows = -(-longest // 32) * 32
    whole = max(longest * row, total * tiles * work)
    if longest > SCAN_WHOLE_ROWS and whole > twice * total * tiles * work + 2 * SCAN_LEAST_ROWS * row + 8:
        args.unit_rows = min(args.unit_rows, max(SCAN_LEAST_ROWS, -(-total * tiles // (SCAN_BLOCKS * 32)) * 32))
    units = np.maximum(-(-a.lengths // args.unit_rows), 1)
    tokens = dict.fromkeys(("units", "ends", "sums"))
    tokens["units"], args.n_units = a.units(args.unit_rows)
    if args.n_units > len(a.lengths):
        tokens["ends"] = a.scratch(args.n_units * a.channels * args.n_states, passes=4)  # (the join reads and writes it)
        tokens["sums"] = a.scratch(args.n_units * a.channels)
    return np.cumsum(units) - units, tokens


def plan_selective_scan(queue, X, dt, A, B, C, Y, D=None, Z=None, dt_bias=None, softplus=False, state=None,
                        new_state=None, keep=False, tag=None):
    """The linear filter whose step size, input and output weights depend on the row::

        s = softplus(dt + dt_bias)  (or dt + dt_bias)
        h[c, n] = exp(s[c] A[c, n]) h[c, n] + s[c] x[c] B[g, n]
        y[c] = (sum_n C[g, n] h[c, n] + D[c] x[c]) * (Z is None or z[c] sigmoid(z[c]))

    ``X``, ``dt``, ``Y``, ``Z``: (rows, channels); ``A``: (channels, n_states) float32, n_states <= 128;
    ``B``, ``C``: (rows, groups * n_states), group g being that many channels' share of them (their width
    tells the number of groups); ``D``, ``dt_bias``: (channels,).  ``state`` / ``new_state``: float32
    (channels, n_states) items, h before the first and after the last row (zeros if None); they may be the
    same items, and several sequences may start from one.  ``keep``: keep what the backward pass needs."""
    a = _Arguments(queue, X)
    if not isinstance(A, DeviceArray) or len(A.shape) != 2 or A.shape[0] != a.channels:
        raise ValueError("A must be a (channels, n_states) DeviceArray")
    n = A.shape[1]
    if not 1 <= n <= MAX_STATES:
        raise NotImplementedError("%d states: 1 to %d are supported" % (n, MAX_STATES))
    if not isinstance(B, CUDARaggedArray) or len(B) == 0:
        raise ValueError("B must be a CUDARaggedArray with an item per sequence")
    width = int(B.shape1s[0])
    groups = width // n
    if groups < 1 or width % n or a.channels % groups:
        raise ValueError("B has %d columns: a multiple of the %d states that divides the channels is expected"
                         % (width, n))
    per = np.full(len(a.lengths), a.channels, np.int64)
    args = _capi.nb2_selective_scan_args(x=a.rows("X", X), dt=a.rows("dt", dt), n_states=n, groups=groups,
                                         softplus=int(bool(softplus)), **a.common())
    each = 16 // a.dtype.itemsize  # elements of a 16-byte access
    a.aligned, rows_aligned = True, a.aligned
    args.B, args.C = a.rows("B", B, columns=width), a.rows("C", C, columns=width)
    args.vec = int(a.aligned and n % each == 0)
    a.aligned = rows_aligned
    args.y, args.z = a.rows("Y", Y, written=True), a.rows("Z", Z, optional=True)
    args.rows_vec = int(a.aligned and (a.channels // groups) % each == 0)
    a.aligned = True
    args.state = a.rows("state", state, columns=n, lengths=per, dtype=np.float32, optional=True)
    args.new_state = a.rows("new_state", new_state, columns=n, lengths=per, dtype=np.float32, written=True, optional=True)
    args.state_vec = int(a.aligned and n % 4 == 0)
    args.A = a.param("A", A, (a.channels, n))
    args.a_vec = int(args.A % 16 == 0)
    args.D = a.param("D", D, (a.channels,), optional=True)
    args.dt_bias = a.param("dt_bias", dt_bias, (a.channels,), optional=True)
    a.check_overlaps(in_place=("state", "new_state"))
    blocks = -(-a.lengths // KEEP_ROWS)
    first = np.cumsum(blocks) - blocks
    kept = a.scratch(int(blocks.sum()) * a.channels * n, passes=1) if keep else None
    longest = int(a.lengths.max())
    args.tokens = int(longest <= TOKEN_ROWS and not keep)
    launches, first_unit, tokens = 1, np.arange(len(a.lengths)), {}
    if not args.tokens:
        first_unit, tokens = _scan_units(a, args, groups * -(-(a.channels // groups) // scan_tile(n)), 0.135, 4.2e-4,
                                         2.2)
        launches = 3 if tokens["ends"] is not None else 1
    a.place(args, table=a.table(first, first_unit), keep=kept, **tokens)
    total = int(a.lengths.sum())
    plan = _make_plan(queue, "cura_selective_scan", "nb2_selective_scan", args, a.kept, len(a.lengths) * a.channels,
                      launches, tag, total * a.channels * (7 * n + 20), a.moved())
    plan.sequence_args = dict(X=X, dt=dt, A=A, B=B, C=C, D=D, Z=Z, dt_bias=dt_bias, softplus=bool(softplus), state=state,
                              keep=args.keep, kept=a.kept, first=first, n=n, groups=groups)
    return plan


def plan_selective_scan_grad(queue, plan, dY, dX, ddt, dA, dB, dC, dD=None, dZ=None, ddt_bias=None, dstate=None,
                             dnew_state=None, tag=None):
    """Backward pass of ``plan`` (from ``plan_selective_scan`` with ``keep=True``, run before it on the same
    inputs): sets the gradients of its inputs, parameters and initial state from ``dY`` and ``dnew_state``
    (zeros if None).  The gradients of B and C are summed over their group's channels."""
    f = plan.sequence_args
    if not f["keep"]:
        raise ValueError("the forward plan keeps nothing: build it with keep=True")
    for name, grad in (("D", dD), ("Z", dZ), ("dt_bias", ddt_bias), ("state", dstate)):
        if grad is not None and f[name] is None:
            raise ValueError("d%s: the forward plan has no %s" % (name, name))
    a = _Arguments(queue, f["X"])
    n, groups = f["n"], f["groups"]
    width = n * groups
    per = np.full(len(a.lengths), a.channels, np.int64)
    args = _capi.nb2_selective_scan_grad_args(x=a.rows("X", f["X"]), dt=a.rows("dt", f["dt"]), n_states=n, groups=groups,
                                              softplus=int(f["softplus"]), **a.common())
    each = 16 // a.dtype.itemsize
    a.aligned, rows_aligned = True, a.aligned
    args.B, args.C = a.rows("B", f["B"], columns=width), a.rows("C", f["C"], columns=width)
    args.vec = int(a.aligned and n % each == 0)
    a.aligned = rows_aligned
    args.z, args.dy = a.rows("Z", f["Z"], optional=True), a.rows("dY", dY)
    args.dx, args.ddt = a.rows("dX", dX, written=True), a.rows("ddt", ddt, written=True)
    a.aligned, rows_aligned = True, a.aligned
    args.dB, args.dC = a.rows("dB", dB, columns=width, written=True), a.rows("dC", dC, columns=width, written=True)
    a.aligned = rows_aligned
    args.dz = a.rows("dZ", dZ, written=True, optional=True)
    args.rows_vec = int(a.aligned and (a.channels // groups) % each == 0)
    a.aligned = True
    args.dstate = a.rows("dstate", dstate, columns=n, lengths=per, dtype=np.float32, written=True, optional=True)
    args.dnew_state = a.rows("dnew_state", dnew_state, columns=n, lengths=per, dtype=np.float32, optional=True)
    args.state_vec = int(a.aligned and n % 4 == 0)
    args.A = a.param("A", f["A"], (a.channels, n))
    args.D = a.param("D", f["D"], (a.channels,), optional=True)
    args.dt_bias = a.param("dt_bias", f["dt_bias"], (a.channels,), optional=True)
    args.dA = a.param("dA", dA, (a.channels, n), written=True)
    args.dD = a.param("dD", dD, (a.channels,), written=True, optional=True)
    args.ddt_bias = a.param("ddt_bias", ddt_bias, (a.channels,), written=True, optional=True)
    a.check_overlaps()
    args.keep = f["keep"]
    a.scratched += 4 * int((-(-a.lengths // KEEP_ROWS)).sum()) * a.channels * n
    a.kept.append(f["kept"])
    total = int(a.lengths.sum())
    args.total_rows = total
    tiles = -(-(a.channels // groups) // scan_tile(n, backward=True))
    first_unit, tokens = _scan_units(a, args, groups * tiles, 0.5, 1.3e-3, 1.25)
    a.place(args, table=a.table(f["first"], np.cumsum(a.lengths) - a.lengths, first_unit, np.zeros_like(first_unit)),
            part_bc=a.scratch(tiles * total * 2 * width), part_a=a.scratch(args.n_units * a.channels * n),
            part_d=a.scratch(args.n_units * a.channels), part_s=a.scratch(args.n_units * a.channels), **tokens)
    return _make_plan(queue, "cura_selective_scan_grad", "nb2_selective_scan_grad", args, a.kept,
                      len(a.lengths) * a.channels, 3 + 2 * bool(args.ends), tag, total * a.channels * (19 * n + 30), a.moved())


# ---- norms around a block --------------------------------------------------------------------
def plan_residual_norm(queue, X, Y=None, H=None, gate=None, gate_first=True, residual=None, weight=None, scale=1.0,
                       norm_weight=None, groups=1, eps=1e-5, tag=None):
    """What stands between two blocks, row by row::

        u = x silu(gate) if gate_first else x
        u = u / sqrt(mean(u^2 over its group of channels) + eps) * weight        (if weight is given)
        u = u if gate_first else u silu(gate)
        Y = residual + scale * u
        H = Y / sqrt(mean(Y^2) + eps) * norm_weight

    ``X``, ``gate``, ``residual``, ``Y``, ``H``: sequence arrays, all but X optional (without ``gate``,
    ``residual`` or ``weight`` their part is left out); one of Y and H is needed.  ``scale``: a number or a
    (channels,) array; ``weight``, ``norm_weight``: (channels,) (None: ones for ``norm_weight``).  H is
    computed from Y before Y's rounding."""
    a = _Arguments(queue, X)
    if Y is None and H is None:
        raise ValueError("neither Y nor H is given")
    groups = int(groups)
    if groups < 1 or a.channels % groups:
        raise ValueError("%d groups do not divide the %d channels" % (groups, a.channels))
    if groups > 1 and weight is None:
        raise ValueError("groups are those of the norm with `weight`, which is missing")
    if a.channels > MAX_NORM_CHANNELS:
        raise NotImplementedError("%d channels: at most %d are supported" % (a.channels, MAX_NORM_CHANNELS))
    if norm_weight is not None and H is None:
        raise ValueError("norm_weight is given but H is not")
    if not float(eps) >= 0:
        raise ValueError("eps must not be negative")
    number = is_number(scale)
    args = _capi.nb2_residual_norm_args(
        x=a.rows("X", X), y=a.rows("Y", Y, written=True, optional=True), h=a.rows("H", H, written=True, optional=True),
        gate=a.rows("gate", gate, optional=True), residual=a.rows("residual", residual, optional=True),
        weight=a.param("weight", weight, (a.channels,), optional=True),
        scale=None if number else a.param("scale", scale, (a.channels,)), scale_value=float(scale) if number else 0.0,
        norm_weight=a.param("norm_weight", norm_weight, (a.channels,), optional=True),
        groups=groups, gate_first=int(bool(gate_first)), eps=float(eps), **a.common())
    a.check_overlaps()
    args.vec = int(a.aligned and (a.channels // groups) % (16 // a.dtype.itemsize) == 0)
    args.param_vec = int(not any(p % 16 for p in (args.weight, args.scale, args.norm_weight) if p))
    total = int(a.lengths.sum())
    args.unit_rows = max(1, -(-total // (148 * NORM_UNITS)))
    units, args.n_units = a.units(args.unit_rows)
    a.place(args, table=a.table(), units=units)
    plan = _make_plan(queue, "cura_residual_norm", "nb2_residual_norm", args, a.kept, total * a.channels, 1, tag,
                      total * a.channels * 16, a.moved())
    plan.sequence_args = dict(X=X, gate=gate, gate_first=gate_first, residual=residual, weight=weight, scale=scale,
                              norm_weight=norm_weight, groups=groups, eps=eps)
    return plan


def plan_residual_norm_grad(queue, plan, dX, dY=None, dH=None, dgate=None, dresidual=None, dweight=None, dscale=None,
                            dnorm_weight=None, tag=None):
    """Backward pass of ``plan`` (from ``plan_residual_norm``): sets the gradients of its inputs and
    parameters from ``dY`` and ``dH`` (zeros if None; one of them is needed).  Reads the forward pass's
    inputs again."""
    f = plan.sequence_args
    if dY is None and dH is None:
        raise ValueError("neither dY nor dH is given")
    for name, grad in (("gate", dgate), ("residual", dresidual), ("weight", dweight)):
        if grad is not None and f[name] is None:
            raise ValueError("d%s: the forward plan has no %s" % (name, name))
    number = is_number(f["scale"])
    if dscale is not None and number:
        raise ValueError("dscale: the forward plan's scale is a number")
    if dnorm_weight is not None and (f["norm_weight"] is None or dH is None):
        raise ValueError("dnorm_weight needs dH and a forward plan with a norm_weight")
    a = _Arguments(queue, f["X"])
    vector = (a.channels,)
    args = _capi.nb2_residual_norm_grad_args(
        x=a.rows("X", f["X"]), gate=a.rows("gate", f["gate"], optional=True),
        residual=a.rows("residual", f["residual"], optional=True), dy=a.rows("dY", dY, optional=True),
        dh=a.rows("dH", dH, optional=True), dx=a.rows("dX", dX, written=True),
        dgate=a.rows("dgate", dgate, written=True, optional=True),
        dresidual=a.rows("dresidual", dresidual, written=True, optional=True),
        weight=a.param("weight", f["weight"], vector, optional=True),
        scale=None if number else a.param("scale", f["scale"], vector), scale_value=float(f["scale"]) if number else 0.0,
        norm_weight=a.param("norm_weight", f["norm_weight"], vector, optional=True),
        dweight=a.param("dweight", dweight, vector, written=True, optional=True),
        dscale=a.param("dscale", dscale, vector, written=True, optional=True),
        dnorm_weight=a.param("dnorm_weight", dnorm_weight, vector, written=True, optional=True),
        groups=f["groups"], gate_first=int(bool(f["gate_first"])), eps=float(f["eps"]), **a.common())
    a.check_overlaps()
    args.vec = int(a.aligned and (a.channels // f["groups"]) % (16 // a.dtype.itemsize) == 0)
    args.param_vec = int(not any(p % 16 for p in (args.weight, args.scale, args.norm_weight) if p))
    total = int(a.lengths.sum())
    args.unit_rows = max(1, -(-total // (148 * NORM_GRAD_UNITS)))
    units, args.n_units = a.units(args.unit_rows)
    a.place(args, table=a.table(), units=units, part=a.scratch(args.n_units * 2 * a.channels))
    return _make_plan(queue, "cura_residual_norm_grad", "nb2_residual_norm_grad", args, a.kept, total * a.channels,
                      2, tag, total * a.channels * 40, a.moved())
