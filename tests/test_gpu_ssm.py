"""The causal convolution and the selective scan over sequences of a batch, against loops in 64 bits.

Bounds, element by element, with u = 2^-24 (half a step of f32):
  convolution: taps + 2 roundings of the sum of the magnitudes, an activation's slope (SiLU 1.1) and a few roundings.
  scan: the reference carries a bound E of its state's error along,
      E <- a E + |a h| (|sA| (r + 3u) + 3u) + |s B x| (r + 3u) + u |h|
    where a = e^(sA) comes from the exponent's error (r: the relative error of s: its sum is off by u |v|, softplus
    passes on its slope's share and adds 4u) and the hardware's exponential (one step).  A scan that is split
    along its rows joins pieces with e^(A sum s), whose sum over a piece adds no more than that again: twice E.  The
    output adds N + 4 roundings of its terms' magnitudes and those of the gate.
  bf16 outputs: half a step, 2^-8, more.
"""
import ctypes as C

import numpy as np
import pytest

import nemoasr
import oracle
from fp4_ref import quant, random_rows, row_bytes, values

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16 = 0, 1


def _sig(v):
    with np.errstate(over="ignore"):
        return 1 / (1 + np.exp(-v))


def _bits(x, typ):
    return oracle.f32_to_bf16(x) if typ == BF16 else np.ascontiguousarray(x, np.float32)


def _kept(x, typ):
    """What rows of the type hold of x, in 64 bits."""
    return (oracle.bf16_to_f32(oracle.f32_to_bf16(x)) if typ == BF16 else np.asarray(x, np.float32)).astype(np.float64)


def _back(b, typ):
    return oracle.bf16_to_f32(b) if typ == BF16 else b


def _seqs(lens, slots, gap=0, start=0):
    """Table rows for sequences one after another, `gap` rows apart."""
    out, first = [], start
    for n, (a, b) in zip(lens, slots):
        out.append((first, n, a, b))
        first += n + gap
    return np.array(out, np.int32).reshape(-1, 4), first


# ---- convolution -------------------------------------------------------------------------------------


def conv_ref(x, w, bias, state, seqs, act):
    """(rows, bound, new state) of the convolution; x [M][D] and the rest in 64 bits."""
    taps = w.shape[1]
    y, e, new = np.zeros_like(x), np.zeros_like(x), state.copy()
    for first, n, a, b in seqs:
        line = np.concatenate([state[a] if a >= 0 else np.zeros((taps - 1, x.shape[1])), x[first:first + n]])
        s, m = np.zeros((n, x.shape[1])), np.zeros((n, x.shape[1]))
        for j in range(taps):
            s += line[j:j + n] * w[:, j]
            m += np.abs(line[j:j + n] * w[:, j])
        if bias is not None:
            s, m = s + bias, m + np.abs(bias)
        err = (taps + 2) * U * m
        if act == 1:
            y[first:first + n], e[first:first + n] = s * _sig(s), 1.1 * err + 8 * U * np.abs(s * _sig(s))
        else:
            y[first:first + n], e[first:first + n] = (np.maximum(s, 0) if act == 2 else s), err
        if b >= 0:
            new[b] = line[n:]
    return y, e, new


def run_conv(gpu, typ, x, w, bias, state, seqs, M, max_rows, act=1, ldx=None, ldy=None, off=0):
    """(output rows with what was there before, state) from the GPU."""
    D, taps = w.shape
    ldx, ldy = ldx or D, ldy or D
    dt = np.uint16 if typ == BF16 else np.float32
    xb = np.zeros((M, ldx), dt)
    xb[:, :D] = _bits(x, typ)
    d = [gpu.put(np.concatenate([np.zeros(off, dt), xb.ravel()])), gpu.put(w.astype(np.float32)), gpu.put(state.astype(np.float32)),
         gpu.put(seqs), gpu.put(np.full(off + (M + 2) * ldy, 9, dt))]
    db = gpu.put(bias.astype(np.float32)) if bias is not None else None
    size = xb.itemsize
    gpu.begin()
    gpu.check(nemoasr.lib().nk_causal_conv(gpu.h, d[0].at(off * size), typ, ldx, d[1].ptr, db.ptr if db else None, d[2].ptr,
                                           state.shape[0], d[3].ptr, len(seqs), max_rows, d[4].at(off * size), ldy, M, D, taps, act))
    gpu.end()
    y, st = d[4].read((off + (M + 2) * ldy,), dt), d[2].read(state.shape)
    for b in d + ([db] if db else []):
        b.free()
    assert (y[:off] == 9).all()
    return y[off:].reshape(M + 2, ldy), st


CONV_CASES = [  # lengths, (slot read, slot written), rows between the sequences
    ([1], [(0, 0)], 0),
    ([1, 1, 1, 1, 1], [(0, 0), (1, 4), (-1, 2), (3, -1), (5, 5)], 0),
    ([2, 0, 3, 1, 0], [(0, 0), (1, 1), (2, 3), (4, 4), (-1, 5)], 2),
    ([7, 33, 32, 64, 100], [(0, 1), (-1, 5), (2, 2), (3, -1), (4, 4)], 1),
    ([200], [(-1, -1)], 0),
]


@pytest.mark.parametrize("case", range(len(CONV_CASES)))
@pytest.mark.parametrize("D", [1, 100, 256, 1026, 2048])
@pytest.mark.parametrize("typ", [F32, BF16])
@pytest.mark.parametrize("taps", [2, 3, 4])
def test_conv(gpu, case, D, typ, taps):
    lens, slots, gap = CONV_CASES[case]
    rng = np.random.default_rng([case, D, taps])
    seqs, M = _seqs(lens, slots, gap)
    x, w = rng.standard_normal((M, D)), rng.standard_normal((D, taps)).astype(np.float32)
    bias = rng.standard_normal(D).astype(np.float32) if taps != 3 else None
    state = rng.standard_normal((6, taps - 1, D)).astype(np.float32)
    act = (case + taps) % 3
    more = [dict(), dict(ldx=2 * D + 8, ldy=D + 8), dict(ldx=D + 3, ldy=D + 1, off=1)][case % 3]
    y, st = run_conv(gpu, typ, x, w, bias, state, seqs, M, max(lens) + (case % 2) * 5, act, **more)
    xk = _kept(x, typ)
    ref, tol, new = conv_ref(xk, w.astype(np.float64), None if bias is None else bias.astype(np.float64), state.astype(np.float64), seqs, act)
    mine = np.zeros(M + 2, bool)
    for first, n, _, _ in seqs:
        mine[first:first + n] = True
    if typ == BF16:
        tol = tol + 2.0 ** -8 * (np.abs(ref) + tol)
    got = _back(y[:M, :D], typ)[mine[:M]]
    assert (np.abs(got - ref[mine[:M]]) <= tol[mine[:M]] + 1e-37).all()
    assert (y[~mine] == 9).all() and (y[:, D:] == 9).all()
    np.testing.assert_array_equal(st, new.astype(np.float32))


@pytest.mark.parametrize("typ,D,more", [(BF16, 2050, dict()), (BF16, 2050, dict(ldx=2051)), (F32, 2050, dict(ldy=2052))])
def test_conv_long(gpu, typ, D, more):
    """Enough values for longer tiles and two channels a thread (bf16 rows of an even stride)."""
    rng = np.random.default_rng(D)
    seqs, M = _seqs([8100, 37, 200], [(0, 0), (-1, 1), (2, 2)], 1)
    x, w, b = rng.standard_normal((M, D)), rng.standard_normal((D, 4)).astype(np.float32), rng.standard_normal(D).astype(np.float32)
    state = rng.standard_normal((3, 3, D)).astype(np.float32)
    y, st = run_conv(gpu, typ, x, w, b, state, seqs, M, 8100, 1, **more)
    ref, tol, new = conv_ref(_kept(x, typ), w.astype(np.float64), b.astype(np.float64), state.astype(np.float64), seqs, 1)
    if typ == BF16:
        tol = tol + 2.0 ** -8 * (np.abs(ref) + tol)
    for first, n, _, _ in seqs:
        assert (np.abs(_back(y[first:first + n, :D], typ) - ref[first:first + n]) <= tol[first:first + n] + 1e-37).all()
    np.testing.assert_array_equal(st, new.astype(np.float32))
    assert (y[M:] == 9).all() and (y[8100] == 9).all() and (y[:, D:] == 9).all()


@pytest.mark.parametrize("taps,act", [(2, 2), (3, 1), (3, 0)])
def test_conv_long_of_fewer_taps(gpu, taps, act):
    """Two bf16 channels a thread with two and three taps."""
    rng = np.random.default_rng(taps)
    D = 2050
    seqs, M = _seqs([8100, 1, 37, 200], [(0, 0), (3, 3), (-1, 1), (2, 2)], 1)
    x, w = rng.standard_normal((M, D)), rng.standard_normal((D, taps)).astype(np.float32)
    b = rng.standard_normal(D).astype(np.float32) if act else None
    state = rng.standard_normal((4, taps - 1, D)).astype(np.float32)
    y, st = run_conv(gpu, BF16, x, w, b, state, seqs, M, 8100, act, ldx=2052, ldy=2054)
    ref, tol, new = conv_ref(_kept(x, BF16), w.astype(np.float64), None if b is None else b.astype(np.float64), state.astype(np.float64),
                             seqs, act)
    tol = tol + 2.0 ** -8 * (np.abs(ref) + tol)
    for first, n, _, _ in seqs:
        assert (np.abs(_back(y[first:first + n, :D], BF16) - ref[first:first + n]) <= tol[first:first + n] + 1e-37).all()
    np.testing.assert_array_equal(st, new.astype(np.float32))
    assert (y[M:] == 9).all() and (y[8100] == 9).all() and (y[:, D:] == 9).all()


@pytest.mark.parametrize("typ,D,taps", [(F32, 2048, 4), (BF16, 2048, 3), (F32, 70, 2), (BF16, 512, 4)])
def test_conv_skewed_batch(gpu, typ, D, taps):
    """One long sequence among hundreds of tokens, in any order, and a max_rows far above it: the long one goes round
    a grid of fewer tiles, and max_rows changes no bit."""
    rng = np.random.default_rng(D)
    lens = np.concatenate([rng.integers(0, 4, 300), [3001, 64, 9]])
    seqs, M = _seqs(lens.tolist(), [((-1, i)[i % 2], i if i % 3 else -1) for i in range(len(lens))], 1)
    seqs = np.ascontiguousarray(seqs[rng.permutation(len(seqs))])
    x, w, b = rng.standard_normal((M, D)), rng.standard_normal((D, taps)).astype(np.float32), rng.standard_normal(D).astype(np.float32)
    state = rng.standard_normal((len(lens), taps - 1, D)).astype(np.float32)
    y, st = run_conv(gpu, typ, x, w, b, state, seqs, M, 3001)
    ref, tol, new = conv_ref(_kept(x, typ), w.astype(np.float64), b.astype(np.float64), state.astype(np.float64), seqs, 1)
    if typ == BF16:
        tol = tol + 2.0 ** -8 * (np.abs(ref) + tol)
    mine = np.zeros(M + 2, bool)
    for first, n, _, _ in seqs:
        mine[first:first + n] = True
    assert (np.abs(_back(y[:M], typ) - ref)[mine[:M]] <= tol[mine[:M]] + 1e-37).all() and (y[~mine] == 9).all()
    np.testing.assert_array_equal(st, new.astype(np.float32))
    for max_rows in (1 << 18, 1 << 30):
        y2, st2 = run_conv(gpu, typ, x, w, b, state, seqs, M, max_rows)
        np.testing.assert_array_equal(y2, y)
        np.testing.assert_array_equal(st2, st)


@pytest.mark.parametrize("typ", [F32, BF16])
def test_silu_of_far_values(gpu, typ):
    """SiLU of values down to the lowest: zero there, NaN at -infinity as the quotient gives, in the convolution and
    the gate (8 roundings, and 2e-36 where the hardware's reciprocal flushes)."""
    far = np.array([-3e38, -1e30, -1e10, -1000, -104.5, -103, -89, -88, -87, -80, 80, 87, 88.5, 104.5, 1e10, 3e38, np.inf, -np.inf, np.nan])
    D, v = len(far), _kept(far, typ)
    with np.errstate(invalid="ignore"):
        want = v * _sig(v)
    ok = np.isfinite(want)

    def check(row):
        got = _back(row, typ)
        tol = (8 * U + (2.0 ** -8 if typ == BF16 else 0)) * np.abs(want) + 2e-36
        assert (np.isnan(got) == np.isnan(want)).all() and (got[np.isinf(want)] == np.inf).all()
        assert (np.abs(got[ok] - want[ok]) <= tol[ok]).all()

    y, _ = run_conv(gpu, typ, far[None], np.repeat([[0.0, 1.0]], D, 0), None, np.zeros((1, 1, D)), np.array([[0, 1, -1, -1]], np.int32), 1, 1)
    check(y[0])
    for rows in (1, 40, 700):
        o = operands(np.random.default_rng(0), typ, rows, D, 4, 1, 1)
        o["z"] = np.repeat(v[None], rows, 0)
        o["x"], o["B"], o["C"], o["skip"] = np.ones((rows, D)), 0 * o["B"], 0 * o["C"], np.ones(D)
        c = ScanCall(gpu, typ, o, np.array([[0, rows, -1, -1]], np.int32), rows, 1)
        y, _ = c.run()
        c.free()
        for r in y[:rows]:
            check(r)


@pytest.mark.parametrize("typ", [F32, BF16])
@pytest.mark.parametrize("act", [0, 1, 2])
def test_conv_keeps_nan(gpu, typ, act):
    """A NaN reaches the rows of its channel that its taps reach, through every activation."""
    rng = np.random.default_rng(act)
    D, n = 70, 40
    x, w = rng.standard_normal((n, D)), 1 + rng.standard_normal((D, 3)).astype(np.float32) ** 2
    x[11, 5] = np.nan
    y, _ = run_conv(gpu, typ, x, w, None, np.zeros((1, 2, D)), np.array([[0, n, -1, -1]], np.int32), n, n, act)
    bad = np.zeros((n, D), bool)
    bad[11:14, 5] = True
    np.testing.assert_array_equal(np.isnan(_back(y[:n], typ)), bad)


def test_conv_in_pieces(gpu):
    """A sequence fed in pieces of any length, in one slot, gives the bits of the whole."""
    rng = np.random.default_rng(5)
    D, taps, n = 192, 4, 90
    x, w, b = rng.standard_normal((n, D)), rng.standard_normal((D, taps)), rng.standard_normal(D)
    state = np.zeros((1, taps - 1, D))
    whole, end = run_conv(gpu, F32, x, w, b, state, np.array([[0, n, -1, 0]], np.int32), n, n)
    parts, t, st = [], 0, state
    for c in (1, 1, 2, 0, 3, 40, 33, 1, 9):
        y, st = run_conv(gpu, F32, x[t:t + c] if c else x[:1], w, b, st, np.array([[0, c, 0, 0]], np.int32), max(c, 1), c)
        parts.append(y[:c])
        t += c
    assert t == n
    np.testing.assert_array_equal(np.concatenate(parts), whole[:n])
    np.testing.assert_array_equal(st, end)


# ---- scan --------------------------------------------------------------------------------------------


def scan_ref(o, seqs, softplus):
    """(rows, bound, states, their bound) of the scan in 64 bits; o: the operands as 64-bit arrays (None: left out)."""
    x, dt, B, Cm, z, A, skip, db, state = (o[k] for k in ("x", "dt", "B", "C", "z", "A", "skip", "dt_bias", "state"))
    M, D = x.shape
    G, N = B.shape[1:]
    y, e = np.zeros((M, D)), np.zeros((M, D))
    new, enew = state.copy(), np.zeros_like(state)
    for first, n, a0, b0 in seqs:
        h = state[a0].copy() if a0 >= 0 else np.zeros((D, N))
        E = np.zeros((D, N))
        for t in range(first, first + n):
            v = dt[t] + (db if db is not None else 0)
            ev = U * np.abs(v) if db is not None else np.zeros(D)
            if softplus:
                s = np.maximum(v, 0) + np.log1p(np.exp(-np.abs(v)))
                r = _sig(v) * ev / s + 4 * U
            else:
                s, r = v, np.where(v != 0, ev / np.where(v != 0, np.abs(v), 1), 0)
            s, r = s[:, None], r[:, None]
            a = np.exp(s * A)
            Bt, Ct = np.repeat(B[t], D // G, 0), np.repeat(Cm[t], D // G, 0)
            add = s * Bt * x[t][:, None]
            E = a * E + np.abs(a * h) * (np.abs(s * A) * (r + 3 * U) + 3 * U) + np.abs(add) * (r + 3 * U)
            h = a * h + add
            E = E + U * np.abs(h) + 1e-38
            o_, m = (Ct * h).sum(1), np.abs(Ct * h).sum(1)
            err = (np.abs(Ct) * 2 * E).sum(1)
            if skip is not None:
                o_, m = o_ + skip * x[t], m + np.abs(skip * x[t])
            err = err + (N + 4) * U * m
            if z is not None:
                gate = z[t] * _sig(z[t])
                o_, err = o_ * gate, err * np.abs(gate) + 8 * U * np.abs(o_ * gate)
            y[t], e[t] = o_, err
        if b0 >= 0:
            new[b0], enew[b0] = h, 2 * E
    return y, e, new, enew


def operands(rng, typ, M, D, N, G, slots, z=True, skip=True, db=True):
    x, dt, B, Cm = (rng.standard_normal(s).astype(np.float32) for s in ((M, D), (M, D), (M, G, N), (M, G, N)))
    o = {"x": x, "dt": 0.7 * dt - (0 if db else 3), "B": B, "C": Cm, "z": rng.standard_normal((M, D)) if z else None,
         "A": (-np.arange(1, N + 1) * np.exp(0.1 * rng.standard_normal((D, N)))).astype(np.float32),
         "skip": rng.standard_normal(D).astype(np.float32) if skip else None,
         "dt_bias": (-3 + rng.standard_normal(D)).astype(np.float32) if db else None,
         "state": rng.standard_normal((slots, D, N)).astype(np.float32)}
    return {k: v if v is None else _kept(v, typ if k in ("x", "dt", "B", "C", "z") else F32) for k, v in o.items()}


class ScanCall:
    """The operands on the GPU: x, dt and y rows of `pad` more values, z beside x, B and C parts of one projection's
    rows; what is left out is NaN, and the output's room 9."""

    def __init__(self, gpu, typ, o, seqs, max_rows, softplus, pad=0):
        self.gpu, self.typ = gpu, typ
        M, D = o["x"].shape
        G, N = o["B"].shape[1:]
        self.shape, self.M = (M + 2, D + pad), M
        nan = np.full
        xz = nan((M, 2 * D + pad), np.nan, np.float32)
        xz[:, :D] = o["x"]
        if o["z"] is not None:
            xz[:, D:2 * D] = o["z"]
        dt = nan((M, D + 2 * pad), np.nan, np.float32)
        dt[:, :D] = o["dt"]
        bc = nan((M, pad + 2 * G * N), np.nan, np.float32)
        bc[:, pad:pad + G * N], bc[:, pad + G * N:] = o["B"].reshape(M, -1), o["C"].reshape(M, -1)
        size = 2 if typ == BF16 else 4
        self.dt = np.uint16 if typ == BF16 else np.float32
        put = gpu.put
        self.bufs = b = {"xz": put(self._b(xz)), "dt": put(self._b(dt)), "bc": put(self._b(bc)), "seqs": put(seqs),
                         "y": put(np.full(self.shape, 9, self.dt)), "state": put(o["state"].astype(np.float32))}
        for k in ("A", "skip", "dt_bias"):
            if o[k] is not None:
                b[k] = put(o[k].astype(np.float32))
        at = lambda k: b[k].ptr if k in b else None  # noqa: E731
        self.state_shape = o["state"].shape
        self.args = nemoasr.Scan(type=typ, ldx=2 * D + pad, lddt=D + 2 * pad, ldbc=pad + 2 * G * N, ldz=2 * D + pad, ldy=D + pad,
                                 x=b["xz"].ptr, dt=b["dt"].ptr, B=b["bc"].at(size * pad), C=b["bc"].at(size * (pad + G * N)),
                                 z=b["xz"].at(size * D) if o["z"] is not None else None, y=b["y"].ptr, A=at("A"), skip=at("skip"),
                                 dt_bias=at("dt_bias"), state=b["state"].ptr, seqs=b["seqs"].ptr, slots=self.state_shape[0],
                                 nseq=len(seqs), max_rows=max_rows, M=M, D=D, N=N, groups=G, softplus=softplus)

    def _b(self, x):
        if self.typ == F32:
            return x
        bits = oracle.f32_to_bf16(np.nan_to_num(x))
        bits[np.isnan(x)] = 0x7FC0
        return bits

    def launch(self):
        self.gpu.check(nemoasr.lib().nk_ssm_scan(self.gpu.h, C.byref(self.args)))

    def run(self):
        self.gpu.begin()
        self.launch()
        self.gpu.end()
        return self.read()

    def read(self):
        return self.bufs["y"].read(self.shape, self.dt), self.bufs["state"].read(self.state_shape)

    def free(self):
        for b in self.bufs.values():
            b.free()


def check_scan(gpu, typ, o, seqs, max_rows, softplus=1, pad=0):
    c = ScanCall(gpu, typ, o, seqs, max_rows, softplus, pad)
    y, st = c.run()
    c.free()
    ref, tol, new, enew = scan_ref(o, seqs, softplus)
    M, D = ref.shape
    mine = np.zeros(M + 2, bool)
    for first, n, _, _ in seqs:
        mine[first:first + n] = True
    if typ == BF16:
        tol = tol + 2.0 ** -8 * (np.abs(ref) + tol)
    assert (y[~mine] == 9).all() and (y[:, D:] == 9).all()
    if mine.any():
        over = np.abs(_back(y[:M, :D], typ) - ref)[mine[:M]] / (tol[mine[:M]] + 1e-37)
        assert over.max() <= 1, (over.max(), np.unravel_index(over.argmax(), over.shape))
    over = np.abs(st - new) / (enew + 1e-37)
    assert over.max() <= 1, ("state", over.max(), np.unravel_index(over.argmax(), over.shape))
    return y, st


SCAN_CASES = [
    ([1], [(0, 0)], 0),
    ([1] * 6, [(0, 0), (1, 6), (-1, 2), (3, -1), (5, 5), (-1, 4)], 0),
    ([2, 0, 3, 1, 0], [(0, 0), (1, 1), (2, 3), (4, 4), (-1, 5)], 2),
    ([7, 33, 32, 64, 100], [(0, 1), (-1, 5), (2, 2), (3, -1), (4, 4)], 1),
    ([300], [(2, 3)], 0),
    ([700, 0, 1, 130], [(0, 0), (1, 2), (-1, 3), (-1, -1)], 3),
]


@pytest.mark.parametrize("case", range(len(SCAN_CASES)))
@pytest.mark.parametrize("D,N,G", [(64, 16, 1), (100, 5, 2), (256, 16, 4), (130, 1, 1), (96, 33, 3), (70, 64, 1), (320, 8, 1), (4, 12, 4)])
@pytest.mark.parametrize("typ", [F32, BF16])
def test_scan(gpu, case, D, N, G, typ):
    lens, slots, gap = SCAN_CASES[case]
    rng = np.random.default_rng([case, D, N])
    seqs, M = _seqs(lens, slots, gap)
    k = (case + D) % 4
    o = operands(rng, typ, M, D, N, G, 7, z=k != 0, skip=k != 1, db=k != 2)
    check_scan(gpu, typ, o, seqs, max(lens) + (case % 2) * 40, 1, [0, 8, 3][(case + N) % 3])


@pytest.mark.parametrize("case", range(len(SCAN_CASES)))
@pytest.mark.parametrize("D,N,G", [(64, 17, 1), (100, 20, 2), (96, 32, 3), (70, 31, 1), (260, 32, 1), (66, 48, 1)])
@pytest.mark.parametrize("typ", [F32, BF16])
def test_scan_more_states(gpu, case, D, N, G, typ):
    """17 to 32 states, and 48, in every form."""
    test_scan(gpu, case, D, N, G, typ)


@pytest.mark.parametrize("D,N,G", [(40, 20, 2), (24, 32, 1)])
@pytest.mark.parametrize("typ", [F32, BF16])
def test_scan_many_sequences_of_more_states(gpu, typ, D, N, G):
    test_scan_many_sequences(gpu, typ, D, N, G)


@pytest.mark.parametrize("rows", [1, 2, 500])
@pytest.mark.parametrize("typ", [F32, BF16])
def test_scan_wide(gpu, rows, typ):
    """More channels than a few workgroups."""
    rng = np.random.default_rng(rows)
    seqs, M = _seqs([rows, rows], [(0, 0), (1, 2)])
    check_scan(gpu, typ, operands(rng, typ, M, 2048, 16, 1, 3), seqs, rows)


@pytest.mark.parametrize("rows", [1, 5, 400])
def test_scan_no_softplus_and_far_steps(gpu, rows):
    """Steps given as they are (zero and below among them, with A of either sign), and softplus of far values."""
    rng = np.random.default_rng(rows)
    seqs, M = _seqs([rows], [(0, 1)])
    o = operands(rng, F32, M, 128, 16, 1, 2, db=False)
    o["dt"] = _kept(0.01 * np.abs(rng.standard_normal((M, 128))), F32)
    o["dt"][::3] = 0
    o["A"][:, ::2] *= -0.01
    check_scan(gpu, F32, o, seqs, rows, softplus=0)
    o = operands(rng, F32, M, 128, 16, 1, 2)
    o["dt"] = _kept(rng.choice([-200.0, -88.0, -20.0, 0.0, 3.0, 30.0, 90.0], (M, 128)) + rng.standard_normal((M, 128)), F32)
    check_scan(gpu, F32, o, seqs, rows)


@pytest.mark.parametrize("typ,D,N", [(F32, 64, 16), (BF16, 100, 5)])
@pytest.mark.parametrize("max_rows", [650, 1 << 18])
def test_scan_skewed_batch(gpu, typ, D, N, max_rows):
    """Long sequences among many short ones, in any order and with rows between them, and a max_rows far above the
    longest: the scratch goes by the rows that there are, so a capture finds room without a call before it."""
    L = nemoasr.lib()
    rng = np.random.default_rng(D)
    lens = np.concatenate([rng.integers(0, 4, 120), [650, 65, 64, 333, 1, 24, 25]])
    seqs, M = _seqs(lens.tolist(), [((-1, i)[i % 2], i if i % 3 else -1) for i in range(len(lens))], 1)
    seqs = np.ascontiguousarray(seqs[rng.permutation(len(seqs))])
    o = operands(rng, typ, M, D, N, 1, len(lens))
    c = ScanCall(gpu, typ, o, seqs, max_rows, 1)
    gpu.begin()
    gpu.check(L.gpu_capture_begin(gpu.h))
    c.launch()
    gr = L.gpu_capture_end(gpu.h)
    gpu.end()
    assert gr
    want = check_scan(gpu, typ, o, seqs, max_rows)
    gpu.begin()
    gpu.check(L.gpu_graph_launch(gpu.h, gr))
    gpu.end()
    for a, b in zip(want, c.read()):
        np.testing.assert_array_equal(a, b)
    L.gpu_graph_free(gr)
    c.free()


@pytest.mark.parametrize("D,N,G", [(24, 16, 1), (40, 5, 2), (70, 8, 1), (12, 33, 3), (9, 64, 1)])
@pytest.mark.parametrize("typ", [F32, BF16])
def test_scan_many_sequences(gpu, typ, D, N, G):
    """Thousands of sequences, most of them tokens or empty, a few of several tiles, in any order: each whole."""
    rng = np.random.default_rng([D, N])
    lens = np.concatenate([rng.integers(0, 3, 4196), [130, 64, 65, 41]])
    seqs, M = _seqs(lens.tolist(), [((-1, i)[i % 2], i if i % 3 else -1) for i in range(len(lens))], 1)
    seqs = np.ascontiguousarray(seqs[rng.permutation(len(seqs))])
    k = (D + typ) % 3
    o = operands(rng, typ, M, D, N, G, len(lens), z=k != 0, skip=k != 1, db=k != 2)
    check_scan(gpu, typ, o, seqs, 130, pad=3 * (k == 1))


@pytest.mark.parametrize("rows", [36, 129])
def test_scan_whole_of_wide_rows(gpu, rows):
    """Enough channels and sequences that a split does not pay."""
    rng = np.random.default_rng(rows)
    seqs, M = _seqs([rows] * 60, [(i, i) for i in range(60)])
    check_scan(gpu, BF16, operands(rng, BF16, M, 512, 16, 1, 60), seqs, rows)


@pytest.mark.parametrize("rows", [3, 37, 90, 601])
def test_scan_forgets_at_once(gpu, rows):
    """A of -infinity: every row's state is its own input's, also where rows do not fill a tile."""
    rng = np.random.default_rng(rows)
    seqs, M = _seqs([rows], [(0, 1)])
    o = operands(rng, F32, M, 64, 16, 1, 2)
    o["dt"] = np.maximum(o["dt"], -8.0)
    o["A"][:, ::3] = -np.inf
    c = ScanCall(gpu, F32, o, seqs, rows, 1)
    y, st = c.run()
    c.free()
    o["A"][:, ::3] = -1e30  # the same: e^(sA) is zero for every step here
    ref, tol, new, enew = scan_ref(o, seqs, 1)
    assert (np.abs(y[:M] - ref) <= tol + 1e-37).all() and (np.abs(st - new) <= enew + 1e-37).all()


def test_scan_of_growing_steps(gpu):
    """Steps below zero, which let states grow: a factor over many rows that passes the type's range takes a state
    of zero, or a tiny one, to where the recurrence does."""
    rng = np.random.default_rng(4)
    rows = 600
    seqs, M = _seqs([rows], [(0, 1)])
    o = operands(rng, F32, M, 64, 16, 1, 2, db=False)
    o["A"] = np.full((64, 16), -1.0)
    o["x"] *= 0
    o["state"][0, ::2] = 0
    o["state"][0, 1::2] = _kept(1e-37 * (1 + np.abs(o["state"][0, 1::2])), F32)
    o["dt"] = np.full((M, 64), -0.25)  # e^150 = 2^216 over the rows, e^8 over a piece of 32
    check_scan(gpu, F32, o, seqs, rows, softplus=0)
    o["dt"] = np.where(np.arange(M)[:, None] < 16, -9.0, 0.0) * np.ones((M, 64))  # 2^104 over 8 rows, 2^207 over 16
    check_scan(gpu, F32, o, seqs, rows, softplus=0)


@pytest.mark.parametrize("rows", [4, 600])
def test_scan_not_finite(gpu, rows):
    """An infinity or NaN in one channel's row reaches that channel's later rows of that sequence, and nothing else."""
    rng = np.random.default_rng(rows)
    seqs, M = _seqs([rows, rows], [(0, 0), (1, 1)])
    o = operands(rng, F32, M, 96, 16, 1, 2)
    clean = ScanCall(gpu, F32, o, seqs, rows, 1)
    y0, s0 = clean.run()
    clean.free()
    o["x"][rows // 2, 7], o["dt"][rows + 1, 40] = np.nan, np.inf
    c = ScanCall(gpu, F32, o, seqs, rows, 1)
    y, s = c.run()
    c.free()
    hit = np.zeros(y.shape, bool)
    hit[rows // 2:rows, 7], hit[rows + 1:2 * rows, 40] = True, True
    np.testing.assert_array_equal(y[~hit], y0[~hit])
    assert np.isnan(y[:M][hit[:M]]).all()
    hs = np.zeros(s.shape, bool)
    hs[0, 7], hs[1, 40] = True, True
    np.testing.assert_array_equal(s[~hs], s0[~hs])
    assert np.isnan(s[0, 7]).all()


def plain_scan(o, seqs, softplus):
    """Rows and states of the recurrence in 64 bits, infinities and NaN as they come."""
    M, D = o["x"].shape
    G, N = o["B"].shape[1:]
    y, new = np.zeros((M, D)), o["state"].copy()
    with np.errstate(all="ignore"):
        for first, n, a0, b0 in seqs:
            h = o["state"][a0].copy() if a0 >= 0 else np.zeros((D, N))
            for t in range(first, first + n):
                v = o["dt"][t] + (o["dt_bias"] if o["dt_bias"] is not None else 0)
                s = (np.maximum(v, 0) + np.log1p(np.exp(-np.abs(v))) if softplus else v)[:, None]
                h = np.exp(s * o["A"]) * h + s * np.repeat(o["B"][t], D // G, 0) * o["x"][t][:, None]
                y[t] = (np.repeat(o["C"][t], D // G, 0) * h).sum(1)
                if o["skip"] is not None:
                    y[t] += o["skip"] * o["x"][t]
                if o["z"] is not None:
                    y[t] *= o["z"][t] * _sig(o["z"][t])
            if b0 >= 0:
                new[b0] = h
    return y, new


def same_kind(got, want):
    """NaN where the recurrence has it, infinities with its sign, finite elsewhere."""
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    np.testing.assert_array_equal(np.where(np.isinf(got), got, 0), np.where(np.isinf(want), want, 0))


@pytest.mark.parametrize("N", [1, 3, 5, 8, 11, 16, 24, 33])
@pytest.mark.parametrize("rows,nseq", [(4, 2), (40, 2), (90, 60), (600, 2)])
@pytest.mark.parametrize("typ", [F32, BF16])
def test_scan_infinite_inputs(gpu, N, rows, nseq, typ):
    """Infinite inputs and steps give what the recurrence gives, whatever the number of states and whichever kernel
    runs: rows with the states over lanes, whole sequences, split ones.  Channels beside them keep their bits."""
    rng = np.random.default_rng([N, rows])
    D = 512 if nseq > 2 else 96
    seqs, M = _seqs([rows] * nseq, [(i, i) for i in range(nseq)])
    o = operands(rng, typ, M, D, N, 1, nseq)
    o["dt_bias"] = _kept(-4 + 0.3 * rng.standard_normal(D), F32)
    clean = ScanCall(gpu, typ, o, seqs, rows, 1)
    y0, s0 = clean.run()
    clean.free()
    o["x"][1, 7], o["x"][rows // 2, 9], o["x"][2, 30], o["dt"][rows + 1, 40] = np.inf, -np.inf, np.nan, np.inf
    o["B"][rows + 2, 0, N - 1] = np.inf
    o["B"][rows + 2, 0, :N - 1] = 0
    c = ScanCall(gpu, typ, o, seqs, rows, 1)
    y, s = c.run()
    c.free()
    want, new = plain_scan(o, seqs, 1)
    same_kind(_back(y[:M, :D], typ), want)
    same_kind(s, new)
    np.testing.assert_array_equal(y[:rows, 50:D], y0[:rows, 50:D])
    np.testing.assert_array_equal(s[0, 50:], s0[0, 50:])


@pytest.mark.parametrize("rows", [20, 200, 600])
def test_scan_infinite_state_is_kept(gpu, rows):
    """A state that is infinite stays so over any number of rows, of long steps too, as it does row by row; a rate of
    -infinity makes it NaN."""
    rng = np.random.default_rng(rows)
    seqs, M = _seqs([rows, rows], [(0, 0), (1, 1)])
    o = operands(rng, F32, M, 64, 16, 1, 2, db=False)
    o["A"] = _kept(np.full((64, 16), -16.0), F32)
    o["B"], o["C"], o["skip"] = np.abs(o["B"]), np.abs(o["C"]) + 0.1, np.abs(o["skip"])
    o["z"] = np.abs(o["z"]) + 0.1
    o["dt"] = np.full((M, 64), 1.0)  # e^-16 a row
    o["x"][3, 7], o["state"][1, 20, 4], o["x"][rows + 1, 33] = np.inf, -np.inf, np.inf
    o["A"][33, 2] = -np.inf
    c = ScanCall(gpu, F32, o, seqs, rows, 0)
    y, s = c.run()
    c.free()
    want, new = plain_scan(o, seqs, 0)
    same_kind(y[:M], want)
    same_kind(s, new)
    assert np.isposinf(y[rows - 1, 7]) and np.isneginf(s[1, 20, 4]) and np.isnan(s[1, 33, 2]) and np.isposinf(s[1, 33, 1])


def test_scan_in_pieces(gpu):
    """A sequence fed in pieces of any length, tokens among them, in one slot: the whole's result within the bounds."""
    rng = np.random.default_rng(8)
    D, N, n = 192, 16, 700
    o = operands(rng, F32, n, D, N, 1, 1)
    ref, tol, new, enew = scan_ref(o, np.array([[0, n, 0, 0]]), 1)
    t, st, got = 0, o["state"], []
    for c in (1, 1, 0, 2, 17, 300, 1, 300, 77, 1):
        p = {k: v[t:t + max(c, 1)] if k in ("x", "dt", "B", "C", "z") else v for k, v in o.items()}
        p["state"] = st
        if t == n:
            break
        call = ScanCall(gpu, F32, p, np.array([[0, c, 0, 0]], np.int32), c, 1)
        y, st = call.run()
        call.free()
        got.append(y[:c, :D])
        t += c
    assert t == n
    assert (np.abs(np.concatenate(got) - ref) <= 2 * tol).all() and (np.abs(st - new) <= 2 * enew).all()


def test_bad_entries_are_left_out(gpu):
    """Entries past the rows, the slots or max_rows write nothing; the sequences beside them are whole."""
    rng = np.random.default_rng(1)
    D, N, M = 70, 16, 40
    good = [(0, 10, 0, 1), (10, 12, -1, 2)]
    bad = [(35, 6, -1, 3), (-1, 4, -1, 3), (22, -3, -1, 3), (22, 4, 5, 3), (22, 4, -2, 3), (22, 4, -1, 5), (22, 4, -1, -2), (22, 13, -1, 3),
           (2 ** 31 - 1, 2, -1, 3), (41, 0, -1, 3)]
    seqs = np.array(good + bad, np.int32)
    o = operands(rng, F32, M, D, N, 1, 5)
    ref, tol, new, enew = scan_ref(o, good, 1)
    c = ScanCall(gpu, F32, o, seqs, 12, 1)
    y, st = c.run()
    c.free()
    assert (np.abs(y[:22, :D] - ref[:22]) <= tol[:22]).all() and (y[22:] == 9).all()
    assert (np.abs(st - new) <= enew + 1e-37).all()
    w, state = rng.standard_normal((D, 4)), rng.standard_normal((5, 3, D)).astype(np.float32)
    y, st = run_conv(gpu, F32, o["x"], w, None, state, seqs, M, 12)
    ref, tol, new = conv_ref(o["x"], w.astype(np.float32).astype(np.float64), None, state.astype(np.float64), good, 1)
    assert (np.abs(y[:22] - ref[:22]) <= tol[:22] + 1e-37).all() and (y[22:] == 9).all()
    np.testing.assert_array_equal(st, new.astype(np.float32))


def test_scan_without_slots(gpu):
    """No state anywhere: sequences from zero that leave none."""
    rng = np.random.default_rng(2)
    seqs, M = _seqs([5, 90], [(-1, -1), (-1, -1)])
    o = operands(rng, F32, M, 64, 16, 1, 1)
    c = ScanCall(gpu, F32, o, seqs, 90, 1)
    c.args.state, c.args.slots = None, 0
    y, _ = c.run()
    c.free()
    ref, tol, _, _ = scan_ref(o, seqs, 1)
    assert (np.abs(y[:M] - ref) <= tol).all()


@pytest.mark.parametrize("rows", [1, 3, 900])
def test_scan_captures(gpu, rows):
    """Replays of a captured scan that goes on in its own slots follow the same launches made one by one, other
    scans that use the context's scratch between them; two captured scans are replayed in turn."""
    L = nemoasr.lib()
    rng = np.random.default_rng(rows)
    seqs, M = _seqs([rows, rows], [(0, 0), (1, 1)])
    o, o2 = operands(rng, F32, M, 128, 16, 1, 2), operands(rng, F32, 1500, 64, 16, 1, 2)
    a, b = ScanCall(gpu, F32, o, seqs, rows, 1), ScanCall(gpu, F32, o, seqs, rows, 1)
    other = ScanCall(gpu, F32, o2, np.array([[0, 1500, 0, 1]], np.int32), 1500, 1)
    want_other = other.run()
    graphs = []
    for call in (a, other):
        gpu.begin()
        gpu.check(L.gpu_capture_begin(gpu.h))
        call.launch()
        graphs.append(L.gpu_capture_end(gpu.h))
        gpu.end()
        assert graphs[-1]
    for _ in range(3):
        want = b.run()
        for gr in graphs:
            gpu.begin()
            gpu.check(L.gpu_graph_launch(gpu.h, gr))
            gpu.end()
        got, got_other = a.read(), other.read()
        for x, y in zip(want + want_other, got + got_other):
            np.testing.assert_array_equal(x, y)
        check_scan(gpu, F32, o2, np.array([[0, 1400, 0, 1]], np.int32), 1400)
    for gr in graphs:
        L.gpu_graph_free(gr)
    for c in (a, b, other):
        c.free()


@pytest.mark.parametrize("typ,D,N,max_rows", [(F32, 128, 16, 700), (BF16, 70, 5, 700), (F32, 64, 16, 1 << 18), (F32, 100, 24, 32)])
def test_captured_block_takes_other_tables(gpu, typ, D, N, max_rows):
    """A captured convolution and scan, replayed with other sequences in the table: each replay gives the bits of the
    same calls made one by one, and of empty or unfitting entries nothing."""
    L = nemoasr.lib()
    rng = np.random.default_rng(D)
    M, ns, taps = 900, 6, 4
    o = operands(rng, typ, M, D, N, 1, ns)
    w, bias, cs = (rng.standard_normal(s).astype(np.float32) for s in ((D, taps), (D,), (ns, taps - 1, D)))
    long = min(max_rows, 650)
    tables = [[(0, long, 0, 0), (long, 30, -1, 1), (700, 1, 2, 3)] + [(0, 0, -1, -1)] * 3,
              [(i * 20, 1 + 3 * i, i, i) for i in range(ns)],
              [(800, 31, 5, 5), (0, 0, 4, 4), (M, 1, 3, 3), (100, 32, -1, 2), (40, 7, ns, 1), (60, 2, 0, 0)]]
    c = ScanCall(gpu, typ, o, np.array(tables[0], np.int32), max_rows, 1)
    f = [gpu.put(a) for a in (w, bias, cs, np.full((M, D), 9, c.dt))]

    def launch():
        gpu.check(L.nk_causal_conv(gpu.h, c.args.x, typ, c.args.ldx, f[0].ptr, f[1].ptr, f[2].ptr, ns, c.args.seqs, ns, max_rows, f[3].ptr, D,
                                   M, D, taps, 1))
        c.launch()

    def clear(table):
        f[2].write(cs)
        f[3].write(np.full((M, D), 9, c.dt))
        c.bufs["seqs"].write(np.array(table, np.int32))
        c.bufs["state"].write(o["state"].astype(np.float32))
        c.bufs["y"].write(np.full(c.shape, 9, c.dt))

    def result():
        return [f[2].read(cs.shape), f[3].read((M, D), c.dt), *c.read()]

    want = []
    for t in tables:
        clear(t)
        gpu.begin()
        launch()
        gpu.end()
        want.append(result())
    gpu.begin()
    gpu.check(L.gpu_capture_begin(gpu.h))
    launch()
    gr = L.gpu_capture_end(gpu.h)
    gpu.end()
    assert gr
    for i in (1, 0, 2, 1):
        clear(tables[i])
        gpu.begin()
        gpu.check(L.gpu_graph_launch(gpu.h, gr))
        gpu.end()
        for a, b in zip(want[i], result()):
            np.testing.assert_array_equal(a, b)
    L.gpu_graph_free(gr)
    c.free()
    for b in f:
        b.free()


@pytest.mark.parametrize("typ", [F32, BF16])
def test_most_sequences(gpu, typ):
    """65535 tokens in a call, their slots in another order."""
    rng = np.random.default_rng(7)
    n, D, N = 65535, 8, 4
    slot = rng.permutation(n)
    seqs = np.stack([np.arange(n), np.ones(n), slot, slot], 1).astype(np.int32)
    o = operands(rng, typ, n, D, N, 1, n)
    c = ScanCall(gpu, typ, o, seqs, 1, 1)
    y, st = c.run()
    c.free()
    v = o["dt"] + o["dt_bias"]
    s = (np.maximum(v, 0) + np.log1p(np.exp(-np.abs(v))))[:, :, None]
    h0, add = o["state"][slot], s * o["B"][:, 0, None] * o["x"][:, :, None]
    h = np.exp(s * o["A"]) * h0 + add
    # s is off by 4u and what its sum's rounding makes of it, as in scan_ref; |s A| is below 40 here
    r = _sig(v)[:, :, None] * U * np.abs(v)[:, :, None] / s + 4 * U
    e = np.abs(np.exp(s * o["A"]) * h0) * (np.abs(s * o["A"]) * (r + 3 * U) + 3 * U) + np.abs(add) * (r + 3 * U) + U * np.abs(h) + 1e-38
    assert (np.abs(st[slot] - h) <= 2 * e).all()
    gate = o["z"] * _sig(o["z"])
    m = (np.abs(o["C"][:, 0, None] * h)).sum(2) + np.abs(o["skip"] * o["x"])
    ref = ((o["C"][:, 0, None] * h).sum(2) + o["skip"] * o["x"]) * gate
    tol = ((np.abs(o["C"][:, 0, None]) * 2 * e).sum(2) + (N + 4) * U * m) * np.abs(gate) + 8 * U * np.abs(ref)
    if typ == BF16:
        tol = tol + 2.0 ** -8 * (np.abs(ref) + tol)
    assert (np.abs(_back(y[:n, :D], typ) - ref) <= tol + 1e-37).all()
    w, cs = rng.standard_normal((D, 4)).astype(np.float32), rng.standard_normal((n, 3, D)).astype(np.float32)
    y, st = run_conv(gpu, typ, o["x"], w, None, cs, seqs, n, 1, act=0)
    line = np.concatenate([cs[slot].astype(np.float64), o["x"][:, None]], 1)
    terms = line * w.T.astype(np.float64)
    tol = 6 * U * np.abs(terms).sum(1)
    if typ == BF16:
        tol = tol + 2.0 ** -8 * (np.abs(terms.sum(1)) + tol)
    assert (np.abs(_back(y[:n], typ) - terms.sum(1)) <= tol + 1e-37).all()
    np.testing.assert_array_equal(st[slot], line[:, 1:].astype(np.float32))


# ---- a block -----------------------------------------------------------------------------------------


@pytest.mark.parametrize("lens", [[1, 1, 1], [9, 0, 40], [350]])
def test_block(gpu, lens):
    """A selective-scan block as a program runs it: 4-bit projection in, convolution, 4-bit projections to the
    step, B and C, scan with its gate, 4-bit projection out added to the residual; against the same in 64 bits.
    The bound carries each operator's through the next as a norm: every product is off by at most 2^-16 + (K + 2)
    2^-23 of its magnitudes, the operators between by less; 1e-3 of the result's largest value holds that chain with
    magnitudes up to 30 times the values."""
    L = nemoasr.lib()
    rng = np.random.default_rng(lens)
    Dm, D, N, R, taps = 128, 256, 16, 8, 4
    seqs, M = _seqs(lens, [(-1 if i == 1 else i, i) for i in range(len(lens))])
    ns = len(lens)

    def matrix(n, k):
        w = quant(rng.standard_normal((n, k)) / np.sqrt(k))
        return w, values(*w, k), [gpu.put(w[0]), gpu.put(w[1])]

    win, wx, wdt, wout = matrix(2 * D, Dm), matrix(R + 2 * N, D), matrix(D, R), matrix(Dm, D)
    x0 = rng.standard_normal((M, Dm)).astype(np.float32)
    cw, cb = rng.standard_normal((D, taps)).astype(np.float32) / 2, rng.standard_normal(D).astype(np.float32) / 4
    A = (-np.arange(1, N + 1) * np.ones((D, 1))).astype(np.float32)
    skip, db = np.ones(D, np.float32), np.full(D, -4, np.float32)
    cs, ss = rng.standard_normal((ns, taps - 1, D)).astype(np.float32), rng.standard_normal((ns, D, N)).astype(np.float32)
    f = {k: gpu.put(v) for k, v in dict(x0=x0, cw=cw, cb=cb, A=A, skip=skip, db=db, cs=cs, ss=ss, seqs=seqs).items()}
    for k, w in (("xz", 2 * D), ("u", D), ("p", R + 2 * N), ("dt", D), ("y", D)):
        f[k] = gpu.put(np.zeros((M, w), np.float32))
    P = {k: b.ptr for k, b in f.items()}
    longest = max(lens)

    def w4(a, lda, w, c, ldc, n, k, acc=0):
        gpu.check(L.nk_gemm_w4(gpu.h, P[a], lda, w[2][0].ptr, row_bytes(k), w[2][1].ptr, row_bytes(k) // 16, None, P[c], ldc, M, n, k, 0,
                               acc, 1.0))

    gpu.begin()
    w4("x0", Dm, win, "xz", 2 * D, 2 * D, Dm)
    gpu.check(L.nk_causal_conv(gpu.h, P["xz"], F32, 2 * D, P["cw"], P["cb"], P["cs"], ns, P["seqs"], ns, longest, P["u"], D, M, D, taps, 1))
    w4("u", D, wx, "p", R + 2 * N, R + 2 * N, D)
    w4("p", R + 2 * N, wdt, "dt", D, D, R)
    a = nemoasr.Scan(type=F32, ldx=D, lddt=D, ldbc=R + 2 * N, ldz=2 * D, ldy=D, x=P["u"], dt=P["dt"], B=P["p"] + 4 * R, C=P["p"] + 4 * (R + N),
                     z=P["xz"] + 4 * D, y=P["y"], A=P["A"], skip=P["skip"], dt_bias=P["db"], state=P["ss"], seqs=P["seqs"], slots=ns, nseq=ns,
                     max_rows=longest, M=M, D=D, N=N, groups=1, softplus=1)
    gpu.check(L.nk_ssm_scan(gpu.h, C.byref(a)))
    w4("y", D, wout, "x0", Dm, Dm, D, acc=1)
    gpu.end()
    got = [f["x0"].read((M, Dm)), f["cs"].read(cs.shape), f["ss"].read(ss.shape)]

    xz = x0.astype(np.float64) @ win[1].T
    u, _, cn = conv_ref(xz[:, :D], cw.astype(np.float64), cb.astype(np.float64), cs.astype(np.float64), seqs, 1)
    p = u @ wx[1].T
    o = dict(x=u, dt=p[:, :R] @ wdt[1].T, B=p[:, None, R:R + N], C=p[:, None, R + N:], z=xz[:, D:], A=A.astype(np.float64),
             skip=skip.astype(np.float64), dt_bias=db.astype(np.float64), state=ss.astype(np.float64))
    y, _, sn, _ = scan_ref(o, seqs, 1)
    for g, w in zip(got, (x0 + y @ wout[1].T, cn, sn)):
        assert np.abs(g - w).max() <= 1e-3 * np.abs(w).max()
    for b in list(f.values()) + [b for w in (win, wx, wdt, wout) for b in w[2]]:
        b.free()
