"""4-bit rows and the products with 4-bit weights, against the same in 64 bits.

Quantisation and its inverse are exact.  A product's bound, element by element, from the arithmetic: products
of two 4-bit values are exact, the sum of K of them in f32 and the few operations of the epilogue are off by
at most a whole step (2^-23, so that a sum that cuts instead of rounding is covered) of the sum of the
magnitudes each; f32 rows enter as three bf16 terms that add up to them, three products for one.
An activation passes an error on by at most its slope (SiLU 1.1, the gate's sigmoid 1/4) and adds a few roundings
of its own.
"""
import numpy as np
import pytest

import oracle
from fp4_ref import quant, random_rows, row_bytes, values

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -23
NONE, SILU, RELU, GLU = 0, 1, 2, 3


def _lib():
    import nemoasr

    return nemoasr.lib()


def _sig(v):
    with np.errstate(over="ignore"):
        return 1 / (1 + np.exp(-v))


def _ref(x, w, bias, act, alpha, c0, extra):
    """(result, bound) in 64 bits; extra: the error of each product relative to its magnitude."""
    k = x.shape[1]
    s, mag = x @ w.T, np.abs(x) @ np.abs(w).T
    if bias is not None:
        s, mag = s + bias, mag + np.abs(bias)
    err = mag * (STEP * (k + 2) + extra)
    if act == GLU:
        n = s.shape[1] // 2
        a, g, ea, eg = s[:, :n], s[:, n:], err[:, :n], err[:, n:]
        y = a * _sig(g)
        e = ea * _sig(g) + np.abs(a) * eg / 4 + ea * eg + 4 * STEP * np.abs(y)
    elif act == SILU:
        y = s * _sig(s)
        e = 1.1 * err + 4 * STEP * np.abs(y)
    elif act == RELU:
        y, e = np.maximum(s, 0), err
    else:
        y, e = s, err
    y, e = alpha * y, np.abs(alpha) * e + STEP * np.abs(alpha * y)
    if c0 is not None:
        y = y + c0
        e = e + STEP * (np.abs(y) + np.abs(c0))
    return y, e + 1e-37


# ---- quantisation ------------------------------------------------------------------------------------


def _quant(gpu, x, ld=None, typ=None, off=0):
    """Codes and scales from the GPU (buffers with room behind, which has to stay) of f32 or bf16 bits x."""
    m, k = x.shape
    ld = k if ld is None else ld
    typ = int(x.dtype == np.uint16) if typ is None else typ
    buf = np.zeros(off + m * ld, x.dtype)
    buf[off:].reshape(m, ld)[:, :k] = x
    ldq, lds = row_bytes(k) + 16, row_bytes(k) // 16 + 4
    dx, dq, ds = gpu.put(buf), gpu.put(np.full(m * ldq, 0xAA, np.uint8)), gpu.put(np.full(m * lds, 0xAA, np.uint8))
    gpu.begin()
    gpu.check(_lib().nk_fp4_quant(gpu.h, dx.at(off * x.itemsize), typ, ld, dq.ptr, ldq, ds.ptr, lds, m, k))
    gpu.end()
    q, s = dq.read((m, ldq), np.uint8), ds.read((m, lds), np.uint8)
    assert (q[:, row_bytes(k):] == 0xAA).all() and (s[:, row_bytes(k) // 16:] == 0xAA).all()
    out = []
    for t, dt in ((0, np.float32), (1, np.uint16)):
        ldy = k + 3
        dy = gpu.put(np.full(m * ldy, 7, dt))
        gpu.begin()
        gpu.check(_lib().nk_fp4_dequant(gpu.h, dq.ptr, ldq, ds.ptr, lds, dy.ptr, t, ldy, m, k))
        gpu.end()
        y = dy.read((m, ldy), dt)
        assert (y[:, k:] == 7).all()
        out.append(y[:, :k])
        dy.free()
    for b in (dx, dq, ds):
        b.free()
    return q[:, :row_bytes(k)], s[:, :row_bytes(k) // 16], out


@pytest.mark.parametrize("m,k", [(1, 1), (3, 31), (5, 32), (2, 33), (7, 127), (4, 128), (3, 129), (9, 1000), (64, 1024), (33, 4096)])
@pytest.mark.parametrize("bf16", [False, True])
def test_quant_and_back(gpu, m, k, bf16):
    rng = np.random.default_rng([m, k])
    x = (rng.standard_normal((m, k)) * np.exp2(rng.integers(-30, 30, (m, 1)))).astype(np.float32)
    if bf16:
        x = oracle.bf16_to_f32(oracle.f32_to_bf16(x))
    arg = oracle.f32_to_bf16(x) if bf16 else x
    for ld, off in ((k, 0), (-(-k // 8) * 8 + 8, 0), (k + 3, 1)):
        q, s, back = _quant(gpu, arg, ld, off=off)
        rq, rs = quant(x)
        np.testing.assert_array_equal(s, rs)
        np.testing.assert_array_equal(q, rq)
        np.testing.assert_array_equal(back[0], values(rq, rs, k))
        np.testing.assert_array_equal(oracle.bf16_to_f32(back[1]), values(rq, rs, k))


def test_quant_borders(gpu):
    """Every tie and its neighbours in f32, at scales from the smallest to the largest, with either sign; whole
    blocks of zeros; subnormal blocks; the largest finite value."""
    t = np.array([0, 0.25, 0.5, 0.75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7], np.float32)
    t = np.concatenate([t, np.nextafter(t, np.float32(0)), np.nextafter(t, np.float32(9))])[:31]
    rows = []
    for e in (-126, -125, -124, -60, -1, 0, 1, 60, 120, 124):
        with np.errstate(over="ignore"):
            b = (np.append(t, np.float32(7.5)) * np.float32(2.0) ** e).astype(np.float32)
        rows += [b, -b]
    rows += [np.zeros(32, np.float32), np.full(32, 1e-45, np.float32), np.full(32, -3e-39, np.float32),
             np.full(32, np.finfo(np.float32).max)]
    x = np.stack(rows)
    q, s, back = _quant(gpu, x)
    rq, rs = quant(x)
    np.testing.assert_array_equal(s, rs)
    np.testing.assert_array_equal(q, rq)
    np.testing.assert_array_equal(back[0].astype(np.float64), values(rq, rs, 32))


def test_quant_not_finite(gpu):
    """An infinity or a NaN makes its block NaN and no other."""
    rng = np.random.default_rng(4)
    x = rng.standard_normal((6, 160)).astype(np.float32)
    x[0, 33], x[1, 0], x[2, 159], x[3, 64] = np.nan, np.inf, -np.inf, np.float32(np.nan)
    q, s, back = _quant(gpu, x)
    rq, rs = quant(x)
    np.testing.assert_array_equal(s, rs)
    np.testing.assert_array_equal(back[0], values(rq, rs, 160))
    assert np.isnan(back[0]).sum() == 4 * 32 and np.isnan(oracle.bf16_to_f32(back[1])).sum() == 4 * 32
    assert not (back[1][~np.isnan(back[0])] == 0x7FC0).any()


def test_dequant_every_code_and_scale(gpu):
    """All 16 codes under all 256 scales; f32 overflows where the value does."""
    q = np.tile(np.array([2 * i | (2 * i + 1) << 4 for i in range(8)], np.uint8), (256, 8))
    s = np.repeat(np.arange(256, dtype=np.uint8)[:, None], 4, 1)
    dq, ds, dy = gpu.put(q), gpu.put(s), gpu.alloc(256 * 128 * 4)
    gpu.begin()
    gpu.check(_lib().nk_fp4_dequant(gpu.h, dq.ptr, 64, ds.ptr, 4, dy.ptr, 0, 128, 256, 128))
    gpu.end()
    with np.errstate(over="ignore"):
        np.testing.assert_array_equal(dy.read((256, 128)), values(q, s, 128).astype(np.float32))
    for b in (dq, ds, dy):
        b.free()


@pytest.mark.parametrize("m,k,more", [(5, 64, 0), (9, 1000, 0), (9, 1000, 8), (33, 4096, 16), (3, 40, 8), (7, 1003, 5)])
@pytest.mark.parametrize("typ", [0, 1])
def test_dequant_rows_of_whole_16_bytes(gpu, m, k, more, typ):
    """Rows whose values are stored 16 bytes at a time, their last run cut off or not."""
    ld, dt = k + more, (np.float32, np.uint16)[typ]
    assert ld % 8 == 0
    q, s = random_rows(np.random.default_rng([m, k]), m, k)
    dq, ds, dy = gpu.put(q), gpu.put(s), gpu.put(np.full((m, ld), 7, dt))
    gpu.begin()
    gpu.check(_lib().nk_fp4_dequant(gpu.h, dq.ptr, q.shape[1], ds.ptr, s.shape[1], dy.ptr, typ, ld, m, k))
    gpu.end()
    y = dy.read((m, ld), dt)
    assert (y[:, k:] == 7).all()
    np.testing.assert_array_equal(oracle.bf16_to_f32(y[:, :k]) if typ else y[:, :k], values(q, s, k))
    for b in (dq, ds, dy):
        b.free()


# ---- products ----------------------------------------------------------------------------------------


def _product(gpu, kind, x, w, bias=None, act=NONE, c0=None, alpha=1.0, ldc=None, pad=0, off=0):
    """The GPU's result; x: f32 rows, or (codes, scales); w: (codes, scales); ldc and pad leave room behind the
    output rows, which has to stay; off moves C off its 16-byte alignment."""
    wq, ws = w
    n, k = wq.shape[0], x[2] if kind == "fp4" else x.shape[1]
    m = x[0].shape[0] if kind == "fp4" else x.shape[0]
    nout = n // 2 if act == GLU else n
    ldc = nout if ldc is None else ldc
    fill = np.full(off + (m + pad) * ldc, 7.0, np.float32)
    if c0 is not None:
        fill[off:].reshape(m + pad, ldc)[:m, :nout] = c0
    bufs = [gpu.put(wq), gpu.put(ws), gpu.put(fill)]
    db = gpu.put(bias) if bias is not None else None
    end = (bufs[0].ptr, wq.shape[1], bufs[1].ptr, ws.shape[1], db.ptr if db else None, bufs[2].at(4 * off), ldc, m, n, k, act,
           int(c0 is not None), alpha)
    gpu.begin()
    if kind == "fp4":
        bufs += [gpu.put(x[0]), gpu.put(x[1])]
        gpu.check(_lib().nk_gemm_fp4(gpu.h, bufs[3].ptr, x[0].shape[1], bufs[4].ptr, x[1].shape[1], *end))
    else:
        lda = -(-k // 4) * 4
        rows = np.full((m, lda), np.nan, np.float32)  # what lies behind a row is not read
        rows[:, :k] = x
        bufs.append(gpu.put(rows))
        gpu.check(_lib().nk_gemm_w4(gpu.h, bufs[3].ptr, lda, *end))
    gpu.end()
    out = bufs[2].read(fill.shape)
    for b in bufs + ([db] if db else []):
        b.free()
    assert (out[:off] == 7).all()
    out = out[off:].reshape(m + pad, ldc)
    assert (out[m:] == 7).all() and (out[:, nout:] == 7).all()
    return out[:m, :nout]


def _check(gpu, kind, m, n, k, act=NONE, bias=False, resid=False, alpha=1.0, **more):
    rng = np.random.default_rng([m, n, k, act])
    w = random_rows(rng, n, k)
    wv = values(*w, k)
    b = rng.standard_normal(n).astype(np.float32) if bias else None
    nout = n // 2 if act == GLU else n
    c0 = rng.standard_normal((m, nout)).astype(np.float32) if resid else None
    if kind == "fp4":
        x = random_rows(rng, m, k, 124, 130)
        got = _product(gpu, kind, (*x, k), w, b, act, c0, alpha, **more)
        ref, tol = _ref(values(*x, k), wv, b, act, alpha, c0, 0.0)
    else:
        x = rng.standard_normal((m, k)).astype(np.float32)
        got = _product(gpu, kind, x, w, b, act, c0, alpha, **more)
        ref, tol = _ref(x.astype(np.float64), wv, b, act, alpha, c0, 2 * STEP * k)
    over = np.abs(got - ref) / tol
    assert np.isfinite(got).all() and over.max() <= 1, (over.max(), np.unravel_index(over.argmax(), over.shape))


KINDS = pytest.mark.parametrize("kind", ["fp4", "w4"])


@KINDS
@pytest.mark.parametrize("m", [1, 2, 5, 15, 16, 17, 31, 33, 48, 64, 65, 100, 129, 200, 257])
@pytest.mark.parametrize("n,k", [(64, 128), (96, 512), (200, 1024), (33, 97), (1, 1), (130, 2304)])
def test_product_sizes(gpu, kind, m, n, k):
    _check(gpu, kind, m, n, k)


@KINDS
@pytest.mark.parametrize("m,n,k", [(1, 4096, 1024), (7, 1024, 4096), (16, 640, 1024), (24, 2048, 2048), (448, 1024, 512),
                                   (300, 520, 8192), (700, 4100, 260), (1030, 2048, 1024)])
@pytest.mark.parametrize("act,bias,resid,alpha", [(NONE, True, True, 0.5), (SILU, True, False, 1.0), (RELU, False, True, -2.0),
                                                  (GLU, True, True, 1.0)])
def test_product_epilogues(gpu, kind, m, n, k, act, bias, resid, alpha):
    _check(gpu, kind, m, n, k, act, bias, resid, alpha)


@KINDS
@pytest.mark.parametrize("m,n,k,act", [(2040, 4090, 2180, NONE), (1000, 8190, 2180, GLU)])
def test_product_widest_tiles(gpu, kind, m, n, k, act):
    """Enough outputs for the widest tiles, cut off at every side; an odd number of 128 values."""
    _check(gpu, kind, m, n, k, act, True, act == NONE)


@pytest.mark.parametrize("m", [1, 3, 5])
@pytest.mark.parametrize("n,k", [(4100, 650), (8192, 2048), (5001, 97)])
@pytest.mark.parametrize("act,bias,resid", [(NONE, True, False), (SILU, False, True)])
def test_w4_up_to_five_rows_of_wide_weights(gpu, m, n, k, act, bias, resid):
    """32 columns a workgroup, cut off too."""
    _check(gpu, "w4", m, n, k, act, bias, resid, 0.5)


@pytest.mark.parametrize("m,n,k", [(448, 4096, 1024), (440, 4090, 1000), (500, 4001, 1500)])
@pytest.mark.parametrize("act,bias,resid", [(NONE, True, True), (SILU, False, False)])
def test_w4_of_hundreds_of_rows(gpu, m, n, k, act, bias, resid):
    """Tiles of 64 x 128, cut off too."""
    _check(gpu, "w4", m, n, k, act, bias, resid, 0.5)


@KINDS
@pytest.mark.parametrize("m,n,k,act", [(200, 1000, 513, NONE), (200, 1000, 640, NONE), (200, 1000, 770, NONE), (200, 1000, 640, GLU),
                                       (1024, 4096, 1152, NONE), (1000, 4090, 1130, NONE), (1000, 8180, 1400, GLU),
                                       (2040, 4090, 2170, NONE), (1000, 8190, 2170, GLU), (70, 333, 4870, NONE)])
def test_product_odd_groups(gpu, kind, m, n, k, act):
    """Rows of an odd number of groups of 128 values (5, 7, 9, 11, 17, 39): the last step of 256 is half one, its
    scales alone behind the others'."""
    assert -(-k // 128) % 2 == 1
    _check(gpu, kind, m, n, k, act, True, act == NONE)


@pytest.mark.parametrize("m,n,k", [(24, 4090, 2300), (6, 8190, 1100), (50, 2047, 4100)])
@pytest.mark.parametrize("act", [NONE, SILU, GLU])
def test_w4_few_rows_of_wide_weights(gpu, m, n, k, act):
    """Rows by 16 and columns by 32, both cut off."""
    n -= act == GLU and n % 2
    _check(gpu, "w4", m, n, k, act, True, True, 0.5, ldc=n + 3, pad=2, off=1)
    _check(gpu, "w4", m, n, k, act, False, True, 1.0, ldc=-(-n // 4) * 4 + 4, pad=1)


@KINDS
@pytest.mark.parametrize("m,n,k", [(3, 70, 200), (40, 70, 200), (200, 262, 384)])
@pytest.mark.parametrize("act", [NONE, GLU])
def test_product_strides_and_room(gpu, kind, m, n, k, act):
    """Output rows apart and off their 16 bytes: nothing beside them is written."""
    _check(gpu, kind, m, n, k, act, True, True, 1.0, ldc=n + 5, pad=3, off=1)
    _check(gpu, kind, m, n, k, act, False, False, 1.0, ldc=-(-n // 4) * 4 + 4, pad=1)


@KINDS
@pytest.mark.parametrize("m", [5, 9, 40, 200])
@pytest.mark.parametrize("k", [128, 640])
def test_product_of_far_scales(gpu, kind, m, k):
    """Rows and weights under scales from the least to the largest (of f32 rows' weights those below 2^128), every pair of
    them whose sums of magnitudes are between 1e-30 and 1e38.  f32 rows lose what is below 2^-133 of a value."""
    rng = np.random.default_rng([m, k])
    ss = np.array([0, 1, 2, 7, 60, 126, 200, 250, 252] + [253, 254] * (kind == "fp4"))
    n = 5 * len(ss)
    w = random_rows(rng, n, k)
    w[1][:] = ss[np.arange(n) % len(ss)][:, None]
    wv, xs = values(*w, k), ss[np.arange(m) % len(ss)]
    if kind == "fp4":
        x = random_rows(rng, m, k)
        x[1][:] = xs[:, None]
        got, xv = _product(gpu, kind, (*x, k), w), values(*x, k)
    else:
        x = (rng.standard_normal((m, k)) * np.exp2(xs - 127.0)[:, None]).astype(np.float32)
        got, xv = _product(gpu, kind, x, w), x.astype(np.float64)
    ref, mag = xv @ wv.T, np.abs(xv) @ np.abs(wv).T
    tol = mag * STEP * (k + 2)
    if kind == "w4":
        tol = tol + mag * STEP * 2 * k + 2.0 ** -133 * np.abs(wv).sum(1)
    ok = (mag < 1e38) & (mag > 1e-30)
    assert ok.sum() > m * n / 3 and (np.abs(got - ref)[ok] <= tol[ok]).all()


@KINDS
@pytest.mark.parametrize("m", [2, 20, 300])
def test_product_not_finite(gpu, kind, m):
    """A NaN in a row, or in a block of weights, reaches that row, or that column, and no other."""
    rng = np.random.default_rng(m)
    n, k = 160, 320
    w = random_rows(rng, n, k)
    w[1][17, 3] = 255
    x = rng.standard_normal((m, k)).astype(np.float32)
    x[1, 5] = np.nan
    if kind == "fp4":
        got = _product(gpu, kind, (*quant(x), k), w)
    else:
        got = _product(gpu, kind, x, w)
    bad = np.zeros((m, n), bool)
    bad[1], bad[:, 17] = True, True
    np.testing.assert_array_equal(np.isnan(got), bad)
    assert np.isfinite(got[~bad]).all()


@KINDS
@pytest.mark.parametrize("m", [2, 20, 300])
@pytest.mark.parametrize("act", [SILU, RELU, GLU])
def test_activations_keep_nan(gpu, kind, m, act):
    """A NaN goes through every activation: what the quantisation marks in a block is not lost."""
    rng = np.random.default_rng([m, act])
    n, k = 160, 420
    w = random_rows(rng, n, k)
    w[1][17, 3] = 255
    x = rng.standard_normal((m, k)).astype(np.float32)
    x[1, 5] = np.inf if kind == "fp4" else np.nan
    got = _product(gpu, kind, (*quant(x), k) if kind == "fp4" else x, w, act=act)
    bad = np.zeros(got.shape, bool)
    bad[1], bad[:, 17] = True, True
    np.testing.assert_array_equal(np.isnan(got), bad)


@pytest.mark.parametrize("m", [3, 9, 40, 200])
def test_w4_infinite_row(gpu, m):
    """An infinite value of a row meets weights of either sign: infinite with the product's sign, NaN against zeros."""
    k, n = 64, 16
    code = np.zeros((n, 128), np.uint8)
    code[:, 3] = np.arange(16)
    w = (code[:, 0::2] | code[:, 1::2] << 4, np.full((n, 4), 127, np.uint8))
    x = np.ones((m, k), np.float32)
    x[1, 3] = np.inf
    got = _product(gpu, "w4", x, w)
    assert np.isfinite(np.delete(got, 1, 0)).all()
    np.testing.assert_array_equal(got[1], [np.nan] + [np.inf] * 7 + [np.nan] + [-np.inf] * 7)


@pytest.mark.parametrize("m,n", [(3, 16), (4, 4112), (9, 16), (24, 4096), (40, 16), (200, 16)])
@pytest.mark.parametrize("scale,count", [(140, 1), (127, 48), (252, 1)])
def test_w4_infinite_row_of_large_weights(gpu, m, n, scale, count):
    """An infinite value stays one however large its weights are, and however many it has."""
    k = 64
    code = np.zeros((n, 128), np.uint8)
    code[:, 3:3 + count] = (np.arange(n) % 16)[:, None]
    w = (code[:, 0::2] | code[:, 1::2] << 4, np.full((n, 4), scale, np.uint8))
    x = np.zeros((m, k), np.float32)
    x[1, 3:3 + count] = np.inf
    x[2, 3] = -np.inf
    got = _product(gpu, "w4", x, w)
    want = np.tile(np.array([np.nan] + [np.inf] * 7 + [np.nan] + [-np.inf] * 7, np.float32), n // 16)
    assert not np.delete(got, (1, 2), 0).any()
    np.testing.assert_array_equal(got[1], want)
    np.testing.assert_array_equal(got[2], -want)


@pytest.mark.parametrize("m", [3, 9, 40, 200])
def test_w4_signalling_nan(gpu, m):
    """A NaN whose payload lies in its lower half alone is a NaN in its row, no infinity."""
    w = random_rows(np.random.default_rng(m), 64, 200)
    x = np.ones((m, 200), np.float32)
    x.view(np.uint32)[1, 77] = 0x7F800001
    got = _product(gpu, "w4", x, w)
    assert np.isnan(got[1]).all() and np.isfinite(np.delete(got, 1, 0)).all()


@KINDS
def test_product_is_repeatable_and_captures(gpu, kind):
    """The same bits from every replay of a captured product, with other work between the replays."""
    L = _lib()
    rng = np.random.default_rng(3)
    for m, n, k in ((1, 2048, 1024), (12, 1024, 4096), (70, 512, 1024)):
        w, x = random_rows(rng, n, k), rng.standard_normal((m, k)).astype(np.float32)
        xq = quant(x)
        d = [gpu.put(a) for a in (w[0], w[1], x, xq[0], xq[1], np.zeros((m, n), np.float32))]

        def launch():
            end = (d[0].ptr, w[0].shape[1], d[1].ptr, w[1].shape[1], None, d[5].ptr, n, m, n, k, NONE, 0, 1.0)
            if kind == "fp4":
                gpu.check(L.nk_gemm_fp4(gpu.h, d[3].ptr, xq[0].shape[1], d[4].ptr, xq[1].shape[1], *end))
            else:
                gpu.check(L.nk_gemm_w4(gpu.h, d[2].ptr, k, *end))

        gpu.begin()
        launch()
        gpu.end()
        first = d[5].read((m, n))
        gpu.begin()
        gpu.check(L.gpu_capture_begin(gpu.h))
        launch()
        gr = L.gpu_capture_end(gpu.h)
        gpu.end()
        assert gr
        for _ in range(3):
            d[5].write(np.full((m, n), 9.0, np.float32))
            _check(gpu, kind, 9, 130, 1100)
            gpu.begin()
            gpu.check(L.gpu_graph_launch(gpu.h, gr))
            gpu.end()
            np.testing.assert_array_equal(d[5].read((m, n)), first)
        L.gpu_graph_free(gr)
        for b in d:
            b.free()
