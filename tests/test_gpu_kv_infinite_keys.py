"""Keys with infinite values behind what a head's fragments hold of it, on the GPU: a logit of -inf has no weight (a row
of nothing else is NaN), one of +inf makes its row NaN, and rows that do not see the key are as they are without it.  Heads of all widths, those that fill
their fragments and those that do not; few rows and many, split along the tokens or not."""
import numpy as np
import pytest

import oracle
from kv_ref import BF16, E4M3, F32, Pages
from test_gpu_kv import Cache, back, close, kept, run_attend, sequences, tokens_of
from test_gpu_kv_splits import attend_rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("typ", [F32, BF16])
@pytest.mark.parametrize("dh", [16, 32, 48, 64, 80, 96, 112, 128, 144, 192, 240, 256])
@pytest.mark.parametrize("rows,start", [(1, 70), (1, 3000), (20, 10), (11, 2500), (130, 0), (130, 2600)])
def test_attend_infinite_keys(gpu, typ, dh, rows, start):
    rng = np.random.default_rng([28, typ, dh, rows, start])
    hk, group = 2, 2
    seqs, M = sequences([rows, 2], [start, 30])
    pages = Pages(rng, BF16, hk, dh, 16, tokens_of(seqs))
    row, n = seqs[0, 3], start + rows
    at = [(start + rows // 3, dh - 1), (start // 2, dh - 8), (start + 2 * rows // 3, dh - 3)]  # tokens and their infinite value
    inf = oracle.f32_to_bf16(np.array([-np.inf], np.float32))[0]
    for j, d in at:
        pages.k[pages.table[row, j // 16], 0, j % 16, d] = inf
    q = rng.standard_normal((M, hk * group, dh)) * 2
    signs = np.where(np.arange(M)[:, None] % 4 == 3, -1.0, 1.0)  # of every fourth row the logits are +inf
    for _, d in at:
        q[:, :, d] = signs * (np.abs(q[:, :, d]) + 0.1)
    q = kept(q, typ)
    cache = Cache(gpu, pages)
    out = back(run_attend(gpu, cache, typ, q.reshape(M, -1), seqs, hk * group, fill=7.0), typ).reshape(q.shape)
    cache.free()
    scale = np.float64(np.float32(dh ** -0.5))
    for first, r, before, row in seqs:
        (k, ok), (v, _) = (pages.tokens(x, row, before + r) for x in "kv")
        pos = before + np.arange(r)
        for h in range(hk * group):
            kh = k[:, h // group]
            inf_at = ~np.isfinite(kh).all(1)
            with np.errstate(invalid="ignore"):  # a row that sees no other keys
                ref, bound = attend_rows(q[first:first + r, h], np.where(inf_at[:, None], 0.0, kh), v[:, h // group], ok & ~inf_at, pos, 0, 0, scale,
                                         typ, before + r)
            seen = (np.flatnonzero(inf_at) <= pos[:, None]).any(1)
            nan = seen & (signs[first:first + r, 0] < 0) | (pos < np.argmin(inf_at))  # or all that it sees are -inf
            got = out[first:first + r, h]
            assert np.isnan(got[nan]).all()
            close(got[~nan], ref[~nan], bound[~nan])


@pytest.mark.parametrize("typ", [F32, BF16])
@pytest.mark.parametrize("dh", [48, 80, 192])
@pytest.mark.parametrize("rows,start", [(1, 700), (140, 0)])
def test_attend_nan_codes(gpu, typ, dh, rows, start):
    """Keys of an 8-bit cache that are NaN, in the head's last value: the rows that see them are, no others."""
    rng = np.random.default_rng([29, typ, dh, rows])
    seqs, M = sequences([rows, 2], [start, 30])
    pages = Pages(rng, E4M3, 1, dh, 32, tokens_of(seqs))
    row, j = seqs[0, 3], start + rows // 2
    pages.k[pages.table[row, j // 32], 0, j % 32, dh - 1] = 0x7f
    q = kept(rng.standard_normal((M, 2, dh)), typ)
    cache = Cache(gpu, pages)
    out = back(run_attend(gpu, cache, typ, q.reshape(M, -1), seqs, 2, fill=7.0), typ).reshape(q.shape)
    cache.free()
    scale = np.float64(np.float32(dh ** -0.5))
    nan = np.zeros(M, bool)
    nan[j - start:rows] = True
    assert np.isnan(out[nan]).all()
    for first, r, before, row in seqs:
        (k, ok), (v, _) = (pages.tokens(x, row, before + r) for x in "kv")
        ok = ok & np.isfinite(k).all((1, 2))
        for h in range(2):
            ref, bound = attend_rows(q[first:first + r, h], np.nan_to_num(k[:, 0]), v[:, 0], ok, before + np.arange(r), 0, 0, scale, typ, before + r)
            live = ~nan[first:first + r]
            close(out[first:first + r, h][live], ref[live], bound[live])
