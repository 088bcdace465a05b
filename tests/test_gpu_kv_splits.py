"""Attention of prompts whose tiles are split along their tokens, on the GPU: every row against the formula in 64 bits, the rows
that no sequence has as they were.  A causal prompt's first tiles see next to nothing and its last ones all of it, so that the
pieces, which all tiles of a sequence have alike, are most where there are somewhat fewer tiles than workgroups wanted."""
import numpy as np
import pytest

from kv_ref import BF16, E4M3, F32, U, Pages
from test_gpu_kv import Cache, back, close, kept, run_attend, sequences, tokens_of

pytestmark = pytest.mark.gpu


def attend_rows(q, k, v, ok, pos, window, sinks, scale, typ, n):
    """(rows, bounds) of one head's rows q [R][dh] at positions pos over keys and values of n tokens: the formula and bound of
    kv_ref.attend for many rows at once."""
    dh = q.shape[1]
    j = np.arange(n)
    see = ok & (j <= pos[:, None])
    if window:
        see &= (j > pos[:, None] - window) | (j < sinks)
    s = np.where(see, scale * (q @ k.T), -np.inf)
    w = np.exp(s - s.max(1, keepdims=True))
    w /= w.sum(1, keepdims=True)
    o = w @ v
    mag = np.where(see, np.abs(s), 0.0)
    d = w * (U * ((dh + 16) * scale * (np.abs(q) @ np.abs(k).T) + 4 * (mag + mag.max(1, keepdims=True)) + 2))
    a = w @ np.abs(v)
    err = d @ np.abs(v) + d.sum(1, keepdims=True) * np.abs(o) + U * (n / 32 + 40) * a
    if typ == BF16:
        err += 2.0 ** -8 * (a + np.abs(o) + err)
    return o, err + 1e-36


def check(gpu, typ, cache_type, hk, group, dh, rows, starts, window=0, sinks=0, **more):
    rng = np.random.default_rng([27, typ, hk, group, sum(rows), window])
    heads = hk * group
    seqs, M = sequences(rows, starts, gap=2)
    pages = Pages(rng, cache_type, hk, dh, 32, tokens_of(seqs))
    cache = Cache(gpu, pages)
    q = rng.standard_normal((M, heads * dh)) * 2
    out = back(run_attend(gpu, cache, typ, q, seqs, heads, window, sinks, fill=7.0, **more), typ).reshape(M, heads, dh)
    cache.free()
    q = kept(q, typ).reshape(M, heads, dh)
    scale = np.float64(np.float32(dh ** -0.5))
    left = np.ones(M, bool)
    for first, r, start, row in seqs:
        n = start + r
        left[first:first + r] = False
        (k, ok), (v, _) = (pages.tokens(x, row, n) for x in "kv")
        for h in range(heads):
            for i in range(0, r, 512):
                at = slice(first + i, first + min(r, i + 512))
                ref, bound = attend_rows(q[at, h], k[:, h // group], v[:, h // group], ok, start + np.arange(i, min(r, i + 512)), window, sinks,
                                         scale, typ, n)
                close(out[at, h], ref, bound)
    assert (out[left] == 7.0).all()


@pytest.mark.parametrize("typ,cache_type,hk,group,rows,starts,window", [
    (BF16, BF16, 8, 1, [2944], [0], 0),
    (BF16, E4M3, 8, 2, [1472], [0], 0),
    (BF16, BF16, 4, 4, [1472], [0], 0),
    (BF16, BF16, 4, 4, [1, 1500, 3], [90, 7, 0], 0),
    (BF16, E4M3, 2, 4, [3000], [0], 0),
    (BF16, BF16, 1, 8, [1987, 119], [0, 1788], 0),
    (BF16, BF16, 8, 1, [2900], [0], 2890),
    (F32, BF16, 8, 4, [1472], [0], 0),
    (F32, E4M3, 8, 1, [4300], [0], 0),
])
def test_attend_prompts_split_along_their_tokens(gpu, typ, cache_type, hk, group, rows, starts, window):
    check(gpu, typ, cache_type, hk, group, 32, rows, starts, window, 4)
    if len(rows) > 1 or window:  # and as a captured call has it, bounds far above
        check(gpu, typ, cache_type, hk, group, 32, rows, starts, window, 4, max_rows=5000, max_len=1 << 17)
