"""Attention over long 4-bit caches, so closely that one position left out or counted twice, or a part of the weights lost, is seen."""
import numpy as np
import pytest

import kv4_ref as ref
from hip_rt import Hip
from test_kv4 import _attend, _cache, _data, _store

U = ref.U


@pytest.fixture
def hip(gq):
    h = Hip(gq)
    yield h
    h.close()


def exact(q, k, v, pos, num, window, scale):
    """All rows in float64; rows without a position NaN."""
    n_seq, n_tok, nh, hd = q.shape
    y = np.full(q.shape, np.nan)
    g = nh // k.shape[2]
    for s in range(n_seq):
        for t in range(num[s]):
            p = pos[s] + t
            if not 0 <= p < k.shape[1]:
                continue
            lo = max(0, p - window + 1) if window else 0
            for h in range(k.shape[2]):
                x = q[s, t, h * g:(h + 1) * g].astype(np.float64) @ np.ascontiguousarray(k[s, lo:p + 1, h].T) * scale
                w = np.exp(x - x.max(1, keepdims=True))
                y[s, t, h * g:(h + 1) * g] = w @ v[s, lo:p + 1, h] / w.sum(1, keepdims=True)
    return y


def close(y, want, smax, n, hd):
    """The error of each row, as a part of the row, in root mean squares. With u = 2^-24, and roundings that are independent of one another:
    a score is off by about sqrt(hd) u times its products' magnitudes (their sum, the query's parts: 22 bits) and by 2 u of itself
    (the scale), a weight by that as a factor, by 4 u from its parts and by 2 u from the exponential; a row of independent values is
    off by as much of itself, plus u sqrt(n / 32) of the sums' steps and 4 u of joins and division. The largest of many rows: 4 times
    that. One position of n left out is about 1 / sqrt(n) of the row, at 9000 some 900 times the bound; the weights' lower parts are 1e-4."""
    live = ~np.isnan(want).any(-1)
    err = np.sqrt(((y - want) ** 2).mean(-1) / (want ** 2).mean(-1))[live]
    bound = 4 * U * (np.sqrt(hd) + 2 * smax + 6 + np.sqrt(n / 32) + 4)
    print(f"[kv4 long] rows {live.sum()} error {err.max():.2e} median {np.median(err):.2e} bound {bound:.2e}", flush=True)
    assert (err <= bound).all(), float(err.max() / bound)


@pytest.mark.gpu
@pytest.mark.parametrize("nh,nkv,hd", [(4, 2, 32), (6, 3, 64), (8, 2, 128), (4, 1, 256), (16, 2, 64)])
@pytest.mark.parametrize("n_tok,pos,num", [(1, [8999], [1]), (1, [8991, 31, 4128], [1, 1, 1]), (3, [8997, 4001, 127], [3, 2, 3]),
                                           (70, [5010], [70]), (33, [2047, 700], [33, 20])])
@pytest.mark.parametrize("window", [0, 2500])
def test_long_rows(gq, hip, nh, nkv, hd, n_tok, pos, num, window):
    n = 9000
    rng = np.random.default_rng(hd + n_tok)
    k, v = _data(rng, len(pos), n, nkv, hd)
    q = rng.standard_normal((len(pos), n_tok, nh, hd)).astype(np.float32)
    kv, _ = _cache(gq, hip, len(pos), n, nkv, hd)
    _store(gq, hip, kv, k, v, [0] * len(pos))
    y = _attend(gq, hip, kv, q, pos, num, window, hd ** -0.5)
    want = exact(q, ref.values(k), ref.values(v), pos, num, window, hd ** -0.5)
    smax = max(np.abs(q[s, :, h * nh // nkv:(h + 1) * nh // nkv].reshape(-1, hd) @ k[s, :, h].T).max() for s in range(len(pos)) for h in range(nkv)) * hd ** -0.5
    close(y, want, smax, n, hd)


@pytest.mark.gpu
@pytest.mark.parametrize("hd,n_tok", [(64, 1), (128, 17), (256, 1)])
def test_every_position_counts_once(gq, hip, hd, n_tok):
    """Scores of 0 and values that tell their positions apart: 1, which sets the block's scale, and +-1/2 by the bits of the position, exact in
    4 bits. Length times output is a whole number of halves, and a position that is missing or twice in the sum moves every element by a
    half at least. FP32 is off by a few u times the length. Rows of many lengths around the ends of records, and so of ranges."""
    nh, nkv, n = 4, 2, 9000
    bits = np.arange(n)[:, None] >> np.arange(14) & 1
    v = np.zeros((1, n, nkv, hd), np.float32)
    for blk in range(0, hd, 32):
        v[0, ..., blk] = 1
        v[0, ..., blk + 1:blk + 15] = (0.5 - bits)[:, None]
    kv, _ = _cache(gq, hip, 1, n, nkv, hd)
    _store(gq, hip, kv, np.ones_like(v), v, [0])
    assert np.array_equal(ref.values(v), v)
    total = np.cumsum(v[0, :, 0].astype(np.float64), 0)
    q = np.zeros((1, n_tok, nh, hd), np.float32)
    for first in (0, 30, 31, 32, 33, 127, 128, 500, 1023, 1024, 4095, 4096, 8000, n - n_tok):
        y = _attend(gq, hip, kv, q, [first], None, 0, 1.0)[0]
        for t in range(n_tok):
            assert (np.abs(y[t] * (first + t + 1.0) - total[first + t]) < 0.1).all(), (first, t)
