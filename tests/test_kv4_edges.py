"""Attention over the 4-bit cache at the ends of its numbers: scores of any finite size, weights far below the largest,
infinities and NaN where a row does not look."""
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


@pytest.mark.gpu
@pytest.mark.parametrize("nh,nkv,hd", [(4, 2, 32), (8, 2, 128), (4, 1, 256)])
@pytest.mark.parametrize("size", [1e6, 3e8, 1e10, 1e15, 1e25, 1e33, 1e36, "one element"])
@pytest.mark.parametrize("first,n_tok", [(0, 6), (700, 1)])
def test_scores_of_any_size(gq, hip, nh, nkv, hd, size, first, n_tok):
    """Scores so far apart that a token's output is the value of its best position, and so large that a rounding of one is many powers of e.
    FP32 sums of hd products and the query in two parts leave a score off by (hd + 8) u times its products' magnitudes: heads whose two best
    positions are not further apart than that are left out. The value comes back as a weight of 1 in two parts (22 bits) times quants
    and scale, over the sum of weights: a few u."""
    rng = np.random.default_rng(hd)
    n = first + n_tok
    k, v = _data(rng, 1, n, nkv, hd)
    q = rng.standard_normal((1, n_tok, nh, hd)).astype(np.float32)
    if size == "one element":  # up to the end of FP32's range
        q *= 0
        q[..., 3] = rng.uniform(1.1e38, 3.4e38, q.shape[:-1]) * rng.choice([-1, 1], q.shape[:-1])
        k *= np.float32(1e-3)
    else:
        q *= np.float32(size)
    kv, _ = _cache(gq, hip, 1, n, nkv, hd)
    _store(gq, hip, kv, k, v, [0])
    scale = hd ** -0.5
    y = _attend(gq, hip, kv, q, [first], None, 0, scale)
    kk, vv = ref.values(k)[0], ref.values(v)[0]
    seen = 0
    for t in range(n_tok):
        for h in range(nh):
            x = kk[:first + t + 1, h * nkv // nh]
            s = x @ q[0, t, h].astype(np.float64) * scale
            off = (hd + 8) * U * (np.abs(x) @ np.abs(q[0, t, h].astype(np.float64))).max() * scale
            best = int(s.argmax())
            if (np.delete(s, best) > s[best] - 2 * off - 30).any():
                continue
            seen += 1
            want = vv[best, h * nkv // nh]
            assert (np.abs(y[0, t, h] - want) <= 16 * U * np.abs(want)).all(), (t, h, y[0, t, h], want)
    assert seen >= nh // 2


@pytest.mark.gpu
@pytest.mark.parametrize("hd,n_tok", [(32, 1), (64, 40), (128, 1), (128, 20), (256, 3)])
@pytest.mark.parametrize("at", [11, 500])
def test_a_dominant_position_without_values(gq, hip, hd, n_tok, at):
    """One position far above all others, whose values are zero: the output is made of the others' weights alone. All of them are equal, so
    what rounding leaves of one adds up. A weight is held no finer than 2^-31 of the largest (off by half of that), a weight times a
    value scale no finer than 2^-24 beside a largest product of at least 2^7 * 2^6 (8 quants of the largest scale: 2^-35 of the values)."""
    nh, nkv, n = 8, 2, 700
    rng = np.random.default_rng(hd)
    first = n - n_tok
    k = np.zeros((1, n, nkv, hd), np.float32)
    v = rng.uniform(0.5, 1.5, (1, n, nkv, hd)).astype(np.float32)
    k[0, at, :, 3], v[0, at] = 1, 0
    q = rng.standard_normal((1, n_tok, nh, hd)).astype(np.float32)
    q[..., 3] = np.linspace(9, 22, n_tok * nh).reshape(n_tok, nh)  # how far above, in nats
    kv, _ = _cache(gq, hip, 1, n, nkv, hd)
    _store(gq, hip, kv, k, v, [0])
    y = _attend(gq, hip, kv, q, [first], None, 0, 1.0)
    kk, vv = ref.values(k)[0], ref.values(v)[0]
    for t in range(n_tok):
        for h in range(nh):
            g = h * nkv // nh
            want, tol = ref.attention(q[0, t, h].astype(np.float64), kk[:, g], vv[:, g], first + t, 0, 1.0)
            seen = vv[:first + t + 1, g]
            tol = tol + 2.0 ** -32 * seen.sum(0) + 2.0 ** -35 * len(seen) * seen.max()
            assert (np.abs(y[0, t, h] - want) <= tol).all(), (t, h, float((np.abs(y[0, t, h] - want) / tol).max()))


@pytest.mark.gpu
@pytest.mark.parametrize("nh,nkv,hd,n_tok", [(4, 2, 32, 70), (6, 2, 64, 33), (8, 2, 128, 20), (4, 1, 256, 9)])
@pytest.mark.parametrize("first,window", [(0, 0), (45, 0), (0, 7), (600, 33), (9, 900)])
def test_infinities_and_nan_out_of_sight(gq, hip, nh, nkv, hd, n_tok, first, window):
    """Keys and values of later tokens, and of positions behind a token's window, that are infinite, NaN or too large for an fp16 scale: the
    tokens that do not see them come out as if they were not there, the others not finite where they are."""
    rng = np.random.default_rng(n_tok + first)
    n = first + n_tok
    k, v = _data(rng, 1, n, nkv, hd)
    q = rng.standard_normal((1, n_tok, nh, hd)).astype(np.float32)
    bad_v, bad_k = {first + n_tok // 2: (np.inf, 3), first + n_tok - 2: (np.nan, 31)}, {first + n_tok - 1: np.nan}
    if window:
        bad_v[max(first - 3, 0)] = (-3e6, 0)
    kv, _ = _cache(gq, hip, 1, n, nkv, hd)
    clean_k, clean_v = k.copy(), v.copy()
    for p, (x, e) in bad_v.items():
        v[0, p, :, e] = x
    for p, x in bad_k.items():
        k[0, p] = x
    _store(gq, hip, kv, k, v, [0])
    y = _attend(gq, hip, kv, q, [first], None, window, hd ** -0.5)[0]
    kk, vv = ref.values(clean_k)[0], ref.values(clean_v)[0]
    for t in range(n_tok):
        p = first + t
        seen = range(max(0, p - window + 1) if window else 0, p + 1)
        for h in range(nh):
            if any(x in seen for x in bad_k):
                assert np.isnan(y[t, h]).all()
                continue
            want, tol = ref.attention(q[0, t, h].astype(np.float64), kk[:, h * nkv // nh], vv[:, h * nkv // nh], p, window, hd ** -0.5)
            fine = np.ones(hd, bool)
            if any(x in seen for x in bad_v):
                fine[:32] = False
                assert not np.isfinite(y[t, h, :32]).all()
            assert (np.abs(y[t, h] - want) <= tol)[fine].all(), (t, h)
