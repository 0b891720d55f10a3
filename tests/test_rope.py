"""Rotary positions on caller-owned memory: the table against its formulas, turned rows against extended precision, strides, rows
that stay, in place, refusals, captured calls."""
import ctypes as C
import math

import numpy as np
import pytest

from hip_rt import Hip

U = 2.0 ** -24  # half a step of FP32, relative


@pytest.fixture
def hip(gq):
    h = Hip(gq)
    yield h
    h.close()


def turned(x, at, freqs, n_rot, layout):
    """Rows x [tokens, heads, dim] at positions `at`, in extended precision, and a bound of the error: three roundings to FP32 of each
    product (of the cosine or sine, of itself, of the sum; the sum's counted for both), the 64-bit product of position and
    frequency (half a step of it, in turns) and 1e-12 for the series."""
    half = n_rot // 2
    turn = np.asarray(at, np.longdouble)[:, None] * freqs[:half].astype(np.longdouble)
    off = 2 * math.pi * np.abs(turn).astype(np.float64) * 2.0 ** -53 + 1e-12
    a = (turn - np.rint(turn)).astype(np.longdouble) * (2 * np.longdouble(math.pi) + np.longdouble(2.4492935982947064e-16))
    c, s = (f(a)[:, None] * freqs[half] for f in (np.cos, np.sin))
    i0, i1 = (np.arange(half), half + np.arange(half)) if layout == 0 else (2 * np.arange(half), 2 * np.arange(half) + 1)
    x = x.astype(np.longdouble)
    y, tol = x.copy(), np.zeros(x.shape)
    x0, x1 = x[..., i0], x[..., i1]
    y[..., i0], y[..., i1] = x0 * c - x1 * s, x0 * s + x1 * c
    for i, (p, q) in ((i0, (c, s)), (i1, (s, c))):
        tol[..., i] = 3.01 * U * (np.abs(x0 * p) + np.abs(x1 * q)) + off[:, None] * abs(freqs[half]) * (np.abs(x0) + np.abs(x1)) + 1e-37
    return y.astype(np.float64), tol


def rotate(gq, hip, xs, n_rot, layout, freqs, pos, num=None, pad=0, in_place=False, stream=0):
    """xs: arrays [seqs, tokens, heads, dim]; pad: floats between heads and behind rows (NaN, and 7 in the outputs)."""
    rows, outs = [], []
    for x in xs:
        s, t, h, d = x.shape
        buf = np.full((s, t, h * (d + pad) + pad), np.nan, np.float32)
        buf[..., :h * (d + pad)].reshape(s, t, h, d + pad)[..., :d] = x
        px = hip.upload(buf)
        py = px if in_place else hip.upload(np.full(buf.shape, 7.0, np.float32))
        rows.append(gq.RopeRows(px, py, buf.shape[2], d + pad, buf.shape[2], d + pad, h))
        outs.append((py, buf.shape, x.shape))
    s, t, _, d = xs[0].shape
    gq.rope_static(rows, s, t, d, n_rot, layout, hip.upload(freqs), hip.upload(np.asarray(pos, np.int32)),
                   hip.upload(np.asarray(num, np.int32)) if num is not None else 0, stream)
    got = []
    for py, shape, (s, t, h, d) in outs:
        y = hip.download(py, shape, np.float32)
        inner = y[..., :h * (d + pad)].reshape(s, t, h, d + pad)
        if pad:
            rest = np.concatenate([inner[..., d:].ravel(), y[..., h * (d + pad):].ravel()])
            assert np.isnan(rest).all() if in_place else (rest == 7.0).all()
        got.append(inner[..., :d].copy())
    return got


def check(xs, got, n_rot, layout, freqs, pos, num, in_place=False):
    for x, y in zip(xs, got):
        for s in range(x.shape[0]):
            n = x.shape[1] if num is None else max(0, min(num[s], x.shape[1]))
            live = np.array([t < n and pos[s] + t >= 0 for t in range(x.shape[1])])
            assert (y[s, ~live] == (x[s, ~live] if in_place else 7.0)).all()
            want, tol = turned(x[s, live], (pos[s] + np.arange(x.shape[1]))[live], freqs, n_rot, layout)
            assert np.array_equal(y[s, live][..., n_rot:], x[s, live][..., n_rot:])
            err = np.abs(y[s, live] - want)
            assert (err <= tol).all(), (s, float((err / np.maximum(tol, 1e-300)).max()))


DIMS = [(256, 64), (128, 128), (64, 58), (4, 2), (32, 10), (1024, 1024), (20, 6), (96, 96), (256, 8)]


@pytest.mark.gpu
@pytest.mark.parametrize("dim,n_rot", DIMS)
@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n_tok,pos,num", [(1, [0, 131071, 77], None), (5, [3, -2, 2 ** 31 - 6], [5, 5, 0]), (70, [1, 0, 2 ** 20], [70, 1, 33])])
def test_rope(gq, hip, dim, n_rot, layout, in_place, n_tok, pos, num):
    print(f"[rope] {n_rot} of {dim}, layout {layout}, tokens {n_tok}, in place {in_place}", flush=True)
    rng = np.random.default_rng(dim + n_tok)
    xs = [rng.standard_normal((3, n_tok, h, dim)).astype(np.float32) for h in (5, 2)]
    freqs = gq.rope_freqs(n_rot, 1e4, 4.0, 4096)
    got = rotate(gq, hip, xs, n_rot, layout, freqs, pos, num, 4 if n_tok == 5 else 0, in_place)
    check(xs, got, n_rot, layout, freqs, pos, num, in_place)


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [(1,), (3, 1, 2, 7), (40,), (300, 1)])
@pytest.mark.parametrize("n_tok", [1, 9, 2000])
def test_arrays_and_heads(gq, hip, heads, n_tok):
    """One to four arrays in a launch, from a single head to hundreds, few rows and many."""
    if sum(heads) * n_tok > 100000:
        n_tok = 300
    rng = np.random.default_rng(n_tok)
    xs = [rng.standard_normal((1, n_tok, h, 64)).astype(np.float32) for h in heads]
    freqs = gq.rope_freqs(32, 1e6)
    check(xs, rotate(gq, hip, xs, 32, 0, freqs, [100], None), 32, 0, freqs, [100], None)


@pytest.mark.gpu
def test_graph_and_streams(gq, hip):
    """A call captured once and replayed at other positions, with eager ones on another stream between; the same bits."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((4, 1, 6, 128)).astype(np.float32)
    freqs = gq.rope_freqs(128, 1e6)
    a, b = hip.stream(), hip.stream()
    pos, tab, px = hip.alloc(16), hip.upload(freqs), hip.upload(x)
    py = [hip.alloc(x.nbytes) for _ in range(2)]
    rows = [[gq.RopeRows(px, p, 768, 128, 768, 128, 6)] for p in py]
    graph = hip.capture(a, lambda: gq.rope_static(rows[0], 4, 1, 128, 128, 1, tab, pos, 0, a))
    for i in range(4):
        at = [i, 1000 * i, 77, 2 ** 20 + i]
        hip.write(pos, np.asarray(at, np.int32))
        hip.launch(graph, a)
        gq.rope_static(rows[1], 4, 1, 128, 128, 1, tab, pos, 0, b)
        got = [hip.download(p, x.shape, np.float32) for p in py]
        assert np.array_equal(got[0].view(np.uint32), got[1].view(np.uint32))
        check([x], [got[0]], 128, 1, freqs, at, None)


def test_table(gq):
    """Against the formulas, in plain Python floats: a few roundings of 2^-53 each, the power's among them (16)."""
    for n_rot, base, factor, ctx, fast, slow, factors in [(64, 1e7, 1.0, 0, 32, 1, None), (128, 1e4, 8.0, 0, 32, 1, None), (128, 1e6, 4.0, 32768, 32, 1, None),
                                                          (10, 1e4, 2.0, 4096, 32, 1, None), (2, 1e4, 16.0, 8192, 64, 2, None),
                                                          (64, 5e5, 2.0, 8192, 32, 1, [1 + i / 7 for i in range(32)])]:
        got = gq.rope_freqs(n_rot, base, factor, ctx, fast, slow, factors)
        lo, hi = (n_rot * math.log(ctx / (2 * math.pi * b)) / (2 * math.log(base)) if ctx else 0 for b in (fast, slow))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), n_rot - 1)
        for i in range(n_rot // 2):
            w = base ** (-2 * i / n_rot) / (factors[i] if factors else 1)
            ramp = min(max((i - lo) / max(hi - lo, 1e-3), 0), 1) if ctx else 1
            want = ((1 - ramp) * w + ramp * w / factor) / (2 * math.pi)
            assert abs(got[i] - want) <= 16 * 2.0 ** -53 * want
        assert abs(got[-1] - (0.1 * math.log(factor) + 1 if ctx else 1)) <= 4 * 2.0 ** -53


def test_refusals(gq):
    """Arguments that are refused before anything is launched (no device is touched)."""
    lib, P = gq.hip_lib(), 1 << 20
    out = np.zeros(600)
    ok = dict(n_rot=64, base=1e4, factor=1.0, ctx=0, fast=32.0, slow=1.0, factors=None, out=out.ctypes.data)
    assert lib.gemvq_rope_freqs(*ok.values()) == 0
    bad_factor = np.ones(32)
    bad_factor[3] = 0
    for b in (dict(n_rot=0), dict(n_rot=63), dict(n_rot=1026), dict(n_rot=-2), dict(base=1.0), dict(base=math.nan), dict(base=math.inf), dict(factor=0.0),
              dict(factor=-1.0), dict(factor=math.inf), dict(ctx=-1), dict(ctx=4096, slow=0.0), dict(ctx=4096, fast=0.5),
              dict(ctx=4096, fast=math.inf), dict(out=None), dict(factors=bad_factor.ctypes.data)):
        assert lib.gemvq_rope_freqs(*{**ok, **b}.values()) == gq.EINVAL, b
    with pytest.raises(gq.GemvqError):
        gq.rope_freqs(64, 1e4, factors=[1.0])

    def rows(x=P, y=P * 2, xr=1024, xh=128, yr=1024, yh=128, h=8):
        return gq.RopeRows(x, y, xr, xh, yr, yh, h)

    ok = dict(arrays=[rows()], n_seq=2, n_tok=3, dim=128, n_rot=64, layout=0, freqs=P, pos=P, num=P)
    bad = [dict(arrays=[rows(**b)]) for b in (dict(x=0), dict(y=0), dict(x=P + 4), dict(y=P + 8), dict(xr=124), dict(xr=1022), dict(xh=126), dict(xh=64),
                                              dict(yr=64), dict(yh=130), dict(yh=-128), dict(h=0), dict(h=65536), dict(y=P, yr=2048),
                                              dict(xr=1 << 41))]
    bad += [dict(arrays=[rows()] * 5), dict(arrays=[rows(h=40000)] * 2), dict(n_seq=0), dict(n_tok=0), dict(n_seq=1 << 16, n_tok=1 << 15), dict(n_seq=1 << 12, n_tok=1 << 12), dict(dim=0),
            dict(dim=126, n_rot=64), dict(dim=1028), dict(n_rot=0), dict(n_rot=63), dict(n_rot=130), dict(layout=2), dict(layout=-1),
            dict(freqs=0), dict(freqs=P + 4), dict(pos=0), dict(pos=P + 2), dict(num=P + 1)]
    for b in bad:
        a = {**ok, **b}
        arr = (gq.RopeRows * len(a["arrays"]))(*a["arrays"])
        assert lib.gemvq_rope_static(arr, len(arr), *list(a.values())[1:], 0) == gq.EINVAL, b
    arr = (gq.RopeRows * 1)(rows())
    assert lib.gemvq_rope_static(None, 1, *list(ok.values())[1:], 0) == gq.EINVAL
    assert lib.gemvq_rope_static(arr, 0, *list(ok.values())[1:], 0) == gq.EINVAL
    with pytest.raises(gq.GemvqError):
        gq.rope_static([rows(h=0)], 1, 1, 128, 64, 0, P, P)
    assert C.sizeof(gq.RopeRows) == 56
