"""Verification of drafted tokens on caller-owned memory: against float64 with ragged sequences, masks and the values at the ends of
FP32; certain drafts, temperature 0, sampling without a draft; the distribution of what comes out; refusals, captured calls."""
import numpy as np
import pytest

from hip_rt import Hip

INF = np.inf


@pytest.fixture
def hip(gq):
    h = Hip(gq)
    yield h
    h.close()


def clean(x):
    return np.minimum(np.where(np.isnan(x), -INF, x).astype(np.float64), float(np.finfo(np.float32).max))


def dist(x, temp):
    """A row's distribution, None for one of nothing but -inf."""
    x = clean(x)
    if x.max() == -INF:
        return None
    e = np.exp((x - x.max()) / (temp or 1.0))
    return e / e.sum()


def reference(target, draft, token, num, uniform, temp, dtemp):
    """n_accept, out and logp; sequences not in use at 7."""
    s, k1, n = target.shape
    k = k1 - 1
    n_accept, out, logp = np.full(s, 7), np.full((s, k1), 7), np.full((s, k1), 7.0)
    for i in range(s):
        m = k if num is None else min(num[i], k)
        if m < 0:
            continue
        out[i], logp[i] = -1, 0
        for a in range(m + 1):
            p = dist(target[i, a], temp)
            w = p
            if p is None or a == m:
                break
            d = token[i, a]
            inside = 0 <= d < n
            if temp == 0:
                if d != p.argmax():
                    break
            else:
                q = np.zeros(n)
                if draft is not None:
                    q = dist(draft[i, a], dtemp)
                    q = np.zeros(n) if q is None else q
                elif inside:
                    q[d] = 1
                if not inside or not uniform[i, a] * q[d] < p[d]:
                    w = np.maximum(p - q, 0)
                    w = w if w.sum() > 0 else p
                    break
            out[i, a], logp[i, a] = d, np.log(p[d])
        n_accept[i] = a
        if w is not None:
            if temp == 0:
                new = int(w.argmax())
            else:
                c = np.cumsum(w)
                at = int(np.searchsorted(c, float(uniform[i, k]) * c[-1], side="right"))
                new = at if at < n and w[at] > 0 else int(np.flatnonzero(w > 0)[-1])
            out[i, a], logp[i, a] = new, np.log(p[new])
    return n_accept, out, logp


def verify(gq, hip, target, draft, token, num, uniform, temp=1.0, dtemp=1.0, skew=0, stream=0):
    """skew: floats that rows start past a 16-byte line, and that lie between rows."""
    s, k1, n = target.shape

    def rows(x):
        buf = np.full(x.shape[0] * x.shape[1] * (n + skew) + 8, np.nan, np.float32)
        for r, row in enumerate(x.reshape(-1, n)):
            buf[skew + r * (n + skew):][:n] = row
        return hip.upload(buf) + 4 * skew

    outs = [hip.upload(np.full(m, 7, t)) for m, t in ((s, np.int32), (s * k1, np.int32), (s * k1, np.float32))]
    nw = gq.draft_work(s, k1 - 1, n)
    assert nw > 0
    gq.draft_verify_static(rows(target), n + skew, rows(draft) if draft is not None else 0, n + skew, n, s, k1 - 1,
                           hip.upload(np.asarray(token, np.int32)), hip.upload(np.asarray(num, np.int32)) if num is not None else 0,
                           hip.upload(np.asarray(uniform, np.float32)), temp, dtemp, *outs, hip.upload(np.full(nw, 0xFF, np.uint8)), nw, stream)
    return hip.download(outs[0], (s,), np.int32), hip.download(outs[1], (s, k1), np.int32), hip.download(outs[2], (s, k1), np.float32)


def check(got, want):
    assert np.array_equal(got[0], want[0]), (got[0], want[0])
    assert np.array_equal(got[1], want[1]), (got[1], want[1])
    # One rounding to FP32 (half a step), and a sum of exponentials each of which is 2^(N / 256) (1 + E), |E| < 2^-9, with E formed in
    # FP32: its argument r + e (|.| < 2^-8.9) is rounded by 2^-34, times ln 2; the slope g (0.69) by 2^-25 and its constants by 2^-25,
    # times 2^-9; the product by 2^-34: 2^-34 (0.7 + 1 + 1 + 1) < 2.2e-10. A sum of such terms, and its logarithm, is off by no more.
    assert (np.abs(got[2] - want[2]) <= 2.0 ** -24 * np.abs(want[2]) + 2.2e-10).all()


def inputs(rng, s, k, n, noise=1.0, temp=1.0):
    target = (2.5 * rng.standard_normal((s, k + 1, n))).astype(np.float32)
    draft = (target[:, :k] + noise * rng.standard_normal((s, k, n))).astype(np.float32)
    token = np.zeros((s, k), np.int32)
    for i in range(s):
        for t in range(k):
            c = np.cumsum(dist(draft[i, t], temp))
            token[i, t] = min(np.searchsorted(c, rng.random() * c[-1], side="right"), n - 1)
    return target, draft, token, rng.random((s, k + 1)).astype(np.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("s,k,n", [(1, 4, 1), (3, 1, 7), (2, 3, 255), (5, 2, 2048), (4, 4, 2049), (3, 5, 8193), (1, 32, 1000), (40, 8, 9001),
                                   (2, 4, 151936), (12, 4, 151936), (1, 2, 1 << 20), (1000, 3, 50), (7, 0, 5000), (1, 0, 151936)])
@pytest.mark.parametrize("skew", [0, 3])
def test_verification(gq, hip, s, k, n, skew):
    print(f"[draft] {s} x {k} of {n}, skew {skew}", flush=True)
    rng = np.random.default_rng(n + skew)
    x = inputs(rng, s, k, n)
    num = rng.integers(-1, k + 2, s) if s > 2 else None
    check(verify(gq, hip, x[0], x[1], x[2], num, x[3], skew=skew), reference(*x[:3], num, x[3], 1.0, 1.0))
    check(verify(gq, hip, x[0], None, x[2], num, x[3], 0.7, skew=skew), reference(x[0], None, x[2], num, x[3], 0.7, 1.0))
    check(verify(gq, hip, x[0], x[1], x[2], num, x[3], 0.0, skew=skew), reference(*x[:3], num, x[3], 0.0, 1.0))


@pytest.mark.gpu
@pytest.mark.parametrize("temp,dtemp", [(0.5, 1.0), (1.0, 0.25), (3.0, 2.0), (0.01, 0.01), (100.0, 100.0)])
def test_temperatures(gq, hip, temp, dtemp):
    rng = np.random.default_rng(4)
    x = inputs(rng, 20, 4, 5000, temp=dtemp)
    check(verify(gq, hip, x[0], x[1], x[2], None, x[3], temp, dtemp), reference(*x[:3], None, x[3], temp, dtemp))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [300, 20000])
@pytest.mark.parametrize("what", ["same", "masked", "masked token", "all masked", "draft all masked", "one left", "nan", "inf", "extremes", "outside",
                                  "u 0", "u 1", "u above 1", "certain and sure", "equal logits", "wide"])
def test_edges(gq, hip, what, n):
    print(f"[draft] {what} of {n}", flush=True)
    rng = np.random.default_rng(5)
    s, k = 6, 3
    target, draft, token, u = inputs(rng, s, k, n)
    num, with_draft = [3, 3, 2, 0, -1, 3], True
    if what == "same":  # every token is accepted
        draft = target[:, :k].copy()
    elif what == "masked":
        target[:, :, rng.random(n) < 0.9] = -INF
    elif what == "masked token":
        np.put_along_axis(target[:, :k], token[..., None].astype(np.int64), -INF, -1)
    elif what == "all masked":
        target[0, 0] = target[1, 1] = target[2, 2] = target[3, 0] = -INF
    elif what == "draft all masked":
        draft[:] = -INF
    elif what == "one left":
        target[:] = -INF
        target[..., n - 1] = -3.0
        token[0] = n - 1
    elif what == "nan":
        target[rng.random(target.shape) < 0.3] = np.nan
        draft[rng.random(draft.shape) < 0.3] = np.nan
        target[0, 0] = np.nan
    elif what == "inf":
        target[:, :, 5] = INF
        target[1, :, 9] = INF
        draft[:, :, 9] = INF
    elif what == "extremes":
        target *= np.float32(1e37)
        draft *= np.float32(1e37)
    elif what == "outside":
        token[0], token[1], token[2], token[5] = -1, n, 2 ** 31 - 1, -2 ** 31
    elif what == "u 0":
        u[:] = 0
    elif what == "u 1":
        u[:] = 1
    elif what == "u above 1":
        u[:] = 1.5
    elif what == "certain and sure":  # the one token with a probability, refused by a number of 1
        with_draft, u[:] = False, 1.0
        target[:] = -INF
        target[:, :, 4] = 1.0
        token[:] = 4
    elif what == "equal logits":
        target[:], draft[:] = 1.5, -2.0
    elif what == "wide":  # probabilities down to e^-600
        target *= 50
        draft *= 50
    d = draft if with_draft else None
    check(verify(gq, hip, target, d, token, num, u), reference(target, d, token, num, u, 1.0, 1.0))
    check(verify(gq, hip, target, None, token, num, u), reference(target, None, token, num, u, 1.0, 1.0))
    check(verify(gq, hip, target, d, token, num, u, 0.0), reference(target, d, token, num, u, 0.0, 1.0))


@pytest.mark.gpu
@pytest.mark.parametrize("certain", [False, True])
def test_tokens_are_distributed_as_the_targets(gq, hip, certain):
    """Two drafted tokens of 13000 sequences with one and the same model, whose rows do not depend on the tokens before: the first two
    tokens that come out are draws from the target's rows. Counts stay within 5.5 standard deviations (4e-8 for one of them, 16 of
    them). A certain token is accepted with p(d) and else another one, so the first token out is p's draw whatever d is."""
    rng = np.random.default_rng(6)
    s, n = 13000, 8
    row = (1.5 * rng.standard_normal((3, n))).astype(np.float32)
    drow = (1.5 * rng.standard_normal((2, n))).astype(np.float32)
    token = np.stack([rng.choice(n, s, p=dist(drow[t], 1.0)) for t in range(2)], 1).astype(np.int32)
    u = rng.random((s, 3)).astype(np.float32)
    target, draft = np.broadcast_to(row, (s, 3, n)), np.broadcast_to(drow, (s, 2, n))
    n_accept, out, _ = verify(gq, hip, target, None if certain else draft, token, None, u)
    for t in range(2):
        some = out[n_accept >= t, t]  # sequences that have a token there
        p = dist(row[t], 1.0)
        got = np.bincount(some, minlength=n)
        assert (np.abs(got - len(some) * p) <= 5.5 * np.sqrt(len(some) * p * (1 - p))).all(), (t, got, len(some) * p)


@pytest.mark.gpu
def test_graph_and_streams(gq, hip):
    """A call captured once and replayed with other logits and numbers, with eager ones on another stream between."""
    rng = np.random.default_rng(8)
    s, k, n = 4, 3, 30000
    a, b = hip.stream(), hip.stream()
    nw = gq.draft_work(s, k, n)
    sides = [[hip.alloc(m) for m in (4 * s * (k + 1) * n, 4 * s * k * n, 4 * s * k, 4 * s * (k + 1), 4 * s, 4 * s * (k + 1), 4 * s * (k + 1), nw)]
             for _ in range(2)]

    def call(side, stream):
        t, d, tok, u, na, out, lp, w = side
        gq.draft_verify_static(t, n, d, n, n, s, k, tok, 0, u, 0.9, 1.0, na, out, lp, w, nw, stream)

    graph = hip.capture(a, lambda: call(sides[0], a))
    for _ in range(4):
        x = inputs(rng, s, k, n)
        for side in sides:
            for p, v in zip(side, x):
                hip.write(p, v)
        hip.launch(graph, a)
        call(sides[1], b)
        want = reference(*x[:3], None, x[3], 0.9, 1.0)
        for side in sides:
            check((hip.download(side[4], (s,), np.int32), hip.download(side[5], (s, k + 1), np.int32), hip.download(side[6], (s, k + 1), np.float32)),
                  want)


@pytest.mark.gpu
def test_without_log_probabilities(gq, hip):
    rng = np.random.default_rng(9)
    x = inputs(rng, 3, 2, 700)
    na, out = hip.alloc(12), hip.alloc(36)
    nw = gq.draft_work(3, 2, 700)
    gq.draft_verify_static(hip.upload(x[0]), 700, hip.upload(x[1]), 700, 700, 3, 2, hip.upload(x[2]), 0, hip.upload(x[3]), 1.0, 1.0, na, out, 0,
                           hip.alloc(nw), nw)
    want = reference(*x[:3], None, x[3], 1.0, 1.0)
    assert np.array_equal(hip.download(na, (3,), np.int32), want[0]) and np.array_equal(hip.download(out, (3, 3), np.int32), want[1])


def test_refusals(gq):
    """Arguments that are refused before anything is launched (no device is touched)."""
    lib, P = gq.hip_lib(), 1 << 20
    for bad in ((0, 1, 10), (1, -1, 10), (1, 33, 10), (1, 1, 0), (1, 1, (1 << 20) + 1), (22000, 1, 10), (1 << 30, 32, 10)):
        assert gq.draft_work(*bad) == 0
    assert gq.draft_work(65535, 0, 10) > 0
    ok = dict(target=P, ts=1000, draft=P, ds=1000, n=1000, s=2, k=3, token=P, num=P, uniform=P, temp=1.0, dtemp=1.0, n_accept=P, out=P, logp=P,
              work=P, nw=1 << 40)
    nan = float("nan")
    for b in (dict(target=0), dict(target=P + 2), dict(ts=999), dict(ts=1 << 41), dict(draft=P + 1), dict(ds=999), dict(n=0), dict(n=(1 << 20) + 1), dict(s=0),
              dict(s=30000), dict(k=-1), dict(k=33), dict(token=0), dict(token=P + 2), dict(num=P + 2), dict(uniform=0), dict(uniform=P + 1),
              dict(temp=-1.0), dict(temp=nan), dict(temp=INF), dict(dtemp=0.0), dict(dtemp=nan), dict(dtemp=-2.0), dict(n_accept=0), dict(n_accept=P + 2),
              dict(out=0), dict(out=P + 1), dict(logp=P + 2), dict(work=0), dict(work=P + 8), dict(nw=gq.draft_work(2, 3, 1000) - 1)):
        assert lib.gemvq_draft_verify_static(*{**ok, **b}.values(), 0) == gq.EINVAL, b
    with pytest.raises(gq.GemvqError):
        gq.draft_verify_static(0, 10, 0, 10, 10, 1, 1, P, 0, P, 1.0, 1.0, P, P, P, P, 1 << 20)


@pytest.mark.gpu
def test_rows_far_apart(gq, hip):
    """Rows 2 GiB apart: the last ones beyond 32 bits of bytes and of floats."""
    rng = np.random.default_rng(10)
    s, k, n = 2, 2, 3000
    x = inputs(rng, s, k, n)
    stride = (1 << 29) + 64
    big = hip.alloc(4 * (5 * stride + n))
    for r in range(6):
        hip.write(big + 4 * r * stride, x[0].reshape(6, n)[r])
    na, out, lp = hip.alloc(8), hip.alloc(24), hip.alloc(24)
    nw = gq.draft_work(s, k, n)
    gq.draft_verify_static(big, stride, hip.upload(x[1]), n, n, s, k, hip.upload(x[2]), 0, hip.upload(x[3]), 1.0, 1.0, na, out, lp, hip.alloc(nw), nw)
    check((hip.download(na, (s,), np.int32), hip.download(out, (s, k + 1), np.int32), hip.download(lp, (s, k + 1), np.float32)),
          reference(*x[:3], None, x[3], 1.0, 1.0))


@pytest.mark.gpu
def test_calls_at_once(gq, hip):
    """Calls on two streams with workspaces of their own, many times over, do not disturb one another."""
    rng = np.random.default_rng(11)
    s, k, n = 6, 3, 9000
    streams = [hip.stream(), hip.stream()]
    sides, wants = [], []
    for _ in range(2):
        x = inputs(rng, s, k, n)
        nw = gq.draft_work(s, k, n)
        sides.append([hip.upload(x[0]), hip.upload(x[1]), hip.upload(x[2]), hip.upload(x[3]), hip.alloc(4 * s), hip.alloc(4 * s * (k + 1)),
                      hip.alloc(4 * s * (k + 1)), hip.alloc(nw), nw])
        wants.append(reference(*x[:3], None, x[3], 1.0, 1.0))
    for _ in range(20):
        for (t, d, tok, u, na, out, lp, w, nw), stream in zip(sides, streams):
            gq.draft_verify_static(t, n, d, n, n, s, k, tok, 0, u, 1.0, 1.0, na, out, lp, w, nw, stream)
    for (_, _, _, _, na, out, lp, _, _), want in zip(sides, wants):
        check((hip.download(na, (s,), np.int32), hip.download(out, (s, k + 1), np.int32), hip.download(lp, (s, k + 1), np.float32)), want)
