"""Attention over 4-bit caches with sinks, and of groups of sequences that share a prefix: against float64 at lengths around the
records' borders, windows that end in the prefix, in the sequences' own caches and in the sinks, padded and empty sequences, many
sequences, infinities where a row does not look; refusals, captured calls, and a whole step of drafted tokens."""

import numpy as np
import pytest

import kv4_ref as ref
from hip_rt import Hip
from test_kv4 import _cache, _data, _store

U = ref.U


@pytest.fixture
def hip(gq):
    h = Hip(gq)
    yield h
    h.close()


def seen_by(p, window, sinks):
    """The positions that the token at position p sees."""
    j = np.arange(p + 1)
    return j if not window else j[(j > p - window) | (j < sinks)]


def want_of(q, k, v, scale):
    """One row over the positions given: y and a bound of FP32 arithmetic's error, as in kv4_ref.attention, with two more joins of
    ranges (4 u each) in the sum."""
    s = k @ q * scale
    p = np.exp(s - s.max())
    p /= p.sum()
    ds = (q.size + 4) * U * np.max(np.abs(k) @ np.abs(q)) * abs(scale) + 4 * U * np.max(np.abs(s))
    return p @ v, (2 * ds + (2 * len(k) + 32) * U) * (p @ np.abs(v)) + 1e-30


def attend(gq, hip, kv, q, pos, num=None, window=0, sinks=0, scale=1.0, prefix=None, plen=None, stream=0):
    n_seq, n_tok, nh, hd = q.shape
    y = hip.upload(np.full(q.shape, 7.0, np.float32))
    nw = gq.kv4_attn_shared_work(kv, prefix, n_tok, nh) if prefix else gq.kv4_attn_sink_work(kv, n_tok, nh)
    rest = (hip.upload(q), nh * hd, hd, y, nh * hd, n_tok, nh, hip.upload(np.asarray(pos, np.int32)),
            hip.upload(np.asarray(num, np.int32)) if num is not None else 0, window, sinks, scale,
            hip.upload(np.full(max(nw, 16), 0xFF, np.uint8)), nw, stream)
    if prefix:
        gq.kv4_attn_shared_static(kv, prefix, hip.upload(np.asarray(plen, np.int32)), *rest)
    else:
        gq.kv4_attn_sink_static(kv, *rest)
    return hip.download(y, q.shape, np.float32)


def check(q, k, v, y, pos, num, window, sinks, scale, pk=None, pv=None, plen=None):
    """k, v: what the sequences' own caches hold, pk, pv: the prefixes'."""
    n_seq, n_tok, nh, hd = q.shape
    g = nh // k.shape[2]
    members = n_seq // len(plen) if plen is not None else 1
    for s in range(n_seq):
        n = 0 if plen is None else max(0, min(plen[s // members], pk.shape[1]))
        for t in range(n_tok):
            p = pos[s] + t
            if t >= (n_tok if num is None else num[s]) or p < 0 or p >= k.shape[1]:
                assert (y[s, t] == 7.0).all(), (s, t)
                continue
            j = seen_by(n + p, window, sinks)
            for h in range(nh):
                kk, vv = k[s, j[j >= n] - n, h // g], v[s, j[j >= n] - n, h // g]
                if n:
                    kk, vv = (np.concatenate([a[s // members, j[j < n], h // g], b]) for a, b in ((pk, kk), (pv, vv)))
                want, tol = want_of(q[s, t, h].astype(np.float64), kk, vv, scale)
                err = np.abs(y[s, t, h] - want)
                assert (err <= tol).all(), (s, t, h, p, float((err / tol).max()))


HEADS = [(4, 1, 32), (6, 3, 64), (8, 2, 128), (4, 1, 256), (20, 1, 64), (2, 2, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("nh,nkv,hd", HEADS)
@pytest.mark.parametrize("n_tok,first", [(1, 0), (1, 31), (1, 517), (3, 30), (40, 100), (70, 0)])
@pytest.mark.parametrize("window,sinks", [(0, 4), (33, 0), (33, 4), (1, 1), (100, 70), (64, 1000), (32, 32)])
def test_sinks(gq, hip, nh, nkv, hd, n_tok, first, window, sinks):
    print(f"[kv4 sinks] heads {nh}/{nkv} dim {hd} tokens {n_tok} at {first} window {window} sinks {sinks}", flush=True)
    rng = np.random.default_rng(n_tok + first)
    n = first + n_tok
    k, v = _data(rng, 2, n, nkv, hd)
    q = (1.5 * rng.standard_normal((2, n_tok, nh, hd))).astype(np.float32)
    kv, _ = _cache(gq, hip, 2, n + 3, nkv, hd)  # past the tokens: NaN scales
    _store(gq, hip, kv, k, v, [0, 0])
    y = attend(gq, hip, kv, q, [first, first], None, window, sinks, hd ** -0.5)
    check(q, ref.values(k), ref.values(v), y, [first, first], None, window, sinks, hd ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 128), (4, 1, 256), (6, 3, 64), (4, 2, 32)])
def test_sinks_long_and_ragged(gq, hip, nh, nkv, hd):
    """Sequences of very unlike lengths in one call, one not in use, one past its end, one with a single position."""
    n_ctx = 9000
    pos, num = [8997, 0, -1, 4001, 8999, 70], [3, 1, 3, 2, 3, 0]
    rng = np.random.default_rng(5)
    k, v = _data(rng, len(pos), n_ctx, nkv, hd)
    q = rng.standard_normal((len(pos), 3, nh, hd)).astype(np.float32)
    kv, _ = _cache(gq, hip, len(pos), n_ctx, nkv, hd)
    _store(gq, hip, kv, k, v, [0] * len(pos), [9000, 1, 9000, 4003, 9000, 0])
    for window, sinks in ((2500, 4), (2500, 3000), (100, 1), (8999, 200)):
        y = attend(gq, hip, kv, q, pos, num, window, sinks, hd ** -0.5)
        check(q, ref.values(k), ref.values(v), y, pos, num, window, sinks, hd ** -0.5)


def shared(gq, hip, groups, members, n_tok, heads, prefix_ctx, own_ctx, plen, pos, num, windows, seed=0, fill=0xFF):
    nh, nkv, hd = heads
    rng = np.random.default_rng(seed)
    n_seq = groups * members
    pk, pv = _data(rng, groups, prefix_ctx, nkv, hd)
    k, v = _data(rng, n_seq, own_ctx, nkv, hd)
    q = (1.5 * rng.standard_normal((n_seq, n_tok, nh, hd))).astype(np.float32)
    prefix, _ = _cache(gq, hip, groups, prefix_ctx, nkv, hd, fill)
    kv, _ = _cache(gq, hip, n_seq, own_ctx, nkv, hd, fill)
    _store(gq, hip, prefix, pk, pv, [0] * groups, np.clip(plen, 0, prefix_ctx))  # NaN behind the prefixes
    last = [max(0, min(p + (n_tok if num is None else num[s]), own_ctx)) for s, p in enumerate(pos)]  # (tokens of p < 0 may have places)
    _store(gq, hip, kv, k, v, [0] * n_seq, last)
    vals = [ref.values(x) for x in (k, v, pk, pv)]
    for window, sinks in windows:
        y = attend(gq, hip, kv, q, pos, num, window, sinks, hd ** -0.5, prefix, plen)
        check(q, vals[0], vals[1], y, pos, num, window, sinks, hd ** -0.5, vals[2], vals[3], plen)


@pytest.mark.gpu
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("n_tok", [1, 5, 37])
@pytest.mark.parametrize("plen,own", [(1, 0), (32, 31), (100, 32), (515, 3), (0, 70), (33, 200)])
def test_shared(gq, hip, heads, n_tok, plen, own):
    print(f"[kv4 shared] heads {heads} tokens {n_tok} prefix {plen} own {own}", flush=True)
    pos = [own, max(own - 7, 0), own, own + 2, 0, own]
    shared(gq, hip, 2, 3, n_tok, heads, 520, own + n_tok + 2, [plen, max(plen - 5, 0)], pos, None,
           [(0, 0), (40, 0), (40, 3), (plen + 10, 2), (7, 90), (3, plen + 2)], plen + own)


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [(8, 2, 128), (4, 1, 256), (8, 8, 64), (6, 2, 32)])
@pytest.mark.parametrize("members", [1, 4, 17])
def test_shared_long_and_ragged(gq, hip, heads, members):
    """Prefixes of very unlike lengths, empty ones and one that ends past its cache; sequences not in use, a group of them, tokens past
    the end of their caches."""
    rng = np.random.default_rng(members)
    groups, own_ctx = 5, 700
    plen = [4000, 0, 333, 4000, 5000]
    pos = rng.integers(-2, own_ctx, groups * members)
    pos[2 * members:3 * members] = -5  # nobody reads the third prefix
    num = rng.integers(0, 4, groups * members)
    num[0] = 3
    pos[0] = own_ctx - 2
    shared(gq, hip, groups, members, 3, heads, 4000, own_ctx, plen, [int(p) for p in pos], [int(n) for n in num],
           [(0, 0), (900, 0), (900, 5), (300, 64), (4500, 1)], 1)


@pytest.mark.gpu
@pytest.mark.parametrize("groups,members", [(1, 64), (64, 1), (65, 1), (1, 65), (33, 4), (2, 100)])
def test_shared_of_many_sequences(gq, hip, groups, members):
    """More sequences or groups than a wave looks at in one go."""
    rng = np.random.default_rng(groups)
    n = groups * members
    shared(gq, hip, groups, members, 2, (4, 2, 64), 400, 90, [int(x) for x in rng.integers(0, 401, groups)],
           [int(x) for x in rng.integers(-1, 90, n)], [int(x) for x in rng.integers(0, 3, n)], [(0, 0), (100, 0), (60, 33)], 2)


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [(4, 1, 256), (8, 2, 128), (4, 4, 32)])
def test_shared_equals_the_whole_cache(gq, hip, heads):
    """The same positions in one cache and split into prefix and own: within both bounds of each other, with 300 tokens."""
    nh, nkv, hd = heads
    rng = np.random.default_rng(9)
    n, plen, n_tok = 900, 555, 300
    k, v = _data(rng, 1, n, nkv, hd)
    q = rng.standard_normal((1, n_tok, nh, hd)).astype(np.float32)
    whole, _ = _cache(gq, hip, 1, n, nkv, hd)
    prefix, _ = _cache(gq, hip, 1, plen, nkv, hd)
    own, _ = _cache(gq, hip, 1, n - plen, nkv, hd)
    _store(gq, hip, whole, k, v, [0])
    _store(gq, hip, prefix, k[:, :plen], v[:, :plen], [0])
    _store(gq, hip, own, k[:, plen:], v[:, plen:], [0])
    a = attend(gq, hip, whole, q, [n - n_tok], None, 400, 10, hd ** -0.5)
    b = attend(gq, hip, own, q, [n - n_tok - plen], None, 400, 10, hd ** -0.5, prefix, [plen])
    kk, vv = ref.values(k), ref.values(v)
    check(q, kk, vv, a, [n - n_tok], None, 400, 10, hd ** -0.5)
    check(q, kk[:, plen:], vv[:, plen:], b, [n - n_tok - plen], None, 400, 10, hd ** -0.5, kk[:, :plen], vv[:, :plen], [plen])


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [32, 128, 256])
def test_infinities_reach_only_the_rows_that_see_them(gq, hip, hd):
    """Values beyond fp16's range (infinite scales) at a sink, in the prefix's middle and in one sequence's own cache."""
    nh, nkv, plen, own = 4, 2, 200, 50
    rng = np.random.default_rng(11)
    pk, pv = _data(rng, 1, plen, nkv, hd)
    k, v = _data(rng, 2, own, nkv, hd)
    q = rng.standard_normal((2, 1, nh, hd)).astype(np.float32)
    pv[0, 1, 0, :32] = 3e6
    pv[0, 100, 1, :32] = -3e6
    v[1, 20, 0, :32] = 3e6
    prefix, _ = _cache(gq, hip, 1, plen, nkv, hd)
    kv, _ = _cache(gq, hip, 2, own, nkv, hd)
    _store(gq, hip, prefix, pk, pv, [0])
    _store(gq, hip, kv, k, v, [0, 0])
    for window, sinks, hurt in ((0, 0, {0: (0, 1), 1: (0, 1)}), (120, 0, {1: (0,)}), (120, 1, {1: (0,)}), (120, 2, {0: (0,), 1: (0,)}), (160, 0, {0: (1,), 1: (0, 1)}),
                                (20, 0, {}), (20, 102, {0: (0, 1), 1: (0, 1)})):
        y = attend(gq, hip, kv, q, [own - 1, own - 1], None, window, sinks, 0.1, prefix, [plen])
        for s in range(2):
            for h in range(nh):
                bad = h // 2 in hurt.get(s, ())
                assert np.isfinite(y[s, 0, h, 32:]).all()
                assert np.isnan(y[s, 0, h, :32]).all() if bad else np.isfinite(y[s, 0, h, :32]).all(), (window, sinks, s, h)


@pytest.mark.gpu
def test_strides(gq, hip):
    """Queries interleaved with gates, rows apart from one another; y rows apart, what is between them untouched."""
    nh, nkv, hd, n_tok, plen, own = 4, 2, 64, 5, 100, 40
    rng = np.random.default_rng(7)
    pk, pv = _data(rng, 1, plen, nkv, hd)
    k, v = _data(rng, 2, own, nkv, hd)
    prefix, _ = _cache(gq, hip, 1, plen, nkv, hd)
    kv, _ = _cache(gq, hip, 2, own, nkv, hd)
    _store(gq, hip, prefix, pk, pv, [0])
    _store(gq, hip, kv, k, v, [0, 0])
    qrow, yrow = nh * 2 * hd + 8, nh * hd + 4
    q = np.full((2, n_tok, qrow), np.nan, np.float32)
    plain = rng.standard_normal((2, n_tok, nh, hd)).astype(np.float32)
    q[:, :, :nh * 2 * hd].reshape(2, n_tok, nh, 2, hd)[:, :, :, 0] = plain
    y = hip.upload(np.full((2, n_tok, yrow), 7.0, np.float32))
    pos = [own - n_tok, 3]
    nw = gq.kv4_attn_shared_work(kv, prefix, n_tok, nh)
    gq.kv4_attn_shared_static(kv, prefix, hip.upload(np.int32([plen])), hip.upload(q), qrow, 2 * hd, y, yrow, n_tok, nh,
                              hip.upload(np.asarray(pos, np.int32)), 0, 0, 0, 0.1, hip.alloc(nw), nw)
    got = hip.download(y, (2, n_tok, yrow), np.float32)
    assert (got[:, :, nh * hd:] == 7.0).all()
    check(plain, ref.values(k), ref.values(v), got[:, :, :nh * hd].reshape(2, n_tok, nh, hd), pos, None, 0, 0, 0.1, ref.values(pk), ref.values(pv), [plen])


@pytest.mark.gpu
def test_graph_and_streams(gq, hip):
    """Calls captured once, replayed at other positions and prefix lengths with eager calls on another stream between; every replay
    gives the bits of the eager call."""
    nh, nkv, hd, plen, own = 8, 2, 128, 900, 300
    rng = np.random.default_rng(8)
    pk, pv = _data(rng, 2, plen, nkv, hd)
    k, v = _data(rng, 4, own, nkv, hd)
    q = rng.standard_normal((4, 1, nh, hd)).astype(np.float32)
    streams = [hip.stream(), hip.stream()]
    side = []
    for _ in range(2):
        prefix, _ = _cache(gq, hip, 2, plen, nkv, hd)
        kv, _ = _cache(gq, hip, 4, own, nkv, hd)
        nw, ns = gq.kv4_attn_shared_work(kv, prefix, 1, nh), gq.kv4_attn_sink_work(kv, 1, nh)
        side.append((prefix, kv, hip.upload(q), hip.alloc(q.nbytes), hip.alloc(q.nbytes), hip.alloc(16), hip.alloc(8), hip.alloc(nw), nw, hip.alloc(ns), ns))
        _store(gq, hip, prefix, pk, pv, [0, 0])
        _store(gq, hip, kv, k, v, [0] * 4)

    def step(s, stream):
        prefix, kv, qd, y, y2, pos, ln, work, nw, work2, ns = s
        gq.kv4_attn_shared_static(kv, prefix, ln, qd, nh * hd, hd, y, nh * hd, 1, nh, pos, 0, 700, 4, 0.1, work, nw, stream)
        gq.kv4_attn_sink_static(kv, qd, nh * hd, hd, y2, nh * hd, 1, nh, pos, 0, 100, 4, 0.1, work2, ns, stream)

    graph = hip.capture(streams[0], lambda: step(side[0], streams[0]))
    vals = [ref.values(x) for x in (k, v, pk, pv)]
    for i in range(4):
        pos, ln = [i, 60 * i, 299 - i, 150], [900 - 250 * i, 31 * i]
        for s in side:
            hip.write(s[5], np.asarray(pos, np.int32))
            hip.write(s[6], np.asarray(ln, np.int32))
        hip.launch(graph, streams[0])
        step(side[1], streams[1])
        for which in (3, 4):
            got = [hip.download(s[which], q.shape, np.float32) for s in side]
            assert np.array_equal(got[0].view(np.uint32), got[1].view(np.uint32))
            if which == 3:
                check(q, vals[0], vals[1], got[0], pos, None, 700, 4, 0.1, vals[2], vals[3], ln)
            else:
                check(q, vals[0], vals[1], got[0], pos, None, 100, 4, 0.1)


@pytest.mark.gpu
def test_a_step_of_drafted_tokens(gq, hip):
    """The calls of a step together: queries and keys turned, keys and values stored behind the prefix, attention with sinks, and the
    drafted tokens verified on logits made of its outputs."""
    nh, nkv, hd, groups, members, n_tok, vocab, plen = 4, 2, 64, 2, 3, 4, 500, [150, 77]
    rng = np.random.default_rng(12)
    n_seq, own = groups * members, 40
    pk, pv = _data(rng, groups, 160, nkv, hd)
    k, v = _data(rng, n_seq, own, nkv, hd)
    pos = [int(p) for p in rng.integers(0, own - n_tok, n_seq)]
    q = rng.standard_normal((n_seq, n_tok, nh, hd)).astype(np.float32)
    kn, vn = _data(rng, n_seq, n_tok, nkv, hd)
    head = (rng.standard_normal((nh * hd, vocab)) / 8).astype(np.float32)
    prefix, _ = _cache(gq, hip, groups, 160, nkv, hd)
    kv, _ = _cache(gq, hip, n_seq, own, nkv, hd)
    _store(gq, hip, prefix, pk, pv, [0] * groups, plen)
    _store(gq, hip, kv, k, v, [0] * n_seq, pos)
    # the tokens' places behind the prefixes: positions for the angles, places for the caches
    at = np.int32([plen[s // members] + pos[s] for s in range(n_seq)])
    freqs = gq.rope_freqs(hd, 1e4)
    dq, dk = hip.upload(q), hip.upload(kn)
    dpos = hip.upload(np.int32(pos))
    gq.rope_static([gq.RopeRows(dq, dq, nh * hd, hd, nh * hd, hd, nh), gq.RopeRows(dk, dk, nkv * hd, hd, nkv * hd, hd, nkv)], n_seq, n_tok, hd, hd,
                   gq.ROPE_HALF, hip.upload(freqs), hip.upload(at))
    gq.kv4_store_static(kv, dk, hip.upload(vn), nkv * hd, n_tok, dpos)
    y = hip.alloc(q.nbytes)
    nw = gq.kv4_attn_shared_work(kv, prefix, n_tok, nh)
    gq.kv4_attn_shared_static(kv, prefix, hip.upload(np.int32(plen)), dq, nh * hd, hd, y, nh * hd, n_tok, nh, dpos, 0, 120, 5, hd ** -0.5, hip.alloc(nw), nw)
    got = hip.download(y, q.shape, np.float32)
    qt, kt = hip.download(dq, q.shape, np.float32), hip.download(dk, kn.shape, np.float32)
    for x, z in ((q, qt), (kn, kt)):  # against the formula in 64 bits (angles below 200 turns: 1e-13; three roundings)
        for s in range(n_seq):
            a = np.outer(at[s] + np.arange(n_tok), 1e4 ** (-2 * np.arange(hd // 2) / hd))[:, None]
            x0, x1 = x[s, ..., :hd // 2].astype(float), x[s, ..., hd // 2:].astype(float)
            want = np.concatenate([x0 * np.cos(a) - x1 * np.sin(a), x0 * np.sin(a) + x1 * np.cos(a)], -1)
            size = np.concatenate([np.abs(x0) + np.abs(x1)] * 2, -1)
            assert (np.abs(z[s] - want) <= (3.01 * U + 1e-12) * size).all()
    for s in range(n_seq):
        k[s, pos[s]:pos[s] + n_tok], v[s, pos[s]:pos[s] + n_tok] = kt[s], vn[s]
    check(qt, ref.values(k), ref.values(v), got, pos, None, 120, 5, hd ** -0.5, ref.values(pk), ref.values(pv), plen)
    logits = (got.reshape(n_seq, n_tok, -1) @ head).astype(np.float32)
    token = logits[:, :-1].argmax(-1).astype(np.int32)
    token[::2, 1] = (token[::2, 1] + 1) % vocab  # every other sequence loses its second token
    na, out, lp = hip.alloc(4 * n_seq), hip.alloc(4 * n_seq * n_tok), hip.alloc(4 * n_seq * n_tok)
    nw = gq.draft_work(n_seq, n_tok - 1, vocab)
    gq.draft_verify_static(hip.upload(logits), vocab, 0, 0, vocab, n_seq, n_tok - 1, hip.upload(token), 0, 0, 0.0, 1.0, na, out, lp, hip.alloc(nw), nw)
    na, out = hip.download(na, (n_seq,), np.int32), hip.download(out, (n_seq, n_tok), np.int32)
    best = logits.argmax(-1)
    for s in range(n_seq):
        m = 1 if s % 2 == 0 else n_tok - 1
        assert na[s] == m and np.array_equal(out[s, :m + 1], best[s, :m + 1]) and (out[s, m + 1:] == -1).all()


def test_refusals(gq):
    """Arguments that are refused before anything is launched (no device is touched)."""
    lib, P = gq.hip_lib(), 1 << 20

    def kv(data=P, n_seq=4, n_ctx=4096, nkv=2, hd=64):
        return gq.Kv4(data, n_seq, n_ctx, nkv, hd)

    a = dict(kv=kv(), q=P, qs=256, qh=64, y=P, ys=256, n_tok=4, nh=4, pos=P, num=0, window=0, sinks=0, scale=1.0, work=P, nw=1 << 40)
    need, need2 = lib.gemvq_kv4_attn_sink_work(kv(), 4, 4), lib.gemvq_kv4_attn_shared_work(kv(), kv(n_seq=2), 4, 4)
    assert need > 0 and need2 > 0
    bad = [dict(kv=None), dict(kv=kv(0)), dict(kv=kv(P + 128)), dict(kv=kv(hd=96)), dict(q=0), dict(q=P + 4), dict(qs=62), dict(qh=60), dict(qh=66), dict(y=0),
           dict(y=P + 8), dict(ys=252), dict(ys=258), dict(n_tok=0), dict(n_tok=65536), dict(nh=0), dict(nh=3), dict(pos=0),
           dict(num=P + 2), dict(window=-1), dict(sinks=-1), dict(work=0), dict(work=P + 8), dict(n_tok=1 << 13, nh=256, ys=64 << 8)]
    for b in bad + [dict(nw=need - 1)]:
        x = {**a, **b}
        assert lib.gemvq_kv4_attn_sink_static(*x.values(), 0) == gq.EINVAL, b
    ok = dict(kv=kv(), prefix=kv(n_seq=2), plen=P, **{k: v for k, v in a.items() if k != "kv"})
    bad += [dict(prefix=None), dict(prefix=kv(0, 2)), dict(prefix=kv(P + 4, 2)), dict(prefix=kv(n_seq=3)), dict(prefix=kv(n_seq=8)), dict(prefix=kv(n_seq=2, nkv=1)),
            dict(prefix=kv(n_seq=2, hd=128)), dict(prefix=kv(n_seq=2, n_ctx=0)), dict(plen=0), dict(plen=P + 2), dict(nw=need2 - 1)]
    for b in bad:
        x = {**ok, **b}
        assert lib.gemvq_kv4_attn_shared_static(*x.values(), 0) == gq.EINVAL, b
    assert lib.gemvq_kv4_attn_sink_work(kv(), 1 << 13, 256) == 0 and lib.gemvq_kv4_attn_shared_work(kv(), kv(n_seq=3), 4, 4) == 0
    with pytest.raises(gq.GemvqError):
        gq.kv4_attn_sink_static(kv(0), P, 256, 64, P, 256, 4, 4, P)
    with pytest.raises(gq.GemvqError):
        gq.kv4_attn_shared_static(kv(), kv(n_seq=3), P, P, 256, 64, P, 256, 4, 4, P)


@pytest.mark.gpu
def test_far_into_large_caches(gq, hip):
    """A prefix of which the last KV heads lie beyond 4 GiB, seen by its sinks and a window at its end."""
    nh, nkv, hd, plen, window, sinks = 8, 8, 256, 2200000, 60, 3
    rng = np.random.default_rng(13)
    nb = gq.kv4_bytes(1, plen, nkv, hd)
    assert nb // nkv * (nkv - 1) > 4 << 30
    prefix = gq.Kv4(hip.alloc(nb), 1, plen, nkv, hd)
    kv, _ = _cache(gq, hip, 2, 40, nkv, hd)
    tail = 70
    pk, pv = _data(rng, 1, sinks + tail, nkv, hd)
    k, v = _data(rng, 2, 40, nkv, hd)
    q = rng.standard_normal((2, 2, nh, hd)).astype(np.float32)
    _store(gq, hip, prefix, pk[:, :sinks], pv[:, :sinks], [0])
    _store(gq, hip, prefix, pk[:, sinks:], pv[:, sinks:], [plen - tail])
    _store(gq, hip, kv, k, v, [0, 0])
    pos = [0, 30]
    y = attend(gq, hip, kv, q, pos, None, window, sinks, hd ** -0.5, prefix, [plen])
    kk, vv, ppk, ppv = (ref.values(x) for x in (k, v, pk, pv))
    for s in range(2):
        for t in range(2):
            p = pos[s] + t
            first = plen + p - window + 1  # of the window: some of it in the prefix
            from_prefix = np.concatenate([np.arange(sinks), sinks + tail - (plen - first) + np.arange(plen - first)])
            for h in range(nh):
                want, tol = want_of(q[s, t, h].astype(np.float64), np.concatenate([ppk[0, from_prefix, h], kk[s, :p + 1, h]]),
                                    np.concatenate([ppv[0, from_prefix, h], vv[s, :p + 1, h]]), hd ** -0.5)
                assert (np.abs(y[s, t, h] - want) <= tol).all(), (s, t, h)


@pytest.mark.gpu
def test_numbers_of_tokens_that_are_too_large(gq, hip):
    """num above n_tok counts as n_tok; prefix lengths below 0 as none."""
    shared(gq, hip, 2, 2, 2, (4, 2, 64), 100, 50, [-5, 60], [3, 10, 0, 44], [2, 2, 2, 2], [(0, 0), (30, 2)], 3)
    nh, nkv, hd = 4, 2, 64
    rng = np.random.default_rng(14)
    k, v = _data(rng, 2, 60, nkv, hd)
    q = rng.standard_normal((2, 2, nh, hd)).astype(np.float32)
    kv, _ = _cache(gq, hip, 2, 60, nkv, hd)
    _store(gq, hip, kv, k, v, [0, 0])
    y = attend(gq, hip, kv, q, [20, 50], [9, 70000], 16, 2, 0.1)
    check(q, ref.values(k), ref.values(v), y, [20, 50], None, 16, 2, 0.1)
