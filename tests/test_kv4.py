"""The 4-bit KV cache on caller-owned memory: stored bytes and values, attention against float64, refusals, padded and empty
sequences, strides, other streams, captured calls."""
import ctypes as C

import numpy as np
import pytest

import kv4_ref as ref
from hip_rt import Hip


@pytest.fixture
def hip(gq):
    h = Hip(gq)
    yield h
    h.close()


def _cache(gq, hip, n_seq, n_ctx, nkv, hd, fill=0xFF):
    """A cache full of bytes that are NaN as scales."""
    nb = gq.kv4_bytes(n_seq, n_ctx, nkv, hd)
    return gq.Kv4(hip.upload(np.full(nb, fill, np.uint8)), n_seq, n_ctx, nkv, hd), nb


def _store(gq, hip, kv, k, v, pos, num=None, stream=0):
    n_seq, n_tok = k.shape[:2]
    row = int(np.prod(k.shape[2:]))
    gq.kv4_store_static(kv, hip.upload(k), hip.upload(v), row, n_tok, hip.upload(np.asarray(pos, np.int32)),
                        hip.upload(np.asarray(num, np.int32)) if num is not None else 0, stream)


def _attend(gq, hip, kv, q, pos, num=None, window=0, scale=1.0, stream=0):
    n_seq, n_tok, nh, hd = q.shape
    y = hip.upload(np.full(q.shape, 7.0, np.float32))
    nw = gq.kv4_attn_work(kv, n_tok, nh)
    gq.kv4_attn_static(kv, hip.upload(q), nh * hd, hd, y, nh * hd, n_tok, nh, hip.upload(np.asarray(pos, np.int32)),
                       hip.upload(np.asarray(num, np.int32)) if num is not None else 0, window, scale,
                       hip.upload(np.full(max(nw, 16), 0xFF, np.uint8)), nw, stream)
    return hip.download(y, q.shape, np.float32)


def _data(rng, n_seq, n, nkv, hd):
    gain = np.exp(0.3 * rng.standard_normal((2, nkv, hd)))
    return [(rng.standard_normal((n_seq, n, nkv, hd)) * gain[i]).astype(np.float32) for i in range(2)]


def _check(q, k, v, y, pos, num, window, scale):
    """Rows of live tokens against float64 (k and v: all positions' stored values), the others left at 7."""
    n_seq, n_tok, nh, hd = q.shape
    g = nh // k.shape[2]
    for s in range(n_seq):
        for t in range(n_tok):
            p = pos[s] + t
            if t >= num[s] or p < 0 or p >= k.shape[1]:
                assert (y[s, t] == 7.0).all()
                continue
            for h in range(nh):
                want, tol = ref.attention(q[s, t, h].astype(np.float64), k[s, :, h // g], v[s, :, h // g], p, window, scale)
                err = np.abs(y[s, t, h] - want)
                assert (err <= tol).all(), (s, t, h, p, float((err / tol).max()))


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("n_tok,pos,num", [(1, [0, 37, 63], None), (1, [95, -1, 5], None), (70, [0, 3, 32], None),
                                           (33, [31, 64, 90], [33, 0, 20]), (5, [-2, 94, 60], [5, 5, 3])])
def test_store_writes_its_bytes_alone(gq, hip, hd, n_tok, pos, num):
    n_seq, n_ctx, nkv = 3, 96, 2
    print(f"[kv4 store] hd {hd} tokens {n_tok} pos {pos} num {num}", flush=True)
    rng = np.random.default_rng(1)
    k, v = _data(rng, n_seq, n_tok, nkv, hd)
    k[0, 0, 0, :32] = 0  # a block of zeros
    v[0, 0, 0, :32] = np.where(np.arange(32) % 2, 1.5, -1.5)  # the largest magnitude with both signs: the first decides
    kv, nb = _cache(gq, hip, n_seq, n_ctx, nkv, hd, 0xA5)
    _store(gq, hip, kv, k, v, pos, num)
    want = np.full((n_seq, nkv, n_ctx // 32, 36 * hd), 0xA5, np.uint8)
    for s in range(n_seq):
        for t in range(n_tok if num is None else num[s]):
            if 0 <= pos[s] + t < n_ctx:
                for h in range(nkv):
                    ref.put(want[s, h, (pos[s] + t) // 32], (pos[s] + t) % 32, k[s, t, h], v[s, t, h])
    got = hip.download(kv.data, want.shape, np.uint8)
    assert np.array_equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("n_ctx,n_tok,pos,num", [(100, 40, [2, 59], [40, 33]), (700, 400, [33, 299], [400, 395]), (400, 400, [0, 31], [400, 17])])
def test_load_gives_what_was_stored(gq, hip, hd, n_ctx, n_tok, pos, num):
    n_seq, nkv = 2, 3
    rng = np.random.default_rng(2)
    k, v = _data(rng, n_seq, n_tok, nkv, hd)
    kv, _ = _cache(gq, hip, n_seq, n_ctx, nkv, hd)
    _store(gq, hip, kv, k, v, pos, num)
    row = nkv * hd + 12  # rows with room between them, which stays as it was
    out = [hip.upload(np.full((n_seq, n_tok, row), 7.0, np.float32)) for _ in range(2)]
    gq.kv4_load_static(kv, *out, row, n_tok, hip.upload(np.asarray(pos, np.int32)), hip.upload(np.asarray(num, np.int32)))
    for x, p in zip((k, v), out):
        got = hip.download(p, (n_seq, n_tok, row), np.float32)
        assert (got[:, :, nkv * hd:] == 7.0).all()
        want = ref.values(x)
        for s in range(n_seq):
            assert np.array_equal(got[s, :num[s], :nkv * hd], want[s, :num[s]].reshape(num[s], -1).astype(np.float32))
            assert (got[s, num[s]:] == 7.0).all()


SHAPES = [(4, 1, 32), (6, 3, 64), (8, 2, 128), (4, 1, 256), (2, 2, 128), (20, 1, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("nh,nkv,hd", SHAPES)
@pytest.mark.parametrize("n_tok,first", [(1, 0), (1, 31), (1, 32), (1, 517), (3, 30), (17, 100), (40, 0)])
@pytest.mark.parametrize("window", [0, 33])
def test_attention(gq, hip, nh, nkv, hd, n_tok, first, window):
    print(f"[kv4 attention] heads {nh}/{nkv} dim {hd} tokens {n_tok} at {first} window {window}", flush=True)
    rng = np.random.default_rng(n_tok + first)
    n = first + n_tok
    k, v = _data(rng, 2, n, nkv, hd)
    q = (1.5 * rng.standard_normal((2, n_tok, nh, hd))).astype(np.float32)
    kv, _ = _cache(gq, hip, 2, n + 3, nkv, hd)  # past the tokens: NaN scales
    pos = [first, first]
    _store(gq, hip, kv, k, v, [0, 0])
    y = _attend(gq, hip, kv, q, pos, None, window, hd ** -0.5)
    _check(q, ref.values(k), ref.values(v), y, pos, [n_tok] * 2, window, hd ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 128), (4, 1, 256), (6, 3, 64), (4, 2, 32)])
def test_attention_long_and_ragged(gq, hip, nh, nkv, hd):
    """Sequences of very unlike lengths in one call, one not in use, one past its end, one with a single position."""
    n_ctx, n_tok = 9000, 3
    pos, num = [8997, 0, -1, 4001, 8999, 70], [3, 1, 3, 2, 3, 0]
    rng = np.random.default_rng(5)
    k, v = _data(rng, len(pos), n_ctx, nkv, hd)
    q = rng.standard_normal((len(pos), n_tok, nh, hd)).astype(np.float32)
    kv, _ = _cache(gq, hip, len(pos), n_ctx, nkv, hd)
    _store(gq, hip, kv, k, v, [0] * len(pos), [9000, 1, 9000, 4003, 9000, 0])
    for window in (0, 2500):
        y = _attend(gq, hip, kv, q, pos, num, window, hd ** -0.5)
        _check(q, ref.values(k), ref.values(v), y, pos, [3, 1, 3, 2, 3, 0], window, hd ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("n_seq,n_ctx", [(64, 600), (65, 90), (150, 600)])
def test_attention_of_many_sequences(gq, hip, n_seq, n_ctx):
    """More sequences than a wave looks at in one go, some without tokens, with one range or several each."""
    nh, nkv, hd = 4, 2, 128
    rng = np.random.default_rng(n_seq)
    k, v = _data(rng, n_seq, n_ctx, nkv, hd)
    q = rng.standard_normal((n_seq, 2, nh, hd)).astype(np.float32)
    kv, _ = _cache(gq, hip, n_seq, n_ctx, nkv, hd)
    _store(gq, hip, kv, k, v, [0] * n_seq)
    for most in (n_ctx, 40):
        pos = [int(p) for p in rng.integers(-1, most, n_seq)]
        num = [int(n) for n in rng.integers(0, 3, n_seq)]
        y = _attend(gq, hip, kv, q, pos, num, 0, hd ** -0.5)
        _check(q, ref.values(k), ref.values(v), y, pos, num, 0, hd ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["large scores", "tiny values", "huge values", "one value block far above"])
def test_attention_ranges(gq, hip, what):
    """Scores of hundreds, value scales at both ends of fp16's range, and one position whose values dwarf the others'."""
    nh, nkv, hd, n = 4, 2, 64, 300
    rng = np.random.default_rng(6)
    k, v = _data(rng, 1, n, nkv, hd)
    q = rng.standard_normal((1, 1, nh, hd)).astype(np.float32)
    if what == "large scores":
        q *= 100
    elif what == "tiny values":
        v *= np.float32(2.0 ** -12)  # scales of about 2^-14, fp16's smallest normal number
    elif what == "huge values":
        v *= np.float32(50000)
    else:
        v[0, 17] *= np.float32(10000)
    kv, _ = _cache(gq, hip, 1, n, nkv, hd)
    _store(gq, hip, kv, k, v, [0])
    y = _attend(gq, hip, kv, q, [n - 1], None, 0, hd ** -0.5)
    _check(q, ref.values(k), ref.values(v), y, [n - 1], [1], 0, hd ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 256])
def test_keys_with_an_outlier_channel(gq, hip, hd):
    """One key channel far above the others of its block, which become zeros, and small in the queries."""
    nh, nkv, n = 4, 2, 200
    rng = np.random.default_rng(16)
    k, v = _data(rng, 1, n, nkv, hd)
    q = rng.standard_normal((1, 1, nh, hd)).astype(np.float32)
    k[..., 5::32] *= 100
    q[..., 5::32] *= np.float32(0.01)
    kv, _ = _cache(gq, hip, 1, n, nkv, hd)
    _store(gq, hip, kv, k, v, [0])
    y = _attend(gq, hip, kv, q, [n - 1], None, 0, hd ** -0.5)
    _check(q, ref.values(k), ref.values(v), y, [n - 1], [1], 0, hd ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, -0.0, -0.2, 1e-30, 30.0])
def test_attention_scales(gq, hip, scale):
    """A scale of either sign, none at all (the mean of the values), and ends of its range."""
    nh, nkv, hd, n = 4, 2, 128, 210
    rng = np.random.default_rng(17)
    k, v = _data(rng, 1, n, nkv, hd)
    q = rng.standard_normal((1, 3, nh, hd)).astype(np.float32)
    q[0, 1] = 0
    kv, _ = _cache(gq, hip, 1, n, nkv, hd)
    _store(gq, hip, kv, k, v, [0])
    y = _attend(gq, hip, kv, q, [n - 3], None, 0, scale)
    scale = float(np.float32(scale))
    for t in range(3):
        for h in range(nh):
            # the bound takes the scale's magnitude
            want, tol = ref.attention(np.sign(scale) * q[0, t, h].astype(np.float64), ref.values(k)[0, :, h // 2], ref.values(v)[0, :, h // 2], n - 3 + t, 0,
                                      abs(scale))
            assert (np.abs(y[0, t, h] - want) <= tol).all(), (t, h)


@pytest.mark.gpu
def test_attention_strides(gq, hip):
    """Queries interleaved with gates, rows apart from one another; y rows apart, what is between them untouched."""
    nh, nkv, hd, n_tok, n = 4, 2, 64, 5, 130
    rng = np.random.default_rng(7)
    k, v = _data(rng, 2, n, nkv, hd)
    kv, _ = _cache(gq, hip, 2, n, nkv, hd)
    _store(gq, hip, kv, k, v, [0, 0])
    qrow, yrow = nh * 2 * hd + 8, nh * hd + 4
    q = np.full((2, n_tok, qrow), np.nan, np.float32)
    plain = rng.standard_normal((2, n_tok, nh, hd)).astype(np.float32)
    q[:, :, :nh * 2 * hd].reshape(2, n_tok, nh, 2, hd)[:, :, :, 0] = plain
    y = hip.upload(np.full((2, n_tok, yrow), 7.0, np.float32))
    pos = [n - n_tok, 3]
    nw = gq.kv4_attn_work(kv, n_tok, nh)
    gq.kv4_attn_static(kv, hip.upload(q), qrow, 2 * hd, y, yrow, n_tok, nh, hip.upload(np.asarray(pos, np.int32)), 0, 0, 0.1,
                       hip.alloc(nw), nw)
    got = hip.download(y, (2, n_tok, yrow), np.float32)
    assert (got[:, :, nh * hd:] == 7.0).all()
    _check(plain, ref.values(k), ref.values(v), got[:, :, :nh * hd].reshape(2, n_tok, nh, hd), pos, [n_tok] * 2, 0, 0.1)


@pytest.mark.gpu
def test_decode_in_a_graph_and_on_streams(gq, hip):
    """A store and its attention captured once, replayed at other positions with eager calls on another stream between; every
    replay gives the bits of the eager call."""
    nh, nkv, hd, n = 8, 2, 128, 700
    rng = np.random.default_rng(8)
    k, v = _data(rng, 2, n, nkv, hd)
    q = rng.standard_normal((2, 1, nh, hd)).astype(np.float32)
    streams = [hip.stream(), hip.stream()]
    side = []
    for _ in range(2):
        kv, _ = _cache(gq, hip, 2, n, nkv, hd)
        nw = gq.kv4_attn_work(kv, 1, nh)
        side.append((kv, hip.alloc(8 * nkv * hd), hip.alloc(8 * nkv * hd), hip.upload(q), hip.alloc(q.nbytes), hip.alloc(8),
                     hip.alloc(nw), nw))
        _store(gq, hip, kv, k[:, :600], v[:, :600], [0, 0])

    def step(s, stream):
        kv, kn, vn, qd, y, pos, work, nw = s
        gq.kv4_store_static(kv, kn, vn, nkv * hd, 1, pos, 0, stream)
        gq.kv4_attn_static(kv, qd, nh * hd, hd, y, nh * hd, 1, nh, pos, 0, 0, 0.1, work, nw, stream)

    graph = hip.capture(streams[0], lambda: step(side[0], streams[0]))
    for i in range(4):
        for s in side:
            hip.write(s[1], k[:, 600 + i])
            hip.write(s[2], v[:, 600 + i])
            hip.write(s[5], np.full(2, 600 + i, np.int32))
        hip.launch(graph, streams[0])
        step(side[1], streams[1])
        got = [hip.download(s[4], q.shape, np.float32) for s in side]
        assert np.array_equal(got[0].view(np.uint32), got[1].view(np.uint32))
        _check(q, ref.values(k), ref.values(v), got[0], [600 + i] * 2, [1, 1], 0, 0.1)


def test_sizes(gq):
    assert gq.kv4_bytes(1, 1, 1, 32) == 36 * 32
    assert gq.kv4_bytes(3, 33, 2, 128) == 3 * 2 * 2 * 36 * 128
    assert gq.kv4_bytes(1, 2 ** 31 - 1, 1, 256) == 2 ** 26 * 36 * 256
    for bad in ((0, 1, 1, 32), (1, 0, 1, 32), (1, 1, 0, 32), (1, 1, 1, 48), (1, 1, 1, 512), (65536, 1, 1, 32), (1, 1, 65536, 32)):
        assert gq.kv4_bytes(*bad) == 0


def test_refusals(gq):
    """Arguments that are refused before anything is launched (no device is touched)."""
    lib, P = gq.hip_lib(), 1 << 20

    def kv(data=P, n_seq=2, n_ctx=64, nkv=2, hd=64):
        return gq.Kv4(data, n_seq, n_ctx, nkv, hd)

    rows = dict(kv=kv(), k=P, v=P, row=128, n_tok=4, pos=P, num=P)
    bad = [dict(kv=None), dict(kv=kv(0)), dict(kv=kv(P + 128)), dict(kv=kv(n_seq=0)), dict(kv=kv(n_ctx=0)), dict(kv=kv(nkv=0)),
           dict(kv=kv(hd=48)), dict(kv=kv(n_seq=65536)), dict(k=0), dict(v=0), dict(k=P + 4), dict(v=P + 8), dict(row=124),
           dict(row=130), dict(row=-128), dict(n_tok=0), dict(n_tok=65536), dict(pos=0), dict(pos=P + 2), dict(num=P + 1)]
    for b in bad:
        a = {**rows, **b}
        for f in (lib.gemvq_kv4_store_static, lib.gemvq_kv4_load_static):
            assert f(a["kv"], a["k"], a["v"], a["row"], a["n_tok"], a["pos"], a["num"], 0) == gq.EINVAL, b
    attn = dict(kv=kv(), q=P, qs=256, qh=64, y=P, ys=256, n_tok=4, nh=4, pos=P, num=0, window=0, scale=1.0, work=P, nw=1 << 30)
    bad = [dict(kv=kv(0)), dict(kv=kv(hd=96)), dict(q=0), dict(q=P + 4), dict(qs=62), dict(qh=60), dict(qh=66), dict(y=0),
           dict(y=P + 8), dict(ys=252), dict(ys=258), dict(n_tok=0), dict(n_tok=65536), dict(nh=0), dict(nh=3), dict(pos=0),
           dict(num=P + 2), dict(window=-1)]
    if lib.gemvq_kv4_attn_work(kv(), 4, 4):
        bad += [dict(work=0), dict(work=P + 8), dict(nw=lib.gemvq_kv4_attn_work(kv(), 4, 4) - 1)]
    for b in bad:
        a = {**attn, **b}
        assert lib.gemvq_kv4_attn_static(*[a[n] for n in attn], 0) == gq.EINVAL, b
    a = dict(attn, n_tok=1 << 15, nh=1 << 13, ys=64 << 13)  # 2^28 query rows
    assert lib.gemvq_kv4_attn_static(*[a[n] for n in attn], 0) == gq.EINVAL
    long = dict(attn, kv=kv(n_ctx=4096))
    need = lib.gemvq_kv4_attn_work(long["kv"], 4, 4)
    assert need > 0 and lib.gemvq_kv4_attn_work(kv(), 4, 4) == 0  # 64 positions: one range a sequence
    for b in (dict(work=0), dict(work=P + 8), dict(nw=need - 1)):
        a = {**long, **b}
        assert lib.gemvq_kv4_attn_static(*[a[n] for n in attn], 0) == gq.EINVAL, b
    with pytest.raises(gq.GemvqError):
        gq.kv4_store_static(kv(), P, P, 100, 1, P)
    assert C.sizeof(gq.Kv4) == 24
