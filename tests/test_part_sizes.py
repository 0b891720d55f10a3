"""Workspaces of the calls on caller-owned memory that verify drafted tokens or attend with sinks and prefixes: one that serves a
loop's largest call serves its smaller ones."""
import itertools

import numpy as np
import pytest

import kv4_ref as ref
from hip_rt import Hip
from test_kv4 import _cache, _data, _store
from test_kv4_shared import check


@pytest.fixture
def hip(gq):
    h = Hip(gq)
    yield h
    h.close()


def growing(sizes):
    """Neighbours of a grid of sizes, the second no smaller anywhere."""
    for at in itertools.product(*(range(len(s)) for s in sizes)):
        for i, s in enumerate(sizes):
            if at[i] + 1 < len(s):
                more = at[:i] + (at[i] + 1,) + at[i + 1:]
                yield tuple(s[k] for s, k in zip(sizes, at)), tuple(s[k] for s, k in zip(sizes, more))


def test_verification_of_fewer_tokens_needs_no_more(gq):
    for small, large in growing(([1, 2, 3, 7, 8, 12, 13, 16, 31, 32, 33, 64, 500, 1000], [0, 1, 3, 4, 5, 31, 32], [1, 7, 2048, 2049, 4096, 4097, 32003, 151936, 1 << 20])):
        assert 0 < gq.draft_work(*small) <= gq.draft_work(*large), (small, large)


HEADS = [(32, 8, 128), (16, 4, 256), (6, 1, 64), (40, 1, 32)]


@pytest.mark.parametrize("nh,nkv,hd", HEADS)
def test_attention_with_sinks_of_fewer_tokens_needs_no_more(gq, nh, nkv, hd):
    def work(n_seq, n_ctx, n_tok):
        return gq.kv4_attn_sink_work(gq.Kv4(0, n_seq, n_ctx, nkv, hd), n_tok, nh)

    for small, large in growing(([1, 2, 3, 12, 13, 31, 32, 63, 64, 95, 96, 97, 200, 1000], [1, 64, 65, 256, 500, 1024, 8192, 100001], [1, 2, 3, 4, 5, 8, 9, 17, 96, 512])):
        few, many = work(*small), work(*large)
        if large[0] * large[2] * nh <= 1 << 22 and many:
            assert 16 <= few <= many, (small, large)
    assert work(96, 32, 1) == 16 and work(1 << 16, 32, 512) == 0  # none needed, not served


@pytest.mark.parametrize("nh,nkv,hd", HEADS)
def test_attention_behind_fewer_prefixes_needs_no_more(gq, nh, nkv, hd):
    sizes = [(g, g * m, p, n, t) for g in (1, 2, 3, 5, 16) for m in (1, 2, 3, 9, 32) for p in (1, 500, 30000) for n in (32, 1000, 8192) for t in (1, 3, 5, 40)]
    needs = np.array([gq.kv4_attn_shared_work(gq.Kv4(0, s, n, nkv, hd), gq.Kv4(0, g, p, nkv, hd), t, nh) for g, s, p, n, t in sizes])
    table = np.array(sizes)
    assert (needs >= 16).all()
    for x, need in zip(table, needs):
        smaller = (table <= x).all(1)
        assert needs[smaller].max() <= need, (x, table[smaller][needs[smaller].argmax()])


@pytest.mark.gpu
def test_a_loop_with_the_workspace_of_its_largest_call(gq, hip):
    """64 sequences of 32/8 heads fill the device without split records, fewer do not; the same behind one or two prefixes, one token or
    several."""
    nh, nkv, hd, own, plen = 32, 8, 128, 500, 300
    rng = np.random.default_rng(15)
    k, v = _data(rng, 96, own, nkv, hd)
    pk, pv = _data(rng, 2, plen, nkv, hd)
    kv, _ = _cache(gq, hip, 96, own, nkv, hd)
    prefix, _ = _cache(gq, hip, 2, plen, nkv, hd)
    _store(gq, hip, kv, k, v, [0] * 96)
    _store(gq, hip, prefix, pk, pv, [0] * 2)
    kk, vv, ppk, ppv = (ref.values(x) for x in (k, v, pk, pv))
    nw = max(gq.kv4_attn_sink_work(kv, 5, nh), gq.kv4_attn_shared_work(kv, prefix, 5, nh))
    work = hip.upload(np.full(nw, 0xFF, np.uint8))
    for n_seq, n_tok, groups in ((96, 1, 0), (95, 1, 0), (3, 5, 0), (96, 1, 2), (9, 5, 1), (1, 1, 1), (1, 1, 0)):
        print(f"[parts] {n_seq} x {n_tok}, {groups} prefixes", flush=True)
        few = gq.Kv4(kv.data, n_seq, own, nkv, hd)
        q = rng.standard_normal((n_seq, n_tok, nh, hd)).astype(np.float32)
        pos = rng.integers(0, own - n_tok, n_seq)
        y = hip.upload(np.full(q.shape, 7.0, np.float32))
        rest = (hip.upload(q), nh * hd, hd, y, nh * hd, n_tok, nh, hip.upload(pos.astype(np.int32)), 0, 200, 3, 0.1, work, nw)
        if groups:
            gq.kv4_attn_shared_static(few, gq.Kv4(prefix.data, groups, plen, nkv, hd), hip.upload(np.int32([plen, 77])), *rest)
        else:
            gq.kv4_attn_sink_static(few, *rest)
        some = rng.choice(n_seq, min(n_seq, 6), replace=False) if not groups else np.arange(n_seq)
        got = hip.download(y, q.shape, np.float32)
        if groups:
            check(q, kk[:n_seq], vv[:n_seq], got, pos, None, 200, 3, 0.1, ppk[:groups], ppv[:groups], [plen, 77][:groups])
        else:
            check(q[some], kk[some], vv[some], got[some], pos[some], None, 200, 3, 0.1)


@pytest.mark.gpu
def test_a_loop_of_verifications_with_the_workspace_of_its_largest(gq, hip):
    """13 sequences of 4 drafted tokens of 151936 have half as many chunks as 12."""
    from test_draft import check as check_tokens, inputs, reference

    rng = np.random.default_rng(16)
    s, k, n = 13, 4, 151936
    x = inputs(rng, s, k, n)
    nw = gq.draft_work(s, k, n)
    bufs, work = [hip.upload(a) for a in x], hip.alloc(nw)
    for few in (13, 12, 1):
        na, out, lp = hip.alloc(4 * few), hip.alloc(4 * few * (k + 1)), hip.alloc(4 * few * (k + 1))
        gq.draft_verify_static(bufs[0], n, bufs[1], n, n, few, k, bufs[2], 0, bufs[3], 1.0, 1.0, na, out, lp, work, nw)
        check_tokens((hip.download(na, (few,), np.int32), hip.download(out, (few, k + 1), np.int32), hip.download(lp, (few, k + 1), np.float32)),
                     reference(*(a[:few] for a in x[:3]), None, x[3][:few], 1.0, 1.0))


@pytest.mark.gpu
def test_calls_that_are_not_split_take_no_workspace(gq, hip):
    """Short caches, and sequences enough to fill the device by themselves."""
    for n_seq, own, (nh, nkv, hd) in ((3, 200, (8, 2, 128)), (96, 600, (32, 8, 128))):
        rng = np.random.default_rng(18)
        k, v = _data(rng, n_seq, own, nkv, hd)
        kv, _ = _cache(gq, hip, n_seq, own, nkv, hd)
        _store(gq, hip, kv, k, v, [0] * n_seq)
        q, y = rng.standard_normal((n_seq, 1, nh, hd)).astype(np.float32), hip.alloc(4 * n_seq * nh * hd)
        pos = rng.integers(0, own, n_seq)
        gq.kv4_attn_sink_static(kv, hip.upload(q), nh * hd, hd, y, nh * hd, 1, nh, hip.upload(pos.astype(np.int32)), 0, 70, 3, 0.1)
        few = slice(0, 5)
        check(q[few], ref.values(k[few]), ref.values(v[few]), hip.download(y, q.shape, np.float32)[few], pos[few], None, 70, 3, 0.1)
