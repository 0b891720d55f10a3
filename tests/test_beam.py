"""The beam search's step on caller-owned memory: selection against float64 with ties, masks, ended beams and the values at the ends
of FP32; reordering byte by byte; both with a 4-bit cache as a search uses them."""
import numpy as np
import pytest

import kv4_ref
from hip_rt import Hip

INF = np.inf


@pytest.fixture
def hip(gq):
    h = Hip(gq)
    yield h
    h.close()


def reference(x, score, last, eos, groups, beams):
    """score, token and parent of a selection, in float64."""
    v = x.shape[1]
    x = np.minimum(np.where(np.isnan(x), -INF, x).astype(np.float64), float(np.finfo(np.float32).max))
    score = np.where(np.isnan(score), -INF, score).astype(np.float64)
    top = x.max(1, keepdims=True)
    with np.errstate(invalid="ignore", divide="ignore"):
        lp = (x - top) - np.log(np.exp(x - top).sum(1, keepdims=True))
        c = np.where((x == -INF) | (score[:, None] == -INF), -INF, score[:, None] + lp)
    if last is not None and 0 <= eos < v:
        over = last == eos
        c[over] = -INF
        c[over, eos] = score[over]
    out = []
    for g in range(groups):
        flat = c[g * beams:(g + 1) * beams].ravel()
        some = np.flatnonzero(flat >= np.partition(flat, -beams)[-beams])
        out.append(some[np.argsort(-flat[some], kind="stable")[:beams]])
    flat = np.stack(out)
    val = np.take_along_axis(c.reshape(groups, -1), flat, 1)
    return val, flat % v, flat // v


def select(gq, hip, x, score, last, eos, groups, beams, skew=0, alias=False, stream=0):
    """skew: floats that rows start past a 16-byte line, and that lie between rows."""
    rows, v = x.shape
    stride = v + skew
    buf = np.full(rows * stride + 8, np.nan, np.float32)
    for r in range(rows):
        buf[skew + r * stride:skew + r * stride + v] = x[r]
    px = hip.upload(buf) + 4 * skew
    ps = hip.upload(score.astype(np.float32))
    pl = hip.upload(np.asarray(last, np.int32)) if last is not None else 0
    po = ps if alias else hip.alloc(4 * rows)
    pt = pl if alias and pl else hip.alloc(4 * rows)
    pp, nw = hip.alloc(4 * rows), gq.beam_work(groups, beams, v)
    gq.beam_select_static(px, stride, v, groups, beams, ps, pl, eos, po, pt, pp, hip.upload(np.full(nw, 0xFF, np.uint8)), nw, stream)
    return [hip.download(p, (groups, beams), t) for p, t in ((po, np.float32), (pt, np.int32), (pp, np.int32))]


def check(got, want):
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2])
    fin = np.isfinite(want[0])
    assert np.array_equal(got[0][~fin], want[0][~fin].astype(np.float32))
    # one rounding to FP32 of a 64-bit value that is good to 1e-9
    assert (np.abs(got[0][fin] - want[0][fin]) <= kv4_ref.U * np.abs(want[0][fin]) + 1e-9).all()


@pytest.mark.gpu
@pytest.mark.parametrize("groups,beams,v", [(1, 1, 1), (1, 1, 7), (2, 3, 5), (1, 4, 2047), (1, 4, 2048), (2, 4, 2049), (3, 5, 8193),
                                            (1, 32, 40), (2, 32, 5000), (16, 8, 40001), (600, 1, 300), (1, 2, 1 << 20),
                                            (1, 32, 151936), (1, 32, 300001), (2, 8, 1 << 20), (1, 32, 1 << 20)])
@pytest.mark.parametrize("skew", [0, 1, 3])
def test_selection(gq, hip, groups, beams, v, skew):
    print(f"[beam selection] {groups} x {beams} of {v}, skew {skew}", flush=True)
    rng = np.random.default_rng(v + skew)
    x = (2.5 * rng.standard_normal((groups * beams, v))).astype(np.float32)
    score = -20 * rng.random(groups * beams)
    last = rng.integers(0, 3, groups * beams).astype(np.int32)
    eos = min(2, v - 1)
    score = score.astype(np.float32)
    check(select(gq, hip, x, score, last, eos, groups, beams, skew), reference(x, score, last, eos, groups, beams))
    check(select(gq, hip, x, score, None, eos, groups, beams, skew, alias=True), reference(x, score, None, -1, groups, beams))


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["equal", "few values", "ascending", "descending", "masked", "all masked", "one left", "start",
                                  "dead", "all ended", "nan", "inf", "extremes", "spikes"])
@pytest.mark.parametrize("beams,v", [(4, 5000), (32, 9000), (1, 100), (8, 60000), (24, 230000)])
def test_selection_at_the_edges(gq, hip, what, beams, v):
    """The groups' beams share their logits, so equal candidates are equal bits and their order is that of the indexes."""
    print(f"[beam selection] {what}, {beams} of {v}", flush=True)
    rng = np.random.default_rng(3)
    groups = 2
    x = np.repeat(rng.standard_normal((groups, v)).astype(np.float32), beams, 0)
    score = np.repeat(np.float32([-1.5, -2.25]), beams)
    last, eos = np.zeros(groups * beams, np.int32), 77
    if what == "equal":
        x[:] = 1.25
    elif what == "few values":
        x = np.repeat(rng.integers(-1, 2, (groups, v)).astype(np.float32), beams, 0)
    elif what == "ascending":
        x[:] = np.arange(v, dtype=np.float32) / 64
    elif what == "descending":
        x[:] = -np.arange(v, dtype=np.float32) / 64
    elif what == "masked":
        x[:, rng.random(v) < 0.9] = -INF
    elif what == "all masked":
        x[:] = -INF
    elif what == "one left":
        x[:] = -INF
        x[:, v - 1] = 3.0
    elif what == "start":
        score = np.tile(np.float32([0.0] + [-INF] * (beams - 1)), groups)
    elif what == "dead":
        score[:] = -INF
    elif what == "all ended":
        last[:] = eos
        score = -np.arange(groups * beams, dtype=np.float32)
    elif what == "nan":
        x[:, ::3] = np.nan
        score[1::2] = np.nan
    elif what == "inf":
        x[:, [5, v // 2]] = INF
    elif what == "extremes":
        x[:, 0], x[:, 1] = 3e38, -3e38
    else:  # the best of a chunk in one thread's hands
        x[:, 1024::1024] += 50
    check(select(gq, hip, x, score, last, eos, groups, beams), reference(x, score, last, eos, groups, beams))


def _arrays(gq, hip, groups, beams, rng, wide):
    """Arrays of every kind: (BeamArray, host copy as bytes, parts of the rows)."""
    rows, unit = groups * beams, 16 if wide else 4
    used = rng.integers(0, 12, rows).astype(np.int32)
    pu = hip.upload(used)
    out = []
    for parts, first, count, ub, ul, order, pad in ((1, 0, 1, 64 * unit, 0, "rp", 0), (3, 0, 1, 1000 * unit, 0, "pr", 0),
                                                    (2, 3, 11, 37 * unit, 1, "pr", 0), (4, 1, 6, 9 * unit, 2, "rp", 2 * unit),
                                                    (1, 5, 5, unit, 1, "rp", 0), (1, 0, 9, unit, 1, "rp", unit)):
        size = count * ub + pad
        rs, ps = (parts * size, size) if order == "rp" else (size, rows * size)
        host = rng.integers(0, 256, rows * parts * size).astype(np.uint8)
        host = np.concatenate([host, np.zeros(64, np.uint8)])
        a = gq.BeamArray(hip.upload(host), rs, ps, parts, first, count, ub, ul, pu if ul else 0, 1)
        out.append((a, host, lambda r, rs=rs, ps=ps, parts=parts: [r * rs + p * ps for p in range(parts)],
                    (first, count, ub, ul)))
    return out, used


@pytest.mark.gpu
@pytest.mark.parametrize("groups,beams", [(1, 1), (1, 2), (3, 4), (2, 7), (1, 16), (2, 32)])
@pytest.mark.parametrize("wide", [True, False])
@pytest.mark.parametrize("who", ["random", "same", "stay", "first", "cycle", "bad"])
def test_reordering(gq, hip, groups, beams, wide, who):
    print(f"[beam reordering] {groups} x {beams} wide {wide} parents {who}", flush=True)
    rng = np.random.default_rng(beams)
    arrays, used = _arrays(gq, hip, groups, beams, rng, wide)
    par = {"random": rng.integers(0, beams, (groups, beams)), "same": np.full((groups, beams), beams - 1),
           "stay": np.tile(np.arange(beams), (groups, 1)), "first": np.zeros((groups, beams), int),
           "cycle": np.tile((np.arange(beams) + 1) % beams, (groups, 1)),
           "bad": np.tile(np.arange(beams)[::-1], (groups, 1))}[who].astype(np.int32)
    if who == "bad":
        par[:, 0], par[:, -1] = -1, beams
    many = (gq.BeamArray * len(arrays))(*[a[0] for a in arrays])
    gq.beam_reorder_static(many, hip.upload(par), groups, beams)
    for i, (a, host, parts_of, (first, count, ub, ul)) in enumerate(arrays):
        want = host.copy()
        for g in range(groups):
            for b in range(beams):
                p = par[g, b]
                if not 0 <= p < beams:
                    continue
                src, dst = g * beams + p, g * beams + b
                end = min(count, -(-int(used[src]) // ul)) if ul else count
                if end > first:
                    for s, d in zip(parts_of(src), parts_of(dst)):
                        want[d + first * ub:d + end * ub] = host[s + first * ub:s + end * ub]
        assert np.array_equal(hip.download(a.data, want.shape, np.uint8), want), i


@pytest.mark.gpu
def test_reordering_more_arrays_than_a_launch_takes(gq, hip):
    rng = np.random.default_rng(9)
    host = [rng.integers(0, 1 << 30, (4, 33)).astype(np.int32) for _ in range(60)]
    arrays = (gq.BeamArray * 60)(*[gq.BeamArray(hip.upload(h), 132, 0, 1, 0, 33, 4) for h in host])
    gq.beam_reorder_static(arrays, hip.upload(np.int32([2, 2, 0, 1])), 1, 4)
    for h, a in zip(host, arrays):
        assert np.array_equal(hip.download(a.data, h.shape, np.int32), h[[2, 2, 0, 1]])


@pytest.mark.gpu
def test_a_search_over_4_bit_caches(gq, hip):
    """Store, attention, selection and reordering as a search runs them, captured once and replayed with eager selections between: a toy
    decoder whose next keys, values and queries are rows of tables, whose logits are another table's row (by the beam's last two tokens)
    plus a part of its attention's output. Scores, tokens and their histories against the same search in float64."""
    groups, beams, v, nh, nkv, hd, prompt, steps, eos = 2, 4, 96, 4, 2, 32, 37, 30, 3
    rows, n_ctx = groups * beams, prompt + steps
    rng = np.random.default_rng(11)
    tk, tv = (rng.standard_normal((v, nkv, hd)).astype(np.float32) for _ in range(2))
    tq = rng.standard_normal((v, nh, hd)).astype(np.float32)
    big = (2 * rng.standard_normal((v, v))).astype(np.float32)
    mix = (0.5 * rng.standard_normal((nh * hd, v))).astype(np.float32)
    prompts = rng.integers(4, v, (groups, prompt))
    kv = gq.Kv4(hip.upload(np.full(gq.kv4_bytes(rows, n_ctx, nkv, hd), 0xFF, np.uint8)), rows, n_ctx, nkv, hd)
    ids = np.zeros((rows, n_ctx), np.int32)
    ids[:, :prompt] = np.repeat(prompts, beams, 0)
    d = {n: hip.alloc(s) for n, s in (("k", 4 * rows * nkv * hd), ("v", 4 * rows * nkv * hd), ("q", 4 * rows * nh * hd),
                                      ("y", 4 * rows * nh * hd), ("x", 4 * rows * v), ("parent", 4 * rows), ("token", 4 * rows))}
    d["pos"], d["used"] = hip.alloc(4 * rows), hip.alloc(4 * rows)
    start = np.tile(np.float32([0.0] + [-INF] * (beams - 1)), groups)
    d["score"], d["ids"] = hip.upload(start), hip.upload(ids)
    hip.write(d["pos"], np.zeros(rows, np.int32))
    gq.kv4_store_static(kv, hip.upload(tk[ids[:, :prompt - 1]]), hip.upload(tv[ids[:, :prompt - 1]]), nkv * hd, prompt - 1, d["pos"])
    nw, na = gq.beam_work(groups, beams, v), gq.kv4_attn_work(kv, 1, nh)
    work, awork = hip.alloc(nw), hip.alloc(na)
    rec = 36 * hd
    per_row = nkv * (-(-n_ctx // 32)) * rec
    moves = (gq.BeamArray * 2)(
        gq.BeamArray(kv.data, per_row, per_row // nkv, nkv, prompt // 32, -(-n_ctx // 32), rec, 32, d["used"], 1),
        gq.BeamArray(d["ids"], 4 * n_ctx, 0, 1, prompt, n_ctx, 4, 1, d["used"], 1))
    stream = hip.stream()

    def attend():
        gq.kv4_store_static(kv, d["k"], d["v"], nkv * hd, 1, d["pos"], 0, stream)
        gq.kv4_attn_static(kv, d["q"], nh * hd, hd, d["y"], nh * hd, 1, nh, d["pos"], 0, 0, hd ** -0.5, awork, na, stream)

    def search():
        gq.beam_select_static(d["x"], v, v, groups, beams, d["score"], d["token"], eos, d["score"], d["token"], d["parent"], work, nw,
                              stream)
        gq.beam_reorder_static(moves, d["parent"], groups, beams, stream)

    g_attend, g_search = hip.capture(stream, attend), hip.capture(stream, search)
    token = np.repeat(prompts[:, -1], beams).astype(np.int32)
    hip.write(d["token"], token)
    keys, vals = kv4_ref.values(tk), kv4_ref.values(tv)
    w_ids, w_score, w_token = ids.copy(), start.astype(np.float64), token.copy()  # the search in float64
    for step in range(steps):
        p = prompt - 1 + step
        hip.write(d["k"], tk[token])
        hip.write(d["v"], tv[token])
        hip.write(d["q"], tq[token])
        hip.write(d["pos"], np.full(rows, p, np.int32))
        hip.write(d["used"], np.full(rows, p + 1, np.int32))
        hip.launch(g_attend, stream) if step % 3 else attend()
        y = hip.download(d["y"], (rows, nh * hd), np.float32)
        want_y, tol = np.empty((rows, nh * hd)), np.empty((rows, nh * hd))
        for r in range(rows):
            for h in range(nh):
                at = w_ids[r, :p + 1], h * nkv // nh
                a, b = kv4_ref.attention(tq[w_token[r], h].astype(np.float64), keys[at], vals[at], p, 0, hd ** -0.5)
                want_y[r, h * hd:(h + 1) * hd], tol[r, h * hd:(h + 1) * hd] = a, b
        assert (np.abs(y - want_y) <= tol).all(), step
        x = (big[token].astype(np.float64) + y.astype(np.float64) @ mix).astype(np.float32)
        hip.write(d["x"], x)
        hip.launch(g_search, stream) if step % 2 else search()
        val, tok, par = reference(x, w_score, w_token, eos, groups, beams)
        src = (par + beams * np.arange(groups)[:, None]).ravel()
        w_ids, w_score = w_ids[src].copy(), val.ravel().astype(np.float32)
        token = hip.download(d["token"], (rows,), np.int32)
        score = hip.download(d["score"], (rows,), np.float32)
        assert np.array_equal(token, tok.ravel()), step
        assert (np.abs(score - w_score) <= 2 * kv4_ref.U * np.abs(w_score) + 1e-9).all()
        w_score, w_token = score, token  # the next step's inputs are the same bits
        if p + 1 < n_ctx:
            w_ids[:, p + 1] = token
            got = hip.download(d["ids"], ids.shape, np.int32)
            got[:, p + 1] = token
            hip.write(d["ids"], got)
            assert np.array_equal(got[:, :p + 2], w_ids[:, :p + 2])


def test_refusals(gq):
    """Arguments that are refused before anything is launched (no device is touched)."""
    lib, P = gq.hip_lib(), 1 << 20
    ok = dict(x=P, stride=100, v=100, groups=2, beams=4, score=P, last=0, eos=1, so=P, tok=P, par=P, work=P, nw=1 << 30)
    need = gq.beam_work(2, 4, 100)
    assert need > 0
    for b in (dict(x=0), dict(x=P + 2), dict(stride=99), dict(v=0), dict(v=(1 << 20) + 1, stride=1 << 21), dict(groups=0), dict(beams=0),
              dict(beams=33), dict(groups=20000), dict(score=0), dict(score=P + 1), dict(last=P + 2), dict(so=0), dict(tok=0),
              dict(par=0), dict(par=P + 3), dict(work=0), dict(work=P + 8), dict(nw=need - 1)):
        a = {**ok, **b}
        assert lib.gemvq_beam_select_static(*a.values(), 0) == gq.EINVAL, b
    assert gq.beam_work(0, 4, 100) == gq.beam_work(1, 33, 100) == gq.beam_work(1, 1, 0) == gq.beam_work(65536, 1, 5) == 0

    def arr(**k):
        d = dict(data=P, row_stride=64, part_stride=0, n_part=1, first=0, count=16, unit_bytes=4, unit_len=1, used=0, used_stride=1)
        return (gq.BeamArray * 1)(gq.BeamArray(*{**d, **k}.values()))

    for b in (dict(data=0), dict(data=P + 2), dict(row_stride=60), dict(row_stride=66), dict(n_part=0), dict(first=17),
              dict(unit_bytes=0), dict(unit_bytes=6, row_stride=96), dict(n_part=2), dict(n_part=2, part_stride=128),
              dict(n_part=2, part_stride=32, row_stride=64), dict(used=P + 1), dict(used=P, unit_len=0), dict(used=P, used_stride=0),
              dict(row_stride=1 << 50), dict(count=1 << 31, unit_bytes=1 << 31, row_stride=1 << 46)):
        assert lib.gemvq_beam_reorder_static(arr(**b), 1, P, 2, 4, 0) == gq.EINVAL, b
    for a in ((None, 1, P, 2, 4), (arr(), 0, P, 2, 4), (arr(), 1, 0, 2, 4), (arr(), 1, P + 2, 2, 4), (arr(), 1, P, 0, 4),
              (arr(), 1, P, 2, 0), (arr(), 1, P, 2, 33), (arr(), 1, P, 65535, 2)):
        assert lib.gemvq_beam_reorder_static(*a, 0) == gq.EINVAL
    # both nestings are taken (nothing moves: first == count, so nothing is launched)
    for k in (dict(n_part=2, part_stride=512), dict(n_part=2, part_stride=64, row_stride=128)):
        assert lib.gemvq_beam_reorder_static(arr(first=16, **k), 1, P, 2, 4, 0) == 0
