"""4-bit KV buffers and the beam search in command lists and in the model driver: the ATTN command against float64 (its norms, rotation and
quantization repeated in FP32, so the cache's values are known exactly), the BEAM commands against numpy, a whole search against
teacher-forced lockstep decodes."""
import numpy as np
import pytest

import kv4_ref as ref
from test_beam import reference

pytestmark = pytest.mark.gpu
F = np.float32
EPS = 1e-6


@pytest.fixture(scope="module")
def q35():
    import qwen35

    return qwen35


def _norm_rope(x, w, cs, n_rot):
    """RMS norm with weight and NEOX rotation of one row in FP32, in the kernels' order of operations."""
    s = (x * x).astype(F)
    while s.size > 1:
        s = (s[0::2] + s[1::2]).astype(F)
    sc = F(1) / np.sqrt(F(s[0] / F(x.size)) + F(EPS), dtype=F)
    y = ((x * sc).astype(F) * w).astype(F)
    h = n_rot // 2
    c, sn = cs[0::2], cs[1::2]
    a, b = y[:h].copy(), y[h:n_rot].copy()
    y[:h] = (a * c).astype(F) - (b * sn).astype(F)
    y[h:n_rot] = (a * sn).astype(F) + (b * c).astype(F)
    return y


def _attn_case(gq, nh, nkv, hd, n_rot, gate, runs, n_ctx, seqs=0):
    """Runs ATTN commands on a 4-bit buffer: each of `runs` a (first position, tokens); with seqs, each a position list. Returns per run the
    outputs, and the rows' queries, gates, positions and sequence, and the cache's exact values per sequence."""
    rng = np.random.default_rng(hd + nh)
    qstride = 2 * hd if gate else hd
    most = max(seqs or n for _, n in runs)
    off, at = 64, {}
    for name, n in (("q", most * nh * qstride), ("k", most * nkv * hd), ("v", most * nkv * hd), ("y", most * nh * hd), ("qn", hd),
                    ("kn", hd), ("cs", n_ctx * n_rot), ("pos", 16 * 32)):
        at[name] = off
        off += -(-n // 16) * 16
    qn, kn = (rng.uniform(0.5, 1.5, hd).astype(F) for _ in range(2))
    ang = np.arange(n_ctx)[:, None] * 1e4 ** (-2.0 * np.arange(n_rot // 2) / max(n_rot, 1))
    cs = np.stack([np.cos(ang), np.sin(ang)], -1).reshape(n_ctx, n_rot).astype(F)
    ns = seqs or 1
    cap = n_ctx
    keys, vals = (np.zeros((ns, cap, nkv, hd)) for _ in range(2))
    out = []
    with gq.Context(act_floats=off + 64, weight_bytes=1 << 12) as ctx:
        ctx.set_kv_type(gq.KV_Q4_0)
        kv = ctx.kv_create(n_ctx * ns, nkv, hd)
        for name, x in (("qn", qn), ("kn", kn), ("cs", cs)):
            if x.size:
                ctx.write(at[name], x)
        for first, n in runs:
            rows = ns if seqs else n
            q = rng.standard_normal((rows, nh, qstride)).astype(F)
            k, v = (rng.standard_normal((rows, nkv, hd)).astype(F) for _ in range(2))
            pos = list(first) if seqs else [first + t for t in range(n)]
            slots = np.zeros(16 * 32, np.int32)
            if seqs:
                slots[0:16 * rows:16] = pos
            else:
                slots[0] = first
            for name, x in (("q", q), ("k", k), ("v", v), ("pos", slots)):
                ctx.write(at[name], x)
            ctx.write(at["y"], np.full(rows * nh * hd, 7, F))
            c = gq.attn(nh, nkv, at["q"], kv, at["y"], hd, n_rot, at["pos"], at["k"], at["v"], hd ** -0.5, EPS, at["qn"], at["kn"],
                        at["cs"], gate=at["q"] + hd if gate else None, n_tok=rows)
            if seqs:
                c[7] |= 2
            assert ctx.run(c) == 0, ctx.error()
            y = ctx.read(at["y"], rows * nh * hd).reshape(rows, nh, hd)
            qr = np.zeros((rows, nh, hd), F)
            for r in range(rows):
                s, p = (r if seqs else 0), pos[r]
                if not 0 <= p < cap:
                    continue
                for h in range(nkv):
                    keys[s, p, h] = ref.values(_norm_rope(k[r, h], kn, cs[p], n_rot))
                    vals[s, p, h] = ref.values(v[r, h])
                for h in range(nh):
                    qr[r, h] = _norm_rope(q[r, h, :hd], qn, cs[p], n_rot)
            for r in range(rows):
                s, p = (r if seqs else 0), pos[r]
                if not 0 <= p < cap:
                    assert (y[r] == 7).all()
                    continue
                for h in range(nh):
                    want, tol = ref.attention(qr[r, h].astype(np.float64), keys[s, :, h * nkv // nh], vals[s, :, h * nkv // nh], p, 0,
                                              hd ** -0.5)
                    if gate:  # sigmoid in FP32: an exponential and a division, a few steps
                        f = 1 / (1 + np.exp(-q[r, h, hd:].astype(np.float64)))
                        want, tol = want * f, tol + 8 * ref.U * np.abs(want)
                    assert (np.abs(y[r, h] - want) <= tol).all(), (r, h, p)
            out.append(y)
        got_k, got_v = ctx.kv_read(kv, 0, n_ctx * ns, nkv * hd)
    for got, x in ((got_k, keys), (got_v, vals)):
        assert np.array_equal(got.view(np.float16).reshape(x.shape).astype(F), x.astype(np.float16).astype(F))
    return out


@pytest.mark.parametrize("nh,nkv,hd,n_rot,gate", [(4, 1, 32, 0, False), (4, 2, 64, 64, True), (8, 2, 128, 32, True), (16, 4, 256, 64, True)])
def test_attn_command(gq, nh, nkv, hd, n_rot, gate):
    """Tokens one by one, in batches, over the ends of records, past the buffer's end."""
    print(f"[kv4 ATTN] {nh}/{nkv} of {hd}", flush=True)
    _attn_case(gq, nh, nkv, hd, n_rot, gate, [(0, 1), (1, 1), (2, 29), (31, 32), (63, 5), (68, 1), (69, 3), (71, 1)], 72)


@pytest.mark.parametrize("n_ctx", [64, 41])
def test_attn_command_in_sequences(gq, n_ctx):
    """Regions of whole records and regions that end inside one; a sequence past its end."""
    _attn_case(gq, 4, 2, 64, 32, True, [([0, 0, 0], 1), ([1, 1, 1], 1), ([2, 2, 2], 1), ([3, n_ctx, 3], 1)], n_ctx, seqs=3)


def test_attn_command_without_scratch(gq, monkeypatch):
    """No memory for partial sums: every sequence is one range."""
    monkeypatch.setenv("GEMVQ_SCRATCH_LIMIT", "0")
    _attn_case(gq, 8, 2, 128, 32, False, [(0, 32), (32, 32), (64, 32), (96, 32), (128, 32), (160, 1)], 192)


@pytest.mark.parametrize("scratch", [True, False])
def test_attn_command_over_ranges(gq, monkeypatch, scratch):
    """Buffers long enough to be split into ranges, with and without memory for their partial sums (unstored positions are zeros)."""
    if not scratch:
        monkeypatch.setenv("GEMVQ_SCRATCH_LIMIT", "0")
    _attn_case(gq, 16, 4, 256, 64, True, [(0, 32), (500, 32), (890, 5), (899, 1), (310, 1)], 900)
    _attn_case(gq, 8, 2, 128, 32, False, [([600, 3, 1199], 1), ([601, 4, 1200], 1), ([1198, 1198, 600], 1)], 1200, seqs=3)


def test_attn_command_rejections(gq):
    with gq.Context(act_floats=1 << 16, weight_bytes=1 << 12) as ctx:
        with pytest.raises(gq.GemvqError):
            ctx.set_kv_type(3)
        ctx.set_kv_type(gq.KV_Q4_0)
        with pytest.raises(gq.GemvqError):
            ctx.kv_create(64, 2, 48)
        assert ctx.usable()
        kv = ctx.kv_create(64, 2, 64)
        c = gq.attn(4, 2, 64, kv, 1024, 64, 0, 32, 2048, 2304, 0.125, EPS, 4096, 4160, 4224)
        assert ctx.run(c) == 0, ctx.error()
        ctx.set_arith(gq.ARITH_REFERENCE)
        assert ctx.run(c) == 1 and "4-bit" in ctx.error()
        ctx.set_arith(gq.ARITH_CANONICAL)
        assert ctx.run(gq.attn(4, 2, 64, kv, 1024, 64, 0, 32, 2048, 2304, 0.125, EPS, 4096, 4160, 4224, n_tok=33)) == 1
        assert ctx.run(gq.attn(0, 2, 64, kv, 1024, 64, 0, 32, 2048, 2304, 0.125, EPS, 4096, 4160, 4224)) == 1
        ctx.set_kv_type(gq.KV_F16)  # buffers of both kinds side by side
        kv16 = ctx.kv_create(64, 2, 64)
        both = c + gq.attn(4, 2, 64, kv16, 1024, 64, 0, 32, 2048, 2304, 0.125, EPS, 4096, 4160, 4224)
        assert ctx.run(both) == 0, ctx.error()


def test_beam_commands(gq):
    """Prompt steps and selections of two groups in a captured list, with every kind of move."""
    ng, nb, v, cap, win = 2, 3, 512, 40, 48
    ns = ng * nb
    rng = np.random.default_rng(4)
    off, at = 64, {}
    for name, n in (("x", ns * v), ("score", 16 * ns), ("parent", 16 * ns), ("tok", 16 * ns), ("pos", 16 * ns), ("len", 16 * ns),
                    ("prompt", ns * cap), ("out", ns * cap), ("win", 2 * ns * win)):
        at[name] = off
        off += -(-n // 16) * 16
    prompts = np.repeat(rng.integers(10, v, (ng, cap)).astype(np.int32), nb, 0)
    lens = np.repeat([2, 4], nb)
    slot = lambda x: np.concatenate([np.append(np.asarray([a]), np.zeros(15, np.asarray(x).dtype)) for a in x])  # noqa: E731
    cmds = gq.beam(v, at["x"], v, nb, ng, 5, at["score"], at["parent"], at["tok"], at["pos"], at["len"], at["prompt"], cap)
    cmds += gq.beam_move(gq.BEAM_STATE, 0, 4, 4, at["parent"], nb, ng, 2, 4 * ns)
    cmds += gq.beam_move(gq.BEAM_ACT, at["win"], win, win, at["parent"], nb, ng, 2, ns * win)
    cmds += gq.beam_move(gq.BEAM_ACT, at["out"], cap, cap, at["parent"], nb, ng, pos=at["pos"])
    cmds += gq.beam_next(at["tok"], at["pos"], at["out"], cap, ns)
    state = rng.standard_normal((2, ns, 4 * 128)).astype(F)
    wins = rng.standard_normal((2, ns, win)).astype(F)
    score = np.tile(F([0, -np.inf, -np.inf]), ng)
    tok, pos = prompts[:, 0].copy(), np.zeros(ns, np.int32)
    out = np.full((ns, cap), -1, np.int32)
    out[:, 0] = tok
    with gq.Context(act_floats=off + 64, weight_bytes=1 << 12, state_rows=8 * ns) as ctx:
        ctx.state_write(0, state)
        for name, x in (("score", slot(score)), ("tok", slot(tok)), ("pos", slot(pos)), ("len", slot(lens.astype(np.int32))),
                        ("prompt", prompts), ("out", out), ("win", wins)):
            ctx.write(at[name], x)
        g = ctx.graph(cmds)
        assert ctx.launch_count() == 4  # two for the selection, one for the moves, one for the ids
        for step in range(8):
            x = (3 * rng.standard_normal((ns, v))).astype(F)
            if step == 5:
                x[:, 5] += 30  # eos wins
            ctx.write(at["x"], x)
            ctx.replay(g)
            last = np.where(pos >= lens, tok, -1)
            val, t2, p2 = reference(x, score, last, 5, ng, nb)
            par = np.arange(ns)
            for i in range(ng):
                rows = slice(i * nb, i * nb + nb)
                if pos[i * nb] + 1 < lens[i * nb]:
                    tok[rows] = prompts[rows, pos[i * nb] + 1]
                else:
                    tok[rows], score[rows], par[rows] = t2[i], val[i].astype(F), p2[i] + i * nb
            state, wins = state[:, par], wins[:, par]
            for r, o in enumerate(out.copy()[par]):
                out[r, :pos[r] + 1] = o[:pos[r] + 1]
            pos = pos + 1
            out[np.arange(ns), pos] = tok
            got = {n: ctx.read(at[n], 16 * ns, dt)[::16] for n, dt in (("tok", np.int32), ("pos", np.int32), ("score", F))}
            assert np.array_equal(got["tok"], tok) and np.array_equal(got["pos"], pos), step
            fin = np.isfinite(score)
            assert np.array_equal(got["score"][~fin], score[~fin])
            assert (np.abs(got["score"][fin] - score[fin]) <= 2 * ref.U * np.abs(score[fin]) + 1e-9).all()
            score = got["score"].copy()
            assert np.array_equal(ctx.read(at["out"], ns * cap, np.int32).reshape(ns, cap), out), step
            assert np.array_equal(ctx.read(at["win"], wins.size).reshape(wins.shape), wins)
            assert np.array_equal(ctx.state_read(0, 8 * ns).reshape(state.shape), state)


def test_beam_moves_that_meet_run_in_order(gq):
    """Two moves of one array, and of overlapping ones, in one list: as if run one by one."""
    rng = np.random.default_rng(6)
    x = rng.standard_normal(400).astype(F)
    parent = np.zeros(48, np.int32)
    parent[0:48:16] = [2, 0, 1]
    moves = [gq.beam_move(gq.BEAM_ACT, 64, 32, 32, 16, 3, 1), gq.beam_move(gq.BEAM_ACT, 64, 32, 32, 16, 3, 1),
             gq.beam_move(gq.BEAM_ACT, 80, 48, 40, 16, 3, 1), gq.beam_move(gq.BEAM_ACT, 320, 16, 10, 16, 3, 1)]
    got = []
    with gq.Context(act_floats=512, weight_bytes=1 << 12) as ctx:
        for lists in ([sum(moves, [])], moves):
            ctx.write(64, x)
            ctx.write(16, parent)
            for c in lists:
                assert ctx.run(c) == 0, ctx.error()
            got.append(ctx.read(64, 400))
    assert np.array_equal(got[0], got[1])


def test_beam_command_rejections(gq):
    with gq.Context(act_floats=1 << 14, weight_bytes=1 << 12, state_rows=64) as ctx:
        ctx.set_kv_type(gq.KV_Q4_0)
        kv = ctx.kv_create(64, 2, 64)
        ok = dict(n_vocab=100, x=1024, row_stride=112, n_beam=2, n_group=2, eos=1, score=64, parent=128, tok=192, pos=256, plen=320,
                  prompt=2048, cap=20)
        assert ctx.run(gq.beam(**ok)) == 0, ctx.error()
        for b in (dict(n_vocab=0), dict(row_stride=96), dict(row_stride=100), dict(n_beam=0), dict(n_beam=33), dict(n_group=0),
                  dict(n_group=17), dict(x=16300), dict(x=1025), dict(score=65), dict(parent=16380), dict(tok=16380), dict(pos=16380),
                  dict(plen=16380), dict(prompt=16368), dict(cap=0)):
            assert ctx.run(gq.beam(**{**ok, **b})) == 1, b
        move = dict(kind=gq.BEAM_ACT, off=1024, row_stride=64, n=64, parent=128, n_beam=2, n_group=2)
        for good in ({}, dict(kind=gq.BEAM_STATE, off=0, row_stride=4, n=4), dict(kind=gq.BEAM_KV, off=kv, pos=256),
                     dict(n_part=2, part_stride=256), dict(n_part=2, part_stride=64, row_stride=128)):
            assert ctx.run(gq.beam_move(**{**move, **good})) == 0, (good, ctx.error())
        for b in (dict(kind=3), dict(n=0), dict(row_stride=60), dict(off=16300), dict(off=1025), dict(parent=129), dict(n_beam=0),
                  dict(n_group=20), dict(first=65), dict(n_part=2, part_stride=128), dict(off=128, row_stride=64), dict(pos=16380),
                  dict(kind=gq.BEAM_STATE, off=0, row_stride=40, n=40), dict(kind=gq.BEAM_KV, off=kv), dict(kind=gq.BEAM_KV, off=7, pos=256),
                  dict(kind=gq.BEAM_KV, off=kv, pos=256, n_group=1, n_beam=3), dict(kind=gq.BEAM_KV, off=kv, pos=256, first=17)):
            assert ctx.run(gq.beam_move(**{**move, **b})) == 1, b
        assert ctx.run(gq.beam_move(**move)[:8]) == 1 and ctx.run(gq.beam(**ok)[:8]) == 1
        assert ctx.run(gq.beam_next(192, 256, 2048, 20, 4)) == 0
        for a in ((193, 256, 2048, 20, 4), (192, 256, 2048, 0, 4), (192, 256, 2048, 20, 0), (192, 256, 2048, 20, 33), (192, 256, 16368, 20, 4)):
            assert ctx.run(gq.beam_next(*a)) == 1
        assert ctx.usable()


def small(q35, n_ctx=48):
    return q35.Config(n_layer=4, n_embd=1024, n_ff=2048, n_vocab=2048, n_head=4, n_head_kv=1, head_dim=128, n_rot=32, ssm_k_heads=2,
                      ssm_v_heads=4, n_ctx=n_ctx)


def test_model_over_a_4_bit_cache(gq, q35):
    """The first attention layer's keys and values do not depend on any attention: what the 4-bit caches hold of them is the fp16 caches'
    to a quantization step, the same bits for single steps, a batched prompt and sequences in lockstep."""
    cfg = small(q35, 41)
    blob = q35.generate(cfg, seed=3)
    ids = q35.prompt_ids(cfg, 40, 3)
    row = cfg.n_head_kv * cfg.head_dim
    got = {}
    for kind in (gq.KV_F16, gq.KV_Q4_0):
        with q35.Model(blob, kv_type=kind) as m:
            m.reset(ids)
            m.step(39)
            got[kind, "steps"] = m.ctx.kv_read(0, 0, 39, row)
            m.step(1)
            tokens = m.tokens(41)
            m.reset(ids)
            assert m.prefill(39)
            got[kind, "prefill"] = m.ctx.kv_read(0, 0, 39, row)
            m.step(1)
            assert np.array_equal(m.tokens(40), tokens[:40])
            assert np.isfinite(m.logits()).all()
    with q35.BatchModel(blob, 2, kv_type=gq.KV_Q4_0) as bm:
        bm.reset([ids, ids[:7]])
        bm.step(39)
        got["lockstep"] = bm.ctx.kv_read(0, 0, 39, row)
    for i in range(2):
        x = got[gq.KV_F16, "steps"][i].view(np.float16).astype(np.float64).reshape(-1, 32)
        q = got[gq.KV_Q4_0, "steps"][i].view(np.float16).astype(np.float64).reshape(-1, 32)
        # a step is an eighth of the block's largest element; the far end of the range (7 steps of 8) is a whole step off; fp16 twice
        step = np.abs(x).max(1, keepdims=True) / 8
        assert (np.abs(x - q) <= step * (1 + 2.0 ** -7)).all()
        assert np.array_equal(got[gq.KV_Q4_0, "steps"][i], got[gq.KV_Q4_0, "prefill"][i])
        assert np.array_equal(got[gq.KV_Q4_0, "steps"][i], got["lockstep"][i])


@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 2, 64), (4, 1, 256)])
def test_long_prompt_over_a_4_bit_cache(gq, q35, monkeypatch, heads, kv_heads, dim):
    """Prompt chunks of 512 tokens (their rotated queries in the context's scratch) and of as many as the buffers' own scratch holds: the first
    attention layer's cache is the same bits. The second's depends on the first's attention, whose FP32 rounding differs by chunk; that turns
    few activations' 8-bit roundings, each a 254th of its block's largest, so that few of 16 levels change, by one: 1 in 20 at most is
    asked for, where a wrong row would change nearly all."""
    cfg = q35.Config(n_layer=8, n_embd=1024, n_ff=2048, n_vocab=2048, n_head=heads, n_head_kv=kv_heads, head_dim=dim, n_rot=32,
                     ssm_k_heads=2, ssm_v_heads=4, n_ctx=1100)
    blob = q35.generate(cfg, seed=7)
    ids = q35.prompt_ids(cfg, 1050, 5)
    row, got = kv_heads * dim, []
    for limit in (None, "0"):
        if limit:
            monkeypatch.setenv("GEMVQ_SCRATCH_LIMIT", limit)
        with q35.Model(blob, kv_type=gq.KV_Q4_0) as m:
            m.reset(ids)
            assert m.prefill(1049)
            m.step(20)
            assert np.isfinite(m.logits()).all()
            got.append([m.ctx.kv_read(layer, 0, 1049, row) for layer in (0, 1)])
    for i in range(2):
        assert np.array_equal(got[0][0][i], got[1][0][i])
        a, b = (np.asarray(g[1][i]).view(np.float16).astype(np.float64).reshape(-1, 32) for g in got)
        step = np.maximum(np.abs(a).max(1), np.abs(b).max(1))[:, None] / 8
        assert (np.abs(a - b) > step / 2).mean() < 0.05


@pytest.mark.parametrize("kind", ["f16", "q4_0"])
@pytest.mark.parametrize("groups,beams,lens", [(2, 3, (9, 4)), (1, 4, (33,))])
def test_beam_search_of_the_model(gq, q35, kind, groups, beams, lens):
    """Every step's selection from the logits of teacher-forced lockstep decodes of the beams' own ids (the same bits, whatever rows the
    beams moved through), the scores and ids after each."""
    kv = gq.KV_Q4_0 if kind == "q4_0" else gq.KV_F16
    cfg = small(q35)
    blob = q35.generate(cfg, seed=5, types={"output.weight": gq.Q8_0})
    ns, steps = groups * beams, 6
    rng = np.random.default_rng(7)
    prompts = [rng.integers(0, cfg.n_vocab, n).astype(np.int32) for n in lens]
    ids = [prompts[s // beams] for s in range(ns)]
    print(f"[beam search] {groups} x {beams}, {kind} caches", flush=True)

    def search(eos, check):
        score = np.tile(F([0.0] + [-np.inf] * (beams - 1)), groups)
        seqs = [list(p[:1]) for p in ids]
        with q35.BatchModel(blob, ns, kv_type=kv) as bm, q35.BatchModel(blob, ns, kv_type=kv) as forced:
            bm.set_beam(beams, eos)
            bm.reset(ids)
            for step in range(max(lens) - 1 + steps):
                bm.step()
                if check:  # row s reads its own ids so far
                    forced.reset([np.asarray(q, np.int32) for q in seqs])
                    forced.step(step + 1)
                    x = np.stack([forced.logits(s) for s in range(ns)])
                    last = np.asarray([q[-1] if len(q) > len(ids[s]) else -1 for s, q in enumerate(seqs)])
                    val, tok, par = reference(x, score, last, eos, groups, beams)
                    new = []
                    for s in range(ns):
                        g = s // beams
                        if step + 1 < len(ids[s]):
                            new.append(seqs[s] + [ids[s][step + 1]])
                        else:
                            new.append(seqs[g * beams + par[g, s % beams]] + [tok[g, s % beams]])
                    moved = np.asarray([step + 1 >= len(p) for p in ids])
                    seqs = new
                    got = bm.scores()
                    want = np.where(moved, val.ravel(), score)
                    fin = np.isfinite(want)
                    assert np.array_equal(got[~fin], want[~fin].astype(F))
                    assert (np.abs(got[fin] - want[fin]) <= 2 * ref.U * np.abs(want[fin]) + 1e-9).all(), step
                    score = got
                    for s in range(ns):
                        assert np.array_equal(bm.tokens(s, step + 2), seqs[s]), (step, s)
            return [bm.tokens(s, max(lens) + steps) for s in range(ns)], bm.scores()

    free, _ = search(-1, True)
    eos = int(free[0][max(lens) + 1])  # a token that the best beam takes: now the search ends there
    ended, scores = search(eos, True)
    again, scores2 = search(eos, False)
    assert all(np.array_equal(a, b) for a, b in zip(ended, again)) and np.array_equal(scores, scores2)
    for row in ended:  # behind eos: eos
        gen = row[max(lens):]
        at = np.nonzero(gen == eos)[0]
        if at.size and groups == 1:
            assert (gen[at[0]:] == eos).all()
    assert any((row[max(lens):] == eos).any() for row in ended)


def test_beam_refusals_of_the_model(gq, q35):
    blob = q35.generate(small(q35), seed=5)
    with q35.BatchModel(blob, 4) as bm:
        for n in (3, 5, -1, 8):
            with pytest.raises(gq.GemvqError):
                bm.set_beam(n)
        bm.set_beam(2)
        with pytest.raises(gq.GemvqError, match="reset first"):
            bm.step(1)
        with pytest.raises(gq.GemvqError, match="same prompt"):
            bm.reset([[1, 2], [1, 3], [4], [4]])
        with pytest.raises(gq.GemvqError, match="reset first"):
            bm.step(1)
        bm.reset([[1, 2], [1, 2], [4], [4]])
        bm.step(3)
        bm.set_beam(0)  # greedy again
        bm.reset([[1, 2], [1, 3], [4], [4]])
        bm.step(3)
        with pytest.raises(gq.GemvqError):
            bm.scores()
        greedy = [bm.tokens(s, 4) for s in range(4)]
    with q35.BatchModel(blob, 4) as bm:
        bm.reset([[1, 2], [1, 3], [4], [4]])
        bm.step(3)
        assert all(np.array_equal(bm.tokens(s, 4), greedy[s]) for s in range(4))
