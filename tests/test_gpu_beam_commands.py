"""The beam search's commands in lists and in the model driver at their edges."""
import numpy as np
import pytest

from test_gpu_kv4_commands import small

pytestmark = pytest.mark.gpu
F = np.float32


def slots(x):
    """Values 16 floats apart."""
    x = np.asarray(x)
    out = np.zeros(16 * x.size, x.dtype)
    out[::16] = x.ravel()
    return out


def test_a_group_with_prompts_of_unlike_lengths(gq):
    """While a group's first sequence reads its prompt, every sequence of it is its own parent, whatever its parent slot held, and one
    behind its own prompt keeps its token; the moves then leave the group's rows where they are."""
    ng, nb, v, cap, win = 2, 3, 64, 16, 16
    ns = ng * nb
    rng = np.random.default_rng(12)
    prompts = rng.integers(0, v, (ns, cap)).astype(np.int32)
    lens = np.int32([5, 2, 5, 4, 4, 1])
    tok, parent = prompts[:, 0].copy(), np.int32([2, 2, 0, 1, 0, 0])
    at = {n: 64 + 16 * 1024 * i for i, n in enumerate(("x", "score", "parent", "tok", "pos", "len", "prompt", "win"))}
    cmds = gq.beam(v, at["x"], v, nb, ng, -1, at["score"], at["parent"], at["tok"], at["pos"], at["len"], at["prompt"], cap)
    cmds += gq.beam_move(gq.BEAM_ACT, at["win"], win, win, at["parent"], nb, ng)
    rows = rng.standard_normal((ns, win)).astype(F)
    score = F([0, -1, -2, 0, -1, -2])
    with gq.Context(act_floats=8 * 16 * 1024 + 64, weight_bytes=1 << 12) as ctx:
        for name, x in (("x", rng.standard_normal((ns, v)).astype(F)), ("score", slots(score)), ("parent", slots(parent)), ("tok", slots(tok)),
                        ("len", slots(lens)), ("prompt", prompts), ("win", rows)):
            ctx.write(at[name], x)
        for p in range(3):
            ctx.write(at["pos"], slots(np.full(ns, p, np.int32)))
            assert ctx.run(cmds) == 0, ctx.error()
            tok = np.where(p + 1 < lens, prompts[:, p + 1], tok)
            assert np.array_equal(ctx.read(at["tok"], 16 * ns, np.int32)[::16], tok), p
            assert np.array_equal(ctx.read(at["parent"], 16 * ns, np.int32)[::16], np.tile(np.arange(nb), ng)), p
            assert np.array_equal(ctx.read(at["score"], 16 * ns)[::16], score)
            assert np.array_equal(ctx.read(at["win"], rows.size).reshape(rows.shape), rows), p


def test_beam_under_a_scratch_limit(gq, monkeypatch):
    """The limit is on scratch that a launch can do without; the selection's workspace is none of it. Larger ones follow smaller ones."""
    monkeypatch.setenv("GEMVQ_SCRATCH_LIMIT", "0")
    rng = np.random.default_rng(2)
    with gq.Context(act_floats=1 << 18, weight_bytes=1 << 12) as ctx:
        ctx.write(64, slots(F([-1.0, -2.0])))
        for v in (64, 512, 40000):
            x = rng.standard_normal((2, v)).astype(F)
            ctx.write(1024, x)
            ctx.write(64, slots(F([-1.0, -2.0])))
            assert ctx.run(gq.beam(v, 1024, v, 2, 1, -1, 64, 128, 192)) == 0, ctx.error()
            lp = x - np.log(np.exp(x.astype(np.float64)).sum(1, keepdims=True)) + np.array([[-1.0], [-2.0]])
            best = np.argsort(-lp.ravel(), kind="stable")[:2]
            assert np.array_equal(ctx.read(192, 32, np.int32)[::16], best % v)
            assert np.array_equal(ctx.read(128, 32, np.int32)[::16], best // v)


def test_no_scores_of_an_earlier_search(gq):
    """Between set_beam and reset there are no scores: those in memory are another search's, in other groups."""
    import qwen35

    with qwen35.BatchModel(qwen35.generate(small(qwen35), seed=5), 4) as bm:
        bm.set_beam(2)
        with pytest.raises(gq.GemvqError, match="reset first"):
            bm.scores()
        bm.reset([[1, 2]] * 4)
        assert np.array_equal(bm.scores(), F([0, -np.inf, 0, -np.inf]))
        bm.step(3)
        assert np.isfinite(bm.scores()).all()
        bm.set_beam(4)
        with pytest.raises(gq.GemvqError, match="reset first"):
            bm.scores()
        bm.reset([[1, 2]] * 4)
        assert np.array_equal(bm.scores(), F([0, -np.inf, -np.inf, -np.inf]))
