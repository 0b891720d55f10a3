"""4-bit KV buffers between command lists."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
F = np.float32


def test_a_rejected_list_changes_nothing(gq):
    """A list with ATTN or BEAM_MOVE on a 4-bit buffer that is rejected further on leaves the buffer's regions as they were: positions read
    back are those of the last list that was compiled."""
    nh, nkv, hd, ns, cap = 4, 2, 64, 3, 41
    rng = np.random.default_rng(3)
    at = {n: 64 + 4096 * i for i, n in enumerate(("q", "k", "v", "y", "qn", "kn", "cs", "pos", "parent"))}
    with gq.Context(act_floats=9 * 4096 + 64, weight_bytes=1 << 12) as ctx:
        ctx.set_kv_type(gq.KV_Q4_0)
        kv = ctx.kv_create(ns * cap, nkv, hd)
        for name, n in (("q", ns * nh * hd), ("k", ns * nkv * hd), ("v", ns * nkv * hd), ("qn", hd), ("kn", hd)):
            ctx.write(at[name], rng.standard_normal(n).astype(F))
        slots = np.zeros(16 * ns, np.int32)
        slots[::16] = [0, 40, 17]
        ctx.write(at["pos"], slots)

        def attn(n_tok, seqs):
            c = gq.attn(nh, nkv, at["q"], kv, at["y"], hd, 0, at["pos"], at["k"], at["v"], 0.125, 1e-6, at["qn"], at["kn"], at["cs"], n_tok=n_tok)
            c[7] |= 2 if seqs else 0
            return c

        assert ctx.run(attn(ns, True)) == 0, ctx.error()
        want = ctx.kv_read(kv, 0, ns * cap, nkv * hd)
        used = [p for p in range(ns * cap) if want[0].view(np.float16).reshape(ns * cap, -1)[p].any()]
        assert used == [0, cap + 40, 2 * cap + 17]
        bad = gq.fill(0, 0, 0.0)
        move = gq.beam_move(gq.BEAM_KV, kv, 0, 0, at["parent"], 1, 1, pos=at["pos"])
        for rejected in (attn(1, False) + bad, move + bad):
            assert ctx.run(rejected) > 1
            got = ctx.kv_read(kv, 0, ns * cap, nkv * hd)
            assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
