"""Rotary positions and verification of drafted tokens at sizes from which on they run in forms of their own: rotated rows of 16 MB and more
(stores that pass the caches by, several pieces a thread), 2^24 logits and more (chunks of 8192). Everything else as in the tests of
smaller sizes: ragged, padded, in place, at borders of groups of rows and heads."""
import numpy as np
import pytest

from hip_rt import Hip
from test_draft import check as check_tokens, inputs, reference, verify
from test_rope import check as check_rows, rotate

MANY_FLOATS, MANY_LOGITS = 4 << 20, 16 << 20


@pytest.fixture
def hip(gq):
    h = Hip(gq)
    yield h
    h.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dim,n_rot", [(256, 64), (128, 128), (96, 96), (1024, 1024), (256, 8), (64, 58)])
@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("in_place", [False, True])
def test_rope(gq, hip, dim, n_rot, layout, in_place):
    heads = (5, 2, 4)
    n_tok = MANY_FLOATS // (3 * sum(heads) * dim) + 2
    n_tok += n_tok * 3 % max(1, 512 // n_rot) == 0  # rows that are left over behind the last whole group
    assert 3 * n_tok * sum(heads) * dim >= MANY_FLOATS
    print(f"[rope] {n_rot} of {dim}, layout {layout}, 3 x {n_tok} tokens, in place {in_place}", flush=True)
    rng = np.random.default_rng(dim + n_rot)
    xs = [rng.standard_normal((3, n_tok, h, dim), dtype=np.float32) for h in heads]
    freqs = gq.rope_freqs(n_rot, 1e6, 4.0, 4096)
    pos, num = [-3, 77, 2 ** 31 - n_tok], [n_tok, 9, n_tok - 1]
    check_rows(xs, rotate(gq, hip, xs, n_rot, layout, freqs, pos, num, 4, in_place), n_rot, layout, freqs, pos, num, in_place)


@pytest.mark.gpu
@pytest.mark.parametrize("s,k,n,skew", [(13, 4, 151936, 0), (16, 4, 151936, 3), (17, 4, 150001, 1), (16, 0, 1 << 20, 0), (700, 3, 3521, 0)])
def test_verification(gq, hip, s, k, n, skew):
    assert s * n * (2 * k + 1) >= MANY_LOGITS
    print(f"[draft] {s} x {k} of {n}, skew {skew}", flush=True)
    rng = np.random.default_rng(n + skew)
    x = inputs(rng, s, k, n)
    num = rng.integers(-1, k + 2, s)
    for draft, temp in ((x[1], 1.0), (None, 0.7), (x[1], 0.0)):
        check_tokens(verify(gq, hip, x[0], draft, x[2], num, x[3], temp, skew=skew), reference(x[0], draft, x[2], num, x[3], temp, 1.0))
