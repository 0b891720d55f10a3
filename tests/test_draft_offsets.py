"""Verification of drafted tokens whose logits over the temperature lie far from 0: up to the last ones that exponentials are formed of
in FP32 (8192 ln 2 = 5678), across that border within a row, and beyond it."""
import numpy as np
import pytest

from hip_rt import Hip
from test_draft import inputs, reference, verify


@pytest.fixture
def hip(gq):
    h = Hip(gq)
    yield h
    h.close()


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [1390.0, 1410.0, 5600.0, -5600.0, 5665.0, -5680.0, 20000.0, -3e5])
@pytest.mark.parametrize("temp", [1.0, 0.0078125, 300.0])
@pytest.mark.parametrize("certain", [False, True])
def test_far_logits(gq, hip, offset, temp, certain):
    """A term is 2^(N / 256) (1 + E), E = s (ln 2 + ..) in FP32 and s what is left of the logit times c = log2(e) / temperature, in two
    parts (of each 24 bits). With X = |c x| < 9192: c is off by 2^-48 of itself, s by 2.3e-11 / ln 2; s is below 2^-9 + 2^-23 X < 0.0031,
    its smaller part rounded by 2^-34, itself by 2^-33; its factor by 2^-25 and by 1.9e-9 (ln 2 in FP32); E, below 0.0022, by 2^-33:
    (2.3 + 4.1 + 8.1 + 9.2 + 0.6 + 11.7) e-11 = 3.6e-10, over 1 + E. Log-probabilities have a rounding to FP32 besides."""
    print(f"[draft] logits around {offset}, temperature {temp}", flush=True)
    rng = np.random.default_rng(17)
    x = inputs(rng, 9, 3, 6000)
    x = [((a + offset) * temp).astype(np.float32) for a in x[:2]] + list(x[2:])
    draft = None if certain else x[1]
    got = verify(gq, hip, x[0], draft, x[2], None, x[3], temp, temp)
    want = reference(x[0], draft, x[2], None, x[3], temp, temp)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
    assert (np.abs(got[2] - want[2]) <= 2.0 ** -24 * np.abs(want[2]) + 3.7e-10).all()
