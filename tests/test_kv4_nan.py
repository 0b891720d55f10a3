"""What the 4-bit cache holds of blocks with NaN, infinities and values too large for an fp16 scale."""
import numpy as np
import pytest

import kv4_ref as ref
from hip_rt import Hip
from test_kv4 import _cache, _store


@pytest.fixture
def hip(gq):
    h = Hip(gq)
    yield h
    h.close()


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [32, 128, 256])
@pytest.mark.parametrize("n_tok", [1, 64])
@pytest.mark.parametrize("what,alone", [(np.nan, False), (-np.nan, False), (np.inf, True), (-np.inf, True), (3e6, True)])
def test_blocks_without_a_scale(gq, hip, hd, n_tok, what, alone):
    """One such element at each place of a block in turn: a NaN makes its whole block NaN; an infinity, or a number whose eighth is past
    fp16's range, makes it infinite itself, and the block's other elements anything but finite. The other blocks stay what they are."""
    rng = np.random.default_rng(hd)
    for e in range(32):
        x = rng.standard_normal((1, n_tok, 1, hd)).astype(np.float32)
        clean = ref.values(x)
        x[..., e] = what
        kv, _ = _cache(gq, hip, 1, 64, 1, hd)
        _store(gq, hip, kv, x, x, [0])
        out = [hip.alloc(4 * n_tok * hd) for _ in range(2)]
        gq.kv4_load_static(kv, *out, hd, n_tok, hip.upload(np.zeros(1, np.int32)))
        for p in out:
            got = hip.download(p, x.shape, np.float32)
            assert np.array_equal(got[..., 32:], clean[..., 32:].astype(np.float32))
            assert not np.isfinite(got[..., :32]).any(), e
            if alone:
                assert (got[..., e] == np.sign(np.float32(what)) * np.float32(np.inf)).all(), (e, got[0, 0, 0, e])
            else:
                assert np.isnan(got[..., :32]).all(), e
