"""Rotary positions: tables at the ends of what their arguments may be are finite, or refused; so are arrays that name one another's
memory. (No device is touched.)"""
import math

import numpy as np
import pytest


def test_tables_are_finite_or_refused(gq):
    tiny, most = 1e-310, 1.7e308
    ones = np.ones(32)
    for bad in (dict(factor=tiny), dict(factor=tiny, yarn_ctx=4096), dict(factor=5e-324, yarn_ctx=4096, beta_fast=1e-3, beta_slow=1e-3),
                dict(factors=ones * tiny), dict(factors=np.where(np.arange(32) == 31, 5e-324, ones))):
        with pytest.raises(gq.GemvqError):
            gq.rope_freqs(64, 1e4, **bad)
    for ok in (dict(factor=most), dict(factor=most, yarn_ctx=2 ** 31 - 1), dict(factor=1e-9, yarn_ctx=1), dict(factors=ones * most), dict(base=1 + 2.0 ** -52),
               dict(base=1 + 2.0 ** -52, yarn_ctx=2 ** 31 - 1, factor=8.0, beta_slow=5e-324), dict(base=most), dict(base=most, yarn_ctx=1, factor=2.0, beta_fast=most, beta_slow=most)):
        got = gq.rope_freqs(64, **{"base": 1e4, **ok})
        assert np.isfinite(got).all() and (got[:-1] >= 0).all(), ok


def test_pairs_that_keep_their_angle_do_not_depend_on_the_factor(gq):
    """A share of 0 of the angle over `factor` is nothing, whatever it is."""
    plain, stretched = gq.rope_freqs(64, 1e4), gq.rope_freqs(64, 1e4, factor=1e300, yarn_ctx=4096)
    kept = max(math.floor(64 * math.log(4096 / (2 * math.pi * 32)) / (2 * math.log(1e4))), 0)
    assert kept > 0 and np.array_equal(plain[:kept + 1], stretched[:kept + 1])


def test_an_array_named_twice_is_refused(gq):
    """In place or not: its heads would turn twice, or be read while another workgroup writes them."""
    lib, P = gq.hip_lib(), 1 << 20
    a, b, c, d = P, 2 * P, 3 * P, 4 * P
    for pairs in ([(a, a), (a, a)], [(a, b), (c, b)], [(a, b), (b, d)], [(b, d), (a, b)], [(a, b), (c, d), (P * 5, a)], [(a, a), (b, b), (c, c), (b, d)]):
        arr = (gq.RopeRows * len(pairs))(*(gq.RopeRows(x, y, 1024, 128, 1024, 128, 8) for x, y in pairs))
        assert lib.gemvq_rope_static(arr, len(arr), 2, 3, 128, 64, 0, P, P, P, 0) == gq.EINVAL, pairs
