"""Sizes of 4-bit caches whose bytes would pass 64 bits."""
import pytest

N = 2 ** 31 - 1


def test_sizes_past_64_bits_are_not_served(gq):
    """(No device is touched.)"""
    assert gq.kv4_bytes(65535, 32, 65535, 256) == 65535 * 65535 * 36 * 256
    assert gq.kv4_bytes(100, N, 1, 256) == 100 * 2 ** 26 * 36 * 256
    lib, P = gq.hip_lib(), 1 << 20
    for sizes in ((65535, N, 65535, 256), (65535, N, 65535, 32), (65535, N, 1, 256), (1, N, 65535, 32), (65535, 1 << 20, 65535, 128)):
        assert gq.kv4_bytes(*sizes) == 0, sizes
        kv = gq.Kv4(P, *sizes)
        row = sizes[2] * sizes[3]
        for f in (lib.gemvq_kv4_store_static, lib.gemvq_kv4_load_static):
            assert f(kv, P, P, row, 1, P, 0, 0) == gq.EINVAL
        assert lib.gemvq_kv4_attn_work(kv, 1, sizes[2]) == 0
        assert lib.gemvq_kv4_attn_static(kv, P, row, sizes[3], P, row, 1, sizes[2], P, 0, 0, 1.0, P, 1 << 40, 0) == gq.EINVAL


@pytest.mark.gpu
def test_buffers_of_heads_that_no_command_names(gq):
    with gq.Context(act_floats=1 << 10, weight_bytes=1 << 12) as ctx:
        ctx.set_kv_type(gq.KV_Q4_0)
        for heads in (65536, N):
            with pytest.raises(gq.GemvqError, match="shape"):
                ctx.kv_create(64, heads, 64)
        assert ctx.usable() and ctx.kv_create(64, 2, 64) == 0
