"""The 4-bit KV cache on the CPU: its quantization in FP32, its layout, and attention over it in float64."""
import numpy as np

U = 2.0 ** -24  # half a step of FP32, relative


def quantize(x):
    """Q4_0 of the last axis: quants (0..15) and fp16 scales per block of 32, in FP32 as ggml does."""
    b = x.astype(np.float32).reshape(*x.shape[:-1], -1, 32)
    at = np.abs(b).argmax(-1)[..., None]  # the first of the largest
    d = (np.take_along_axis(b, at, -1) / np.float32(-8)).astype(np.float32)
    inv = np.divide(np.float32(1), d, out=np.zeros_like(d), where=d != 0)
    q = np.clip(np.trunc((b * inv).astype(np.float32) + np.float32(8.5)), 0, 15).astype(np.uint8)
    return q, d[..., 0].astype(np.float16)


def values(x):
    """What the cache holds of rows x, in float64."""
    q, d = quantize(x)
    return ((q.astype(np.float64) - 8) * d.astype(np.float64)[..., None]).reshape(x.shape)


def put(rec, p, k, v):
    """Writes one position's key and value (head_dim floats) into a record (uint8 array)."""
    hd = k.size
    nb, kb, vb = hd // 32, min(hd // 32, 4), min(hd // 32, 2)
    for x, value in ((k, 0), (v, 1)):
        q, d = quantize(x)
        for blk in range(nb):
            for e in range(16):
                byte = int(q[blk, e]) | int(q[blk, e + 16]) << 4
                if value:
                    at = 16 * hd + np.ravel_multi_index((blk // vb, p % 16 // 4, e, blk % vb, p // 16, p % 4),
                                                        (nb // vb, 4, 16, vb, 2, 4))
                else:
                    at = np.ravel_multi_index((p // 16, blk // kb, e // 4, p % 16, blk % kb, e % 4), (2, nb // kb, 4, 16, kb, 4))
                rec[at] = byte
            at = 32 * hd + value * 2 * hd + 2 * np.ravel_multi_index((p % 16 // 4, blk, p // 16, p % 4), (4, nb, 2, 4))
            rec[at:at + 2] = np.frombuffer(d[blk].tobytes(), np.uint8)


def attention(q, k, v, pos, window, scale):
    """One query row over positions 0..pos of k and v [positions, head_dim] (float64): y, and a bound of the error of FP32
    arithmetic on it. With u = 2^-24: a score's sum of hd products is off by at most (hd + 4) u sum |q_i k_i| scale (4: the
    query taken in two parts, the scale); e^s by that, as a factor, plus a few u; the weighted sum and the sum of weights over n
    positions by n u and 8 u more (weights times scales taken in two parts, joins, the division)."""
    lo = max(0, pos - window + 1) if window else 0
    kk, vv = k[lo:pos + 1], v[lo:pos + 1]
    s = kk @ q * scale
    p = np.exp(s - s.max())
    p /= p.sum()
    hd = q.size
    ds = (hd + 4) * U * np.max(np.abs(kk) @ np.abs(q)) * scale + 4 * U * np.max(np.abs(s))
    return p @ vv, (2 * ds + (2 * len(kk) + 24) * U) * (p @ np.abs(vv)) + 1e-30
