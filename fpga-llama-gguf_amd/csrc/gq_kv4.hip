// Kernels on the 4-bit KV cache (gq_kv4.h): storing new keys and values, reading them back, attention.
#include "gq_device.h"
#include "gq_kv4.h"

#include <type_traits>

namespace gq {
namespace {

// One block of 32 elements, one per lane of a half wave: returns the lane's quant and, in d, the block's fp16 scale.
__device__ __forceinline__ uint32_t kv4_quantize(float x, uint32_t & d16) {
    const int lane = threadIdx.x & 63;
    float am = fabsf(x);
#pragma unroll
    for (int s = 16; s >= 1; s >>= 1) am = fmaxf(am, __shfl_xor(am, s, WAVE));
    const unsigned long long at = __ballot(fabsf(x) == am);
    const uint32_t half = lane < 32 ? uint32_t(at) : uint32_t(at >> 32);
    const float m = __shfl(x, (lane & 32) + (half ? __ffs(int(half)) - 1 : 0), WAVE);
    const float d = m / -8.0f;
    const float id = d != 0.0f ? 1.0f / d : 0.0f;
    const float v = x * id + 8.5f;
    d16 = f2h(d);
    return uint32_t(int(fminf(fmaxf(v, 0.0f), 15.0f)));
}

// The sequence's first position and number of tokens.
__device__ __forceinline__ void kv4_span(const Kv4Tokens & t, int s, long long & p0, int & n) {
    p0 = t.pos[size_t(s) * t.pos_stride];
    n = t.num ? min(t.num[s], t.n_tok) : t.n_tok;
}

__device__ __forceinline__ uint8_t * kv4_rec(const Kv4Cache & c, int s, int h, int tile) {
    return c.data + ((size_t(s) * c.n_head_kv + h) * c.tiles + tile) * kv4_record(c.head_dim);
}

// Workgroup (record of the tokens' span, KV head, sequence): half waves take the blocks of its positions in turn. A record that the
// tokens fill is put together in LDS and written in 16-byte pieces; of the others only the tokens' own bytes are written.
template <int HD>
__global__ __launch_bounds__(256) void kv4_store_kernel(Kv4RowsArgs a) {
    using L = Kv4Layout<HD>;
    __shared__ __align__(16) uint8_t img[L::RECORD];
    const int h = blockIdx.y, s = blockIdx.z, tid = threadIdx.x, hw = tid >> 5, e = tid & 31;
    long long p0;
    int n;
    kv4_span(a.t, s, p0, n);
    const long long lo = p0 < 0 ? 0 : p0, hi = p0 + n < a.c.n_ctx ? p0 + n : a.c.n_ctx;  // positions to store
    const long long tile = lo / KV4_TILE + blockIdx.x;
    if (lo >= hi || tile * KV4_TILE >= hi) return;
    const int first = int(lo - tile * KV4_TILE > 0 ? lo - tile * KV4_TILE : 0);
    const int end = int(hi - tile * KV4_TILE < KV4_TILE ? hi - tile * KV4_TILE : KV4_TILE);
    uint8_t * rec = kv4_rec(a.c, s, h, int(tile));
    const bool full = end - first == KV4_TILE;
    uint8_t * out = full ? img : rec;
    for (int u = hw; u < (end - first) * L::NB * 2; u += 8) {
        const int p = first + u / (2 * L::NB), blk = u % L::NB;
        const bool val = (u / L::NB) & 1;
        const size_t row = size_t(s) * a.t.n_tok + size_t(tile * KV4_TILE + p - p0);
        uint32_t d;
        const uint32_t q = kv4_quantize((val ? a.v : a.k)[row * size_t(a.row_stride) + size_t(h) * HD + blk * 32 + e], d);
        const uint32_t up = __shfl_xor(q, 16, WAVE);
        if (e < 16) out[val ? L::vq(p, blk, e) : L::kq(p, blk, e)] = uint8_t(q | up << 4);
        if (e == 0) *reinterpret_cast<uint16_t *>(out + (val ? L::VD : L::KD) + L::scale(p, blk)) = uint16_t(d);
    }
    if (!full) return;
    __syncthreads();
    for (int i = tid; i < L::RECORD / 16; i += 256) reinterpret_cast<uint4 *>(rec)[i] = reinterpret_cast<const uint4 *>(img)[i];
}

template <int HD>
__device__ __forceinline__ float kv4_key(const uint8_t * rec, int p, int e) {
    using L = Kv4Layout<HD>;
    const int blk = e >> 5, q = rec[L::kq(p, blk, e & 15)] >> ((e & 16) ? 4 : 0) & 15;
    return h2f(*reinterpret_cast<const uint16_t *>(rec + L::KD + L::scale(p, blk))) * float(q - 8);
}
template <int HD>
__device__ __forceinline__ float kv4_value(const uint8_t * rec, int p, int e) {
    using L = Kv4Layout<HD>;
    const int blk = e >> 5, q = rec[L::vq(p, blk, e & 15)] >> ((e & 16) ? 4 : 0) & 15;
    return h2f(*reinterpret_cast<const uint16_t *>(rec + L::VD + L::scale(p, blk))) * float(q - 8);
}

// Workgroup (token, KV head, sequence), a thread an element.
template <int HD>
__global__ __launch_bounds__(256) void kv4_load_kernel(Kv4RowsArgs a) {
    const int h = blockIdx.y, s = blockIdx.z, t = blockIdx.x;
    long long p0;
    int n;
    kv4_span(a.t, s, p0, n);
    const long long p = p0 + t;
    if (t >= n || p < 0 || p >= a.c.n_ctx) return;
    const uint8_t * rec = kv4_rec(a.c, s, h, int(p / KV4_TILE));
    const size_t row = (size_t(s) * a.t.n_tok + t) * size_t(a.row_stride) + size_t(h) * HD;
    for (int e = threadIdx.x; e < HD; e += 256) {
        a.k[row + e] = kv4_key<HD>(rec, int(p % KV4_TILE), e);
        a.v[row + e] = kv4_value<HD>(rec, int(p % KV4_TILE), e);
    }
}

// Workgroup (q head, token, sequence): records in order, 8 threads a position for the scores, a thread an element for the values.
template <int HD>
__global__ __launch_bounds__(256) void kv4_attn_kernel(Kv4AttnArgs a) {
    __shared__ float qs[HD], pr[KV4_TILE];
    const int hq = blockIdx.x, t = blockIdx.y, s = blockIdx.z, tid = threadIdx.x, h = hq / (a.n_head / a.c.n_head_kv);
    long long p0;
    int n;
    kv4_span(a.t, s, p0, n);
    const long long pl = p0 + t;
    if (t >= n || pl < 0 || pl >= a.c.n_ctx) return;
    const int pos = int(pl), from = a.window && pos >= a.window ? pos - a.window + 1 : 0;
    const size_t row = size_t(s) * a.t.n_tok + t;
    if (tid < HD) qs[tid] = a.q[row * size_t(a.q_row) + size_t(hq) * size_t(a.q_head) + tid];
    __syncthreads();
    float m = -__builtin_inff(), l = 0.0f, o = 0.0f;
    for (int tile = from / KV4_TILE; tile <= pos / KV4_TILE; ++tile) {
        const uint8_t * rec = kv4_rec(a.c, s, h, tile);
        const int p = tid >> 3, part = tid & 7, at = tile * KV4_TILE + p;
        float dot = 0.0f;
        for (int e = part; e < HD; e += 8) dot += qs[e] * kv4_key<HD>(rec, p, e);
        dot += __shfl_xor(dot, 1, WAVE);
        dot += __shfl_xor(dot, 2, WAVE);
        dot += __shfl_xor(dot, 4, WAVE);
        if (part == 0) pr[p] = at >= from && at <= pos ? dot * a.scale : -__builtin_inff();
        __syncthreads();
        float mt = m;
        for (int j = 0; j < KV4_TILE; ++j) mt = fmaxf(mt, pr[j]);
        const float f = expf_(m - mt);
        l *= f;
        o *= f;
        m = mt;
        for (int j = 0; j < KV4_TILE; ++j) {
            if (pr[j] == -__builtin_inff()) continue;
            const float w = expf_(pr[j] - m);
            l += w;
            if (tid < HD) o += w * kv4_value<HD>(rec, j, tid);
        }
        __syncthreads();
    }
    if (tid < HD) {
        const size_t g = row * size_t(a.q_row) + size_t(hq) * size_t(a.q_head) + tid;
        a.y[row * size_t(a.y_row) + size_t(hq) * HD + tid] = a.gate ? sigmoid_(a.gate[g]) * (o / l) : o / l;
    }
}

template <typename F>
hipError_t by_dim(int hd, F f) {
    switch (hd) {
    case 32: f(std::integral_constant<int, 32>()); break;
    case 64: f(std::integral_constant<int, 64>()); break;
    case 128: f(std::integral_constant<int, 128>()); break;
    case 256: f(std::integral_constant<int, 256>()); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_kv4_store(const Kv4RowsArgs & a, hipStream_t s) {
    const unsigned span = unsigned((a.t.n_tok + KV4_TILE - 2) / KV4_TILE + 1);  // records that n_tok positions can touch
    return by_dim(a.c.head_dim, [&](auto hd) {
        GQ_LAUNCH(kv4_store_kernel<hd.value>, dim3(span, a.c.n_head_kv, a.t.n_seq), dim3(256), 0, s, a);
    });
}

hipError_t launch_kv4_load(const Kv4RowsArgs & a, hipStream_t s) {
    return by_dim(a.c.head_dim, [&](auto hd) {
        GQ_LAUNCH(kv4_load_kernel<hd.value>, dim3(a.t.n_tok, a.c.n_head_kv, a.t.n_seq), dim3(256), 0, s, a);
    });
}

hipError_t launch_kv4_attn(const Kv4AttnArgs & a, hipStream_t s) {
    return by_dim(a.c.head_dim, [&](auto hd) {
        GQ_LAUNCH(kv4_attn_kernel<hd.value>, dim3(a.n_head, a.t.n_tok, a.t.n_seq), dim3(256), 0, s, a);
    });
}

}  // namespace gq
