// Kernels on the 4-bit KV cache (gq_kv4.h): storing new keys and values, reading them back, attention.
#include "gq_device.h"
#include "gq_kv4.h"

#include <algorithm>
#include <cfloat>
#include <climits>
#include <type_traits>

namespace gq {
namespace {

// A block of 32 elements held by 8 lanes, lane j elements 4 j .. 4 j + 3: returns the lane's four quants as the low nibbles of four
// bytes and, in d16, the block's fp16 scale.
__device__ __forceinline__ uint32_t kv4_quantize(const float * x, uint32_t & d16) {
    // magnitudes as words: a NaN is above all numbers and becomes the scale, so the block reads back as NaN
    const auto size = [](float y) { return __float_as_uint(y) & 0x7fffffffu; };
    uint32_t am = size(x[0]);
    float m = x[0];
#pragma unroll
    for (int i = 1; i < 4; ++i) {
        const bool more = size(x[i]) > am;
        am = more ? size(x[i]) : am;
        m = more ? x[i] : m;
    }
    const int lane = threadIdx.x;
    const auto take = [&](float m2, bool later) {  // the other lanes' largest; of equal ones the first
        const bool other = size(m2) > am || (later && size(m2) == am);
        am = other ? size(m2) : am;
        m = other ? m2 : m;
    };
    take(dpp_f32<DPP_XOR1>(m), lane & 1);
    take(dpp_f32<DPP_XOR2>(m), lane & 2);
    take(dpp_f32<DPP_HALF_MIRROR>(m), lane & 4);
    const float d = m / -8.0f, id = d != 0.0f ? 1.0f / d : 0.0f;
    d16 = f2h(d);
    uint32_t q = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float v = x[i] * id + 8.5f;
        q |= uint32_t(int(fminf(fmaxf(v, 0.0f), 15.0f))) << (8 * i);
    }
    return q;
}

// The sequence's first position and number of tokens.
__device__ __forceinline__ void kv4_span(const Kv4Tokens & t, int s, long long & p0, int & n) {
    p0 = t.pos[size_t(s) * t.pos_stride];
    n = t.num ? min(t.num[s], t.n_tok) : t.n_tok;
}

__device__ __forceinline__ uint8_t * kv4_rec(const Kv4Cache & c, int s, int h, int tile) {
    return c.data + size_t(s * c.seq + h * c.head + tile) * kv4_record(c.head_dim);
}

// Workgroup (record of the tokens' span; keys or values; four blocks | KV head | sequence): 8 lanes a block. A record that the tokens
// fill is put together in LDS and written in 16-byte pieces; of the others only the tokens' own bytes are written. So small a share of
// a record (2.3 KB) that a prompt of 512 tokens still has a few hundred workgroups, each with its 4 reads in flight together.
// 1983 tokens of 4 heads of 256 (18.5 MB): 8.0 us, 2.3 TB/s; 512 of them 4.9 us; one token of each of 32 sequences, 8 heads of 128, 3 us.
// The launch and one trip to memory are 3 to 4 us of each; behind them the largest is bound by the shuffles and conversions of its
// blocks.
constexpr int KV4_STORE = 256;  // threads (1983 tokens of 4 heads of 256 with their reading back: 17.6, 15.3 and 14.3 us with 64, 128 and 256)
template <int HD>
__global__ __launch_bounds__(KV4_STORE) void kv4_store_kernel(Kv4RowsArgs a) {
    using L = Kv4Layout<HD>;
    constexpr int BG = L::NB < 4 ? L::NB : 4, GROUPS = L::NB / BG, UNITS = KV4_STORE / 8, ITER = KV4_TILE * BG / UNITS;
    constexpr int QB = 512 * BG;  // bytes of the quants of BG blocks, keys or values
    __shared__ __align__(16) uint8_t img[QB + 64 * BG];
    const int h = blockIdx.y, s = blockIdx.z, tid = threadIdx.x, j = tid & 7;
    const int val = blockIdx.x & 1, bg = (blockIdx.x >> 1) % GROUPS;
    long long p0;
    int n;
    kv4_span(a.t, s, p0, n);
    const long long lo = p0 < 0 ? 0 : p0, hi = p0 + n < a.c.n_ctx ? p0 + n : a.c.n_ctx;  // positions to store
    const long long at = (lo / KV4_TILE + (blockIdx.x >> 1) / GROUPS) * KV4_TILE;        // the record's first position
    if (lo >= hi || at >= hi) return;
    const int first = int(lo - at > 0 ? lo - at : 0), end = int(hi - at < KV4_TILE ? hi - at : KV4_TILE);
    uint8_t * rec = kv4_rec(a.c, s, h, int(at / KV4_TILE));
    const bool full = end - first == KV4_TILE;
    const float * src = (val ? a.v : a.k) + size_t(h) * HD + bg * 128 + j * 4;
    const long long row0 = (long long)s * a.t.n_tok + (at - p0);
    const int units = (end - first) * BG;
    typedef float f32x4 __attribute__((ext_vector_type(4)));
    float x[ITER][4];
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        const int u = i * UNITS + (tid >> 3);
        if (u < units) *reinterpret_cast<f32x4 *>(x[i]) = *reinterpret_cast<const f32x4 *>(src + (row0 + first + u / BG) * a.row_stride + u % BG * 32);
    }
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        const int u = i * UNITS + (tid >> 3);
        if (u >= units) break;
        const int p = first + u / BG, b = u % BG, blk = bg * BG + b;
        uint32_t d;
        const uint32_t q = kv4_quantize(x[i], d), bytes = q | uint32_t(dpp_i32<0x104>(int(q))) << 4;  // lanes j < 4: with those of lane j + 4
        uint8_t * to = full ? img : rec;
        if (j < 4) {
            if (val) {
                uint8_t * v = to + (full ? L::vq(p, blk, 4 * j) - L::VQ - bg * QB : L::vq(p, blk, 4 * j));
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e * 8 * L::VB] = uint8_t(bytes >> (8 * e));
            } else {
                uint8_t * k = to + (full ? L::kq(p, blk, 4 * j) - (p >> 4) * (8 * HD - 256 * BG) - bg * 256 * L::KB : L::kq(p, blk, 4 * j));
                *reinterpret_cast<uint32_t *>(k) = bytes;
            }
        }
        if (j == 0)
            *reinterpret_cast<uint16_t *>(full ? img + QB + ((p & 15) >> 2) * 16 * BG + b * 16 + (p >> 4) * 8 + (p & 3) * 2
                                               : rec + (val ? L::VD : L::KD) + L::scale(p, blk)) = uint16_t(d);
    }
    if (!full) return;
    __syncthreads();
    for (int i = tid; i < QB / 16; i += KV4_STORE) {
        const int sub = i / (QB / 32);  // keys: the record's halves lie apart
        const int to = val ? L::VQ + bg * QB + i * 16 : sub * 8 * HD + bg * 256 * L::KB + (i - sub * (QB / 32)) * 16;
        *reinterpret_cast<uint4 *>(rec + to) = *reinterpret_cast<const uint4 *>(img + i * 16);
    }
    for (int i = tid; i < 4 * BG; i += KV4_STORE)
        *reinterpret_cast<uint4 *>(rec + (val ? L::VD : L::KD) + (i / BG * L::NB + bg * BG + i % BG) * 16) = *reinterpret_cast<const uint4 *>(img + QB + i * 16);
}

// Workgroup (q head, or KV head behind them | token | sequence): the ATTN command's norm and rotation of one vector, in the order of
// the F16 cache's kernels; a q head's goes to qr, a key's into the cache with its value, 8 lanes a block. One vector a workgroup: a
// decode step has few, each a chain of two sums and two trips to memory (4 us).
template <int HD>
__global__ __launch_bounds__(256) void kv4_append_kernel(Kv4AppendArgs a) {
    using L = Kv4Layout<HD>;
    __shared__ __align__(16) float xs[HD], rot[HD];
    __shared__ float red[4];
    const int t = blockIdx.y, s = blockIdx.z, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    long long p0;
    int n;
    kv4_span(a.t, s, p0, n);
    const long long pl = p0 + t;
    if (t >= n || pl < 0 || pl >= a.c.n_ctx) return;
    const int pos = int(pl), half = a.n_rot / 2;
    const bool isq = int(blockIdx.x) < a.n_head;
    const int h = isq ? blockIdx.x : blockIdx.x - a.n_head;
    const size_t row = size_t(s) * a.t.n_tok + t;
    const bool el = tid < HD;
    const int e = el ? tid : 0;
    const float x = !el ? 0.0f : isq ? a.q[(row * a.n_head + h) * size_t(a.q_stride) + e] : a.k[(row * a.c.n_head_kv + h) * HD + e];
    const float w = isq ? a.qn[e] : a.kn[e];
    const int pi = e < half ? e : e - half;
    const bool turn = e < a.n_rot;
    const float cs0 = turn ? a.cs[size_t(pos) * a.n_rot + 2 * pi] : 0.0f, cs1 = turn ? a.cs[size_t(pos) * a.n_rot + 2 * pi + 1] : 0.0f;
    float sq[1] = {x * x};
    pair_sum_lanes_n<64, 1>(sq);
    if (lane == 0) red[wave] = sq[0];
    __syncthreads();
    const float sc = 1.0f / sqrtf(((red[0] + red[1]) + (red[2] + red[3])) / float(HD) + a.eps);
    if (el) xs[e] = (x * sc) * w;
    __syncthreads();
    if (el) {
        const float x0 = xs[pi], x1 = turn ? xs[pi + half] : 0.0f;
        const float r = e < half ? x0 * cs0 - x1 * cs1 : turn ? x0 * cs1 + x1 * cs0 : xs[e];
        if (isq) a.qr[(row * a.n_head + h) * HD + e] = r;
        else rot[e] = r;
    }
    if (isq) return;
    __syncthreads();
    if (tid >= HD / 2) return;  // HD / 4 threads the key, as many the value
    const bool val = tid >= HD / 4;
    const int u = val ? tid - HD / 4 : tid, blk = u >> 3, j = u & 7, p = pos % KV4_TILE;
    const float * src = val ? a.v + (row * a.c.n_head_kv + h) * HD + 4 * u : rot + 4 * u;
    const float y[4] = {src[0], src[1], src[2], src[3]};
    uint32_t d;
    const uint32_t q = kv4_quantize(y, d), bytes = q | uint32_t(dpp_i32<0x104>(int(q))) << 4;
    uint8_t * rec = kv4_rec(a.c, s, h, pos / KV4_TILE);
    if (j < 4) {
        uint8_t * to = rec + (val ? L::vq(p, blk, 4 * j) : L::kq(p, blk, 4 * j));
#pragma unroll
        for (int i = 0; i < 4; ++i) to[i * (val ? 8 * L::VB : 1)] = uint8_t(bytes >> (8 * i));
    }
    if (j == 0) *reinterpret_cast<uint16_t *>(rec + (val ? L::VD : L::KD) + L::scale(p, blk)) = uint16_t(d);
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

// Workgroup (token, KV head, sequence), a thread an element: the writes, 7 times what is read, are whole lines. Few tokens: a trip to
// memory after the positions' one, 3 us.
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

// Many tokens: workgroup (record of the tokens' span; keys or values | KV head | sequence) takes its half of the record to LDS in
// 16-byte pieces and writes the rows in 16-byte pieces. 1983 tokens of 4 heads of 256 (18.5 MB): 7.1 us, 2.6 TB/s, 3 to 4 of them the
// launch and two trips to memory.
template <int HD>
__global__ __launch_bounds__(256) void kv4_load_records_kernel(Kv4RowsArgs a) {
    using L = Kv4Layout<HD>;
    constexpr int QB = 16 * HD, ROW = HD / 4;  // bytes of the keys' or the values' quants; threads of a row
    __shared__ __align__(16) uint8_t img[QB + 2 * HD];
    const int h = blockIdx.y, s = blockIdx.z, tid = threadIdx.x, val = blockIdx.x & 1;
    long long p0;
    int n;
    kv4_span(a.t, s, p0, n);
    const long long lo = p0 < 0 ? 0 : p0, hi = p0 + n < a.c.n_ctx ? p0 + n : a.c.n_ctx;  // positions to read
    const long long at = (lo / KV4_TILE + (blockIdx.x >> 1)) * KV4_TILE;                  // the record's first position
    if (lo >= hi || at >= hi) return;
    const int first = int(lo - at > 0 ? lo - at : 0), end = int(hi - at < KV4_TILE ? hi - at : KV4_TILE);
    const uint8_t * rec = kv4_rec(a.c, s, h, int(at / KV4_TILE));
    for (int i = tid; i < QB / 16; i += 256) reinterpret_cast<uint4 *>(img)[i] = reinterpret_cast<const uint4 *>(rec + (val ? L::VQ : 0))[i];
    for (int i = tid; i < HD / 8; i += 256) reinterpret_cast<uint4 *>(img + QB)[i] = reinterpret_cast<const uint4 *>(rec + (val ? L::VD : L::KD))[i];
    __syncthreads();
    const int e = tid % ROW * 4, blk = e >> 5, up = e & 16 ? 4 : 0;
    float * to = (val ? a.v : a.k) + ((long long)s * a.t.n_tok + (at - p0)) * a.row_stride + size_t(h) * HD + e;
    for (int p = first + tid / ROW; p < end; p += 256 / ROW) {
        const float d = h2f(*reinterpret_cast<const uint16_t *>(img + QB + L::scale(p, blk)));
        typedef float f32x4 __attribute__((ext_vector_type(4)));
        f32x4 y;
        if (val) {
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = d * float((img[L::vq(p, blk, (e & 15) + i) - L::VQ] >> up & 15) - 8);
        } else {
            const uint32_t w = *reinterpret_cast<const uint32_t *>(img + L::kq(p, blk, e & 15));
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = d * float(int(w >> (8 * i + up) & 15) - 8);
        }
        *reinterpret_cast<f32x4 *>(to + p * a.row_stride) = y;
    }
}

// ---- attention ----
// A wave takes the rows (token, q head) of one KV head 16 at a time (NQ such groups) and records of 32 positions one after another:
//   S^T = K Q^T   16x16x32 fp16 matrix instructions, a block of 32 elements each: the quants minus 8 are whole numbers, exact in fp16;
//                 the query, scaled to its row's largest element, is the sum of two fp16 numbers (22 bits). Each block's sums are
//                 multiplied by its scales in FP32. (The quants' bits as they are, 2^-24 n, with the 8 taken off through the
//                 accumulator's start, are a tenth fewer vector instructions, but the instruction's sums of such small factors keep
//                 several bits less: results are off by 5e-6 in place of 3e-7.)
//   P = 2^(S - c) in FP32, c = m - 4 with m the query's running maximum, or m - 7 where that is far above the one before it, taken anew
//                 when a score passes c by 9 (so P <= 2^9). P is the sum of two fp16 numbers: 22 bits, but no finer than 2^-24: at most
//                 2^-28 of the largest weight, and 2^-31 where one position is 2^9 above all others and the sum is made of small
//                 weights beside it. (FP32 would keep 24 bits of the smallest ones too, in three parts: half as many matrix instructions
//                 again. m - 7 always: 512 tokens at 7680, us with m - 4, so, and m - 7: 16/4 heads of 256 175.0 / 174.9 / 178.1,
//                 16/2 of 64 59.8 / 60.4 / 63.9.) Lane 16 g + q holds query q's weights of the 8 positions that it feeds to
//   O^T += V^T P^T: the quants minus 8 again; a block's scales go to the weights, P d = h + l: h the rounded product of d and P's upper
//                 part, l, by two fused multiply-adds, what that rounding left and the lower part's product (22 bits). The scales
//                 are brought up by a power of two 2^e common to the wave, the largest so far to 2^6..2^7, its 11 bits below 2^7, so
//                 P d is at most 65504, fp16's largest number; a scale 2^20 below the largest is still a normal number.
// The accumulators stay with the query's lanes and nothing crosses lanes in the loop. The four waves of a workgroup take the records of
// its range in turn and join at the end; ranges of one sequence are joined by kv4_join_kernel.
// A record and 16 rows, heads of 256, are 64 matrix instructions and about 540 others, half of them unpacking; wider heads than 128
// leave no registers for more than 16 rows to share that. What bounds it, by the counters:
//   512 tokens at 7680, 16/4 heads of 256: 180 us, 370 TFLOP/s of the formula's 66.6 GFLOP (twice that in parts). Vector instructions
//     are issued in 64 % of the cycles, and without any matrix instruction it would still be 160 us: each hundred instructions less a
//     record are 21 us. (Kernel times, here and below, by rocprofv3.)
//   32 sequences of up to 8192, 32/8 heads of 128 (152 MB): 40 us, 3.8 TB/s; vector instructions in 47 %, matrix instructions in 16 %,
//     the rest the beginnings and ends of workgroups that have some ten records a wave.
//   one sequence of 32768, 16/4 heads of 256 (38 MB): 14.6 us, 2.6 TB/s, two records a wave: the chain of position, record, sums and
//     joining is half of it; of 640: 7.2 us, that chain alone.
// Tried and taken back, for the 512 tokens, then at 202 us: workgroups whose waves share one record's unpacking for 64 rows through LDS
// (two barriers a record; 190 us and 16 us of joining); 32 rows a wave at heads of 256 with one wave a SIMD (244 us). A raised wave
// priority around the matrix instructions, and other orders of them, change less than 1 %.
typedef _Float16 half2 __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef uint16_t __attribute__((may_alias)) half_word;  // 16 bits of memory that is read as words

constexpr float KV4_LOW = -FLT_MAX;  // no score is below it: the maximum before the first one

template <int N>
__device__ __forceinline__ void load_words(const uint8_t * p, uint32_t * w) {
    if constexpr (N == 4) {
        const u32x4 x = *reinterpret_cast<const u32x4 *>(p);
        for (int i = 0; i < 4; ++i) w[i] = x[i];
    } else if constexpr (N == 2) {
        const u32x2 x = *reinterpret_cast<const u32x2 *>(p);
        w[0] = x[0];
        w[1] = x[1];
    } else {
        w[0] = *reinterpret_cast<const uint32_t *>(p);
    }
}

// What a lane holds of a record: its quants in registers; the scales, which 16 lanes share, go through LDS (a lane loads, masks and
// scales 4 HD / 64 bytes of them: the keys' in lanes 0..31, the values' in 32..63).
template <int HD>
struct Kv4Tile {
    static constexpr int NB = HD / 32, KB = Kv4Layout<HD>::KB, VB = Kv4Layout<HD>::VB;
    static constexpr int NS = HD / 32;              // scales a lane loads
    static constexpr int NW = NS > 1 ? NS / 2 : 1;  // words of them
    uint32_t k[2][NB];  // its position's key bytes, by half of the record and block
    uint32_t v[NB][2];  // its element's value bytes at its 8 positions
    uint32_t d[NW];

    __device__ __forceinline__ void load_keys(const uint8_t * rec, int lane) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int c = 0; c < NB / KB; ++c) load_words<KB>(rec + u * 8 * HD + c * 256 * KB + lane * 4 * KB, &k[u][c * KB]);
    }
    __device__ __forceinline__ void load_scales(const uint8_t * rec, int lane) {
        if constexpr (NS > 1) load_words<NW>(rec + Kv4Layout<HD>::KD + lane * 4 * NW, d);
        else d[0] = *reinterpret_cast<const uint16_t *>(rec + Kv4Layout<HD>::KD + lane * 2);
    }
    __device__ __forceinline__ void load_values(const uint8_t * rec, int lane) {
#pragma unroll
        for (int c = 0; c < NB / VB; ++c) load_words<2 * VB>(rec + Kv4Layout<HD>::VQ + c * 512 * VB + lane * 8 * VB, v[c * VB]);
    }
    // The position of the record that the lane's scale i belongs to.
    __device__ static int at(int lane, int i) {
        const int w = (lane & 31) * NS + i;
        return ((w >> 2) & 1) * 16 + w / (8 * NB) * 4 + (w & 3);
    }
    // Scales to LDS, each group of four in the order 0, 2, 1, 3 of nibbles(), times f (fp16 pairs; 1 for the keys').
    __device__ __forceinline__ void stage(uint32_t * lds, int lane, half2 f) const {
        uint32_t x[NW];
#pragma unroll
        for (int i = 0; i < NW; ++i) x[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2, d[i]) * f);
        if constexpr (NS >= 4) {
#pragma unroll
            for (int i = 0; i < NW; i += 2) {
                lds[lane * NW + i] = __builtin_amdgcn_perm(x[i + 1], x[i], 0x05040100u);
                lds[lane * NW + i + 1] = __builtin_amdgcn_perm(x[i + 1], x[i], 0x07060302u);
            }
        } else {
            half_word * p = reinterpret_cast<half_word *>(lds);
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                const int w = lane * NS + i;
                p[(w & ~3) + ((w & 1) << 1) + ((w >> 1) & 1)] = uint16_t(x[0] >> (16 * i));
            }
        }
    }
};

// Orders a wave's LDS writes before its other lanes' reads (a wave's LDS operations are carried out in order).
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

__device__ __forceinline__ float half_of(uint32_t w, int hi) { return h2f((hi ? w >> 16 : w) & 0xffffu); }

__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const half2 h = {_Float16(a), _Float16(b)};
    return __builtin_bit_cast(uint32_t, h);
}

// Constants that the compiler is kept from seeing: masks and exponents whose and-or then is one instruction (two literals would not
// fit it), and a -1 whose multiply-add with an fp16 operand is one.
struct Kv4Const {
    uint32_t m0, m1, x0, x1;
    float minus;
    __device__ __forceinline__ Kv4Const() {
        __asm__("s_mov_b32 %0, 0x000f000f" : "=s"(m0));
        __asm__("s_mov_b32 %0, 0x00f000f0" : "=s"(m1));
        __asm__("v_mov_b32 %0, 0x64006400" : "=v"(x0));
        __asm__("v_mov_b32 %0, 0x54005400" : "=v"(x1));
        __asm__("s_mov_b32 %0, -1.0" : "=s"(minus));
    }
};

// Two numbers as the sums of two fp16 numbers each: hi + lo, 22 bits. The empty asms make the numbers and their upper parts exist
// (see f2h): folded into the conversion, a product's nearest fp16 number can differ from the one that lo is formed against.
__device__ __forceinline__ void split2(float a, float b, uint32_t & hi, uint32_t & lo, const Kv4Const & k) {
    __asm__("" : "+v"(a), "+v"(b));
    hi = pack2(a, b);
    __asm__("" : "+v"(hi));
    lo = pack2(__builtin_fmaf(half_of(hi, 0), k.minus, a), __builtin_fmaf(half_of(hi, 1), k.minus, b));
}

// The 8 nibbles of four bytes minus 8, as fp16: low nibbles of bytes 0, 2, 1, 3, then the high ones.
__device__ __forceinline__ u32x4 nibbles(uint32_t w, const Kv4Const & k) {
    const half2 c0 = {_Float16(-1032.0f), _Float16(-1032.0f)}, c1 = {_Float16(-72.0f), _Float16(-72.0f)};
    const uint32_t x = w >> 8;
    u32x4 r;
    r[0] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2, (w & k.m0) | k.x0) + c0);  // 1024 + n
    r[1] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2, (x & k.m0) | k.x0) + c0);
    r[2] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2, (w & k.m1) | k.x1) + c1);  // 64 + n
    r[3] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2, (x & k.m1) | k.x1) + c1);
    return r;
}

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int s = 32; s >= 1; s >>= 1) x = fmaxf(x, __shfl_xor(x, s, WAVE));
    return x;
}

// How the sequences' records are dealt to workgroups: a sequence's `tiles` records from `first` on, in ranges of `per`; its ranges
// are number `slot` on of all. Every lane of a wave has the same.
struct Kv4Range {
    int first, tiles, per, slot, n;  // n: tokens of the sequence
    long long p0;
};

// Records that the tokens of a sequence see (r.p0 and r.n are set): from the first token's first position to the last one's own.
__device__ __forceinline__ void kv4_seen(const Kv4AttnArgs & a, Kv4Range & r) {
    const long long lo = r.p0 < 0 ? 0 : r.p0, hi = r.p0 + r.n < a.c.n_ctx ? r.p0 + r.n : a.c.n_ctx;  // positions of live tokens
    if (lo >= hi) {
        r.first = r.tiles = 0;
        return;
    }
    r.first = a.window && lo >= a.window ? int((lo - a.window + 1) / KV4_TILE) : 0;
    r.tiles = int((hi - 1) / KV4_TILE) - r.first + 1;
}

// A wave's sum (DPP: the rows of 16 upwards, then row 15 into the next and 31 into the upper half).
__device__ __forceinline__ int wave_total(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);  // row_shr:1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2 and 3
    return __builtin_amdgcn_readlane(x, 63);
}

// The ranges' length: all records over the ranges that the grid has room for, a sequence's last one being short. `most`: the longest
// sequence's records; up to half of KV4_ALONE, each sequence stays one range.
__device__ __forceinline__ int kv4_per(long long records, int ranges, int n_seq, int most, int hd) {
    int per = most;
    if (ranges > n_seq && most > KV4_ALONE / 2 / hd) {
        if (n_seq == 1) per = int((unsigned(records) + unsigned(ranges) - 1u) / unsigned(ranges));
        else per = int(ceil(double(records) / double(ranges - n_seq)));  // (quotients below 2^27 with fractions of at least 2^-16)
    }
    return per > KV4_LEAST ? per : KV4_LEAST;
}

// The sequence that range number `range` belongs to (BY_RANGE), or sequence s itself, with its ranges; false: no such range. A wave's
// lanes look at the sequences together, 64 at a time: first at all records, for the ranges' length, then at each sequence's ranges.
template <bool BY_RANGE>
__device__ __forceinline__ bool kv4_find(const Kv4AttnArgs & a, int range, int & s, Kv4Range & r) {
    if (a.t.n_seq == 1) {
        s = 0;
        kv4_span(a.t, 0, r.p0, r.n);
        kv4_seen(a, r);
        r.per = kv4_per(r.tiles, a.ranges, 1, r.tiles, a.c.head_dim);
        r.slot = 0;
        return (long long)(BY_RANGE ? range : 0) * r.per < r.tiles;
    }
    const int lane = threadIdx.x & 63;
    Kv4Range x;  // the lane's sequence
    const auto look = [&](int i) {
        x.p0 = x.n = 0;
        if (i < a.t.n_seq) kv4_span(a.t, i, x.p0, x.n);
        kv4_seen(a, x);
    };
    long long sum = 0;
    int most = 0;
    for (int i0 = 0; i0 < a.t.n_seq; i0 += 64) {
        look(i0 + lane);
        sum += x.tiles;
        most = max(most, x.tiles);
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
        sum += __shfl_xor(sum, d, WAVE);
        most = max(most, __shfl_xor(most, d, WAVE));
    }
    int per = kv4_per(sum, a.ranges, a.t.n_seq, most, a.c.head_dim);
    // That leaves room for a short range of every sequence; less will do. Worth its 0.3 us where the sequences are many (32 of up to
    // 8192, 32/8 heads of 128: 46 and 51 us).
    if (a.t.n_seq <= 64 && 8 * a.t.n_seq > a.ranges && per < most) {
        int low = max(int((sum + a.ranges - 1) / a.ranges), KV4_LEAST);
        for (int i = 0; i < 4 && low < per; ++i) {
            const int mid = (low + per) >> 1;
            if (wave_total(int(unsigned(x.tiles + mid - 1) / unsigned(mid))) <= a.ranges) per = mid;
            else low = mid + 1;
        }
    }
    int before = 0;
    for (int i0 = 0; i0 < a.t.n_seq; i0 += 64) {
        if (a.t.n_seq > 64) look(i0 + lane);  // (up to 64 sequences: as they are)
        const int mine = int(unsigned(x.tiles + per - 1) / unsigned(per));
        int upto = before + mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int y = __shfl_up(upto, d, WAVE);
            if (lane >= d) upto += y - before;
        }
        const int all = __shfl(upto, 63, WAVE);
        if (BY_RANGE ? range < all : s < i0 + 64) {
            const int l = BY_RANGE ? __ffsll(__ballot(upto > range)) - 1 : s - i0;
            s = i0 + l;
            r.slot = __shfl(upto - mine, l, WAVE);
            r.first = __shfl(x.first, l, WAVE);
            r.tiles = __shfl(x.tiles, l, WAVE);
            r.p0 = __shfl(int(x.p0), l, WAVE);
            r.n = __shfl(x.n, l, WAVE);
            r.per = per;
            return r.tiles > 0;
        }
        before = all;
    }
    return false;
}

// Four elements of an output row.
template <int HD>
__device__ __forceinline__ void kv4_out(const Kv4AttnArgs & a, size_t row, int hq, int e, f32x4 y, float l) {
    if (a.gate) {
        const f32x4 g = *reinterpret_cast<const f32x4 *>(a.gate + row * size_t(a.g_row) + size_t(hq) * size_t(a.g_head) + e);
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = sigmoid_(g[i]) * (y[i] / l);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = y[i] / l;
    }
    *reinterpret_cast<f32x4 *>(a.y + row * size_t(a.y_row) + size_t(hq) * HD + e) = y;
}

// Which rows and records a workgroup has: those of one sequence's range of records (kv4_attn_kernel).
struct Kv4Rows {
    int s, h, G, row0, p0, t_lo, t_hi, n_tok, n_head, window, range;  // tokens t_lo .. t_hi are in the rows and have positions
    int lo, hi;       // the positions that they see
    int first, last;  // the range's records of those
    bool alone;       // the sequence's one range
    const uint8_t * head;
    float * work;
    __device__ __forceinline__ int record(int at) const { return at; }
    // Row i of the workgroup: whether it has a position, its token's row and its q head (of some row with a position otherwise).
    __device__ __forceinline__ bool row(int i, size_t & token, int & hq) const {
        const int r = row0 + i, t = int(unsigned(r) / unsigned(G));
        const bool ok = t >= t_lo && t <= t_hi;
        token = size_t(s) * n_tok + (ok ? t : t_lo);
        hq = h * G + (ok ? r - t * G : 0);
        return ok;
    }
    // The positions from..to that row i sees, to -1: none.
    __device__ __forceinline__ void limits(int i, int & from, int & to) const {
        const int t = int(unsigned(row0 + i) / unsigned(G));
        const bool ok = t >= t_lo && t <= t_hi;
        to = ok ? p0 + t : -1;
        from = ok && window ? p0 + t - window + 1 : 0;
    }
    __device__ __forceinline__ bool sees(int p, int from, int to) const { return p >= from && p <= to; }
    __device__ __forceinline__ bool hidden(int p, int from, int to) const { return p < from || p > to; }
    __device__ __forceinline__ bool unseen(int p) const { return p < lo || p > hi; }  // by any row
    // Some row does not see all of the record at position `from`.
    __device__ __forceinline__ bool edge(int from) const { return from < (window ? p0 + t_hi - window + 1 : 0) || from + KV4_TILE - 1 > p0 + t_lo; }
    // This range's set of a row: [range][token][head][HD + 4], C and L behind the sums.
    __device__ __forceinline__ float * set(int, size_t token, int hq, int hd) const {
        return work + ((size_t(range) * n_tok + (token - size_t(s) * n_tok)) * n_head + hq) * (hd + 4);
    }
};

template <int HD, int NQ, typename Rows>
__device__ __forceinline__ void kv4_attend(const Kv4AttnArgs & a, const Rows & rows) {
    constexpr int NB = HD / 32, ROWS = 16 * NQ;
    // Blocks of 32 elements that the waves' sums are joined in at a time; threads of a row there.
    constexpr int JB = NQ == 1 ? NB : 1, PAD = 32 * JB + 4, JT = 256 / ROWS;
    constexpr size_t QBYTES = size_t(NQ) * NB * 2 * 1024, JBYTES = size_t(4) * ROWS * PAD * 4;
    __shared__ __align__(16) uint8_t both[QBYTES > JBYTES ? QBYTES : JBYTES];
    u32x4(*ql)[64] = reinterpret_cast<u32x4(*)[64]>(both);              // the queries' parts
    float(*part)[ROWS][PAD] = reinterpret_cast<float(*)[ROWS][PAD]>(both);  // later the waves' sums
    // The queries' parts that stay in registers, as many as leave room for two waves a SIMD (512 tokens at 7680, us with two, one and
    // none: 16/4 heads of 256 175.0 / 178.8 / 182.9, 32/8 of 128 no room / 161.3 / 164.9). The others are read from LDS for every
    // record.
    constexpr int QR = NQ == 1 || HD * NQ <= 128 ? 2 : 1;
    __shared__ float kqs[ROWS], cs[4][ROWS], ls[4][ROWS];
    __shared__ __align__(16) uint32_t scales[4][HD];  // a wave's record's key scales, then its value scales: [g][block][8] each
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, col = lane & 15;
    const int first = rows.first, last = rows.last;
    const uint8_t * head = rows.head;
    const Kv4Const k4;

    Kv4Tile<HD> tile;
    int at = first + wave;
    {
        const uint8_t * rec = head + size_t(rows.record(min(at, last))) * kv4_record(HD);
        tile.load_scales(rec, lane);
        tile.load_keys(rec, lane);
        tile.load_values(rec, lane);
    }
    // the queries to LDS, 16 threads a row with 4 elements at a time (elements in the order of nibbles())
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        constexpr int NP = HD >= 64 ? HD / 64 : 1;
        const int pc = tid & 15;
        size_t token;
        int hq;
        rows.row(n * 16 + (tid >> 4), token, hq);
        const float * src = a.q + token * size_t(a.q_row) + size_t(hq) * size_t(a.q_head);
        f32x4 x[NP];
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            x[i] = *reinterpret_cast<const f32x4 *>(src + ((pc + 16 * i) * 4 & (HD - 1)));
            top = fmaxf(fmaxf(fmaxf(top, fabsf(x[i][0])), fmaxf(fabsf(x[i][1]), fabsf(x[i][2]))), fabsf(x[i][3]));
        }
        top = fmaxf(top, dpp_f32<DPP_XOR1>(top));
        top = fmaxf(top, dpp_f32<DPP_XOR2>(top));
        top = fmaxf(top, dpp_f32<DPP_HALF_MIRROR>(top));
        top = fmaxf(top, dpp_f32<DPP_MIRROR>(top));
        // the largest element to 2^13..2^14 (rows of zeros: some power of two), times the mantissa and sign of the scale and log2(e), which
        // leaves it below 2^15.6; what brings the products back is a power of two, so scores times it are exact at any size, and a
        // row's largest score less itself is 0
        const int e = min(max(int((__float_as_uint(top) >> 23) & 255), 40), 254);
        const float up = __uint_as_float(uint32_t(127 + 13 + 127 - e) << 23) * (__builtin_amdgcn_frexp_mantf(a.scale) * 2.88539008177792681f);
        if (pc == 0) kqs[n * 16 + (tid >> 4)] = __uint_as_float(uint32_t(min(max(e - 14 + __builtin_amdgcn_frexp_expf(a.scale), 1), 254)) << 23);
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int piece = (pc + 16 * i) & (HD / 4 - 1), to = (piece & 3) * 16 + (tid >> 4);  // 8 block + 4 half + g
            u32x2 hi2, lo2;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                uint32_t hw, lw;
                split2(x[i][k] * up, x[i][k + 2] * up, hw, lw, k4);
                hi2[k] = hw;
                lo2[k] = lw;
            }
            u32x4 * dst = ql[(n * NB + (piece >> 3)) * 2];
            *reinterpret_cast<u32x2 *>(reinterpret_cast<uint8_t *>(dst + to) + (piece & 4) * 2) = hi2;
            *reinterpret_cast<u32x2 *>(reinterpret_cast<uint8_t *>(dst + 64 + to) + (piece & 4) * 2) = lo2;
        }
    }
    __syncthreads();
    u32x4 q[NQ][NB][QR];
    float kq[NQ];  // what brings the products back: the scale's power of two over the row's
    int my_lo[NQ], my_hi[NQ];
    f32x4 o[NQ][NB][2];
    float c[NQ], l[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        rows.limits(n * 16 + col, my_lo[n], my_hi[n]);
        kq[n] = kqs[n * 16 + col];
        c[n] = KV4_LOW;
        l[n] = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            o[n][b][0] = o[n][b][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < QR; ++i) q[n][b][i] = ql[(n * NB + b) * 2 + i][lane];
        }
    }
    bool sums = false;  // o holds something
    int e = 15;  // the value scales' exponent: the largest so far times 2^e is below 2^7 (scales below 2^-8 keep 2^15)
    for (; at <= last; at += 4) {
        const uint8_t * ahead = head + size_t(rows.record(min(at + 4, last))) * kv4_record(HD);  // (the last one again where there is none)
        const int from = rows.record(at) * KV4_TILE;
        const bool edge = rows.edge(from);
        if (edge) {  // positions that no row sees may never have been stored: their scales become 0
#pragma unroll
            for (int i = 0; i < Kv4Tile<HD>::NS; ++i) {
                const int p = from + Kv4Tile<HD>::at(lane, i);
                if (rows.unseen(p)) tile.d[i / 2] &= i & 1 ? 0x0000ffffu : 0xffff0000u;
            }
        }
        uint32_t dtop = 0;  // the largest value scale's magnitude, as fp16 bits
#pragma unroll
        for (int i = 0; i < Kv4Tile<HD>::NW; ++i) dtop = max(dtop, max(tile.d[i] & 0x7fffu, (tile.d[i] >> 16) & 0x7fffu));
        if (lane < 32) dtop = 0;
        if (__any(int(dtop >> 10) - 15 + e >= 7)) {  // a larger value scale: bring it to 2^6
            if (__any(dtop >= 0x7c00u)) {
                // Infinities or NaN among the value scales: their blocks come out NaN in the rows that see the positions, and they become 0 (a
                // weight of 0 times an infinity would be NaN in the other rows too)
                tile.stage(scales[wave], lane, half2{_Float16(1.0f), _Float16(1.0f)});
                wave_sync();
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const u32x4 vd = *reinterpret_cast<const u32x4 *>(&scales[wave][HD / 2 + (g * NB + b) * 4]);
#pragma unroll
                    for (int n = 0; n < NQ; ++n) {
                        bool hit = false;
#pragma unroll
                        for (int i = 0; i < 8; ++i) {  // word i / 2: positions 0 and 2, 1 and 3 of the lane's four, and 16 further
                            const int p = from + (i >> 2) * 16 + 4 * g + ((i >> 1) & 1) + 2 * (i & 1);
                            hit |= rows.sees(p, my_lo[n], my_hi[n]) && (vd[i >> 1] >> 16 * (i & 1) & 0x7c00u) == 0x7c00u;
                        }
                        unsigned long long hits = __ballot(hit);
                        hits |= hits >> 32;
                        const float add = uint32_t(hits | hits >> 16) >> col & 1 ? __builtin_nanf("") : 0.0f;
                        o[n][b][0] += add;
                        o[n][b][1] += add;
                    }
                }
                wave_sync();
                dtop = 0;
#pragma unroll
                for (int i = 0; i < 2 * Kv4Tile<HD>::NW; ++i) {
                    const uint32_t d = (tile.d[i >> 1] >> 16 * (i & 1)) & 0x7fffu;
                    if (lane >= 32 && d >= 0x7c00u) tile.d[i >> 1] &= i & 1 ? 0x0000ffffu : 0xffff0000u;
                    else if (lane >= 32) dtop = max(dtop, d);
                }
            }
            int top = max(int(dtop >> 10), 6 + 15 - e);
#pragma unroll
            for (int d = 32; d >= 1; d >>= 1) top = max(top, __shfl_xor(top, d, WAVE));
            const int e2 = 6 + 15 - top;  // (e where no finite scale asks for less)
            const float f = __uint_as_float(uint32_t(127 + e2 - e) << 23);
            e = e2;
            if (sums)
#pragma unroll
                for (int n = 0; n < NQ; ++n)
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        o[n][b][0] *= f;
                        o[n][b][1] *= f;
                    }
        }
        {
            const _Float16 f = lane < 32 ? _Float16(1.0f) : _Float16(__uint_as_float(uint32_t(127 + e) << 23));
            tile.stage(scales[wave], lane, half2{f, f});
        }
        wave_sync();
        tile.load_scales(ahead, lane);
        float sc[NQ][8];
        {
            f32x4 acc[NQ][2];
#pragma unroll
            for (int n = 0; n < NQ; ++n) acc[n][0] = acc[n][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const u32x4 kd = *reinterpret_cast<const u32x4 *>(&scales[wave][(g * NB + b) * 4]);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const u32x4 kk = nibbles(tile.k[u][b], k4);
#pragma unroll
                    for (int n = 0; n < NQ; ++n) {
                        f32x4 x = mfma(kk, q[n][b][0], f32x4{0.0f, 0.0f, 0.0f, 0.0f});
                        x = mfma(kk, QR == 2 ? q[n][b][QR - 1] : ql[(n * NB + b) * 2 + 1][lane], x);
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[n][u][i] = __builtin_fmaf(x[i], half_of(kd[2 * u + (i & 1)], i >> 1), acc[n][u][i]);
                    }
                }
            }
            tile.load_keys(ahead, lane);
#pragma unroll
            for (int n = 0; n < NQ; ++n)
#pragma unroll
                for (int i = 0; i < 8; ++i) sc[n][i] = acc[n][i >> 2][i & 3];
        }
        bool again = false;
        float top[NQ];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            if (edge)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int p = from + (i >> 2) * 16 + 4 * g + (i & 3);
                    if (rows.hidden(p, my_lo[n], my_hi[n])) sc[n][i] = -__builtin_inff();
                }
            top[n] = fmaxf(fmaxf(fmaxf(sc[n][0], sc[n][1]), fmaxf(sc[n][2], sc[n][3])), fmaxf(fmaxf(sc[n][4], sc[n][5]), fmaxf(sc[n][6], sc[n][7]))) * kq[n];
            again |= bool(__any(top[n] - c[n] > 9.0f));  // (not c + 9, which may round to the maximum)
        }
        if (again) {  // new maxima
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                float m = fmaxf(top[n], __shfl_xor(top[n], 16, WAVE));
                m = fmaxf(m, __shfl_xor(m, 32, WAVE));
                const float c2 = fmaxf(m - (m - c[n] > 13.0f ? 7.0f : 4.0f), c[n]), f = __builtin_amdgcn_exp2f(c[n] - c2);
                c[n] = c2;
                l[n] *= f;
                if (sums)
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        o[n][b][0] *= f;
                        o[n][b][1] *= f;
                    }
            }
        }
        sums = true;
        u32x4 ph[NQ], pl[NQ];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
#pragma unroll
            for (int i = 0; i < 8; ++i) sc[n][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[n][i], kq[n], -c[n]));
            l[n] += ((sc[n][0] + sc[n][1]) + (sc[n][2] + sc[n][3])) + ((sc[n][4] + sc[n][5]) + (sc[n][6] + sc[n][7]));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int i0 = (i >> 1) * 4 + (i & 1);
                uint32_t hi2, lo2;
                split2(sc[n][i0], sc[n][i0 + 2], hi2, lo2, k4);
                ph[n][i] = hi2;
                pl[n][i] = lo2;
            }
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const u32x4 vd = *reinterpret_cast<const u32x4 *>(&scales[wave][HD / 2 + (g * NB + b) * 4]);
            const u32x4 v0 = nibbles(tile.v[b][0], k4), v1 = nibbles(tile.v[b][1], k4);  // positions 0, 2, 1, 3 and 4, 6, 5, 7 of the lane's 8
            u32x4 dh[NQ], dl[NQ];
#pragma unroll
            for (int n = 0; n < NQ; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t h32 = ph[n][i], l32 = pl[n][i], d32 = vd[i];
                    const half2 h = __builtin_bit_cast(half2, h32), d = __builtin_bit_cast(half2, d32), x = h * d;
                    dh[n][i] = __builtin_bit_cast(uint32_t, x);
                    dl[n][i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(half2, l32), d, __builtin_elementwise_fma(h, d, -x)));
                }
#pragma unroll
            for (int u = 0; u < 2; ++u) {  // the lane's element, and the one 16 further
                const u32x4 w = {v0[2 * u], v0[2 * u + 1], v1[2 * u], v1[2 * u + 1]};
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    o[n][b][u] = mfma(w, dh[n], o[n][b][u]);
                    o[n][b][u] = mfma(w, dl[n], o[n][b][u]);
                }
            }
        }
        tile.load_values(ahead, lane);
        wave_sync();  // the scales have been read
    }
    // ---- the waves' sums joined ----
    const float down = __uint_as_float(uint32_t(127 - e) << 23);
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        l[n] += __shfl_xor(l[n], 16, WAVE);
        l[n] += __shfl_xor(l[n], 32, WAVE);
        if (g == 0) {
            cs[wave][n * 16 + col] = c[n];
            ls[wave][n * 16 + col] = l[n];
        }
    }
    const int rj = tid / JT;
    size_t token;
    int hq;
    const bool mine = rows.row(rj, token, hq);
    float f[4] = {0.0f, 0.0f, 0.0f, 0.0f}, C = KV4_LOW, L = 0.0f;
#pragma unroll
    for (int b0 = 0; b0 < NB; b0 += JB) {
        __syncthreads();  // (the queries, or the blocks before, have been read)
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int b = 0; b < JB; ++b)
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    *reinterpret_cast<f32x4 *>(&part[wave][n * 16 + col][b * 32 + u * 16 + 4 * g]) = o[n][b0 + b][u] * down;
        __syncthreads();
        if (b0 == 0) {
#pragma unroll
            for (int w = 0; w < 4; ++w) C = fmaxf(C, cs[w][rj]);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                f[w] = __builtin_amdgcn_exp2f(cs[w][rj] - C);
                L += ls[w][rj] * f[w];
            }
        }
        if (!mine) continue;
#pragma unroll 1
        for (int ej = tid % JT * 4; ej < 32 * JB; ej += 4 * JT) {
            f32x4 y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < 4; ++w) y += *reinterpret_cast<const f32x4 *>(&part[w][rj][ej]) * f[w];
            const int el = b0 * 32 + ej;
            if (rows.alone) {
                kv4_out<HD>(a, token, hq, el, y, L);
            } else {
                float * w = rows.set(rj, token, hq, HD);
                *reinterpret_cast<f32x4 *>(w + el) = y;
                if (el == 0) {
                    w[HD] = C;
                    w[HD + 1] = L;
                }
            }
        }
    }
}

template <int HD, int NQ>
__global__ __launch_bounds__(256, kv4_resident(HD, NQ)) void kv4_attn_kernel(Kv4AttnArgs a) {
    constexpr int ROWS = 16 * NQ;
    // Workgroup (KV head, group of rows behind it | range): the groups of one KV head, which read the same records, stay on an XCD or
    // a few. Rows of the KV head: token row / G, q head row % G
    const int G = a.group, h = int(unsigned(blockIdx.x) % unsigned(a.c.n_head_kv)), row0 = int(unsigned(blockIdx.x) / unsigned(a.c.n_head_kv)) * ROWS;
    const int range = blockIdx.y;
    int s = 0;
    Kv4Range r;
    if (!kv4_find<true>(a, range, s, r)) return;
    s = __builtin_amdgcn_readfirstlane(s);
    const int p0 = __builtin_amdgcn_readfirstlane(int(r.p0));
    // tokens -p0 (where p0 < 0) .. live - 1 have positions
    const int live = int(min((long long)__builtin_amdgcn_readfirstlane(r.n), (long long)a.c.n_ctx - p0));
    const int t_lo = max(int(unsigned(row0) / unsigned(G)), -p0), t_hi = min(int(unsigned(row0 + ROWS - 1) / unsigned(G)), live - 1);
    if (t_lo > t_hi) return;
    // the group's positions: lo .. hi, the rows' own ranges within them
    const int lo = a.window ? max(0, p0 + t_lo - a.window + 1) : 0, hi = p0 + t_hi;
    const int j = range - r.slot;
    const bool alone = __builtin_amdgcn_readfirstlane(int(r.tiles <= r.per));  // the sequence's one range
    const int first = __builtin_amdgcn_readfirstlane(max(r.first + j * r.per, lo / KV4_TILE));
    const int last = __builtin_amdgcn_readfirstlane(min(r.first + min((j + 1) * r.per, r.tiles) - 1, hi / KV4_TILE));
    if (first > last) return;  // none of the range's positions are seen
    kv4_attend<HD, NQ>(a, Kv4Rows{s, h, G, row0, p0, t_lo, t_hi, a.t.n_tok, a.n_head, a.window, range, lo, hi, first, last, alone, kv4_rec(a.c, s, h, 0), a.work});
}

// ---- attention with a prefix and sinks ----
// Segments: the groups' prefixes (number g), then the sequences' own caches (n_group + s). Each range of a segment's records has a
// workgroup for every KV head and group of rows.
struct Kv4Seg {
    // Records that some row sees: n_sink from 0 on, and those from `rest` on, `tiles` in all.
    int n_sink, rest, tiles;
};

__device__ __forceinline__ int kv4_group_of(const Kv4PartsArgs & x, int s) { return x.member_mul ? int(__umulhi(unsigned(s), x.member_mul)) : s; }
__device__ __forceinline__ int kv4_prefix(const Kv4PartsArgs & x, int group) { return max(0, min(x.pre_len[group], x.pre.n_ctx)); }

// The records of a segment of which the positions from .. to - 1 and the first `sinks` are seen.
__device__ __forceinline__ Kv4Seg kv4_records(int from, int to, int sinks) {
    if (to <= 0) return {0, 0, 0};
    const int end = (to - 1) / KV4_TILE + 1, rest = from >= to ? end : max(from, 0) / KV4_TILE;
    const int n_sink = min(sinks > 0 ? (min(sinks, to) - 1) / KV4_TILE + 1 : 0, rest);
    return {n_sink, rest, n_sink + end - rest};
}
// The positions of a sequence's live tokens in its own cache: low .. high - 1, none: high 0.
__device__ __forceinline__ void kv4_live(const Kv4PartsArgs & x, int s, int & low, int & high) {
    const int p0 = x.a.t.pos[s], n = x.a.t.num ? min(x.a.t.num[s], x.a.t.n_tok) : x.a.t.n_tok;
    low = max(p0, 0);
    high = n > 0 && p0 < x.a.c.n_ctx && p0 > -n ? p0 + min(n, p0 < 0 ? n : x.a.c.n_ctx - p0) : 0;
    high = min(high, x.a.c.n_ctx);
}
__device__ __forceinline__ Kv4Seg kv4_own_seg(const Kv4PartsArgs & x, int s) {
    int low, high;
    kv4_live(x, s, low, high);
    if (!x.a.window) return kv4_records(0, high, 0);
    // (a window begins at -2^31 + 1 or after)
    return kv4_records(low - x.a.window + 1, high, x.n_group ? x.sinks - kv4_prefix(x, kv4_group_of(x, s)) : x.sinks);
}
__device__ __forceinline__ Kv4Seg kv4_prefix_seg(const Kv4PartsArgs & x, int group) {
    const int n = kv4_prefix(x, group);
    if (!x.a.window || !n) return kv4_records(0, n, 0);
    int least = INT_MAX;  // the group's first live position
    for (int i = 0; i < x.members; ++i) {
        int low, high;
        kv4_live(x, group * x.members + i, low, high);
        if (high) least = min(least, low);
    }
    return least == INT_MAX ? Kv4Seg{0, 0, 0} : kv4_records(int(min((long long)n + least - x.a.window + 1, (long long)INT_MAX)), n, x.sinks);
}

// The workspace: every segment's first workgroup and number of ranges, then the workgroups' sets, [workgroup][row][HD + 4] each.
__host__ __device__ inline size_t kv4_table_floats(long long segs) { return size_t(segs + 1) / 2 * 4; }
__device__ __forceinline__ float * kv4_sets(const Kv4PartsArgs & x) { return x.a.work + kv4_table_floats(x.n_group + (long long)x.a.t.n_seq); }

// A segment's workgroups: its ranges times KV heads, 8 of these side by side, for every group of rows in turn: the groups that read the
// same records are on one XCD, close in time (workgroups are dealt to the 8 XCDs in turn).
struct Kv4Order {
    int n, groups;  // ranges times KV heads, groups of rows
    __device__ __forceinline__ int to(int q, int group) const {
        const int c = q & ~7;
        return c * groups + group * min(8, n - c) + (q & 7);
    }
    __device__ __forceinline__ void from(int k, int & q, int & group) const {
        const int c = int(unsigned(k) / unsigned(8 * groups)), rest = k - c * 8 * groups, width = min(8, n - 8 * c);
        group = int(unsigned(rest) / unsigned(width));
        q = 8 * c + rest - group * width;
    }
};

// What a workgroup has to do, the same in every lane: a group of rows and a KV head of a range of a segment.
struct Kv4Piece {
    int seg, head, group, from, to;  // records from .. to - 1 of the segment's
    Kv4Seg r;
};

// Sums of a wave's lanes up to each (DPP: within rows of 16, then row 15 into the next and 31 into the upper half).
__device__ __forceinline__ int wave_upto(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
    return x;
}
__device__ __forceinline__ float wave_sum_f(float x) {
    const auto step = [&](auto ctrl, auto rows) {
        x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), ctrl.value, rows.value, 0xf, rows.value == 0xf));
    };
    step(std::integral_constant<int, 0x111>(), std::integral_constant<int, 0xf>());
    step(std::integral_constant<int, 0x112>(), std::integral_constant<int, 0xf>());
    step(std::integral_constant<int, 0x114>(), std::integral_constant<int, 0xf>());
    step(std::integral_constant<int, 0x118>(), std::integral_constant<int, 0xf>());
    step(std::integral_constant<int, 0x142>(), std::integral_constant<int, 0xa>());
    step(std::integral_constant<int, 0x143>(), std::integral_constant<int, 0xc>());
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}
__device__ __forceinline__ int kv4_parts_of(int tiles, int per) { return int(unsigned(tiles + per - 1) / unsigned(per)); }

// Workgroup `id`'s piece; false: it has none. Every wave's lanes look at the segments together, 64 at a time (the groups, then the
// sequences): first at all records times workgroups, for the ranges' length, then for the segment that the workgroup falls into. The
// last workgroup, which mostly has no piece, writes the table of them.
__device__ __forceinline__ bool kv4_place(const Kv4PartsArgs & x, int id, Kv4Piece & piece) {
    const int lane = threadIdx.x & 63, n_group = x.n_group, n_seq = x.a.t.n_seq, heads = x.a.c.n_head_kv;
    const int pre_batches = (n_group + 63) / 64, batches = pre_batches + (n_seq + 63) / 64;
    const bool few = n_seq <= 64;  // at most one batch of each, looked at once
    const auto look = [&](int b) {
        const int i = (b < pre_batches ? b : b - pre_batches) * 64 + lane;
        if (b < pre_batches) return i < n_group ? kv4_prefix_seg(x, i) : Kv4Seg{0, 0, 0};
        return i < n_seq ? kv4_own_seg(x, i) : Kv4Seg{0, 0, 0};
    };
    Kv4Seg pre = {0, 0, 0}, own = {0, 0, 0};
    if (few) {
        own = look(pre_batches);
        if (n_group) pre = look(0);
    }
    const auto seg = [&](int b) { return few ? b < pre_batches ? pre : own : look(b); };
    int per = 1 << 30;
    if (!x.whole) {
        float sum = 0.0f;
        if (few) {
            sum = float(own.tiles) * float(x.own_units) + (n_group ? float(pre.tiles) * float(x.pre_units) : 0.0f);
        } else {
            double all = 0.0;
            for (int b = 0; b < batches; ++b) all += double(seg(b).tiles) * (b < pre_batches ? x.pre_units : x.own_units);
            sum = float(all);
        }
        // (roundings to FP32 are within 2^-17: the ranges are never more than the target and one a segment)
        const float each = wave_sum_f(sum) * (1.00002f / float(x.target));
        per = max(each < 1e9f ? int(each) + 1 : 1 << 30, KV4_LEAST);
        // That leaves room for a short range of every segment, and a few workgroups that start when the others are done cost more
        // than they bring: the shortest ranges, nearly, that are all there at once (us with the ones above and so: 30 and 25 at 32
        // sequences behind 8192, 32/8 heads of 128, 22 and 18 at windows of 1024 of them; twice as many ranges 35 and 24).
        if (few)
            for (int k = 0, low = per, high = 2 * min(per, 1 << 29); k < 5 && low < high; ++k) {
                const int mid = k ? (low + high) >> 1 : low;
                const int n = kv4_parts_of(own.tiles, mid) * x.own_units + (n_group ? kv4_parts_of(pre.tiles, mid) * x.pre_units : 0);
                const bool fits = __builtin_amdgcn_readlane(wave_upto(n), 63) <= x.target;
                per = fits ? mid : per;
                if (fits) high = mid;
                else low = mid + 1;
                if (!fits && k == 4) per = high;
            }
    }
    const bool table = id == int(gridDim.x) - 1 && x.a.work;
    bool found = false;
    int before = 0;
    for (int b = 0; b < batches; ++b) {
        const Kv4Seg y = seg(b);
        const bool is_pre = b < pre_batches;
        const int units = is_pre ? x.pre_units : x.own_units, n = kv4_parts_of(y.tiles, per), upto = wave_upto(n * units);
        const int all = __builtin_amdgcn_readlane(upto, 63);
        if (table) {
            const int i = (is_pre ? b : b - pre_batches) * 64 + lane;
            if (threadIdx.x < 64 && i < (is_pre ? n_group : n_seq))
                reinterpret_cast<int2 *>(x.a.work)[(is_pre ? 0 : n_group) + i] = int2{before + upto - n * units, n};
        }
        if (!found && id - before < all) {
            const int l = __ffsll(__ballot(before + upto > id)) - 1;
            const auto get = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
            const int k = id - before - get(upto - n * units), m = get(n), tiles = get(y.tiles);
            int q;
            Kv4Order{m * heads, is_pre ? x.pre_groups : x.own_groups}.from(k, q, piece.group);
            const int j = int(unsigned(q) / unsigned(heads)), each = int(unsigned(tiles) / unsigned(m)), more = tiles - each * m;
            piece.seg = (is_pre ? b * 64 : n_group + (b - pre_batches) * 64) + l;
            piece.head = q - j * heads;
            piece.r = {get(y.n_sink), get(y.rest), tiles};
            piece.from = each * j + min(j, more);  // ranges of a segment are alike
            piece.to = piece.from + each + (j < more);
            found = true;
            if (!table) return true;
        }
        before += all;
    }
    return found;
}

// The rows and records of kv4_parts_kernel's workgroup.
struct Kv4PartRows {
    int h, G, row0, sink;
    int lo, hi;                       // positions (of the segment's cache) that some row sees, besides the first `sink`
    int lo_most, hi_least;            // every row sees those
    int first, last, n_sink, skip;    // records: `first` on, from number n_sink on `skip` further
    bool alone, pre, windowed;
    int len, window;
    const uint8_t * head;
    float * sets;
    const int2 * at;                  // in LDS: a row's token row (-1: none) and place in its own cache

    template <int ROWS>
    __device__ __forceinline__ bool find(const Kv4PartsArgs & x, const Kv4Piece & p, int2 * at_) {
        const Kv4AttnArgs & a = x.a;
        const int tid = threadIdx.x, n_group = x.n_group, seg = __builtin_amdgcn_readfirstlane(p.seg);
        pre = seg < n_group;
        const int id = pre ? seg : seg - n_group, members = pre ? x.members : 1;
        G = a.group;
        h = __builtin_amdgcn_readfirstlane(p.head);
        row0 = __builtin_amdgcn_readfirstlane(p.group) * ROWS;
        len = n_group ? __builtin_amdgcn_readfirstlane(kv4_prefix(x, pre ? id : kv4_group_of(x, id))) : 0;
        window = a.window;
        windowed = window != 0;
        sink = !windowed ? 0 : pre ? min(x.sinks, len) : max(x.sinks - len, 0);
        // every lane a row (ROWS are at most 64), the workgroup's positions from all of them
        const int rows = members * a.t.n_tok * G, i = tid & (ROWS - 1);
        const bool in = row0 + i < rows;
        const int token = id * members * a.t.n_tok + (G == 1 ? in ? row0 + i : 0 : int(unsigned(in ? row0 + i : 0) / unsigned(G)));
        const int sq = a.t.n_tok == 1 ? token : int(unsigned(token) / unsigned(a.t.n_tok)), t = token - sq * a.t.n_tok;
        long long p0;
        int n;
        kv4_span(a.t, sq, p0, n);
        const bool ok = in && t < n && p0 + t >= 0 && p0 + t < a.c.n_ctx;
        const int place = int(p0 + t);
        if (tid < ROWS) at_[tid] = int2{ok ? token : -1, place};
        at = at_;
        int from = 0, to = -1;
        if (ok) span(place, from, to);
        int v[4] = {ok ? from : INT_MAX, ok ? -to : INT_MAX, ok ? -from : INT_MAX, ok ? to : INT_MAX};
#pragma unroll
        for (int d = 1; d < 64; d <<= 1)
            if (d < ROWS)
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = min(v[k], __shfl_xor(v[k], d, WAVE));
        lo = __builtin_amdgcn_readfirstlane(v[0]);
        hi = -__builtin_amdgcn_readfirstlane(v[1]);
        lo_most = -__builtin_amdgcn_readfirstlane(v[2]);
        hi_least = __builtin_amdgcn_readfirstlane(v[3]);
        if (hi_least == INT_MAX) return false;  // no row has a position
        // the range's records of the sinks, then those behind them, as far as the rows see any
        const Kv4Seg r = {__builtin_amdgcn_readfirstlane(p.r.n_sink), __builtin_amdgcn_readfirstlane(p.r.rest), __builtin_amdgcn_readfirstlane(p.r.tiles)};
        const int f = __builtin_amdgcn_readfirstlane(p.from), e = __builtin_amdgcn_readfirstlane(p.to), end = hi / KV4_TILE + 1;
        const int s1 = min(min(e, r.n_sink), end);
        int b0 = max(f, r.n_sink) - r.n_sink + r.rest;
        const int b1 = min(e - r.n_sink + r.rest, end);
        if ((long long)b0 * KV4_TILE >= sink) b0 = max(b0, lo / KV4_TILE);  // (there are sinks behind it otherwise)
        const int sinks = max(s1 - f, 0), others = max(b1 - b0, 0);
        first = sinks ? f : b0;
        last = first + sinks + others - 1;
        n_sink = sinks ? f + sinks : INT_MAX;
        skip = sinks ? b0 - (f + sinks) : 0;
        alone = !a.work || (!len && r.tiles == e - f);
        head = pre ? kv4_rec(x.pre, id, h, 0) : kv4_rec(a.c, id, h, 0);
        sets = a.work ? kv4_sets(x) + size_t(blockIdx.x) * x.rows * (a.c.head_dim + 4) : nullptr;
        __syncthreads();  // the rows' places are there
        if (first <= last) return true;
        if (!alone && tid < ROWS && at[tid].x >= 0) {  // the rows see nothing of the range
            sets[tid * (a.c.head_dim + 4) + a.c.head_dim] = KV4_LOW;
            sets[tid * (a.c.head_dim + 4) + a.c.head_dim + 1] = 0.0f;
        }
        return false;
    }
    // The positions of the segment that a token at that place sees, besides the sinks.
    __device__ __forceinline__ void span(int place, int & from, int & to) const {
        to = pre ? len - 1 : place;
        from = windowed ? int(min(max((pre ? (long long)len : 0ll) + place - window + 1, 0ll), (long long)INT_MAX - 1)) : 0;
    }
    __device__ __forceinline__ int record(int i) const { return i < n_sink ? i : i + skip; }
    __device__ __forceinline__ bool row(int i, size_t & token, int & hq) const {
        const int t = at[i].x;
        token = size_t(max(t, 0));
        hq = t < 0 ? 0 : h * G + int(unsigned(row0 + i) % unsigned(G));
        return t >= 0;
    }
    __device__ __forceinline__ void limits(int i, int & from, int & to) const {
        const int2 x = at[i];
        from = 0;
        to = -1;
        if (x.x >= 0) span(x.y, from, to);
    }
    __device__ __forceinline__ bool sees(int p, int from, int to) const { return (p >= from || p < sink) && p <= to; }
    __device__ __forceinline__ bool hidden(int p, int from, int to) const { return !sees(p, from, to); }
    __device__ __forceinline__ bool unseen(int p) const { return (p < lo && p >= sink) || p > hi; }
    __device__ __forceinline__ bool edge(int from) const { return (from < lo_most && from + KV4_TILE > sink) || from + KV4_TILE - 1 > hi_least; }
    __device__ __forceinline__ float * set(int i, size_t, int, int hd) const { return sets + size_t(i) * (hd + 4); }
};

// Times (rocprofv3): 32 sequences behind 8192 positions and up to 1024 of their own, 32/8 heads of 128 27 us, two groups of 16 behind
// 30000, 16/4 heads of 256 72 us (a wave takes 2.6 to 3.3 us for a record, with one or two waves a SIMD: 600 instructions, one after
// another); windows of 1024 and 64 sinks of 32 sequences, 32/8 heads of 128 18 us; of 512 tokens, 16/4 of 256 40 us (35 in calls one after
// another); 4 sequences behind 512 positions 10.5 us, a chain of four trips to memory around one record. A group's rows are taken as many
// at a time as one sequence's are (kv4_nq), whatever its members. With all members' rows counted, up to 32 or 64, a call alone in a graph:
// 32 sequences behind 8192, 32/8 heads of 128, 35.0 and 38.9 us, 15 of 4 tokens behind 1503, heads of 64, 16.9 and 22.3; but 64 behind
// 30000 138 and 113, of heads of 64 87 and 67.
template <int HD, int NQ>
__global__ __launch_bounds__(256, kv4_resident(HD, NQ)) void kv4_parts_kernel(Kv4PartsArgs x) {
    __shared__ int2 at[16 * NQ];
    Kv4Piece p;
    Kv4PartRows rows;
    if (kv4_place(x, int(blockIdx.x), p) && rows.find<16 * NQ>(x, p, at)) kv4_attend<HD, NQ>(x.a, rows);
}

// Workgroup (rows: q heads of tokens): WAVES waves a row, each its share of the row's sets, lanes HD / 4 to a set; WAVES 1: four rows
// a workgroup.
template <int HD, int WAVES>
__global__ __launch_bounds__(256) void kv4_parts_join_kernel(Kv4PartsArgs x) {
    constexpr int PER = HD / 4, SETS = 64 / PER, AHEAD = 4;
    __shared__ float cl[4][2];
    __shared__ __align__(16) float part[4][HD];
    const Kv4AttnArgs & a = x.a;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane / PER, e = lane % PER * 4;
    const long long all = (long long)a.t.n_seq * a.t.n_tok * a.n_head, at = WAVES == 1 ? blockIdx.x * 4ll + wave : blockIdx.x;
    if (at >= all) return;
    const int token = int(unsigned(at) / unsigned(a.n_head)), hq = int(at) - token * a.n_head, s = int(unsigned(token) / unsigned(a.t.n_tok)), t = token - s * a.t.n_tok;
    const int n_group = x.n_group, group = n_group ? kv4_group_of(x, s) : 0, G = a.group, h = int(unsigned(hq) / unsigned(G));
    const int2 * table = reinterpret_cast<const int2 *>(a.work);
    const int2 own = table[n_group + s], pre = n_group ? table[group] : int2{0, 0};
    const int len = n_group ? kv4_prefix(x, group) : 0;
    long long p0;
    int n_tok;
    kv4_span(a.t, s, p0, n_tok);
    if (t >= n_tok || p0 + t < 0 || p0 + t >= a.c.n_ctx || (!len && own.y == 1)) return;
    // its row in its workgroups: those of the sequence's own ranges and those of the prefix's
    constexpr size_t SET = HD + 4;
    const int orow = t * G + hq - h * G, prow = orow + (s - group * x.members) * a.t.n_tok * G;
    const int og = int(unsigned(orow) / unsigned(x.rows)), pg = n_group ? int(unsigned(prow) / unsigned(x.rows)) : 0;
    const Kv4Order oo{own.y * a.c.n_head_kv, x.own_groups}, po{pre.y * a.c.n_head_kv, x.pre_groups};
    const float * sets = kv4_sets(x);
    const int n = pre.y + own.y, n0 = WAVES == 1 ? 0 : n * wave / WAVES, n1 = WAVES == 1 ? n : n * (wave + 1) / WAVES;
    const auto set = [&](int j) {
        const bool first = j < pre.y;
        const int q = (first ? j : j - pre.y) * a.c.n_head_kv + h;
        const int k = first ? pre.x + po.to(q, pg) : own.x + oo.to(q, og), row = first ? prow - pg * x.rows : orow - og * x.rows;
        return sets + (size_t(k) * x.rows + row) * SET;
    };
    f32x4 y = {0.0f, 0.0f, 0.0f, 0.0f};
    float C = KV4_LOW, L = 0.0f;
    for (int b = n0; b < n1; b += 64) {  // 64 sets (often all) at a time: their statistics and the first sums read together
        const float2 c = b + lane < n1 ? *reinterpret_cast<const float2 *>(set(b + lane) + HD) : float2{KV4_LOW, 0.0f};
        const int m = min(n1 - b, 64);
        f32x4 v[AHEAD];
        const auto fetch = [&](int j0) {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i)
                v[i] = j0 + i * SETS < m ? *reinterpret_cast<const f32x4 *>(set(b + j0 + i * SETS) + e) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        };
        fetch(sub);
        const float top = fmaxf(wave_max(c.x), C), old = __builtin_amdgcn_exp2f(C - top), f = __builtin_amdgcn_exp2f(c.x - top);
        C = top;
        L = L * old + c.y * f;  // the lane's own sets'
        y *= old;
        for (int j0 = sub; j0 < m + sub; j0 += AHEAD * SETS) {  // (as often in every lane)
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int j = (j0 + i * SETS) & 63;
                const float fj = __shfl(f, j, WAVE), lj = __shfl(c.y, j, WAVE);
                if (j0 + i * SETS < m && !(lj == 0.0f)) y += v[i] * fj;  // (sets of nothing have no sums)
            }
            if (j0 + AHEAD * SETS < m + sub) fetch(j0 + AHEAD * SETS);
        }
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) L += __shfl_xor(L, d, WAVE);
#pragma unroll
    for (int d = 32; d >= PER; d >>= 1)
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] += __shfl_xor(y[i], d, WAVE);
    if constexpr (WAVES > 1) {
        if (lane == 0) {
            cl[wave][0] = C;
            cl[wave][1] = L;
        }
        if (sub == 0) *reinterpret_cast<f32x4 *>(&part[wave][e]) = y;
        __syncthreads();
        if (wave) return;
        float top = KV4_LOW;
        for (int w = 0; w < WAVES; ++w) top = fmaxf(top, cl[w][0]);
        y = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        L = 0.0f;
        for (int w = 0; w < WAVES; ++w) {
            const float f = __builtin_amdgcn_exp2f(cl[w][0] - top);
            y += *reinterpret_cast<const f32x4 *>(&part[w][e]) * f;
            L += cl[w][1] * f;
        }
    }
    if (sub == 0) kv4_out<HD>(a, token, hq, e, y, L);
}

// Workgroup (q head and EL of its elements, token, sequence): the sets of a sequence with several ranges. The factors of all sets
// first, then EL / 4 threads a set, 1024 / EL sets at a time. 128 sets of 16 heads of 256 (2.1 MB): 4.4 us with 64 elements a
// workgroup, two trips to memory in a row (positions, sets).
template <int HD, int EL>
__global__ __launch_bounds__(256) void kv4_join_kernel(Kv4AttnArgs a) {
    constexpr int PER = EL / 4, SETS = 256 / PER;
    __shared__ float f[KV4_GROUPS], red[2][4];
    __shared__ __align__(16) float part[SETS][EL];
    const int hq = blockIdx.x / (HD / EL), e0 = blockIdx.x % (HD / EL) * EL, t = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int s = blockIdx.z;
    Kv4Range r;
    if (!kv4_find<false>(a, 0, s, r)) return;
    const long long p = r.p0 + t;
    if (r.tiles <= r.per || t >= r.n || p < 0 || p >= a.c.n_ctx) return;
    // the ranges that hold positions this token sees
    const int j0 = ((a.window && p >= a.window ? int((p - a.window + 1) / KV4_TILE) : 0) - r.first) / r.per;
    const int n = (int(p / KV4_TILE) - r.first) / r.per - j0 + 1;
    const size_t step = size_t(a.t.n_tok) * a.n_head * (HD + 4);
    const float * w = a.work + (size_t(r.slot + j0) * a.t.n_tok + t) * a.n_head * (HD + 4) + size_t(hq) * (HD + 4);
    // every first read before the first use: the sets' c and sums of weights, AHEAD sets of the thread's elements
    constexpr int STATS = KV4_GROUPS / 256, AHEAD = 8;
    static_assert(KV4_GROUPS % 256 == 0, "a thread's sets");
    float2 cl[STATS];
#pragma unroll
    for (int i = 0; i < STATS; ++i) cl[i] = tid + 256 * i < n ? *reinterpret_cast<const float2 *>(w + (tid + 256 * i) * step + HD) : float2{KV4_LOW, 0.0f};
    const int e = tid % PER * 4, j1 = tid / PER;
    f32x4 x[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) x[i] = j1 + i * SETS < n ? *reinterpret_cast<const f32x4 *>(w + (j1 + i * SETS) * step + e0 + e) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float C = KV4_LOW, L = 0.0f;
#pragma unroll
    for (int i = 0; i < STATS; ++i) C = fmaxf(C, cl[i].x);
    C = wave_max(C);
    if (lane == 0) red[0][wave] = C;
    __syncthreads();
    C = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
#pragma unroll
    for (int i = 0; i < STATS; ++i) {
        const float g = __builtin_amdgcn_exp2f(cl[i].x - C);
        if (tid + 256 * i < n) f[tid + 256 * i] = g;
        L += cl[i].y * g;
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) L += __shfl_xor(L, d, WAVE);
    if (lane == 0) red[1][wave] = L;
    __syncthreads();
    f32x4 y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
        if (j1 + i * SETS < n) y += x[i] * f[j1 + i * SETS];
#pragma unroll 4
    for (int j = j1 + AHEAD * SETS; j < n; j += SETS) y += *reinterpret_cast<const f32x4 *>(w + j * step + e0 + e) * f[j];
    *reinterpret_cast<f32x4 *>(&part[tid / PER][e]) = y;
    __syncthreads();
    if (tid >= PER) return;
#pragma unroll
    for (int i = 1; i < SETS; ++i) y += *reinterpret_cast<const f32x4 *>(&part[i][e]);
    kv4_out<HD>(a, size_t(s) * a.t.n_tok + t, hq, e0 + e, y, (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]));
}

// The same for many rows (q heads of tokens): a wave `per_wave` of them one after another, its lanes HD / 4 to a set. What each
// workgroup does before its first row (finding the sequence's ranges, 2 us) is shared by its rows.
template <int HD>
__global__ __launch_bounds__(256) void kv4_join_rows_kernel(Kv4AttnArgs a, int per_wave) {
    constexpr int PER = HD / 4, SETS = 64 / PER;
    const int lane = threadIdx.x & 63, sub = lane / PER, e = lane % PER * 4;
    int s = blockIdx.y;
    Kv4Range r;
    if (!kv4_find<false>(a, 0, s, r) || r.tiles <= r.per) return;
    const int rows = a.t.n_tok * a.n_head, row0 = int(blockIdx.x * 4 + (threadIdx.x >> 6)) * per_wave;
    const size_t step = size_t(a.t.n_tok) * a.n_head * (HD + 4);
    for (int row = row0; row < min(row0 + per_wave, rows); ++row) {
        const int t = int(unsigned(row) / unsigned(a.n_head)), hq = row - t * a.n_head;
        const long long p = r.p0 + t;
        if (t >= r.n || p < 0 || p >= a.c.n_ctx) continue;
        const int k0 = ((a.window && p >= a.window ? int((p - a.window + 1) / KV4_TILE) : 0) - r.first) / r.per;
        const int n = (int(p / KV4_TILE) - r.first) / r.per - k0 + 1;
        const float * w = a.work + size_t(r.slot + k0) * step + size_t(row) * (HD + 4);
        f32x4 y = {0.0f, 0.0f, 0.0f, 0.0f};
        float C = KV4_LOW, L = 0.0f;
        for (int b = 0; b < n; b += 64) {  // 64 sets (often all) at a time
            const float2 cl = b + lane < n ? *reinterpret_cast<const float2 *>(w + (b + lane) * step + HD) : float2{KV4_LOW, 0.0f};
            const float top = fmaxf(wave_max(cl.x), C), old = __builtin_amdgcn_exp2f(C - top), f = __builtin_amdgcn_exp2f(cl.x - top);
            C = top;
            L = L * old + cl.y * f;  // the lane's own sets'
            y *= old;
            const int m = min(n - b, 64);
            for (int j0 = sub; j0 < m + sub; j0 += 4 * SETS) {  // (as often in every lane)
                f32x4 x[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    x[i] = j0 + i * SETS < m ? *reinterpret_cast<const f32x4 *>(w + (b + j0 + i * SETS) * step + e) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float fj = __shfl(f, (j0 + i * SETS) & 63, WAVE);
                    if (j0 + i * SETS < m) y += x[i] * fj;
                }
            }
        }
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) L += __shfl_xor(L, d, WAVE);
#pragma unroll
        for (int d = 32; d >= PER; d >>= 1)
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] += __shfl_xor(y[i], d, WAVE);
        if (sub == 0) kv4_out<HD>(a, size_t(s) * a.t.n_tok + t, hq, e, y, L);
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

hipError_t launch_kv4_append(const Kv4AppendArgs & a, hipStream_t s) {
    return by_dim(a.c.head_dim, [&](auto hd) {
        GQ_LAUNCH(kv4_append_kernel<hd.value>, dim3(a.n_head + a.c.n_head_kv, a.t.n_tok, a.t.n_seq), dim3(256), 0, s, a);
    });
}

hipError_t launch_kv4_store(const Kv4RowsArgs & a, hipStream_t s) {
    const unsigned span = unsigned((a.t.n_tok + KV4_TILE - 2) / KV4_TILE + 1);  // records that n_tok positions can touch
    return by_dim(a.c.head_dim, [&](auto hd) {
        constexpr unsigned parts = 2 * (hd.value < 128 ? 1 : hd.value / 128);
        GQ_LAUNCH(kv4_store_kernel<hd.value>, dim3(span * parts, a.c.n_head_kv, a.t.n_seq), dim3(KV4_STORE), 0, s, a);
    });
}

// Rows (KV heads of tokens) from which on the records are read whole, where a sequence has tokens for half a record; us with single
// rows and records, and the storing before: 6.6 and 7.6 at 400 rows, 8.5 and 8.8 at 2048, 9.4 and 8.1 at 4096, 16.7 and 14.2 at 7932.
constexpr int KV4_RECORDS = 2048;
hipError_t launch_kv4_load(const Kv4RowsArgs & a, hipStream_t s) {
    const unsigned span = unsigned((a.t.n_tok + KV4_TILE - 2) / KV4_TILE + 1);  // records that n_tok positions can touch
    return by_dim(a.c.head_dim, [&](auto hd) {
        if (a.t.n_tok >= KV4_TILE / 2 && (long long)a.t.n_seq * a.t.n_tok * a.c.n_head_kv >= KV4_RECORDS)
            GQ_LAUNCH(kv4_load_records_kernel<hd.value>, dim3(2 * span, a.c.n_head_kv, a.t.n_seq), dim3(256), 0, s, a);
        else GQ_LAUNCH(kv4_load_kernel<hd.value>, dim3(a.t.n_tok, a.c.n_head_kv, a.t.n_seq), dim3(256), 0, s, a);
    });
}

// Groups of 16 rows that a workgroup takes: as many as there are, up to what the registers hold.
static int kv4_nq(int hd, int n_tok, int per_kv) {
    const long long rows = n_tok * (long long)per_kv;
    return rows <= 16 || hd == 256 ? 1 : rows <= 32 || hd == 128 ? 2 : 4;
}

// How many ranges a call's records are dealt to: as many as give the workgroups that are resident together, but at least one range a
// sequence, and no more than KV4_LEAST records each give; one a sequence where no position needs more.
int kv4_ranges(const Kv4Cache & c, int n_seq, int n_tok, int n_head) {
    if (kv4_tiles(c.n_ctx) <= KV4_ALONE / c.head_dim) return n_seq;
    const int per_kv = n_head / c.n_head_kv, nq = kv4_nq(c.head_dim, n_tok, per_kv), rows = 16 * nq;
    const int groups = 256 * kv4_resident(c.head_dim, nq);
    const long long units = (n_tok * (long long)per_kv + rows - 1) / rows * c.n_head_kv;
    const long long records = (long long)n_seq * kv4_tiles(c.n_ctx), most = (long long)n_seq * ((kv4_tiles(c.n_ctx) + KV4_LEAST - 1) / KV4_LEAST);
    long long ranges = std::max<long long>(n_seq, std::min(groups / units, most));
    // Few long ranges for sequences of unlike lengths come out unlike themselves: twice as many (3 sequences of 96 tokens at up to
    // 10776, 32/8 heads of 128: 53 us, 74 without). Of others twice as many are no gain (182 and 175 us at one of 512 at 7680, 16/4 heads
    // of 256; 25.1 and 23.7 at 3 of 360 at up to 1451, 8 heads of 64; 28.0 and 21.8 at 8 of 8 at up to 8184, 16/4 heads of 128).
    if (n_seq > 1 && records >= 128 * ranges) ranges = std::max<long long>(ranges, std::min<long long>(2 * ranges, KV4_GROUPS));
    return int(std::min<long long>(ranges, 65535));
}

size_t kv4_work_floats(const Kv4Cache & c, int n_seq, int n_tok, int n_head) {
    const int ranges = kv4_ranges(c, n_seq, n_tok, n_head);
    return ranges > n_seq ? size_t(ranges) * n_tok * n_head * (c.head_dim + 4) : 0;
}

bool kv4_joins(const Kv4AttnArgs & a) { return a.work && kv4_ranges(a.c, a.t.n_seq, a.t.n_tok, a.n_head) > a.t.n_seq; }

// Rows (q heads of tokens) up to which each has workgroups of its own: several up to half as many. us with several, one, and a wave's
// share of one: 22.9 / 22.0 / 24.1 at 320 rows (20 tokens at 8172, 16/4 heads of 256), 12.9 / 12.9 / 12.6 at 320 (40 at 1411, 8 heads of 64),
// 22.1 / 20.8 / 20.9 at 512, 51.4 / 48.5 / 46.6 at 1024, 35.9 / 35.9 / 24.0 at 8640.
constexpr int KV4_FEW = 512;
hipError_t launch_kv4_attn(const Kv4AttnArgs & args, hipStream_t s) {
    Kv4AttnArgs a = args;
    const int per_kv = a.n_head / a.c.n_head_kv, nq = kv4_nq(a.c.head_dim, a.t.n_tok, per_kv);
    a.ranges = a.work ? kv4_ranges(a.c, a.t.n_seq, a.t.n_tok, a.n_head) : a.t.n_seq;
    a.group = per_kv;
    const dim3 grid(unsigned((a.t.n_tok * (long long)per_kv + 16 * nq - 1) / (16 * nq) * a.c.n_head_kv), unsigned(a.ranges));
    return by_dim(a.c.head_dim, [&](auto hd) {
        if (nq == 1) GQ_LAUNCH((kv4_attn_kernel<hd.value, 1>), grid, dim3(256), 0, s, a);
        if constexpr (hd.value < 256)
            if (nq == 2) GQ_LAUNCH((kv4_attn_kernel<hd.value, 2>), grid, dim3(256), 0, s, a);
        if constexpr (hd.value < 128)
            if (nq == 4) GQ_LAUNCH((kv4_attn_kernel<hd.value, 4>), grid, dim3(256), 0, s, a);
        if (a.ranges <= a.t.n_seq) return;
        const long long rows = a.t.n_tok * (long long)a.n_head, all = a.t.n_seq * rows;
        if (all <= KV4_FEW / 2) {
            constexpr int narrow = hd.value < 64 ? 32 : 64;
            GQ_LAUNCH((kv4_join_kernel<hd.value, narrow>), dim3(a.n_head * (hd.value / narrow), a.t.n_tok, a.t.n_seq), dim3(256), 0, s, a);
        } else if (all <= KV4_FEW) {
            GQ_LAUNCH((kv4_join_kernel<hd.value, hd.value>), dim3(a.n_head, a.t.n_tok, a.t.n_seq), dim3(256), 0, s, a);
        } else {
            const int per_wave = int(std::min<long long>(std::max<long long>(all / 4096, 1), 16));
            GQ_LAUNCH(kv4_join_rows_kernel<hd.value>, dim3(unsigned((rows + 4 * per_wave - 1) / (4 * per_wave)), a.t.n_seq), dim3(256), 0, s, a, per_wave);
        }
    });
}

// How a call with a prefix or sinks is launched: groups of 16 rows a workgroup, groups of those in a prefix's rows and in a sequence's,
// the workgroups that its ranges are dealt to and the most that they can come to (every segment's workgroups of one range more),
// and whether every segment is one range. That is so of short caches, and where the sequences' workgroups fill the device by themselves (us
// so and split: 64 sequences at up to 8192, 32/8 heads of 256, 172 and 177, all at 8191 245 and 245; 256 at up to 4096, 32/8 of 128, 157 and
// 164; 96 at up to 8192 139 and 137; a window of 1024 of 512 tokens, 16/4 of 256, 36.4 and 38.8). Rows are counted as n_tok says: one live
// token of 512 at 30000 waits 363 us for its four workgroups, 26 in a call of one token.
struct Kv4Plan {
    int nq, pre_groups, own_groups, target;
    bool whole;
    long long grid;
};
static Kv4Plan kv4_plan(const Kv4Cache & c, int n_group, int pre_ctx, int n_seq, int n_tok, int n_head, int window, int sinks) {
    const int members = n_group ? n_seq / n_group : 1, per_kv = n_head / c.n_head_kv;
    const long long rows = n_tok * (long long)per_kv;
    Kv4Plan p;
    p.nq = kv4_nq(c.head_dim, n_tok, per_kv);
    p.own_groups = int((rows + 16 * p.nq - 1) / (16 * p.nq));
    p.pre_groups = n_group ? int((rows * members + 16 * p.nq - 1) / (16 * p.nq)) : 0;
    p.target = 256 * kv4_resident(c.head_dim, p.nq);
    const long long own = (long long)p.own_groups * c.n_head_kv * n_seq, pre = (long long)p.pre_groups * c.n_head_kv * n_group;
    long long tiles = kv4_tiles(c.n_ctx);  // records of a sequence that its tokens see
    if (window) tiles = std::min(tiles, (long long)window / KV4_TILE + n_tok / KV4_TILE + 4 + sinks / KV4_TILE);
    p.whole = !n_group && (own >= p.target || tiles <= KV4_ALONE / c.head_dim);
    p.grid = own + pre + (p.whole ? 0 : p.target);
    if (!p.whole) {  // no more than the longest segments could have
        const auto most = [](int n_ctx) { return (kv4_tiles(n_ctx) + KV4_LEAST - 1) / KV4_LEAST; };
        p.grid = std::min(p.grid, own * most(c.n_ctx) + pre * most(pre_ctx));
    }
    return p;
}

// No less than any call needs that has as much of something as this one and no more of anything: of sequences, groups, positions and
// tokens. Fewer tokens may mean fewer rows a workgroup (nq), whose one group of rows is then full; groups of a prefix's rows are counted
// as if each prefix's last one held a single row; a call without a prefix needs nothing once its sequences' workgroups are the target
// or more, so no more than one less counts.
size_t kv4_parts_floats(const Kv4Cache & c, int n_group, int pre_ctx, int n_seq, int n_tok, int n_head) {
    const long long own_tiles = kv4_tiles(c.n_ctx), pre_tiles = kv4_tiles(pre_ctx), all_rows = n_tok * (long long)(n_head / c.n_head_kv);
    if (!n_group && own_tiles <= KV4_ALONE / c.head_dim) return 0;
    size_t floats = 0;
    for (int nq = 1, most_nq = kv4_nq(c.head_dim, n_tok, n_head / c.n_head_kv); nq <= most_nq; nq *= 2) {
        const long long size = 16 * nq, rows = nq < most_nq ? size : all_rows, target = 256 * kv4_resident(c.head_dim, nq);
        long long own = (rows + size - 1) / size * c.n_head_kv * n_seq;
        if (!n_group) own = std::min(own, target - 1);
        const long long pre = (rows * n_seq + (size - 1) * n_group) / size * c.n_head_kv;
        const auto ranges = [](long long tiles) { return (tiles + KV4_LEAST - 1) / KV4_LEAST; };
        const long long grid = n_group ? std::min(own + pre + target, own * ranges(own_tiles) + pre * ranges(pre_tiles)) : std::min(own + target, own * ranges(own_tiles));
        floats = std::max(floats, size_t(grid * size) * (c.head_dim + 4));
    }
    return kv4_table_floats((long long)n_group + n_seq) + floats;
}
bool kv4_parts_whole(const Kv4Cache & c, int n_group, int pre_ctx, int n_seq, int n_tok, int n_head) {
    return kv4_plan(c, n_group, pre_ctx, n_seq, n_tok, n_head, 0, 0).whole;
}
long long kv4_parts_grid(const Kv4Cache & c, int n_group, int pre_ctx, int n_seq, int n_tok, int n_head) {
    return kv4_plan(c, n_group, pre_ctx, n_seq, n_tok, n_head, 0, 0).grid;
}

hipError_t launch_kv4_parts(const Kv4PartsArgs & args, hipStream_t s) {
    Kv4PartsArgs x = args;
    Kv4AttnArgs & a = x.a;
    const Kv4Plan p = kv4_plan(a.c, x.pre.data ? a.t.n_seq / x.members : 0, x.pre.n_ctx, a.t.n_seq, a.t.n_tok, a.n_head, a.window, x.sinks);
    x.rows = 16 * p.nq;
    x.n_group = x.pre.data ? a.t.n_seq / x.members : 0;
    x.member_mul = x.members > 1 ? unsigned((0x100000000ull + unsigned(x.members) - 1) / unsigned(x.members)) : 0;  // (exact: s below 2^16)
    x.pre_groups = p.pre_groups;
    x.own_groups = p.own_groups;
    x.pre_units = p.pre_groups * a.c.n_head_kv;
    x.own_units = p.own_groups * a.c.n_head_kv;
    x.target = p.target;
    x.whole = p.whole;
    a.group = a.n_head / a.c.n_head_kv;
    const dim3 grid{unsigned(p.grid)};
    return by_dim(a.c.head_dim, [&](auto hd) {
        if (p.nq == 1) GQ_LAUNCH((kv4_parts_kernel<hd.value, 1>), grid, dim3(256), 0, s, x);
        if constexpr (hd.value < 256)
            if (p.nq == 2) GQ_LAUNCH((kv4_parts_kernel<hd.value, 2>), grid, dim3(256), 0, s, x);
        if constexpr (hd.value < 128)
            if (p.nq == 4) GQ_LAUNCH((kv4_parts_kernel<hd.value, 4>), grid, dim3(256), 0, s, x);
        if (p.whole) return;
        const long long rows = (long long)a.t.n_seq * a.t.n_tok * a.n_head;
        if (rows <= KV4_FEW) GQ_LAUNCH((kv4_parts_join_kernel<hd.value, 4>), dim3(unsigned(rows)), dim3(256), 0, s, x);
        else GQ_LAUNCH((kv4_parts_join_kernel<hd.value, 1>), dim3(unsigned((rows + 3) / 4)), dim3(256), 0, s, x);
    });
}

}  // namespace gq
