// Rotary positions (gq_rope.h).
#include "gq_device.h"
#include "gq_rope.h"

#include <algorithm>
#include <cmath>

namespace gq {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

// cos and sin of t full turns, times m. The whole turns are taken off in 64 bits (positions of 2^31 and a turn in six positions are
// 2^28.4 turns, good to 2^-25 of one there), then the nearest quarter; what is left, at most an eighth either way, goes into the
// Taylor series of sine and cosine (to x^13 / 13! and x^12 / 12!: 3e-14 and 2e-13), rounded to FP32 once at the end.
__device__ __forceinline__ float2 rope_turn(double t, double m) {
    t -= rint(t);
    const double q = rint(4.0 * t), x = (t - 0.25 * q) * 6.283185307179586, x2 = x * x;
    double s = 1.0 / 6227020800.0;
    s = __builtin_fma(s, x2, -1.0 / 39916800.0);
    s = __builtin_fma(s, x2, 1.0 / 362880.0);
    s = __builtin_fma(s, x2, -1.0 / 5040.0);
    s = __builtin_fma(s, x2, 1.0 / 120.0);
    s = __builtin_fma(s, x2, -1.0 / 6.0);
    s = __builtin_fma(s * x2, x, x) * m;
    double c = 1.0 / 479001600.0;
    c = __builtin_fma(c, x2, -1.0 / 3628800.0);
    c = __builtin_fma(c, x2, 1.0 / 40320.0);
    c = __builtin_fma(c, x2, -1.0 / 720.0);
    c = __builtin_fma(c, x2, 1.0 / 24.0);
    c = __builtin_fma(c, x2, -0.5);
    c = __builtin_fma(c, x2, 1.0) * m;
    const int k = int(q) & 3;
    const double a = k & 1 ? s : c, b = k & 1 ? c : s;
    return float2{float(k == 1 || k == 2 ? -a : a), float(k >= 2 ? -b : b)};
}

// Workgroup (token rows | heads): the angles of its rows once, to LDS, 64-bit work that all heads share; then its elements, WIDE in
// pieces of four pairs (or of 16 bytes that stay), else pair by pair. The first pieces are read before the angles are there. Memory
// bounds it.
template <bool WIDE, bool PAIRS>
__global__ __launch_bounds__(256) void rope_kernel(RotaryArgs a) {
    constexpr int AHEAD = 4, W = WIDE ? 4 : 1;
    __shared__ float2 cs[ROPE_MAX_DIM / 2];  // tokens * n_rot / 2 of them
    __shared__ int live[256];                // rows with a position
    const int tid = threadIdx.x, half = a.n_rot / 2, tail = a.head_dim - a.n_rot;
    const int per = half / W + tail / W;  // pieces of a head
    const int row0 = int(blockIdx.x) * a.tokens, rows = min(a.tokens, a.n_seq * a.n_tok - row0);
    const int head0 = int(blockIdx.y) * a.heads, heads = min(a.heads, a.a[a.n - 1].end - head0);
    const int items = rows * heads * per;

    struct Piece {
        const float * x;
        float * y;
        int r, c;  // row of the workgroup (-1: no piece), piece of the head
    };
    const auto find = [&](int i) {
        Piece p;
        const int rh = int(unsigned(i) / unsigned(per)), r = int(unsigned(rh) / unsigned(heads));
        int h = head0 + rh - r * heads, k = 0;
        p.c = i - rh * per;
        p.r = i < items ? r : -1;
#pragma unroll
        for (int j = 1; j < ROPE_ARRAYS; ++j)
            if (j < a.n && h >= a.a[j - 1].end) k = j;
        const RotaryArray & m = a.a[k];
        if (k) h -= a.a[k - 1].end;
        const long long row = row0 + r;
        p.x = m.x + row * m.x_row + h * m.x_head;
        p.y = m.y + row * m.y_row + h * m.y_head;
        if (p.x == p.y && p.c >= half / W) p.r = -1;  // in place: nothing to copy
        return p;
    };
    const auto load = [&](const Piece & p, float * v) {  // its pairs' first elements, then the second ones
        if (p.r < 0) return;
        const int o = p.c * W;
        if constexpr (WIDE) {
            f32x4 lo, hi;
            if (o >= half) {
                lo = *reinterpret_cast<const f32x4 *>(p.x + a.n_rot + o - half);
                hi = lo;
            } else if (PAIRS) {
                lo = *reinterpret_cast<const f32x4 *>(p.x + 2 * o);
                hi = *reinterpret_cast<const f32x4 *>(p.x + 2 * o + 4);
            } else {
                lo = *reinterpret_cast<const f32x4 *>(p.x + o);
                hi = *reinterpret_cast<const f32x4 *>(p.x + half + o);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = lo[e];
                v[4 + e] = hi[e];
            }
        } else {
            v[0] = p.x[o >= half ? a.n_rot + o - half : PAIRS ? 2 * o : o];
            v[1] = o >= half ? 0.0f : p.x[PAIRS ? 2 * o + 1 : half + o];
        }
    };
    const auto put = [&](const Piece & p, const float * v) {
        if (p.r < 0 || !live[p.r]) return;
        const int o = p.c * W;
        float z[2 * W];
        if (o < half) {
#pragma unroll
            for (int e = 0; e < W; ++e) {
                const float2 t = cs[p.r * half + o + e];
                const int i0 = WIDE && PAIRS ? 2 * e : e, i1 = WIDE && PAIRS ? 2 * e + 1 : W + e;
                z[i0] = v[i0] * t.x - v[i1] * t.y;
                z[i1] = v[i0] * t.y + v[i1] * t.x;
            }
        }
        if constexpr (WIDE) {
            if (o >= half) {
                *reinterpret_cast<f32x4 *>(p.y + a.n_rot + o - half) = f32x4{v[0], v[1], v[2], v[3]};
            } else {
                *reinterpret_cast<f32x4 *>(p.y + (PAIRS ? 2 * o : o)) = f32x4{z[0], z[1], z[2], z[3]};
                *reinterpret_cast<f32x4 *>(p.y + (PAIRS ? 2 * o + 4 : half + o)) = f32x4{z[4], z[5], z[6], z[7]};
            }
        } else if (o >= half) {
            p.y[a.n_rot + o - half] = v[0];
        } else {
            p.y[PAIRS ? 2 * o : o] = z[0];
            p.y[PAIRS ? 2 * o + 1 : half + o] = z[1];
        }
    };

    Piece p[AHEAD];
    float v[AHEAD][2 * W];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
        p[j] = find(tid + 256 * j);
        load(p[j], v[j]);
    }
    for (int i = tid; i < rows * half; i += 256) {
        const int r = int(unsigned(i) / unsigned(half)), row = row0 + r, s = int(unsigned(row) / unsigned(a.n_tok));
        const long long at = (long long)a.pos[s] + (row - s * a.n_tok);
        cs[i] = rope_turn(double(at) * a.freqs[i - r * half], a.freqs[half]);
    }
    for (int r = tid; r < rows; r += 256) {
        const int row = row0 + r, s = int(unsigned(row) / unsigned(a.n_tok)), t = row - s * a.n_tok;
        live[r] = (!a.num || t < a.num[s]) && (long long)a.pos[s] + t >= 0;
    }
    __syncthreads();
    for (int i = tid;; i += 256 * AHEAD) {
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) put(p[j], v[j]);
        if (i + 256 * AHEAD >= items) break;
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            p[j] = find(i + 256 * (AHEAD + j));
            load(p[j], v[j]);
        }
    }
}

}  // namespace

hipError_t launch_rotary(const RotaryArgs & args, hipStream_t s) {
    RotaryArgs a = args;
    int heads = 0;
    for (int i = 0; i < a.n; ++i) a.a[i].end = heads += a.a[i].n_head;
    const bool wide = a.n_rot % 8 == 0;
    const int w = wide ? 4 : 1, per = a.n_rot / 2 / w + (a.head_dim - a.n_rot) / w;
    const long long rows = (long long)a.n_seq * a.n_tok;
    a.tokens = std::max(1, 512 / a.n_rot);
    // pieces of a workgroup: four a thread, or one where that leaves the device's 256 CUs less than two workgroups each
    const long long all = rows * heads * per;
    const int pieces = all >= 512 * 1024 ? 1024 : 256;
    a.heads = std::min(heads, std::max(1, pieces / (a.tokens * per)));
    const dim3 grid(unsigned((rows + a.tokens - 1) / a.tokens), unsigned((heads + a.heads - 1) / a.heads));
    if (wide && a.pairs) GQ_LAUNCH((rope_kernel<true, true>), grid, dim3(256), 0, s, a);
    else if (wide) GQ_LAUNCH((rope_kernel<true, false>), grid, dim3(256), 0, s, a);
    else if (a.pairs) GQ_LAUNCH((rope_kernel<false, true>), grid, dim3(256), 0, s, a);
    else GQ_LAUNCH((rope_kernel<false, false>), grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

void rope_table(int n_rot, double base, double factor, int yarn_ctx, double beta_fast, double beta_slow, const double * factors,
                double * out) {
    constexpr double turn = 6.283185307179586;
    // the pair that turns b times over yarn_ctx positions
    const auto pair = [&](double b) { return n_rot * std::log(yarn_ctx / (b * turn)) / (2 * std::log(base)); };
    double low = 0, high = 0;
    if (yarn_ctx) {
        low = std::max(std::floor(pair(beta_fast)), 0.0);
        high = std::min(std::ceil(pair(beta_slow)), double(n_rot - 1));
    }
    for (int i = 0; i < n_rot / 2; ++i) {
        const double kept = std::pow(base, -2.0 * i / n_rot) / (factors ? factors[i] : 1.0);
        const double share = yarn_ctx ? std::min(std::max((i - low) / std::max(high - low, 1e-3), 0.0), 1.0) : 1.0;
        out[i] = (kept * (1 - share) + kept / factor * share) / turn;
    }
    out[n_rot / 2] = yarn_ctx ? 0.1 * std::log(factor) + 1 : 1.0;
}

}  // namespace gq
