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
// pieces of four pairs of halves (two times 16 bytes), two neighbouring pairs (16 bytes) or 16 bytes that stay, else pair by pair. The
// first pieces are read before the angles are there. Memory bounds it: 4096 tokens of 32/8 heads of 128 (168 MB) are 29.1 us, 5.8 TB/s,
// of neighbours 31.4 (35.6 with four pairs a piece, where a wave's access covers every other 16 bytes); one token 4.3, a launch and two
// trips.
template <bool WIDE, bool PAIRS, bool MANY>
__global__ __launch_bounds__(256) void rope_kernel(RotaryArgs a) {
    // pairs of a piece, its elements, elements of a piece that stays, pieces that a thread has on their way; ONE: 16 bytes a piece
    constexpr bool ONE = WIDE && PAIRS;
    constexpr int W = !WIDE ? 1 : PAIRS ? 2 : 4, N = 2 * W, TAIL = WIDE ? 4 : 1, AHEAD = ONE ? 8 : 4;
    __shared__ float2 cs[ROPE_MAX_DIM / 2];  // tokens * n_rot / 2 of them
    __shared__ int live[256];                // rows with a position
    const int tid = threadIdx.x, half = a.n_rot / 2, tail = a.head_dim - a.n_rot;
    const int turn = half / W, per = turn + tail / TAIL;  // pieces of a head
    const int row0 = int(blockIdx.x) * a.tokens, rows = min(a.tokens, a.n_seq * a.n_tok - row0);
    const int head0 = int(blockIdx.y) * a.heads, heads = min(a.heads, a.a[a.n - 1].end - head0);
    const int items = rows * heads * per, second = PAIRS ? W : half;  // where a piece's second 16 bytes (or element) are

    struct Piece {
        const float * x;
        float * y;
        int r, c;  // row of the workgroup (-1: no piece), piece of the head
    };
    const auto find = [&](int i) {
        Piece p;
        // quotients of numbers whose product with the divisor is below 2^32
        const int rh = a.per_mul ? int(__umulhi(unsigned(i), a.per_mul)) : i;
        const int r = heads == 1 ? rh : heads == a.heads ? int(__umulhi(unsigned(rh), a.heads_mul)) : int(unsigned(rh) / unsigned(heads));
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
        if (p.x == p.y && p.c >= turn) p.r = -1;  // in place: nothing to copy
        const int at = p.c >= turn ? a.n_rot + (p.c - turn) * TAIL : PAIRS ? N * p.c : W * p.c;
        p.x += at;
        p.y += at;
        return p;
    };
    const auto load = [&](const Piece & p, float * v) {  // of halves the first elements, then the second ones
        if (p.r < 0) return;
        if constexpr (WIDE) {
            *reinterpret_cast<f32x4 *>(v) = *reinterpret_cast<const f32x4 *>(p.x);
            if (!ONE && p.c < turn) *reinterpret_cast<f32x4 *>(v + N - 4) = *reinterpret_cast<const f32x4 *>(p.x + second);
        } else {
            v[0] = p.x[0];
            if (p.c < turn) v[1] = p.x[second];
        }
    };
    const auto store = [&](f32x4 z, float * to) {
        if constexpr (MANY) __builtin_nontemporal_store(z, reinterpret_cast<f32x4 *>(to));
        else *reinterpret_cast<f32x4 *>(to) = z;
    };
    const auto put = [&](const Piece & p, const float * v) {
        if (p.r < 0 || !live[p.r]) return;
        const bool turns = p.c < turn;
        float z[N];
#pragma unroll
        for (int e = 0; e < N; ++e) z[e] = v[e];
        if (turns) {
#pragma unroll
            for (int e = 0; e < W; ++e) {
                const float2 t = cs[p.r * half + p.c * W + e];
                const int i0 = PAIRS ? 2 * e : e, i1 = PAIRS ? 2 * e + 1 : W + e;
                z[i0] = v[i0] * t.x - v[i1] * t.y;
                z[i1] = v[i0] * t.y + v[i1] * t.x;
            }
        }
        if constexpr (WIDE) {
            store(f32x4{z[0], z[1], z[2], z[3]}, p.y);
            if (!ONE && turns) store(f32x4{z[N - 4], z[N - 3], z[N - 2], z[N - 1]}, p.y + second);
        } else {
            p.y[0] = z[0];
            if (turns) p.y[second] = z[1];
        }
    };

    Piece p[AHEAD];
    float v[AHEAD][N];
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
    const int per = a.n_rot / 2 / (wide ? a.pairs ? 2 : 4 : 1) + (a.head_dim - a.n_rot) / (wide ? 4 : 1);  // pieces of a head
    const long long rows = (long long)a.n_seq * a.n_tok;
    a.tokens = std::max(1, 512 / a.n_rot);
    // Pieces of a workgroup: one a thread, or, where that is more than the device has room for, eight (16 of 16 bytes). us with one,
    // four and eight: 4.3 / 4.4 / 4.1 at 1 token of 16/4 heads of 256, 4.3 / 4.8 / 6.6 at 8 of 32/8 of 128, 62 / 42 / 38.5 at 4096 of them
    // (29.4 with stores that pass the caches by, which these, 16 MB and more, do not fit; loads that do are 3 us longer). Few pieces and
    // stores that stay, many and stores that pass by: 4.8 / 6.8 us at 128 of them (2 MB out), 8.2 / 7.2 at 512 (10 MB; neighbours 16.2 / 9.5),
    // 13.1 / 9.7 at 1024 (20 MB; 29 / 12.9), 105 / 54 at 8192; with a kernel that reads the queries afterwards 13.5 / 12.0, 19.2 / 18.1 and
    // 148 / 117. Where n_rot is no multiple of 8, element by element: 4096 of 32/8 heads, 58 of 128 58 us (neighbours 51), 122 of 256 155
    // (140), for 33 and 66 at the rate of a copy; 64 of 256 53 (56).
    const bool many = rows * heads * a.head_dim >= 4 << 20;
    const int pieces = many ? a.pairs ? 4096 : 2048 : 256;
    a.heads = std::min(heads, std::max(1, pieces / (a.tokens * per)));
    const auto mul = [](int d) { return d > 1 ? unsigned((0x100000000ull + unsigned(d) - 1) / unsigned(d)) : 0u; };
    a.per_mul = mul(per);
    a.heads_mul = mul(a.heads);
    const dim3 grid(unsigned((rows + a.tokens - 1) / a.tokens), unsigned((heads + a.heads - 1) / a.heads));
    if (wide && a.pairs && many) GQ_LAUNCH((rope_kernel<true, true, true>), grid, dim3(256), 0, s, a);
    else if (wide && many) GQ_LAUNCH((rope_kernel<true, false, true>), grid, dim3(256), 0, s, a);
    else if (wide && a.pairs) GQ_LAUNCH((rope_kernel<true, true, false>), grid, dim3(256), 0, s, a);
    else if (wide) GQ_LAUNCH((rope_kernel<true, false, false>), grid, dim3(256), 0, s, a);
    else if (a.pairs) GQ_LAUNCH((rope_kernel<false, true, false>), grid, dim3(256), 0, s, a);
    else GQ_LAUNCH((rope_kernel<false, false, false>), grid, dim3(256), 0, s, a);
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
