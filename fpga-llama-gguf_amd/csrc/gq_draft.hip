// Verification of drafted tokens (gq_draft.h), in two launches. The first reads every logit once: the maximum and the sum of
// exponentials of every chunk of a row (and, at temperature 0, the place of the maximum). In the second, every workgroup of a sequence
// joins its rows' chunks, decides how many tokens stand, and sums what is left of one chunk of the one row that a new token comes
// from; the last workgroup of the sequence to be done finds the token. Sums are in 64 bits and their terms good to 2.2e-10 (3.6e-10 where logits over the
// temperature pass 1400), up and down by chance: a token is found where a sum of up to 2^20 terms passes a given number, and the borders of all of them have to be where
// they belong.
// 32 sequences of 4 tokens, 151936 logits (175 MB, 39 MB of them twice): 36 us (4.8 TB/s; reading them alone 31 us) and 22 us; one of
// them: 5.4 and 11 us, the second a chain of six trips to memory.
#include "gq_device.h"
#include "gq_draft.h"

#include <cfloat>
#include <type_traits>

namespace gq {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_at_4 __attribute__((ext_vector_type(4), aligned(4)));

// 2^t for |t| <= 1000: t = n + f with |f| <= 1/2, 1 + f q(f) with q interpolating (2^f - 1) / f at 10 Chebyshev points (off by at
// most 5.7e-16 of 2^f). n comes out of u = t + 1.5 * 2^52 as its low word.
__device__ __forceinline__ double draft_exp2(double t) {
    constexpr double magic = 6755399441055744.0;
    const double u = t + magic, f = t - (u - magic);
    double p = 7.070977866508139e-09;
    p = __builtin_fma(p, f, 1.0205905413765595e-07);
    p = __builtin_fma(p, f, 1.3215451633221434e-06);
    p = __builtin_fma(p, f, 1.5252672924850737e-05);
    p = __builtin_fma(p, f, 0.00015403530424776529);
    p = __builtin_fma(p, f, 0.0013333558200794592);
    p = __builtin_fma(p, f, 0.009618129107618665);
    p = __builtin_fma(p, f, 0.05550410866465167);
    p = __builtin_fma(p, f, 0.24022650695910075);
    p = __builtin_fma(p, f, 0.6931471805599462);
    p = __builtin_fma(p, f, 1.0);
    return __builtin_amdgcn_ldexp(p, __double2loint(u));
}
// e^((x - m) / temperature) for x <= m, with c = log2(e) / temperature; from 2^-1000 on, which also stands for what is below, -inf and
// NaN. (Not 0 there: that would be a branch around each.) What counts as a weight is above DRAFT_NONE.
__device__ __forceinline__ double draft_term(float x, double m, double c) { return draft_exp2(fmin(fmax((double(x) - m) * c, -1000.0), 0.0)); }
constexpr double DRAFT_NONE = 1e-290;

// The same for many logits of a row, most of it in FP32: instructions in 64 bits are what the kernels wait for otherwise (16 of them a
// logit: 32 x 4 of 151936 took 43 us without reading anything, 31 us to read without them). x c in two parts, p + e, whose sum has 40
// bits and more; p = N / 256 + r exactly, |r| <= 2^-9; 2^(r + e) = 1 + E in FP32; 2^(N / 256) from a table of 256 in 64 bits, its
// exponent moved. With X = |x c| (below 9192), |r + e| < 2^-9 + 2^-23 X < 0.0031. What is rounded, in parts of a term: r + e by 2^-33
// (8.1e-11), its factor by 2^-25 and ln 2 in it by 1.9e-9 (times |r + e|), E, up to 0.0022, by 2^-33 (2^-34 below 2^-9), e by half a step of
// 2^-23 X and c by 2^-48: 2.2e-10 for X up to 2024, 3.6e-10 for all (the most that was seen: 2.1e-10, 2.4e-10).
// The reference is 2^K, K the whole number next to c times the row's maximum, `unit` the exact 2^(c max - K): a term is the same whatever
// maximum it is formed with, so a row's sums and its weights have the same errors. Only where |c max| is below 8192 (`fast`): N comes
// out of u = 256 p + 1.5 * 2^23 - 256 K, as its low bits.
struct DraftExp {
    double m, c, unit;
    float top, ch, cl, base, low;
    bool fast;
    __device__ __forceinline__ DraftExp(float max, const DraftScale & s) {
        m = top = max;
        c = s.c;
        const double t = m * c, k = rint(t);
        fast = fabs(t) < 8192.0 && s.fast;
        ch = s.ch;
        cl = s.cl;
        base = 12582912.0f - 256.0f * float(fast ? k : 0.0);
        low = float(m - s.reach);
        unit = fast ? draft_exp2(t - k) : 1.0;
    }
    __device__ __forceinline__ double quick(float x, const double * table) const {
        x = __builtin_amdgcn_fmed3f(x, low, top);  // (NaN: low)
        const float p = x * ch, e = __builtin_fmaf(x, cl, __builtin_fmaf(x, ch, -p));
        const float u = __builtin_fmaf(p, 256.0f, base), r = __builtin_fmaf(u - base, -1.0f / 256.0f, p) + e;
        const float E = r * __builtin_fmaf(r, __builtin_fmaf(r, 0.0555041086648216f, 0.240226506959101f), 0.693147180559945f);
        const uint32_t n = __float_as_uint(u);
        const double t = table[n & 255u];
        const double v = __hiloint2double(int(uint32_t(__double2hiint(t)) + (n << 12)), __double2loint(t));  // (N / 256 in the exponent's place)
        return __builtin_fma(v, double(E), v);
    }
    __device__ __forceinline__ double slow(float x) const { return draft_term(x, m, c); }
};
// The table, by all threads of the workgroup (before a barrier): of 2^(i / 256) with i / 256 taken off where an exponent is added.
__device__ __forceinline__ void draft_table(double * table) {
    const double t = draft_exp2(double(threadIdx.x) / 256.0);
    table[threadIdx.x] = __hiloint2double(int(uint32_t(__double2hiint(t)) - (threadIdx.x << 12)), __double2loint(t));
}

__device__ __forceinline__ float draft_clean(float x) { return x == x ? fminf(x, FLT_MAX) : -__builtin_inff(); }
// Over aligned groups of 2^SH lanes (8 to 64): DPP within rows of 16, then across them.
template <typename F>
__device__ __forceinline__ float over_lanes(float x, int sh, F f) {
    x = f(x, dpp_f32<DPP_XOR1>(x));
    x = f(x, dpp_f32<DPP_XOR2>(x));
    x = f(x, dpp_f32<DPP_HALF_MIRROR>(x));
    if (sh > 3) x = f(x, dpp_f32<DPP_MIRROR>(x));
    if (sh > 4) x = f(x, __shfl_xor(x, 16, WAVE));
    if (sh > 5) x = f(x, __shfl_xor(x, 32, WAVE));
    return x;
}
__device__ __forceinline__ double sum_lanes(double x, int sh) {
    const auto step = [&](auto ctrl) { x += __longlong_as_double(dpp_i64<ctrl.value>(__double_as_longlong(x))); };
    step(std::integral_constant<int, DPP_XOR1>());
    step(std::integral_constant<int, DPP_XOR2>());
    step(std::integral_constant<int, DPP_HALF_MIRROR>());
    if (sh > 3) step(std::integral_constant<int, DPP_MIRROR>());
    if (sh > 4) x += __shfl_xor(x, 16, WAVE);
    if (sh > 5) x += __shfl_xor(x, 32, WAVE);
    return x;
}
// A wave's sums up to each lane.
__device__ __forceinline__ double scan_wave(double x) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const double y = __shfl_up(x, d, WAVE);
        if (lane >= d) x += y;
    }
    return x;
}
__device__ __forceinline__ float max_f(float a, float b) { return fmaxf(a, b); }

struct DraftStat {  // of a chunk: its maximum, that one's first token, the sum of the terms relative to it
    float m;
    int at;
    double sum;
};
// Of two chunks, or rows' parts, the one with the larger maximum, of equal ones the first token.
__device__ __forceinline__ void draft_best(float & m, int & at, float m2, int at2) {
    const bool other = m2 > m || (m2 == m && at2 < at);
    m = other ? m2 : m;
    at = other ? at2 : at;
}

// The workspace: what each chunk of every row comes to (target rows, then draft rows), the sums of what is left of the quarters of a
// sequence's chunks, the rows' logits of their drafted tokens, and how many workgroups of each sequence are done (a line each).
constexpr int DRAFT_LINE = 64;  // words between counters
struct DraftWork {
    DraftStat * stat;
    double * left;
    float * logit;
    unsigned * done;
};
__host__ __device__ inline long long draft_rows(const DraftArgs & a) { return (long long)a.n_seq * (2 * a.n_draft + 1); }
__device__ __forceinline__ DraftWork draft_at(const DraftArgs & a) {
    DraftWork w;
    w.stat = static_cast<DraftStat *>(a.work);
    w.left = reinterpret_cast<double *>(w.stat + draft_rows(a) * a.chunks);
    w.logit = reinterpret_cast<float *>(w.left + 4ll * a.n_seq * a.parts);
    w.done = reinterpret_cast<unsigned *>(w.logit + draft_rows(a));
    return w;
}
__device__ __forceinline__ int draft_num(const DraftArgs & a, int s) { return a.num ? min(a.num[s], a.n_draft) : a.n_draft; }

// The first of a lane's logits 4 i .. 4 i + 3 of a chunk: a wave's 64 * PER follow one another.
template <int PER>
__device__ __forceinline__ int draft_place(int chunk, int i) {
    return chunk * 256 * PER + (threadIdx.x >> 6) * 64 * PER + 4 * (64 * i + (threadIdx.x & 63));
}
// The lane's PER logits of a chunk; behind the row: -inf. (One branch for a wave's loads: they stay in flight over it.)
template <int PER>
__device__ __forceinline__ void draft_load(const float * x, int n, int chunk, float * v) {
    if (chunk * 256 * PER + (__builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6)) + 1) * 64 * PER <= n) {
#pragma unroll
        for (int i = 0; i < PER / 4; ++i) *reinterpret_cast<f32x4 *>(v + 4 * i) = *reinterpret_cast<const f32x4_at_4 *>(x + draft_place<PER>(chunk, i));
    } else {
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int t = draft_place<PER>(chunk, j >> 2) + (j & 3);
            v[j] = x[min(t, n - 1)];
            v[j] = t < n ? v[j] : -__builtin_inff();
        }
    }
}

// Workgroup (chunk of 256 * PER logits | row of the target, then of the draft).
template <int PER>
__global__ __launch_bounds__(256) void draft_scan_kernel(DraftArgs a) {
    __shared__ DraftStat red[4];
    __shared__ double table[256];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, chunk = blockIdx.x, trows = a.n_seq * (a.n_draft + 1);
    const bool own = int(blockIdx.y) < trows;
    const int row = own ? blockIdx.y : blockIdx.y - trows, each = own ? a.n_draft + 1 : a.n_draft, s = row / each, t = row - s * each;
    const DraftWork w = draft_at(a);
    if (own && t == 0 && chunk == 0 && tid == 0) w.done[(long long)s * DRAFT_LINE] = 0;
    const int num = draft_num(a, s), token = t < a.n_draft ? a.token[(long long)s * a.n_draft + t] : -1;
    if (own ? t > num : t >= num) return;
    const float * x = own ? a.target + row * a.target_stride : a.draft + row * a.draft_stride;
    const DraftScale & sc = own ? a.scale : a.draft_scale;
    const double c = sc.c;
    float v[PER];
    draft_load<PER>(x, a.n_vocab, chunk, v);
    draft_table(table);
    __syncthreads();
    if (token >= 0 && token < a.n_vocab && token / (256 * PER) == chunk)
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (draft_place<PER>(chunk, j >> 2) + (j & 3) == token) w.logit[own ? row : (long long)trows + row] = draft_clean(v[j]);
    float m = -__builtin_inff();  // (NaN: passed by)
    int at = 0x7fffffff;
#pragma unroll
    for (int j = 0; j < PER; ++j) m = fmaxf(m, v[j]);
    if (__any(m == __builtin_inff())) {
        m = fminf(m, FLT_MAX);
#pragma unroll
        for (int j = 0; j < PER; ++j) v[j] = draft_clean(v[j]);
    }
    if (a.greedy) {
#pragma unroll
        for (int j = PER - 1; j >= 0; --j) at = v[j] == m ? draft_place<PER>(chunk, j >> 2) + (j & 3) : at;
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) {
            const float m2 = __shfl_xor(m, d, WAVE);
            const int at2 = __shfl_xor(at, d, WAVE);
            draft_best(m, at, m2, at2);
        }
    } else {
        m = over_lanes(m, 6, max_f);
    }
    m = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(m)));
    double sum = 0.0;
    if (m > -__builtin_inff()) {
        const DraftExp e(m, sc);
        if (e.fast) {
#pragma unroll
            for (int j = 0; j < PER; ++j) sum += e.quick(v[j], table);
        } else {
#pragma unroll
            for (int j = 0; j < PER; ++j) sum += e.slow(v[j]);
        }
        sum = sum_lanes(sum, 6) / e.unit;
    }
    if (lane == 0) red[wave] = {m, at, sum};
    __syncthreads();
    if (tid) return;
    DraftStat r = {red[0].m, red[0].at, 0.0};
    for (int i = 1; i < 4; ++i) draft_best(r.m, r.at, red[i].m, red[i].at);
    for (int i = 0; i < 4; ++i) r.sum += red[i].sum * draft_term(red[i].m, r.m, c);
    w.stat[(own ? row : (long long)trows + row) * a.chunks + chunk] = r;
}

// Workgroup (chunk of 256 * PER logits | sequence). A chain of trips to memory: how many tokens there are; the chunks' statistics and the logits of the
// drafted tokens; a chunk of the rows that the new token comes from; and, in the last workgroup, the sums of all of these, and a quarter
// of a chunk.
template <int PER>
__global__ __launch_bounds__(256) void draft_pick_kernel(DraftArgs a) {
    constexpr int ROWS = 2 * DRAFT_MAX + 1;
    __shared__ float top[ROWS];
    __shared__ int arg[ROWS], accepted, last, hit[8];
    __shared__ double total[ROWS], red[4], rest, table[256];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, chunk = blockIdx.x, s = blockIdx.y;
    const int num = draft_num(a, s);
    const bool greedy = a.greedy, rows_of_draft = a.draft && !greedy;
    const DraftWork w = draft_at(a);
    const double c = a.scale.c, cq = a.draft_scale.c;
    const long long trow = (long long)s * (a.n_draft + 1), drow = (long long)s * a.n_draft, trows = (long long)a.n_seq * (a.n_draft + 1);
    draft_table(table);
    // the drafted tokens, and their logits (read whether or not there are as many)
    int d = -1;
    float xt = 0.0f, xd = 0.0f, u = 0.0f;
    if (wave == 0 && lane < a.n_draft) {
        d = a.token[drow + lane];
        if (!greedy) u = a.uniform[trow + lane];
        xt = w.logit[trow + lane];
        if (rows_of_draft) xd = w.logit[trows + drow + lane];
    }
    // ---- the rows: 0 .. n_draft the target's, then the draft's (those that are not there are not looked at later); 8 to 64 lanes a
    // row, two chunks a lane at a time ----
    const int n1 = a.n_draft + 1, rows = n1 + (rows_of_draft ? a.n_draft : 0), sh = a.chunks > 64 ? 6 : a.chunks > 32 ? 5 : a.chunks > 16 ? 4 : 3;
    for (int r0 = 0; r0 < rows; r0 += 256 >> sh) {
        const int r = r0 + (tid >> sh), c1 = lane & ((1 << sh) - 1);
        const bool mine = r < n1;
        const DraftStat * st = w.stat + (mine ? trow + r : trows + drow + (r - n1)) * a.chunks;
        const double cr = mine ? c : cq;
        float m = -__builtin_inff();
        int at = 0x7fffffff;
        double sum = 0.0;
        for (int i = c1; i < a.chunks + c1; i += 2 << sh) {  // (once but for more than 128 chunks)
            DraftStat x[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) x[k] = r < rows && i + (k << sh) < a.chunks ? st[i + (k << sh)] : DraftStat{-__builtin_inff(), 0x7fffffff, 0.0};
            const float m2 = fmaxf(m, fmaxf(x[0].m, x[1].m));
            sum = sum * draft_term(m, m2, cr) + x[0].sum * draft_term(x[0].m, m2, cr) + x[1].sum * draft_term(x[1].m, m2, cr);
#pragma unroll
            for (int k = 0; k < 2; ++k) draft_best(m, at, x[k].m, x[k].at);
        }
        float m1 = over_lanes(m, sh, max_f);
        sum = sum_lanes(sum * draft_term(m, m1, cr), sh);
        if (greedy)
#pragma unroll
            for (int k = 32; k >= 1; k >>= 1) {
                const float m2 = __shfl_xor(m, k, WAVE);
                const int at2 = __shfl_xor(at, k, WAVE);
                if (k >> sh == 0) draft_best(m, at, m2, at2);
            }
        if (c1 == 0 && r < rows) {
            top[r] = m1;
            arg[r] = at;
            total[r] = sum;
        }
    }
    __syncthreads();
    if (num < 0) return;
    // ---- how many tokens stand ----
    if (wave == 0) {
        bool ok = lane < num && d >= 0 && d < a.n_vocab && top[lane < num ? lane : 0] > -__builtin_inff();
        if (ok && greedy) {
            ok = d == arg[lane];
        } else if (ok) {
            const double p = (double(xt) - top[lane]) * c > -1000.0 ? draft_term(xt, top[lane], c) : 0.0;
            double q = 1.0, qs = 1.0;  // e and sums, which are no less: u q / qs < p / total
            if (a.draft) {
                const float m = top[n1 + lane];
                q = (double(xd) - m) * cq > -1000.0 ? draft_term(xd, m, cq) : 0.0;
                qs = m > -__builtin_inff() ? fmax(total[n1 + lane], q) : 1.0;
            }
            ok = double(u) * q * fmax(total[lane], p) < p * qs;
        }
        const unsigned long long no = ~__ballot(ok);
        if (lane == 0) accepted = __ffsll(no) - 1;  // (lanes from num on say no)
    }
    __syncthreads();
    const int k = accepted;
    const float m = top[k];
    double logsum = 0.0;
    const auto finish = [&](int token) {  // by the first wave
        if (lane > a.n_draft) return;
        const int tok = lane < k ? d : lane == k ? token : -1;
        a.out[trow + lane] = tok;
        if (lane == 0) a.n_accept[s] = k;
        if (!a.logp) return;
        double l = 0.0;
        if (tok >= 0) {
            if (lane == k) xt = draft_clean(a.target[(trow + k) * a.target_stride + tok]);
            l = (double(xt) - top[lane]) * c * 0.6931471805599453 - logsum;
        }
        a.logp[trow + lane] = float(fmin(l, 0.0));
    };
    if (greedy || !(m > -__builtin_inff())) {
        if (chunk == 0 && a.logp && lane <= k) logsum = log(total[lane]);
        if (chunk == 0 && wave == 0) finish(m > -__builtin_inff() ? arg[k] : -1);
        return;
    }
    // ---- what is left of this chunk, a sum a wave (weights in units of the target's row) ----
    const float * xp = a.target + (trow + k) * a.target_stride;
    const bool less = k < num && a.draft && top[n1 + k] > -__builtin_inff();
    const float * xq = less ? a.draft + (drow + k) * a.draft_stride : xp;
    const int certain = k < num && !a.draft ? a.token[drow + k] : -1, subs = 4 * a.parts;
    float px[PER], qx[PER];
    draft_load<PER>(xp, a.n_vocab, chunk, px);
    if (less) draft_load<PER>(xq, a.n_vocab, chunk, qx);
    const DraftExp ep(m, a.scale), eq(less ? top[n1 + k] : m, less ? a.draft_scale : a.scale);
    const double share = less ? total[k] * ep.unit / (total[n1 + k] * eq.unit) : 0.0;
    const bool fast = ep.fast && eq.fast;
    const auto weight = [&](float p, float q, int token, bool whole) {
        const double x = ep.fast ? ep.quick(p, table) : ep.slow(p);
        if (whole) return x;
        if (less) return fmax(__builtin_fma(eq.fast ? eq.quick(q, table) : eq.slow(q), -share, x), 0.0);
        return token == certain ? 0.0 : x;
    };
    double * left = w.left + (long long)s * subs;
    double sum = 0.0;
    if (fast && less) {
#pragma unroll
        for (int j = 0; j < PER; ++j) sum += fmax(__builtin_fma(eq.quick(qx[j], table), -share, ep.quick(px[j], table)), 0.0);
    } else if (fast) {
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const double x = ep.quick(px[j], table);
            sum += draft_place<PER>(chunk, j >> 2) + (j & 3) == certain ? 0.0 : x;
        }
    } else {
#pragma unroll
        for (int j = 0; j < PER; ++j) sum += weight(px[j], less ? qx[j] : 0.0f, draft_place<PER>(chunk, j >> 2) + (j & 3), false);
    }
    sum = sum_lanes(sum, 6);
    if (lane == 0) __hip_atomic_store(left + 4 * chunk + wave, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    // The sums are agent-scope atomic stores, coherent across the XCDs without an L2 writeback, and have arrived (stores count in vmcnt
    // on gfx950) before the count goes up; the last workgroup's loads are such loads, issued after its count came back.
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (tid == 0) last = __hip_atomic_fetch_add(w.done + (long long)s * DRAFT_LINE, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == unsigned(a.parts) - 1;
    __syncthreads();
    if (!last) return;
    // ---- the token: the quarter of a chunk where the sums pass the goal (or the last one with any weight, where rounding leaves
    // none), then itself ----
    constexpr int EACH = DRAFT_MAX_VOCAB / (64 * PER) / 256 > 1 ? DRAFT_MAX_VOCAB / (64 * PER) / 256 : 1;  // sums a thread
    const int each = (subs + 255) / 256, i0 = tid * each;
    double part[EACH], mine = 0.0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        part[i] = i < each && i0 + i < subs ? __hip_atomic_load(left + i0 + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.0;
        mine += part[i];
    }
    const auto before_of = [&](double x, double & all) {  // the sums of the threads before this one, and of all
        const double upto = scan_wave(x);
        __syncthreads();
        if (lane == 63) red[wave] = upto;
        __syncthreads();
        double before = upto - x;
        for (int i = 0; i < wave; ++i) before += red[i];
        all = (red[0] + red[1]) + (red[2] + red[3]);
        return before;
    };
    double all, before = before_of(mine, all);
    const bool whole = !(all > DRAFT_NONE * DRAFT_MAX_VOCAB);
    if (whole) {  // nothing is left: the row as it is
        for (int i = wave; i < subs; i += 4) {
            double sum = 0.0;
            for (int j = lane; j < 64 * PER && i * 64 * PER + j < a.n_vocab; j += 64) sum += weight(xp[i * 64 * PER + j], 0.0f, 0, true);
            sum = sum_lanes(sum, 6);
            if (lane == 0) __hip_atomic_store(left + i, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        mine = 0.0;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            part[i] = i < each && i0 + i < subs ? __hip_atomic_load(left + i0 + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.0;
            mine += part[i];
        }
        before = before_of(mine, all);
    }
    const double goal = all * double(a.uniform[trow + a.n_draft]);
    if (wave == 0 && a.logp && lane <= k) logsum = log(total[lane]);
    // the first of the threads' first ones, and the last of their last ones
    const auto choose = [&](int first, int end, int & f, int & e) {
        const unsigned long long has = __ballot(first >= 0), any = __ballot(end >= 0);
        const int f1 = __shfl(first, has ? __ffsll(has) - 1 : 0, WAVE), e1 = __shfl(end, any ? 63 - __clzll(any) : 0, WAVE);
        __syncthreads();
        if (lane == 0) {
            hit[wave] = has ? f1 : -1;
            hit[4 + wave] = any ? e1 : -1;
        }
        __syncthreads();
        f = e = -1;
        for (int i = 3; i >= 0; --i) f = hit[i] >= 0 ? hit[i] : f;
        for (int i = 0; i < 4; ++i) e = hit[4 + i] >= 0 ? hit[4 + i] : e;
    };
    int first = -1, end = -1, f, e;
    double run = before, at_first = 0.0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        if (part[i] > DRAFT_NONE) {
            end = i0 + i;
            if (first < 0 && run + part[i] > goal) {
                first = end;
                at_first = run;
            }
        }
        run += part[i];
    }
    choose(first, end, f, e);
    if (first >= 0 && first == f) rest = goal - at_first;
    if (f < 0 && tid == 0) rest = __builtin_inf();
    __syncthreads();
    const double goal2 = rest;
    const int sub = f >= 0 ? f : e;
    // a thread's tokens: PER / 4 in a row
    constexpr int N = PER / 4;
    const int t0 = sub * 64 * PER + tid * N;
    double v[N];
    mine = 0.0;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const bool in = t0 + j < a.n_vocab;
        v[j] = weight(in ? xp[t0 + j] : -__builtin_inff(), in && less ? xq[t0 + j] : -__builtin_inff(), t0 + j, whole);
        mine += v[j];
    }
    double upto = before_of(mine, all);
    first = end = -1;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        upto += v[j];
        if (v[j] > DRAFT_NONE) {
            end = t0 + j;
            if (first < 0 && upto > goal2) first = end;
        }
    }
    choose(first, end, f, e);
    if (wave == 0) finish(f >= 0 ? f : e);
}

// Logits of a chunk in either kernel: the longer ones where there are enough to fill the device with them. Both kernels, us, with
// 4096 and 2048 / 8192 and 4096: 5.4 + 11.1 / 6.2 + 11.2 at 1 x 4 of 151936, 11.2 + 11.6 / 12.1 + 10.4 at 61 x 3 of 32003 (certain,
// half of them there), 45 + 28 / 41 + 21 at 32 x 4 of 151936, before the last steps (5.3 + 11.3, 9.9 + 10.4 and 36 + 22 now).
constexpr int DRAFT_SCAN = 4096, DRAFT_PICK = 2048;  // the shorter ones
struct DraftSizes {
    int scan, pick;
};
DraftSizes draft_sizes(int n_seq, int n_draft, int n_vocab) {
    const long long row = (long long)n_seq * n_vocab;
    return {row * (2 * n_draft + 1) >= 16 << 20 ? 2 * DRAFT_SCAN : DRAFT_SCAN, row >= 1 << 20 ? 2 * DRAFT_PICK : DRAFT_PICK};
}
int draft_chunks(int n_vocab, int each) { return (n_vocab + each - 1) / each; }

}  // namespace

DraftScale draft_scale(double temperature) {
    DraftScale s;
    s.c = 1.4426950408889634 / temperature;
    s.reach = 1000.0 / s.c;
    s.fast = s.c < 1e30 && s.c > 1e-30;
    s.ch = s.fast ? float(s.c) : 0.0f;
    s.cl = s.fast ? float(s.c - double(s.ch)) : 0.0f;
    return s;
}

// Of the shorter chunks whatever a call's own are (twice as many numbers at most): what a call needs never falls as its sizes grow.
size_t draft_work(int n_seq, int n_draft, int n_vocab) {
    return size_t(n_seq) * (size_t(2 * n_draft + 1) * (sizeof(DraftStat) * draft_chunks(n_vocab, DRAFT_SCAN) + sizeof(float)) +
                            4 * sizeof(double) * draft_chunks(n_vocab, DRAFT_PICK) + DRAFT_LINE * sizeof(unsigned));
}

hipError_t launch_draft(const DraftArgs & args, hipStream_t s) {
    DraftArgs a = args;
    const DraftSizes z = draft_sizes(a.n_seq, a.n_draft, a.n_vocab);
    a.chunks = draft_chunks(a.n_vocab, z.scan);
    a.parts = draft_chunks(a.n_vocab, z.pick);
    const bool draft = a.draft && !a.greedy;
    const dim3 rows(unsigned(a.chunks), unsigned(a.n_seq * (a.n_draft + 1 + (draft ? a.n_draft : 0)))), seqs(unsigned(a.parts), unsigned(a.n_seq));
    if (z.scan > DRAFT_SCAN) GQ_LAUNCH(draft_scan_kernel<32>, rows, dim3(256), 0, s, a);
    else GQ_LAUNCH(draft_scan_kernel<16>, rows, dim3(256), 0, s, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (z.pick > DRAFT_PICK) GQ_LAUNCH(draft_pick_kernel<16>, seqs, dim3(256), 0, s, a);
    else GQ_LAUNCH(draft_pick_kernel<8>, seqs, dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace gq
