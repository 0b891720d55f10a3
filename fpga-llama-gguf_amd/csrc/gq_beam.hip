// The beam search's kernels (gq_beam.h).
#include "gq_beam.h"
#include "gq_device.h"

#include <cfloat>
#include <type_traits>

namespace gq {
namespace {

// ---- selection ----
// Two launches. The first reads every logit once: workgroup (256 * PER logits of a row) forms their maximum m and sum of e^(x - m), and
// their n_beam best in order. The second, a workgroup per group, joins the rows' sums, and takes the best candidate off the sorted
// lists n_beam times (or, of many, merges them). Values are 64-bit from the logits on (candidates of two beams may lie next to each
// other). A list entry is one word that orders as the candidates of one row do: the logit's bits made monotone, above the token
// inverted.
// 8 groups of 8 beams of 151936 logits (39 MB): 16.2 us (2.4 TB/s: a workgroup's own way of read, reduce and rank is 7 us, the 64-bit
// exponentials another 5, partly behind the reads) and 8.6 us, of which n_beam steps of about 0.4 us that wait for one another; one
// group of 4: 6.8 and 4.7 us, both latency. (Kernel times by rocprofv3; those of the rules below are calls replayed in a graph.)

// 2^t for -1020 <= t <= 0: t = n + f with |f| <= 1/2, 1 + f q(f) with q interpolating (2^f - 1) / f at 7 Chebyshev points (off by at
// most 1.1e-10 of 2^f, exact at 0), and n added to the exponent. n comes out of u = t + 1.5 * 2^52 as its low word.
__device__ __forceinline__ double beam_poly(double f, double u) {
    double p = 1.5297323765018243e-05;
    p = __builtin_fma(p, f, 0.00015461444698569867);
    p = __builtin_fma(p, f, 0.001333350238614389);
    p = __builtin_fma(p, f, 0.009618056678524634);
    p = __builtin_fma(p, f, 0.05550410883909642);
    p = __builtin_fma(p, f, 0.24022650922288757);
    p = __builtin_fma(p, f, 0.6931471805599453);
    p = __builtin_fma(p, f, 1.0);
    return __hiloint2double(__double2hiint(p) + (__double2loint(u) << 20), __double2loint(p));
}
__device__ __forceinline__ double beam_exp2(double t) {
    const double magic = 6755399441055744.0, u = t + magic;
    return beam_poly(t - (u - magic), u);
}
// e^(x - m) for x <= m and m finite; below m - 700, and for NaN, e^-700. As beam_exp2, with the multiplication by log2(e) in both of
// its sums.
__device__ __forceinline__ double beam_term(float x, double m, double low) {
    constexpr double magic = 6755399441055744.0, log2e = 1.4426950408889634;
    const double d = fmax(double(x) - m, low), u = __builtin_fma(d, log2e, magic);
    return beam_poly(__builtin_fma(d, log2e, magic - u), u);
}
__device__ __forceinline__ double beam_term(float x, float m) { return beam_term(x, double(m), -700.0); }

// log x for 1 <= x < 2^64: the hardware's FP32 logarithm y, and one step from it: x e^-y = 1 + r with r below 1e-6.
__device__ __forceinline__ double beam_log(double x) {
    const double y = double(__builtin_amdgcn_logf(float(x))), r = x * beam_exp2(-y) - 1.0;
    return y * 0.6931471805599453 + r * (1.0 - 0.5 * r);
}

// Over a wave: by DPP within rows of 16, then across them.
template <typename F>
__device__ __forceinline__ uint32_t wave_u32(uint32_t x, F f) {
    x = f(x, uint32_t(dpp_i32<DPP_XOR1>(int(x))));
    x = f(x, uint32_t(dpp_i32<DPP_XOR2>(int(x))));
    x = f(x, uint32_t(dpp_i32<DPP_HALF_MIRROR>(int(x))));
    x = f(x, uint32_t(dpp_i32<DPP_MIRROR>(int(x))));
    x = f(x, uint32_t(__shfl_xor(int(x), 16, WAVE)));
    return f(x, uint32_t(__shfl_xor(int(x), 32, WAVE)));
}
template <typename F>
__device__ __forceinline__ double wave_f64(double x, F f) {
    const auto step = [&](auto ctrl) { x = f(x, __longlong_as_double(dpp_i64<ctrl.value>(__double_as_longlong(x)))); };
    step(std::integral_constant<int, DPP_XOR1>());
    step(std::integral_constant<int, DPP_XOR2>());
    step(std::integral_constant<int, DPP_HALF_MIRROR>());
    step(std::integral_constant<int, DPP_MIRROR>());
    x = f(x, __shfl_xor(x, 16, WAVE));
    return f(x, __shfl_xor(x, 32, WAVE));
}
__device__ __forceinline__ uint32_t max_u(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint32_t min_u(uint32_t a, uint32_t b) { return a < b ? a : b; }
__device__ __forceinline__ double sum_d(double a, double b) { return a + b; }

struct BeamStat {
    float m;
    uint32_t pad;
    double sum;
};
// The workspace: the statistics of every chunk of every row, then their lists.
__device__ __forceinline__ BeamStat * beam_stats(const BeamSelectArgs & a) { return static_cast<BeamStat *>(a.work); }
__device__ __forceinline__ unsigned long long * beam_lists(const BeamSelectArgs & a) {
    return reinterpret_cast<unsigned long long *>(beam_stats(a) + size_t(a.n_group) * a.n_beam * a.chunks);
}

// A row that takes no logits: a beam that has ended (its one candidate), or one without a score (none, also where its last token is eos:
// its candidates are all at -inf, so their order is that of the tokens).
__device__ __forceinline__ bool beam_closed(const BeamSelectArgs & a, int row, bool & ended) {
    const size_t at = size_t(row) * a.slot;
    const bool scored = a.score[at] > -__builtin_inff();
    ended = scored && a.last && a.last[at] == a.eos && a.eos >= 0 && a.eos < a.n_vocab && !(a.pos && a.pos[at] < a.n_prompt[at]);
    return ended || !scored;
}
// Whether the row's prompt has a next id; its place in the prompt.
__device__ __forceinline__ bool beam_prompted(const BeamSelectArgs & a, int row, int & next) {
    if (!a.pos) return false;
    next = a.pos[size_t(row) * a.slot] + 1;
    return next >= 0 && next < min(a.n_prompt[size_t(row) * a.slot], a.cap);
}

// Orders a wave's LDS writes before its other lanes' reads (a wave's LDS operations are carried out in order).
__device__ __forceinline__ void wave_lds() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <int PER>
__global__ __launch_bounds__(256) void beam_scan_kernel(BeamSelectArgs a) {
    constexpr int CH = 256 * PER;
    extern __shared__ unsigned long long list[];  // the waves' candidates: beam_list each
    __shared__ float red[4];
    __shared__ double sums[4];
    __shared__ int count[4];
    __shared__ unsigned long long best[4][BEAM_MAX];
    const int row = blockIdx.y, chunk = blockIdx.x, k = a.n_beam, tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), v0 = chunk * CH, cap = beam_list(k, PER);
    const size_t at = size_t(row) * a.chunks + chunk;
    unsigned long long * out = beam_lists(a) + at * k;
    const float * x = a.x + size_t(row) * size_t(a.stride);
    // elements 4 (256 i + tid) + e of the chunk, wherever the row starts (a 16-byte load takes any multiple of 4): what a lane holds goes by
    // the tokens alone, so beams with the same logits have the same sums and tie. Read before it is known whether the row takes
    // logits at all, which is a microsecond later
    typedef float f32x4 __attribute__((ext_vector_type(4)));
    typedef float f32x4_at_4 __attribute__((ext_vector_type(4), aligned(4)));
    float v[PER];
#pragma unroll
    for (int i = 0; i < PER / 4; ++i) {
        const int t = v0 + 4 * (256 * i + tid);
        if (t + 4 <= a.n_vocab) {
            *reinterpret_cast<f32x4 *>(v + 4 * i) = *reinterpret_cast<const f32x4_at_4 *>(x + t);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * i + e] = t + e < a.n_vocab ? x[t + e] : -__builtin_inff();
        }
    }
    bool ended;
    int next;
    if (beam_prompted(a, row - row % k, next)) return;  // the group reads its prompt (its first beam says so, here and below)
    if (beam_closed(a, row, ended)) {
        // the first chunk lists the tokens in order at -inf, an ended beam's eos before them at 0 (of sum 1)
        for (int i = tid; i < k; i += 256) {
            const int token = ended ? (i == 0 ? a.eos : i - 1 < a.eos ? i - 1 : i) : i;
            const float x = ended && i == 0 ? 0.0f : -__builtin_inff();
            out[i] = chunk == 0 && token < a.n_vocab ? (unsigned long long)beam_order(x) << 32 | uint32_t(~token) : 0ull;
        }
        if (tid == 0) beam_stats(a)[at] = {ended && chunk == 0 ? 0.0f : -__builtin_inff(), 0, ended && chunk == 0 ? 1.0 : 0.0};
        return;
    }
    const auto token_of = [&](int j) { return v0 + 4 * (256 * (j >> 2) + tid) + (j & 3); };
    const auto real = [&](int j) { return token_of(j) < a.n_vocab; };
    const auto clean = [](float y) { return y == y ? fminf(y, FLT_MAX) : -__builtin_inff(); };
    float tv = v[0];
#pragma unroll
    for (int j = 1; j < PER; ++j) tv = fmaxf(tv, v[j]);
    const auto clean_all = [&] {
        __asm__ volatile("");  // (a branch of its own: not done ahead of it and selected)
#pragma unroll
        for (int j = 0; j < PER; ++j) v[j] = clean(v[j]);
    };
    if (__any(tv == __builtin_inff())) {
        clean_all();
        tv = fminf(tv, FLT_MAX);
    }
    tv = clean(tv);  // (NaN: the lane has no number; the others pass maxima and terms by)
    const uint32_t top = real(0) ? beam_order(tv) : 0;  // the lane's best; 0: it has none
    // ---- maximum and sum ----
    const uint32_t wtop = __builtin_amdgcn_readfirstlane(wave_u32(top, max_u)), wlow = __builtin_amdgcn_readfirstlane(wave_u32(top, min_u));
    const float wm = wtop ? beam_number(wtop) : -__builtin_inff();  // each wave's sum is relative to its own maximum
    double sum = 0.0;
    if (wm > -__builtin_inff()) {
#pragma unroll
        for (int j = 0; j < PER; ++j) sum += beam_term(v[j], wm);
    }
    sum = wave_f64(sum, sum_d);
    // ---- the wave's candidates: those that pass a bound on the lanes' best ----
    int n;
    const uint32_t lo = beam_bound([&](uint32_t w) { return __popcll(__ballot(top >= w)); }, k, wlow, wtop, n);
    unsigned long long * mylist = list + wave * cap;
    int have = 0;
    const auto put = [&](bool in, float y, int t) {
        const unsigned long long who = __ballot(in);
        if (!who) return;
        if (in) mylist[have + __popcll(who & ((1ull << lane) - 1))] = (unsigned long long)beam_order(y) << 32 | uint32_t(~t);
        have += __popcll(who);
    };
    const uint32_t bottom = beam_order(-__builtin_inff());
    if (n <= k + BEAM_SLACK && lo > bottom) {
        const float bound = beam_number(lo);
#pragma unroll
        for (int j = 0; j < PER; ++j) put(v[j] >= bound, v[j], token_of(j));
    } else {
        clean_all();
        // every element counts, or many lanes' best are equal: of the elements at the bound itself, the tokens up to `until`
        int until = INT_MAX;
        if (n > k + BEAM_SLACK) {
            int mine = INT_MAX;
            if (top == lo) {
#pragma unroll
                for (int j = PER - 1; j >= 0; --j)
                    if (real(j) && beam_order(v[j]) == lo) mine = token_of(j);
            }
            const int above = __popcll(__ballot(top > lo));
            int l = v0 - 1, h = v0 + CH;  // fewer than k with tokens <= l, at least k with <= h
            while (h - l > 1) {
                const int mid = l + (h - l) / 2;
                if (above + __popcll(__ballot(mine <= mid)) >= k) h = mid;
                else l = mid;
            }
            until = h;
        }
        const auto passes = [&](float y, int t) { return beam_order(y) > lo || (beam_order(y) == lo && t <= until); };
#pragma unroll
        for (int j = 0; j < PER; ++j) put(real(j) && passes(v[j], token_of(j)), v[j], token_of(j));
    }
    if (lane < 8) {  // up to whole eights of entries
        const int i = have + lane;
        if (i < (have + 7) / 8 * 8) mylist[i] = 0;
    }
    if (lane == 0) {
        red[wave] = wm;
        sums[wave] = sum;
        count[wave] = min(have, k);
    }
    // ---- in order: the wave's, each candidate's place being the number of better ones; then the chunk's, a place further for every
    // better one of the other waves ----
    wave_lds();
    if (lane < BEAM_MAX && lane >= have) best[wave][lane] = 0;
    for (int i = lane; i < have; i += 64) {
        const unsigned long long key = mylist[i];
        int place = 0;
        for (int j = 0; j < have; j += 8) {
            unsigned long long y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = mylist[j + e];
#pragma unroll
            for (int e = 0; e < 8; ++e) place += y[e] > key;
        }
        if (place < BEAM_MAX) best[wave][place] = key;
    }
    __syncthreads();
    if (lane < count[wave]) {
        const unsigned long long key = best[wave][lane];
        int before[3] = {0, 0, 0};
#pragma unroll
        for (int st = BEAM_MAX / 2; st >= 1; st /= 2)
#pragma unroll
            for (int w = 0; w < 3; ++w) before[w] += best[(wave + 1 + w) & 3][before[w] + st - 1] > key ? st : 0;
        int place = lane;
#pragma unroll
        for (int w = 0; w < 3; ++w) place += before[w] + (best[(wave + 1 + w) & 3][before[w]] > key);
        if (place < k) out[place] = key;
    }
    for (int i = count[0] + count[1] + count[2] + count[3] + tid; i < k; i += 256) out[i] = 0;
    if (tid == 0) {
        const float m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        double s = 0.0;
        for (int w = 0; w < 4; ++w)
            if (red[w] > -__builtin_inff()) s += sums[w] * beam_term(red[w], m);
        beam_stats(a)[at] = {m, 0, s};
    }
}

// The second launch's beginning: the rows' maxima, the logarithms of their sums and their scores, 8 to 64 lanes a row. What is read of
// score and last is read here (score_out and token may be the same memory). False: the group reads its prompt.
template <int W>
__device__ __forceinline__ bool beam_rows(const BeamSelectArgs & a, int g, double * top, double * logsum, double * scores) {
    const int k = a.n_beam, tid = threadIdx.x, lane = tid & 63;
    int ahead;
    if (beam_prompted(a, g * k, ahead)) {  // the group's beams read their prompt
        if (tid < k) {
            if (beam_prompted(a, g * k + tid, ahead)) a.token[(g * k + tid) * a.slot] = a.prompt[size_t(g * k + tid) * a.cap + ahead];
            a.parent[(g * k + tid) * a.slot] = tid;
        }
        return false;
    }
    const BeamStat * st = beam_stats(a) + size_t(g) * k * a.chunks;
    const int sh = a.chunks > 32 ? 6 : a.chunks > 16 ? 5 : a.chunks > 8 ? 4 : 3, each = 64 >> sh;
    const auto over = [&](auto x, auto f, auto get) {  // over a row's lanes
        x = f(x, get(x, std::integral_constant<int, DPP_XOR1>()));
        x = f(x, get(x, std::integral_constant<int, DPP_XOR2>()));
        x = f(x, get(x, std::integral_constant<int, DPP_HALF_MIRROR>()));
        if (sh > 3) x = f(x, get(x, std::integral_constant<int, DPP_MIRROR>()));
        if (sh > 4) x = f(x, __shfl_xor(x, 16, WAVE));
        if (sh > 5) x = f(x, __shfl_xor(x, 32, WAVE));
        return x;
    };
    for (int b0 = 0; b0 < k; b0 += W * each) {
        const int b = b0 + (tid >> 6) * each + (lane >> sh), c1 = lane & ((1 << sh) - 1);
        const float sc = b < k ? a.score[(g * k + b) * a.slot] : 0.0f;
        BeamStat x[2];
        float m = -__builtin_inff();
        double s = 0.0;
        for (int c0 = c1; c0 < a.chunks + c1; c0 += 2 << sh) {  // (once but for more than 128 chunks)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int c = c0 + (i << sh);
                x[i] = b < k && c < a.chunks ? st[b * a.chunks + c] : BeamStat{-__builtin_inff(), 0, 0.0};
            }
            const float m1 = fmaxf(m, fmaxf(x[0].m, x[1].m));
            if (m1 > -__builtin_inff()) s = (m > -__builtin_inff() ? s * beam_term(m, m1) : 0.0) + x[0].sum * beam_term(x[0].m, m1) + x[1].sum * beam_term(x[1].m, m1);
            m = m1;
        }
        const float wm = over(m, [](float y, float z) { return fmaxf(y, z); }, [](float y, auto c) { return dpp_f32<c.value>(y); });
        s = over(m > -__builtin_inff() ? s * beam_term(m, wm) : 0.0, sum_d,
                 [](double y, auto c) { return __longlong_as_double(dpp_i64<c.value>(__double_as_longlong(y))); });
        if (c1 == 0 && b < k) {
            top[b] = wm;
            logsum[b] = beam_log(s);
            scores[b] = sc == sc ? double(sc) : -__builtin_inf();
        }
    }
    __syncthreads();
    return true;
}

// The beam of a list.
__device__ __forceinline__ int beam_of(const BeamSelectArgs & a, int list) {
    return min(a.chunk_mul ? int(__umulhi(unsigned(list), a.chunk_mul)) : list, a.n_beam - 1);
}

// A list entry's value.
__device__ __forceinline__ double beam_value(unsigned long long e, int b, const double * top, const double * logsum, const double * scores) {
    const float x = beam_number(uint32_t(e >> 32));
    return x > -__builtin_inff() && scores[b] > -__builtin_inf() ? scores[b] + ((double(x) - top[b]) - logsum[b]) : -__builtin_inf();
}
constexpr uint32_t BEAM_NONE = 0xffffffffu;  // beam * n_vocab + token of an empty list's head

// The lists' first `depth` entries in LDS as values and indexes, formed by all threads at once. Lists of which more is taken are read
// further from memory (a microsecond each).
constexpr int BEAM_LDS = 4096;  // entries: one at least of each list
struct BeamLists {
    const unsigned long long * li;
    double * v;
    uint32_t * id;
    const double * top, * logsum, * scores;
    int k, depth;

    __device__ __forceinline__ void form(const BeamSelectArgs & a, unsigned long long e, int l, double & value, uint32_t & index) const {
        const int b = beam_of(a, l);
        value = e ? beam_value(e, b, top, logsum, scores) : -__builtin_inf();
        index = e ? uint32_t(b) * uint32_t(a.n_vocab) + ~uint32_t(e) : BEAM_NONE;
    }
    __device__ __forceinline__ void at(const BeamSelectArgs & a, int l, int i, double & value, uint32_t & index) const {
        if (i < depth) {
            value = v[l * depth + i];
            index = id[l * depth + i];
        } else {
            form(a, i < k ? li[size_t(l) * k + i] : 0, l, value, index);
        }
    }
};
struct BeamShared {
    double v[BEAM_LDS], top[BEAM_MAX], logsum[BEAM_MAX], scores[BEAM_MAX], won[BEAM_MAX];
    uint32_t id[BEAM_LDS], taken[BEAM_MAX];
};
// False: the group reads its prompt.
template <int T>
__device__ __forceinline__ bool beam_fetch(const BeamSelectArgs & a, int g, BeamShared & sh, BeamLists & out) {
    const int k = a.n_beam, lists = k * a.chunks, depth = min(k, BEAM_LDS / lists), n = lists * depth;
    const unsigned long long * li = beam_lists(a) + size_t(g) * lists * k;
    out = {li, sh.v, sh.id, sh.top, sh.logsum, sh.scores, k, depth};
    constexpr int AHEAD = BEAM_LDS / T < 8 ? BEAM_LDS / T : 8;  // reads in flight a thread, beside the rows' sums
    unsigned long long x[AHEAD];
    const auto where = [&](int i) { return depth == k ? i : i / depth * k + i % depth; };
#pragma unroll
    for (int e = 0; e < AHEAD; ++e) {
        const int i = threadIdx.x + e * T;
        x[e] = i < n ? li[where(i)] : 0;
    }
    if (!beam_rows<T / 64>(a, g, sh.top, sh.logsum, sh.scores)) return false;
#pragma unroll
    for (int e = 0; e < AHEAD; ++e) {
        const int i = threadIdx.x + e * T;
        if (i < n) out.form(a, x[e], i / depth, sh.v[i], sh.id[i]);
    }
    for (int i = threadIdx.x + AHEAD * T; i < n; i += T) out.form(a, li[where(i)], i / depth, sh.v[i], sh.id[i]);
    __syncthreads();
    return true;
}

// The winners, written at the end (a store in a step would be waited for in the next one's reads).
__device__ __forceinline__ void beam_write(const BeamSelectArgs & a, int g, const BeamShared & sh, int j) {
    const uint32_t b = sh.taken[j] / uint32_t(a.n_vocab);
    const int to = (g * a.n_beam + j) * a.slot;
    a.score_out[to] = float(sh.won[j]);
    a.token[to] = int32_t(sh.taken[j] - b * uint32_t(a.n_vocab));
    a.parent[to] = int32_t(b);
}

__device__ __forceinline__ bool beam_better(double v2, uint32_t i2, double v1, uint32_t i1) { return v2 > v1 || (v2 == v1 && i2 < i1); }

// The best of N heads, as a tree.
template <int N>
__device__ __forceinline__ void beam_best(const double * v, const uint32_t * id, double & bv, uint32_t & bi) {
    if constexpr (N == 1) {
        bv = v[0];
        bi = id[0];
    } else {
        double v2;
        uint32_t i2;
        beam_best<N / 2>(v, id, bv, bi);
        beam_best<N - N / 2>(v + N / 2, id + N / 2, v2, i2);
        const bool other = beam_better(v2, i2, bv, bi);
        bv = other ? v2 : bv;
        bi = other ? i2 : bi;
    }
}

// The wave's largest value, in every lane (by DPP alone: the rows of 16 upwards, then row 15 into the next and 31 into the upper half).
__device__ __forceinline__ double wave_best(double x) {
    const auto step = [&](auto ctrl, auto rows) {
        const long long y = __double_as_longlong(x);
        const int lo = __builtin_amdgcn_update_dpp(int(y), int(y), ctrl.value, rows.value, 0xf, false);
        const int hi = __builtin_amdgcn_update_dpp(int(y >> 32), int(y >> 32), ctrl.value, rows.value, 0xf, false);
        x = fmax(x, __hiloint2double(hi, lo));
    };
    using std::integral_constant;
    step(integral_constant<int, 0x111>(), integral_constant<int, 0xf>());  // row_shr:1, 2, 4, 8
    step(integral_constant<int, 0x112>(), integral_constant<int, 0xf>());
    step(integral_constant<int, 0x114>(), integral_constant<int, 0xf>());
    step(integral_constant<int, 0x118>(), integral_constant<int, 0xf>());
    step(integral_constant<int, 0x142>(), integral_constant<int, 0xa>());  // row_bcast:15 into rows 1 and 3
    step(integral_constant<int, 0x143>(), integral_constant<int, 0xc>());  // row_bcast:31 into rows 2 and 3
    const long long y = __double_as_longlong(x);
    return __hiloint2double(__builtin_amdgcn_readlane(int(y >> 32), 63), __builtin_amdgcn_readlane(int(y), 63));
}

// Workgroup per group of up to 64 * OWN lists: after the rows' sums its first wave alone, one winner a step. A lane holds the heads of
// OWN lists, the best of them and, read ahead, what follows it in its list.
template <int OWN>
__global__ __launch_bounds__(256) void beam_pick_wave_kernel(BeamSelectArgs a) {
    __shared__ BeamShared sh;
    const int g = blockIdx.x, k = a.n_beam, tid = threadIdx.x, lists = k * a.chunks;
    BeamLists li;
    if (!beam_fetch<256>(a, g, sh, li) || tid >= 64) return;
    double v[OWN], bv, nv;
    uint32_t id[OWN], bi, ni;
    int taken[OWN];
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
        taken[i] = 0;
        v[i] = -__builtin_inf();
        id[i] = BEAM_NONE;
        if (tid + 64 * i < lists) li.at(a, tid + 64 * i, 0, v[i], id[i]);
    }
    const auto best = [&] {
        beam_best<OWN>(v, id, bv, bi);
        int l = 0, t = 0;
#pragma unroll
        for (int i = 0; i < OWN; ++i)
            if (id[i] == bi) {
                l = tid + 64 * i;
                t = taken[i];
            }
        nv = -__builtin_inf();
        ni = BEAM_NONE;
        if (bi != BEAM_NONE) li.at(a, l, t + 1, nv, ni);
    };
    best();
    for (int j = 0; j < k; ++j) {
        const double wv = wave_best(bv);
        const unsigned long long who = __ballot(bv == wv);
        uint32_t wi;
        if (__popcll(who) == 1) {
            wi = uint32_t(__builtin_amdgcn_readlane(int(bi), __ffsll(who) - 1));
        } else {  // equal values: the lowest index
            wi = __builtin_amdgcn_readfirstlane(wave_u32(bv == wv ? bi : BEAM_NONE, min_u));
        }
        if (bi == wi) {
            sh.won[j] = wv;
            sh.taken[j] = wi;
#pragma unroll
            for (int i = 0; i < OWN; ++i)
                if (id[i] == wi) {
                    ++taken[i];
                    v[i] = nv;
                    id[i] = ni;
                }
            best();
        }
    }
    wave_lds();
    if (tid < k) beam_write(a, g, sh, tid);
}

// A better candidate of the pair keeps the lane where `first`, the other one the lane's partner.
__device__ __forceinline__ void beam_exchange(double & v, uint32_t & id, double v2, uint32_t i2, bool first) {
    const bool take = beam_better(v2, i2, v, id) == first;
    v = take ? v2 : v;
    id = take ? i2 : id;
}
template <int XOR>
__device__ __forceinline__ void beam_stage(double & v, uint32_t & id, int lane) {  // lanes XOR apart, in groups of 32
    constexpr int PATTERN = XOR << 10 | 0x1f;
    const long long x = __double_as_longlong(v);
    const int lo = __builtin_amdgcn_ds_swizzle(int(x), PATTERN), hi = __builtin_amdgcn_ds_swizzle(int(x >> 32), PATTERN);
    const uint32_t i2 = uint32_t(__builtin_amdgcn_ds_swizzle(int(id), PATTERN));
    beam_exchange(v, id, __hiloint2double(hi, lo), i2, (lane & XOR) == 0);
}
// 32 lanes' candidates, in order, become the best 32 of them and of another 32 in order, whose number 31 - lane the lane brings.
__device__ __forceinline__ void beam_merge(double & v, uint32_t & id, double v2, uint32_t i2, int lane) {
    beam_exchange(v, id, v2, i2, true);  // the best 32, rising and then falling
    beam_stage<16>(v, id, lane);
    beam_stage<8>(v, id, lane);
    beam_stage<4>(v, id, lane);
    beam_stage<2>(v, id, lane);
    beam_stage<1>(v, id, lane);
}

// Many winners, or many lists: halves of waves each merge their share of the lists into their best 32 in order (a list whose head is no
// better than the k-th so far is passed by), and those then pairwise.
__global__ __launch_bounds__(1024) void beam_pick_merge_kernel(BeamSelectArgs a) {
    constexpr int T = 1024, H = T / 32;
    __shared__ BeamShared sh;
    __shared__ double bestv[H / 2][32];
    __shared__ uint32_t besti[H / 2][32];
    const int g = blockIdx.x, k = a.n_beam, tid = threadIdx.x, lane = tid & 31, half = tid >> 5, lists = k * a.chunks;
    BeamLists li;
    if (!beam_fetch<T>(a, g, sh, li)) return;
    double v = -__builtin_inf();
    uint32_t id = BEAM_NONE;
    const int there = 31 - lane;
    for (int l = half; l < lists; l += H) {
        double hv, v2 = -__builtin_inf();
        uint32_t hi, i2 = BEAM_NONE;
        li.at(a, l, 0, hv, hi);
        const bool worth = beam_better(hv, hi, __shfl(v, k - 1, 32), uint32_t(__shfl(int(id), k - 1, 32)));
        if (!__any(worth)) continue;
        if (worth && there < k) li.at(a, l, there, v2, i2);
        beam_merge(v, id, v2, i2, lane);
    }
    for (int n = H / 2; n >= 1; n /= 2) {
        if (half >= n && half < 2 * n) {
            bestv[half - n][there] = v;
            besti[half - n][there] = id;
        }
        __syncthreads();
        if (half < n) beam_merge(v, id, bestv[half][lane], besti[half][lane], lane);
        __syncthreads();
    }
    if (tid < k) {
        sh.won[tid] = v;
        sh.taken[tid] = id;
        beam_write(a, g, sh, tid);
    }
}

// ---- reordering ----
// Workgroup (4 KB of one part of an array, group): a thread takes the same 16 bytes of all the group's rows, first
// the sources of every row that changes, then the writes: in place, each moved byte read from HBM and written once (a source with
// several heirs is read again from the caches). Rows that stay cost nothing. Bound by the memory: 4 groups of 8, 8 caches of 2000
// positions (2.3 GB read and written): 419 us, 5.5 TB/s; one group of 4 with 24 layers of states (327 MB): 66 us, 5.0 TB/s. Few and
// short arrays: three trips to memory (one group of 15, 2.6 MB: 8.4 us).

// The rows from I on at `at` in the tile: row I's source is read, the further rows' all follow, then row I is written. (A recursion:
// with an array of 8 pieces the compiler keeps one value of 32 registers, and copies of it.)
template <int I, int NB, typename V>
__device__ __forceinline__ void beam_rows_move(uint8_t * at, int off, int bytes, int p, unsigned long long row_stride) {
    if constexpr (I < NB) {
        const bool on = off < __builtin_amdgcn_readlane(bytes, I);
        V x = {};
        if (on) x = *reinterpret_cast<const V *>(at + __builtin_amdgcn_readlane(p, I) * row_stride);
        beam_rows_move<I + 1, NB, V>(at, off, bytes, p, row_stride);
        if (on) *reinterpret_cast<V *>(at + I * row_stride) = x;
    }
}

// Each wave's lanes look at a row each first: its parent and the bytes that move, which all lanes then take from there.
template <int NB, typename V>
__device__ __forceinline__ void beam_move(const BeamMove & m, const int32_t * parent, int slot, uint8_t * part, unsigned long long from, int n_beam,
                                          int row0) {
    const int lane = threadIdx.x & 63;
    int p = lane < n_beam ? parent[size_t(row0 + lane) * slot] : -1;
    if (p == lane || p >= n_beam) p = -1;
    unsigned long long hi = p < 0 ? 0 : m.hi;
    if (m.used && p >= 0) {
        const long long u = (long long)m.used[size_t(row0 + p) * m.used_stride] + m.used_more;
        const unsigned long long units = u > 0 ? ((unsigned long long)u + m.unit_len - 1) / m.unit_len : 0;
        hi = min(hi, units * m.unit_bytes);
    }
    const int bytes = hi > from ? int(min(hi - from, (unsigned long long)BEAM_TILE)) : 0;  // of this tile
    if (!__any(bytes > 0)) return;
#pragma unroll 1
    for (int off = threadIdx.x * sizeof(V); off < int(BEAM_TILE); off += 256 * sizeof(V))
        beam_rows_move<0, NB, V>(part + from + off, off, bytes, p, m.row_stride);
}

template <int NB>
__global__ __launch_bounds__(256) void beam_reorder_kernel(BeamReorderArgs a) {
    int i = 0;
    while (blockIdx.x >= a.m[i].end) ++i;
    const BeamMove & m = a.m[i];
    const uint32_t t = blockIdx.x - (i ? a.m[i - 1].end : 0), p = t / m.tiles;
    const int row0 = blockIdx.y * a.n_beam;
    uint8_t * part = m.data + row0 * m.row_stride + p * m.part_stride;
    const unsigned long long from = m.lo + (unsigned long long)(t - p * m.tiles) * BEAM_TILE;
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    if (m.wide) beam_move<NB, u32x4>(m, a.parent, a.parent_stride, part, from, a.n_beam, row0);
    else beam_move<NB, uint32_t>(m, a.parent, a.parent_stride, part, from, a.n_beam, row0);
}

// A launch (5 us in a list): its ids follow the moves of the id lists, which follow the selection.
__global__ void beam_next_kernel(BeamNextArgs a) {
    const int s = threadIdx.x;
    if (s >= a.n_seq) return;
    const int p = a.pos[16 * s] + 1;
    if (p >= 0 && p < a.cap) a.out[size_t(s) * a.cap + p] = a.tok[16 * s];
    a.pos[16 * s] = p;
}

int beam_chunks(int n_vocab, int per) { return (n_vocab + 256 * per - 1) / (256 * per); }
// Logits a thread of the first kernel takes: 8, the shorter way through one workgroup, or 32 where those would give the second kernel
// 192 lists a group or the first more workgroups than the device holds at once. Both kernels with 8 and 32: 10.0 and 11.0 us at one
// group of 4 of 32000, 10.4 and 10.8 at one of 2 of 151936, 14.6 and 16.5 at 70 of 8 of 4000; 12.6 and 11.6 at one of 4 of 151936, 15.5
// and 14.4 at one of 12 of 32000, 16.0 and 14.1 at 20 of 5 of 32003, 41.6 and 25.0 at 8 of 8 of 151936.
int beam_per(int n_group, int n_beam, int n_vocab) {
    const int lists = n_beam * beam_chunks(n_vocab, 8);
    return lists >= 192 || (long long)n_group * lists >= 1536 ? 32 : 8;
}

}  // namespace

size_t beam_work(int n_group, int n_beam, int n_vocab) {
    const long long rows = (long long)n_group * n_beam;
    const int per = beam_per(n_group, n_beam, n_vocab);
    return size_t(rows) * beam_chunks(n_vocab, per) * (sizeof(BeamStat) + 8 * size_t(n_beam));
}

// Winners from which on the lists are merged; also where a group has more lists than a wave's registers take the heads of. Both
// kernels, winners one by one and merged: 11.6 and 14.5 us at one group of 4 of 151936, 25.4 and 25.5 at 8 of 8, 18.2 and 17.0 at one of
// 10, 28.7 and 25.5 at 4 of 12; 27.3 and 20.0 at 17 of 29 of 4687. One by one with 2 and 5 lists a lane: 12.1 and 13.6 us at one of 8 of
// 32000.
constexpr int BEAM_MANY = 10;
hipError_t launch_beam_select(const BeamSelectArgs & args, hipStream_t s) {
    BeamSelectArgs a = args;
    const int rows = a.n_group * a.n_beam;
    a.per = beam_per(a.n_group, a.n_beam, a.n_vocab);
    a.chunks = beam_chunks(a.n_vocab, a.per);
    a.chunk_mul = a.chunks > 1 ? unsigned((0x100000000ull + unsigned(a.chunks) - 1) / unsigned(a.chunks)) : 0;
    const unsigned lds = unsigned(beam_list(a.n_beam, a.per) * 4 * sizeof(unsigned long long));
    const dim3 grid(unsigned(a.chunks), unsigned(rows));
    if (a.per == 32) GQ_LAUNCH(beam_scan_kernel<32>, grid, dim3(256), lds, s, a);
    else GQ_LAUNCH(beam_scan_kernel<8>, grid, dim3(256), lds, s, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    // lists of a group: at most 32 * 128
    const int lists = a.n_beam * a.chunks;
    const dim3 groups(unsigned(a.n_group));
    if (a.n_beam >= BEAM_MANY || lists > 64 * 5) GQ_LAUNCH(beam_pick_merge_kernel, groups, dim3(1024), 0, s, a);
    else if (lists <= 64 * 2) GQ_LAUNCH(beam_pick_wave_kernel<2>, groups, dim3(256), 0, s, a);
    else GQ_LAUNCH(beam_pick_wave_kernel<5>, groups, dim3(256), 0, s, a);
    return hipGetLastError();
}

hipError_t launch_beam_next(const BeamNextArgs & a, hipStream_t s) {
    GQ_LAUNCH(beam_next_kernel, dim3(1), dim3(64), 0, s, a);
    return hipGetLastError();
}

hipError_t launch_beam_reorder(const BeamReorderArgs & a, hipStream_t s) {
    const dim3 grid(a.m[a.n - 1].end, unsigned(a.n_group));
    if (a.n_beam <= 4) GQ_LAUNCH(beam_reorder_kernel<4>, grid, dim3(256), 0, s, a);
    else if (a.n_beam <= 8) GQ_LAUNCH(beam_reorder_kernel<8>, grid, dim3(256), 0, s, a);
    else if (a.n_beam <= 16) GQ_LAUNCH(beam_reorder_kernel<16>, grid, dim3(256), 0, s, a);
    else GQ_LAUNCH(beam_reorder_kernel<32>, grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace gq
