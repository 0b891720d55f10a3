// Verification of drafted tokens (gq_draft.h), in two launches. The first reads every logit once: the maximum and the sum of
// exponentials of every chunk of a row (and, at temperature 0, the place of the maximum). In the second, every workgroup of a sequence
// joins its rows' chunks, decides how many tokens stand, and sums what is left of one chunk of the one row that a new token comes
// from; the last workgroup of the sequence to be done finds the token. Distributions are in 64 bits throughout: a token is found where a
// sum of up to 2^20 terms passes a given number, and the borders of all of them have to be where they belong.
#include "gq_device.h"
#include "gq_draft.h"

#include <cfloat>
#include <type_traits>

namespace gq {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_at_4 __attribute__((ext_vector_type(4), aligned(4)));

// 2^t for -1020 < t <= 0 (0 for others): t = n + f with |f| <= 1/2, 1 + f q(f) with q interpolating (2^f - 1) / f at 10 Chebyshev
// points (off by at most 5.7e-16 of 2^f), and n added to the exponent. n comes out of u = t + 1.5 * 2^52 as its low word.
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
    return t > -1020.0 ? __hiloint2double(__double2hiint(p) + (__double2loint(u) << 20), __double2loint(p)) : 0.0;
}
// e^((x - m) / temperature) with c = log2(e) / temperature, for x <= m; 0 for x = -inf, whatever m is.
__device__ __forceinline__ double draft_term(float x, double m, double c) { return draft_exp2((double(x) - m) * c); }
__device__ __forceinline__ float draft_clean(float x) { return x == x ? fminf(x, FLT_MAX) : -__builtin_inff(); }
__device__ __forceinline__ double draft_scale(double temperature) {
    return 1.4426950408889634 / (temperature > 0.0 ? temperature : 1.0);
}

template <typename T, typename F>
__device__ __forceinline__ T over_wave(T x, F f) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) x = f(x, __shfl_xor(x, d, WAVE));
    return x;
}
__device__ __forceinline__ double sum_d(double a, double b) { return a + b; }
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

// The workspace: what each chunk of every row comes to (target rows, then draft rows), the chunks' sums of what is left, and how many
// workgroups of each sequence are done.
struct DraftWork {
    DraftStat * stat;
    double * left;
    unsigned * done;
};
__host__ __device__ inline long long draft_rows(const DraftArgs & a) { return (long long)a.n_seq * (2 * a.n_draft + 1); }
__device__ __forceinline__ DraftWork draft_at(const DraftArgs & a) {
    DraftWork w;
    w.stat = static_cast<DraftStat *>(a.work);
    w.left = reinterpret_cast<double *>(w.stat + draft_rows(a) * a.chunks);
    w.done = reinterpret_cast<unsigned *>(w.left + (long long)a.n_seq * a.chunks);
    return w;
}
__device__ __forceinline__ int draft_num(const DraftArgs & a, int s) { return a.num ? min(a.num[s], a.n_draft) : a.n_draft; }

// PER logits a thread, four in a row each; behind the row: -inf.
template <int PER, typename F>
__device__ __forceinline__ void draft_load(const float * x, int n, F place, float * v) {
#pragma unroll
    for (int i = 0; i < PER / 4; ++i) {
        const int t = place(i);
        if (t + 4 <= n) {
            *reinterpret_cast<f32x4 *>(v + 4 * i) = *reinterpret_cast<const f32x4_at_4 *>(x + t);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * i + e] = t + e < n ? x[t + e] : -__builtin_inff();
        }
    }
}

// Workgroup (chunk of 256 * PER logits | row of the target, then of the draft).
template <int PER>
__global__ __launch_bounds__(256) void draft_scan_kernel(DraftArgs a) {
    __shared__ DraftStat red[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, chunk = blockIdx.x, trows = a.n_seq * (a.n_draft + 1);
    const bool own = int(blockIdx.y) < trows;
    const int row = own ? blockIdx.y : blockIdx.y - trows, each = own ? a.n_draft + 1 : a.n_draft, s = row / each, t = row - s * each;
    const DraftWork w = draft_at(a);
    if (own && t == 0 && chunk == 0 && tid == 0) w.done[s] = 0;
    const int num = draft_num(a, s);
    if (own ? t > num : t >= num) return;
    const float * x = own ? a.target + row * a.target_stride : a.draft + row * a.draft_stride;
    const int v0 = chunk * 256 * PER;
    float v[PER];
    draft_load<PER>(x, a.n_vocab, [&](int i) { return v0 + 4 * (256 * i + tid); }, v);
    float m = -__builtin_inff();
    int at = 0x7fffffff;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        v[j] = draft_clean(v[j]);
        m = fmaxf(m, v[j]);
    }
    if (a.temperature == 0.0) {
#pragma unroll
        for (int j = PER - 1; j >= 0; --j) at = v[j] == m ? v0 + 4 * (256 * (j >> 2) + tid) + (j & 3) : at;
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) {
            const float m2 = __shfl_xor(m, d, WAVE);
            const int at2 = __shfl_xor(at, d, WAVE);
            draft_best(m, at, m2, at2);
        }
    } else {
        m = over_wave(m, max_f);
    }
    const double c = draft_scale(own ? a.temperature : a.draft_temperature);
    double sum = 0.0;
    if (m > -__builtin_inff()) {
#pragma unroll
        for (int j = 0; j < PER; ++j) sum += draft_term(v[j], m, c);
    }
    sum = over_wave(sum, sum_d);
    if (lane == 0) red[wave] = {m, at, sum};
    __syncthreads();
    if (tid) return;
    DraftStat r = {red[0].m, red[0].at, 0.0};
    for (int i = 1; i < 4; ++i) draft_best(r.m, r.at, red[i].m, red[i].at);
    for (int i = 0; i < 4; ++i) r.sum += red[i].sum * draft_term(red[i].m, r.m, c);
    w.stat[(own ? row : (long long)trows + row) * a.chunks + chunk] = r;
}

// Workgroup (chunk | sequence).
template <int PER>
__global__ __launch_bounds__(256) void draft_pick_kernel(DraftArgs a) {
    constexpr int ROWS = 2 * DRAFT_MAX + 1;
    __shared__ float top[ROWS], rowsum_m[4];
    __shared__ int arg[ROWS], accepted, last, found;
    __shared__ double total[ROWS], red[4], base;
    __shared__ double part[256];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, chunk = blockIdx.x, s = blockIdx.y;
    const int num = draft_num(a, s);
    if (num < 0) return;
    const bool greedy = a.temperature == 0.0, rows_of_draft = a.draft && !greedy;
    const DraftWork w = draft_at(a);
    const double c = draft_scale(a.temperature), cq = draft_scale(a.draft_temperature);
    const long long trow = (long long)s * (a.n_draft + 1), drow = (long long)s * a.n_draft, trows = (long long)a.n_seq * (a.n_draft + 1);
    // ---- the rows: 0 .. num the target's, then the draft's ----
    for (int r = wave; r < num + 1 + (rows_of_draft ? num : 0); r += 4) {
        const bool mine = r <= num;
        const DraftStat * st = w.stat + (mine ? trow + r : trows + drow + (r - num - 1)) * a.chunks;
        const double cr = mine ? c : cq;
        float m = -__builtin_inff();
        int at = 0x7fffffff;
        double sum = 0.0;
        for (int i = lane; i < a.chunks; i += 64) {
            const DraftStat x = st[i];
            const float m2 = fmaxf(m, x.m);
            if (m2 > -__builtin_inff()) sum = sum * draft_term(m, m2, cr) + x.sum * draft_term(x.m, m2, cr);
            draft_best(m, at, x.m, x.at);
        }
        float m1 = m;
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) {
            const float m2 = __shfl_xor(m1, d, WAVE);
            const int at2 = __shfl_xor(at, d, WAVE);
            draft_best(m1, at, m2, at2);
        }
        sum = over_wave(m > -__builtin_inff() ? sum * draft_term(m, m1, cr) : 0.0, sum_d);
        if (lane == 0) {
            top[r] = m1;
            arg[r] = at;
            total[r] = sum;
        }
    }
    __syncthreads();
    // ---- how many tokens stand ----
    if (wave == 0) {
        const int d = lane < num ? a.token[drow + lane] : -1;
        bool ok = lane < num && d >= 0 && d < a.n_vocab && top[lane] > -__builtin_inff();
        if (ok && greedy) {
            ok = d == arg[lane];
        } else if (ok) {
            const double p = draft_term(draft_clean(a.target[(trow + lane) * a.target_stride + d]), top[lane], c) / total[lane];
            double q = 1.0;
            if (a.draft) {
                const float m = top[num + 1 + lane];
                q = m > -__builtin_inff() ? draft_term(draft_clean(a.draft[(drow + lane) * a.draft_stride + d]), m, cq) / total[num + 1 + lane] : 0.0;
            }
            ok = double(a.uniform[trow + lane]) * q < p;
        }
        const unsigned long long no = ~__ballot(ok);
        if (lane == 0) accepted = __ffsll(no) - 1;  // (lanes from num on say no)
    }
    __syncthreads();
    const int k = accepted;
    const float m = top[k];
    const auto finish = [&](int token) {  // by the first wave
        if (lane > a.n_draft) return;
        const int tok = lane < k ? a.token[drow + lane] : lane == k ? token : -1;
        a.out[trow + lane] = tok;
        if (lane == 0) a.n_accept[s] = k;
        if (!a.logp) return;
        double l = 0.0;
        if (tok >= 0) l = (double(draft_clean(a.target[(trow + lane) * a.target_stride + tok])) - top[lane]) * c * 0.6931471805599453 - log(total[lane]);
        a.logp[trow + lane] = float(l);
    };
    if (greedy || !(m > -__builtin_inff())) {
        if (chunk == 0 && wave == 0) finish(m > -__builtin_inff() ? arg[k] : -1);
        return;
    }
    // ---- what is left of this chunk ----
    const float * xp = a.target + (trow + k) * a.target_stride;
    const float * xq = k < num && a.draft ? a.draft + (drow + k) * a.draft_stride : nullptr;
    const double ip = 1.0 / total[k];
    double iq = 0.0;
    float mq = 0.0f;
    if (xq && top[num + 1 + k] > -__builtin_inff()) {
        iq = 1.0 / total[num + 1 + k];
        mq = top[num + 1 + k];
    }
    const int certain = k < num && !a.draft ? a.token[drow + k] : -1;
    const auto weights = [&](auto place, double * v, bool whole) {  // of PER tokens, four in a row each
        float p[PER], q[PER];
        draft_load<PER>(xp, a.n_vocab, place, p);
        if (xq) draft_load<PER>(xq, a.n_vocab, place, q);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            v[j] = draft_term(draft_clean(p[j]), m, c) * ip;
            if (whole) continue;
            if (xq) v[j] = fmax(v[j] - draft_term(draft_clean(q[j]), mq, cq) * iq, 0.0);
            else if (place(j >> 2) + (j & 3) == certain) v[j] = 0.0;
        }
    };
    const int v0 = chunk * 256 * PER;
    {
        double v[PER], sum = 0.0;
        weights([&](int i) { return v0 + 4 * (256 * i + tid); }, v, false);
#pragma unroll
        for (int j = 0; j < PER; ++j) sum += v[j];
        sum = over_wave(sum, sum_d);
        if (lane == 0) red[wave] = sum;
    }
    __syncthreads();
    if (tid == 0) {
        __hip_atomic_store(w.left + (long long)s * a.chunks + chunk, (red[0] + red[1]) + (red[2] + red[3]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last = __hip_atomic_fetch_add(w.done + s, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == unsigned(a.chunks) - 1;
    }
    __syncthreads();
    if (!last) return;
    // ---- the token: its chunk, its thread's PER tokens, itself ----
    if (wave == 0) {
        double all = 0.0;
        const double * left = w.left + (long long)s * a.chunks;
        const DraftStat * st = w.stat + (trow + k) * a.chunks;
        const auto of = [&](int i, bool whole) {
            if (i >= a.chunks) return 0.0;
            return whole ? st[i].sum * draft_term(st[i].m, m, c) * ip : __hip_atomic_load(left + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        };
        for (int i = lane; i < a.chunks; i += 64) all += of(i, false);
        all = over_wave(all, sum_d);
        const bool whole = !(all > 0.0);  // nothing is left: the row as it is
        if (whole) {
            all = 0.0;
            for (int i = lane; i < a.chunks; i += 64) all += of(i, true);
            all = over_wave(all, sum_d);
        }
        const float u = a.uniform[trow + a.n_draft];
        const double goal = all * double(u);
        double before = 0.0, start = 0.0;
        int at = -1;
        for (int i0 = 0; i0 < a.chunks && at < 0; i0 += 64) {
            const double mine = of(i0 + lane, whole);
            double upto = mine;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const double y = __shfl_up(upto, d, WAVE);
                if (lane >= d) upto += y;
            }
            upto += before;
            const unsigned long long past = __ballot(mine > 0.0 && upto > goal), some = __ballot(mine > 0.0);
            if (past) {
                at = i0 + __ffsll(past) - 1;
                start = __shfl(upto - mine, __ffsll(past) - 1, WAVE);
            } else if (some) {  // the last one with anything, where rounding leaves no sum above the goal
                found = i0 + 63 - __clzll(some);
            }
            before = __shfl(upto, 63, WAVE);
        }
        if (lane == 0) {
            base = at < 0 ? __builtin_inf() : goal - start;  // infinite: the last token with a weight
            if (at >= 0) found = at;
            last = whole ? 2 : 1;
        }
    }
    __syncthreads();
    const int w0 = found * 256 * PER + tid * PER;
    const double goal = base;
    const bool whole = last == 2;
    double v[PER], sum = 0.0;
    weights([&](int i) { return w0 + 4 * i; }, v, whole);
#pragma unroll
    for (int j = 0; j < PER; ++j) sum += v[j];
    double upto = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const double y = __shfl_up(upto, d, WAVE);
        if (lane >= d) upto += y;
    }
    if (lane == 63) red[wave] = upto;
    __syncthreads();
    double start = upto - sum;
    for (int i = 0; i < wave; ++i) start += red[i];
    // a thread's first token past the goal, and its last one with a weight; the first thread's of all, else the last's
    int first = -1, end = -1;
    double run = start;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        run += v[j];
        if (v[j] > 0.0) {
            end = w0 + j;
            if (first < 0 && run > goal) first = w0 + j;
        }
    }
    int * firsts = reinterpret_cast<int *>(part);
    const unsigned long long has = __ballot(first >= 0), any = __ballot(end >= 0);
    const int f = __shfl(first, has ? __ffsll(has) - 1 : 0, WAVE), e = __shfl(end, any ? 63 - __clzll(any) : 0, WAVE);
    if (lane == 0) {
        firsts[wave] = has ? f : -1;
        firsts[4 + wave] = any ? e : -1;
    }
    __syncthreads();
    if (wave) return;
    int token = -1;
    for (int i = 3; i >= 0; --i) token = firsts[i] >= 0 ? firsts[i] : token;
    if (token < 0)
        for (int i = 0; i < 4; ++i) token = firsts[4 + i] >= 0 ? firsts[4 + i] : token;
    finish(token);
}

int draft_chunks(int n_vocab, int per) { return (n_vocab + 256 * per - 1) / (256 * per); }
int draft_per(int n_seq, int n_draft, int n_vocab) { return (long long)n_seq * (2 * n_draft + 1) * draft_chunks(n_vocab, 8) >= 1536 ? 32 : 8; }

}  // namespace

size_t draft_work(int n_seq, int n_draft, int n_vocab) {
    const size_t chunks = size_t(draft_chunks(n_vocab, draft_per(n_seq, n_draft, n_vocab)));
    return size_t(n_seq) * ((size_t(2 * n_draft + 1) * sizeof(DraftStat) + sizeof(double)) * chunks + sizeof(unsigned));
}

hipError_t launch_draft(const DraftArgs & args, hipStream_t s) {
    DraftArgs a = args;
    a.per = draft_per(a.n_seq, a.n_draft, a.n_vocab);
    a.chunks = draft_chunks(a.n_vocab, a.per);
    const bool draft = a.draft && a.temperature > 0.0;
    const dim3 rows(unsigned(a.chunks), unsigned(a.n_seq * (a.n_draft + 1 + (draft ? a.n_draft : 0)))), seqs(unsigned(a.chunks), unsigned(a.n_seq));
    if (a.per == 32) GQ_LAUNCH(draft_scan_kernel<32>, rows, dim3(256), 0, s, a);
    else GQ_LAUNCH(draft_scan_kernel<8>, rows, dim3(256), 0, s, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (a.per == 32) GQ_LAUNCH(draft_pick_kernel<32>, seqs, dim3(256), 0, s, a);
    else GQ_LAUNCH(draft_pick_kernel<8>, seqs, dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace gq
