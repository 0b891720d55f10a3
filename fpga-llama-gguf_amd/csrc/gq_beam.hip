// The beam search's kernels (gq_beam.h).
#include "gq_beam.h"
#include "gq_device.h"

#include <cfloat>

namespace gq {
namespace {

// ---- selection ----
// Two launches. The first reads every logit once: workgroup (256 * PER logits of a row) forms their maximum m and sum of e^(x - m),
// and their n_beam best in order. The second, a workgroup per group, joins the rows' sums, and takes the best candidate off the
// sorted lists n_beam times. Values are 64-bit from the logits on (candidates of two beams may lie next to each other): e^(x - m) as
// 2^n times a polynomial of degree 9, with an error below 1e-11.
// A list entry is one word that orders as the candidates of one row do: the logit's bits made monotone, above the token inverted.
constexpr int BEAM_SLACK = 8;

__device__ __forceinline__ uint32_t order_of(float x) {  // monotone in x, > 0 for every number
    const uint32_t b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }

// e^t for t <= 0 (t = -inf and below the range: 0).
__device__ __forceinline__ double beam_exp(double t) {
    t = fmax(t * 1.4426950408889634, -1100.0);
    const double n = __builtin_rint(t), r = (t - n) * 0.6931471805599453;
    double p = 1.0 / 362880;
    p = __builtin_fma(p, r, 1.0 / 40320);
    p = __builtin_fma(p, r, 1.0 / 5040);
    p = __builtin_fma(p, r, 1.0 / 720);
    p = __builtin_fma(p, r, 1.0 / 120);
    p = __builtin_fma(p, r, 1.0 / 24);
    p = __builtin_fma(p, r, 1.0 / 6);
    p = __builtin_fma(p, r, 0.5);
    p = __builtin_fma(p, r, 1.0);
    p = __builtin_fma(p, r, 1.0);
    return __builtin_ldexp(p, int(n));
}

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

// A row that takes no logits: a beam that has ended (its one candidate), or one without a score (none).
__device__ __forceinline__ bool beam_closed(const BeamSelectArgs & a, int row, bool & ended) {
    const size_t at = size_t(row) * a.slot;
    ended = a.last && a.last[at] == a.eos && a.eos >= 0 && a.eos < a.n_vocab && !(a.pos && a.pos[at] < a.n_prompt[at]);
    return ended || !(a.score[at] > -__builtin_inff());
}
// Whether the row's prompt has a next id; its place in the prompt.
__device__ __forceinline__ bool beam_prompted(const BeamSelectArgs & a, int row, int & next) {
    if (!a.pos) return false;
    next = a.pos[size_t(row) * a.slot] + 1;
    return next >= 0 && next < min(a.n_prompt[size_t(row) * a.slot], a.cap);
}

template <int PER>
__global__ __launch_bounds__(256) void beam_scan_kernel(BeamSelectArgs a) {
    constexpr int CH = 256 * PER;
    extern __shared__ unsigned long long list[];  // the waves' candidates: (n_beam + BEAM_SLACK) * PER each
    __shared__ float red[4];
    __shared__ double sums[4];
    __shared__ int count[4];
    const int row = blockIdx.y, chunk = blockIdx.x, k = a.n_beam, tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), v0 = chunk * CH, cap = (k + BEAM_SLACK) * PER;
    const size_t at = size_t(row) * a.chunks + chunk;
    unsigned long long * out = beam_lists(a) + at * k;
    bool ended;
    int next;
    if (beam_prompted(a, row - row % k, next)) return;  // the group reads its prompt (its first beam says so, here and below)
    if (beam_closed(a, row, ended)) {
        // the first chunk lists the tokens in order at -inf, an ended beam's eos before them at 0 (of sum 1)
        for (int i = tid; i < k; i += 256) {
            const int token = ended ? (i == 0 ? a.eos : i - 1 < a.eos ? i - 1 : i) : i;
            const float x = ended && i == 0 ? 0.0f : -__builtin_inff();
            out[i] = chunk == 0 && token < a.n_vocab ? (unsigned long long)order_of(x) << 32 | uint32_t(~token) : 0ull;
        }
        if (tid == 0) beam_stats(a)[at] = {ended && chunk == 0 ? 0.0f : -__builtin_inff(), 0, ended && chunk == 0 ? 1.0 : 0.0};
        return;
    }
    const float * x = a.x + size_t(row) * size_t(a.stride);
    // elements 4 (256 i + tid) + e from the chunk's start; rows start anywhere, so the pieces are brought to 16 bytes
    const int skew = int((reinterpret_cast<uintptr_t>(x + v0) >> 2) & 3);
    typedef float f32x4 __attribute__((ext_vector_type(4)));
    float v[PER];
#pragma unroll
    for (int i = 0; i < PER / 4; ++i) {
        const int t = v0 - skew + 4 * (256 * i + tid);
        if (t >= v0 && t + 4 <= a.n_vocab) {
            *reinterpret_cast<f32x4 *>(v + 4 * i) = *reinterpret_cast<const f32x4 *>(x + t);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * i + e] = t + e >= v0 && t + e < a.n_vocab ? x[t + e] : 0.0f;
        }
    }
    const auto token_of = [&](int j) { return v0 - skew + 4 * (256 * (j >> 2) + tid) + (j & 3); };
    // the last `skew` elements of the chunk are the pieces' overhang: one more each in the first threads
    float extra = 0.0f;
    const int xt = v0 + CH - skew + tid;
    const bool more = tid < skew && xt < a.n_vocab;
    if (more) extra = x[xt];
    uint32_t o[PER];  // monotone bits, 0: no element
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int t = token_of(j);
        const float y = v[j] == v[j] ? fminf(v[j], FLT_MAX) : -__builtin_inff();
        v[j] = y;
        o[j] = t >= v0 && t < a.n_vocab ? order_of(y) : 0;
        top = max(top, o[j]);
    }
    extra = extra == extra ? fminf(extra, FLT_MAX) : -__builtin_inff();
    const uint32_t oe = more ? order_of(extra) : 0;
    top = max(top, oe);
    // ---- maximum and sum ----
    uint32_t wtop = top, wlow = top;
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
        wtop = max(wtop, uint32_t(__shfl_xor(int(wtop), d, WAVE)));
        wlow = min(wlow, uint32_t(__shfl_xor(int(wlow), d, WAVE)));
    }
    wtop = __builtin_amdgcn_readfirstlane(wtop);
    wlow = __builtin_amdgcn_readfirstlane(wlow);
    const float wm = wtop ? value_of(wtop) : -__builtin_inff();  // each wave's sum is relative to its own maximum
    double sum = 0.0;
    if (wm > -__builtin_inff()) {
#pragma unroll
        for (int j = 0; j < PER; ++j) sum += o[j] ? beam_exp(double(v[j]) - double(wm)) : 0.0;
        if (oe) sum += beam_exp(double(extra) - double(wm));
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) sum += __shfl_xor(sum, d, WAVE);
    // ---- the wave's candidates: a bound that at least k lanes' best pass, and not many more ----
    uint32_t lo = 1, hi = wtop + 1;  // at least k lanes' best are >= lo (if so many lanes have any), fewer than k are >= hi
    int n = __popcll(__ballot(top >= 1));
    if (n > k + BEAM_SLACK) {
        if (wlow) lo = wlow;
        while (hi - lo > 1 && n > k + BEAM_SLACK) {
            const uint32_t mid = lo + (hi - lo) / 2;
            const int c = __popcll(__ballot(top >= mid));
            if (c >= k) {
                lo = mid;
                n = c;
            } else {
                hi = mid;
            }
        }
    }
    int until = INT_MAX;  // of the elements at the bound itself, the tokens up to this one
    if (n > k + BEAM_SLACK) {  // many lanes' best are equal: the ones with the lowest tokens
        int mine = INT_MAX;
        if (top == lo) {
            if (oe == lo) mine = xt;
#pragma unroll
            for (int j = PER - 1; j >= 0; --j)
                if (o[j] == lo) mine = token_of(j);
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
    unsigned long long * mylist = list + wave * cap;
    int have = 0;
    const auto put = [&](uint32_t ord, int t) {
        const bool in = ord > lo || (ord == lo && t <= until);
        const unsigned long long who = __ballot(in);
        if (!who) return;
        if (in) mylist[have + __popcll(who & ((1ull << lane) - 1))] = (unsigned long long)ord << 32 | uint32_t(~t);
        have += __popcll(who);
    };
#pragma unroll
    for (int j = 0; j < PER; ++j) put(o[j], token_of(j));
    put(oe, xt);
    if (lane == 0) {
        red[wave] = wm;
        sums[wave] = sum;
        count[wave] = have;
    }
    __syncthreads();
    // ---- the chunk's: each candidate's place is the number of better ones ----
    int all = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) all += count[w];
    for (int i = lane; i < have; i += 64) {
        const unsigned long long key = mylist[i];
        int place = 0;
        for (int w = 0; w < 4; ++w)
            for (int j = 0, c = count[w]; j < c; ++j) place += list[w * cap + j] > key;
        if (place < k) out[place] = key;
    }
    for (int i = all + tid; i < k; i += 256) out[i] = 0;
    if (tid == 0) {
        const float m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        double s = 0.0;
        for (int w = 0; w < 4; ++w)
            if (red[w] > -__builtin_inff()) s += sums[w] * beam_exp(double(red[w]) - double(m));
        beam_stats(a)[at] = {m, 0, s};
    }
}

// Workgroup per group. A thread holds the heads of up to 4 of the group's lists.
template <int T>
__global__ __launch_bounds__(T) void beam_pick_kernel(BeamSelectArgs a) {
    constexpr int OWN = 4, W = T / 64;
    __shared__ double top[BEAM_MAX], logsum[BEAM_MAX], scores[BEAM_MAX];
    __shared__ double bestv[2][W];
    __shared__ uint32_t besti[2][W];
    const int g = blockIdx.x, k = a.n_beam, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lists = k * a.chunks;
    const size_t first = size_t(g) * k * a.chunks;
    int ahead;
    if (beam_prompted(a, g * k, ahead)) {  // the group's beams read their prompt
        if (tid < k && beam_prompted(a, g * k + tid, ahead)) {
            a.token[(g * k + tid) * a.slot] = a.prompt[size_t(g * k + tid) * a.cap + ahead];
            a.parent[(g * k + tid) * a.slot] = tid;
        }
        return;
    }
    const BeamStat * st = beam_stats(a) + first;
    const unsigned long long * li = beam_lists(a) + first * k;
    // the lists' first two entries, while the rows' sums are joined
    unsigned long long next[OWN], head[OWN];
    int taken[OWN];
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
        const int l = tid + i * T;
        head[i] = l < lists ? li[size_t(l) * k] : 0;
        next[i] = l < lists && k > 1 ? li[size_t(l) * k + 1] : 0;
        taken[i] = 2;
    }
    for (int b = wave; b < k; b += W) {
        float m = -__builtin_inff();
        for (int c = lane; c < a.chunks; c += 64) m = fmaxf(m, st[b * a.chunks + c].m);
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) m = fmaxf(m, __shfl_xor(m, d, WAVE));
        double s = 0.0;
        if (m > -__builtin_inff())
            for (int c = lane; c < a.chunks; c += 64) s += st[b * a.chunks + c].sum * beam_exp(double(st[b * a.chunks + c].m) - double(m));
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) s += __shfl_xor(s, d, WAVE);
        if (lane == 0) {
            const float sc = a.score[(g * k + b) * a.slot];
            top[b] = m;
            logsum[b] = log(s);
            scores[b] = sc == sc ? double(sc) : -__builtin_inf();
        }
    }
    __syncthreads();  // (score_out and token may be score and last: everything of them has been read)
    const auto value = [&](unsigned long long e, int b) {
        const float x = value_of(uint32_t(e >> 32));
        return x > -__builtin_inff() && scores[b] > -__builtin_inf() ? scores[b] + ((double(x) - top[b]) - logsum[b]) : -__builtin_inf();
    };
    double v[OWN];
    uint32_t id[OWN];  // beam * n_vocab + token; all ones: the list is empty
    const auto show = [&](int i, int b) {
        v[i] = value(head[i], b);
        id[i] = head[i] ? uint32_t(b) * uint32_t(a.n_vocab) + ~uint32_t(head[i]) : 0xffffffffu;
    };
#pragma unroll
    for (int i = 0; i < OWN; ++i) show(i, (tid + i * T) / a.chunks < k ? (tid + i * T) / a.chunks : 0);
    for (int j = 0; j < k; ++j) {
        double bv = v[0];
        uint32_t bi = id[0];
        const auto better = [](double v2, uint32_t i2, double v1, uint32_t i1) { return i2 != 0xffffffffu && (i1 == 0xffffffffu || v2 > v1 || (v2 == v1 && i2 < i1)); };
#pragma unroll
        for (int i = 1; i < OWN; ++i)
            if (better(v[i], id[i], bv, bi)) {
                bv = v[i];
                bi = id[i];
            }
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) {
            const double v2 = __shfl_xor(bv, d, WAVE);
            const uint32_t i2 = uint32_t(__shfl_xor(int(bi), d, WAVE));
            if (better(v2, i2, bv, bi)) {
                bv = v2;
                bi = i2;
            }
        }
        if (lane == 0) {
            bestv[j & 1][wave] = bv;
            besti[j & 1][wave] = bi;
        }
        __syncthreads();
        bv = bestv[j & 1][0];
        bi = besti[j & 1][0];
#pragma unroll
        for (int w = 1; w < W; ++w)
            if (better(bestv[j & 1][w], besti[j & 1][w], bv, bi)) {
                bv = bestv[j & 1][w];
                bi = besti[j & 1][w];
            }
        if (tid == 0) {
            const uint32_t b = bi / uint32_t(a.n_vocab);
            const int to = (g * k + j) * a.slot;
            a.score_out[to] = float(bv);
            a.token[to] = int32_t(bi - b * uint32_t(a.n_vocab));
            a.parent[to] = int32_t(b);
        }
#pragma unroll
        for (int i = 0; i < OWN; ++i)
            if (id[i] == bi) {  // taken: the list's next entry becomes its head
                const int l = tid + i * T;
                head[i] = next[i];
                next[i] = taken[i] < k ? li[size_t(l) * k + taken[i]] : 0;
                ++taken[i];
                show(i, l / a.chunks);
            }
    }
}

// ---- reordering ----
// Workgroup (4 KB of one part of an array, group): a thread takes the same 16 bytes of all the group's rows, first the sources of
// every row that changes, then the writes: in place, each moved byte read from HBM and written once (a source with several heirs is read again from
// the caches). Rows that stay cost nothing.
template <int NB, typename V>
__device__ __forceinline__ void beam_move(const BeamMove & m, const int32_t * parent, int slot, uint8_t * part, unsigned long long from, int n_beam,
                                          int row0) {
    constexpr int STEP = 256 * sizeof(V), N = BEAM_TILE / STEP;
    for (int it = 0; it < N; ++it) {
        const unsigned long long off = from + it * STEP + threadIdx.x * sizeof(V);
        V x[NB];
        bool moved[NB];
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            moved[i] = false;
            if (i >= n_beam) continue;
            const int p = parent[size_t(row0 + i) * slot];
            if (p == i || p < 0 || p >= n_beam) continue;
            unsigned long long hi = m.hi;
            if (m.used) {
                const long long u = (long long)m.used[size_t(row0 + p) * m.used_stride] + m.used_more;
                const unsigned long long units = u > 0 ? ((unsigned long long)u + m.unit_len - 1) / m.unit_len : 0;
                hi = min(hi, units * m.unit_bytes);
            }
            moved[i] = off < hi;
            if (moved[i]) x[i] = *reinterpret_cast<const V *>(part + p * m.row_stride + off);
        }
#pragma unroll
        for (int i = 0; i < NB; ++i)
            if (moved[i]) *reinterpret_cast<V *>(part + i * m.row_stride + off) = x[i];
    }
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

__global__ void beam_next_kernel(BeamNextArgs a) {
    const int s = threadIdx.x;
    if (s >= a.n_seq) return;
    const int p = a.pos[16 * s] + 1;
    if (p >= 0 && p < a.cap) a.out[size_t(s) * a.cap + p] = a.tok[16 * s];
    a.pos[16 * s] = p;
}

// Logits a thread of the first kernel takes: 32, or 8 where that gives too few workgroups to read at the memory's rate.
int beam_per(int rows, int n_vocab) { return (long long)rows * ((n_vocab + 8191) / 8192) >= 512 ? 32 : 8; }
// (a chunk's first piece may start up to 3 elements before it, so 256 * per elements and 3 more are read by a workgroup)
int beam_chunks(int n_vocab, int per) { return (n_vocab + 256 * per - 1) / (256 * per); }

}  // namespace

size_t beam_work(int n_group, int n_beam, int n_vocab) {
    const long long rows = (long long)n_group * n_beam;
    const int per = beam_per(int(rows), n_vocab);
    return size_t(rows) * beam_chunks(n_vocab, per) * (sizeof(BeamStat) + 8 * size_t(n_beam));
}

hipError_t launch_beam_select(const BeamSelectArgs & args, hipStream_t s) {
    BeamSelectArgs a = args;
    const int rows = a.n_group * a.n_beam;
    a.per = beam_per(rows, a.n_vocab);
    a.chunks = beam_chunks(a.n_vocab, a.per);
    const unsigned lds = unsigned((a.n_beam + BEAM_SLACK) * a.per * 4 * sizeof(unsigned long long));
    const dim3 grid(unsigned(a.chunks), unsigned(rows));
    if (a.per == 32) GQ_LAUNCH(beam_scan_kernel<32>, grid, dim3(256), lds, s, a);
    else GQ_LAUNCH(beam_scan_kernel<8>, grid, dim3(256), lds, s, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (a.n_beam * a.chunks <= 1024) GQ_LAUNCH(beam_pick_kernel<256>, dim3(unsigned(a.n_group)), dim3(256), 0, s, a);
    else GQ_LAUNCH(beam_pick_kernel<1024>, dim3(unsigned(a.n_group)), dim3(1024), 0, s, a);
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
