// The allocation-free batched GEMV (gemvq_gemm_static in include/gemvq_hip.h): the GEMM command's two kernels on
// caller-owned device buffers. The quantized activation rows, which the GEMM command stages in its context's
// buffers, are staged here in `scratch`, a fixed device array of this file (one copy per device, held until the
// process ends). Nothing here allocates: the array's address on a device is looked up once, on the first call on
// that device, and kept.
// The 4-bit KV cache (gemvq_kv4_*_static) and the beam search's step (gemvq_beam_*_static) on caller-owned memory: their arguments'
// checks and launches. So for rotary positions (gemvq_rope_*) and the verification of drafted tokens (gemvq_draft_*).
#include "gemvq_hip.h"
#include "gq_beam.h"
#include "gq_draft.h"
#include "gq_kernels.h"
#include "gq_kv4.h"
#include "gq_rope.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <mutex>

using namespace gq;

namespace {

constexpr size_t Q_BYTES = size_t(GEMM_MAX_TOK) * GEMV_MAXK;          // quants of up to 32 token rows
constexpr size_t BLOCKS = size_t(GEMM_MAX_TOK) * (GEMV_MAXK / 32);    // their per-block scale words
constexpr size_t SCRATCH_BYTES = GEMVQ_STATIC_SCRATCH_BYTES;          // 640 KiB
static_assert(Q_BYTES + 2 * BLOCKS * sizeof(uint16_t) + BLOCKS / 16 * sizeof(float) <= SCRATCH_BYTES, "scratch size in the header");

__device__ __align__(256) uint8_t scratch[SCRATCH_BYTES];

constexpr int MAX_DEVICES = 64;
std::mutex g_mutex;
uint8_t * g_scratch[MAX_DEVICES];  // scratch's device address on each device (the host-side name is not one)

// The address of `scratch` on the current device, looked up on the first call there.
int scratch_on(int dev, uint8_t ** out) {
    std::lock_guard<std::mutex> lock(g_mutex);
    if (!g_scratch[dev]) {
        void * p = nullptr;
        const hipError_t e = hipGetSymbolAddress(&p, HIP_SYMBOL(scratch));
        if (e != hipSuccess) return -int(e);
        g_scratch[dev] = static_cast<uint8_t *>(p);
    }
    *out = g_scratch[dev];
    return 0;
}

bool aligned(const void * p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// Rows of floats that the kernels read and write in 16-byte pieces.
bool rows_ok(const void * p, int64_t stride, int64_t least) {
    return p && aligned(p, 16) && stride % 4 == 0 && stride >= least && stride <= (int64_t(1) << 40);
}

constexpr int GRID_MAX = 65535;

// Bytes of a cache; 0: sizes that are not served (2^46 bytes and more among them, whose offsets would pass 64 bits).
uint64_t kv4_bytes(int n_seq, int n_ctx, int n_head_kv, int head_dim) {
    if (n_seq < 1 || n_seq > GRID_MAX || n_ctx < 1 || n_head_kv < 1 || n_head_kv > GRID_MAX || !kv4_dim_ok(head_dim)) return 0;
    const uint64_t records = uint64_t(n_seq) * uint64_t(n_head_kv) * uint64_t(kv4_tiles(n_ctx));
    return records < (uint64_t(1) << 46) / kv4_record(head_dim) ? records * kv4_record(head_dim) : 0;
}
bool kv4_sizes_ok(const gemvq_kv4 * c) { return c && kv4_bytes(c->n_seq, c->n_ctx, c->n_head_kv, c->head_dim); }
// Query rows of a sequence: their workgroups fit a grid.
bool kv4_heads_ok(const gemvq_kv4 * c, int n_tok, int n_head) {
    return n_tok >= 1 && n_tok <= GEMVQ_KV4_MAX_TOK && n_head >= 1 && n_head <= GRID_MAX && n_head % c->n_head_kv == 0 &&
           int64_t(n_tok) * n_head <= GEMVQ_KV4_MAX_ROWS;
}
bool kv4_ok(const gemvq_kv4 * c) { return kv4_sizes_ok(c) && c->data && aligned(c->data, 256); }

Kv4Cache kv4_cache(const gemvq_kv4 * c) {
    const long long tiles = kv4_tiles(c->n_ctx);
    return {static_cast<uint8_t *>(c->data), c->n_ctx, c->n_head_kv, c->head_dim, tiles * c->n_head_kv, tiles};
}

bool kv4_tokens(const gemvq_kv4 * c, int n_tok, const int32_t * pos, const int32_t * num, Kv4Tokens & t) {
    if (n_tok < 1 || n_tok > GEMVQ_KV4_MAX_TOK || !pos || !aligned(pos, 4) || !aligned(num, 4)) return false;
    t = {pos, num, 1, n_tok, c->n_seq};
    return true;
}

int kv4_rows(const gemvq_kv4 * c, const float * k, const float * v, int64_t row_stride, int n_tok, const int32_t * pos,
             const int32_t * num, Kv4RowsArgs & a) {
    if (!kv4_ok(c) || !kv4_tokens(c, n_tok, pos, num, a.t)) return GEMVQ_EINVAL;
    const int64_t least = int64_t(c->n_head_kv) * c->head_dim;
    if (!rows_ok(k, row_stride, least) || !rows_ok(v, row_stride, least)) return GEMVQ_EINVAL;
    a.c = kv4_cache(c);
    a.k = const_cast<float *>(k);
    a.v = const_cast<float *>(v);
    a.row_stride = row_stride;
    return 0;
}

}  // namespace

extern "C" int gemvq_gemm_static(int type, int rows, int cols, const void * w, const float * x, int n_tok, int x_stride,
                                 float * y, int y_stride, void * stream) {
    if (type != T_Q4_0 && type != T_Q4_1 && type != T_Q8_0) return GEMVQ_EINVAL;
    if (rows < 1 || cols < 512 || cols % 512 || cols > int(GEMVQ_MAX_COLS)) return GEMVQ_EINVAL;
    if (n_tok < 1 || n_tok > int(GEMVQ_GEMM_MAX_TOK)) return GEMVQ_EINVAL;  // the scratch holds 32 token rows
    if (x_stride < cols || x_stride % 16 || y_stride < rows || y_stride % 16) return GEMVQ_EINVAL;
    if (!w || !x || !y || !aligned(w, 256) || !aligned(x, 64) || !aligned(y, 64)) return GEMVQ_EINVAL;
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return -int(e);
    if (dev < 0 || dev >= MAX_DEVICES) return GEMVQ_EINVAL;
    uint8_t * base = nullptr;
    const int st = scratch_on(dev, &base);
    if (st) return st;
    GemmQuantArgs q{};
    q.x = x;
    q.norm_w = nullptr;
    q.q = reinterpret_cast<int8_t *>(base);
    q.d = reinterpret_cast<uint16_t *>(base + Q_BYTES);
    q.s = q.d + BLOCKS;
    q.bound = reinterpret_cast<float *>(q.s + BLOCKS);
    q.n_tok = n_tok;
    q.n_pad = (n_tok + 15) / 16 * 16;  // the quantizer writes the padding rows too: nothing needs clearing
    q.cols = cols;
    q.x_stride = x_stride;
    GemmArgs g{};
    g.w = weight_view(static_cast<const uint8_t *>(w), type, rows, cols);
    g.q = q.q;
    g.d = q.d;
    g.s = q.s;
    g.bound = q.bound;
    g.y = y;
    g.rows = rows;
    g.cols = cols;
    g.n_tok = n_tok;
    g.y_stride = y_stride;
    g.epi = EPI_PLAIN;
    g.wbound[0] = INFINITY;  // the caller's matrix was never scanned: each step's bound is formed from its scales
    const hipStream_t s = static_cast<hipStream_t>(stream);
    e = launch_gemm_quant(q, s);
    if (e == hipSuccess) e = launch_gemm(g, type, s);
    return e == hipSuccess ? 0 : -int(e);
}

extern "C" {

uint64_t gemvq_kv4_bytes(int n_seq, int n_ctx, int n_head_kv, int head_dim) { return kv4_bytes(n_seq, n_ctx, n_head_kv, head_dim); }

int gemvq_kv4_store_static(const gemvq_kv4 * kv, const float * k, const float * v, int64_t row_stride, int n_tok,
                           const int32_t * pos, const int32_t * num, void * stream) {
    Kv4RowsArgs a;
    const int st = kv4_rows(kv, k, v, row_stride, n_tok, pos, num, a);
    if (st) return st;
    const hipError_t e = launch_kv4_store(a, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? 0 : -int(e);
}

int gemvq_kv4_load_static(const gemvq_kv4 * kv, float * k, float * v, int64_t row_stride, int n_tok, const int32_t * pos,
                          const int32_t * num, void * stream) {
    Kv4RowsArgs a;
    const int st = kv4_rows(kv, k, v, row_stride, n_tok, pos, num, a);
    if (st) return st;
    const hipError_t e = launch_kv4_load(a, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? 0 : -int(e);
}

uint64_t gemvq_kv4_attn_work(const gemvq_kv4 * kv, int n_tok, int n_head) {
    if (!kv4_sizes_ok(kv) || !kv4_heads_ok(kv, n_tok, n_head)) return 0;
    return kv4_work_floats(kv4_cache(kv), kv->n_seq, n_tok, n_head) * sizeof(float);
}

int gemvq_kv4_attn_static(const gemvq_kv4 * kv, const float * q, int64_t q_stride, int64_t q_head_stride, float * y,
                          int64_t y_stride, int n_tok, int n_head, const int32_t * pos, const int32_t * num, int window,
                          float scale, void * work, uint64_t work_bytes, void * stream) {
    Kv4AttnArgs a{};
    if (!kv4_ok(kv) || !kv4_tokens(kv, n_tok, pos, num, a.t)) return GEMVQ_EINVAL;
    if (!kv4_heads_ok(kv, n_tok, n_head) || window < 0) return GEMVQ_EINVAL;
    const uint64_t need = gemvq_kv4_attn_work(kv, n_tok, n_head);
    if (work_bytes < need || (need && (!work || !aligned(work, 16)))) return GEMVQ_EINVAL;
    const int64_t hd = kv->head_dim;
    if (!rows_ok(q, q_stride, hd) || q_head_stride % 4 || q_head_stride < hd || q_head_stride > (int64_t(1) << 40) ||
        !rows_ok(y, y_stride, n_head * hd))
        return GEMVQ_EINVAL;
    a.c = kv4_cache(kv);
    a.q = q;
    a.y = y;
    a.q_row = q_stride;
    a.q_head = q_head_stride;
    a.y_row = y_stride;
    a.n_head = n_head;
    a.window = window;
    a.scale = scale;
    a.work = need ? static_cast<float *>(work) : nullptr;
    const hipError_t e = launch_kv4_attn(a, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? 0 : -int(e);
}

}  // extern "C"

namespace {

// Sizes of a call with parts: rows and workgroups fit one-dimensional grids.
bool kv4_parts_ok(const gemvq_kv4 * kv, const gemvq_kv4 * prefix, int n_tok, int n_head) {
    if (!kv4_sizes_ok(kv) || !kv4_heads_ok(kv, n_tok, n_head) || int64_t(kv->n_seq) * n_tok * n_head > GEMVQ_KV4_MAX_PART_ROWS) return false;
    if (prefix && (!kv4_sizes_ok(prefix) || prefix->n_head_kv != kv->n_head_kv || prefix->head_dim != kv->head_dim || kv->n_seq % prefix->n_seq)) return false;
    return kv4_parts_grid(kv4_cache(kv), prefix ? prefix->n_seq : 0, prefix ? prefix->n_ctx : 0, kv->n_seq, n_tok, n_head) < (1 << 24);  // below 2^32 threads
}
// At least 16 bytes (0 says that sizes are not served).
uint64_t kv4_parts_work(const gemvq_kv4 * kv, const gemvq_kv4 * prefix, int n_tok, int n_head) {
    return std::max<uint64_t>(16, kv4_parts_floats(kv4_cache(kv), prefix ? prefix->n_seq : 0, prefix ? prefix->n_ctx : 0, kv->n_seq, n_tok, n_head) * sizeof(float));
}

int kv4_parts(const gemvq_kv4 * kv, const gemvq_kv4 * prefix, const int32_t * prefix_len, const float * q, int64_t q_stride,
              int64_t q_head_stride, float * y, int64_t y_stride, int n_tok, int n_head, const int32_t * pos, const int32_t * num,
              int window, int sinks, float scale, void * work, uint64_t work_bytes, void * stream) {
    Kv4PartsArgs x{};
    if (!kv4_ok(kv) || !kv4_tokens(kv, n_tok, pos, num, x.a.t) || !kv4_parts_ok(kv, prefix, n_tok, n_head) || window < 0 || sinks < 0) return GEMVQ_EINVAL;
    if (prefix && (!kv4_ok(prefix) || !prefix_len || !aligned(prefix_len, 4))) return GEMVQ_EINVAL;
    const bool none = kv4_parts_whole(kv4_cache(kv), prefix ? prefix->n_seq : 0, prefix ? prefix->n_ctx : 0, kv->n_seq, n_tok, n_head);
    const uint64_t need = none ? 0 : kv4_parts_work(kv, prefix, n_tok, n_head);
    if (work_bytes < need || (need && (!work || !aligned(work, 16)))) return GEMVQ_EINVAL;
    const int64_t hd = kv->head_dim;
    if (!rows_ok(q, q_stride, hd) || q_head_stride % 4 || q_head_stride < hd || q_head_stride > (int64_t(1) << 40) ||
        !rows_ok(y, y_stride, n_head * hd))
        return GEMVQ_EINVAL;
    x.a.c = kv4_cache(kv);
    x.a.q = q;
    x.a.y = y;
    x.a.q_row = q_stride;
    x.a.q_head = q_head_stride;
    x.a.y_row = y_stride;
    x.a.n_head = n_head;
    x.a.window = window;
    x.a.scale = scale;
    x.a.work = need ? static_cast<float *>(work) : nullptr;
    if (prefix) x.pre = kv4_cache(prefix);
    x.pre_len = prefix_len;
    x.members = prefix ? kv->n_seq / prefix->n_seq : 1;
    x.sinks = sinks;
    const hipError_t e = launch_kv4_parts(x, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? 0 : -int(e);
}

}  // namespace

extern "C" {

uint64_t gemvq_kv4_attn_sink_work(const gemvq_kv4 * kv, int n_tok, int n_head) {
    return kv4_parts_ok(kv, nullptr, n_tok, n_head) ? kv4_parts_work(kv, nullptr, n_tok, n_head) : 0;
}

int gemvq_kv4_attn_sink_static(const gemvq_kv4 * kv, const float * q, int64_t q_stride, int64_t q_head_stride, float * y,
                               int64_t y_stride, int n_tok, int n_head, const int32_t * pos, const int32_t * num, int window,
                               int sinks, float scale, void * work, uint64_t work_bytes, void * stream) {
    return kv4_parts(kv, nullptr, nullptr, q, q_stride, q_head_stride, y, y_stride, n_tok, n_head, pos, num, window, sinks, scale, work, work_bytes, stream);
}

uint64_t gemvq_kv4_attn_shared_work(const gemvq_kv4 * kv, const gemvq_kv4 * prefix, int n_tok, int n_head) {
    return prefix && kv4_parts_ok(kv, prefix, n_tok, n_head) ? kv4_parts_work(kv, prefix, n_tok, n_head) : 0;
}

int gemvq_kv4_attn_shared_static(const gemvq_kv4 * kv, const gemvq_kv4 * prefix, const int32_t * prefix_len, const float * q,
                                 int64_t q_stride, int64_t q_head_stride, float * y, int64_t y_stride, int n_tok, int n_head,
                                 const int32_t * pos, const int32_t * num, int window, int sinks, float scale, void * work,
                                 uint64_t work_bytes, void * stream) {
    if (!prefix) return GEMVQ_EINVAL;
    return kv4_parts(kv, prefix, prefix_len, q, q_stride, q_head_stride, y, y_stride, n_tok, n_head, pos, num, window, sinks, scale, work, work_bytes, stream);
}

}  // extern "C"

static_assert(GEMVQ_BEAM_MAX == BEAM_MAX && GEMVQ_BEAM_MAX_VOCAB == BEAM_MAX_VOCAB, "limits in the header");

namespace {
bool beam_rows_ok(int n_group, int n_beam) {
    return n_beam >= 1 && n_beam <= BEAM_MAX && n_group >= 1 && int64_t(n_group) * n_beam <= GRID_MAX;
}
}  // namespace

extern "C" {

uint64_t gemvq_beam_work(int n_group, int n_beam, int n_vocab) {
    if (!beam_rows_ok(n_group, n_beam) || n_vocab < 1 || n_vocab > BEAM_MAX_VOCAB) return 0;
    return beam_work(n_group, n_beam, n_vocab);
}

int gemvq_beam_select_static(const float * logits, int64_t row_stride, int n_vocab, int n_group, int n_beam, const float * score,
                             const int32_t * last, int eos, float * score_out, int32_t * token, int32_t * parent, void * work,
                             uint64_t work_bytes, void * stream) {
    const uint64_t need = gemvq_beam_work(n_group, n_beam, n_vocab);
    if (!need || !logits || row_stride < n_vocab || row_stride > (int64_t(1) << 40) || !score || !score_out || !token || !parent ||
        !work || work_bytes < need)
        return GEMVQ_EINVAL;
    if (!aligned(logits, 4) || !aligned(score, 4) || !aligned(last, 4) || !aligned(score_out, 4) || !aligned(token, 4) ||
        !aligned(parent, 4) || !aligned(work, 16))
        return GEMVQ_EINVAL;
    BeamSelectArgs a{};
    a.x = logits;
    a.stride = row_stride;
    a.n_vocab = n_vocab;
    a.n_group = n_group;
    a.n_beam = n_beam;
    a.eos = eos;
    a.score = score;
    a.last = last;
    a.score_out = score_out;
    a.token = token;
    a.parent = parent;
    a.slot = 1;
    a.work = work;
    const hipError_t e = launch_beam_select(a, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? 0 : -int(e);
}

int gemvq_beam_reorder_static(const gemvq_beam_array * arrays, int n_arrays, const int32_t * parent, int n_group, int n_beam,
                              void * stream) {
    if (!arrays || n_arrays < 1 || !parent || !aligned(parent, 4) || !beam_rows_ok(n_group, n_beam)) return GEMVQ_EINVAL;
    const uint64_t rows = uint64_t(n_group) * uint64_t(n_beam), most = uint64_t(1) << 46;  // (sums below stay below 2^63)
    for (int i = 0; i < n_arrays; ++i) {
        const gemvq_beam_array & x = arrays[i];
        const uint64_t size = uint64_t(x.count) * x.unit_bytes;
        if (!x.data || !aligned(x.data, 4) || x.n_part < 1 || x.n_part > uint32_t(GRID_MAX) || x.first > x.count || x.unit_bytes < 4 ||
            x.unit_bytes % 4 || x.row_stride % 4 || x.part_stride % 4 || x.row_stride > most || x.part_stride > most || size > most)
            return GEMVQ_EINVAL;
        if (x.used && (!aligned(x.used, 4) || x.unit_len < 1 || x.used_stride < 1)) return GEMVQ_EINVAL;
        if (!beam_rows_apart(rows, size, x.row_stride, x.part_stride, x.n_part)) return GEMVQ_EINVAL;
        if (beam_move_groups(uint64_t(x.first) * x.unit_bytes, size, x.n_part) > BEAM_GRID) return GEMVQ_EINVAL;
    }
    for (int i = 0; i < n_arrays;) {
        BeamReorderArgs a{};
        a.parent = parent;
        a.n_group = n_group;
        a.n_beam = n_beam;
        a.parent_stride = 1;
        uint32_t end = 0;
        for (; i < n_arrays && a.n < BEAM_MOVES; ++i) {
            const gemvq_beam_array & x = arrays[i];
            if (x.first == x.count) continue;
            if (end + beam_move_groups(uint64_t(x.first) * x.unit_bytes, uint64_t(x.count) * x.unit_bytes, x.n_part) > BEAM_GRID) break;
            BeamMove & m = a.m[a.n++];
            m.data = static_cast<uint8_t *>(x.data);
            m.row_stride = x.row_stride;
            m.part_stride = x.part_stride;
            m.lo = uint64_t(x.first) * x.unit_bytes;
            m.hi = uint64_t(x.count) * x.unit_bytes;
            m.used = x.used;
            m.unit_bytes = x.unit_bytes;
            m.unit_len = x.unit_len;
            m.used_stride = x.used_stride;
            beam_move_shape(m, x.n_part, end);
        }
        if (!a.n) break;
        const hipError_t e = launch_beam_reorder(a, static_cast<hipStream_t>(stream));
        if (e != hipSuccess) return -int(e);
    }
    return 0;
}

}  // extern "C"

static_assert(GEMVQ_ROPE_MAX_ARRAYS == ROPE_ARRAYS && GEMVQ_ROPE_MAX_DIM == ROPE_MAX_DIM, "limits in the header");
static_assert(GEMVQ_DRAFT_MAX == DRAFT_MAX && GEMVQ_DRAFT_MAX_VOCAB == DRAFT_MAX_VOCAB, "limits in the header");

extern "C" {

int gemvq_rope_freqs(int n_rot, double base, double factor, int yarn_ctx, double beta_fast, double beta_slow, const double * factors,
                     double * freqs) {
    if (n_rot < 2 || n_rot % 2 || n_rot > ROPE_MAX_DIM || !freqs) return GEMVQ_EINVAL;
    if (!(base > 1) || !std::isfinite(base) || !(factor > 0) || !std::isfinite(factor) || yarn_ctx < 0) return GEMVQ_EINVAL;
    if (yarn_ctx && !(beta_slow > 0 && beta_fast >= beta_slow && std::isfinite(beta_fast))) return GEMVQ_EINVAL;
    for (int i = 0; factors && i < n_rot / 2; ++i)
        if (!(factors[i] > 0) || !std::isfinite(factors[i])) return GEMVQ_EINVAL;
    double table[ROPE_MAX_DIM / 2 + 1];
    rope_table(n_rot, base, factor, yarn_ctx, beta_fast, beta_slow, factors, table);
    for (int i = 0; i <= n_rot / 2; ++i)
        if (!std::isfinite(table[i])) return GEMVQ_EINVAL;  // divisors next to 0
    std::copy(table, table + n_rot / 2 + 1, freqs);
    return 0;
}

int gemvq_rope_static(const gemvq_rope_rows * arrays, int n_arrays, int n_seq, int n_tok, int head_dim, int n_rot, int layout,
                      const double * freqs, const int32_t * pos, const int32_t * num, void * stream) {
    if (!arrays || n_arrays < 1 || n_arrays > ROPE_ARRAYS || n_seq < 1 || n_tok < 1 || int64_t(n_seq) * n_tok >= GEMVQ_ROPE_MAX_ROWS)
        return GEMVQ_EINVAL;
    if (head_dim < 4 || head_dim % 4 || head_dim > ROPE_MAX_DIM || n_rot < 2 || n_rot % 2 || n_rot > head_dim) return GEMVQ_EINVAL;
    if ((layout != GEMVQ_ROPE_HALF && layout != GEMVQ_ROPE_PAIRS) || !freqs || !aligned(freqs, 8) || !pos || !aligned(pos, 4) || !aligned(num, 4))
        return GEMVQ_EINVAL;
    RotaryArgs a{};
    int64_t heads = 0;
    for (int i = 0; i < n_arrays; ++i) {
        const gemvq_rope_rows & r = arrays[i];
        if (r.n_head < 1 || r.n_head > GRID_MAX || (heads += r.n_head) > GRID_MAX) return GEMVQ_EINVAL;
        if (!rows_ok(r.x, r.x_row, head_dim) || !rows_ok(r.y, r.y_row, head_dim) || !rows_ok(r.x, r.x_head, head_dim) || !rows_ok(r.y, r.y_head, head_dim))
            return GEMVQ_EINVAL;
        if (r.x == r.y && (r.x_row != r.y_row || r.x_head != r.y_head)) return GEMVQ_EINVAL;
        for (int j = 0; j < i; ++j)  // one array's first head is written while another's is read or written
            if (r.y == arrays[j].y || r.y == arrays[j].x || r.x == arrays[j].y) return GEMVQ_EINVAL;
        a.a[i] = {r.x, r.y, r.x_row, r.x_head, r.y_row, r.y_head, r.n_head, 0};
    }
    a.freqs = freqs;
    a.pos = pos;
    a.num = num;
    a.n = n_arrays;
    a.n_seq = n_seq;
    a.n_tok = n_tok;
    a.head_dim = head_dim;
    a.n_rot = n_rot;
    a.pairs = layout == GEMVQ_ROPE_PAIRS;
    const hipError_t e = launch_rotary(a, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? 0 : -int(e);
}

// Differences of logits over it, and its reciprocal, are 64-bit numbers.
static bool draft_temperature_ok(double t) { return t >= 1e-30 && t <= 1e30; }

uint64_t gemvq_draft_work(int n_seq, int n_draft, int n_vocab) {
    if (n_seq < 1 || n_draft < 0 || n_draft > DRAFT_MAX || int64_t(n_seq) * (2 * n_draft + 1) > GRID_MAX || n_vocab < 1 || n_vocab > DRAFT_MAX_VOCAB)
        return 0;
    return draft_work(n_seq, n_draft, n_vocab);
}

int gemvq_draft_verify_static(const float * target, int64_t target_stride, const float * draft, int64_t draft_stride, int n_vocab,
                              int n_seq, int n_draft, const int32_t * token, const int32_t * num, const float * uniform,
                              double temperature, double draft_temperature, int32_t * n_accept, int32_t * out, float * logp, void * work,
                              uint64_t work_bytes, void * stream) {
    const uint64_t need = gemvq_draft_work(n_seq, n_draft, n_vocab);
    const int64_t most = int64_t(1) << 40;
    if (!need || !target || target_stride < n_vocab || target_stride > most || !n_accept || !out || !work || work_bytes < need) return GEMVQ_EINVAL;
    if (draft && (draft_stride < n_vocab || draft_stride > most)) return GEMVQ_EINVAL;
    if ((n_draft && !token) || (temperature != 0.0 && (!draft_temperature_ok(temperature) || !uniform))) return GEMVQ_EINVAL;
    if (temperature != 0.0 && draft && !draft_temperature_ok(draft_temperature)) return GEMVQ_EINVAL;
    if (!aligned(target, 4) || !aligned(draft, 4) || !aligned(token, 4) || !aligned(num, 4) || !aligned(uniform, 4) || !aligned(n_accept, 4) ||
        !aligned(out, 4) || !aligned(logp, 4) || !aligned(work, 16))
        return GEMVQ_EINVAL;
    DraftArgs a{};
    a.target = target;
    a.draft = n_draft ? draft : nullptr;
    a.target_stride = target_stride;
    a.draft_stride = draft_stride;
    a.token = token;
    a.num = num;
    a.uniform = uniform;
    a.n_accept = n_accept;
    a.out = out;
    a.logp = logp;
    a.greedy = temperature == 0.0;
    a.scale = draft_scale(a.greedy ? 1.0 : temperature);
    a.draft_scale = draft_scale(a.greedy || !draft ? 1.0 : draft_temperature);
    a.n_vocab = n_vocab;
    a.n_seq = n_seq;
    a.n_draft = n_draft;
    a.work = work;
    const hipError_t e = launch_draft(a, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? 0 : -int(e);
}

}  // extern "C"
