// The allocation-free batched GEMV (gemvq_gemm_static in include/gemvq_hip.h): the GEMM command's two kernels on
// caller-owned device buffers. The quantized activation rows, which the GEMM command stages in its context's
// buffers, are staged here in `scratch`, a fixed device array of this file (one copy per device, held until the
// process ends). Nothing here allocates: the array's address on a device is looked up once, on the first call on
// that device, and kept.
// The 4-bit KV cache (gemvq_kv4_*_static) and the beam search's step (gemvq_beam_*_static) on caller-owned memory: their arguments'
// checks and launches.
#include "gemvq_hip.h"
#include "gq_beam.h"
#include "gq_kernels.h"
#include "gq_kv4.h"

#include <hip/hip_runtime.h>

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
