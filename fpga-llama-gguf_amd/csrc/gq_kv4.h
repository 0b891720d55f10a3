// The 4-bit KV cache (Q4_0 blocks of 32 elements along head_dim): its layout, and the launch descriptors of the kernels on it.
//
// A block x[0..31]: m = its element of largest magnitude (the first of them), d = m / -8, q = min(15, int(x / d + 8.5)) with
// x / d formed as x * (1 / d), all in FP32 (ggml's Q4_0); it holds fp16(d) and the sixteen values, and stands for fp16(d) * (q - 8).
//
// Per sequence and KV head the cache is a row of records of 32 positions each, NB = head_dim / 32 blocks a position:
//   Kq  16 head_dim bytes  [sub 2][c][g 4][p 16][b][e 4]: byte of block 4 c + b (b < min(NB, 4)) at position 16 sub + p; low nibble
//                          element 32 block + 4 g + e, high nibble the one 16 further (the two halves of a byte as in ggml)
//   Vq  16 head_dim bytes  [c][g 4][n 16][b][sub 2][r 4]: byte of block 2 c + b (b < min(NB, 2)) at position 16 sub + 4 g + r; low
//                          nibble element 32 block + n, high nibble the one 16 further
//   Kd, Vd  2 head_dim bytes each  [g 4][block][sub 2][r 4]: fp16 scale of position 16 sub + 4 g + r
// The order is that of the matrix instructions' operands (16x16x32): lane 16 g + p of a wave finds the key bytes of its position, and
// lane 16 g + n the value bytes of its element at 8 positions, as consecutive 16-byte pieces, whole 1 KB lines a load. Every byte
// belongs to one position, so a position is written without reading its neighbours.
#pragma once
#include "gq_kernels.h"

namespace gq {

constexpr int KV4_TILE = 32;  // positions of a record

__host__ __device__ constexpr bool kv4_dim_ok(int hd) { return hd == 32 || hd == 64 || hd == 128 || hd == 256; }
__host__ __device__ constexpr size_t kv4_record(int hd) { return size_t(36) * hd; }
__host__ __device__ constexpr int kv4_tiles(int n_ctx) { return (n_ctx - 1) / KV4_TILE + 1; }

// Offsets in a record of position p (0..31): the key byte of element e < 16 of block blk (its high nibble: element e + 16),
// the value byte likewise, and the scale of the block (bytes from the start of Kd or Vd).
template <int HD>
struct Kv4Layout {
    static constexpr int NB = HD / 32, KB = NB < 4 ? NB : 4, VB = NB < 2 ? NB : 2;
    static constexpr int VQ = 16 * HD, KD = 32 * HD, VD = 34 * HD, RECORD = 36 * HD;
    __host__ __device__ static int kq(int p, int blk, int e) {
        return (p >> 4) * 8 * HD + (blk / KB) * 256 * KB + ((e >> 2) * 16 + (p & 15)) * 4 * KB + (blk % KB) * 4 + (e & 3);
    }
    __host__ __device__ static int vq(int p, int blk, int e) {
        return VQ + (blk / VB) * 512 * VB + (((p & 15) >> 2) * 16 + e) * 8 * VB + (blk % VB) * 8 + (p >> 4) * 4 + (p & 3);
    }
    __host__ __device__ static int scale(int p, int blk) { return ((((p & 15) >> 2) * NB + blk) * 8 + (p >> 4) * 4 + (p & 3)) * 2; }
};

// Tokens t < num[s] (num NULL: n_tok) of sequence s are at positions pos[s * pos_stride] + t; the ones outside 0 .. n_ctx - 1 are
// not touched.
struct Kv4Tokens {
    const int32_t * pos;
    const int32_t * num;
    int pos_stride, n_tok, n_seq;
};

struct Kv4Cache {  // the records of sequence s and KV head h start at record s * seq + h * head
    uint8_t * data;
    int n_ctx, n_head_kv, head_dim;  // n_ctx: positions of a sequence
    long long seq, head;
};

struct Kv4RowsArgs {  // store or load: row (s * n_tok + t) of k and v at row_stride floats, KV heads packed
    Kv4Cache c;
    Kv4Tokens t;
    float * k;
    float * v;
    long long row_stride;
};

struct Kv4AttnArgs {
    Kv4Cache c;
    Kv4Tokens t;
    const float * q;  // row (s * n_tok + t) at q_row floats, head h at q_head floats
    float * y;        // row (s * n_tok + t) at y_row floats, heads packed
    long long q_row, q_head, y_row;
    int n_head, window;  // window 0: every position up to the token's own
    float scale;
    const float * gate;  // NULL, or gate rows (the output times sigmoid(gate)), g_row and g_head floats apart
    long long g_row, g_head;
    float * work;        // kv4_work_floats; NULL: one range a sequence
    int ranges;          // set at launch: ranges of records that the grid has workgroups for
    int group;           // set at launch: n_head / n_head_kv
};

// Times of these rules, here and in gq_kv4.hip: a call alone (attention and joining; storing and reading back) replayed in a graph.
// Workgroups of the attention a CU holds at once (nq groups of 16 query rows each): three where the registers can be kept to that (32
// ragged sequences of up to 8192, 32/8 heads of 128: 46 us, 50 with two). A call's records are dealt to as many as the device holds, each
// with its share: twice as many, each with half of it, are 25.1 us in place of 20.1 (4 sequences of 8192, 32/8 heads of 128), 32.5 and
// 27.6 (8 of 5 tokens at 8000, 32/8 heads of 64), 37.0 and 29.3 (8 of 8 tokens at 8184, 16/4 heads of 128); 23.5 and 18.4 (one of 32768,
// 16/4 heads of 256).
__host__ __device__ constexpr int kv4_resident(int hd, int nq) { return hd * nq <= 128 ? 3 : 2; }
constexpr int KV4_GROUPS = 768;   // at most
constexpr int KV4_LEAST = 4;      // records of a range at least: one a wave
// Records times head_dim up to which a cache's sequences are not split, which needs no second launch: its waves' few records more take
// less than joining. Half as many where the cache is longer, but no sequence in it (us whole, whole with the second launch, and split:
// one sequence of 320, 16/4 heads of 256, 10.2 / 11.5 / 10.3, of 640 13.5 / 15.0 / 10.4; 4 of 1500 26.0 / 27.9 / 14.8; 32 of 256, 32/8
// heads of 128, in caches of 8192, 7.7 / 10.2 / 12.8; 7 of 5 tokens in a window of 1000, 8 heads of 64, 10.5 / 12.8 / 11.1).
constexpr int KV4_ALONE = 2048;
bool kv4_joins(const Kv4AttnArgs & a);  // the launch is followed by that of kv4_join_kernel
size_t kv4_work_floats(const Kv4Cache & c, int n_seq, int n_tok, int n_head);

// The ATTN command's part before the attention: every q head and new key normalized and rotated (gq_kernels.h, AttnArgs; q stays FP32
// in qr), the keys and values stored. Tokens as t says.
struct Kv4AppendArgs {
    Kv4Cache c;
    Kv4Tokens t;
    const float * q;   // row (s * n_tok + t) at n_head * q_stride floats
    const float * k;   // rows of n_head_kv * head_dim floats
    const float * v;
    const float * qn;
    const float * kn;
    const float * cs;  // n_rot floats a position
    float * qr;        // rows of n_head * head_dim floats
    int n_head, n_rot, q_stride;
    float eps;
};

hipError_t launch_kv4_append(const Kv4AppendArgs & a, hipStream_t s);
hipError_t launch_kv4_store(const Kv4RowsArgs & a, hipStream_t s);
hipError_t launch_kv4_load(const Kv4RowsArgs & a, hipStream_t s);
hipError_t launch_kv4_attn(const Kv4AttnArgs & a, hipStream_t s);

}  // namespace gq
