// Layout of the paged key/value cache (include/litenn_kv.h) and what its kernels share: where a value lies, the sequences of
// a call, checked page numbers.
//
// A tile holds 16 tokens of one kv head: key quants, key scales, value quants, value scales.  The quant planes are in the order
// in which the attention kernels' MMA operands want them, so that a lane reads its share of a tile as whole vectors without
// shuffles, and a tile is one run of bytes that one bulk copy brings in:
//   keys    A operand of K . q^T (mma m16n8k16, row = token): lane 4g + t holds, for tokens g and g + 8 (half j = 0, 1), the eight
//           dimensions 32b + 8t + {0..7} of every block b.  A block is two k16 steps, so its scale meets the sum of exactly those.
//   values  A operand of V^T . P^T (row = dimension, k = token): lane 4g + t holds, for tokens 8j + 2t and 8j + 2t + 1, the four
//           dimensions 32b + 4g + {0..3} of every block, the two tokens' values of a dimension in one 32-bit operand register.
// The prompt kernel stores the same registers as 8 x 8 matrices.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "qmm_common.cuh"

namespace qmm {

constexpr int KV_F16 = 0;
constexpr int KV_TILE = 16;  // tokens per tile

__host__ __device__ constexpr int kv_unit(int fmt)
{
    return fmt == FMT_Q4_0 ? 4 : fmt == FMT_Q8_0 ? 8 : 16;  // bytes of eight values
}
__host__ __device__ constexpr int kv_lane_bytes(int fmt, int hd)
{
    return hd / 32 * kv_unit(fmt);  // of one lane and eight tokens
}
__host__ __device__ constexpr int kv_vec(int fmt, int hd)
{
    return kv_lane_bytes(fmt, hd) % 16 == 0 ? 16 : kv_lane_bytes(fmt, hd) % 8 == 0 ? 8 : 4;
}
__host__ __device__ constexpr int kv_plane_bytes(int fmt, int hd)
{
    return 64 * kv_lane_bytes(fmt, hd);
}
__host__ __device__ constexpr int kv_scale_bytes(int fmt, int hd)
{
    return fmt == KV_F16 ? 0 : hd;  // 16 tokens x hd / 32 blocks x 2 bytes
}
__host__ __device__ constexpr int kv_tile_bytes(int fmt, int hd)
{
    return 2 * (kv_plane_bytes(fmt, hd) + kv_scale_bytes(fmt, hd));
}
// Byte of a quant plane: half j, lane p, byte x of block b.
__host__ __device__ constexpr int kv_place(int fmt, int hd, int j, int p, int b, int x)
{
    const int at = b * kv_unit(fmt) + x, vec = kv_vec(fmt, hd);
    return j * 32 * kv_lane_bytes(fmt, hd) + at / vec * 32 * vec + p * vec + at % vec;
}
// Byte of a scale plane: token of the tile, block b.
__host__ __device__ constexpr int kv_scale_place(int hd, int token, int b)
{
    return ((((token >> 1) & 3) * 2 + (token >> 3)) * (hd / 32) + b) * 4 + (token & 1) * 2;
}

// Status codes (qmm_kernel_status).
constexpr int KV_BAD_PAGE = 21, KV_BAD_ROWS = 22, KV_LATE_COPY = 23;

struct KvPool {
    uint8_t* base;
    int fmt, kv_heads, head_dim, page_tokens;
    int64_t n_pages;
};
struct KvSeqs {
    int batch, table_width;
    const int* table;
    const int* kv_len;
    const int* row_begin;  // null: one row per sequence
    int64_t rows;
    int* status;
};

// Rows and length of sequence s, checked: n = 0 where they cannot be right.  `bad` tells so.
struct KvSeq {
    int64_t row0;
    int n, len;
};
__host__ __device__ __forceinline__ KvSeq kv_seq(const KvPool& c, const KvSeqs& b, int s, bool& bad)
{
    KvSeq q;
    const int64_t b0 = b.row_begin ? b.row_begin[s] : s, b1 = b.row_begin ? b.row_begin[s + 1] : s + 1;
    const int len = b.kv_len[s];
    bad = b0 < 0 || b1 < b0 || b1 > b.rows || len < 0 || len > (int64_t)b.table_width * c.page_tokens;
    q.row0 = b0;
    q.n = bad ? 0 : (int)(b1 - b0);
    q.len = bad ? 0 : len;
    return q;
}
// Page of a token of sequence s (pos below its checked length), -1 where the table names none of the pool's.
__host__ __device__ __forceinline__ int kv_page(const KvPool& c, const KvSeqs& b, int s, int pos)
{
    const int page = b.table[(int64_t)s * b.table_width + pos / c.page_tokens];
    return page >= 0 && page < c.n_pages ? page : -1;
}
__host__ __device__ __forceinline__ int64_t kv_tile_index(const KvPool& c, int page, int head, int pos)
{
    return ((int64_t)page * c.kv_heads + head) * (c.page_tokens / KV_TILE) + pos % c.page_tokens / KV_TILE;
}

}  // namespace qmm
