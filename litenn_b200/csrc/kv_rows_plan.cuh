// How kv_rows.cu cuts its work: one list of tiles over all (sequence, kv head, pass of eight columns), equal shares of it per CTA.
// Host code too, so that the tests walk it without a GPU.
#pragma once

#include "kv_layout.cuh"

namespace qmm {

constexpr int KV_COLS = 8;  // columns (query heads of a kv head, times rows) of a pass

__host__ __device__ __forceinline__ int kv_max(int a, int b)
{
    return a > b ? a : b;
}
__host__ __device__ __forceinline__ int kv_min(int a, int b)
{
    return a < b ? a : b;
}

// A sequence's part of the list: w = kv heads * passes * tiles entries.
struct SeqWork {
    KvSeq q;
    int tile0, tiles, passes;
    long long w;
};
__host__ __device__ __forceinline__ SeqWork seq_work(const KvPool& c, const KvSeqs& b, int group, int window, int s, bool& bad)
{
    SeqWork x;
    x.q = kv_seq(c, b, s, bad);
    // tiles from the first that the first row's window reaches to the last token's; a sequence without any still has its
    // rows' zeros to write
    const int first = x.q.len - x.q.n;
    const int low = window > 0 ? kv_max(0, first - window + 1) : 0;
    x.tile0 = low / KV_TILE;
    x.tiles = kv_max(1, (x.q.len + KV_TILE - 1) / KV_TILE - x.tile0);
    x.passes = (int)(((long long)x.q.n * group + KV_COLS - 1) / KV_COLS);
    x.w = (long long)c.kv_heads * x.passes * x.tiles;
    return x;
}

// What one pass of a sequence sees.
struct PassView {
    int col0, cols;
    int pos_lo, pos_hi;   // positions of the first and the last column's row
    int seen_lo, all_lo;  // some column sees seen_lo .. pos_hi, every column all_lo .. pos_lo
    int tile_begin, tile_end;  // of the given tiles, those that some column sees
};
__host__ __device__ __forceinline__ PassView pass_view(const SeqWork& x, int group, int window, int pass, int tile_begin,
                                                       int tile_end)
{
    PassView v;
    const long long columns = (long long)x.q.n * group;
    v.col0 = pass * KV_COLS;
    v.cols = columns - v.col0 < KV_COLS ? (int)(columns - v.col0) : KV_COLS;
    const int first = x.q.len - x.q.n;
    v.pos_lo = first + v.col0 / group;
    v.pos_hi = first + (v.col0 + v.cols - 1) / group;
    v.seen_lo = window > 0 ? kv_max(0, v.pos_lo - window + 1) : 0;
    v.all_lo = window > 0 ? kv_max(0, v.pos_hi - window + 1) : 0;
    v.tile_begin = kv_max(tile_begin, v.seen_lo / KV_TILE);
    v.tile_end = kv_min(tile_end, v.pos_hi < 0 ? 0 : v.pos_hi / KV_TILE + 1);
    return v;
}

// `ctas` equal shares of `total` list entries: where share i begins, and which share has an entry.
__host__ __device__ __forceinline__ long long share_begin(long long total, long long ctas, long long i)
{
    return total * i / ctas;
}
__host__ __device__ __forceinline__ long long share_of(long long total, long long ctas, long long entry)
{
    return ((entry + 1) * ctas - 1) / total;
}

}  // namespace qmm
