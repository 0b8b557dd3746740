// How kv_rows.cu cuts its work: one list over all (sequence, kv head, pass of columns), equal shares of it per CTA.  A list entry
// has a unit for every tile of 16 tokens, behind KV_ENTRY_UNITS for what an entry costs beside its tiles.
// Host code too, so that the tests walk it without a GPU.
#pragma once

#include "kv_layout.cuh"

namespace qmm {

// Starting an entry (queries, page numbers, the first copies) and joining its warps takes a CTA about as long as this many tiles.
// 64 sequences of up to 600 tokens of 32 kv heads of 128, Q4_0: 93 us with 8, 84 with 12, 81 with 16, 80 with 24; one of 8000 tokens 27.5, 25.8,
// 24.3, 24.6.  (With 2, and 4, 149 and 116 us: a share that ends just past an entry's head does nothing but its start and its join.)
constexpr int KV_ENTRY_UNITS = 16;

__host__ __device__ __forceinline__ int kv_max(int a, int b)
{
    return a > b ? a : b;
}
__host__ __device__ __forceinline__ int kv_min(int a, int b)
{
    return a < b ? a : b;
}
// First position that a row at `pos` sees (window 0: no limit).  No difference is taken where it could leave 32 bits: rows in front of
// a sequence's first token have negative positions, and a window may be 2^31 - 1.
__host__ __device__ __forceinline__ int kv_first_seen(int pos, int window)
{
    return window > 0 && pos >= window ? pos - window + 1 : 0;
}
// Division of numbers below 2^63, in 32 bits where they fit (a 64-bit division is a hundred dependent instructions, and a short
// call waits for half a dozen of them).
__host__ __device__ __forceinline__ long long kv_div(long long x, long long y)
{
    if (((unsigned long long)(x | y) >> 32) == 0) {
        return (unsigned int)x / (unsigned int)y;
    }
    return x / y;
}

// A sequence's part of the list: kv heads * passes entries.
struct SeqWork {
    KvSeq q;
    int tile0, tiles, passes;
    long long units;
};
// `cols` columns (query heads of a kv head, times rows) to a pass.
__host__ __device__ __forceinline__ SeqWork seq_work(const KvPool& c, const KvSeqs& b, int group, int window, int cols, int s,
                                                     bool& bad)
{
    SeqWork x;
    x.q = kv_seq(c, b, s, bad);
    // tiles from the first that the first row's window reaches to the last token's; a sequence without any still has its
    // rows' zeros to write
    const int first = x.q.len - x.q.n;
    x.tile0 = kv_first_seen(first, window) / KV_TILE;
    x.tiles = kv_max(1, (x.q.len + KV_TILE - 1) / KV_TILE - x.tile0);
    x.passes = (int)(((long long)x.q.n * group + cols - 1) / cols);
    x.units = (long long)c.kv_heads * x.passes * (x.tiles + KV_ENTRY_UNITS);
    return x;
}

// What one pass of a sequence sees.
struct PassView {
    int col0, cols;
    int pos_lo, pos_hi;   // positions of the first and the last column's row
    int seen_lo, all_lo;  // some column sees seen_lo .. pos_hi, every column all_lo .. pos_lo
    int tile_begin, tile_end;  // of the given tiles, those that some column sees
};
__host__ __device__ __forceinline__ PassView pass_view(const SeqWork& x, int group, int window, int cols, int pass, int tile_begin,
                                                       int tile_end)
{
    PassView v;
    const long long columns = (long long)x.q.n * group;
    v.col0 = pass * cols;
    v.cols = columns - v.col0 < cols ? (int)(columns - v.col0) : cols;
    const int first = x.q.len - x.q.n;
    v.pos_lo = first + v.col0 / group;
    v.pos_hi = first + (v.col0 + v.cols - 1) / group;
    v.seen_lo = kv_first_seen(v.pos_lo, window);
    v.all_lo = kv_first_seen(v.pos_hi, window);
    v.tile_begin = kv_max(tile_begin, v.seen_lo / KV_TILE);
    v.tile_end = kv_min(tile_end, v.pos_hi < 0 ? 0 : v.pos_hi / KV_TILE + 1);
    return v;
}

// CTAs that take a share: all where each gets eight tiles (a CTA has four warps, which take two at a time), else one for every
// eight, as a whole number to an entry, so that equal entries end where shares end: 130 tokens of 32 kv heads of 128, Q4_0, take
// 10.4 us on 32 CTAs and 18.1 us on 36.  (One for every four: 16 sequences of 100 tokens 24 us instead of 12; for every sixteen: one of
// 700 tokens 21 instead of 15.)
__host__ __device__ __forceinline__ long long share_count(long long units, long long entries, long long grid)
{
    const long long want = (units - entries * KV_ENTRY_UNITS) / 8;
    if (want >= grid || entries >= want) {
        return want >= grid || entries >= grid ? grid : entries;
    }
    const long long per = kv_div(want + entries / 2, entries);
    return entries * per <= grid ? entries * per : entries * (per - 1);
}
// `ctas` equal shares of `units`, the first ones a unit longer: where share i begins, and which share has a unit.
__host__ __device__ __forceinline__ long long share_begin(long long units, long long ctas, long long i)
{
    const long long each = kv_div(units, ctas), more = units - each * ctas;
    return i * each + (i < more ? i : more);
}
__host__ __device__ __forceinline__ long long share_of(long long units, long long ctas, long long unit)
{
    const long long each = kv_div(units, ctas), more = units - each * ctas, longer = more * (each + 1);
    return unit < longer ? kv_div(unit, each + 1) : more + kv_div(unit - longer, each);
}

}  // namespace qmm
