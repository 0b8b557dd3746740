// Test-only helper: the paged cache's index functions and the walk over its list of tiles, on the host.
#include <cstdint>
#include <cstring>
#include <set>
#include <vector>

#include "../../litenn_b200/csrc/kv_rows_plan.cuh"

using namespace qmm;

// Every (half, lane, block, byte) of a quant plane and every scale has a byte of its own; 0 if so.
extern "C" int kv_places(int fmt, int hd)
{
    std::vector<int> seen(kv_plane_bytes(fmt, hd), 0), scales(kv_scale_bytes(fmt, hd), 0);
    for (int j = 0; j < 2; ++j) {
        for (int p = 0; p < 32; ++p) {
            for (int b = 0; b < hd / 32; ++b) {
                for (int x = 0; x < kv_unit(fmt); ++x) {
                    const int at = kv_place(fmt, hd, j, p, b, x);
                    if (at < 0 || at >= (int)seen.size() || seen[at]++) {
                        return 1;
                    }
                }
            }
        }
    }
    for (int token = 0; token < 16 && fmt != KV_F16; ++token) {
        for (int b = 0; b < hd / 32; ++b) {
            const int at = kv_scale_place(hd, token, b);
            if (at < 0 || at + 1 >= (int)scales.size() || scales[at]++ || scales[at + 1]++) {
                return 2;
            }
        }
    }
    return 0;
}

// Walks the list as the CTAs do, with `cols` columns to a pass.  visits[row][kv head][head of the group][token]: how often each is
// visited, `tokens` per row; returns 0, or what went wrong.
extern "C" int kv_walk(int fmt, int kv_heads, int hd, int page_tokens, long long n_pages, int batch, int table_width,
                       const int* table, const int* kv_len, const int* row_begin, long long rows, int group, int window, int cols,
                       int grid, int tokens, int* visits, int* bad_rows, int* bad_pages)
{
    const KvPool pool = {nullptr, fmt, kv_heads, hd, page_tokens, n_pages};
    const KvSeqs seqs = {batch, table_width, table, kv_len, row_begin, rows, nullptr};
    const long long pool_tiles = n_pages * kv_heads * (page_tokens / KV_TILE);
    long long units = 0, entries = 0;
    for (int s = 0; s < batch; ++s) {
        bool bad;
        const SeqWork x = seq_work(pool, seqs, group, window, cols, s, bad);
        units += x.units;
        entries += (long long)kv_heads * x.passes;
        *bad_rows += bad;
    }
    if (units == 0) {
        return 0;
    }
    const long long ctas = share_count(units, entries, grid);
    if (ctas < 1 || ctas > grid) {
        return 14;
    }
    long long next = 0;
    std::vector<int> parts(ctas, 0), wanted(ctas, 0), slots(2 * ctas, 0);
    for (long long c = 0; c < ctas; ++c) {
        const long long begin = share_begin(units, ctas, c), end = share_begin(units, ctas, c + 1);
        if (begin != next || end <= begin) {
            return 1;
        }
        next = end;
        int seq = 0;
        long long first = 0;
        bool bad;
        SeqWork x = seq_work(pool, seqs, group, window, cols, 0, bad);
        for (long long at = begin; at < end;) {
            while (at >= first + x.units) {
                first += x.units;
                if (++seq >= batch) {
                    return 2;
                }
                x = seq_work(pool, seqs, group, window, cols, seq, bad);
            }
            const int each = x.tiles + KV_ENTRY_UNITS;
            const long long entry = kv_div(at - first, each);
            const long long e0 = first + entry * each + KV_ENTRY_UNITS, e1 = e0 + x.tiles;
            const int head = (int)(entry / x.passes), pass = (int)(entry % x.passes);
            const long long from = at > e0 ? at : e0, to = end < e1 ? end : e1;
            at = to;
            if (end < e1) {
                at = end;
            }
            if (from >= to) {
                continue;
            }
            if (head >= kv_heads) {
                return 3;
            }
            const PassView v = pass_view(x, group, window, cols, pass, x.tile0 + (int)(from - e0), x.tile0 + (int)(to - e0));
            if (v.cols < 1 || v.cols > cols || v.col0 + v.cols > (long long)x.q.n * group) {
                return 4;
            }
            for (int tile = v.tile_begin; tile < v.tile_end; ++tile) {
                if (tile * KV_TILE / page_tokens >= table_width) {
                    return 5;
                }
                const int page = kv_page(pool, seqs, seq, tile * KV_TILE);
                if (page < 0) {
                    ++*bad_pages;
                    continue;
                }
                const long long index = kv_tile_index(pool, page, head, tile * KV_TILE);
                if (index < 0 || index >= pool_tiles) {
                    return 6;
                }
                for (int col = v.col0; col < v.col0 + v.cols; ++col) {
                    const long long row = x.q.row0 + col / group;
                    if (row < 0 || row >= rows) {
                        return 7;
                    }
                    const int pos = x.q.len - x.q.n + col / group, lo = window > 0 ? kv_max(0, pos - window + 1) : 0;
                    for (int t = tile * KV_TILE; t < tile * KV_TILE + KV_TILE; ++t) {
                        const bool whole = t >= v.all_lo && t <= v.pos_lo, sees = t <= pos && t >= lo;
                        if (whole && !sees) {
                            return 8;
                        }
                        if (sees && (t > v.pos_hi || t < v.seen_lo || t >= tokens)) {
                            return 9;
                        }
                        if (sees) {
                            ++visits[((row * kv_heads + head) * group + col % group) * tokens + t];
                        }
                    }
                }
            }
            const long long c0 = share_of(units, ctas, e0), c1 = share_of(units, ctas, e1 - 1);
            if (c < c0 || c > c1 || share_begin(units, ctas, c0) > e0 || share_begin(units, ctas, c0 + 1) <= e0) {
                return 10;
            }
            if (((from == e0) != (c == c0)) || ((e1 <= end) != (c == c1))) {
                return 11;
            }
            if (c0 != c1) {
                ++parts[c0];
                wanted[c0] = (int)(c1 - c0 + 1);
                if (slots[2 * c + (from == e0 ? 1 : 0)]++) {
                    return 15;  // a place of the workspace for two parts
                }
            }
        }
    }
    return next != units ? 12 : parts != wanted ? 13 : 0;
}
