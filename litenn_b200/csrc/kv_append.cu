// Appending to the paged cache and reading it back (include/litenn_kv.h).
//
// Append: a row's queries and keys are turned by their position's angles, keys and values are quantized in blocks of 32
// dimensions and stored where the attention kernels' operands want them (kv_layout.cuh).  The angles and the rotation are
// taken in fp64: a position of 10^5 times a frequency near 1 has lost eight of fp32's bits before the cosine is taken, and the
// blocks' rounding turns a last-bit difference into another quant.  Rounding the rotated value to fp32 once makes the stored
// bytes a function of the inputs alone, whichever form wrote them.
#include <type_traits>

#include "kv_kernels.h"

#include "../../include/litenn_qmm.h"

namespace qmm {

namespace {

__device__ __forceinline__ void pdl_trigger()
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void pdl_sync()
{
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

// Four consecutive values of a row.
__device__ __forceinline__ void load4(const void* p, int64_t at, int type, float (&x)[4])
{
    if (type == QMM_OUT_F32) {
        const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + at);
        x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
    } else {
        const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(p) + at);
        x[0] = __uint_as_float(v.x << 16), x[1] = __uint_as_float(v.x & 0xFFFF0000u);
        x[2] = __uint_as_float(v.y << 16), x[3] = __uint_as_float(v.y & 0xFFFF0000u);
    }
}
__device__ __forceinline__ void store4(void* p, int64_t at, int type, const float (&x)[4])
{
    if (type == QMM_OUT_F32) {
        *reinterpret_cast<float4*>(static_cast<float*>(p) + at) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
        const __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
        uint2 v;
        v.x = *reinterpret_cast<const uint32_t*>(&a);
        v.y = *reinterpret_cast<const uint32_t*>(&b);
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p) + at) = v;
    }
}

// (x, y) turned by (c, s), rounded to fp32 once.
__device__ __forceinline__ float2 turned(float x, float y, double2 cs)
{
    return make_float2((float)((double)x * cs.x - (double)y * cs.y), (float)((double)x * cs.y + (double)y * cs.x));
}

// The eight lanes of a 32-dimension block hold four values each: the block's scale and this lane's four quants, by GGUF's
// rules in fp32 (no contraction: the bytes must not depend on how the compiler joins a product and a sum).  Magnitudes are
// compared as their bits, which puts infinities and NaN above all else.
template <int FMT>
__device__ __forceinline__ float quantize4(const float (&x)[4], int lane, uint32_t (&q)[4])
{
    float top = x[0];
    uint32_t size = __float_as_uint(x[0]) & 0x7FFFFFFFu;
#pragma unroll
    for (int i = 1; i < 4; ++i) {
        const uint32_t bits = __float_as_uint(x[i]) & 0x7FFFFFFFu;
        top = bits > size ? x[i] : top;  // the first of equals
        size = max(size, bits);
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        const float other = __shfl_xor_sync(0xFFFFFFFFu, top, o);
        const uint32_t bits = __float_as_uint(other) & 0x7FFFFFFFu;
        const bool lower = (lane & o) != 0;  // the other lane's values come first
        top = bits > size || (lower && bits == size) ? other : top;
        size = max(size, bits);
    }
    const bool odd = size >= 0x7F800000u;
    constexpr float MOST = FMT == FMT_Q4_0 ? 8188.0f : 515.5f;  // q * d stays within fp16's range
    float d = FMT == FMT_Q4_0 ? top * -0.125f : __fdiv_rn(__uint_as_float(size), 127.0f);
    d = fminf(fmaxf(d, -MOST), MOST);
    const float inverse = d == 0.0f ? 0.0f : __frcp_rn(d);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        // the whole part of a number from 0 to 2^23: the last bits of its sum with 2^23, rounded down (no conversion unit)
        const float y = __fmul_rn(x[i], inverse);
        if (FMT == FMT_Q4_0) {
            q[i] = __float_as_uint(__fadd_rd(fminf(fmaxf(__fadd_rn(y, 8.5f), 0.0f), 15.0f), 8388608.0f)) & 15u;
        } else {
            // half added rounding down: to the nearest, 0.5 - 2^-25 would become 1
            const uint32_t r = __float_as_uint(__fadd_rd(fminf(__fadd_rd(fabsf(y), 0.5f), 127.0f), 8388608.0f)) & 127u;
            q[i] = y < 0.0f ? 128u - r : 128u + r;
        }
        q[i] = odd ? (FMT == FMT_Q4_0 ? 8u : 128u) : q[i];
    }
    return odd ? __uint_as_float(0x7FC00000u) : d;
}

// Four consecutive values of a token as the cache holds them.
template <int FMT>
struct Packed {
    uint32_t w[FMT == KV_F16 ? 2 : 1];
    float d;
};
// All 32 lanes call it: a block's eight join in its maximum, and a Q4_0 key word is two lanes'.
template <int FMT>
__device__ __forceinline__ Packed<FMT> pack4(bool keys, int dim, const float (&x)[4], int lane)
{
    Packed<FMT> p;
    if constexpr (FMT == KV_F16) {
        const __half2 lo = __floats2half2_rn(x[0], x[1]), hi = __floats2half2_rn(x[2], x[3]);
        p.w[0] = *reinterpret_cast<const uint32_t*>(&lo);
        p.w[1] = *reinterpret_cast<const uint32_t*>(&hi);
        p.d = 0.0f;
    } else {
        uint32_t q[4];
        p.d = quantize4<FMT>(x, lane, q);
        if (FMT == FMT_Q4_0) {
            // keys: dims 4h.. of a lane's eight are bytes h and h + 2 of its word, the pair of lanes joins them.  All lanes take
            // part: a warp may hold keys and values
            const uint32_t mine = ((q[0] | q[2] << 4) | (q[1] | q[3] << 4) << 16) << (8u * ((uint32_t)(dim >> 2) & 1u));
            const uint32_t word = mine | __shfl_xor_sync(0xFFFFFFFFu, mine, 1);
            p.w[0] = keys ? word : q[0] | q[1] << 4 | q[2] << 8 | q[3] << 12;
        } else {
            p.w[0] = q[0] | q[1] << 8 | q[2] << 16 | q[3] << 24;
        }
    }
    return p;
}
// Stores them: `keys` tells which plane's order.
template <int FMT>
__device__ __forceinline__ void place4(uint8_t* tile, int hd, bool keys, int token, int dim, const Packed<FMT>& p)
{
    const int b = dim >> 5, first = keys ? 0 : kv_plane_bytes(FMT, hd) + kv_scale_bytes(FMT, hd);
    const int j = token >> 3, e = token & 1;
    const int lane = keys ? 4 * (token & 7) + (dim >> 3 & 3) : 4 * (dim >> 2 & 7) + (token >> 1 & 3);
    uint8_t* at = tile + first + kv_place(FMT, hd, j, lane, b, 0);  // the lane's eight values of the block
    if constexpr (FMT == KV_F16) {
        if (keys) {
            *reinterpret_cast<uint2*>(at + 2 * (dim & 4)) = make_uint2(p.w[0], p.w[1]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                *reinterpret_cast<uint16_t*>(at + 4 * i + 2 * e) = (uint16_t)(p.w[i >> 1] >> (16 * (i & 1)));
            }
        }
    } else {
        if (FMT == FMT_Q4_0) {
            if (!keys) {
                *reinterpret_cast<uint16_t*>(at + 2 * e) = (uint16_t)p.w[0];
            } else if ((dim & 4) == 0) {
                *reinterpret_cast<uint32_t*>(at) = p.w[0];
            }
        } else if (keys) {
            *reinterpret_cast<uint32_t*>(at + (dim & 4)) = p.w[0];
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                at[2 * i + e] = (uint8_t)(p.w[0] >> (8 * i));
            }
        }
        if ((dim & 31) == 0) {
            *reinterpret_cast<__half*>(tile + first + kv_plane_bytes(FMT, hd) + kv_scale_place(hd, token, b)) =
                __float2half_rn(p.d);
        }
    }
}

// Four consecutive values of a token as fp32.
template <int FMT>
__device__ __forceinline__ void get4(const uint8_t* tile, int hd, bool keys, int token, int dim, float (&x)[4])
{
    const int b = dim >> 5, first = keys ? 0 : kv_plane_bytes(FMT, hd) + kv_scale_bytes(FMT, hd);
    const int j = token >> 3, e = token & 1;
    const int lane = keys ? 4 * (token & 7) + (dim >> 3 & 3) : 4 * (dim >> 2 & 7) + (token >> 1 & 3);
    const uint8_t* at = tile + first + kv_place(FMT, hd, j, lane, b, 0);  // the lane's eight values of the block
    const int half = dim >> 2 & 1;                                        // keys: which four of them
    if (FMT == KV_F16) {
        if (keys) {
            const uint2 w = *reinterpret_cast<const uint2*>(at + 8 * half);
            const float2 lo = __half22float2(*reinterpret_cast<const __half2*>(&w.x)), hi = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
            x[0] = lo.x, x[1] = lo.y, x[2] = hi.x, x[3] = hi.y;
        } else {
            const uint4 w = *reinterpret_cast<const uint4*>(at);  // pairs of tokens
            const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = __half2float(__ushort_as_half((unsigned short)(v[i] >> (16 * e))));
            }
        }
        return;
    }
    const float d = __half2float(
        *reinterpret_cast<const __half*>(tile + first + kv_plane_bytes(FMT, hd) + kv_scale_place(hd, token, b)));
    int q[4];
    if (FMT == FMT_Q4_0) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(at);
        // keys: dimension 4 half + i is nibble 2 half + (i >> 1) of the lower (i even) or the upper 16 bits; values: nibble i of
        // the token's 16 bits
        const uint32_t lo = keys ? w >> (8 * half) : w >> (16 * e), hi = keys ? w >> (16 + 8 * half) : lo >> 8;
        q[0] = (int)(lo & 15u);
        q[1] = (int)(keys ? hi & 15u : lo >> 4 & 15u);
        q[2] = (int)(keys ? lo >> 4 & 15u : hi & 15u);
        q[3] = (int)(hi >> 4 & 15u);
    } else {
        const uint2 w = *reinterpret_cast<const uint2*>(at);
        const uint32_t k = half ? w.y : w.x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            q[i] = (int)(keys ? k >> (8 * i) & 255u : (i < 2 ? w.x : w.y) >> (16 * (i & 1) + 8 * e) & 255u);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[i] = (float)(q[i] - (FMT == FMT_Q4_0 ? 8 : 128)) * d;
    }
}

// Sequence of a row: the lowest that claims it (there is one unless row_begin is not rising).  Whole CTA; reports what is bad.
struct RowPlace {
    int seq, pos;  // seq < 0: no sequence has the row
};
__device__ __forceinline__ RowPlace find_row(const KvPool& c, const KvSeqs& b, int64_t row, int* found)
{
    if (threadIdx.x == 0) {
        *found = b.batch;
    }
    __syncthreads();
    if (!b.row_begin) {
        if (threadIdx.x == 0) {
            *found = row < b.batch ? (int)row : b.batch;
        }
    } else {
        for (int s = threadIdx.x; s < b.batch; s += blockDim.x) {
            if (__ldg(b.row_begin + s) <= row && row < __ldg(b.row_begin + s + 1)) {
                atomicMin(found, s);
            }
            if (row == 0) {  // what cannot be right may have no rows
                bool bad;
                kv_seq(c, b, s, bad);
                if (bad) {
                    atomicExch(b.status, KV_BAD_ROWS);
                }
            }
        }
    }
    __syncthreads();
    RowPlace p;
    p.seq = *found < b.batch ? *found : -1;
    p.pos = 0;
    if (p.seq >= 0) {
        bool bad;
        const KvSeq q = kv_seq(c, b, p.seq, bad);
        const int first = q.len - q.n;
        if (bad || first < 0) {
            if (threadIdx.x == 0) {
                atomicExch(b.status, KV_BAD_ROWS);
            }
            p.seq = -1;
        } else {
            p.pos = first + (int)(row - q.row0);
        }
    }
    return p;
}

// One row per blockIdx.y, its work cut over blockIdx.x: every thread takes four dimensions of a head.  For few rows, where a call's
// time is its latency: one token of 8 kv heads of 128 and 32 query heads 3.0 us in Q4_0, 16 tokens 3.3 us (its bytes would take 0.1 us).
template <int FMT>
__global__ void __launch_bounds__(256) kv_append_kernel(const KvAppendArgs a)
{
    __shared__ int found;
    __shared__ double2 turn[128];
    pdl_trigger();
    pdl_sync();
    const int hd = a.pool.head_dim, lane = threadIdx.x & 31;
    for (int64_t row = blockIdx.y; row < a.seqs.rows; row += gridDim.y) {
        __syncthreads();
        const RowPlace at = find_row(a.pool, a.seqs, row, &found);
        if (at.seq < 0) {
            continue;
        }
        const int page = kv_page(a.pool, a.seqs, at.seq, at.pos);
        if (page < 0 && threadIdx.x == 0) {
            atomicExch(a.seqs.status, KV_BAD_PAGE);
        }
        const int n = a.rope.dim / 2;
        for (int i = threadIdx.x; i < n; i += blockDim.x) {
            double s, c;
            sincos((double)at.pos * a.rope.inv_freq[i], &s, &c);
            turn[i] = make_double2(c * a.rope.gain, s * a.rope.gain);
        }
        __syncthreads();
        const int q_items = a.heads * hd / 4, kv_items = a.pool.kv_heads * hd / 4;
        const int all = q_items + 2 * kv_items, step = gridDim.x * blockDim.x;
        // whole warps: q_items and kv_items are multiples of 8, and the block sums of eight lanes want their warp
        for (int base = blockIdx.x * blockDim.x + (threadIdx.x & ~31); base < all; base += step) {
            const int item = base + lane;
            const bool is_q = item < q_items, on = item < all;
            const bool keys = item < q_items + kv_items;
            const int mine = is_q ? item : keys ? item - q_items : item - q_items - kv_items;
            const int head = mine / (hd / 4), dim = mine % (hd / 4) * 4;
            const void* src = is_q ? a.q : keys ? a.k : a.v;
            const int64_t in = row * (is_q ? a.q_stride : keys ? a.k_stride : a.v_stride) + (int64_t)head * hd;
            float x[4] = {0.0f, 0.0f, 0.0f, 0.0f}, y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            bool both = false, skip = false;  // queries in halves: the first half's lanes turn and store the second's too
            if (on) {
                load4(src, in + dim, a.type, x);
                if (keys && dim < 2 * n) {
                    if (!a.rope.halves) {
#pragma unroll
                        for (int i = 0; i < 4; i += 2) {
                            if (dim + i < 2 * n) {
                                const float2 r = turned(x[i], x[i + 1], turn[(dim + i) >> 1]);
                                x[i] = r.x, x[i + 1] = r.y;
                            }
                        }
                    } else {
                        const bool second = dim >= n;
                        both = is_q && !second;
                        skip = is_q && second;
                        if (!skip) {
                            load4(src, in + (second ? dim - n : dim + n), a.type, y);
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const float2 r = second ? turned(y[i], x[i], turn[dim - n + i]) : turned(x[i], y[i], turn[dim + i]);
                                x[i] = second ? r.y : r.x;
                                y[i] = second ? r.x : r.y;
                            }
                        }
                    }
                }
                if (is_q && !skip) {
                    const int64_t out = row * a.q_out_stride + (int64_t)head * hd + dim;
                    store4(a.q_out, out, a.q_type, x);
                    if (both) {
                        store4(a.q_out, out + n, a.q_type, y);
                    }
                }
            }
            uint8_t* tile = a.pool.base + kv_tile_index(a.pool, max(page, 0), is_q || !on ? 0 : head, at.pos) * kv_tile_bytes(FMT, hd);
            const Packed<FMT> p = pack4<FMT>(keys, dim, x, lane);
            if (on && !is_q && page >= 0) {
                place4<FMT>(tile, hd, keys, at.pos % KV_TILE, dim, p);
            }
        }
    }
}

template <int FMT>
__global__ void __launch_bounds__(256) kv_read_kernel(const KvReadArgs a)
{
    __shared__ int found;
    pdl_trigger();
    pdl_sync();
    const int hd = a.pool.head_dim;
    for (int64_t row = blockIdx.y; row < a.seqs.rows; row += gridDim.y) {
        __syncthreads();
        const RowPlace at = find_row(a.pool, a.seqs, row, &found);
        if (at.seq < 0) {
            continue;
        }
        const int page = kv_page(a.pool, a.seqs, at.seq, at.pos);
        if (page < 0) {
            if (threadIdx.x == 0) {
                atomicExch(a.seqs.status, KV_BAD_PAGE);
            }
            continue;
        }
        const int items = a.pool.kv_heads * hd / 4;
        for (int item = blockIdx.x * blockDim.x + threadIdx.x; item < 2 * items; item += gridDim.x * blockDim.x) {
            const bool keys = item < items;
            const int mine = keys ? item : item - items;
            const int head = mine / (hd / 4), dim = mine % (hd / 4) * 4;
            const uint8_t* tile = a.pool.base + kv_tile_index(a.pool, page, head, at.pos) * kv_tile_bytes(FMT, hd);
            float x[4];
            get4<FMT>(tile, hd, keys, at.pos % KV_TILE, dim, x);
            store4(keys ? a.k : a.v, row * (keys ? a.k_stride : a.v_stride) + (int64_t)head * hd + dim, a.type, x);
        }
    }
}

// ---- prompts: one tile of 16 tokens per CTA and group of heads -----------------------------------------------------------
// A token's values lie in pieces of 1 to 4 bytes all over a tile (two tokens share an operand register), so whole tiles are put
// together in shared memory and leave as 16-byte stores; a sequence's first and last tile may be shared with tokens that are
// there already and are stored piece by piece.  Bound: bytes (rows in, queries out, tiles out).

// A tile of a call: 16 positions of a sequence, those from `begin` to `end` being rows of the call from `row` on.
struct TilePlace {
    int seq, pos0, begin, end;  // seq < 0: there is no such tile
    int64_t row;
};
// The `want`-th tile over all sequences.  Whole CTA; the first reports what is bad.  A lane counts the tiles of batch / 32 sequences in
// a row, and the one that has the tile counts again.
__device__ __forceinline__ TilePlace find_tile(const KvPool& c, const KvSeqs& b, int64_t want, TilePlace* shared)
{
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x, each = (b.batch + 31) / 32, s0 = lane * each, s1 = min(b.batch, s0 + each);
        const auto look = [&](int s, bool& bad) {
            KvSeq q = kv_seq(c, b, s, bad);
            bad = bad || q.len < q.n;
            q.n = bad ? 0 : q.n;
            return q;
        };
        const auto tiles = [](const KvSeq& q) { return q.n > 0 ? (q.len - 1) / KV_TILE - (q.len - q.n) / KV_TILE + 1 : 0; };
        int64_t mine = 0;
        bool any_bad = false;
#pragma unroll 4
        for (int s = s0; s < s1; ++s) {
            bool bad;
            mine += tiles(look(s, bad));
            any_bad = any_bad || bad;
        }
        if (any_bad && want == 0) {
            atomicExch(b.status, KV_BAD_ROWS);
        }
        int64_t upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t u = __shfl_up_sync(0xFFFFFFFFu, upto, o);
            upto += lane >= o ? u : 0;
        }
        int64_t before = upto - mine;
        const bool here = before <= want && want < upto;
        if (here) {
            for (int s = s0; s < s1; ++s) {
                bool bad;
                const KvSeq q = look(s, bad);
                const int n = tiles(q);
                if (want < before + n) {
                    TilePlace p;
                    const int first = q.len - q.n, tile = first / KV_TILE + (int)(want - before);
                    p.seq = s;
                    p.pos0 = tile * KV_TILE;
                    p.begin = max(0, first - p.pos0);
                    p.end = min(KV_TILE, q.len - p.pos0);
                    p.row = q.row0 + (p.pos0 + p.begin - first);
                    *shared = p;
                    break;
                }
                before += n;
            }
        }
        if (!__any_sync(0xFFFFFFFFu, here) && lane == 0) {
            shared->seq = -1;
        }
    }
    __syncthreads();
    return *shared;
}
// At most this many tiles hold rows of a call.
int64_t tiles_of(const KvSeqs& b)
{
    return b.rows / KV_TILE + 2 * (int64_t)b.batch;
}

constexpr int TILE_WARPS = 8;
constexpr int TILE_Q_HEADS = 16;  // query heads of a CTA that has those
template <int FMT, int HD>
struct TileShape {
    static constexpr int BYTES = kv_tile_bytes(FMT, HD);
    static constexpr int KV_HEADS = BYTES <= 4608 ? 8 : BYTES <= 8192 ? 4 : 2;  // kv heads of a CTA that has those
    static constexpr int LANES = HD / 4;                    // that a head's row takes, four values each
    // A warp's lane keeps its dimensions from head to head, so it reads its angles once per row: LW lanes and SEGS turns to a
    // head, HPW heads at once.
    static constexpr int LW = LANES < 32 ? LANES : 32, SEGS = LANES / LW, HPW = 32 / LW;
};

// A lane's angles: of its pairs (dim, dim + 1), (dim + 2, dim + 3), or in halves of its four dimensions (either half's).
template <bool HALVES>
struct Angles {
    double2 cs[HALVES ? 4 : 2];
    __device__ __forceinline__ void load(const double2* turn, int dim, int n)
    {
        const int first = HALVES ? (dim >= n ? dim - n : dim) : dim >> 1;
        if (dim < 2 * n) {
#pragma unroll
            for (int i = 0; i < (HALVES ? 4 : 2); ++i) {
                cs[i] = HALVES || first + i < n ? turn[first + i] : make_double2(1.0, 0.0);
            }
        }
    }
};

// One row's queries in halves, by one warp: n / 4 lanes to a head, each with four dimensions of the first half and the four
// they turn with, so that every lane has pairs whatever part of the head turns; then the dimensions behind, copied.
template <int UNROLL>
__device__ __forceinline__ void turn_halves(const KvAppendArgs& a, const double2* turn, int n, int64_t in, int64_t out, int heads,
                                            int hd, int lane)
{
    if (n) {
        const int lanes = n / 4, per_warp = 32 / lanes, dim = lane % lanes * 4;
        Angles<true> t;
        t.load(turn, dim, n);
        for (int base = lane / lanes; base < heads && lane < per_warp * lanes; base += UNROLL * per_warp) {
            float x[UNROLL][4], y[UNROLL][4];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const int h = base + u * per_warp;
                if (h < heads) {
                    load4(a.q, in + h * hd + dim, a.type, x[u]);
                    load4(a.q, in + h * hd + dim + n, a.type, y[u]);
                }
            }
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const int h = base + u * per_warp;
                if (h < heads) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 z = turned(x[u][i], y[u][i], t.cs[i]);
                        x[u][i] = z.x, y[u][i] = z.y;
                    }
                    store4(a.q_out, out + h * hd + dim, a.q_type, x[u]);
                    store4(a.q_out, out + h * hd + dim + n, a.q_type, y[u]);
                }
            }
        }
    }
    const int rest = hd / 4 - n / 2;
    if (rest && (a.q_out != a.q || a.q_type != a.type)) {
        const int lanes = rest < 32 ? rest : 32, per_warp = 32 / lanes;
        for (int base = lane / lanes; base < heads && lane < per_warp * lanes; base += UNROLL * per_warp) {
            for (int dim = 2 * n + lane % lanes * 4; dim < hd; dim += 128) {
                float x[UNROLL][4];
#pragma unroll
                for (int u = 0; u < UNROLL; ++u) {
                    if (base + u * per_warp < heads) {
                        load4(a.q, in + (base + u * per_warp) * hd + dim, a.type, x[u]);
                    }
                }
#pragma unroll
                for (int u = 0; u < UNROLL; ++u) {
                    if (base + u * per_warp < heads) {
                        store4(a.q_out, out + (base + u * per_warp) * hd + dim, a.q_type, x[u]);
                    }
                }
            }
        }
    }
}

// Many rows.  blockIdx.x: groups of kv heads, then groups of query heads; blockIdx.y: tiles.  A warp takes a row at a time.  A whole
// tile is put together in shared memory: stored from the registers, its two- and four-byte pieces made a sector of DRAM traffic
// each.  1999 rows of 32 heads of 128 with as many kv heads, fp32 to Q4_0, are 140 MB in 47 us (46 % of the copy rate), to Q8_0 148 MB
// in 51, to fp16 164 MB in 46; sixteen prompts of 33 to 901 rows, 64 query and 8 kv heads of 128, half of each rotated, bf16 to fp16,
// 306 MB in 105 us (44 %).  Bound: latency, at 4.8 warps a scheduler (half of the issue slots, 7 % of the fp64 units): a tile's place, its
// angles and a barrier come before the first rows are asked for.  With the read of the same rows behind it (42 MB in 20 us, 61 MB in 21):
// registers for three CTAs of an SM 64 and 124 us, two left loads exposed (ragged prompts 218), four spill (144); sixteen warps a CTA 64
// and 147.
template <int FMT, int HD, bool HALVES>
__global__ void __launch_bounds__(TILE_WARPS * 32, 24 / TILE_WARPS) kv_append_tile_kernel(const KvAppendArgs a)
{
    using Shape = TileShape<FMT, HD>;
    constexpr int UNROLL = HALVES ? 2 : 4;
    extern __shared__ __align__(16) uint8_t append_smem[];
    __shared__ TilePlace place;
    double2* turn = reinterpret_cast<double2*>(append_smem);  // [16][rope.dim / 2]
    const int n = a.rope.dim / 2;
    uint8_t* tiles = append_smem + (size_t)KV_TILE * n * sizeof(double2);  // [KV_HEADS]
    pdl_trigger();
    pdl_sync();
    const TilePlace at = find_tile(a.pool, a.seqs, blockIdx.y, &place);
    if (at.seq < 0) {
        return;
    }
    const int rows = at.end - at.begin;
    for (int i = threadIdx.x; i < rows * n; i += blockDim.x) {
        double s, c;
        sincos((double)(at.pos0 + at.begin + i / n) * a.rope.inv_freq[i % n], &s, &c);
        turn[i] = make_double2(c * a.rope.gain, s * a.rope.gain);
    }
    __syncthreads();
    const int kv_groups = (a.pool.kv_heads + Shape::KV_HEADS - 1) / Shape::KV_HEADS;
    const int lane = threadIdx.x & 31;
    if ((int)blockIdx.x >= kv_groups) {
        const int h0 = ((int)blockIdx.x - kv_groups) * TILE_Q_HEADS, heads = min(TILE_Q_HEADS, a.heads - h0);
        for (int r = threadIdx.x >> 5; r < rows; r += TILE_WARPS) {
            const int64_t in = (at.row + r) * a.q_stride + (int64_t)h0 * HD, out = (at.row + r) * a.q_out_stride + (int64_t)h0 * HD;
            if (HALVES) {
                turn_halves<UNROLL>(a, turn + r * n, n, in, out, heads, HD, lane);
                continue;
            }
#pragma unroll
            for (int seg = 0; seg < Shape::SEGS; ++seg) {
                const int dim = lane % Shape::LW * 4 + seg * 128;
                const bool turns = dim < 2 * n;
                Angles<false> t;
                t.load(turn + r * n, dim, n);
                for (int base = lane / Shape::LW; base < heads; base += UNROLL * Shape::HPW) {
                    float x[UNROLL][4];
#pragma unroll
                    for (int u = 0; u < UNROLL; ++u) {
                        const int h = base + u * Shape::HPW;
                        if (lane < Shape::HPW * Shape::LW && h < heads) {
                            load4(a.q, in + h * HD + dim, a.type, x[u]);
                        }
                    }
#pragma unroll
                    for (int u = 0; u < UNROLL; ++u) {
                        const int h = base + u * Shape::HPW;
                        if (lane >= Shape::HPW * Shape::LW || h >= heads) {
                            continue;
                        }
                        if (turns) {
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                if (dim + 2 * i < 2 * n) {
                                    const float2 z = turned(x[u][2 * i], x[u][2 * i + 1], t.cs[i]);
                                    x[u][2 * i] = z.x, x[u][2 * i + 1] = z.y;
                                }
                            }
                        }
                        store4(a.q_out, out + h * HD + dim, a.q_type, x[u]);
                    }
                }
            }
        }
        return;
    }
    const int h0 = (int)blockIdx.x * Shape::KV_HEADS, heads = min(Shape::KV_HEADS, a.pool.kv_heads - h0);
    const int page = kv_page(a.pool, a.seqs, at.seq, at.pos0);
    if (page < 0) {
        if (threadIdx.x == 0) {
            atomicExch(a.seqs.status, KV_BAD_PAGE);
        }
        return;
    }
    // a whole tile is put together in shared memory, a part of one goes to its bytes among the others'
    const bool whole = rows == KV_TILE;
    const int64_t between = whole ? (int64_t)Shape::BYTES : (int64_t)(a.pool.page_tokens / KV_TILE) * Shape::BYTES;
    uint8_t* const first = whole ? tiles : a.pool.base + kv_tile_index(a.pool, page, h0, at.pos0) * Shape::BYTES;
    for (int r = threadIdx.x >> 5; r < rows; r += TILE_WARPS) {
#pragma unroll
        for (int seg = 0; seg < Shape::SEGS; ++seg) {
            const int dim = lane % Shape::LW * 4 + seg * 128;
            const bool turns = dim < 2 * n;
            Angles<HALVES> t;
            t.load(turn + r * n, dim, n);
            // every lane packs, those that have a head store
            const auto strip = [&](auto is_keys) {
                constexpr bool KEYS = decltype(is_keys)::value;
                const int64_t in = (at.row + r) * (KEYS ? a.k_stride : a.v_stride) + (int64_t)h0 * HD + dim;
                for (int base = 0; base < heads; base += UNROLL * Shape::HPW) {
                    float x[UNROLL][4], y[KEYS && HALVES ? UNROLL : 1][4];
                    const int h = base + lane / Shape::LW;
                    const auto on = [&](int u) { return lane < Shape::HPW * Shape::LW && h + u * Shape::HPW < heads; };
#pragma unroll
                    for (int u = 0; u < UNROLL; ++u) {
                        x[u][0] = x[u][1] = x[u][2] = x[u][3] = 0.0f;
                        if (on(u)) {
                            load4(KEYS ? a.k : a.v, in + (h + u * Shape::HPW) * HD, a.type, x[u]);
                            if (KEYS && HALVES && turns) {
                                load4(a.k, in + (h + u * Shape::HPW) * HD + (dim >= n ? -n : n), a.type, y[u % (KEYS && HALVES ? UNROLL : 1)]);
                            }
                        }
                    }
                    if (KEYS && turns) {
#pragma unroll
                        for (int u = 0; u < UNROLL; ++u) {
#pragma unroll
                            for (int i = 0; i < (HALVES ? 4 : 2); ++i) {
                                if (HALVES) {
                                    const float other = y[u % (KEYS && HALVES ? UNROLL : 1)][i];
                                    x[u][i] = dim >= n ? turned(other, x[u][i], t.cs[i]).y : turned(x[u][i], other, t.cs[i]).x;
                                } else {
                                    const float2 z = turned(x[u][2 * i % 4], x[u][(2 * i + 1) % 4], t.cs[i % 2]);
                                    const bool both = dim + 2 * i < 2 * n;
                                    x[u][2 * i % 4] = both ? z.x : x[u][2 * i % 4];
                                    x[u][(2 * i + 1) % 4] = both ? z.y : x[u][(2 * i + 1) % 4];
                                }
                            }
                        }
                    }
                    Packed<FMT> p[UNROLL];
#pragma unroll
                    for (int u = 0; u < UNROLL; ++u) {
                        p[u] = pack4<FMT>(KEYS, dim, x[u], lane);
                    }
#pragma unroll
                    for (int u = 0; u < UNROLL; ++u) {
                        if (on(u)) {
                            place4<FMT>(first + (h + u * Shape::HPW) * between, HD, KEYS, at.begin + r, dim, p[u]);
                        }
                    }
                }
            };
            strip(std::true_type{});
            strip(std::false_type{});
        }
    }
    if (whole) {
        __syncthreads();
        for (int i = threadIdx.x; i < heads * (Shape::BYTES / 16); i += blockDim.x) {
            const int h = i / (Shape::BYTES / 16), k = i % (Shape::BYTES / 16);
            reinterpret_cast<uint4*>(a.pool.base + kv_tile_index(a.pool, page, h0 + h, at.pos0) * Shape::BYTES)[k] =
                reinterpret_cast<const uint4*>(tiles + h * Shape::BYTES)[k];
        }
    }
}

template <int FMT, int HD>
__global__ void __launch_bounds__(TILE_WARPS * 32) kv_read_tile_kernel(const KvReadArgs a)
{
    using Shape = TileShape<FMT, HD>;
    extern __shared__ __align__(16) uint8_t read_smem[];
    __shared__ TilePlace place;
    pdl_trigger();
    pdl_sync();
    const TilePlace at = find_tile(a.pool, a.seqs, blockIdx.y, &place);
    if (at.seq < 0) {
        return;
    }
    const int page = kv_page(a.pool, a.seqs, at.seq, at.pos0);
    if (page < 0) {
        if (threadIdx.x == 0) {
            atomicExch(a.seqs.status, KV_BAD_PAGE);
        }
        return;
    }
    const int h0 = (int)blockIdx.x * Shape::KV_HEADS, heads = min(Shape::KV_HEADS, a.pool.kv_heads - h0);
    for (int i = threadIdx.x; i < heads * (Shape::BYTES / 16); i += blockDim.x) {
        const int h = i / (Shape::BYTES / 16), k = i % (Shape::BYTES / 16);
        reinterpret_cast<uint4*>(read_smem + h * Shape::BYTES)[k] =
            reinterpret_cast<const uint4*>(a.pool.base + kv_tile_index(a.pool, page, h0 + h, at.pos0) * Shape::BYTES)[k];
    }
    __syncthreads();
    const int rows = at.end - at.begin;
    const int lane = threadIdx.x & 31;
    for (int r = threadIdx.x >> 5; r < rows; r += TILE_WARPS) {
#pragma unroll
        for (int seg = 0; seg < Shape::SEGS; ++seg) {
            const int dim = lane % Shape::LW * 4 + seg * 128;
            if (lane >= Shape::HPW * Shape::LW) {
                continue;
            }
#pragma unroll 4
            for (int h = lane / Shape::LW; h < 2 * heads; h += Shape::HPW) {
                const bool keys = h < heads;
                const int mine = keys ? h : h - heads;
                float x[4];
                get4<FMT>(read_smem + mine * Shape::BYTES, HD, keys, at.begin + r, dim, x);
                store4(keys ? a.k : a.v, (at.row + r) * (keys ? a.k_stride : a.v_stride) + (int64_t)(h0 + mine) * HD + dim, a.type, x);
            }
        }
    }
}

template <typename Args>
cudaError_t launch_tiles(void (*kernel)(Args), const Args& a, int groups, int64_t tiles, size_t smem, bool (&configured)[64],
                         size_t most_smem, cudaStream_t stream)
{
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) {
        return e;
    }
    if (device < 0 || device >= 64 || !configured[device]) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most_smem);
        if (e != cudaSuccess) {
            return e;
        }
        if (device >= 0 && device < 64) {
            configured[device] = true;
        }
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)groups, (unsigned)tiles);
    cfg.blockDim = dim3(TILE_WARPS * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <int FMT, int HD, bool HALVES>
cudaError_t append_tiles(const KvAppendArgs& a, cudaStream_t stream)
{
    using Shape = TileShape<FMT, HD>;
    static bool configured[64] = {};
    const int groups = (a.pool.kv_heads + Shape::KV_HEADS - 1) / Shape::KV_HEADS + (a.heads + TILE_Q_HEADS - 1) / TILE_Q_HEADS;
    constexpr size_t TILES = (size_t)Shape::KV_HEADS * Shape::BYTES;
    return launch_tiles(kv_append_tile_kernel<FMT, HD, HALVES>, a, groups, tiles_of(a.seqs),
                        (size_t)KV_TILE * (a.rope.dim / 2) * sizeof(double2) + TILES, configured,
                        (size_t)KV_TILE * (HD / 2) * sizeof(double2) + TILES, stream);
}
template <int FMT, int HD>
cudaError_t read_tiles(const KvReadArgs& a, cudaStream_t stream)
{
    using Shape = TileShape<FMT, HD>;
    static bool configured[64] = {};
    constexpr size_t TILES = (size_t)Shape::KV_HEADS * Shape::BYTES;
    return launch_tiles(kv_read_tile_kernel<FMT, HD>, a, (a.pool.kv_heads + Shape::KV_HEADS - 1) / Shape::KV_HEADS, tiles_of(a.seqs),
                        TILES, configured, TILES, stream);
}
template <int FMT>
cudaError_t append_tiles_fmt(const KvAppendArgs& a, cudaStream_t stream)
{
    const bool halves = a.rope.halves;
    switch (a.pool.head_dim) {
    case 64: return halves ? append_tiles<FMT, 64, true>(a, stream) : append_tiles<FMT, 64, false>(a, stream);
    case 96: return halves ? append_tiles<FMT, 96, true>(a, stream) : append_tiles<FMT, 96, false>(a, stream);
    case 128: return halves ? append_tiles<FMT, 128, true>(a, stream) : append_tiles<FMT, 128, false>(a, stream);
    default: return halves ? append_tiles<FMT, 256, true>(a, stream) : append_tiles<FMT, 256, false>(a, stream);
    }
}
template <int FMT>
cudaError_t read_tiles_fmt(const KvReadArgs& a, cudaStream_t stream)
{
    switch (a.pool.head_dim) {
    case 64: return read_tiles<FMT, 64>(a, stream);
    case 96: return read_tiles<FMT, 96>(a, stream);
    case 128: return read_tiles<FMT, 128>(a, stream);
    default: return read_tiles<FMT, 256>(a, stream);
    }
}
// Whether a call goes by tiles: many rows, and sequences of half a tile and more on average; and no more tiles than a grid has.
// A row's CTA is done sooner, a tile's does less work.  8 kv heads of 128, Q4_0, 32 query heads, rows / tiles: append of one
// sequence of 400 rows 12.6 / 16.0 us, 1000 rows 20.8 / 21.1 us (fp16 18.3 / 13.1), 2000 rows 38.8 / 25.1 us, 8000 rows 156 / 66 us;
// of 500 sequences of 4 rows 39.6 / 51.3 us; read of 1000 rows 6.3 / 6.2 us, of 8000 rows 33.8 / 16.8 us.
// The rule goes by rows, not by heads or formats: fp16 would cross earlier.
bool by_tiles(const KvSeqs& b)
{
    return b.rows >= 800 && b.rows >= (int64_t)8 * b.batch && tiles_of(b) <= 65535;
}

template <typename Args>
cudaError_t launch_rows(void (*kernel)(Args), const Args& a, int64_t rows, int items, cudaStream_t stream)
{
    cudaLaunchConfig_t cfg = {};
    // A few rows are cut over several CTAs each, many rows take one: 256 single tokens of 8 kv heads of 128 and 32 query heads,
    // Q4_0, 10.1 us cut and 11.5 us whole, 400 rows 15.2 us and 12.6 us.
    const int per_row = rows >= 300 ? 1 : (items + 255) / 256;
    cfg.gridDim = dim3((unsigned)per_row, (unsigned)(rows < 65535 ? rows : 65535));
    cfg.blockDim = dim3(256);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

}  // namespace

cudaError_t launch_kv_append(const KvAppendArgs& a, cudaStream_t stream)
{
    const int items = (a.heads + 2 * a.pool.kv_heads) * a.pool.head_dim / 4;
    if (by_tiles(a.seqs)) {
        return a.pool.fmt == FMT_Q4_0   ? append_tiles_fmt<FMT_Q4_0>(a, stream)
               : a.pool.fmt == FMT_Q8_0 ? append_tiles_fmt<FMT_Q8_0>(a, stream)
                                        : append_tiles_fmt<KV_F16>(a, stream);
    }
    switch (a.pool.fmt) {
    case FMT_Q4_0: return launch_rows(kv_append_kernel<FMT_Q4_0>, a, a.seqs.rows, items, stream);
    case FMT_Q8_0: return launch_rows(kv_append_kernel<FMT_Q8_0>, a, a.seqs.rows, items, stream);
    default: return launch_rows(kv_append_kernel<KV_F16>, a, a.seqs.rows, items, stream);
    }
}

cudaError_t launch_kv_read(const KvReadArgs& a, cudaStream_t stream)
{
    const int items = 2 * a.pool.kv_heads * a.pool.head_dim / 4;
    if (by_tiles(a.seqs)) {
        return a.pool.fmt == FMT_Q4_0   ? read_tiles_fmt<FMT_Q4_0>(a, stream)
               : a.pool.fmt == FMT_Q8_0 ? read_tiles_fmt<FMT_Q8_0>(a, stream)
                                        : read_tiles_fmt<KV_F16>(a, stream);
    }
    switch (a.pool.fmt) {
    case FMT_Q4_0: return launch_rows(kv_read_kernel<FMT_Q4_0>, a, a.seqs.rows, items, stream);
    case FMT_Q8_0: return launch_rows(kv_read_kernel<FMT_Q8_0>, a, a.seqs.rows, items, stream);
    default: return launch_rows(kv_read_kernel<KV_F16>, a, a.seqs.rows, items, stream);
    }
}

}  // namespace qmm
