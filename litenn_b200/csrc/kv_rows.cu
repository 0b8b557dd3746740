// Attention over the paged cache for few query rows per key: single tokens, drafted tokens, fp32 prompts (include/litenn_kv.h).
//
//   out[r] = sum_t p_t v_t / sum_t p_t,  p_t = exp2(s_t - m),  s_t = log2(e) * scale * q_r . k_t,  m the running maximum
//
// Bound: the cached bytes, 144 per token and kv head of 128 dimensions in Q4_0.  The query heads of a kv head (and a
// sequence's rows) are columns, eight to a pass, so that one read of the cache serves a whole group of heads.
//
// A warp takes tiles of 16 tokens from a ring of its own that bulk copies fill, and multiplies them on the tensor cores
// (mma m16n8k16, fp16 operands, fp32 sums) as they lie in shared memory:
//   scores  A = queries, rows 0..7 the eight columns' upper fp16 parts, rows 8..15 their lower parts (22 bits together);
//           B = the tile's keys.  Quants go in as they are: a nibble n is the fp16 subnormal n * 2^-24, exact, one mask
//           instead of a conversion; "- 8" is the accumulator's start value, -8 times the block's sum of the query.  A block
//           of 32 dimensions is two MMAs, then its scale multiplies the sum in fp32.
//   values  A = probabilities times the value scales of the block, again in two fp16 parts; B = the values, whose "- 8" has to
//           be taken before the product here (a long flat attention averages thousands of values to nearly nothing, and a
//           subtraction behind the sum would leave only its rounding).
// The score's accumulator layout (row = column g, two tokens) is the probabilities' operand layout, so nothing is moved
// between lanes; running maxima cost two shuffles per tile.
//
// Work is cut evenly: the tiles of all (sequence, kv head, eight columns) follow one another in one list, and every CTA takes
// the same share of it, computed on the device from the lengths, so that ragged batches and single long sequences both fill
// the GPU and a captured launch follows the lengths.  Where a list entry spans CTAs, each leaves its part in the workspace and
// the last to arrive joins them, always in order.
#include <algorithm>

#include "kv_kernels.h"
#include "kv_rows_plan.cuh"

#include "../../include/litenn_kv.h"

namespace qmm {

namespace {

constexpr uint32_t SPIN_LIMIT = 1u << 22;
constexpr int COLS = KV_COLS;

__device__ __forceinline__ uint32_t smem_u32(const void* p)
{
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity)
{
    const uint32_t addr = smem_u32(bar);
    for (uint32_t spin = 0; spin < SPIN_LIMIT; ++spin) {
        uint32_t done;
        asm volatile(
            "{\n"
            ".reg .pred p;\n"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
            "selp.u32 %0, 1, 0, p;\n"
            "}\n"
            : "=r"(done)
            : "r"(addr), "r"(parity)
            : "memory");
        if (done) {
            return true;
        }
    }
    return false;
}
__device__ __forceinline__ void bulk_copy(void* dst, const void* src, uint32_t bytes, uint64_t* bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
                 "l"(src), "r"(bytes), "r"(smem_u32(bar))
                 : "memory");
}
// c += a (16 x 16, row) * b (16 x 8, col)
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t h2_bits(__half2 h)
{
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ __half2 as_h2(uint32_t u)
{
    return *reinterpret_cast<const __half2*>(&u);
}
__device__ __forceinline__ float exp2_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A lane's share of eight tokens: `L` bytes as vectors of kv_vec.
template <int FMT, int HD>
struct Share {
    static constexpr int L = kv_lane_bytes(FMT, HD), V = kv_vec(FMT, HD);
    uint32_t w[L / 4];
    __device__ __forceinline__ void load(const uint8_t* plane, int j, int lane)
    {
        const uint8_t* p = plane + j * 32 * L + lane * V;
#pragma unroll
        for (int i = 0; i < L / V; ++i) {
            if (V == 16) {
                const uint4 v = *reinterpret_cast<const uint4*>(p + i * 32 * V);
                w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
            } else if (V == 8) {
                const uint2 v = *reinterpret_cast<const uint2*>(p + i * 32 * V);
                w[2 * i] = v.x, w[2 * i + 1] = v.y;
            } else {
                w[i] = *reinterpret_cast<const uint32_t*>(p + i * 32 * V);
            }
        }
    }
};

// Scores take the stored codes as fp16 subnormals: the key values' operand registers (r = 0..3) of a block, and which dimension
// of the lane's eight each half holds.  A code's unit in register r is 2^-24 * KEY_STEP: the odd nibbles sit four bits higher,
// which their queries make up for.
template <int FMT>
__device__ __forceinline__ uint32_t key_operand(const uint32_t* w, int r)
{
    if (FMT == FMT_Q4_0) {
        const uint32_t x = r >= 2 ? w[0] >> 8 : w[0];
        return x & (r & 1 ? 0x00F000F0u : 0x000F000Fu);
    }
    if (FMT == FMT_Q8_0) {  // bytes 0, 2 and 1, 3 of a word
        return (r & 1 ? w[r >> 1] >> 8 : w[r >> 1]) & 0x00FF00FFu;
    }
    return w[r];
}
template <int FMT>
__host__ __device__ constexpr int key_dim(int r, int e)  // of the lane's eight dimensions
{
    return FMT == FMT_Q8_0 ? 4 * (r >> 1) + (r & 1) + 2 * e : 2 * r + e;
}
// Values as exact fp16: the operand register of dimension i (0..3) of a block, two tokens.
template <int FMT>
__device__ __forceinline__ uint32_t value_operand(const uint32_t* w, int i)
{
    if (FMT == FMT_Q4_0) {
        const uint32_t x = i >= 2 ? w[0] >> 8 : w[0];
        const uint32_t bits = (x & (i & 1 ? 0x00F000F0u : 0x000F000Fu)) | 0x64006400u;  // 1024 + n, or 1024 + 16 n
        return i & 1 ? h2_bits(__hfma2(as_h2(bits), as_h2(0x2C002C00u), as_h2(0xD480D480u)))  // / 16 - 72
                     : h2_bits(__hadd2(as_h2(bits), as_h2(0xE408E408u)));                      // - 1032
    }
    if (FMT == FMT_Q8_0) {
        const uint32_t bits = __byte_perm(w[i >> 1], 0x64646464u, i & 1 ? 0x4342u : 0x4140u);  // 1024 + (q + 128)
        return h2_bits(__hadd2(as_h2(bits), as_h2(0xE480E480u)));                              // - 1152
    }
    return w[i];
}

template <int FMT, int HD>
struct RowsShape {
    static constexpr int TILE = kv_tile_bytes(FMT, HD);
    static constexpr int WARPS = 4;
    // CTAs per SM, by the registers the accumulators take (HD / 2 of them)
    static constexpr int BY_REGISTERS = HD == 256 ? 1 : HD == 64 ? 4 : 3;
    static constexpr int DEPTH = TILE <= 2304 ? 4 : TILE <= 4608 ? 3 : 2;
    static constexpr int RING = WARPS * DEPTH * TILE;
    static constexpr int QFRAG = HD / 16 * 32 * 16;  // query operand registers
    static constexpr int PART = COLS * HD + 2 * COLS; // floats of one partial result: sums, maxima, totals
    static constexpr int MERGE = WARPS * PART * 4;
    static constexpr int SMEM = RING + QFRAG + MERGE + COLS * (HD / 32) * 4 + COLS * 4 + WARPS * DEPTH * 8 + 64 * 8;
    static constexpr int BY_SMEM = 228 * 1024 / (SMEM + 1024);
    static constexpr int CTAS = BY_REGISTERS < BY_SMEM ? BY_REGISTERS : BY_SMEM;
};

// Block-wide inclusive prefix sum of one value per thread.
template <int WARPS>
__device__ __forceinline__ long long block_scan(long long v, long long* sums)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xFFFFFFFFu, v, o);
        v += lane >= o ? u : 0;
    }
    __syncthreads();
    if (lane == 31) {
        sums[warp] = v;
    }
    __syncthreads();
    for (int i = 0; i < warp; ++i) {
        v += sums[i];
    }
    return v;
}

template <int FMT, int HD>
__global__ void __launch_bounds__(RowsShape<FMT, HD>::WARPS * 32, RowsShape<FMT, HD>::CTAS) kv_rows_kernel(const KvAttnArgs a)
{
    using Shape = RowsShape<FMT, HD>;
    constexpr int WARPS = Shape::WARPS, DEPTH = Shape::DEPTH, TILE = Shape::TILE, NB = HD / 32, PART = Shape::PART;
    constexpr int PLANE = kv_plane_bytes(FMT, HD), SCALES = kv_scale_bytes(FMT, HD), THREADS = WARPS * 32;
    constexpr bool QUANT = FMT != KV_F16;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t* ring = smem;
    uint32_t* qfrag = reinterpret_cast<uint32_t*>(ring + Shape::RING);             // [HD / 16][32 lanes][4]
    float* merge = reinterpret_cast<float*>(ring + Shape::RING + Shape::QFRAG);    // [WARPS][PART]
    float* qsum = merge + WARPS * PART;                                            // [COLS][NB]
    float* qscale = qsum + COLS * NB;                                              // [COLS]
    uint64_t* bars = reinterpret_cast<uint64_t*>(qscale + COLS);                   // [WARPS][DEPTH]
    long long* scan = reinterpret_cast<long long*>(bars + WARPS * DEPTH);          // [WARPS + 8]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;

    if (threadIdx.x < WARPS * DEPTH) {
        mbar_init(&bars[threadIdx.x], 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    __syncthreads();

    // ---- this CTA's share of the list of tiles ----
    long long total = 0;
    for (int base = 0; base < a.seqs.batch; base += THREADS) {
        const int s = base + threadIdx.x;
        bool bad = false;
        const long long w = s < a.seqs.batch ? seq_work(a.pool, a.seqs, a.group, a.window, s, bad).w : 0;
        if (bad && blockIdx.x == 0) {
            atomicExch(a.seqs.status, KV_BAD_ROWS);
        }
        const long long v = block_scan<WARPS>(w, scan);
        if (threadIdx.x == THREADS - 1) {
            scan[WARPS] = total + v;
        }
        __syncthreads();
        total = scan[WARPS];
        __syncthreads();
    }
    if (total == 0) {
        return;
    }
    const long long least = 2 * WARPS;  // tiles that a CTA is worth starting for
    const long long ctas = min((long long)gridDim.x, max(1LL, total / least));
    if (blockIdx.x >= ctas) {
        return;
    }
    const long long begin = share_begin(total, ctas, blockIdx.x), end = share_begin(total, ctas, blockIdx.x + 1);
    // the sequence that holds tile `begin` of the list
    if (threadIdx.x == 0) {
        scan[WARPS + 1] = -1;
    }
    long long before = 0;
    for (int base = 0; base < a.seqs.batch; base += THREADS) {
        const int s = base + threadIdx.x;
        bool bad;
        const long long w = s < a.seqs.batch ? seq_work(a.pool, a.seqs, a.group, a.window, s, bad).w : 0;
        const long long v = before + block_scan<WARPS>(w, scan);
        if (w > 0 && v - w <= begin && begin < v) {
            scan[WARPS + 1] = s;
            scan[WARPS + 2] = v - w;
        }
        if (threadIdx.x == THREADS - 1) {
            scan[WARPS] = v;
        }
        __syncthreads();
        before = scan[WARPS];
        const bool found = scan[WARPS + 1] >= 0;
        __syncthreads();
        if (found) {
            break;
        }
    }
    int seq = (int)scan[WARPS + 1];
    long long seq_first = scan[WARPS + 2];  // list index of the sequence's first tile
    bool bad;
    SeqWork x = seq_work(a.pool, a.seqs, a.group, a.window, seq, bad);

    uint64_t* my_bars = bars + warp * DEPTH;
    uint8_t* my_ring = ring + warp * DEPTH * TILE;
    uint32_t phases = 0;  // bit d: parity of the next completion of slot d
    bool late = false;
    unsigned int* counters = reinterpret_cast<unsigned int*>(a.workspace);                 // [gridDim.x]
    float* parts = reinterpret_cast<float*>(a.workspace + 16384);                           // [gridDim.x][2][PART]

    for (long long at = begin; at < end;) {
        while (at >= seq_first + x.w) {
            seq_first += x.w;
            ++seq;
            x = seq_work(a.pool, a.seqs, a.group, a.window, seq, bad);
        }
        // the list entry (kv head, pass) that holds tile `at`
        const long long entry = (at - seq_first) / x.tiles;
        const long long entry_first = seq_first + entry * x.tiles, entry_end = entry_first + x.tiles;
        const int head = (int)(entry / x.passes), pass = (int)(entry % x.passes);
        const long long here_end = min(end, entry_end);
        const PassView view = pass_view(x, a.group, a.window, pass, x.tile0 + (int)(at - entry_first),
                                        x.tile0 + (int)(here_end - entry_first));
        const int col0 = view.col0, cols = view.cols, pos_lo = view.pos_lo, pos_hi = view.pos_hi;
        const int seen_lo = view.seen_lo, all_lo = view.all_lo, tile_begin = view.tile_begin, tile_end = view.tile_end;
        const int first_pos = x.q.len - x.q.n;  // position of row 0
        const int my_tiles = tile_end - tile_begin > warp ? (tile_end - tile_begin - warp + WARPS - 1) / WARPS : 0;

        // ---- start the ring: page numbers of the next 32 tiles, one per lane ----
        auto page_of = [&](int i) -> int {  // of this warp's i-th tile
            return i < my_tiles ? kv_page(a.pool, a.seqs, seq, (tile_begin + warp + i * WARPS) * KV_TILE) : -1;
        };
        int pages = page_of(lane), pages_next = page_of(32 + lane);
        auto start_copy = [&](int i, int page) {  // lane 0
            const int slot = i % DEPTH, tile = tile_begin + warp + i * WARPS;
            if (page >= 0) {
                mbar_expect_tx(&my_bars[slot], TILE);
                bulk_copy(my_ring + slot * TILE, a.pool.base + kv_tile_index(a.pool, page, head, tile * KV_TILE) * TILE, TILE,
                          &my_bars[slot]);
            } else {
                atomicExch(a.seqs.status, KV_BAD_PAGE);
            }
        };
#pragma unroll
        for (int i = 0; i < DEPTH; ++i) {
            const int page = __shfl_sync(0xFFFFFFFFu, pages, i);
            if (lane == 0 && i < my_tiles && !late) {
                start_copy(i, page);
            }
        }

        // ---- queries: two fp16 parts of q * 2^e with the largest near 2^14, in operand order ----
        for (int c = warp; c < COLS; c += WARPS) {
            const bool on = c < cols;
            const int row = (col0 + c) / a.group, qh = head * a.group + (col0 + c) % a.group;
            const int64_t src = (x.q.row0 + (on ? row : 0)) * a.q_stride + (int64_t)(on ? qh : 0) * HD;
            float v[NB];
            float top = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const int64_t i = src + 32 * b + lane;
                v[b] = !on ? 0.0f
                       : a.q_type == QMM_OUT_F32 ? static_cast<const float*>(a.q)[i]
                                                 : __bfloat162float(static_cast<const __nv_bfloat16*>(a.q)[i]);
                top = fmaxf(top, fabsf(v[b]));
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
            }
            int e = 0;
            if (top > 0.0f && top < INFINITY) {
                e = max(-120, min(120, 14 - ilogbf(top)));
            }
            const float up = scalbnf(1.0f, e);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const float y = v[b] * up;
                const __half hi = __float2half_rn(y);
                const __half lo = __float2half_rn(y - __half2float(hi));
                float sum = __half2float(hi) + __half2float(lo);
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
                }
                if (lane == 0) {
                    qsum[c * NB + b] = sum;
                }
                // dimension 8 tt + d of the block is half ee of register rr in the lanes 4 c + tt
                const int tt = lane >> 3, d = lane & 7;
                const int rr = FMT == FMT_Q8_0 ? 2 * (d >> 2) + (d & 1) : d >> 1, ee = FMT == FMT_Q8_0 ? d >> 1 & 1 : d & 1;
                const bool high = FMT == FMT_Q4_0 && (rr & 1);  // the nibble above: 16 times the code
                __half* f = reinterpret_cast<__half*>(qfrag + ((2 * b + (rr >> 1)) * 32 + 4 * c + tt) * 4 + 2 * (rr & 1));
                f[ee] = high ? __hmul(hi, __float2half_rn(0.0625f)) : hi;
                f[2 + ee] = high ? __hmul(lo, __float2half_rn(0.0625f)) : lo;
            }
            if (lane == 0) {
                qscale[c] = a.scale * 1.44269504088896340736f * scalbnf(1.0f, -e) * (QUANT ? 16777216.0f : 1.0f);
            }
        }
        __syncthreads();
        uint32_t qf[HD <= 128 ? HD / 16 : 1][4];
        if (HD <= 128) {
#pragma unroll
            for (int i = 0; i < HD / 16; ++i) {
                const uint4 v = *reinterpret_cast<const uint4*>(qfrag + (i * 32 + lane) * 4);
                qf[i % (HD <= 128 ? HD / 16 : 1)][0] = v.x, qf[i % (HD <= 128 ? HD / 16 : 1)][1] = v.y;
                qf[i % (HD <= 128 ? HD / 16 : 1)][2] = v.z, qf[i % (HD <= 128 ? HD / 16 : 1)][3] = v.w;
            }
        }
        float start[QUANT ? NB : 1];
#pragma unroll
        for (int b = 0; b < (QUANT ? NB : 1); ++b) {
            start[b] = QUANT ? qsum[g * NB + b] * (FMT == FMT_Q4_0 ? -8.0f : -128.0f) * 0x1p-24f : 0.0f;
        }
        const float qs = qscale[g];
        const int my_pos = first_pos + (col0 + g) / a.group;  // of column g; columns past `cols` see what comes, unstored
        const int my_lo = a.window > 0 ? my_pos - a.window + 1 : 0;

        float m = -INFINITY, l = 0.0f, o[4 * NB][4] = {};
        float vs = 0.0f, limit = 0.0f;  // power of two that brings value scales near one; scales above `limit` lower it

        for (int i = 0; i < my_tiles; ++i) {
            const int slot = i % DEPTH, tile = tile_begin + warp + i * WARPS, tok0 = tile * KV_TILE;
            if ((i & 31) == 0 && i > 0) {
                pages = pages_next;
                pages_next = page_of(i + 32 + lane);
            }
            const int page_ahead = i + DEPTH < my_tiles ? __shfl_sync(0xFFFFFFFFu, ((i + DEPTH) >> 5) == (i >> 5) ? pages : pages_next, (i + DEPTH) & 31) : -1;
            const bool have = __shfl_sync(0xFFFFFFFFu, pages, i & 31) >= 0;
            if (have && !late) {
                late = !__all_sync(0xFFFFFFFFu, mbar_wait(&my_bars[slot], phases >> slot & 1u));
                phases ^= 1u << slot;
                if (late && lane == 0) {
                    atomicExch(a.seqs.status, KV_LATE_COPY);
                }
            }
            if (have && !late) {
                const uint8_t* base = my_ring + slot * TILE;
                const bool whole = tok0 >= all_lo && tok0 + KV_TILE - 1 <= pos_lo;

                // ---- scores ----
                float s[2][2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    Share<FMT, HD> k;
                    k.load(base, j, lane);
                    s[j][0] = s[j][1] = 0.0f;
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        const uint32_t* w = k.w + b * (kv_unit(FMT) / 4);
                        float c[4] = {QUANT ? start[b % (QUANT ? NB : 1)] : 0.0f, QUANT ? start[b % (QUANT ? NB : 1)] : 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            if (HD <= 128) {
                                const uint32_t* q = qf[(2 * b + h) % (HD <= 128 ? HD / 16 : 1)];
                                mma(c, q[0], q[1], q[2], q[3], key_operand<FMT>(w, 2 * h), key_operand<FMT>(w, 2 * h + 1));
                            } else {
                                const uint4 q = *reinterpret_cast<const uint4*>(qfrag + ((2 * b + h) * 32 + lane) * 4);
                                mma(c, q.x, q.y, q.z, q.w, key_operand<FMT>(w, 2 * h), key_operand<FMT>(w, 2 * h + 1));
                            }
                        }
                        if (QUANT) {
                            const float2 d = __half22float2(*reinterpret_cast<const __half2*>(base + PLANE + ((t * 2 + j) * NB + b) * 4));
                            s[j][0] += d.x * (c[0] + c[2]);
                            s[j][1] += d.y * (c[1] + c[3]);
                        } else {
                            s[j][0] += c[0] + c[2];
                            s[j][1] += c[1] + c[3];
                        }
                    }
                }
                uint32_t keep[2] = {0xFFFFFFFFu, 0xFFFFFFFFu};  // per half of a register: the column sees the token
#pragma unroll
                for (int j = 0; j < 2; ++j) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        s[j][e] *= qs;
                        if (!whole) {
                            const int pos = tok0 + 8 * j + 2 * t + e;
                            if (pos > my_pos || pos < my_lo) {
                                s[j][e] = -INFINITY;
                                keep[j] &= e ? 0x0000FFFFu : 0xFFFF0000u;
                            }
                        }
                    }
                }

                // ---- running maximum ----
                float top = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1]));
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
                const bool higher = top > m;
                if (__any_sync(0xFFFFFFFFu, higher)) {
                    const float down = higher ? exp2_fast(m - top) : 1.0f;  // 0 for the first
                    m = higher ? top : m;
                    l *= down;
#pragma unroll
                    for (int n = 0; n < 4 * NB; ++n) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            o[n][r] *= down;
                        }
                    }
                }
                const float ref = m == -INFINITY ? 0.0f : m;
                float p[2][2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        p[j][e] = exp2_fast(s[j][e] - ref);
                        l += p[j][e];
                    }
                }

                // ---- values ----
                const uint8_t* vbase = base + PLANE + SCALES;
                if (QUANT) {
                    // probabilities times scales stay within fp16: `vs` is set by the first tile's largest scale and lowered
                    // when a later one is 2^15 times as large, so what fp16 rounds away is relative to the largest values
                    uint32_t d[2][NB];
                    __half2 most = as_h2(0u);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
#pragma unroll
                        for (int b = 0; b < NB; ++b) {
                            d[j][b] = *reinterpret_cast<const uint32_t*>(vbase + PLANE + ((t * 2 + j) * NB + b) * 4) & keep[j];
                            most = __hmax2(most, __habs2(as_h2(d[j][b])));
                        }
                    }
                    const float largest = fmaxf(__low2float(most), __high2float(most));
                    if (__any_sync(0xFFFFFFFFu, largest > limit)) {
                        float all = largest;
#pragma unroll
                        for (int sh = 16; sh > 0; sh >>= 1) {
                            all = fmaxf(all, __shfl_xor_sync(0xFFFFFFFFu, all, sh));
                        }
                        const int e = max(-15, min(15, -ilogbf(fminf(all, 65504.0f))));
                        const float now = scalbnf(1.0f, e);
                        if (vs != 0.0f) {
                            const float down = now / vs;
#pragma unroll
                            for (int n = 0; n < 4 * NB; ++n) {
#pragma unroll
                                for (int r = 0; r < 4; ++r) {
                                    o[n][r] *= down;
                                }
                            }
                        }
                        vs = now;
                        limit = 0x1p15f / now;
                    }
                    __half2 ph[2], pl[2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float p0 = p[j][0] * vs, p1 = p[j][1] * vs;
                        ph[j] = __floats2half2_rn(p0, p1);
                        const float2 f = __half22float2(ph[j]);
                        pl[j] = __floats2half2_rn(p0 - f.x, p1 - f.y);
                    }
                    Share<FMT, HD> v0, v1;
                    v0.load(vbase, 0, lane);
                    v1.load(vbase, 1, lane);
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        uint32_t hi[2], lo[2];
#pragma unroll
                        for (int j = 0; j < 2; ++j) {  // the product's upper part, and what rounding it left over
                            const __half2 dd = as_h2(d[j][b]), up = __hmul2(ph[j], dd);
                            const __half2 rest = __hfma2(ph[j], dd, __hneg2(up));
                            hi[j] = h2_bits(up);
                            lo[j] = h2_bits(__hfma2(pl[j], dd, rest));
                        }
#pragma unroll
                        for (int n = 0; n < 4; ++n) {
                            mma(o[4 * b + n], hi[0], lo[0], hi[1], lo[1], value_operand<FMT>(v0.w + b * (kv_unit(FMT) / 4), n),
                                value_operand<FMT>(v1.w + b * (kv_unit(FMT) / 4), n));
                        }
                    }
                } else {
                    uint32_t hi[2], lo[2], all_see[2] = {0xFFFFFFFFu, 0xFFFFFFFFu};
                    if (!whole) {
                        // tokens that not every column sees are kept out of the product, whose operand all columns share
                        // (0 times an infinity), and added one by one to the columns that see them
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const int pos = tok0 + 8 * j + 2 * t + e;
                                if (pos > pos_lo || pos < all_lo) {
                                    all_see[j] &= e ? 0x0000FFFFu : 0xFFFF0000u;
                                }
                            }
                        }
                        for (int tok = 0; tok < KV_TILE; ++tok) {
                            const int pos = tok0 + tok;
                            if ((pos <= pos_lo && pos >= all_lo) || pos > pos_hi || pos < seen_lo) {
                                continue;
                            }
                            const int j = tok >> 3, tt = tok >> 1 & 3, e = tok & 1;
                            const float mine = j ? (e ? p[1][1] : p[1][0]) : (e ? p[0][1] : p[0][0]);
                            const float weight = __shfl_sync(0xFFFFFFFFu, mine, 4 * g + tt);
                            if (pos <= my_pos && pos >= my_lo) {
                                // accumulator column c of n-tile (b, n) is dimension 32 b + 4 c + n
#pragma unroll
                                for (int b = 0; b < NB; ++b) {
#pragma unroll
                                    for (int r = 0; r < 2; ++r) {
                                        const __half* v = reinterpret_cast<const __half*>(
                                            vbase + kv_place(FMT, HD, j, 4 * (2 * t + r) + tt, b, 0));
#pragma unroll
                                        for (int n = 0; n < 4; ++n) {
                                            o[4 * b + n][r] += weight * __half2float(v[2 * n + e]);
                                        }
                                    }
                                }
                            }
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const __half2 up = __floats2half2_rn(p[j][0], p[j][1]);
                        const float2 f = __half22float2(up);
                        hi[j] = h2_bits(up) & all_see[j];
                        lo[j] = h2_bits(__floats2half2_rn(p[j][0] - f.x, p[j][1] - f.y)) & all_see[j];
                    }
                    Share<FMT, HD> v0, v1;
                    v0.load(vbase, 0, lane);
                    v1.load(vbase, 1, lane);
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
#pragma unroll
                        for (int n = 0; n < 4; ++n) {
                            mma(o[4 * b + n], hi[0], lo[0], hi[1], lo[1],
                                value_operand<FMT>(v0.w + b * (kv_unit(FMT) / 4), n) & all_see[0],
                                value_operand<FMT>(v1.w + b * (kv_unit(FMT) / 4), n) & all_see[1]);
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0 && i + DEPTH < my_tiles && !late) {
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                start_copy(i + DEPTH, page_ahead);
            }
        }

        // ---- the warps' parts ----
        l += __shfl_xor_sync(0xFFFFFFFFu, l, 1);
        l += __shfl_xor_sync(0xFFFFFFFFu, l, 2);
        if (m == -INFINITY && l != l) {
            m = 0.0f;  // nothing but NaN: a part like any other
        }
        float* mine = merge + warp * PART;
        const float back = QUANT ? (vs == 0.0f ? 1.0f : 1.0f / vs) : 1.0f;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                float4 v;
                v.x = (o[4 * b][r] + o[4 * b][2 + r]) * back;
                v.y = (o[4 * b + 1][r] + o[4 * b + 1][2 + r]) * back;
                v.z = (o[4 * b + 2][r] + o[4 * b + 2][2 + r]) * back;
                v.w = (o[4 * b + 3][r] + o[4 * b + 3][2 + r]) * back;
                *reinterpret_cast<float4*>(mine + g * HD + 32 * b + 4 * (2 * t + r)) = v;
            }
        }
        if (t == 0) {
            mine[COLS * HD + g] = m;
            mine[COLS * HD + COLS + g] = l;
        }
        __syncthreads();
        const bool begins = entry_first >= begin, ends = entry_end <= end;
        float* part = parts + ((size_t)blockIdx.x * 2 + (begins ? 1 : 0)) * PART;
        auto store = [&](int c, int dim, float value) {
            if (c < cols) {
                const int row = (col0 + c) / a.group, qh = head * a.group + (col0 + c) % a.group;
                const int64_t at_out = (x.q.row0 + row) * a.out_stride + (int64_t)qh * HD + dim;
                if (a.out_type == QMM_OUT_F32) {
                    static_cast<float*>(a.out)[at_out] = value;
                } else {
                    static_cast<__nv_bfloat16*>(a.out)[at_out] = __float2bfloat16_rn(value);
                }
            }
        };
        for (int i = threadIdx.x; i < COLS * HD; i += THREADS) {
            const int c = i / HD;
            float top = -INFINITY, sum = 0.0f, all = 0.0f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                top = fmaxf(top, merge[w * PART + COLS * HD + c]);
            }
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float mw = merge[w * PART + COLS * HD + c];
                const float f = mw == -INFINITY ? 0.0f : exp2_fast(mw - top);
                if (mw != -INFINITY) {
                    sum += f * merge[w * PART + i];
                    all += f * merge[w * PART + COLS * HD + COLS + c];
                }
            }
            if (begins && ends) {
                store(c, i % HD, top == -INFINITY ? 0.0f : sum / all);
            } else {
                __stcg(part + i, sum);
                if (i % HD == 0) {
                    __stcg(part + COLS * HD + c, top);
                    __stcg(part + COLS * HD + COLS + c, all);
                }
            }
        }
        if (!(begins && ends)) {
            // CTAs c0 .. c1 hold a part each: the last to come joins them in order
            const long long c0 = share_of(total, ctas, entry_first), c1 = share_of(total, ctas, entry_end - 1);
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) {
                scan[WARPS + 3] = atomicInc(&counters[c0], (unsigned int)(c1 - c0)) == (unsigned int)(c1 - c0);
            }
            __syncthreads();
            if (scan[WARPS + 3]) {
                __threadfence();
                for (int i = threadIdx.x; i < COLS * HD; i += THREADS) {
                    const int c = i / HD;
                    float top = -INFINITY, sum = 0.0f, all = 0.0f;
                    for (long long k = c0; k <= c1; ++k) {
                        const float* from = parts + ((size_t)k * 2 + (k == c0 ? 1 : 0)) * PART;
                        const float mk = __ldcg(from + COLS * HD + c);
                        if (mk == -INFINITY) {
                            continue;
                        }
                        const float next = fmaxf(top, mk);
                        const float old = top == -INFINITY ? 0.0f : exp2_fast(top - next), f = exp2_fast(mk - next);
                        sum = sum * old + f * __ldcg(from + i);
                        all = all * old + f * __ldcg(from + COLS * HD + COLS + c);
                        top = next;
                    }
                    store(c, i % HD, top == -INFINITY ? 0.0f : sum / all);
                }
            }
        }
        __syncthreads();
        at = here_end;
    }
}

template <int FMT, int HD>
cudaError_t launch_rows(const KvAttnArgs& a, int sm_count, cudaStream_t stream)
{
    using Shape = RowsShape<FMT, HD>;
    auto kernel = kv_rows_kernel<FMT, HD>;
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) {
        return e;
    }
    static bool configured[64] = {};
    if (device < 0 || device >= 64 || !configured[device]) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::SMEM);
        if (e != cudaSuccess) {
            return e;
        }
        if (device >= 0 && device < 64) {
            configured[device] = true;
        }
    }
    // counters and two parts per CTA have to fit the workspace
    const int fit = (int)((QMM_KV_WORKSPACE_BYTES - 16384) / (2 * Shape::PART * 4));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)std::max(1, std::min({sm_count * Shape::CTAS, fit, 4096})));
    cfg.blockDim = dim3(Shape::WARPS * 32);
    cfg.dynamicSmemBytes = Shape::SMEM;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <int FMT>
cudaError_t launch_rows_fmt(const KvAttnArgs& a, int sm_count, cudaStream_t stream)
{
    switch (a.pool.head_dim) {
    case 64: return launch_rows<FMT, 64>(a, sm_count, stream);
    case 96: return launch_rows<FMT, 96>(a, sm_count, stream);
    case 128: return launch_rows<FMT, 128>(a, sm_count, stream);
    case 256: return launch_rows<FMT, 256>(a, sm_count, stream);
    default: return cudaErrorInvalidValue;
    }
}

}  // namespace

cudaError_t launch_kv_attention(const KvAttnArgs& a, int sm_count, cudaStream_t stream)
{
    switch (a.pool.fmt) {
    case FMT_Q4_0: return launch_rows_fmt<FMT_Q4_0>(a, sm_count, stream);
    case FMT_Q8_0: return launch_rows_fmt<FMT_Q8_0>(a, sm_count, stream);
    default: return launch_rows_fmt<KV_F16>(a, sm_count, stream);
    }
}

}  // namespace qmm
