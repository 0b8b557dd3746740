// Attention over the paged cache for few query rows per key: single tokens, drafted tokens, fp32 prompts (include/litenn_kv.h).
//
//   out[r] = sum_t p_t v_t / sum_t p_t,  p_t = exp2(s_t - m),  s_t = log2(e) * scale * q_r . k_t,  m near the running maximum
//
// Bound: the cached bytes, 144 per token and kv head of 128 dimensions in Q4_0.  The query heads of a kv head (and a
// sequence's rows) are columns, eight or sixteen to a pass, so that one read of the cache serves a whole group of heads.
//
// A warp takes tiles of 16 tokens from a ring of its own that bulk copies fill, and multiplies them on the tensor cores
// (mma m16n8k16, fp16 operands, fp32 sums) as they lie in shared memory:
//   scores  A = the tile's keys (rows = tokens), B = eight columns' queries in two fp16 parts (22 bits together), one after the
//           other into the same sums.  Quants go in as they are: a nibble n is the fp16 subnormal n * 2^-22, exact, a shift and
//           masks instead of conversions; "- 8" is the accumulator's start value, -8 times the block's sum of the query.  A
//           block of 32 dimensions is two k16 steps, then its scale multiplies the sum in fp32.
//   values  A = the values (rows = dimensions), whose "- 8" has to be taken before the product here (a long flat attention
//           averages thousands of values to nearly nothing, and a subtraction behind the sum would leave only its rounding);
//           B = probabilities times the block's value scales, again in two fp16 parts.
// Keys and values as A operands take half the accumulators of the other way round (queries' two parts as rows of A): 32
// registers of sums instead of 64 at 128 dimensions, so four CTAs share an SM instead of three.  What it costs are four 8 x 8
// transposes per tile that turn the scores' layout (row = token) into the probabilities' operand layout (row = column).
//
// What bounds it beside the bytes: instructions, about 415 a warp for a Q4_0 tile of 128 dimensions (57 % of the issue
// slots, 3.6 warps a scheduler), and what a call takes beside its tiles: 5 us where every entry is one CTA's, 12 to 15 where entries are
// shared (the lengths' scan 1.5, queries and pages 3, joining warps and CTAs 3 to 5).  One token, us: 131072 tokens of 8 kv heads of 128,
// 64 heads, in Q4_0 61 (2.5 TB/s; its copies alone 45), in Q8_0 80 (floor 44); 16 sequences of 700 to 8191 tokens in Q4_0 44, in Q8_0 53;
// 639 tokens of 32 kv heads 15; 16 sequences of 500 to 2000 tokens of 32 kv heads in fp16 64 (5.1 TB/s, 79 % of the copy rate); 8 sequences
// of 100 to 4000 tokens in Q8_0, 3 to 5 rows each of 32 heads, 28.  Prompts come here too where the prompt kernel does not take them
// (fp32 results, heads of 96 and 256), a pass over all their keys for every 8 or 16 columns: 1999 rows of 32 heads of 128 with fp32
// results 606 us, of 32 heads of 96 490, of 16 heads of 256 655, where the prompt kernel takes 83 for 128 dimensions.
//
// Work is cut evenly (kv_rows_plan.cuh) on the device, from the lengths, so that ragged batches and single long sequences both
// fill the GPU and a captured launch follows the lengths.  Where a list entry spans CTAs, each leaves its part in the workspace
// and the last to arrive joins them, always in order.
#include <algorithm>
#include <type_traits>

#include "kv_kernels.h"
#include "kv_rows_plan.cuh"

#include "../../include/litenn_kv.h"

namespace qmm {

namespace {

constexpr uint32_t SPIN_LIMIT = 1u << 22;
constexpr int JOIN = 8;  // parts that are loaded at once when a list entry's parts are joined
// Probabilities are taken as 2^4 .. 2^11 where the largest score lies: it may grow by SLACK before the sums are scaled down (every
// other tile brings one of eight columns a new maximum), and fp16 parts of small ones keep their bits.
constexpr float BIAS = 4.0f, SLACK = 7.0f;
constexpr float MOST_P = 16.0f;  // and are multiplied by this much at most: 2^15

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
// c = the product
__device__ __forceinline__ void mma_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
// 8 x 8 of fp16: lane 4g + t holds row g, columns 2t and 2t + 1, and gets row g of the transpose.
__device__ __forceinline__ uint32_t transpose8(uint32_t x)
{
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
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

// Packed pairs of fp32.
__device__ __forceinline__ float2 add2(float2 x, float2 y)
{
    float2 z;
    asm("{\n.reg .b64 a, b, c;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nadd.rn.f32x2 c, a, b;\nmov.b64 {%0, %1}, c;\n}"
        : "=f"(z.x), "=f"(z.y)
        : "f"(x.x), "f"(x.y), "f"(y.x), "f"(y.y));
    return z;
}
__device__ __forceinline__ float2 fma2(float2 x, float2 y, float2 w)
{
    float2 z;
    asm("{\n.reg .b64 a, b, c, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmov.b64 c, {%6, %7};\n"
        "fma.rn.f32x2 d, a, b, c;\nmov.b64 {%0, %1}, d;\n}"
        : "=f"(z.x), "=f"(z.y)
        : "f"(x.x), "f"(x.y), "f"(y.x), "f"(y.y), "f"(w.x), "f"(w.y));
    return z;
}

template <int BYTES>
__device__ __forceinline__ void load_words(uint32_t* w, const uint8_t* p)
{
    constexpr int V = BYTES % 16 == 0 ? 16 : BYTES % 8 == 0 ? 8 : 4;
#pragma unroll
    for (int i = 0; i < BYTES / V; ++i) {
        if (V == 16) {
            const uint4 v = *reinterpret_cast<const uint4*>(p + 16 * i);
            w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
        } else if (V == 8) {
            const uint2 v = *reinterpret_cast<const uint2*>(p + 8 * i);
            w[2 * i] = v.x, w[2 * i + 1] = v.y;
        } else {
            w[i] = *reinterpret_cast<const uint32_t*>(p + 4 * i);
        }
    }
}

// Scores take the stored codes as fp16 subnormals: the key values' operand registers (r = 0..3) of a block; a code counts
// KEY_UNIT in them, the odd nibbles 16 times that, which their queries make up for.  The tensor core aligns a product by the
// operands' exponent fields, so a subnormal's leading zeros are bits lost below: nibbles are brought up to bits 2..5 and 6..9
// of the fraction (at bits 0..3 and 4..7 the result of 640 tokens was off by 3.0e-6 of its norm instead of 8.8e-7).
template <int FMT>
constexpr float KEY_UNIT = FMT == FMT_Q4_0 ? 0x1p-22f : FMT == FMT_Q8_0 ? 0x1p-24f : 1.0f;
template <int FMT>
__device__ __forceinline__ uint32_t key_operand(const uint32_t* w, int r)
{
    if (FMT == FMT_Q4_0) {
        return (r >= 2 ? w[0] >> 6 : w[0] << 2) & (r & 1 ? 0x03C003C0u : 0x003C003Cu);
    }
    if (FMT == FMT_Q8_0) {  // bytes 0, 2 and 1, 3 of a word
        return (r & 1 ? w[r >> 1] >> 8 : w[r >> 1]) & 0x00FF00FFu;
    }
    return w[r];
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

template <int FMT, int HD, int NT>
struct RowsShape {
    static constexpr int COLS = 8 * NT;  // columns of a pass
    static constexpr int TILE = kv_tile_bytes(FMT, HD);
    static constexpr int WARPS = 4;
    // Tiles of a step.  Two halve what a step costs beside its products (one token, Q4_0, one / two: 131072 tokens of 8 kv heads of
    // 128 63.4 / 60.8 us, of 96 60.0 / 50.0 us, 8 drafts of 2000 tokens Q8_0 22.1 / 19.9 us; 64 sequences of 1000 tokens, whose warps
    // have a handful each, 45.3 / 49.3 us).  Where the sums take 64 registers one leaves room for more CTAs (16 columns of 64, 8
    // sequences of 2000 tokens, 26.6 / 31.8 us), and fp16 has no scales to share (64 dimensions, 131072 tokens 52.8 / 57.4 us).
    static constexpr int STEP = NT == 1 && HD <= 128 && FMT != KV_F16 ? 2 : 1;
    // CTAs per SM, by the registers the sums take (NT * HD / 4 of them); at four, with 128 registers a thread, the 128-wide Q4_0 form
    // spills 16 bytes, the 96-wide fp16 one 48
    static constexpr int BY_REGISTERS = NT * HD <= 128 ? 4 : NT * HD <= 256 ? 3 : 1;
    static constexpr int DEPTH = 2;  // steps in the ring; three were no faster (131072 tokens, 64/8 heads, Q4_0: 62.8 us, two 60.9)
    static constexpr int QFRAG = NT * HD / 16 * 32 * 16;  // query operand registers
    static constexpr int PART = COLS * HD + 2 * COLS;     // floats of one partial result: sums, maxima, totals
    static constexpr int WARP_RING = DEPTH * STEP * TILE > PART * 4 ? DEPTH * STEP * TILE : PART * 4;  // an entry's part lies over it
    static constexpr int RING = WARPS * WARP_RING;
    static constexpr int SMEM =
        RING + QFRAG + COLS * 4 + WARPS * DEPTH * 8 + (WARPS + 8) * 8 + (int)sizeof(SeqWork);
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

template <int FMT, int HD, int NT>
__global__ void __launch_bounds__(RowsShape<FMT, HD, NT>::WARPS * 32, RowsShape<FMT, HD, NT>::CTAS) kv_rows_kernel(const KvAttnArgs a)
{
    using Shape = RowsShape<FMT, HD, NT>;
    constexpr int COLS = Shape::COLS, WARPS = Shape::WARPS, DEPTH = Shape::DEPTH, TILE = Shape::TILE, STEP = Shape::STEP;
    constexpr int NB = HD / 32, PART = Shape::PART, THREADS = WARPS * 32;
    constexpr int PLANE = kv_plane_bytes(FMT, HD), SCALES = kv_scale_bytes(FMT, HD);
    constexpr bool QUANT = FMT != KV_F16;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t* ring = smem;
    uint32_t* qfrag = reinterpret_cast<uint32_t*>(ring + Shape::RING);             // [NT][HD / 16][32 lanes][4]
    float* merge = reinterpret_cast<float*>(ring);                                 // [WARPS][MERGE]
    constexpr int MERGE = Shape::WARP_RING / 4;
    float* qscale = reinterpret_cast<float*>(ring + Shape::RING + Shape::QFRAG);   // [COLS]
    uint64_t* bars = reinterpret_cast<uint64_t*>(qscale + COLS);                   // [WARPS][DEPTH]
    long long* scan = reinterpret_cast<long long*>(bars + WARPS * DEPTH);          // [WARPS + 8]
    SeqWork* found = reinterpret_cast<SeqWork*>(scan + WARPS + 8);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;

    if (threadIdx.x < WARPS * DEPTH) {
        mbar_init(&bars[threadIdx.x], 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    __syncthreads();

    // ---- this CTA's share of the list of tiles ----
    long long total = 0, w = 0, upto = 0;  // of the list; of this thread's sequence, and up to its end
    SeqWork x = {};
    bool bad = false;
    if (threadIdx.x == 0) {
        scan[WARPS + 1] = -1;
        scan[WARPS + 4] = 0;
    }
    for (int base = 0; base < a.seqs.batch; base += THREADS) {
        const int s = base + threadIdx.x;
        w = 0;
        bad = false;
        if (s < a.seqs.batch) {
            x = seq_work(a.pool, a.seqs, a.group, a.window, COLS, s, bad);
            w = x.units;
        }
        if (bad && blockIdx.x == 0) {
            atomicExch(a.seqs.status, KV_BAD_ROWS);
        }
        upto = total + block_scan<WARPS>(w, scan);
        if (s < a.seqs.batch && w > 0) {
            atomicAdd(reinterpret_cast<unsigned long long*>(&scan[WARPS + 4]), (unsigned long long)a.pool.kv_heads * x.passes);
        }
        if (threadIdx.x == THREADS - 1) {
            scan[WARPS] = upto;
        }
        __syncthreads();
        total = scan[WARPS];
        __syncthreads();
    }
    if (total == 0) {
        return;
    }
    const long long ctas = share_count(total, scan[WARPS + 4], gridDim.x);
    if (blockIdx.x >= ctas) {
        return;
    }
    const long long begin = share_begin(total, ctas, blockIdx.x), end = share_begin(total, ctas, blockIdx.x + 1);
    // the sequence that holds unit `begin` of the list
    long long before = 0;
    for (int base = 0; base < a.seqs.batch; base += THREADS) {
        const int s = base + threadIdx.x;
        if (a.seqs.batch > THREADS) {
            w = 0;
            if (s < a.seqs.batch) {
                x = seq_work(a.pool, a.seqs, a.group, a.window, COLS, s, bad);
                w = x.units;
            }
            upto = before + block_scan<WARPS>(w, scan);
        }
        if (w > 0 && upto - w <= begin && begin < upto) {
            scan[WARPS + 1] = s;
            scan[WARPS + 2] = upto - w;
            *found = x;
        }
        if (threadIdx.x == THREADS - 1) {
            scan[WARPS] = upto;
        }
        __syncthreads();
        before = scan[WARPS];
        if (scan[WARPS + 1] >= 0) {
            break;
        }
        __syncthreads();
    }
    int seq = (int)scan[WARPS + 1];
    long long seq_first = scan[WARPS + 2];  // where the sequence's units begin
    x = *found;

    uint64_t* my_bars = bars + warp * DEPTH;
    uint8_t* my_ring = ring + warp * Shape::WARP_RING;
    uint32_t phases = 0;  // bit d: parity of the next completion of slot d
    bool late = false;
    unsigned int* counters = reinterpret_cast<unsigned int*>(a.workspace);                 // [3][gridDim.x]
    float* parts = reinterpret_cast<float*>(a.workspace + KV_PARTS_AT);                         // [gridDim.x][2][PART]

    for (long long at = begin; at < end;) {
        while (at >= seq_first + x.units) {
            seq_first += x.units;
            ++seq;
            x = seq_work(a.pool, a.seqs, a.group, a.window, COLS, seq, bad);
        }
        // the entry (kv head, pass) that holds unit `at`; its tiles are the units from `entry_first` to `entry_end`
        const int each = x.tiles + KV_ENTRY_UNITS;
        const long long entry = kv_div(at - seq_first, each);
        const long long entry_first = seq_first + entry * each + KV_ENTRY_UNITS, entry_end = entry_first + x.tiles;
        const int head = (int)kv_div(entry, x.passes), pass = (int)(entry - (long long)head * x.passes);
        const long long here_first = max(at, entry_first), here_end = min(end, entry_end);
        at = min(end, entry_end);
        if (here_first >= here_end) {
            continue;
        }
        const PassView view = pass_view(x, a.group, a.window, COLS, pass, x.tile0 + (int)(here_first - entry_first),
                                        x.tile0 + (int)(here_end - entry_first));
        const int col0 = view.col0, cols = view.cols, pos_lo = view.pos_lo, pos_hi = view.pos_hi;
        const int seen_lo = view.seen_lo, all_lo = view.all_lo, tile_begin = view.tile_begin, tile_end = view.tile_end;
        const int first_pos = x.q.len - x.q.n;  // position of row 0
        // step i of this warp: the STEP tiles from tile_begin + (warp + i * WARPS) * STEP on
        const int all_steps = max(0, tile_end - tile_begin + STEP - 1) / STEP;
        const int my_steps = all_steps > warp ? (all_steps - warp + WARPS - 1) / WARPS : 0;

        // ---- queries of this warp's columns, loaded before anything waits ----
        constexpr int QC = COLS / WARPS;
        float qv[QC][NB];
#pragma unroll
        for (int n = 0; n < QC; ++n) {
            const int c = warp + n * WARPS;
            const bool on = c < cols;
            const int row = (col0 + c) / a.group, qh = head * a.group + (col0 + c) % a.group;
            const int64_t src = (x.q.row0 + (on ? row : 0)) * a.q_stride + (int64_t)(on ? qh : 0) * HD + lane;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                qv[n][b] = !on ? 0.0f
                           : a.q_type == QMM_OUT_F32 ? static_cast<const float*>(a.q)[src + 32 * b]
                                                     : __bfloat162float(static_cast<const __nv_bfloat16*>(a.q)[src + 32 * b]);
            }
        }

        // ---- start the ring: lane n holds where this warp's n-th tile lies (0: there is none), and its (32 + n)-th ----
        constexpr int AHEAD = 32 / STEP;  // steps whose places the lanes hold
        auto where = [&](int n) -> unsigned long long {
            const int tile = tile_begin + (warp + n / STEP * WARPS) * STEP + n % STEP;
            if (n >= my_steps * STEP || tile >= tile_end) {
                return 0;
            }
            const int page = kv_page(a.pool, a.seqs, seq, tile * KV_TILE);
            if (page < 0) {
                atomicExch(a.seqs.status, KV_BAD_PAGE);
                return 0;
            }
            return reinterpret_cast<unsigned long long>(a.pool.base + kv_tile_index(a.pool, page, head, tile * KV_TILE) * TILE);
        };
        unsigned long long place = where(lane), place_next = 0;
        unsigned int have_all = __ballot_sync(0xFFFFFFFFu, place != 0), have_next = 0;
        if (my_steps > AHEAD) {
            place_next = where(32 + lane);
            have_next = __ballot_sync(0xFFFFFFFFu, place_next != 0);
        }
        // step i, whose places are `at` and which has the tiles `have` (bits): the lanes that hold a place copy it
        auto start_step = [&](int i, unsigned long long at, unsigned int have) {
            const int first = i * STEP & 31, slot = i % DEPTH;
            if (lane == first && have != 0) {
                mbar_expect_tx(&my_bars[slot], TILE * (STEP == 2 && have == 3 ? 2 : 1));
            }
            __syncwarp();
            if ((lane & ~(STEP - 1)) == first && at != 0) {
                bulk_copy(my_ring + (slot * STEP + lane % STEP) * TILE, reinterpret_cast<const void*>(at), TILE, &my_bars[slot]);
            }
        };
#pragma unroll
        for (int i = 0; i < DEPTH; ++i) {
            if (i < my_steps && !late) {
                start_step(i, place, have_all >> (i * STEP & 31) & ((1u << STEP) - 1));
            }
        }

        // ---- queries: two fp16 parts of q * scale * log2(e) * 2^e with the largest near 2^14, in operand order.  With the scale in
        // them the scores' factor is a power of two: a score and its maximum times that factor are exact, however large, where
        // the roundings of other products would put whole powers of two between scores of 2^25 and their maximum ----
#pragma unroll
        for (int n = 0; n < QC; ++n) {
            const int c = warp + n * WARPS;
            float (&v)[NB] = qv[n];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                v[b] *= a.scale * 1.44269504088896340736f;
            }
            uint32_t bits = 0;  // magnitudes order as their bits; NaN above all
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                bits = max(bits, __float_as_uint(v[b]) & 0x7FFFFFFFu);
            }
            bits = __reduce_max_sync(0xFFFFFFFFu, bits);
            const int exponent = (int)(bits >> 23) - 127;  // of the largest, -127 for a subnormal
            const int e = bits == 0 || exponent == 128 ? 0 : max(-112, min(120, 14 - exponent));
            const float up = __uint_as_float((uint32_t)(e + 127) << 23);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const float y = v[b] * up;
                const __half hi = __float2half_rn(y);
                const __half lo = __float2half_rn(y - __half2float(hi));
                // dimension 8 tt + d of the block is half ee of register rr in the lanes 4 c + tt
                const int tt = lane >> 3, d = lane & 7;
                const int rr = FMT == FMT_Q8_0 ? 2 * (d >> 2) + (d & 1) : d >> 1, ee = FMT == FMT_Q8_0 ? d >> 1 & 1 : d & 1;
                const bool high = FMT == FMT_Q4_0 && (rr & 1);  // the nibble above: 16 times the code
                __half* f = reinterpret_cast<__half*>(
                    qfrag + (((c >> 3) * (HD / 16) + 2 * b + (rr >> 1)) * 32 + 4 * (c & 7) + tt) * 4 + 2 * (rr & 1));
                f[ee] = high ? __hmul(hi, __float2half_rn(0.0625f)) : hi;
                f[2 + ee] = high ? __hmul(lo, __float2half_rn(0.0625f)) : lo;
            }
            if (lane == 0) {
                qscale[c] = __uint_as_float((uint32_t)(127 - e) << 23) * (1.0f / KEY_UNIT<FMT>);
            }
        }
        __syncthreads();
        // -8 (-128) times the blocks' sums of the queries, as the products with keys of one
        float2 start[NT][QUANT ? NB : 1];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int b = 0; b < (QUANT ? NB : 1); ++b) {
                start[n][b] = make_float2(0.0f, 0.0f);
                if (QUANT) {
                    constexpr uint32_t ONE = 0x3C003C00u, HIGH = FMT == FMT_Q4_0 ? 0x4C004C00u : ONE;  // 1, 16
                    float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint4 q = *reinterpret_cast<const uint4*>(qfrag + ((n * (HD / 16) + 2 * b + h) * 32 + lane) * 4);
                        mma(c, ONE, ONE, HIGH, HIGH, q.x, q.z);
                        mma(c, ONE, ONE, HIGH, HIGH, q.y, q.w);
                    }
                    constexpr float OFF = (FMT == FMT_Q4_0 ? -8.0f : -128.0f) * KEY_UNIT<FMT>;
                    start[n][b] = make_float2(c[0] * OFF, c[1] * OFF);
                }
            }
        }
        // columns 2t and 2t + 1 are this lane's of the scores, column g of the probabilities as an operand
        float2 qs[NT], m[NT], l[NT];
        int pos_of[NT][2], op_pos[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            qs[n] = *reinterpret_cast<const float2*>(qscale + 8 * n + 2 * t);
            m[n] = make_float2(-INFINITY, -INFINITY);
            l[n] = make_float2(0.0f, 0.0f);
            // columns past `cols` see what comes, unstored; rows in front of the first token see nothing
            pos_of[n][0] = max(-1, first_pos + (col0 + 8 * n + 2 * t) / a.group);
            pos_of[n][1] = max(-1, first_pos + (col0 + 8 * n + 2 * t + 1) / a.group);
            op_pos[n] = max(-1, first_pos + (col0 + 8 * n + g) / a.group);
        }
        const int key_scale_at = kv_scale_place(HD, g, 0);  // of token g; token g + 8 and block b are a constant away
        const int reach = a.window > 0 ? a.window - 1 : 0x7FFFFFFF;  // a row at pos sees pos - reach .. pos
        float o[NT][HD / 16][4] = {};
        float vs = 0.0f;      // power of two that brings value scales near one; up to MOST_P of it goes into the probabilities
        uint32_t limit = 0;   // fp16 bits: scales above it lower vs
        constexpr int U = kv_unit(FMT), LANE = kv_lane_bytes(FMT, HD), VEC = kv_vec(FMT, HD), VB = VEC / U;  // blocks of a vector
        constexpr int BP = VB % 2 == 0 ? 2 : 1;                                                                 // and those multiplied in turn

        for (int i = 0; i < my_steps; ++i) {
            const int slot = i % DEPTH, step_tok0 = (tile_begin + (warp + i * WARPS) * STEP) * KV_TILE;
            if ((i & (AHEAD - 1)) == 0 && i > 0) {
                place = place_next;
                have_all = have_next;
                place_next = i + AHEAD < my_steps ? where((i + AHEAD) * STEP + lane) : 0ull;
                have_next = __ballot_sync(0xFFFFFFFFu, place_next != 0);
            }
            const unsigned int have = have_all >> (i * STEP & 31) & ((1u << STEP) - 1);
            if (have != 0 && !late) {
                late = !__all_sync(0xFFFFFFFFu, mbar_wait(&my_bars[slot], phases >> slot & 1u));
                if (late) {
                    // no copy is started from here on; those in flight (of this step and of the next ones) are waited for once
                    // more, so that they do not land in what the ring's place is used for
                    if (lane == 0) {
                        atomicExch(a.seqs.status, KV_LATE_COPY);
                    }
                    for (int k = 0; k < DEPTH && i + k < my_steps; ++k) {
                        const bool same = ((i + k) ^ i) < AHEAD;
                        if (((same ? have_all : have_next) >> ((i + k) * STEP & 31) & ((1u << STEP) - 1)) != 0) {
                            mbar_wait(&my_bars[(i + k) % DEPTH], phases >> ((i + k) % DEPTH) & 1u);
                        }
                    }
                }
                phases ^= 1u << slot;
            }
            // Two copies of what is done: whole steps, and single tiles, which pay for masks: those where columns differ in what
            // they see, and a last one that has no second.
            auto multiply = [&](auto whole, int first) {
                constexpr bool WHOLE = decltype(whole)::value;
                constexpr int N = WHOLE ? STEP : 1;
                const uint8_t* base = my_ring + (slot * STEP + first) * TILE;
                const int tok0 = step_tok0 + first * KV_TILE;

                // ---- scores: s[n][j] of token tok0 + 8 j + g and columns 2t, 2t + 1 ----
                float2 s[NT][2 * N];
#pragma unroll
                for (int u = 0; u < N; ++u) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        s[n][2 * u] = s[n][2 * u + 1] = make_float2(0.0f, 0.0f);
                    }
                }
#pragma unroll
                for (int vb = 0; vb < NB / VB; ++vb) {
                    uint32_t w[2 * N][VEC / 4];
#pragma unroll
                    for (int j = 0; j < 2 * N; ++j) {
                        load_words<VEC>(w[j], base + (j >> 1) * TILE + (j & 1) * 32 * LANE + vb * 32 * VEC + lane * VEC);
                    }
#pragma unroll
                    for (int b0 = 0; b0 < VB; b0 += BP) {
                        // BP * N * NT chains of four MMAs, in turn: an MMA's sum is ready for the next after about four others
                        float c[BP][NT][N][4];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            uint32_t k[BP][N][4];
                            uint4 q[BP][NT];
#pragma unroll
                            for (int bb = 0; bb < BP; ++bb) {
#pragma unroll
                                for (int u = 0; u < N; ++u) {
                                    const uint32_t *w0 = w[2 * u] + (b0 + bb) * (U / 4), *w1 = w[2 * u + 1] + (b0 + bb) * (U / 4);
                                    k[bb][u][0] = key_operand<FMT>(w0, 2 * h);
                                    k[bb][u][1] = key_operand<FMT>(w1, 2 * h);
                                    k[bb][u][2] = key_operand<FMT>(w0, 2 * h + 1);
                                    k[bb][u][3] = key_operand<FMT>(w1, 2 * h + 1);
                                }
#pragma unroll
                                for (int n = 0; n < NT; ++n) {
                                    q[bb][n] = *reinterpret_cast<const uint4*>(
                                        qfrag + ((n * (HD / 16) + 2 * (vb * VB + b0 + bb) + h) * 32 + lane) * 4);
                                }
                            }
#pragma unroll
                            for (int part = 0; part < 2; ++part) {
#pragma unroll
                                for (int bb = 0; bb < BP; ++bb) {
#pragma unroll
                                    for (int n = 0; n < NT; ++n) {
#pragma unroll
                                        for (int u = 0; u < N; ++u) {
                                            const uint32_t (&x)[4] = k[bb][u];
                                            const uint32_t q0 = part ? q[bb][n].y : q[bb][n].x, q1 = part ? q[bb][n].w : q[bb][n].z;
                                            if (h == 0 && part == 0) {
                                                mma_first(c[bb][n][u], x[0], x[1], x[2], x[3], q0, q1);
                                            } else {
                                                mma(c[bb][n][u], x[0], x[1], x[2], x[3], q0, q1);
                                            }
                                        }
                                    }
                                }
                            }
                        }
#pragma unroll
                        for (int bb = 0; bb < BP; ++bb) {
                            const int b = vb * VB + b0 + bb;
#pragma unroll
                            for (int u = 0; u < N; ++u) {
#pragma unroll
                                for (int j = 0; j < 2; ++j) {
                                    const float d = QUANT ? __half2float(*reinterpret_cast<const __half*>(
                                                                base + u * TILE + PLANE + kv_scale_place(HD, 8 * j, b) + key_scale_at))
                                                          : 0.0f;
#pragma unroll
                                    for (int n = 0; n < NT; ++n) {
                                        const float2 sum = make_float2(c[bb][n][u][2 * j], c[bb][n][u][2 * j + 1]);
                                        s[n][2 * u + j] = QUANT ? fma2(make_float2(d, d), add2(sum, start[n][b % (QUANT ? NB : 1)]), s[n][2 * u + j])
                                                                : add2(s[n][2 * u + j], sum);
                                    }
                                }
                            }
                        }
                    }
                }
                if (!WHOLE) {
#pragma unroll
                    for (int j = 0; j < 2 * N; ++j) {
                        const int pos = tok0 + 8 * j + g;
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            s[n][j].x = pos <= pos_of[n][0] && pos >= pos_of[n][0] - reach ? s[n][j].x : -INFINITY;
                            s[n][j].y = pos <= pos_of[n][1] && pos >= pos_of[n][1] - reach ? s[n][j].y : -INFINITY;
                        }
                    }
                }

                // ---- running maxima: m is BIAS to BIAS + SLACK below them ----
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float2 top = s[n][0];
#pragma unroll
                    for (int j = 1; j < 2 * N; ++j) {
                        top.x = fmaxf(top.x, s[n][j].x);
                        top.y = fmaxf(top.y, s[n][j].y);
                    }
#pragma unroll
                    for (int sh = 4; sh < 32; sh <<= 1) {
                        top.x = fmaxf(top.x, __shfl_xor_sync(0xFFFFFFFFu, top.x, sh));
                        top.y = fmaxf(top.y, __shfl_xor_sync(0xFFFFFFFFu, top.y, sh));
                    }
                    // rounded so that a probability stays below 2^(BIAS + SLACK) where these are lost in large sums
                    top.x = __fmaf_ru(top.x, qs[n].x, -BIAS);
                    top.y = __fmaf_ru(top.y, qs[n].y, -BIAS);
                    const bool higher0 = top.x > __fadd_rd(m[n].x, SLACK), higher1 = top.y > __fadd_rd(m[n].y, SLACK);
                    if (__any_sync(0xFFFFFFFFu, higher0 || higher1)) {
                        const float down0 = higher0 ? exp2_fast(m[n].x - top.x) : 1.0f;  // 0 for the first
                        const float down1 = higher1 ? exp2_fast(m[n].y - top.y) : 1.0f;
                        m[n].x = higher0 ? top.x : m[n].x;
                        m[n].y = higher1 ? top.y : m[n].y;
                        l[n].x *= down0;
                        l[n].y *= down1;
#pragma unroll
                        for (int mt = 0; mt < HD / 16; ++mt) {
                            o[n][mt][0] *= down0;
                            o[n][mt][1] *= down1;
                            o[n][mt][2] *= down0;
                            o[n][mt][3] *= down1;
                        }
                    }
                    const float2 ref = make_float2(m[n].x == -INFINITY ? 0.0f : -m[n].x, m[n].y == -INFINITY ? 0.0f : -m[n].y);
#pragma unroll
                    for (int j = 0; j < 2 * N; ++j) {  // s becomes the probabilities
                        const float2 x2 = fma2(s[n][j], qs[n], ref);
                        s[n][j] = make_float2(exp2_fast(x2.x), exp2_fast(x2.y));
                    }
                    if (!WHOLE) {
#pragma unroll
                        for (int j = 0; j < 2 * N; ++j) {  // also in a column that has seen nothing yet but NaN
                            const int pos = tok0 + 8 * j + g;
                            s[n][j].x = pos <= pos_of[n][0] && pos >= pos_of[n][0] - reach ? s[n][j].x : 0.0f;
                            s[n][j].y = pos <= pos_of[n][1] && pos >= pos_of[n][1] - reach ? s[n][j].y : 0.0f;
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 2 * N; ++j) {
                        l[n] = add2(l[n], s[n][j]);
                    }
                }

                // ---- values ----
#pragma unroll
                for (int u = 0; u < N; ++u) {
                    const uint8_t* vbase = base + u * TILE + PLANE + SCALES;
                    uint32_t all_see[2] = {0xFFFFFFFFu, 0xFFFFFFFFu};  // tokens that every column sees (fp16 caches)
                    uint32_t keep[NT][2];                              // tokens that column g sees (quants)
                    uint32_t d[QUANT ? 2 * NB : 1];                    // value scales of tokens 2t, 2t + 1
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        keep[n][0] = keep[n][1] = 0xFFFFFFFFu;
                    }
                    if (QUANT) {
                        // probabilities times scales stay within fp16: `vs` is set by the first tile's largest scale and
                        // lowered when a later one may be above `limit`, so what fp16 rounds away is relative to the largest.
                        // What of it the probabilities have no room for (scales below 2^-5) multiplies the scales, exactly: without
                        // that the second parts of small values lie below fp16's last bit (512 tokens of Q8_0 values of size 0.001
                        // were off by 2e-5 of their norm)
                        load_words<(QUANT ? 2 * NB : 1) * 4>(d, vbase + PLANE + t * 2 * NB * 4);
                        if (!WHOLE) {
                            uint32_t any[2] = {0, 0};
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                const int pos = tok0 + 16 * u + 8 * j + 2 * t;
#pragma unroll
                                for (int n = 0; n < NT; ++n) {
                                    keep[n][j] = (pos <= op_pos[n] && pos >= op_pos[n] - reach ? 0x0000FFFFu : 0u) |
                                                 (pos + 1 <= op_pos[n] && pos + 1 >= op_pos[n] - reach ? 0xFFFF0000u : 0u);
                                    any[j] |= keep[n][j];
                                }
                            }
#pragma unroll
                            for (int i2 = 0; i2 < 2 * NB; ++i2) {
                                d[i2 % (QUANT ? 2 * NB : 1)] &= any[i2 / NB];
                            }
                        }
                        uint32_t bits = 0;  // the scales' bits, joined: at least the largest
#pragma unroll
                        for (int i2 = 0; i2 < 2 * NB; ++i2) {
                            bits |= d[i2 % (QUANT ? 2 * NB : 1)];
                        }
                        bits &= 0x7FFF7FFFu;
                        if (__any_sync(0xFFFFFFFFu, (bits >> 16) > limit || (bits & 0xFFFFu) > limit)) {
                            __half2 most = __habs2(as_h2(d[0]));
#pragma unroll
                            for (int i2 = 1; i2 < 2 * NB; ++i2) {
                                most = __hmax2(most, __habs2(as_h2(d[i2 % (QUANT ? 2 * NB : 1)])));
                            }
                            float all = fmaxf(__low2float(most), __high2float(most));
#pragma unroll
                            for (int sh = 16; sh > 0; sh >>= 1) {
                                all = fmaxf(all, __shfl_xor_sync(0xFFFFFFFFu, all, sh));
                            }
                            // 2^11 of probability, 2^5 of room: the joined bits of scales of one size stay below it
                            const int e = max(-17, min(19, -1 - ilogbf(fmaxf(fminf(all, 65504.0f), 0x1p-24f))));
                            const float now = vs == 0.0f ? scalbnf(1.0f, e) : fminf(vs, scalbnf(1.0f, e + 4));
                            if (vs != 0.0f && now != vs) {
                                const float down = now / vs;
#pragma unroll
                                for (int n = 0; n < NT; ++n) {
#pragma unroll
                                    for (int mt = 0; mt < HD / 16; ++mt) {
#pragma unroll
                                        for (int r = 0; r < 4; ++r) {
                                            o[n][mt][r] *= down;
                                        }
                                    }
                                }
                            }
                            vs = now;
                            limit = __half_as_ushort(__float2half_rz(fminf(16.0f / now, 65504.0f)));
                        }
                        if (vs > MOST_P) {
                            const __half2 up = __float2half2_rn(vs * (1.0f / MOST_P));  // at most 2^15
#pragma unroll
                            for (int i2 = 0; i2 < 2 * NB; ++i2) {
                                uint32_t& w2 = d[i2 % (QUANT ? 2 * NB : 1)];
                                w2 = h2_bits(__hmul2(as_h2(w2), up));
                            }
                        }
                    } else if (!WHOLE) {
                        // tokens that not every column sees are kept out of the product, whose operand all columns share
                        // (0 times an infinity), and added one by one to the columns that see them
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const int pos = tok0 + 16 * u + 8 * j + 2 * t;
                            all_see[j] = (pos <= pos_lo && pos >= all_lo ? 0x0000FFFFu : 0u) |
                                         (pos + 1 <= pos_lo && pos + 1 >= all_lo ? 0xFFFF0000u : 0u);
                        }
                        for (int tok = 0; tok < KV_TILE; ++tok) {
                            const int pos = tok0 + 16 * u + tok;
                            if ((pos <= pos_lo && pos >= all_lo) || pos > pos_hi || pos < seen_lo) {
                                continue;
                            }
                            const int j = tok >> 3, tt = tok >> 1 & 3, e = tok & 1;
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                const float2 pj = j ? s[n][2 * u + 1] : s[n][2 * u];
                                const float w0 = __shfl_sync(0xFFFFFFFFu, pj.x, 4 * (tok & 7) + t);
                                const float w1 = __shfl_sync(0xFFFFFFFFu, pj.y, 4 * (tok & 7) + t);
                                const bool see0 = pos <= pos_of[n][0] && pos >= pos_of[n][0] - reach;
                                const bool see1 = pos <= pos_of[n][1] && pos >= pos_of[n][1] - reach;
#pragma unroll
                                for (int b = 0; b < NB; ++b) {
                                    const __half* v = reinterpret_cast<const __half*>(vbase + kv_place(FMT, HD, j, 4 * g + tt, b, 0));
#pragma unroll
                                    for (int i2 = 0; i2 < 4; ++i2) {
                                        const float value = __half2float(v[2 * i2 + e]);
                                        float (&sum)[4] = o[n][2 * b + (i2 >> 1)];
                                        sum[2 * (i2 & 1)] += see0 ? w0 * value : 0.0f;
                                        sum[2 * (i2 & 1) + 1] += see1 ? w1 * value : 0.0f;
                                    }
                                }
                            }
                        }
                    }
                    // two fp16 parts of the probabilities, then row = column g, tokens 2t and 2t + 1
                    __half2 ph[NT][2], pl[NT][2];
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const float in_p = fminf(vs, MOST_P);
                            const float2 pj = QUANT ? make_float2(s[n][2 * u + j].x * in_p, s[n][2 * u + j].y * in_p) : s[n][2 * u + j];
                            const __half2 up = __floats2half2_rn(pj.x, pj.y);
                            const float2 f = __half22float2(up);
                            ph[n][j] = as_h2(transpose8(h2_bits(up)) & (QUANT || WHOLE ? 0xFFFFFFFFu : all_see[j]));
                            pl[n][j] = as_h2(transpose8(h2_bits(__floats2half2_rn(pj.x - f.x, pj.y - f.y))) & (QUANT || WHOLE ? 0xFFFFFFFFu : all_see[j]));
                        }
                    }
#pragma unroll
                    for (int vb = 0; vb < NB / VB; ++vb) {
                        uint32_t w[2][VEC / 4];
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            load_words<VEC>(w[j], vbase + j * 32 * LANE + vb * 32 * VEC + lane * VEC);
                        }
#pragma unroll
                        for (int b0 = 0; b0 < VB; b0 += BP) {
                            uint32_t hi[BP][NT][2], lo[BP][NT][2], v[BP][2][4];
#pragma unroll
                            for (int bb = 0; bb < BP; ++bb) {
                                const int b = vb * VB + b0 + bb;
#pragma unroll
                                for (int n = 0; n < NT; ++n) {
#pragma unroll
                                    for (int j = 0; j < 2; ++j) {
                                        if (QUANT) {  // the product's upper part, and what rounding it left over
                                            __half2 dd = as_h2(d[(j * NB + b) % (QUANT ? 2 * NB : 1)]);
                                            if (!WHOLE) {
                                                dd = as_h2(h2_bits(dd) & keep[n][j]);  // a NaN stays with the columns that see it
                                            }
                                            const __half2 up = __hmul2(ph[n][j], dd);
                                            const __half2 rest = __hfma2(ph[n][j], dd, __hneg2(up));
                                            hi[bb][n][j] = h2_bits(up);
                                            lo[bb][n][j] = h2_bits(__hfma2(pl[n][j], dd, rest));
                                        } else {
                                            hi[bb][n][j] = h2_bits(ph[n][j]);
                                            lo[bb][n][j] = h2_bits(pl[n][j]);
                                        }
                                    }
                                }
#pragma unroll
                                for (int i2 = 0; i2 < 2; ++i2) {  // dimensions 32 b + 4 g + 2 i2 (rows g) and the next (rows g + 8)
#pragma unroll
                                    for (int k = 0; k < 4; ++k) {
                                        v[bb][i2][k] = value_operand<FMT>(w[k >> 1] + (b0 + bb) * (U / 4), 2 * i2 + (k & 1)) &
                                                       (QUANT || WHOLE ? 0xFFFFFFFFu : all_see[k >> 1]);
                                    }
                                }
                            }
#pragma unroll
                            for (int part = 0; part < 2; ++part) {
#pragma unroll
                                for (int bb = 0; bb < BP; ++bb) {
#pragma unroll
                                    for (int i2 = 0; i2 < 2; ++i2) {
#pragma unroll
                                        for (int n = 0; n < NT; ++n) {
                                            const uint32_t (&x)[4] = v[bb][i2], (&y)[2] = part ? lo[bb][n] : hi[bb][n];
                                            mma(o[n][2 * (vb * VB + b0 + bb) + i2], x[0], x[1], x[2], x[3], y[0], y[1]);
                                        }
                                    }
                                }
                            }
                        }
                    }
                }
            };
            if (have != 0 && !late) {
                if (have == (1u << STEP) - 1 && step_tok0 >= all_lo && step_tok0 + STEP * KV_TILE - 1 <= pos_lo) {
                    multiply(std::true_type{}, 0);
                } else {
#pragma unroll 1
                    for (int u = 0; u < STEP; ++u) {
                        if (have >> u & 1u) {
                            multiply(std::false_type{}, u);
                        }
                    }
                }
            }
            __syncwarp();
            if (i + DEPTH < my_steps && !late) {
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                const bool same = ((i + DEPTH) ^ i) < AHEAD;
                start_step(i + DEPTH, same ? place : place_next, (same ? have_all : have_next) >> ((i + DEPTH) * STEP & 31) & ((1u << STEP) - 1));
            }
        }

        // ---- the warps' parts ----
        float* mine = merge + warp * MERGE;
        const float back = QUANT ? (vs == 0.0f ? 1.0f : 1.0f / vs) : 1.0f;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int sh = 4; sh < 32; sh <<= 1) {
                l[n].x += __shfl_xor_sync(0xFFFFFFFFu, l[n].x, sh);
                l[n].y += __shfl_xor_sync(0xFFFFFFFFu, l[n].y, sh);
            }
            if (m[n].x == -INFINITY && l[n].x != l[n].x) {
                m[n].x = 0.0f;  // nothing but NaN: a part like any other
            }
            if (m[n].y == -INFINITY && l[n].y != l[n].y) {
                m[n].y = 0.0f;
            }
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const float (&x0)[4] = o[n][2 * b], (&x1)[4] = o[n][2 * b + 1];
                float* to = mine + (8 * n + 2 * t) * HD + 32 * b + 4 * g;
                *reinterpret_cast<float4*>(to) = make_float4(x0[0] * back, x0[2] * back, x1[0] * back, x1[2] * back);
                *reinterpret_cast<float4*>(to + HD) = make_float4(x0[1] * back, x0[3] * back, x1[1] * back, x1[3] * back);
            }
            if (g == 0) {
                *reinterpret_cast<float2*>(mine + COLS * HD + 8 * n + 2 * t) = m[n];
                *reinterpret_cast<float2*>(mine + COLS * HD + COLS + 8 * n + 2 * t) = l[n];
            }
        }
        __syncthreads();
        const bool begins = here_first == entry_first, ends = entry_end <= end;
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
        auto store4 = [&](int c, int dim, float4 v, float all, bool none) {
            store(c, dim, none ? 0.0f : v.x / all);
            store(c, dim + 1, none ? 0.0f : v.y / all);
            store(c, dim + 2, none ? 0.0f : v.z / all);
            store(c, dim + 3, none ? 0.0f : v.w / all);
        };
        for (int i = threadIdx.x * 4; i < COLS * HD; i += THREADS * 4) {
            const int c = i / HD;
            float mw[WARPS], top = -INFINITY, all = 0.0f;
            float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w2 = 0; w2 < WARPS; ++w2) {
                mw[w2] = merge[w2 * MERGE + COLS * HD + c];
                top = fmaxf(top, mw[w2]);
            }
#pragma unroll
            for (int w2 = 0; w2 < WARPS; ++w2) {
                if (mw[w2] != -INFINITY) {
                    const float f = exp2_fast(mw[w2] - top);
                    const float4 v = *reinterpret_cast<const float4*>(merge + w2 * MERGE + i);
                    sum.x += f * v.x, sum.y += f * v.y, sum.z += f * v.z, sum.w += f * v.w;
                    all += f * merge[w2 * MERGE + COLS * HD + COLS + c];
                }
            }
            if (begins && ends) {
                store4(c, i % HD, sum, all, top == -INFINITY);
            } else {
                __stcg(reinterpret_cast<float4*>(part + i), sum);
                if (i % HD == 0) {
                    __stcg(part + COLS * HD + c, top);
                    __stcg(part + COLS * HD + COLS + c, all);
                }
            }
        }
        if (!(begins && ends)) {
            // CTAs c0 .. c1 hold a part each.  The last to come of every JOIN of them joins theirs, the last of those the
            // joined ones, always in order
            const long long c0 = share_of(total, ctas, entry_first), c1 = share_of(total, ctas, entry_end - 1);
            const int all_parts = (int)(c1 - c0) + 1, mine_at = (int)(blockIdx.x - c0);
            const int group0 = mine_at / JOIN * JOIN, in_group = min(JOIN, all_parts - group0);
            const int groups = (all_parts + JOIN - 1) / JOIN;
            auto part_at = [&](int k) { return parts + ((size_t)(c0 + k) * 2 + (k == 0 ? 1 : 0)) * PART; };
            auto last_of = [&](unsigned int* counter, int n) {
                __syncthreads();
                if (threadIdx.x == 0) {  // releases the CTA's stores, acquires the others'
                    unsigned int old;
                    asm volatile("atom.acq_rel.gpu.global.inc.u32 %0, [%1], %2;" : "=r"(old) : "l"(counter), "r"(n - 1) : "memory");
                    scan[WARPS + 3] = old == (unsigned int)(n - 1);
                }
                __syncthreads();
                return scan[WARPS + 3] != 0;
            };
            // sum of n parts, `step` apart: the result, or a part again
            auto join = [&](int first, int n, int step, bool result) {
                constexpr int UNITS = (COLS * HD / 4 + THREADS - 1) / THREADS;
                float4 sum[UNITS];
                float top[UNITS], all[UNITS];
#pragma unroll
                for (int u = 0; u < UNITS; ++u) {
                    sum[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    top[u] = -INFINITY;
                    all[u] = 0.0f;
                }
                for (int at_part = 0; at_part < n; at_part += JOIN) {
#pragma unroll
                    for (int u = 0; u < UNITS; ++u) {
                        const int i = min((int)threadIdx.x + u * THREADS, COLS * HD / 4 - 1) * 4, c = i / HD;
                        float4 v[JOIN];
                        float mk[JOIN], lk[JOIN];
#pragma unroll
                        for (int k = 0; k < JOIN; ++k) {
                            const float* from = part_at(first + min(at_part + k, n - 1) * step);
                            v[k] = __ldcg(reinterpret_cast<const float4*>(from + i));
                            mk[k] = at_part + k < n ? __ldcg(from + COLS * HD + c) : -INFINITY;
                            lk[k] = __ldcg(from + COLS * HD + COLS + c);
                        }
                        float next = top[u];
#pragma unroll
                        for (int k = 0; k < JOIN; ++k) {
                            next = fmaxf(next, mk[k]);
                        }
                        const float old = top[u] == -INFINITY ? 0.0f : exp2_fast(top[u] - next);
                        sum[u].x *= old, sum[u].y *= old, sum[u].z *= old, sum[u].w *= old;
                        all[u] *= old;
                        top[u] = next;
#pragma unroll
                        for (int k = 0; k < JOIN; ++k) {
                            if (mk[k] != -INFINITY) {
                                const float f = exp2_fast(mk[k] - next);
                                sum[u].x += f * v[k].x, sum[u].y += f * v[k].y, sum[u].z += f * v[k].z, sum[u].w += f * v[k].w;
                                all[u] += f * lk[k];
                            }
                        }
                    }
                }
                __syncthreads();  // every part has been read: the first one's place takes the sum
                float* to = part_at(first);
#pragma unroll
                for (int u = 0; u < UNITS; ++u) {
                    const int i = ((int)threadIdx.x + u * THREADS) * 4, c = i / HD;
                    if (i >= COLS * HD) {
                        continue;
                    }
                    if (result) {
                        store4(c, i % HD, sum[u], all[u], top[u] == -INFINITY);
                    } else {
                        __stcg(reinterpret_cast<float4*>(to + i), sum[u]);
                        if (i % HD == 0) {
                            __stcg(to + COLS * HD + c, top[u]);
                            __stcg(to + COLS * HD + COLS + c, all[u]);
                        }
                    }
                }
            };
            if (last_of(&counters[2 * (c0 + group0) + (group0 == 0 ? 1 : 0)], in_group)) {
                join(group0, in_group, 1, groups == 1);
                if (groups > 1 && last_of(&counters[2 * (int)gridDim.x + (int)c0], groups)) {
                    join(0, groups, JOIN, true);
                }
            }
        }
        // the rings' next copies come after everything that was written over them
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();
    }
}

template <int FMT, int HD, int NT>
cudaError_t launch_rows(const KvAttnArgs& a, int sm_count, cudaStream_t stream)
{
    using Shape = RowsShape<FMT, HD, NT>;
    auto kernel = kv_rows_kernel<FMT, HD, NT>;
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
    // three counters and two parts per CTA have to fit the workspace
    const int fit = (int)((QMM_KV_WORKSPACE_BYTES - KV_PARTS_AT) / (2 * Shape::PART * 4));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)std::max(1, std::min({sm_count * Shape::CTAS, fit, KV_COUNTER_BYTES / 12})));
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
    // Sixteen columns to a pass where sequences have many, else eight: those leave registers for four CTAs an SM instead of three,
    // which carries even two passes over the same keys.  8 sequences of 2000 tokens of 8 kv heads of 128, eight / sixteen: Q4_0 with 8
    // columns each 24.7 / 30.0 us, 16 28.0 / 30.8 us, 32 43.5 / 41.0 us, 64 69.2 / 62.6 us; Q8_0 with 16 25.5 / 30.0 us, 64 62.9 / 62.2 us.
    // At 256 dimensions sixteen leave one CTA and take twice eight's time (16 sequences of 2000 tokens, Q4_0, 92 and 42 us).
    const bool wide = a.seqs.rows * a.group >= (int64_t)32 * a.seqs.batch;
    switch (a.pool.head_dim) {
    case 64: return wide ? launch_rows<FMT, 64, 2>(a, sm_count, stream) : launch_rows<FMT, 64, 1>(a, sm_count, stream);
    case 96: return wide ? launch_rows<FMT, 96, 2>(a, sm_count, stream) : launch_rows<FMT, 96, 1>(a, sm_count, stream);
    case 128: return wide ? launch_rows<FMT, 128, 2>(a, sm_count, stream) : launch_rows<FMT, 128, 1>(a, sm_count, stream);
    case 256: return launch_rows<FMT, 256, 1>(a, sm_count, stream);
    default: return cudaErrorInvalidValue;
    }
}

}  // namespace

cudaError_t launch_kv_rows(const KvAttnArgs& a, int sm_count, cudaStream_t stream)
{
    switch (a.pool.fmt) {
    case FMT_Q4_0: return launch_rows_fmt<FMT_Q4_0>(a, sm_count, stream);
    case FMT_Q8_0: return launch_rows_fmt<FMT_Q8_0>(a, sm_count, stream);
    default: return launch_rows_fmt<KV_F16>(a, sm_count, stream);
    }
}

}  // namespace qmm
