// Attention of prompts over the paged cache on the 5th-generation tensor cores (include/litenn_kv.h), bf16 results.
//
// A CTA takes 256 columns of a kv head (query heads of its group, times rows) as two M tiles of 128, and walks the keys in
// blocks of 128.  Per block and M tile:
//   S = Q K^T   tcgen05.mma, both operands fp16 in shared memory, S fp32 in TMEM
//   P           one thread per column: running maximum, exp2, sum; P in fp16 over S's own TMEM columns
//   O += P V    tcgen05.mma, P from TMEM, V^T from shared memory, O fp32 in TMEM
// Warps: 4 per M tile for the softmax (a warp reaches 32 TMEM lanes), 8 that bring keys and values (a tile of 16 tokens each,
// from the cache to fp16 in swizzled shared memory, two stages), one that issues the MMAs.  While one M tile's softmax runs, the
// tensor core works for the other.
//
// Bound: the chain of a block.  A column's softmax takes about 3000 cycles of 128 keys (128 exponentials and maxima of one thread,
// TMEM loads between them), the two products 1700, and with two M tiles in turn a block takes 2.5 us.  512 rows of 64 heads (8 kv heads of
// 128, Q4_0) behind 16384 tokens: 347 us, 804 TFLOP/s, 50 % of the measured dense peak.  1999 rows of 32 heads from the start: 83 us;
// an item costs 8 us beside its blocks (queries 4, results 2, first keys 2) and has 9 of them on average.  Nothing splits the keys of an
// item: 64 rows of 64 heads behind 131072 tokens are 16 items, 1024 blocks each, and take 2.5 ms (floor 0.17).
// Tried and slower (the first of the two cases): blocks of 64 keys with two score buffers 471 us where 128 took 358; one warp fewer for
// keys and values, the tiles dealt in turn, 460; a softmax in one pass over chunks with a running maximum 452.
//
// Numerics: queries are brought to fp16 by a power of two per row, keys and values are the cache's q * scale rounded to fp16
// once, probabilities are fp16 relative to a maximum that may lag 2^8 behind (O is scaled only when it grows by more).  Each of
// the four roundings is up to 2^-11 of its value where the bf16 result's own is up to 2^-8; probabilities below 2^-21 of the
// largest are off by up to 2^-32.75 of it.  Sums are fp32.  A value that is not finite would reach every column of the product
// (0 times infinity): it enters as 0, and its dimension is made NaN in the columns that see its token.
#include <algorithm>
#include <type_traits>

#include "kv_kernels.h"
#include "kv_rows_plan.cuh"
#include "qmm_gemm_ptx.cuh"

#include "../../include/litenn_kv.h"

namespace qmm {

namespace {

constexpr int BLOCK = 128;                     // keys per block
constexpr int M_TILE = 128, COLS = 2 * M_TILE; // columns of an M tile, of a CTA
constexpr int KV_TILES = BLOCK / KV_TILE;       // tiles of a block
constexpr int SOFT_WARPS = 8, KV_WARPS = KV_TILES;
constexpr int THREADS = (SOFT_WARPS + KV_WARPS + 1) * 32;
constexpr uint32_t TMEM_COLS = 512;            // S0, S1, O0, O1
constexpr int KV_LATE_PROMPT = 24;             // a bounded wait ran out
// Probabilities are taken as 2^BIAS where the reference maximum lies, which may lag SLACK powers of two behind: below 2^15.8 in fp16,
// whose bits end at 2^-24.  Without a bias a long tail 2^-20 of the largest key and below came out as multiples of 2^-24: 3000
// equal keys 2^-20.6 below a key of value 0 gave a result that was off by 4 %, 2^-24.4 below by 32 %.  A shorter lag would leave
// room for more bits, and scales the sums more often: 512 rows behind 16384 tokens 341 us, with 2^6 348 us.
constexpr float BIAS = 7.75f, SLACK = 8.0f;

// A maximum (times its factor) whose rounding is not small beside BIAS and SLACK: of a score of 2^25 and its maximum the roundings
// of the products are whole powers of two apart.  Such a column's scores lose the maximum before the factor.
constexpr float FAR = 65536.0f;
__device__ __forceinline__ bool is_far(float m)
{
    return fabsf(m) > FAR && m != -INFINITY;
}

template <int FMT, int HD>
struct PromptShape {
    static constexpr int PANELS = HD / 64;                     // 64 dimensions: a 128-byte swizzle row
    static constexpr int Q_BYTES = PANELS * M_TILE * 128;      // of an M tile
    static constexpr int K_BYTES = PANELS * BLOCK * 128;       // of a stage
    static constexpr int V_BYTES = BLOCK / 64 * HD * 128;
    static constexpr int CONTROL = 8192;                       // barriers and what the warps tell one another
    static constexpr int SMEM = 1024 + CONTROL + 2 * Q_BYTES + 2 * K_BYTES + 2 * V_BYTES;
};

// What a CTA works on: 256 columns of a kv head of a sequence.
struct Item {
    KvSeq q;
    int seq, head;
    int col0, cols;       // of the sequence's columns
    int first_pos;        // of row 0
    int k0;               // first key, a multiple of 16
    int blocks[2], most;  // of each M tile
    int pos_hi, seen_lo;  // keys that some column sees
};

struct Control {
    uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2][2], o_full, drained;  // probabilities: of either half of the keys
    uint32_t tmem;
    Item item[2];                  // the one that is worked on and the next; seq < 0: there is none
    int late;
    uint32_t poison[8][KV_TILES];  // of the last blocks, per tile: tokens whose value is not finite
    float q_scale[COLS];
    float far_max[COLS];           // the running maximum before its factor, where that is past 2^16
    uint32_t odd[4][COLS];         // dimensions in which a column sees a value that is not finite: bit d of word n is 32 n + d
};

// Instruction descriptor: D fp32, A and B fp16, both K-major, M = 128, N = n.
__device__ __forceinline__ uint32_t idesc_f16(int n)
{
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(M_TILE >> 4) << 24);
}
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add)
{
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
        : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add)
{
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
        "}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
        : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, float (&r)[16])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
        : "r"(addr)
        : "memory");
}
// The loads have come; `r` is named so that nothing reads it earlier.
__device__ __forceinline__ void tmem_wait_ld(float (&r)[16])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]), "+f"(r[8]), "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const float (&r)[16])
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
        "f"(r[0]), "f"(r[1]), "f"(r[2]), "f"(r[3]), "f"(r[4]), "f"(r[5]), "f"(r[6]), "f"(r[7]), "f"(r[8]), "f"(r[9]), "f"(r[10]), "f"(r[11]), "f"(r[12]), "f"(r[13]), "f"(r[14]), "f"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t (&r)[8])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_st()
{
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void fence_before()
{
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_after()
{
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ float exp2_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Packed pairs of fp32, and the largest of three.
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
__device__ __forceinline__ float max3(float x, float y, float z)
{
    float m;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(x), "f"(y), "f"(z));
    return m;
}
// Four 8 x 8 matrices of fp16, rows of 16 bytes: lane 4g + t holds row g, columns 2t and 2t + 1 of each, lane 8m + r names the
// place of row r of matrix m.
__device__ __forceinline__ void store_matrices(void* row, const uint32_t (&x)[4])
{
    asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(g_smem_u32(row)), "r"(x[0]), "r"(x[1]),
                 "r"(x[2]), "r"(x[3])
                 : "memory");
}
__device__ __forceinline__ uint32_t h2_bits(__half2 h)
{
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ __half2 as_h2(uint32_t u)
{
    return *reinterpret_cast<const __half2*>(&u);
}
// Four pairs of a word's (two words', four words') values as exact fp16 quants, in storage order (kv_layout.cuh).
template <int FMT>
__device__ __forceinline__ void quants(const uint32_t* w, uint32_t (&v)[4])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (FMT == FMT_Q4_0) {
            const uint32_t x = i >= 2 ? w[0] >> 8 : w[0];
            const uint32_t bits = (x & (i & 1 ? 0x00F000F0u : 0x000F000Fu)) | 0x64006400u;  // 1024 + n, or 1024 + 16 n
            v[i] = i & 1 ? h2_bits(__hfma2(as_h2(bits), as_h2(0x2C002C00u), as_h2(0xD480D480u)))  // / 16 - 72
                         : h2_bits(__hadd2(as_h2(bits), as_h2(0xE408E408u)));                      // - 1032
        } else if (FMT == FMT_Q8_0) {
            const uint32_t bits = __byte_perm(w[i >> 1], 0x64646464u, i & 1 ? 0x4342u : 0x4140u);  // 1024 + (q + 128)
            v[i] = h2_bits(__hadd2(as_h2(bits), as_h2(0xE480E480u)));                              // - 1152
        } else {
            v[i] = w[i];
        }
    }
}
// Two fp16, those that are not finite made 0.
__device__ __forceinline__ uint32_t finite_or_0(uint32_t x)
{
    return ((x & 0x7C00u) == 0x7C00u ? 0u : x & 0xFFFFu) | ((x & 0x7C000000u) == 0x7C000000u ? 0u : x & 0xFFFF0000u);
}
// Volatile: the loads are issued where they stand (as plain ones they were moved down to their uses, a block later).
template <int BYTES>
__device__ __forceinline__ void load_words(uint32_t* w, const uint8_t* p)
{
    if (BYTES == 16) {
        asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(p));
    } else {
        asm volatile("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
    }
}

template <int FMT, int HD>
__global__ void __launch_bounds__(THREADS, 1) kv_prompt_kernel(const KvAttnArgs a)
{
    using Shape = PromptShape<FMT, HD>;
    constexpr int NB = HD / 32, TILE = kv_tile_bytes(FMT, HD), PLANE = kv_plane_bytes(FMT, HD), SCALES = kv_scale_bytes(FMT, HD);
    constexpr int U = kv_unit(FMT), LANE = kv_lane_bytes(FMT, HD), VEC = kv_vec(FMT, HD);
    constexpr bool QUANT = FMT != KV_F16;
    extern __shared__ uint8_t prompt_smem[];
    uint8_t* smem = prompt_smem + ((1024u - (g_smem_u32(prompt_smem) & 1023u)) & 1023u);
    Control& ctl = *reinterpret_cast<Control*>(smem);
    static_assert(sizeof(Control) <= Shape::CONTROL, "control block");
    uint8_t* q_smem = smem + Shape::CONTROL;                 // [2 M tiles][panels][128 columns][128 B]
    uint8_t* k_smem = q_smem + 2 * Shape::Q_BYTES;           // [2 stages][panels][128 keys][128 B]
    uint8_t* v_smem = k_smem + 2 * Shape::K_BYTES;           // [2 stages][2 halves of the keys][HD rows][128 B]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool mma_warp = warp == SOFT_WARPS + KV_WARPS;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            g_mbar_init(&ctl.k_full[i], KV_WARPS);
            g_mbar_init(&ctl.v_full[i], KV_WARPS);
            g_mbar_init(&ctl.k_empty[i], 1);
            g_mbar_init(&ctl.v_empty[i], 1);
            g_mbar_init(&ctl.s_full[i], 1);
            g_mbar_init(&ctl.p_full[i][0], 4);
            g_mbar_init(&ctl.p_full[i][1], 4);
        }
        g_mbar_init(&ctl.o_full, 1);
        g_mbar_init(&ctl.drained, 1);
        ctl.late = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (mma_warp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(g_smem_u32(&ctl.tmem)), "r"(TMEM_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = ctl.tmem;
    g_pdl_launch_dependents();
    g_pdl_wait();

    unsigned int* next_item = reinterpret_cast<unsigned int*>(a.workspace + KV_COUNTER_BYTES);
    unsigned int* done_ctas = next_item + 1;
    uint32_t blocks_before = 0, before0 = 0, before1 = 0, items_before = 0;  // completed: the barriers' parities
    auto give_up = [&]() {
        atomicExch(a.seqs.status, KV_LATE_PROMPT);
        *reinterpret_cast<volatile int*>(&ctl.late) = 1;
    };

    // The next item, for the warp that issues MMAs: heavy ones (late columns) of a sequence first, its kv heads side by side.
    auto fetch = [&](Item& to, bool first) {
        unsigned int want = blockIdx.x;
        if (!first) {
            if (lane == 0) {
                want = gridDim.x + atomicAdd(next_item, 1u);
            }
            want = __shfl_sync(0xFFFFFFFFu, want, 0);
        }
        long long before = 0;
        int seq = -1, local = 0;
        for (int base = 0; base < a.seqs.batch && seq < 0; base += 32) {
            const int s = base + lane;
            bool bad = false;
            long long n = 0;
            if (s < a.seqs.batch) {
                const KvSeq q = kv_seq(a.pool, a.seqs, s, bad);
                n = ((long long)q.n * a.group + COLS - 1) / COLS * a.pool.kv_heads;
            }
            if (bad) {  // the fetch that finds no item has seen every sequence
                atomicExch(a.seqs.status, KV_BAD_ROWS);
            }
            long long upto = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long u = __shfl_up_sync(0xFFFFFFFFu, upto, o);
                upto += lane >= o ? u : 0;
            }
            const bool mine = n > 0 && before + upto - n <= want && want < before + upto;
            const unsigned int who = __ballot_sync(0xFFFFFFFFu, mine);
            if (who != 0) {
                const int from = __ffs(who) - 1;
                seq = base + from;
                local = (int)(want - (before + __shfl_sync(0xFFFFFFFFu, upto - n, from)));
            }
            before += __shfl_sync(0xFFFFFFFFu, upto, 31);
        }
        if (lane == 0) {
            Item n = {};
            n.seq = seq;
            if (seq >= 0) {
                bool bad;
                n.q = kv_seq(a.pool, a.seqs, n.seq, bad);
                const long long columns = (long long)n.q.n * a.group;
                const int tiles = (int)((columns + COLS - 1) / COLS);
                const int tile = tiles - 1 - local / a.pool.kv_heads;
                n.head = local % a.pool.kv_heads;
                n.col0 = tile * COLS;
                n.cols = (int)min((long long)COLS, columns - n.col0);
                n.first_pos = n.q.len - n.q.n;
                const int pos_lo = n.first_pos + n.col0 / a.group;
                n.pos_hi = n.first_pos + (n.col0 + n.cols - 1) / a.group;
                n.seen_lo = kv_first_seen(pos_lo, a.window);
                n.k0 = n.seen_lo / KV_TILE * KV_TILE;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int last = min(n.cols, (i + 1) * M_TILE) - 1;  // the M tile's last column
                    const int pos = n.first_pos + (n.col0 + last) / a.group;
                    n.blocks[i] = last < i * M_TILE || pos < n.k0 ? 0 : (pos - n.k0) / BLOCK + 1;
                }
                n.most = max(n.blocks[0], n.blocks[1]);
            }
            to = n;
        }
        __syncwarp();
    };
    if (mma_warp) {
        fetch(ctl.item[0], true);
    }
    __syncthreads();

    for (;;) {
        const Item& it = ctl.item[items_before & 1];
        if (it.seq < 0 || ctl.late) {
            break;
        }
        if (mma_warp) {  // while the others load queries
            fetch(ctl.item[(items_before & 1) ^ 1], false);
        }
        // ---- queries ----
        else {
            // Eight lanes to a column, which take four dimensions of every 32 each: four columns share what a column costs beside its
            // values (a warp to a column: 8 us for an item's queries).  Loads go without branches, to column 0 in place of one that is
            // not there.
            constexpr int AT_ONCE = 2, MINE = COLS / (SOFT_WARPS + KV_WARPS);
            const int j = lane & 7;
            for (int c8 = 0; c8 < MINE; c8 += 4 * AT_ONCE) {
                float v[AT_ONCE][NB][4];
                const auto bring = [&](auto f32) {
#pragma unroll
                    for (int k = 0; k < AT_ONCE; ++k) {
                        const int c = warp * MINE + c8 + 4 * k + (lane >> 3), col = it.col0 + (c < it.cols ? c : 0), row = col / a.group;
                        const int64_t src = (it.q.row0 + row) * a.q_stride + (int64_t)(it.head * a.group + col - row * a.group) * HD + 4 * j;
#pragma unroll
                        for (int n = 0; n < NB; ++n) {
                            if (decltype(f32)::value) {
                                const float4 x = *reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + src + 32 * n);
                                v[k][n][0] = x.x, v[k][n][1] = x.y, v[k][n][2] = x.z, v[k][n][3] = x.w;
                            } else {
                                const uint2 x = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(a.q) + src + 32 * n);
                                v[k][n][0] = __uint_as_float(x.x << 16), v[k][n][1] = __uint_as_float(x.x & 0xFFFF0000u);
                                v[k][n][2] = __uint_as_float(x.y << 16), v[k][n][3] = __uint_as_float(x.y & 0xFFFF0000u);
                            }
                        }
                    }
                };
                if (a.q_type == QMM_OUT_F32) {
                    bring(std::true_type{});
                } else {
                    bring(std::false_type{});
                }
#pragma unroll
                for (int k = 0; k < AT_ONCE; ++k) {
                    const int c = warp * MINE + c8 + 4 * k + (lane >> 3);
                    uint32_t bits = 0;
#pragma unroll
                    for (int n = 0; n < NB; ++n) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            v[k][n][i] = c < it.cols ? v[k][n][i] : 0.0f;
                            bits = max(bits, __float_as_uint(v[k][n][i]) & 0x7FFFFFFFu);
                        }
                    }
#pragma unroll
                    for (int o = 1; o < 8; o <<= 1) {
                        bits = max(bits, __shfl_xor_sync(0xFFFFFFFFu, bits, o));
                    }
                    const int exponent = (int)(bits >> 23) - 127;
                    const int e = bits == 0 || exponent == 128 ? 0 : max(-112, min(120, 12 - exponent));
                    const float up = __uint_as_float((uint32_t)(e + 127) << 23 | (a.scale < 0.0f ? 0x80000000u : 0u));
                    uint8_t* row = q_smem + (c / M_TILE) * Shape::Q_BYTES + (c % M_TILE) * 128;
#pragma unroll
                    for (int n = 0; n < NB; ++n) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            // dimension 32 n + 8 t + 2 r + e lies at 32 n + 8 r + 2 t + e, as in the keys: t is j / 2, r is 2 (j % 2) + h
                            const int chunk = n % 2 * 4 + 2 * (j & 1) + h;
                            *reinterpret_cast<__half2*>(row + n / 2 * (M_TILE * 128) + ((chunk ^ (c & 7)) << 4) + (j >> 1) * 4) =
                                __floats2half2_rn(v[k][n][2 * h] * up, v[k][n][2 * h + 1] * up);
                        }
                    }
                    if (j == 0) {
                        ctl.q_scale[c] = fabsf(a.scale) * 1.44269504088896340736f * __uint_as_float((uint32_t)(127 - e) << 23);
                    }
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        __syncthreads();

        if (mma_warp) {
            // ---- MMAs ----
            const uint32_t id_s = idesc_f16(BLOCK), id_o = idesc_f16(HD);
            const uint64_t q_desc = umma_smem_desc(g_smem_u32(q_smem)), k_desc = umma_smem_desc(g_smem_u32(k_smem)),
                           v_desc = umma_smem_desc(g_smem_u32(v_smem));
            bool ok = true;
            auto wait = [&](uint64_t* bar, uint32_t parity) {
                ok = ok && g_mbar_wait_warp(bar, parity);
            };
            auto scores = [&](int i, int kb) {
                const uint32_t stage = (blocks_before + kb) & 1;
                fence_after();
                if (elect_one()) {
#pragma unroll
                    for (int kk = 0; kk < HD / 16; ++kk) {
                        const uint64_t at = 2 * (kk & 3);
                        umma_ss(tmem + i * BLOCK, q_desc + (uint64_t)((i * Shape::Q_BYTES + (kk >> 2) * M_TILE * 128) >> 4) + at,
                                k_desc + (uint64_t)((stage * Shape::K_BYTES + (kk >> 2) * BLOCK * 128) >> 4) + at, id_s, kk > 0);
                    }
                    umma_commit(&ctl.s_full[i]);
                }
                __syncwarp();
            };
            auto values = [&](int i, int kb, int half) {
                const uint32_t stage = (blocks_before + kb) & 1;
                fence_after();
                if (elect_one()) {
#pragma unroll
                    for (int kk = half * BLOCK / 32; kk < (half + 1) * BLOCK / 32; ++kk) {
                        umma_ts(tmem + 2 * BLOCK + i * M_TILE, tmem + i * BLOCK + 8 * kk,
                                v_desc + (uint64_t)((stage * Shape::V_BYTES + (kk >> 2) * HD * 128) >> 4) + 2 * (kk & 3), id_o,
                                kb > 0 || kk > 0);
                    }
                }
                __syncwarp();
            };
            auto commit = [&](uint64_t* bar) {
                if (elect_one()) {
                    umma_commit(bar);
                }
                __syncwarp();
            };
            const int most = it.most, blocks0 = it.blocks[0], blocks1 = it.blocks[1];
            if (most > 0) {
                wait(&ctl.k_full[blocks_before & 1], blocks_before >> 1 & 1);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if ((i ? blocks1 : blocks0) > 0 && ok) {
                        scores(i, 0);
                    }
                }
                commit(&ctl.k_empty[blocks_before & 1]);
            }
            for (int kb = 0; kb < most && ok; ++kb) {
                const uint32_t b = blocks_before + kb;
                wait(&ctl.v_full[b & 1], b >> 1 & 1);
                if (kb + 1 < most) {
                    wait(&ctl.k_full[(b + 1) & 1], (b + 1) >> 1 & 1);
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int mine = i ? blocks1 : blocks0;
                    if (kb < mine && ok) {
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            wait(&ctl.p_full[i][half], ((i ? before1 : before0) + kb) & 1);
                            if (ok) {
                                values(i, kb, half);
                            }
                        }
                    }
                    if (kb + 1 < mine && ok) {
                        scores(i, kb + 1);
                    }
                }
                commit(&ctl.v_empty[b & 1]);
                if (kb + 1 < most) {
                    commit(&ctl.k_empty[(b + 1) & 1]);
                }
            }
            commit(&ctl.o_full);
            if (!ok && lane == 0) {
                give_up();
            }
        } else if (warp >= SOFT_WARPS) {
            // ---- keys and values ----
            const int w = warp - SOFT_WARPS, g = lane >> 2, t = lane & 3;
            bool ok = true;
            const int most = it.most;
            // lane n holds where this warp's tile of block n (and 32 + n, ...) lies, 0 where there is none
            auto where = [&](int kb) -> unsigned long long {
                const int tok0 = it.k0 + kb * BLOCK + w * KV_TILE;
                if (kb >= most || tok0 > it.pos_hi) {
                    return 0;
                }
                const int page = kv_page(a.pool, a.seqs, it.seq, tok0);
                if (page < 0) {
                    atomicExch(a.seqs.status, KV_BAD_PAGE);
                    return 0;
                }
                return reinterpret_cast<unsigned long long>(a.pool.base + kv_tile_index(a.pool, page, it.head, tok0) * TILE);
            };
            unsigned long long places = most > 0 ? where(lane) : 0;
            auto place_of = [&](int kb) -> const uint8_t* {
                return reinterpret_cast<const uint8_t*>(__shfl_sync(0xFFFFFFFFu, places, kb & 31));
            };
            // raw words of a tile's keys and of its values: asked for as soon as the ones before have been converted
            uint32_t kw[2][LANE / 4], vw[2][LANE / 4], ks[2][QUANT ? NB : 1], vs[2][QUANT ? NB : 1];
            auto ask = [&](uint32_t (&x)[2][LANE / 4], uint32_t (&d)[2][QUANT ? NB : 1], const uint8_t* plane, int scale_at) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    if (plane) {
#pragma unroll
                        for (int i = 0; i < LANE / VEC; ++i) {
                            load_words<VEC>(x[j] + i * VEC / 4, plane + j * 32 * LANE + i * 32 * VEC + lane * VEC);
                        }
                        if (QUANT) {
                            load_words<(NB >= 4 ? 16 : 8)>(d[j], plane + PLANE + (scale_at * 2 + j) * NB * 4);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < LANE / 4; ++i) {
                            x[j][i] = 0;
                        }
#pragma unroll
                        for (int i = 0; i < (QUANT ? NB : 1); ++i) {
                            d[j][i] = 0;
                        }
                    }
                }
            };
            const uint8_t* tile = nullptr;
            if (most > 0) {
                tile = place_of(0);
                ask(kw, ks, tile, g >> 1);
                ask(vw, vs, tile ? tile + PLANE + SCALES : nullptr, t);
            }
            for (int kb = 0; kb < most && ok; ++kb) {
                const uint32_t b = blocks_before + kb, stage = b & 1;
                const int tok0 = it.k0 + kb * BLOCK + w * KV_TILE;
                if ((kb & 31) == 31) {
                    places = where(kb + 1 + lane);
                }
                const uint8_t* next = place_of(kb + 1);  // nothing behind the last block
                if (b >= 2) {
                    ok = g_mbar_wait_warp(&ctl.k_empty[stage], ((b >> 1) - 1) & 1);
                }
                if (ok) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
#pragma unroll
                        for (int n = 0; n < NB; ++n) {
                            uint32_t x[4];
                            quants<FMT>(kw[j] + n * (U / 4), x);
                            if (QUANT) {
                                const uint32_t both = ks[j][n % (QUANT ? NB : 1)];
                                const __half2 d = as_h2(__byte_perm(both, both, g & 1 ? 0x3232u : 0x1010u));
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    x[i] = h2_bits(__hmul2(as_h2(x[i]), d));
                                }
                            }
                            // matrix r: keys g, dimensions 32 n + 8 t + 2 r + {0, 1}.  This lane's row for the store is key
                            // lane & 7, its 16 bytes are matrix lane >> 3
                            const int row = w * KV_TILE + 8 * j + (lane & 7), chunk = 4 * (n & 1) + (lane >> 3);
                            store_matrices(k_smem + stage * Shape::K_BYTES + (n >> 1) * BLOCK * 128 + row * 128 +
                                               ((chunk ^ (lane & 7)) << 4),
                                           x);
                        }
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) {
                        g_mbar_arrive(&ctl.k_full[stage]);
                    }
                    ask(kw, ks, next, g >> 1);
                    if (b >= 2) {
                        ok = g_mbar_wait_warp(&ctl.v_empty[stage], ((b >> 1) - 1) & 1);
                    }
                }
                if (ok) {
                    // tokens that no column sees, and values that are not finite, enter as 0
                    uint32_t odd[2];  // tokens 2t, 2t + 1 of either half: some value of this lane's is not finite
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        __half2 sum = as_h2(0u);
#pragma unroll
                        for (int n = 0; n < (QUANT ? NB : LANE / 4); ++n) {  // 0, or NaN behind an infinity or a NaN
                            sum = __hfma2(as_h2(QUANT ? vs[j][n % (QUANT ? NB : 1)] : vw[j][n % (LANE / 4)]), as_h2(0u), sum);
                        }
                        odd[j] = h2_bits(sum) & 0x7FFF7FFFu;
                    }
                    uint32_t poison = 0;
                    const bool edge = tok0 < it.seen_lo || tok0 + KV_TILE - 1 > it.pos_hi;
                    auto put = [&](auto masked, const uint32_t (&keep)[2]) {
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
#pragma unroll
                            for (int n = 0; n < NB; ++n) {
                                uint32_t x[4];
                                quants<FMT>(vw[j] + n * (U / 4), x);
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    if (QUANT) {
                                        x[i] = h2_bits(__hmul2(as_h2(x[i]), as_h2(vs[j][n % (QUANT ? NB : 1)])));
                                    }
                                    if (decltype(masked)::value) {
                                        x[i] &= keep[j];
                                    }
                                }
                                // dimension 32 n + 4 g + i is row 32 n + 8 i + g: four matrices of 8 rows x 8 tokens.  This
                                // lane's row for the store is 32 n + lane; its 16 bytes are tokens 8 j .. of the tile
                                const int chunk = (w * KV_TILE + 8 * j) % 64 / 8;
                                store_matrices(v_smem + stage * Shape::V_BYTES + w * KV_TILE / 64 * HD * 128 + (32 * n + lane) * 128 +
                                                   ((chunk ^ (lane & 7)) << 4),
                                               x);
                            }
                        }
                    };
                    const bool any_odd = __any_sync(0xFFFFFFFFu, (odd[0] | odd[1]) != 0);
                    if (any_odd || edge) {
                        uint32_t keep[2] = {0xFFFFFFFFu, 0xFFFFFFFFu};
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const int pos = tok0 + 8 * j + 2 * t + e;
                                const uint32_t half = e ? 0xFFFF0000u : 0x0000FFFFu;
                                const bool seen = pos >= it.seen_lo && pos <= it.pos_hi;
                                // the token's bit of every lane that has some of its dimensions
                                unsigned int who = __ballot_sync(0xFFFFFFFFu, seen && (odd[j] & half) != 0);
                                who |= who >> 16;
                                who |= who >> 8;
                                who |= who >> 4;
#pragma unroll
                                for (int tt = 0; tt < 4; ++tt) {
                                    poison |= (who >> tt & 1u) << (8 * j + 2 * tt + e);
                                }
                                if (!seen) {
                                    keep[j] &= ~half;
                                }
                            }
                        }
                        if (any_odd) {
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
#pragma unroll
                                for (int n = 0; n < (QUANT ? NB : LANE / 4); ++n) {
                                    uint32_t& x = QUANT ? vs[j][n % (QUANT ? NB : 1)] : vw[j][n % (LANE / 4)];
                                    x = finite_or_0(x);
                                }
                            }
                        }
                        put(std::true_type{}, keep);
                    } else {
                        const uint32_t all[2] = {0xFFFFFFFFu, 0xFFFFFFFFu};
                        put(std::false_type{}, all);
                    }
                    if (lane == 0) {
                        ctl.poison[b & 7][w] = poison;
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) {
                        g_mbar_arrive(&ctl.v_full[stage]);
                    }
                    ask(vw, vs, next ? next + PLANE + SCALES : nullptr, t);
                }
                if (!ok && lane == 0) {
                    give_up();
                }
            }
        } else {
            // ---- softmax: one thread per column ----
            const int i = warp >> 2, c = threadIdx.x;  // M tile, column of the CTA
            const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
            const uint32_t s_at = tmem + lanes + i * BLOCK, o_at = tmem + lanes + 2 * BLOCK + i * M_TILE;
            const float qs = ctl.q_scale[c];
            const int pos = it.first_pos + (it.col0 + c) / a.group;
            const int low = kv_first_seen(pos, a.window);
            float m = -INFINITY, l = 0.0f;
            bool ok = true;
            bool far = false;  // the maximum of some column of the warp has been past FAR
            const int my_blocks = it.blocks[i];
            // The dimensions in which this column sees a value of block kb that is not finite.  The words that name its tokens stay for
            // eight blocks, and the warps that write them are at most two ahead of the values that are multiplied; the dimensions
            // come from the cache, one to a lane.  In shared memory: four registers for them took 5 % of a long prompt's time.
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                ctl.odd[n][c] = 0;
            }
            auto look_for_poison = [&](int kb) {
                const uint32_t mine =
                    lane < KV_TILES ? *reinterpret_cast<volatile uint32_t*>(&ctl.poison[(blocks_before + kb) & 7][lane]) : 0u;
                if (__any_sync(0xFFFFFFFFu, mine != 0)) {
                    for (int w = 0; w < KV_TILES; ++w) {
                        const int tok0 = it.k0 + kb * BLOCK + w * KV_TILE;
                        const uint8_t* values = nullptr;
                        for (uint32_t bits = __shfl_sync(0xFFFFFFFFu, mine, w); bits != 0; bits &= bits - 1) {
                            if (!values) {  // the tile's page has been looked up before: it is the pool's
                                values = a.pool.base + kv_tile_index(a.pool, max(kv_page(a.pool, a.seqs, it.seq, tok0), 0), it.head, tok0) * TILE +
                                         PLANE + SCALES;
                            }
                            const int k = __ffs(bits) - 1;
                            const bool sees = tok0 + k <= pos && tok0 + k >= low;
#pragma unroll 1
                            for (int n = 0; n < NB; ++n) {
                                const uint8_t* x = QUANT ? values + PLANE + kv_scale_place(HD, k, n)
                                                         : values + kv_place(FMT, HD, k >> 3, (lane & ~3) + (k >> 1 & 3), n, 4 * (lane & 3) + 2 * (k & 1));
                                const uint32_t bad = __ballot_sync(0xFFFFFFFFu, (*reinterpret_cast<const uint16_t*>(x) & 0x7C00u) == 0x7C00u);
                                if (sees) {
                                    ctl.odd[n][c] |= bad;
                                }
                            }
                        }
                    }
                }
            };
            const uint32_t my_before = i ? before1 : before0;
            for (int kb = 0; kb < my_blocks && ok; ++kb) {
                const int key0 = it.k0 + kb * BLOCK;
                ok = g_mbar_wait_warp(&ctl.s_full[i], (my_before + kb) & 1);
                if (!ok) {
                    break;
                }
                fence_after();
                // keys key0 + lo .. key0 + hi of the block are this column's
                const int hi = pos - key0, lo = low - key0;
                // Probabilities in a warp with a maximum past FAR: those columns' scores lose it before the factor
                auto far_probabilities = [&]() {
                    const float lost = is_far(m) ? ctl.far_max[c] : 0.0f;
                    const float ref = is_far(m) ? -BIAS : m == -INFINITY ? 0.0f : m - BIAS;
#pragma unroll 1
                    for (int part = 0; part < BLOCK / 16; ++part) {
                        float x[16];
                        tmem_ld16(s_at + 16 * part, x);
                        tmem_wait_ld(x);
                        uint32_t p[8];
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            const float e = exp2_fast(fmaf(x[k] - lost, qs, -ref));
                            x[k] = 16 * part + k <= hi && 16 * part + k >= lo ? e : 0.0f;
                            l += x[k];
                        }
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            p[k] = h2_bits(__floats2half2_rn(x[2 * k], x[2 * k + 1]));
                        }
                        tmem_st8(s_at + 8 * part, p);  // over columns that have been read
                        if (part == BLOCK / 32 - 1) {  // the first half of the product can begin
                            tmem_wait_st();
                            fence_before();
                            __syncwarp();
                            if (lane == 0) {
                                g_mbar_arrive(&ctl.p_full[i][0]);
                            }
                        }
                    }
                    tmem_wait_st();
                };
                auto probabilities = [&](auto all_seen) {
                    constexpr bool WHOLE = decltype(all_seen)::value;
                    constexpr int PARTS = BLOCK / 16;
                    float s[2][16];  // the next 16 scores are on their way while these are worked on
                    float top4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                    tmem_ld16(s_at, s[0]);
                    tmem_wait_ld(s[0]);
#pragma unroll
                    for (int part = 0; part < PARTS; ++part) {
                        float (&x)[16] = s[part & 1];
                        tmem_ld16(s_at + 16 * ((part + 1) % PARTS), s[(part + 1) & 1]);
                        if (!WHOLE) {
#pragma unroll
                            for (int k = 0; k < 16; ++k) {
                                x[k] = 16 * part + k <= hi && 16 * part + k >= lo ? x[k] : -INFINITY;
                            }
                        }
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            top4[k & 3] = max3(top4[k & 3], x[2 * k], x[2 * k + 1]);
                        }
                        tmem_wait_ld(s[(part + 1) & 1]);
                    }
                    float top = fmaxf(top4[0], max3(top4[1], top4[2], top4[3]));
                    const float raw = top;
                    top = top == -INFINITY ? top : top * qs;
                    bool higher = top > m + SLACK || (m == -INFINITY && top > m);
                    if (far && is_far(m)) {
                        higher = raw > ctl.far_max[c] && (raw - ctl.far_max[c]) * qs > SLACK;
                    }
                    if (__any_sync(0xFFFFFFFFu, higher)) {
                        const float down = !higher ? 1.0f : exp2_fast(far && is_far(m) ? (ctl.far_max[c] - raw) * qs : m - top);
                        if (higher) {
                            m = top;
                            ctl.far_max[c] = raw;
                        }
                        far = far || __any_sync(0xFFFFFFFFu, is_far(m));
                        l *= down;
                        if (kb > 0) {
                            float (&x)[16] = s[1];
#pragma unroll 1
                            for (int part = 0; part < HD / 16; ++part) {
                                tmem_ld16(o_at + 16 * part, x);
                                tmem_wait_ld(x);
#pragma unroll
                                for (int k = 0; k < 16; ++k) {
                                    x[k] *= down;
                                }
                                tmem_st16(o_at + 16 * part, x);
                            }
                            tmem_wait_st();
                        }
                    }
                    if (far) {
                        far_probabilities();
                        return;
                    }
                    const float ref = m == -INFINITY ? 0.0f : m - BIAS;
                    static_assert(PARTS % 2 == 0, "the first part is in s[0] again");
                    float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
                    for (int part = 0; part < PARTS; ++part) {
                        float (&x)[16] = s[part & 1];
                        uint32_t p[8];
                        if (part + 1 < PARTS) {
                            tmem_ld16(s_at + 16 * (part + 1), s[(part + 1) & 1]);
                        }
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const float2 y = fma2(make_float2(x[2 * k], x[2 * k + 1]), make_float2(qs, qs), make_float2(-ref, -ref));
                            float2 e = make_float2(exp2_fast(y.x), exp2_fast(y.y));
                            if (!WHOLE) {
                                e.x = 16 * part + 2 * k <= hi && 16 * part + 2 * k >= lo ? e.x : 0.0f;
                                e.y = 16 * part + 2 * k + 1 <= hi && 16 * part + 2 * k + 1 >= lo ? e.y : 0.0f;
                            }
                            sum[k & 1] = add2(sum[k & 1], e);
                            p[k] = h2_bits(__floats2half2_rn(e.x, e.y));
                        }
                        if (part + 1 < PARTS) {
                            tmem_wait_ld(s[(part + 1) & 1]);
                        }
                        tmem_st8(s_at + 8 * part, p);  // over columns that have been read
                        if (part == PARTS / 2 - 1) {  // the first half of the product can begin
                            tmem_wait_st();
                            fence_before();
                            __syncwarp();
                            if (lane == 0) {
                                g_mbar_arrive(&ctl.p_full[i][0]);
                            }
                        }
                    }
                    sum[0] = add2(sum[0], sum[1]);
                    l += sum[0].x + sum[0].y;
                    tmem_wait_st();
                };
                if (__all_sync(0xFFFFFFFFu, hi >= BLOCK - 1 && lo <= 0)) {
                    probabilities(std::true_type{});
                } else {
                    probabilities(std::false_type{});
                }
                fence_before();
                __syncwarp();
                if (lane == 0) {
                    g_mbar_arrive(&ctl.p_full[i][1]);
                }
                if (kb > 0) {  // this block's scores were issued behind the last one's values, which were complete by then
                    look_for_poison(kb - 1);
                }
            }
            // ---- results ----
            ok = ok && g_mbar_wait_warp(&ctl.o_full, items_before & 1);
            if (!ok && lane == 0) {
                give_up();
            }
            fence_after();
            if (ok && my_blocks > 0) {
                look_for_poison(my_blocks - 1);
            }
            const int64_t row = it.q.row0 + (it.col0 + c) / a.group;
            const int qh = it.head * a.group + (it.col0 + c) % a.group;
            const unsigned long long out = c < it.cols && ok
                                               ? reinterpret_cast<unsigned long long>(static_cast<__nv_bfloat16*>(a.out) + row * a.out_stride + (int64_t)qh * HD)
                                               : 0ull;
            // The queries' place, which the products have left (o_full), takes a column's row, so that a warp writes whole rows: 16
            // bytes of 32 rows at a time took 3 us an item.
            uint8_t* place = q_smem + i * Shape::Q_BYTES + (c % M_TILE) * 128;
            const bool none = my_blocks == 0 || (m == -INFINITY && l == 0.0f);
            const float inv = none ? 0.0f : 1.0f / l;
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                float o[2][16];
                if (my_blocks > 0) {
                    tmem_ld16(o_at + 32 * n, o[0]);
                    tmem_ld16(o_at + 32 * n + 16, o[1]);
                    tmem_wait_ld(o[0]);
                    tmem_wait_ld(o[1]);
                }
                if (ok) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {  // dimensions 32 n + 8 k ..: 4 g + j is column 8 j + g
                        uint32_t x[4];
#pragma unroll
                        for (int h = 0; h < 4; ++h) {
                            const int d = 8 * k + 2 * h, from = 8 * (d & 3) + (d >> 2);
                            const float x0 = none ? 0.0f : o[from >> 4][from & 15] * inv, x1 = none ? 0.0f : o[(from + 8) >> 4][(from + 8) & 15] * inv;
                            const __nv_bfloat162 pair = __floats2bfloat162_rn(x0, x1);
                            x[h] = *reinterpret_cast<const uint32_t*>(&pair);
                        }
                        *reinterpret_cast<uint4*>(place + n / 2 * (M_TILE * 128) + (((n % 2 * 4 + k) ^ (c & 7)) << 4)) =
                            make_uint4(x[0], x[1], x[2], x[3]);
                    }
                }
            }
#pragma unroll 1
            for (int n = 0; n < NB; ++n) {
                for (uint32_t odd = ctl.odd[n][c]; odd != 0; odd &= odd - 1) {
                    const int d = __ffs(odd) - 1;
                    *reinterpret_cast<uint16_t*>(place + n / 2 * (M_TILE * 128) + (((n % 2 * 4 + d / 8) ^ (c & 7)) << 4) + d % 8 * 2) = 0x7FC0u;
                }
            }
            __syncwarp();
            constexpr int LANES = HD / 8;  // of a row, 16 bytes each
#pragma unroll
            for (int r = 0; r < LANES; ++r) {
                const int from = r * (32 / LANES) + lane / LANES, chunk = lane % LANES, cc = (warp & 3) * 32 + from;
                const unsigned long long to = __shfl_sync(0xFFFFFFFFu, out, from);
                if (to != 0) {
                    reinterpret_cast<uint4*>(to)[chunk] = *reinterpret_cast<const uint4*>(
                        q_smem + i * Shape::Q_BYTES + chunk / 8 * (M_TILE * 128) + cc * 128 + ((chunk % 8 ^ (cc & 7)) << 4));
                }
            }
            fence_before();
        }
        blocks_before += it.most;
        before0 += it.blocks[0];
        before1 += it.blocks[1];
        __syncthreads();
        ++items_before;
        fence_after();
    }

    fence_before();
    __syncthreads();
    if (mma_warp) {
        fence_after();
        if (ctl.late) {  // products may still be under way: once more, before their operands' and their sums' memory is given back
            if (elect_one()) {
                umma_commit(&ctl.drained);
            }
            __syncwarp();
            g_mbar_wait_warp(&ctl.drained, 0);
        }
        __syncwarp();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
        // the last CTA leaves the counters zeroed for the next call
        if (lane == 0 && atomicAdd(done_ctas, 1u) == gridDim.x - 1) {
            atomicExch(next_item, 0u);
            atomicExch(done_ctas, 0u);
        }
    }
}

template <int FMT, int HD>
cudaError_t launch_prompt(const KvAttnArgs& a, int sm_count, cudaStream_t stream)
{
    using Shape = PromptShape<FMT, HD>;
    auto kernel = kv_prompt_kernel<FMT, HD>;
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
    // no more CTAs than there can be items
    const int64_t items = (a.seqs.rows * a.group / COLS + a.seqs.batch) * a.pool.kv_heads;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)std::max<int64_t>(1, std::min<int64_t>(sm_count, items)));
    cfg.blockDim = dim3(THREADS);
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
cudaError_t launch_prompt_fmt(const KvAttnArgs& a, int sm_count, cudaStream_t stream)
{
    return a.pool.head_dim == 64 ? launch_prompt<FMT, 64>(a, sm_count, stream) : launch_prompt<FMT, 128>(a, sm_count, stream);
}

}  // namespace

// bf16 results of enough columns: a list item (256 columns of a kv head) is one CTA's, from its first key to its last, where the
// rows kernel cuts anything over the whole GPU.  2000 tokens of 128 dimensions, rows / prompt kernel, Q4_0: one sequence of 32 rows
// of 64 heads 43 / 56 us, of 64 rows 69 / 56 us; of 64 rows of 32 heads (one to a kv head) 43 / 49 us, of 128 rows 68 / 51 us; eight
// sequences of 4 rows of 64 heads 44 / 49 us, of 8 rows 69 / 49 us, of 16 rows of 32 heads (16 columns each) 70 / 102 us.
// What the rule does not know are the lengths, which are the device's, and which rows are whose: a prompt of 512 rows of 64 heads and 31 single
// tokens behind 1023 others take 80 us in one call and 75 in two, behind 8191 324 and 150, behind 65535 2266 and 716.
bool kv_takes_prompt(const KvAttnArgs& a)
{
    return a.out_type == QMM_OUT_BF16 && (a.pool.head_dim == 64 || a.pool.head_dim == 128) && a.seqs.row_begin != nullptr &&
           a.seqs.rows * a.group >= (int64_t)64 * a.seqs.batch && a.seqs.rows * a.group * a.pool.kv_heads >= 4096;
}

cudaError_t launch_kv_prompt(const KvAttnArgs& a, int sm_count, cudaStream_t stream)
{
    switch (a.pool.fmt) {
    case FMT_Q4_0: return launch_prompt_fmt<FMT_Q4_0>(a, sm_count, stream);
    case FMT_Q8_0: return launch_prompt_fmt<FMT_Q8_0>(a, sm_count, stream);
    default: return launch_prompt_fmt<KV_F16>(a, sm_count, stream);
    }
}

}  // namespace qmm
