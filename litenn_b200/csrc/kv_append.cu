// Appending to the paged cache and reading it back (include/litenn_kv.h).
//
// Append: a row's queries and keys are turned by their position's angles, keys and values are quantized in blocks of 32
// dimensions and stored where the attention kernels' operands want them (kv_layout.cuh).  The angles and the rotation are
// taken in fp64: a position of 10^5 times a frequency near 1 has lost eight of fp32's bits before the cosine is taken, and the
// blocks' rounding turns a last-bit difference into another quant.  Rounding the rotated value to fp32 once makes the stored
// bytes a function of the inputs alone, whichever form wrote them.
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
// rules in fp32 (no contraction: the bytes must not depend on how the compiler joins a product and a sum).
template <int FMT>
__device__ __forceinline__ float quantize4(const float (&x)[4], int lane, uint32_t (&q)[4])
{
    float top = x[0], size = fabsf(x[0]);
    bool odd = !isfinite(x[0]);
#pragma unroll
    for (int i = 1; i < 4; ++i) {
        odd |= !isfinite(x[i]);
        if (fabsf(x[i]) > size) {  // the first of equals
            size = fabsf(x[i]);
            top = x[i];
        }
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        const float other = __shfl_xor_sync(0xFFFFFFFFu, top, o);
        const bool lower = (lane & o) != 0;  // the other lane's values come first
        if (fabsf(other) > size || (lower && fabsf(other) == size)) {
            size = fabsf(other);
            top = other;
        }
    }
    const bool any_odd = (__ballot_sync(0xFFFFFFFFu, odd) >> (lane & 24) & 0xFFu) != 0;
    float d = FMT == FMT_Q4_0 ? __fdiv_rn(top, -8.0f) : __fdiv_rn(size, 127.0f);
    d = fminf(fmaxf(d, -65504.0f), 65504.0f);  // more than fp16 holds: the values saturate
    const float inverse = d == 0.0f ? 0.0f : __fdiv_rn(1.0f, d);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float y = __fmul_rn(x[i], inverse);
        if (FMT == FMT_Q4_0) {
            q[i] = (uint32_t)fminf(fmaxf(floorf(__fadd_rn(y, 8.5f)), 0.0f), 15.0f);
        } else {
            const float r = fminf(floorf(__fadd_rn(fabsf(y), 0.5f)), 127.0f);
            q[i] = (uint32_t)(int)(copysignf(r, y) + 128.0f);
        }
        if (any_odd) {
            q[i] = FMT == FMT_Q4_0 ? 8u : 128u;
        }
    }
    return any_odd ? __uint_as_float(0x7FC00000u) : d;
}

// Stores four consecutive values of a token: `keys` tells which plane's order.  All 32 lanes call it; `on` lanes store.
template <int FMT>
__device__ __forceinline__ void put4(uint8_t* tile, int hd, bool keys, int token, int dim, const float (&x)[4], int lane, bool on)
{
    const int b = dim >> 5, first = keys ? 0 : kv_plane_bytes(FMT, hd) + kv_scale_bytes(FMT, hd);
    const int j = token >> 3, e = token & 1;
    if (FMT == KV_F16) {
        const __half2 lo = __floats2half2_rn(x[0], x[1]), hi = __floats2half2_rn(x[2], x[3]);
        uint2 w;
        w.x = *reinterpret_cast<const uint32_t*>(&lo);
        w.y = *reinterpret_cast<const uint32_t*>(&hi);
        if (!on) {
            return;
        }
        if (keys) {
            *reinterpret_cast<uint2*>(tile + kv_place(FMT, hd, j, 4 * (token & 7) + (dim >> 3 & 3), b, 2 * (dim & 7))) = w;
        } else {
            uint8_t* at = tile + first + kv_place(FMT, hd, j, 4 * (dim >> 2 & 7) + (token >> 1 & 3), b, 2 * e);
            *reinterpret_cast<uint16_t*>(at) = (uint16_t)w.x;
            *reinterpret_cast<uint16_t*>(at + 4) = (uint16_t)(w.x >> 16);
            *reinterpret_cast<uint16_t*>(at + 8) = (uint16_t)w.y;
            *reinterpret_cast<uint16_t*>(at + 12) = (uint16_t)(w.y >> 16);
        }
        return;
    }
    uint32_t q[4];
    const float d = quantize4<FMT>(x, lane, q);
    if (FMT == FMT_Q4_0) {
        if (keys) {  // dims 4h.. of a lane's eight: bytes h and h + 2 of its word, the pair of lanes joins them
            const uint32_t h = (uint32_t)(dim >> 2) & 1u;
            const uint32_t mine = ((q[0] | q[2] << 4) | (q[1] | q[3] << 4) << 16) << (8u * h);
            const uint32_t word = mine | __shfl_xor_sync(0xFFFFFFFFu, mine, 1);
            if (on && h == 0) {
                *reinterpret_cast<uint32_t*>(tile + kv_place(FMT, hd, j, 4 * (token & 7) + (dim >> 3 & 3), b, 0)) = word;
            }
        } else if (on) {
            *reinterpret_cast<uint16_t*>(tile + first + kv_place(FMT, hd, j, 4 * (dim >> 2 & 7) + (token >> 1 & 3), b, 2 * e)) =
                (uint16_t)(q[0] | q[1] << 4 | q[2] << 8 | q[3] << 12);
        }
    } else if (on) {
        if (keys) {
            *reinterpret_cast<uint32_t*>(tile + kv_place(FMT, hd, j, 4 * (token & 7) + (dim >> 3 & 3), b, dim & 4)) =
                q[0] | q[1] << 8 | q[2] << 16 | q[3] << 24;
        } else {
            uint8_t* at = tile + first + kv_place(FMT, hd, j, 4 * (dim >> 2 & 7) + (token >> 1 & 3), b, e);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                at[2 * i] = (uint8_t)q[i];
            }
        }
    }
    if (on && (lane & 7) == 0) {
        *reinterpret_cast<__half*>(tile + first + kv_plane_bytes(FMT, hd) + kv_scale_place(hd, token, b)) = __float2half_rn(d);
    }
}

// Four consecutive values of a token as fp32.
template <int FMT>
__device__ __forceinline__ void get4(const uint8_t* tile, int hd, bool keys, int token, int dim, float (&x)[4])
{
    const int b = dim >> 5, first = keys ? 0 : kv_plane_bytes(FMT, hd) + kv_scale_bytes(FMT, hd);
    const int j = token >> 3, e = token & 1;
    const uint8_t* at = keys ? tile + kv_place(FMT, hd, j, 4 * (token & 7) + (dim >> 3 & 3), b, 0)
                             : tile + first + kv_place(FMT, hd, j, 4 * (dim >> 2 & 7) + (token >> 1 & 3), b, 0);
    if (FMT == KV_F16) {
        const __half* h = reinterpret_cast<const __half*>(at);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = __half2float(h[keys ? (dim & 4) + i : 2 * i + e]);
        }
        return;
    }
    const float d = __half2float(
        *reinterpret_cast<const __half*>(tile + first + kv_plane_bytes(FMT, hd) + kv_scale_place(hd, token, b)));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        int q;
        if (FMT == FMT_Q4_0) {
            const int r = keys ? (dim >> 1 & 2) + (i >> 1) : i, second = keys ? i & 1 : e;
            q = (at[(r >> 1) + 2 * second] >> (4 * (r & 1)) & 15) - 8;
        } else {
            q = (int)at[keys ? (dim & 4) + i : 2 * i + e] - 128;
        }
        x[i] = (float)q * d;
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

// One row per blockIdx.y, its work cut over blockIdx.x.  Simple form: every thread takes four dimensions of a head.
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
            put4<FMT>(tile, hd, keys, at.pos % KV_TILE, dim, x, lane, on && !is_q && page >= 0);
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

template <typename Args>
cudaError_t launch_rows(void (*kernel)(Args), const Args& a, int64_t rows, int items, cudaStream_t stream)
{
    cudaLaunchConfig_t cfg = {};
    // a few rows are cut over several CTAs each, many rows take one
    const int per_row = rows >= 148 ? 1 : (items + 255) / 256;
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
    switch (a.pool.fmt) {
    case FMT_Q4_0: return launch_rows(kv_append_kernel<FMT_Q4_0>, a, a.seqs.rows, items, stream);
    case FMT_Q8_0: return launch_rows(kv_append_kernel<FMT_Q8_0>, a, a.seqs.rows, items, stream);
    default: return launch_rows(kv_append_kernel<KV_F16>, a, a.seqs.rows, items, stream);
    }
}

cudaError_t launch_kv_read(const KvReadArgs& a, cudaStream_t stream)
{
    const int items = 2 * a.pool.kv_heads * a.pool.head_dim / 4;
    switch (a.pool.fmt) {
    case FMT_Q4_0: return launch_rows(kv_read_kernel<FMT_Q4_0>, a, a.seqs.rows, items, stream);
    case FMT_Q8_0: return launch_rows(kv_read_kernel<FMT_Q8_0>, a, a.seqs.rows, items, stream);
    default: return launch_rows(kv_read_kernel<KV_F16>, a, a.seqs.rows, items, stream);
    }
}

}  // namespace qmm
