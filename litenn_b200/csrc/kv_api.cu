// C ABI of the paged key/value cache (include/litenn_kv.h): argument checks and dispatch.
#include "../../include/litenn_kv.h"

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "kv_kernels.h"
#include "qmm_internal.h"
#include "qmm_kernels.h"

using namespace qmm;

namespace {

int fail(const char* fmt, ...)
{
    char buf[256];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    return qmm_internal_fail(QMM_E_INVALID, buf);
}

int fail_cuda(cudaError_t e, const char* what)
{
    char buf[256];
    snprintf(buf, sizeof buf, "%s failed: %s", what, cudaGetErrorString(e));
    return qmm_internal_fail(QMM_E_CUDA, buf);
}

constexpr int MAX_HEADS = 1 << 16;

int check_cache(const char* who, const qmm_kv_cache* c, bool with_pool)
{
    if (!c) {
        return fail("%s: the cache is null", who);
    }
    if (c->fmt != QMM_KV_F16 && c->fmt != QMM_FMT_Q8_0 && c->fmt != QMM_FMT_Q4_0) {
        return qmm_internal_fail(QMM_E_UNSUPPORTED, "a cache is fp16 (0), Q4_0 (1) or Q8_0 (5)");
    }
    if (c->head_dim != 64 && c->head_dim != 96 && c->head_dim != 128 && c->head_dim != 256) {
        return fail("%s: head_dim %d is not one of 64, 96, 128, 256", who, c->head_dim);
    }
    if (c->kv_heads < 1 || c->kv_heads > MAX_HEADS) {
        return fail("%s: %d kv heads", who, c->kv_heads);
    }
    if (c->page_tokens < KV_TILE || c->page_tokens % KV_TILE != 0 || c->page_tokens > 65536) {
        return fail("%s: page_tokens %d is not a multiple of 16 up to 65536", who, c->page_tokens);
    }
    if (c->n_pages < 1 || c->n_pages > 0x7FFFFFFF) {
        return fail("%s: %lld pages", who, (long long)c->n_pages);
    }
    // the pool's size is a product of numbers that each fit: it has to fit itself
    const double bytes = (double)c->n_pages * c->kv_heads * (c->page_tokens / KV_TILE) * kv_tile_bytes(c->fmt, c->head_dim);
    if (bytes > 1e15) {
        return fail("%s: the pool is larger than any memory", who);
    }
    if (with_pool && (!c->pool_dev || reinterpret_cast<uintptr_t>(c->pool_dev) % 16 != 0)) {
        return fail("%s: the pool is null or not 16-byte aligned", who);
    }
    return QMM_OK;
}

int check_batch(const char* who, const qmm_kv_cache* c, const qmm_kv_batch* b)
{
    if (!b) {
        return fail("%s: the batch is null", who);
    }
    if (b->batch < 0 || b->rows < 0 || b->table_width < 0) {
        return fail("%s: a negative batch, row count or table width", who);
    }
    if (b->batch > 0 && (!b->kv_len_dev || (b->table_width > 0 && !b->page_table_dev))) {
        return fail("%s: page_table or kv_len is null", who);
    }
    for (const int32_t* p : {b->page_table_dev, b->kv_len_dev, b->row_begin_dev}) {
        if (reinterpret_cast<uintptr_t>(p) % sizeof(int32_t) != 0) {
            return fail("%s: page_table, kv_len or row_begin is not 4-byte aligned", who);
        }
    }
    if (!b->row_begin_dev && b->batch > b->rows) {
        return fail("%s: %d sequences have one row each, but there are %lld rows", who, b->batch, (long long)b->rows);
    }
    if (b->rows > (int64_t)1 << 30) {
        return fail("%s: more than 2^30 rows", who);
    }
    if ((int64_t)b->table_width * c->page_tokens > 0x7FFFFFFF - 65536) {
        return fail("%s: a table of %d pages of %d tokens passes 31 bits", who, b->table_width, c->page_tokens);
    }
    return QMM_OK;
}

int check_rows(const char* who, const char* name, const void* p, int type, int64_t stride, int64_t width)
{
    if (type != QMM_OUT_F32 && type != QMM_OUT_BF16) {
        return fail("%s: element type %d of %s is neither fp32 nor bf16", who, type, name);
    }
    const int64_t item = type == QMM_OUT_F32 ? 4 : 2;
    if (!p || reinterpret_cast<uintptr_t>(p) % 16 != 0) {
        return fail("%s: %s is null or not 16-byte aligned", who, name);
    }
    if (stride < width || stride * item % 16 != 0 || stride > (int64_t)1 << 32) {
        return fail("%s: row stride %lld of %s is less than its %lld elements or no multiple of 16 bytes", who, (long long)stride,
                    name, (long long)width);
    }
    return QMM_OK;
}

struct Span {
    uintptr_t begin, end;
};
Span span_of(const void* p, int type, int64_t stride, int64_t rows, int64_t width)
{
    const uintptr_t item = type == QMM_OUT_F32 ? 4 : 2, b = reinterpret_cast<uintptr_t>(p);
    return {b, rows > 0 ? b + ((uintptr_t)(rows - 1) * stride + width) * item : b};
}
bool meet(const Span& a, const Span& b)
{
    return a.begin < b.end && b.begin < a.end;
}
// Rows of the same tensor, side by side: spans that meet although no element does.
bool overlap(const void* p, int pt, int64_t ps, int64_t pw, const void* q, int qt, int64_t qs, int64_t qw, int64_t rows)
{
    if (!meet(span_of(p, pt, ps, rows, pw), span_of(q, qt, qs, rows, qw))) {
        return false;
    }
    const int64_t pi = pt == QMM_OUT_F32 ? 4 : 2, qi = qt == QMM_OUT_F32 ? 4 : 2;
    if (ps * pi != qs * qi) {
        return true;
    }
    const int64_t pitch = ps * pi;
    const int64_t apart = (int64_t)((reinterpret_cast<uintptr_t>(q) - reinterpret_cast<uintptr_t>(p)) % (uintptr_t)pitch);
    const int64_t from_p = reinterpret_cast<uintptr_t>(q) >= reinterpret_cast<uintptr_t>(p)
                               ? apart
                               : (pitch - (int64_t)((reinterpret_cast<uintptr_t>(p) - reinterpret_cast<uintptr_t>(q)) % (uintptr_t)pitch)) % pitch;
    return from_p < pw * pi || from_p + qw * qi > pitch;
}

KvPool pool_of(const qmm_kv_cache& c)
{
    return {static_cast<uint8_t*>(c.pool_dev), c.fmt, c.kv_heads, c.head_dim, c.page_tokens, c.n_pages};
}
KvSeqs seqs_of(const qmm_kv_batch& b, int* status)
{
    return {b.batch, b.table_width, b.page_table_dev, b.kv_len_dev, b.row_begin_dev, b.rows, status};
}

}  // namespace

extern "C" {

int qmm_rope_frequencies(int dim, double theta, const float* factors, const qmm_rope_scaling* scaling, double* inv_freq_out,
                         double* gain_out)
{
    const char* who = "qmm_rope_frequencies";
    if (dim < 2 || dim % 2 != 0 || dim > 65536 || !(theta > 0.0) || !std::isfinite(theta) || !inv_freq_out || !gain_out) {
        return fail("%s: dim is even and positive, theta positive, the outputs not null", who);
    }
    const int kind = scaling ? scaling->kind : QMM_ROPE_SCALE_NONE;
    if (kind != QMM_ROPE_SCALE_NONE && kind != QMM_ROPE_SCALE_LINEAR && kind != QMM_ROPE_SCALE_YARN) {
        return fail("%s: unknown scaling %d", who, kind);
    }
    if (kind != QMM_ROPE_SCALE_NONE && !(scaling->factor >= 1.0f && std::isfinite(scaling->factor))) {
        return fail("%s: a context is scaled by at least 1", who);
    }
    if (kind == QMM_ROPE_SCALE_YARN &&
        !(scaling->trained >= 1.0f && scaling->beta_slow > 0.0f && scaling->beta_fast >= scaling->beta_slow && theta > 1.0 &&
          std::isfinite(scaling->trained) && std::isfinite(scaling->beta_fast))) {
        return fail("%s: YaRN wants trained >= 1, beta_fast >= beta_slow > 0 and theta > 1", who);
    }
    for (int i = 0; factors && i < dim / 2; ++i) {
        if (!(factors[i] > 0.0f) || !std::isfinite(factors[i])) {
            return fail("%s: factor %d is not positive", who, i);
        }
    }
    double low = 0.0, high = 0.0;
    if (kind == QMM_ROPE_SCALE_YARN) {  // the pair that turns `beta` times over the trained positions
        const double pi = 3.14159265358979323846;
        auto pair = [&](double beta) { return dim * std::log(scaling->trained / (beta * 2.0 * pi)) / (2.0 * std::log(theta)); };
        low = std::max(0.0, std::floor(pair(scaling->beta_fast)));
        high = std::min(dim - 1.0, std::ceil(pair(scaling->beta_slow)));
    }
    for (int i = 0; i < dim / 2; ++i) {
        double f = std::pow(theta, -2.0 * i / dim);
        if (factors) {
            f /= factors[i];
        }
        if (kind == QMM_ROPE_SCALE_LINEAR) {
            f /= scaling->factor;
        } else if (kind == QMM_ROPE_SCALE_YARN) {
            const double ramp = std::min(1.0, std::max(0.0, (i - low) / std::max(high - low, 0.001)));
            f = f * (1.0 - ramp) + f / scaling->factor * ramp;
        }
        inv_freq_out[i] = f;
    }
    *gain_out = kind == QMM_ROPE_SCALE_YARN ? 0.1 * std::log((double)scaling->factor) + 1.0 : 1.0;
    return QMM_OK;
}

int qmm_kv_pool_bytes(const qmm_kv_cache* cache, size_t* bytes)
{
    if (!bytes) {
        return fail("qmm_kv_pool_bytes: bytes is null");
    }
    if (int rc = check_cache("qmm_kv_pool_bytes", cache, false)) {
        return rc;
    }
    *bytes = (size_t)cache->n_pages * cache->kv_heads * (cache->page_tokens / KV_TILE) * kv_tile_bytes(cache->fmt, cache->head_dim);
    return QMM_OK;
}

int qmm_kv_append(int device, const qmm_kv_cache* cache, const qmm_kv_batch* batch, const qmm_rope* rope, int heads, int type,
                  const void* q_dev, int64_t q_stride, const void* k_dev, int64_t k_stride, const void* v_dev, int64_t v_stride,
                  void* q_out_dev, int q_type, int64_t q_out_stride, void* stream)
{
    const char* who = "qmm_kv_append";
    if (int rc = check_cache(who, cache, true)) {
        return rc;
    }
    if (int rc = check_batch(who, cache, batch)) {
        return rc;
    }
    if (heads < 0 || heads > MAX_HEADS || (heads > 0) != (q_dev != nullptr)) {
        return fail("%s: %d query heads and q %s", who, heads, q_dev ? "given" : "null");
    }
    KvAppendArgs a = {};
    if (rope && rope->dim != 0) {
        if (rope->dim < 0 || rope->dim % 2 != 0 || rope->dim > cache->head_dim ||
            (rope->layout == QMM_ROPE_HALVES && rope->dim % 8 != 0)) {
            return fail("%s: %d rotated dimensions of %d (even; in halves a multiple of 8)", who, rope->dim, cache->head_dim);
        }
        if (rope->layout != QMM_ROPE_PAIRS && rope->layout != QMM_ROPE_HALVES) {
            return fail("%s: unknown rotary layout %d", who, rope->layout);
        }
        if (!rope->inv_freq_dev || reinterpret_cast<uintptr_t>(rope->inv_freq_dev) % 8 != 0) {
            return fail("%s: inv_freq is null or not 8-byte aligned", who);
        }
        a.rope = {rope->dim, rope->layout == QMM_ROPE_HALVES, rope->inv_freq_dev, rope->gain};
    }
    if (batch->rows == 0 || batch->batch == 0) {
        return QMM_OK;
    }
    const int64_t kv_width = (int64_t)cache->kv_heads * cache->head_dim, q_width = (int64_t)heads * cache->head_dim;
    if (int rc = check_rows(who, "k", k_dev, type, k_stride, kv_width)) {
        return rc;
    }
    if (int rc = check_rows(who, "v", v_dev, type, v_stride, kv_width)) {
        return rc;
    }
    if (heads > 0) {
        if (int rc = check_rows(who, "q", q_dev, type, q_stride, q_width)) {
            return rc;
        }
        if (int rc = check_rows(who, "q_out", q_out_dev, q_type, q_out_stride, q_width)) {
            return rc;
        }
        const bool in_place = q_out_dev == q_dev && q_type == type && q_out_stride == q_stride;
        if (!in_place && overlap(q_dev, type, q_stride, q_width, q_out_dev, q_type, q_out_stride, q_width, batch->rows)) {
            return fail("%s: q_out overlaps q without being q", who);
        }
        if (overlap(k_dev, type, k_stride, kv_width, q_out_dev, q_type, q_out_stride, q_width, batch->rows) ||
            overlap(v_dev, type, v_stride, kv_width, q_out_dev, q_type, q_out_stride, q_width, batch->rows)) {
            return fail("%s: q_out overlaps k or v", who);
        }
    }
    DeviceGuard guard(device);
    if (!guard.ok) {
        return fail_cuda(guard.err, "cudaSetDevice");
    }
    int* status = nullptr;
    if (int rc = qmm_internal_status_word(device, &status)) {
        return rc;
    }
    a.pool = pool_of(*cache);
    a.seqs = seqs_of(*batch, status);
    a.heads = heads;
    a.q = q_dev, a.k = k_dev, a.v = v_dev;
    a.q_stride = q_stride, a.k_stride = k_stride, a.v_stride = v_stride;
    a.q_out = q_out_dev;
    a.q_out_stride = q_out_stride;
    a.type = type, a.q_type = q_type;
    const cudaError_t e = launch_kv_append(a, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? QMM_OK : fail_cuda(e, who);
}

int qmm_kv_read(int device, const qmm_kv_cache* cache, const qmm_kv_batch* batch, void* k_out_dev, int64_t k_stride,
                void* v_out_dev, int64_t v_stride, int type, void* stream)
{
    const char* who = "qmm_kv_read";
    if (int rc = check_cache(who, cache, true)) {
        return rc;
    }
    if (int rc = check_batch(who, cache, batch)) {
        return rc;
    }
    if (batch->rows == 0 || batch->batch == 0) {
        return QMM_OK;
    }
    const int64_t width = (int64_t)cache->kv_heads * cache->head_dim;
    if (int rc = check_rows(who, "k_out", k_out_dev, type, k_stride, width)) {
        return rc;
    }
    if (int rc = check_rows(who, "v_out", v_out_dev, type, v_stride, width)) {
        return rc;
    }
    if (overlap(k_out_dev, type, k_stride, width, v_out_dev, type, v_stride, width, batch->rows)) {
        return fail("%s: k_out overlaps v_out", who);
    }
    DeviceGuard guard(device);
    if (!guard.ok) {
        return fail_cuda(guard.err, "cudaSetDevice");
    }
    int* status = nullptr;
    if (int rc = qmm_internal_status_word(device, &status)) {
        return rc;
    }
    KvReadArgs a = {pool_of(*cache), seqs_of(*batch, status), k_out_dev, v_out_dev, k_stride, v_stride, type};
    const cudaError_t e = launch_kv_read(a, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? QMM_OK : fail_cuda(e, who);
}

int qmm_kv_attention(int device, const qmm_kv_cache* cache, const qmm_kv_batch* batch, int heads, const void* q_dev, int q_type,
                     int64_t q_stride, void* out_dev, int out_type, int64_t out_stride, float scale, int window,
                     void* workspace_dev, void* stream)
{
    const char* who = "qmm_kv_attention";
    if (int rc = check_cache(who, cache, true)) {
        return rc;
    }
    if (int rc = check_batch(who, cache, batch)) {
        return rc;
    }
    if (heads < 1 || heads > MAX_HEADS || heads % cache->kv_heads != 0) {
        return fail("%s: %d query heads do not divide over %d kv heads", who, heads, cache->kv_heads);
    }
    if (window < 0 || !std::isfinite(scale)) {
        return fail("%s: a negative window or a scale that is not finite", who);
    }
    if (batch->rows == 0 || batch->batch == 0) {
        return QMM_OK;
    }
    const int64_t width = (int64_t)heads * cache->head_dim;
    if (int rc = check_rows(who, "q", q_dev, q_type, q_stride, width)) {
        return rc;
    }
    if (int rc = check_rows(who, "out", out_dev, out_type, out_stride, width)) {
        return rc;
    }
    if (overlap(q_dev, q_type, q_stride, width, out_dev, out_type, out_stride, width, batch->rows)) {
        return fail("%s: out overlaps q", who);
    }
    if (!workspace_dev || reinterpret_cast<uintptr_t>(workspace_dev) % 256 != 0) {
        return fail("%s: the workspace is null or not 256-byte aligned", who);
    }
    DeviceGuard guard(device);
    if (!guard.ok) {
        return fail_cuda(guard.err, "cudaSetDevice");
    }
    int* status = nullptr;
    if (int rc = qmm_internal_status_word(device, &status)) {
        return rc;
    }
    KvAttnArgs a = {};
    a.pool = pool_of(*cache);
    a.seqs = seqs_of(*batch, status);
    a.heads = heads;
    a.group = heads / cache->kv_heads;
    a.q = q_dev;
    a.out = out_dev;
    a.q_stride = q_stride, a.out_stride = out_stride;
    a.q_type = q_type, a.out_type = out_type;
    a.scale = scale;
    a.window = window;
    a.workspace = static_cast<uint8_t*>(workspace_dev);
    const int sms = sm_count_of(device);
    const cudaError_t e = kv_takes_prompt(a) ? launch_kv_prompt(a, sms, static_cast<cudaStream_t>(stream))
                                             : launch_kv_rows(a, sms, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? QMM_OK : fail_cuda(e, who);
}

}  // extern "C"
