// Host-callable launchers of the paged cache's kernels (internal to the library).
#pragma once

#include "kv_layout.cuh"

namespace qmm {

struct KvRope {
    int dim;  // 0: nothing is rotated
    bool halves;
    const double* inv_freq;
    double gain;
};
struct KvAppendArgs {
    KvPool pool;
    KvSeqs seqs;
    KvRope rope;
    int heads;  // query heads, 0: none
    const void *q, *k, *v;
    int64_t q_stride, k_stride, v_stride;  // elements
    void* q_out;
    int64_t q_out_stride;
    int type, q_type;  // QMM_OUT_*
};
cudaError_t launch_kv_append(const KvAppendArgs& a, cudaStream_t stream);

struct KvReadArgs {
    KvPool pool;
    KvSeqs seqs;
    void *k, *v;
    int64_t k_stride, v_stride;
    int type;
};
cudaError_t launch_kv_read(const KvReadArgs& a, cudaStream_t stream);

struct KvAttnArgs {
    KvPool pool;
    KvSeqs seqs;
    int heads, group;  // query heads, and how many share a kv head
    const void* q;
    void* out;
    int64_t q_stride, out_stride;
    int q_type, out_type;
    float scale;
    int window;  // 0: none
    uint8_t* workspace;
};
// Workspace: counters of the rows kernel, two of the prompt kernel, parts of the rows kernel's results.
constexpr int KV_COUNTER_BYTES = 16384 - 64, KV_PARTS_AT = 16384;
cudaError_t launch_kv_rows(const KvAttnArgs& a, int sm_count, cudaStream_t stream);
// Long prompts with bf16 results (head_dim 64 or 128).
cudaError_t launch_kv_prompt(const KvAttnArgs& a, int sm_count, cudaStream_t stream);
// Whether a call goes to launch_kv_prompt.
bool kv_takes_prompt(const KvAttnArgs& a);

}  // namespace qmm
