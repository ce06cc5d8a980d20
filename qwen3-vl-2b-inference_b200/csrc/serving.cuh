// Launchers of the operators that serve drafted and multimodal tokens over
// the paged cache (page_plan.cu, mrope_append.cu, tree_attention.cu,
// token_logprobs.cu); the C ABI in capi_serving.cu checks their arguments.
#pragma once
#include <cstddef>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include "common.cuh"

namespace qvl {

// ---- element types: 16- and 32-bit floats to and from fp32 ----
__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// ---- page_plan.cu ----
constexpr int kPlanMaxSeqs = 16384;       // three prefix arrays of this many words fit in shared memory
struct PlanArgs {
    const int32_t *old_len, *new_len;
    int S;
    int32_t *table;
    int P, maxp;
    int32_t *free_pages;
    const int32_t *free_count;
    int capacity;
    int32_t *free_count_out, *missing, *starts, *seq_ids, *positions, *slots;
    int max_tokens;
    // set by the launcher
    unsigned long long inv_p;
    int page_ctas;
};
cudaError_t launch_plan_pages(const PlanArgs &a, cudaStream_t st);

// ---- mrope_append.cu ----
struct NormWeight {
    const void *w;          // NULL: no norm
    const float *scales;    // INT8 weights: one scale per `group` values; NULL otherwise
    int group;
};
struct MropeArgs {
    const void *q, *k, *v;
    long q_stride, k_stride, v_stride;      // elements between tokens
    void *q_out;
    void *k_pages, *v_pages;
    const int32_t *slots, *positions, *axes;
    long pos_stride;                        // elements between the axes' rows of `positions`
    const float *cos_t, *sin_t;
    NormWeight qn, kn;
    float eps;
    int T, NH, NKV, D, P, max_pos, n_axes;
    long num_slots;
    int dtype, kv_dtype, w_dtype;
};
cudaError_t launch_mrope_append(const MropeArgs &a, cudaStream_t st);

// ---- tree_attention.cu ----
constexpr int kTreeMaxNodes = 256;        // drafted tokens of one request
struct TreeArgs {
    const void *q;
    long q_stride;
    const void *k_pages, *v_pages;
    long num_pages;
    const int32_t *table, *ctx_lens, *starts, *parents;
    int S, T, max_ctx, max_nodes;
    float scale;
    void *out;
    int NH, NKV, D, P, maxp;
    int dtype, kv_dtype;
    void *workspace;
};
size_t tree_workspace_bytes(int D);
cudaError_t launch_tree_attention(const TreeArgs &a, cudaStream_t st);
// device address (current device) of the kernel's timeout word, or nullptr
int *tree_timeout_word();

// ---- token_logprobs.cu ----
constexpr int kMaxTopK = 64;
struct LogprobArgs {
    const void *logits;
    long stride;            // elements between rows
    const int32_t *tokens;
    float *logprobs, *entropy;
    int32_t *top_ids;
    float *top_lp;
    int T, V, k, dtype;
};
cudaError_t launch_token_logprobs(const LogprobArgs &a, cudaStream_t st);

}  // namespace qvl
