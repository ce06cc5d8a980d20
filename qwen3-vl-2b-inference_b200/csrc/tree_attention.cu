// Attention of a tree of drafted tokens over the paged cache.
//
// Node i of request s (row starts[s] + i of q) sees the request's cached
// positions [0, ctx) and, of the drafted ones at positions ctx + j, itself and
// its ancestors:  out = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale q.k_t - m).
// A parent is an earlier node, so a chain of parents ends by itself; an entry
// that names no earlier node counts as a root.
#include "serving.cuh"

namespace qvl {
namespace {
constexpr int kWarps = 4;

// Rows of q that no node owns: before the first request, past the last one,
// and nodes beyond max_nodes.
__device__ __forceinline__ int node_count(const TreeArgs &a, int s, int &first) {
    first = min(max(a.starts[s], 0), a.T);
    const int end = min(max(a.starts[s + 1], first), a.T);
    return min(end - first, a.max_nodes);
}
}  // namespace

// One warp per query row and head: the running maximum, sum and weighted sum
// of a softmax in one pass; a lane holds D / 32 of the values.
template <typename T, typename C, int D>
__global__ void __launch_bounds__(kWarps * 32) tree_rows_kernel(const __grid_constant__ TreeArgs a) {
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31;
    const long w = (long)blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (w >= (long)a.T * a.NH) return;
    const int row = (int)(w / a.NH), h = (int)(w - (long)row * a.NH);
    const int kvh = h / (a.NH / a.NKV);
    T *out = reinterpret_cast<T *>(a.out) + ((long)row * a.NH + h) * D + lane * E;
    float m = -INFINITY, l = 0.0f, acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.0f;
    int s = 0, first = 0, n = 0;
    for (; s < a.S; ++s) {
        n = node_count(a, s, first);
        if (row >= first && row < first + n) break;
    }
    if (s < a.S) {
        float q[E];
        const T *qp = reinterpret_cast<const T *>(a.q) + row * a.q_stride + (long)h * D + lane * E;
#pragma unroll
        for (int e = 0; e < E; ++e) q[e] = to_f32(qp[e]) * a.scale;
        const int cap = (int)min((long)a.maxp * a.P, (long)INT32_MAX);
        const int ctx = min(max(a.ctx_lens[s], 0), cap);
        auto see = [&](int t) {
            const int pg = a.table[(size_t)s * a.maxp + t / a.P];
            if (pg < 0 || pg >= a.num_pages) return;
            const long off = (((long)pg * a.NKV + kvh) * a.P + t % a.P) * D + lane * E;
            const C *k = reinterpret_cast<const C *>(a.k_pages) + off, *v = reinterpret_cast<const C *>(a.v_pages) + off;
            float sc = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) sc += q[e] * to_f32(k[e]);
#pragma unroll
            for (int o = 16; o; o >>= 1) sc += __shfl_xor_sync(~0u, sc, o);
            const float mn = fmaxf(m, sc);
            const float al = m == mn ? 1.0f : expf(m - mn), p = expf(sc - mn);
            m = mn;
            l = l * al + p;
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] = acc[e] * al + p * to_f32(v[e]);
        };
        for (int t = 0; t < ctx; ++t) see(t);
        for (int i = row - first; i >= 0;) {
            if (i < cap - ctx) see(ctx + i);
            const int par = a.parents[first + i];
            i = par < i ? par : -1;
        }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) out[e] = from_f32<T>(l == 0.0f ? 0.0f : acc[e] / l);
}

size_t tree_workspace_bytes(int, int, int, int, int, int, int) { return 0; }

namespace {
template <typename T, typename C>
cudaError_t launch_rows(const TreeArgs &a, cudaStream_t st) {
    const long warps = (long)a.T * a.NH;
    const unsigned grid = (unsigned)((warps + kWarps - 1) / kWarps);
    if (a.D == 64) tree_rows_kernel<T, C, 64><<<grid, kWarps * 32, 0, st>>>(a);
    else tree_rows_kernel<T, C, 128><<<grid, kWarps * 32, 0, st>>>(a);
    return cudaGetLastError();
}
}  // namespace

cudaError_t launch_tree_attention(const TreeArgs &a, cudaStream_t st) {
    if (a.kv_dtype == QVL_DTYPE_BF16) return launch_rows<__nv_bfloat16, __nv_bfloat16>(a, st);
    if (a.dtype == QVL_DTYPE_FP16) return launch_rows<__half, __half>(a, st);
    return launch_rows<float, __half>(a, st);
}

}  // namespace qvl
