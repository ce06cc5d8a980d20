// Log-probabilities of given tokens, with the entropy and the top
// alternatives of each row of logits, in one pass over the logits.
//
//   m = max x,  Z = sum e^(x - m),  lse = m + log Z
//   logprob = x_token - lse,  entropy = lse - (sum x e^(x - m)) / Z
//   alternatives: the k largest x, ties to the lowest index; x - lse each
// A masked logit (-inf) adds nothing to any of the sums; a row of nothing but
// -inf has log-probabilities of -inf and entropy 0.
//
// Memory bound.  A cluster of CTAs takes a row, each a slice of the
// vocabulary with 16-byte loads; statistics and candidates meet in the first
// CTA's shared memory.
//
// Candidates: the k-th largest of the threads' maxima over the first block
// of a slice is a lower bound of the slice's k-th largest value (k values reach
// it), so that only values that reach it can be among the alternatives: a few
// hundred of a slice's tens of thousands, kept in shared memory and ranked
// once.  A slice with more of them than the buffer holds (sorted or constant
// rows) finds its k largest one after another instead, each with a pass over
// the slice.
#include <cooperative_groups.h>
#include "serving.cuh"
namespace cg = cooperative_groups;

namespace qvl {
namespace {
constexpr int kThreads = 256;
constexpr int kCand = 1024;
constexpr int kMaxCluster = 8;
constexpr float kLog2e = 1.4426950408889634f;

// (value, index) order of the alternatives: larger value first, then lower index.
__device__ __forceinline__ bool before(float v, int i, float w, int j) { return v > w || (v == w && i < j); }

struct Stats {
    float m, z, s;          // max, sum of e^(x - m), sum of x e^(x - m)
};
__device__ __forceinline__ float scale_of(float m, float mm) { return m == mm ? 1.0f : exp2f((m - mm) * kLog2e); }
__device__ __forceinline__ Stats join(const Stats &a, const Stats &b) {
    const float m = fmaxf(a.m, b.m);
    const float fa = scale_of(a.m, m), fb = scale_of(b.m, m);
    return {m, a.z * fa + b.z * fb, a.s * fa + b.s * fb};
}
__device__ __forceinline__ void take(Stats &t, float x) {
    if (x > t.m) {
        const float f = scale_of(t.m, x);
        t.z *= f;
        t.s *= f;
        t.m = x;
    }
    if (x != -INFINITY) {           // NaN stays in the sums
        const float e = exp2f((x - t.m) * kLog2e);
        t.z += e;
        t.s += x * e;
    }
}
}  // namespace

template <typename T>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(const __grid_constant__ LogprobArgs a) {
    constexpr int VE = 16 / sizeof(T);
    __shared__ float cand_v[kCand];
    __shared__ int cand_i[kCand];
    __shared__ float top_v[kMaxTopK];
    __shared__ int top_i[kMaxTopK];
    __shared__ Stats wst[kThreads / 32];
    __shared__ Stats cst;
    __shared__ float tmax[kThreads];
    __shared__ float tau_s, tok_x;
    __shared__ int n_cand, n_top;
    __shared__ float best_v[kThreads / 32];
    __shared__ int best_i[kThreads / 32];

    cg::cluster_group cl = cg::this_cluster();
    const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    const int row = blockIdx.x / C;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const T *x = reinterpret_cast<const T *>(a.logits) + (long)row * a.stride;
    const int per = ((a.V + C - 1) / C + VE - 1) / VE * VE;
    const int lo = min(rank * per, a.V), hi = min(lo + per, a.V);

    if (tid == 0) {
        n_cand = 0;
        n_top = 0;
        tau_s = -INFINITY;
    }
    // lower bound of the slice's k-th largest
    float mx = -INFINITY;
    for (int i = lo + tid; i < min(hi, lo + 16 * kThreads); i += kThreads) mx = fmaxf(mx, to_f32(x[i]));
    tmax[tid] = mx;
    __syncthreads();
    if (a.k > 0 && a.k <= kThreads) {
        int r = 0;
        for (int i = 0; i < kThreads; ++i) r += before(tmax[i], i, mx, tid);
        if (r == a.k - 1) tau_s = mx;
    }
    __syncthreads();
    const float tau = tau_s;

    Stats st{-INFINITY, 0.0f, 0.0f};
    for (int i = lo + tid; i < hi; i += kThreads) {
        const float v = to_f32(x[i]);
        take(st, v);
        if (a.k > 0 && v >= tau && v != -INFINITY) {
            const int at = atomicAdd(&n_cand, 1);
            if (at < kCand) {
                cand_v[at] = v;
                cand_i[at] = i;
            }
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const Stats b{__shfl_xor_sync(~0u, st.m, o), __shfl_xor_sync(~0u, st.z, o), __shfl_xor_sync(~0u, st.s, o)};
        st = join(st, b);
    }
    if (lane == 0) wst[warp] = st;
    __syncthreads();
    if (tid == 0) {
        Stats t = wst[0];
        for (int w = 1; w < kThreads / 32; ++w) t = join(t, wst[w]);
        cst = t;
    }
    const int nc = n_cand;
    if (nc <= kCand) {
        for (int c = tid; c < nc; c += kThreads) {
            int r = 0;
            const float v = cand_v[c];
            const int i = cand_i[c];
            for (int d = 0; d < nc; ++d) r += before(cand_v[d], cand_i[d], v, i);
            if (r < a.k) {
                top_v[r] = v;
                top_i[r] = i;
            }
        }
        if (tid == 0) n_top = min(nc, a.k);
    } else {
        float pv = INFINITY;
        int pi = -1;
        for (int r = 0; r < a.k; ++r) {
            float bv = -INFINITY;
            int bi = INT32_MAX;
            for (int i = lo + tid; i < hi; i += kThreads) {
                const float v = to_f32(x[i]);
                if (v != -INFINITY && (v < pv || (v == pv && i > pi)) && before(v, i, bv, bi)) {
                    bv = v;
                    bi = i;
                }
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                const float v = __shfl_xor_sync(~0u, bv, o);
                const int i = __shfl_xor_sync(~0u, bi, o);
                if (before(v, i, bv, bi)) {
                    bv = v;
                    bi = i;
                }
            }
            if (lane == 0) {
                best_v[warp] = bv;
                best_i[warp] = bi;
            }
            __syncthreads();
            bv = best_v[0];
            bi = best_i[0];
            for (int w = 1; w < kThreads / 32; ++w)
                if (before(best_v[w], best_i[w], bv, bi)) {
                    bv = best_v[w];
                    bi = best_i[w];
                }
            if (bi == INT32_MAX) break;
            if (tid == 0) {
                top_v[r] = bv;
                top_i[r] = bi;
                n_top = r + 1;
            }
            pv = bv;
            pi = bi;
            __syncthreads();
        }
    }
    cl.sync();
    if (rank == 0) {
        __shared__ int have[kMaxCluster + 1];
        if (tid == 0) {
            Stats t = cst;
            int n = 0;
            for (int c = 0; c < C; ++c) {
                if (c) t = join(t, *cl.map_shared_rank(&cst, c));
                have[c] = n;
                n += *cl.map_shared_rank(&n_top, c);
            }
            have[C] = n;
            const float lse = t.m == -INFINITY && t.z == 0.0f ? -INFINITY : t.m + logf(t.z);
            const int tk = a.tokens[row];
            float lp = 0.0f;
            if (tk >= 0 && tk < a.V) {
                const float v = to_f32(x[tk]);
                lp = v == -INFINITY && t.z == t.z ? -INFINITY : v - lse;
            }
            a.logprobs[row] = lp;
            if (a.entropy) a.entropy[row] = t.z == 0.0f ? 0.0f : lse - t.s / t.z;
            tok_x = lse;
        }
        __syncthreads();
        const int n = have[C];
        const float lse = tok_x;
        for (int e = tid; e < n; e += kThreads) {
            int c = 0;
            while (e >= have[c + 1]) ++c;
            cand_v[e] = cl.map_shared_rank(top_v, c)[e - have[c]];
            cand_i[e] = cl.map_shared_rank(top_i, c)[e - have[c]];
        }
        __syncthreads();
        for (int e = tid; e < n; e += kThreads) {
            int r = 0;
            for (int d = 0; d < n; ++d) r += before(cand_v[d], cand_i[d], cand_v[e], cand_i[e]);
            if (r < a.k) {
                a.top_ids[(long)row * a.k + r] = cand_i[e];
                a.top_lp[(long)row * a.k + r] = cand_v[e] - lse;
            }
        }
        // fewer finite logits than alternatives: the lowest -inf ones follow
        if (n < a.k && warp == 0) {
            int r = n;
            for (int i0 = 0; i0 < a.V && r < a.k; i0 += 32) {
                const bool is = i0 + lane < a.V && to_f32(x[i0 + lane]) == -INFINITY;
                const unsigned b = __ballot_sync(~0u, is);
                const int at = r + __popc(b & ((1u << lane) - 1));
                if (is && at < a.k) {
                    a.top_ids[(long)row * a.k + at] = i0 + lane;
                    a.top_lp[(long)row * a.k + at] = lse == lse ? -INFINITY : lse;
                }
                r += __popc(b);
            }
            // and then nothing is left but NaN
            for (r += lane; r < a.k; r += 32) {
                a.top_ids[(long)row * a.k + r] = -1;
                a.top_lp[(long)row * a.k + r] = NAN;
            }
        }
    }
    cl.sync();
}

namespace {
template <typename T>
cudaError_t launch_t(const LogprobArgs &a, cudaStream_t st) {
    int C = kMaxCluster;
    while (C > 1 && a.V / C < 2048) C >>= 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.T * C);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T>, a);
}
}  // namespace

cudaError_t launch_token_logprobs(const LogprobArgs &a, cudaStream_t st) {
    switch (a.dtype) {
    case QVL_DTYPE_FP32: return launch_t<float>(a, st);
    case QVL_DTYPE_FP16: return launch_t<__half>(a, st);
    default: return launch_t<__nv_bfloat16>(a, st);
    }
}

}  // namespace qvl
