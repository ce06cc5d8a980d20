// Log-probabilities of given tokens, with the entropy and the top
// alternatives of each row of logits, in one pass over the logits.
//
//   m = max x,  Z = sum e^(x - m),  lse = m + log Z
//   logprob = x_token - lse,  entropy = lse - (sum x e^(x - m)) / Z
//   alternatives: the k largest x, ties to the lowest index; x - lse each
// A masked logit (-inf) adds nothing to any of the sums; a row of nothing but
// -inf has log-probabilities of -inf and entropy 0.
//
// Memory bound: one read of the logits, 16 bytes a load and four of them in flight a
// thread.  A cluster of CTAs takes a row, each a slice of the vocabulary;
// statistics and candidates meet in the first CTA's shared memory.  Measured: 512
// rows of 151936 fp32 without alternatives 52 us (6.0 TB/s), with 5 of them 59; 1024 rows of
// bf16 with 5 75.5 us (4.1 TB/s; 64 us without: one exponential a logit and its conversions take
// the issue slots at two bytes a logit); 27 rows of fp32 with 20 13.3 us, without 6.7.
//
// Sums: a thread's exponentials are taken against a reference that moves only when a
// logit passes it by 8, so that almost no load rescales anything; an exponent of up
// to 8 is rounded by 8 u, u = 2^-24, which is what its exponential is then off by (ex2.approx itself by
// 4 u at most).
//
// Candidates: the pass leaves each thread with the largest of its logits.  A thread whose
// maximum is passed by k others has nothing among the alternatives; the logits of the
// rest (about k of 512) are looked through once more, mostly in L2, by all threads.  To
// know them without
// sorting 512 values: with W warps and r = ceil(k / W), the smallest of the warps' r-th
// largest maxima is reached by k maxima at least, so that only those that reach
// it (about a hundred) are counted against one another.  What reaches it in the logits
// of the threads that are left is kept in shared memory and ranked.  A slice
// with more of that than the buffer holds (one value all over) finds its k largest
// one after another instead, a pass each.
#include <type_traits>
#include <cooperative_groups.h>
#include "serving.cuh"
namespace cg = cooperative_groups;

namespace qvl {
namespace {
constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kCand = 1024;
constexpr int kMaxCluster = 8;
constexpr int kShare = 128;             // candidates that a slice may hand on unranked
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kFar = 8.0f;
constexpr float kGone = 1000.0f;        // an exponential from this far below is 0

// Value and index as one number, larger where the alternative comes first: by value, then
// by lower index (both zeros are one value).
using Key = unsigned long long;
__device__ __forceinline__ Key key_of(float v, int i) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return (Key)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (uint32_t)~i;
}
__device__ __forceinline__ float value_of(Key k) {
    const uint32_t b = (uint32_t)(k >> 32);
    return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ int index_of(Key k) { return (int)~(uint32_t)k; }
// How many of keys[0, n) come before k; keys are 16-byte aligned, and what lies between n
// and the next even number is 0.
__device__ __forceinline__ int rank_of(const Key *keys, int n, Key k) {
    int r = 0;
#pragma unroll 4
    for (int d = 0; d < n; d += 2) {
        const ulonglong2 x = *reinterpret_cast<const ulonglong2 *>(keys + d);
        r += (x.x > k) + (x.y > k);
    }
    return r;
}

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float redux_max(float v) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}

// A reference m, z = sum e^(x - m), s = sum (x - m) e^(x - m).
struct Stats {
    float m, z, s;
};
__device__ __forceinline__ Stats rebase(const Stats &a, float m) {
    if (a.z == 0.0f || a.m == m) return {m, a.z, a.s};
    // (from lowest values, as masks write them, the way is so far that z d would pass the type's
    // range: where f is 0 already, any d will do)
    const float d = fmaxf(a.m - m, -kGone), f = ex2(d * kLog2e);
    return {m, a.z * f, (a.s + a.z * d) * f};
}
__device__ __forceinline__ Stats warp_join(const Stats &t) {
    const float m = redux_max(t.z == 0.0f ? -INFINITY : t.m);
    Stats r = rebase(t, m == -INFINITY ? 0.0f : m);
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        r.z += __shfl_xor_sync(~0u, r.z, o);
        r.s += __shfl_xor_sync(~0u, r.s, o);
    }
    return r;
}
// Two fp32 operations in one instruction: the sums are bound by issue next to memory.
__device__ __forceinline__ uint64_t two(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 parts(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
// N logits (even); `top` is the largest of them.
template <int N> __device__ __forceinline__ void take(Stats &t, const float (&x)[N], float top) {
    if (top > t.m + kFar || t.z == 0.0f) t = rebase(t, top == -INFINITY ? 0.0f : top);
    uint64_t z = two(t.z, 0.0f), s = two(t.s, 0.0f);
    const uint64_t m = two(-t.m, -t.m), l = two(kLog2e, kLog2e);
#pragma unroll
    for (int e = 0; e < N; e += 2) {
        const uint64_t d = add2(two(x[e], x[e + 1]), m);
        const float2 y = parts(mul2(d, l)), w = parts(d);
        const uint64_t p = two(ex2(y.x), ex2(y.y));
        z = add2(z, p);                     // (NaN stays in it)
        s = fma2(p, two(fmaxf(w.x, -kGone), fmaxf(w.y, -kGone)), s);     // a masked logit: 0, not 0 * inf
    }
    t.z = parts(z).x + parts(z).y;
    t.s = parts(s).x + parts(s).y;
}
template <typename T> struct Vec {
    static constexpr int N = 16 / sizeof(T);
    uint4 v;
    __device__ __forceinline__ void unpack(float (&x)[N]) const {
        const T *t = reinterpret_cast<const T *>(&v);
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = to_f32(t[e]);
    }
    // The largest value; -inf where there is nothing but NaN.
    __device__ __forceinline__ float largest() const {
        float m;
        if constexpr (sizeof(T) == 4) {
            m = fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
        } else if constexpr (std::is_same<T, __half>::value) {
            const __half2 *h = reinterpret_cast<const __half2 *>(&v);
            const __half2 x = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
            m = __half2float(__hmax(__low2half(x), __high2half(x)));
        } else {
            const __nv_bfloat162 *h = reinterpret_cast<const __nv_bfloat162 *>(&v);
            const __nv_bfloat162 x = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
            m = __bfloat162float(__hmax(__low2bfloat16(x), __high2bfloat16(x)));
        }
        return m == m ? m : -INFINITY;
    }
};
}  // namespace

// kAhead: 16-byte loads of a thread in flight; kPerSM: CTAs on an SM.
template <typename T, int kAhead, int kPerSM>
__global__ void __launch_bounds__(kThreads, kPerSM) token_logprobs_kernel(const __grid_constant__ LogprobArgs a) {
    constexpr int N = Vec<T>::N;
    __shared__ __align__(16) Key cand[kCand + 2];
    __shared__ __align__(16) Key all[kMaxCluster * kShare + 2];      // the first CTA's: everyone's candidates
    __shared__ Stats wst[kWarps];
    __shared__ Stats cst;
    __shared__ float wtau[kWarps];
    __shared__ float lse_s;
    __shared__ float max_s[kThreads];
    __shared__ int asked[kThreads];             // threads whose logits are looked through again
    __shared__ int n_cand, n_max, n_asked;
    __shared__ Key best[kWarps];
    __shared__ int have[kMaxCluster + 1];

    cg::cluster_group cl = cg::this_cluster();
    const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    const int row = blockIdx.x / C;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const T *x = reinterpret_cast<const T *>(a.logits) + (long)row * a.stride;
    // elements before the first 16-byte boundary, whole loads, and the rest; the first CTA
    // takes what is not a whole load
    const int head = min((int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T), a.V);
    const int loads = (a.V - head) / N, tail = head + loads * N;
    const int per = (loads + C - 1) / C, lo = min(rank * per, loads), hi = min(lo + per, loads);
    const int loose = rank == 0 ? head + a.V - tail : 0;
    // (ordinary loads: the launch begins before the one that writes the logits has ended, and the
    // read-only path is for what nobody writes in a kernel's lifetime)
    const uint4 *xv = reinterpret_cast<const uint4 *>(x + head);
    auto loose_at = [&](int i) { return i < head ? i : tail + i - head; };

    pdl_launch_dependents();
    if (tid == 0) {
        n_cand = 0;
        n_max = 0;
        n_asked = 0;
    }
    pdl_wait();
    // no load: -inf, which weighs nothing
    auto none = [] {
        Vec<T> v;
        T *t = reinterpret_cast<T *>(&v.v);
#pragma unroll
        for (int e = 0; e < N; ++e) t[e] = from_f32<T>(-INFINITY);
        return v;
    };
    const float own = tid < loose ? to_f32(x[loose_at(tid)]) : -INFINITY;
    float mx = own == own ? own : -INFINITY;
    Stats st{0.0f, 0.0f, 0.0f};
    if (tid < loose) {
        const float f[2] = {own, -INFINITY};
        take(st, f, mx);
    }
    for (int i = lo + tid; i < hi; i += kAhead * kThreads) {
        Vec<T> v[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (i + u * kThreads < hi) v[u].v = xv[i + u * kThreads];
            else v[u] = none();
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            float f[N];
            v[u].unpack(f);
            const float top = v[u].largest();
            take(st, f, top);
            mx = fmaxf(mx, top);
        }
    }
    st = warp_join(st);
    if (lane == 0) wst[warp] = st;
    __syncthreads();
    if (warp == 0) {
        st = warp_join(lane < kWarps ? wst[lane] : Stats{0.0f, 0.0f, 0.0f});
        if (lane == 0) cst = st;
    }
    int nc = 0;
    if (a.k > 0) {
        const int r = (a.k + kWarps - 1) / kWarps;
        float t = -INFINITY, rest = mx;
        for (int n = 0; n < r; ++n) {
            t = redux_max(rest);
            if (t == -INFINITY) break;
            if (lane == __ffs(__ballot_sync(~0u, rest == t)) - 1) rest = -INFINITY;
        }
        if (lane == 0) wtau[warp] = t;
        __syncthreads();
        float tau = wtau[0];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) tau = fminf(tau, wtau[w]);
        const bool in = mx >= tau && mx != -INFINITY;
        if (in) max_s[atomicAdd(&n_max, 1)] = mx;
        __syncthreads();
        if (in) {
            int passed = 0;
#pragma unroll 8
            for (int d = 0; d < n_max; ++d) passed += max_s[d] > mx;
            if (passed < a.k) asked[atomicAdd(&n_asked, 1)] = tid;
        }
        __syncthreads();
        auto offer = [&](float v, int i) {
            if (v >= tau && v != -INFINITY) {
                const int at = atomicAdd(&n_cand, 1);
                if (at < kCand) cand[at] = key_of(v, i);
            }
        };
        if (tid < loose) offer(own, loose_at(tid));
        const int turns = (per + kThreads - 1) / kThreads;
        for (int j = tid; j < n_asked * turns; j += kThreads) {
            const int q = j / turns, i = lo + asked[q] + (j - q * turns) * kThreads;
            if (i >= hi) continue;
            Vec<T> w;
            w.v = xv[i];
            if (w.largest() >= tau) {
                float f[N];
                w.unpack(f);
#pragma unroll
                for (int e = 0; e < N; ++e) offer(f[e], head + i * N + e);
            }
        }
        __syncthreads();
        nc = n_cand;
    }
    if (nc > kCand) {
        // one value after another
        Key past = ~0ull;
        int n = 0;
        for (; n < a.k; ++n) {
            Key b = 0;
            auto look = [&](float w, int i) {
                if (w > -INFINITY) {
                    const Key k = key_of(w, i);
                    if (k < past && k > b) b = k;
                }
            };
            if (tid < loose) look(own, loose_at(tid));
            for (int i = lo + tid; i < hi; i += kThreads) {
                Vec<T> w;
                w.v = xv[i];
                float f[N];
                w.unpack(f);
#pragma unroll
                for (int e = 0; e < N; ++e) look(f[e], head + i * N + e);
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) b = max(b, __shfl_xor_sync(~0u, b, o));
            if (lane == 0) best[warp] = b;
            __syncthreads();
            b = best[0];
#pragma unroll
            for (int w = 1; w < kWarps; ++w) b = max(b, best[w]);
            __syncthreads();
            if (b == 0) break;
            if (tid == 0) cand[n] = b;
            past = b;
        }
        nc = n;
    } else if (nc > kShare) {
        // (all candidates are read before the best are written over them)
        if (tid < 2) cand[nc + tid] = 0;
        __syncthreads();
        Key mine[kCand / kThreads];
        int at[kCand / kThreads];
#pragma unroll
        for (int u = 0; u < kCand / kThreads; ++u) {
            const int c = tid + u * kThreads;
            mine[u] = c < nc ? cand[c] : 0;
            at[u] = c < nc ? rank_of(cand, nc, mine[u]) : kCand;
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kCand / kThreads; ++u)
            if (at[u] < a.k) cand[at[u]] = mine[u];
        nc = a.k;
    }
    __syncthreads();
    if (tid == 0) n_cand = nc;
    if (C > 1) cl.sync();
    else __syncthreads();
    if (rank == 0) {
        if (warp == 0) {
            const Stats t = warp_join(lane < C ? *cl.map_shared_rank(&cst, lane) : Stats{0.0f, 0.0f, 0.0f});
            int upto = lane < C ? *cl.map_shared_rank(&n_cand, lane) : 0;
#pragma unroll
            for (int o = 1; o < kMaxCluster; o <<= 1) {
                const int up = __shfl_up_sync(~0u, upto, o);
                if (lane >= o) upto += up;
            }
            if (lane < C) have[lane + 1] = upto;
            if (lane == 0) {
                have[0] = 0;
                const float lz = logf(t.z), lse = t.z == 0.0f ? -INFINITY : t.m + lz;
                const int tk = a.tokens[row];
                float lp = 0.0f;
                if (tk >= 0 && tk < a.V) {
                    const float w = to_f32(x[tk]);
                    // (the logits' own size does not round the difference)
                    lp = w == -INFINITY && t.z == t.z ? -INFINITY : (w - t.m) - lz;
                }
                a.logprobs[row] = lp;
                if (a.entropy) a.entropy[row] = t.z == 0.0f ? 0.0f : lz - t.s / t.z;
                lse_s = lse;
                cst = t;
            }
        }
        __syncthreads();
        const int n = have[C];
        const float lse = lse_s, m = cst.m, lz = logf(cst.z);
        for (int e = tid; e < n; e += kThreads) {
            int c = 0;
            while (e >= have[c + 1]) ++c;
            all[e] = cl.map_shared_rank(cand, c)[e - have[c]];
        }
        if (tid < 2) all[n + tid] = 0;
        __syncthreads();
        for (int e = tid; e < n; e += kThreads) {
            const Key k = all[e];
            const int at = rank_of(all, n, k);
            if (at < a.k) {
                a.top_ids[(long)row * a.k + at] = index_of(k);
                a.top_lp[(long)row * a.k + at] = (value_of(k) - m) - lz;
            }
        }
        // fewer finite logits than alternatives: the lowest -inf ones follow
        if (n < a.k && warp == 0) {
            int at0 = n;
            for (int i0 = 0; i0 < a.V && at0 < a.k; i0 += 32) {
                const bool is = i0 + lane < a.V && to_f32(x[i0 + lane]) == -INFINITY;
                const unsigned b = __ballot_sync(~0u, is);
                const int at = at0 + __popc(b & ((1u << lane) - 1));
                if (is && at < a.k) {
                    a.top_ids[(long)row * a.k + at] = i0 + lane;
                    a.top_lp[(long)row * a.k + at] = lse == lse ? -INFINITY : lse;
                }
                at0 += __popc(b);
            }
            // and then nothing is left but NaN
            for (at0 += lane; at0 < a.k; at0 += 32) {
                a.top_ids[(long)row * a.k + at0] = -1;
                a.top_lp[(long)row * a.k + at0] = NAN;
            }
        }
    }
    if (C > 1) cl.sync();           // (the first CTA reads the others' shared memory)
}

namespace {
template <typename T>
cudaError_t launch_t(const LogprobArgs &a, cudaStream_t st) {
    // Slices of 2048 logits at least, and two CTAs per SM at most: what a CTA does beside
    // its loads costs more than a shorter slice gives (128 rows of 151936 fp32, 20
    // alternatives: 51 us with clusters of 8, 38 with 4, 33 with 2, 45 alone)
    int C = kMaxCluster;
    while (C > 1 && (a.V / C < 2048 || (long)a.T * C > 2l * 148)) C >>= 1;
    // One wave of CTAs: more loads in flight a thread; several: more CTAs on an SM, so that
    // one's end goes on beside another's loads (27 rows of 151936 fp32: 14.5 and 19.3 us;
    // 1024 of bf16: 106 and 87; both before the second look was shared out among threads)
    const auto kern = (long)a.T * C <= 2l * 148 ? token_logprobs_kernel<T, 4, 2> : token_logprobs_kernel<T, 2, 4>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.T * C);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kern, a);
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
