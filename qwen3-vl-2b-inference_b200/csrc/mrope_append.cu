// Norms of the query and key heads, rotary positions with several axes, and
// the write of keys and values into their cache slots, in one pass.
//
//   x' = x / sqrt(mean(x^2) + eps) * w            (per head, optional)
//   y_i       = x'_i c_i - x'_{i+D/2} s_i          c_i, s_i: row
//   y_{i+D/2} = x'_{i+D/2} c_i + x'_i s_i          positions[axes[i], t], column i
//                                                  of the rotary table
// q goes to q_out in its own type, k (rotated) and v are rounded to the
// cache's type and written at slot = page * P + offset of [page, NKV, P, D].
//
// Memory bound: (2 NH + 2 NKV) D values and 2 NKV D cache values per token.
// A lane holds four values of a head's first half and the same four of its second
// half, so that both partners of a pair sit in one thread; a head takes 8 to 32
// lanes, and a lane group kRows heads.  A CTA takes all heads of a token (or a
// part of them, blockIdx.y, where 256 threads do not hold them) and goes from
// token to token.  While it works on one, the next token's heads are copied into
// shared memory and its cosines and sines gathered (two dependent reads, positions
// and then up to three rows of the table) by a thread for each frequency; norm
// weights are laid there as fp32 once.  Held in registers instead, the
// heads on their way leave too few of them or too few CTAs.
// fp32 throughout; the only roundings are the outputs'.
// Measured (16 query and 8 key heads of 128, fp32, fp16 cache): 8200 tokens 43 us
// (5.5 TB/s; 47 with the heads in registers), 300 tokens 4.8 us, 27 tokens 3.6 us, both
// a chain of three reads; 2049 tokens of bf16, 32 and 8 heads of 64, 8.9 us (12 with four
// heads to a lane group).  Four CTAs of 256 threads on an SM; five 43 and 11 us, and six
// spill: 55 and 13.
#include <algorithm>
#include "serving.cuh"

namespace qvl {
namespace {
constexpr int kThreads = 256;           // at most
constexpr int kRows = 2;
constexpr int kPerSM = 4;
constexpr int kStages = 2;              // tokens of a CTA in shared memory
constexpr int VE = 4;

// N bytes from memory into shared memory, behind the calling thread's back
template <int N>
__device__ __forceinline__ void copy_async(void *to, const void *from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from), "n"(N)
                 : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// four values as loaded and stored
template <int BYTES> struct RawOf;
template <> struct RawOf<4> { using R = float4; };
template <> struct RawOf<2> { using R = uint2; };
template <typename T> using Raw = typename RawOf<sizeof(T)>::R;
template <typename T>
__device__ __forceinline__ void unpack(const Raw<T> &r, float (&f)[VE]) {
    const T *e = reinterpret_cast<const T *>(&r);
#pragma unroll
    for (int i = 0; i < VE; ++i) f[i] = to_f32(e[i]);
}
__device__ __forceinline__ void load_s(const float *p, float (&f)[VE]) {
    unpack<float>(*reinterpret_cast<const float4 *>(p), f);
}
template <typename T>
__device__ __forceinline__ void store(T *p, const float (&f)[VE]) {
    Raw<T> r;
    T *e = reinterpret_cast<T *>(&r);
#pragma unroll
    for (int i = 0; i < VE; ++i) e[i] = from_f32<T>(f[i]);
    *reinterpret_cast<Raw<T> *>(p) = r;
}

__device__ __forceinline__ float weight_at(const NormWeight &n, int dtype, int j) {
    if (!n.w) return 1.0f;
    switch (dtype) {
    case QVL_DTYPE_INT8: return (float)reinterpret_cast<const int8_t *>(n.w)[j] * n.scales[j / n.group];
    case QVL_DTYPE_FP16: return to_f32(reinterpret_cast<const __half *>(n.w)[j]);
    case QVL_DTYPE_BF16: return to_f32(reinterpret_cast<const __nv_bfloat16 *>(n.w)[j]);
    default: return reinterpret_cast<const float *>(n.w)[j];
    }
}
}  // namespace

// Rows 0..NH-1 of a token are queries, the next NKV keys, the last NKV values; a lane
// group has rows r0, r0 + groups, ... of the CTA's part.
template <typename T, typename C, int D>
__global__ void __launch_bounds__(kThreads, kPerSM) mrope_append_kernel(const __grid_constant__ MropeArgs a) {
    constexpr int H = D / 2, LPH = H / VE;
    __shared__ Raw<T> x_s[kStages][kRows][2][kThreads];     // a thread reads only what it copied itself
    __shared__ __align__(16) float w_s[2][D];
    __shared__ __align__(16) float cs_s[2][2][H];
    const int tid = threadIdx.x, rows = a.NH + 2 * a.NKV;
    const int groups = (int)blockDim.x / LPH, lane_j = (tid % LPH) * VE;
    pdl_launch_dependents();
    pdl_wait();

    const int hop = gridDim.x;
    auto is_q = [&](int r) { return r < a.NH; };
    auto is_k = [&](int r) { return r >= a.NH && r < a.NH + a.NKV; };
    const int r0 = (int)blockIdx.y * kRows * groups + tid / LPH;
    auto fetch = [&](int t, int stage) {
        if (t < a.T) {
#pragma unroll
            for (int u = 0; u < kRows; ++u) {
                const int r = r0 + u * groups;
                if (r >= rows) break;
                const T *p = is_q(r)   ? reinterpret_cast<const T *>(a.q) + t * a.q_stride + (long)r * D
                             : is_k(r) ? reinterpret_cast<const T *>(a.k) + t * a.k_stride + (long)(r - a.NH) * D
                                       : reinterpret_cast<const T *>(a.v) + t * a.v_stride + (long)(r - a.NH - a.NKV) * D;
                copy_async<sizeof(Raw<T>)>(&x_s[stage][u][0][tid], p + lane_j);
                copy_async<sizeof(Raw<T>)>(&x_s[stage][u][1][tid], p + lane_j + H);
            }
        }
        copies_commit();
    };
    int t = blockIdx.x;
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) fetch(t + i * hop, i);

    // frequency tid of the next token: its position, and whether that is in the table
    const bool turns = tid < H;
    const int ax = turns ? a.axes[tid] : 0;
    const bool ax_ok = ax >= 0 && ax < a.n_axes;
    auto position = [&](int t) {
        return turns && ax_ok && t < a.T ? a.positions[ax * a.pos_stride + t] : -1;
    };
    bool bad = false;
    float cn = 0.0f, sn = 0.0f;
    auto gather = [&](int p) {
        bad = turns && (p < 0 || p >= a.max_pos);
        if (turns && !bad) {
            cn = a.cos_t[(size_t)p * H + tid];
            sn = a.sin_t[(size_t)p * H + tid];
        }
    };
    int pn = position(t);
    for (int j = tid; j < 2 * D; j += blockDim.x)
        w_s[0][j] = j < D ? weight_at(a.qn, a.w_dtype, j) : weight_at(a.kn, a.w_dtype, j - D);
    gather(pn);
    pn = position(t + hop);
    if (turns) cs_s[0][0][tid] = cn, cs_s[0][1][tid] = sn;

    for (int buf = 0, stage = 0; t < a.T; t += hop, buf ^= 1, stage = stage + 1 == kStages ? 0 : stage + 1) {
        fetch(t + (kStages - 1) * hop, stage == 0 ? kStages - 1 : stage - 1);
        const long slot = a.slots[t];
        // a token with a position outside the table has no rotation: its query
        // rows are zero and its key and value are not written
        const bool none = __syncthreads_or(bad);
        gather(pn);
        pn = position(t + 2 * hop);
        const bool writes = !none && slot >= 0 && slot < a.num_slots;
        const long page = writes ? (int)slot / a.P : 0;
        const long off = writes ? slot - page * a.P : 0;
        float c[VE], s[VE];
        load_s(&cs_s[buf][0][lane_j], c);
        load_s(&cs_s[buf][1][lane_j], s);
        copies_wait<kStages - 1>();
#pragma unroll
        for (int u = 0; u < kRows; ++u) {
            const int r = r0 + u * groups;
            float x0[VE], x1[VE];
            unpack<T>(x_s[stage][u][0][tid], x0);
            unpack<T>(x_s[stage][u][1][tid], x1);
            const bool isq = is_q(r), isk = is_k(r);
            float ss = 0.0f;
#pragma unroll
            for (int e = 0; e < VE; ++e) ss += x0[e] * x0[e] + x1[e] * x1[e];
#pragma unroll
            for (int o = LPH / 2; o; o >>= 1) ss += __shfl_xor_sync(~0u, ss, o);
            if (r >= rows) continue;
            if (isq || isk) {
                const float inv = (isq ? a.qn.w : a.kn.w) ? rsqrtf(ss * (1.0f / D) + a.eps) : 1.0f;
                const float *w = w_s[isq ? 0 : 1] + lane_j;
                float w0[VE], w1[VE];
                load_s(w, w0);
                load_s(w + H, w1);
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    const float y0 = x0[e] * (inv * w0[e]), y1 = x1[e] * (inv * w1[e]);
                    x0[e] = none ? 0.0f : y0 * c[e] - y1 * s[e];
                    x1[e] = none ? 0.0f : y1 * c[e] + y0 * s[e];
                }
            }
            if (isq) {
                T *o = reinterpret_cast<T *>(a.q_out) + ((long)t * a.NH + r) * D + lane_j;
                store<T>(o, x0);
                store<T>(o + H, x1);
            } else if (writes) {
                C *o = reinterpret_cast<C *>(isk ? a.k_pages : a.v_pages) +
                       ((page * a.NKV + (r - a.NH - (isk ? 0 : a.NKV))) * a.P + off) * D + lane_j;
                store<C>(o, x0);
                store<C>(o + H, x1);
            }
        }
        if (turns) cs_s[buf ^ 1][0][tid] = cn, cs_s[buf ^ 1][1][tid] = sn;
    }
}

namespace {
template <typename T, typename C, int D>
cudaError_t launch_d(const MropeArgs &a, cudaStream_t st) {
    constexpr int LPH = D / 2 / VE;
    const int rows = a.NH + 2 * a.NKV;
    // a token's heads in equal parts of at most 256 threads, a thread a frequency at least
    const int most = kThreads / LPH * kRows, parts = (rows + most - 1) / most;
    const int groups = ((rows + parts - 1) / parts + kRows - 1) / kRows;
    const int threads = (std::max(groups * LPH, D / 2) + 31) / 32 * 32;
    // as many CTAs as the SMs hold at once, the tokens spread evenly over them
    const int held = std::max(148 * (kThreads * kPerSM / threads) / parts, 1);
    const int turns = (a.T + held - 1) / held;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((a.T + turns - 1) / turns, parts);
    cfg.blockDim = dim3(threads);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, mrope_append_kernel<T, C, D>, a);
}
template <typename T, typename C>
cudaError_t launch_tc(const MropeArgs &a, cudaStream_t st) {
    switch (a.D) {
    case 64: return launch_d<T, C, 64>(a, st);
    case 128: return launch_d<T, C, 128>(a, st);
    default: return launch_d<T, C, 256>(a, st);
    }
}
template <typename T>
cudaError_t launch_t(const MropeArgs &a, cudaStream_t st) {
    return a.kv_dtype == QVL_DTYPE_FP16 ? launch_tc<T, __half>(a, st) : launch_tc<T, __nv_bfloat16>(a, st);
}
}  // namespace

cudaError_t launch_mrope_append(const MropeArgs &a, cudaStream_t st) {
    switch (a.dtype) {
    case QVL_DTYPE_FP32: return launch_t<float>(a, st);
    case QVL_DTYPE_FP16: return launch_t<__half>(a, st);
    default: return launch_t<__nv_bfloat16>(a, st);
    }
}

}  // namespace qvl
