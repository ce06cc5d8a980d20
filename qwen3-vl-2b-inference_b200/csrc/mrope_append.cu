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
// A lane holds 16 bytes of a head's first half and the same 16 of its second
// half, so that both partners of a pair sit in one thread and every access is
// a 16-byte one; a head takes 4 to 32 lanes.  Each lane group runs kRows heads
// of one token, whose gathered cos/sin (up to three rows of the table) then
// stay in registers.  fp32 throughout; the only roundings are the outputs'.
#include "serving.cuh"

namespace qvl {
namespace {
constexpr int kThreads = 256;
constexpr int kRows = 4;

template <int BYTES> struct Raw;
template <> struct Raw<16> { using T = uint4; };
template <> struct Raw<8> { using T = uint2; };

template <typename T, int N>
__device__ __forceinline__ void load_n(const T *p, float (&f)[N]) {
    using R = typename Raw<N * sizeof(T)>::T;
    const R r = *reinterpret_cast<const R *>(p);
    const T *e = reinterpret_cast<const T *>(&r);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = to_f32(e[i]);
}
template <typename T, int N>
__device__ __forceinline__ void store_n(T *p, const float (&f)[N]) {
    using R = typename Raw<N * sizeof(T)>::T;
    R r;
    T *e = reinterpret_cast<T *>(&r);
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = from_f32<T>(f[i]);
    *reinterpret_cast<R *>(p) = r;
}

__device__ __forceinline__ float weight_at(const NormWeight &n, int dtype, int j) {
    switch (dtype) {
    case QVL_DTYPE_INT8: return (float)reinterpret_cast<const int8_t *>(n.w)[j] * n.scales[j / n.group];
    case QVL_DTYPE_FP16: return to_f32(reinterpret_cast<const __half *>(n.w)[j]);
    case QVL_DTYPE_BF16: return to_f32(reinterpret_cast<const __nv_bfloat16 *>(n.w)[j]);
    default: return reinterpret_cast<const float *>(n.w)[j];
    }
}
}  // namespace

// One lane group (LPH lanes) per kRows consecutive head rows of one token;
// rows 0..NH-1 are queries, the next NKV keys, the last NKV values.
template <typename T, typename C, int D>
__global__ void __launch_bounds__(kThreads) mrope_append_kernel(const __grid_constant__ MropeArgs a) {
    constexpr int VE = 16 / sizeof(T), H = D / 2, LPH = H / VE;
    const int rows = a.NH + 2 * a.NKV;
    const int chunks = (rows + kRows - 1) / kRows;
    const long unit = ((long)blockIdx.x * kThreads + threadIdx.x) / LPH;
    const int j = (threadIdx.x % LPH) * VE;
    const bool there = unit < (long)a.T * chunks;
    const int t = there ? (int)(unit / chunks) : 0;
    const int r0 = there ? (int)(unit - (long)t * chunks) * kRows : rows;

    float x0[kRows][VE], x1[kRows][VE];
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
        const int r = r0 + u;
        if (r < rows) {
            const T *src = r < a.NH ? reinterpret_cast<const T *>(a.q) + t * a.q_stride + (long)r * D
                           : r < a.NH + a.NKV
                               ? reinterpret_cast<const T *>(a.k) + t * a.k_stride + (long)(r - a.NH) * D
                               : reinterpret_cast<const T *>(a.v) + t * a.v_stride + (long)(r - a.NH - a.NKV) * D;
            load_n<T, VE>(src + j, x0[u]);
            load_n<T, VE>(src + j + H, x1[u]);
        } else {
#pragma unroll
            for (int e = 0; e < VE; ++e) x0[u][e] = x1[u][e] = 0.0f;
        }
    }
    float c[VE], s[VE];
    bool bad = false;
#pragma unroll
    for (int e = 0; e < VE; ++e) {
        const int ax = a.axes[j + e];
        int p = -1;
        if (ax >= 0 && ax < a.n_axes) p = a.positions[ax * a.pos_stride + t];
        if (p < 0 || p >= a.max_pos) {
            bad = true;
            c[e] = s[e] = 0.0f;
        } else {
            c[e] = a.cos_t[(size_t)p * H + j + e];
            s[e] = a.sin_t[(size_t)p * H + j + e];
        }
    }
    // a token with a position outside the table has no rotation: its query
    // rows are zero and its key and value are not written
#pragma unroll
    for (int o = LPH / 2; o; o >>= 1) bad |= __shfl_xor_sync(~0u, (int)bad, o) != 0;
    const long slot = a.slots[t];
    const bool writes = !bad && slot >= 0 && slot < a.num_slots;
    const long page = writes ? slot / a.P : 0;
    const long off = writes ? slot - page * a.P : 0;

#pragma unroll
    for (int u = 0; u < kRows; ++u) {
        const int r = r0 + u;
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < VE; ++e) ss += x0[u][e] * x0[u][e] + x1[u][e] * x1[u][e];
#pragma unroll
        for (int o = LPH / 2; o; o >>= 1) ss += __shfl_xor_sync(~0u, ss, o);
        if (r >= rows) continue;
        if (r < a.NH + a.NKV) {
            const NormWeight &n = r < a.NH ? a.qn : a.kn;
            if (n.w) {
                const float inv = 1.0f / sqrtf(ss * (1.0f / D) + a.eps);
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    x0[u][e] *= inv * weight_at(n, a.w_dtype, j + e);
                    x1[u][e] *= inv * weight_at(n, a.w_dtype, j + H + e);
                }
            }
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const float y0 = x0[u][e] * c[e] - x1[u][e] * s[e];
                x1[u][e] = x1[u][e] * c[e] + x0[u][e] * s[e];
                x0[u][e] = bad ? 0.0f : y0;
                if (bad) x1[u][e] = 0.0f;
            }
        }
        if (r < a.NH) {
            T *o = reinterpret_cast<T *>(a.q_out) + ((long)t * a.NH + r) * D + j;
            store_n<T, VE>(o, x0[u]);
            store_n<T, VE>(o + H, x1[u]);
        } else if (writes) {
            const bool isk = r < a.NH + a.NKV;
            const int h = r - a.NH - (isk ? 0 : a.NKV);
            C *o = reinterpret_cast<C *>(isk ? a.k_pages : a.v_pages) + ((page * a.NKV + h) * a.P + off) * D + j;
            store_n<C, VE>(o, x0[u]);
            store_n<C, VE>(o + H, x1[u]);
        }
    }
}

namespace {
template <typename T, typename C, int D>
cudaError_t launch_d(const MropeArgs &a, cudaStream_t st) {
    constexpr int LPH = D / 2 / (16 / (int)sizeof(T));
    const long chunks = (a.NH + 2 * a.NKV + kRows - 1) / kRows;
    const long threads = (long)a.T * chunks * LPH;
    mrope_append_kernel<T, C, D><<<(unsigned)((threads + kThreads - 1) / kThreads), kThreads, 0, st>>>(a);
    return cudaGetLastError();
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
