// Attention of a tree of drafted tokens over the paged cache.
//
// Node i of request s (row starts[s] + i of q) sees the request's cached
// positions [0, ctx) and, of the drafted ones at positions ctx + j, itself and
// its ancestors:  out = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale q.k_t - m).
// A parent is an earlier node, so a chain of parents ends by itself; an entry
// that names no earlier node counts as a root.
//
// The query rows of one request that share a key head (nodes x heads per
// key head) read the same keys and values: 512 bytes a position (D 128) for up to
// NC rows.  Up to ~128 rows that is bound by memory, so the cache is to be
// read once and everything else has to hide behind it.
//
// Both products run on the tensor cores with the *cache* as the 128-row
// operand and the query rows as its columns, so that any number of rows from 1
// up fills the tile's long side:
//   S^T [128 positions, NC rows] = K [128, D] . Q^T          (K as TMA wrote it)
//   O^T [D, NC rows]            = V^T [D, 128] . P^T         (V as TMA wrote it, read
//                                                            along its rows)
// One CTA takes one request, key head, tile of NC rows and slice of the
// context.  Warps: one softmax warpgroup (two for 64 rows: half the columns each;
// thread = position), one warpgroup that sums the output (thread = value of
// the head), a warp for the TMA loads and one for the MMAs.  Per tile of 128
// positions:
//   maxima of the columns over a warp's 32 positions (redux.f32), joined over
//   the warps in shared memory, p = 2^(s - m) -> shared memory, PV into a fresh
//   accumulator, and acc = acc * 2^(m_old - m) + PV in fp32 registers: the
//   tensor cores' accumulation is not rounded to nearest, so no chain of it is
//   longer than a tile.
// fp32 queries are split q = hi + lo (fp16 each, after a power of two per row
// that keeps both in fp16's normal range), and the probabilities
// p = hi + lo as well, 22 bits in all: the products of 16-bit values are exact in the
// tensor core, so fp32 outputs keep fp32 accuracy, and the second products hide
// behind the cache's loads.  16-bit queries are exact as they are.
// The slices of a context meet in a second launch (tree_join_kernel).
//
// Every wait is bounded (2 s); one that gives up sets this kernel's timeout word,
// and while it is set the kernel computes nothing (qvl_tc_timeout_status).
#include "serving.cuh"
#include "tc_common.cuh"

namespace qvl {

__device__ int g_tree_timeout = 0;

namespace {
constexpr int kTile = 128;              // positions per tile: the MMA's M
constexpr int kMaxWords = kTreeMaxNodes / 32;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kPBias = 8.0f;          // p is held times 2^8: its low half stays normal

// ---- tensor core helpers ----
template <typename C>
__host__ __device__ constexpr uint32_t idesc_16(int n, bool mn_major) {
    const uint32_t t = std::is_same<C, __nv_bfloat16>::value ? 1u : 0u;
    const uint32_t tr = mn_major ? (3u << 15) : 0u;
    return (1u << 4) | (t << 7) | (t << 10) | tr | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
}
// Operand whose contraction index is the slow one, as TMA wrote it with
// 128-byte swizzle: rows of 64 values, 8-row atoms of 1024 bytes, `chunk`
// bytes from one 64-value column block to the next.
__device__ __forceinline__ uint64_t sdesc_mn_sw128(uint32_t addr, uint32_t chunk) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | (uint64_t)(chunk >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 |
           (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// The same without swizzle: 8 x 8 blocks of 128 contiguous bytes, the next 8
// contraction indices 128 bytes on, the next 8 rows `chunk` bytes on.
__device__ __forceinline__ uint64_t sdesc_mn_plain(uint32_t addr, uint32_t chunk) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | (uint64_t)(128 >> 4) << 16 | (uint64_t)(chunk >> 4) << 32 |
           (uint64_t)1 << 46;
}
__device__ __forceinline__ void mma_16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ float redux_max(float v) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void bar_sync(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Two floats to packed 16-bit values (a low, b high) and what is left of them.
template <typename C> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <typename C> __device__ __forceinline__ float2 unpack2(uint32_t v);
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t v) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&v));
}
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
// Some half of a packed pair is infinite or NaN.
template <typename C> __device__ __forceinline__ bool nonfinite2(uint32_t v) {
    constexpr uint32_t e = std::is_same<C, __half>::value ? 0x7c00u : 0x7f80u;
    return (v & e) == e || ((v >> 16) & e) == e;
}

// ---- what a CTA works on ----
struct Plan {
    int chunk;          // tiles per slice
    int splits;         // slices of the longest context
    int row_tiles;
    int box;            // positions per TMA box
};

// Rows of q that a request's nodes own: [first, first + n).
__device__ __forceinline__ int node_count(const TreeArgs &a, int s, int &first) {
    first = min(max(a.starts[s], 0), a.T);
    const int end = min(max(a.starts[s + 1], first), a.T);
    return min(end - first, a.max_nodes);
}
// Cached positions, and all positions with the drafted ones (those that the page table has room for).
__device__ __forceinline__ int context(const TreeArgs &a, int s, int n, int &ctx) {
    const long cap = min((long)a.maxp * a.P, (long)INT32_MAX - 2 * kTile);
    ctx = (int)min((long)max(a.ctx_lens[s], 0), cap);
    return (int)min((long)ctx + n, cap);
}
__device__ __forceinline__ int slices(int L, const Plan &p) {
    return max(1, min(p.splits, (L + p.chunk * kTile - 1) / (p.chunk * kTile)));
}

template <typename T, int D, int NC>
struct Conf {
    static constexpr bool kSplitQ = std::is_same<T, float>::value;
    static constexpr int kSW = NC > 32 ? 2 : 1;                       // softmax warpgroups
    static constexpr int kCols = NC / kSW;                            // columns of a softmax thread
    static constexpr int kThreads = kSW * 128 + 128 + 64;
    static constexpr int kPerSM = NC > 32 ? 1 : 2;
    static constexpr int kQ = NC * D * 2;
    static constexpr int kP = NC * kTile * 2;
    static constexpr int kSlot = kTile * D * 2;
    static constexpr int kFixed = (kSplitQ ? 2 : 1) * kQ + 2 * kP;
    static constexpr int kMiscMask = kTreeMaxNodes * (NC > 32 ? NC / 32 : 1) * 4;
    static constexpr int kMisc = kMiscMask + 4 * NC * 4 + NC * 8 + kSW * 4 * kCols * 4 + 2048;
    static constexpr int kRoom = (kPerSM == 2 ? 113 : 226) * 1024 - kFixed - kMisc - 1024;
    static constexpr int kSlots = kRoom / kSlot > 8 ? 8 : kRoom / kSlot;
    static constexpr int kSmem = 1024 + kSlots * kSlot + kFixed + kMisc;
    static constexpr int kTmem = 4 * NC < 32 ? 32 : 4 * NC;
    static_assert(kSlots >= 2, "keys and values take turns in the slots");
};
}  // namespace

// grid (splits * row_tiles, NKV, S)
template <typename T, typename C, int D, int NC>
__global__ void __launch_bounds__(Conf<T, D, NC>::kThreads, Conf<T, D, NC>::kPerSM)
tree_tc_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
               const __grid_constant__ TreeArgs a, const __grid_constant__ Plan pl) {
    using F = Conf<T, D, NC>;
    constexpr int kSW = F::kSW, kCols = F::kCols, NS = F::kSlots;
    constexpr int kWordsC = NC > 32 ? NC / 32 : 1;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char *smem =
        reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char *slots = smem;
    unsigned char *q_s = slots + NS * F::kSlot;                        // hi, then lo
    unsigned char *p_s = q_s + (F::kSplitQ ? 2 : 1) * F::kQ;           // hi, then lo
    uint32_t *tmask = reinterpret_cast<uint32_t *>(p_s + 2 * F::kP);   // [node][kWordsC]: columns that see it
    float *alpha_s = reinterpret_cast<float *>(tmask + kTreeMaxNodes * kWordsC);      // [4][NC]
    float2 *cm_s = reinterpret_cast<float2 *>(alpha_s + 4 * NC);       // [NC]: {score factor, maximum}
    float *wmax_s = reinterpret_cast<float *>(cm_s + NC);              // [kSW][4][kCols]
    uint32_t *bad_s = reinterpret_cast<uint32_t *>(wmax_s + kSW * 4 * kCols);         // [4][4]: rows of V held back
    uint64_t *bars = reinterpret_cast<uint64_t *>(bad_s + 16);
    const uint32_t kv_full = tc::smem_u32(bars), kv_empty = kv_full + 8 * 8, s_full = kv_empty + 8 * 8,
                   s_empty = s_full + 16, o_full = s_empty + 16, o_empty = o_full + 16, p_ready = o_empty + 16,
                   p_empty = p_ready + 8;
    uint32_t *valid_s = reinterpret_cast<uint32_t *>(bars + 26);       // [8], by tile: its boxes that exist
    uint32_t *tmem_slot = valid_s + 8;
    int *off_s = reinterpret_cast<int *>(tmem_slot + 1);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int s = blockIdx.z, kvh = blockIdx.y;
    const int z = blockIdx.x % pl.splits, rt = blockIdx.x / pl.splits;
    const int G = a.NH / a.NKV;

    pdl_wait();
    int first, ctx;
    const int n = node_count(a, s, first);
    const int L = context(a, s, n, ctx);
    const int r0 = rt * NC;
    T *out = reinterpret_cast<T *>(a.out);
    const int nsl = slices(L, pl);

    // rows that no node owns
    if (z == 0 && rt == 0) {
        auto clear = [&](int from, int to) {
            for (long e = (long)from * G * D + tid; e < (long)to * G * D; e += F::kThreads) {
                const long row = e / (G * D), c = e - row * (G * D);
                out[(row * a.NH + (long)kvh * G) * D + c] = from_f32<T>(0.0f);
            }
        };
        if (s == 0) clear(0, min(max(a.starts[0], 0), a.T));
        // past max_nodes, and behind the last request
        clear(first + n, s + 1 < a.S ? min(max(a.starts[s + 1], first), a.T) : a.T);
    }
    if (n == 0 || r0 >= n * G || z >= nsl) return;
    const int rows = min(NC, n * G - r0);
    const int tile0 = z * pl.chunk;
    const int tiles = (L + kTile - 1) / kTile;
    const int nt = (z == nsl - 1 ? tiles : min(tiles, tile0 + pl.chunk)) - tile0;
    const bool has_tree = (long)(tile0 + nt) * kTile > ctx;

    if (tid == 0) {
        off_s[0] = *reinterpret_cast<volatile int *>(&g_tree_timeout);
        for (int i = 0; i < NS; ++i) {
            tc::mbar_init(kv_full + 8 * i, 1);
            tc::mbar_init(kv_empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(s_full + 8 * i, 1);
            tc::mbar_init(s_empty + 8 * i, kSW * 128);
            tc::mbar_init(o_full + 8 * i, 1);
            tc::mbar_init(o_empty + 8 * i, 128);
        }
        tc::mbar_init(p_ready, kSW * 128);
        tc::mbar_init(p_empty, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        tc::prefetch_tmap(&tm_k);
        tc::prefetch_tmap(&tm_v);
    }
    constexpr int kMmaWarp = kSW * 4 + 4, kTmaWarp = kMmaWarp + 1;
    if (warp == kMmaWarp) {
        tc::tmem_alloc(tc::smem_u32(tmem_slot), F::kTmem);
        tc::tmem_relinquish();
    }

    // query rows into shared memory, K-major with 128-byte swizzle: one warp a
    // row; rows past the last one are zero
    const float qmul = a.scale * kLog2e;
    for (int r = warp; r < NC; r += F::kThreads / 32) {
        constexpr int E = D / 32;           // values of a lane
        float x[E];
        const int node = (r0 + r) / G, hq = (r0 + r) - node * G;
        const T *src = reinterpret_cast<const T *>(a.q) + (long)(first + node) * a.q_stride + (long)(kvh * G + hq) * D + lane * E;
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = r < rows ? to_f32(src[e]) : 0.0f;
        float cs = fabsf(qmul);
        if constexpr (F::kSplitQ) {
            float mx = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                x[e] *= qmul;
                mx = fmaxf(mx, fabsf(x[e]));
            }
            mx = redux_max(mx);
            // largest value into [2^9, 2^10)
            int ex = (int)(__float_as_uint(mx) >> 23);
            if (mx == 0.0f || ex == 255) ex = 127 + 9;
            ex = max(ex, 10);
            const float f = __uint_as_float((uint32_t)min(254, 263 - ex) << 23);
            cs = __uint_as_float((uint32_t)(ex - 9) << 23);
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] *= f;
        } else if (qmul < 0.0f) {
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = -x[e];
        }
        const int half = lane * E >> 6, in = lane * E & 63;
        unsigned char *dst = q_s + half * (NC * 128) + r * 128 + ((((in * 2) >> 4) ^ (r & 7)) << 4) + ((in * 2) & 15);
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            const uint32_t hi = pack2<C>(x[e], x[e + 1]);
            *reinterpret_cast<uint32_t *>(dst + e * 2) = hi;
            if constexpr (F::kSplitQ) {
                const float2 h = unpack2<C>(hi);
                *reinterpret_cast<uint32_t *>(dst + F::kQ + e * 2) = pack2<C>(x[e] - h.x, x[e + 1] - h.y);
            }
        }
        if (lane == 0) cm_s[r] = make_float2(cs, -INFINITY);
    }
    if (tid < 16) bad_s[tid] = 0;

    // columns that see each drafted position: ancestors by doubling (a node's
    // set is its own bit, its parent's set, ...), turned to bits over columns
    if (has_tree) {
        uint32_t *anc = reinterpret_cast<uint32_t *>(slots);           // [2][256][words]; before the first load
        int *up = reinterpret_cast<int *>(slots + 2 * kTreeMaxNodes * kMaxWords * 4);
        const int words = (n + 31) / 32;
        for (int i = tid; i < n; i += F::kThreads) {
            const int p = a.parents[first + i];
            up[i] = p >= 0 && p < i ? p : -1;
            for (int w = 0; w < words; ++w) anc[i * kMaxWords + w] = w == (i >> 5) ? 1u << (i & 31) : 0u;
        }
        __syncthreads();
        int cur = 0;
        for (int d = 1; d < n; d *= 2) {
            const uint32_t *src = anc + cur * kTreeMaxNodes * kMaxWords;
            uint32_t *dst = anc + (cur ^ 1) * kTreeMaxNodes * kMaxWords;
            const int *us = up + cur * kTreeMaxNodes;
            int *ud = up + (cur ^ 1) * kTreeMaxNodes;
            for (int i = tid; i < n; i += F::kThreads) {
                const int p = us[i];
                for (int w = 0; w < words; ++w)
                    dst[i * kMaxWords + w] = src[i * kMaxWords + w] | (p >= 0 ? src[p * kMaxWords + w] : 0u);
                ud[i] = p >= 0 ? us[p] : -1;
            }
            cur ^= 1;
            __syncthreads();
        }
        const uint32_t *res = anc + cur * kTreeMaxNodes * kMaxWords;
        for (int e = tid; e < n * kWordsC; e += F::kThreads) {
            const int j = e / kWordsC, w = e - j * kWordsC;
            uint32_t m = 0;
            for (int c = 0; c < 32 && w * 32 + c < rows; ++c) {
                const int node = (r0 + w * 32 + c) / G;
                m |= ((res[node * kMaxWords + (j >> 5)] >> (j & 31)) & 1u) << c;
            }
            tmask[e] = m;
        }
        fence_async_smem();         // the loads overwrite what the generic proxy read and wrote here
    }
    fence_async_smem();
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    pdl_launch_dependents();
    const uint32_t tmem = *tmem_slot;
    const uint32_t tm_s = tmem, tm_o = tmem + 2 * NC;
    bool ok = off_s[0] == 0;
    int issued = 0;                      // slots that the TMA warp filled

    if (warp == kTmaWarp) {
        // lane l: box l / 2 of the tile's 64-value half l % 2
        const int nb = kTile / pl.box, lanes = nb * (D / 64);
        const int b = lane / (D / 64), half = lane % (D / 64);
        const int oob = (int)(a.num_pages * a.NKV * a.P);          // past the last row: zeros
        for (int i = 0; ok && i < nt; ++i) {
            const int t = (tile0 + i) * kTile + b * pl.box;
            int y = oob;
            if (lane < lanes && t < L) {
                const int c = t / a.P;
                const int pg = a.table[(size_t)s * a.maxp + c];
                if (pg >= 0 && pg < a.num_pages) y = (int)(((long)pg * a.NKV + kvh) * a.P + (t - c * a.P));
            }
            const uint32_t there = __ballot_sync(~0u, y != oob);
            for (int h = 0; h < 2 && ok; ++h) {
                const int u = 2 * i + h, sl = u % NS, k = u / NS;
                if (k > 0) ok = tc::mbar_wait(kv_empty + 8 * sl, (k - 1) & 1, &g_tree_timeout);
                ok = __all_sync(~0u, ok);
                if (!ok) break;
                if (lane == 0) {
                    // (the load of a tile's keys runs at most kSlots / 2 + 1 tiles
                    // ahead of the softmax that reads this)
                    if (h == 0) valid_s[i & 7] = there;
                    tc::mbar_expect_tx(kv_full + 8 * sl, F::kSlot);
                }
                __syncwarp();
                if (lane < lanes)
                    tc::tma_load_2d(tc::smem_u32(slots + sl * F::kSlot + half * (kTile * 128) + b * pl.box * 128),
                                    h ? &tm_v : &tm_k, half * 64, y, kv_full + 8 * sl);
                __syncwarp();
                issued = u + 1;
            }
        }
        // loads in flight land before the CTA ends
        if (!ok)
            for (int u = max(0, issued - NS); u < issued; ++u)
                tc::mbar_wait(kv_full + 8 * (u % NS), (u / NS) & 1, nullptr);
    } else if (warp == kMmaWarp) {
        if (lane == 0) {
            constexpr uint32_t id_s = idesc_16<C>(NC, false), id_o = idesc_16<C>(NC, true);
            const uint32_t qa = tc::smem_u32(q_s), pa = tc::smem_u32(p_s), sa = tc::smem_u32(slots);
            auto scores = [&](int i) {
                const int u = 2 * i, sl = u % NS, b = i & 1;
                ok = ok && tc::mbar_wait(kv_full + 8 * sl, (u / NS) & 1, &g_tree_timeout);
                if (i >= 2) ok = ok && tc::mbar_wait(s_empty + 8 * b, ((i >> 1) - 1) & 1, &g_tree_timeout);
                if (!ok) return;
                tc::tc_fence_after();
                const uint32_t ka = sa + sl * F::kSlot;
#pragma unroll
                for (int l = 0; l < (F::kSplitQ ? 2 : 1); ++l)
#pragma unroll
                    for (int k = 0; k < D / 16; ++k)
                        mma_16(tm_s + b * NC, tc::sdesc_k_sw128(ka + (k >> 2) * (kTile * 128) + (k & 3) * 32),
                               tc::sdesc_k_sw128(qa + l * F::kQ + (k >> 2) * (NC * 128) + (k & 3) * 32), id_s,
                               (l | k) ? 1u : 0u);
                tc::tc_commit(kv_empty + 8 * sl);
                tc::tc_commit(s_full + 8 * b);
            };
            scores(0);
            for (int i = 0; ok && i < nt; ++i) {
                if (i + 1 < nt) scores(i + 1);
                const int u = 2 * i + 1, sl = u % NS, b = i & 1;
                ok = ok && tc::mbar_wait(kv_full + 8 * sl, (u / NS) & 1, &g_tree_timeout);
                ok = ok && tc::mbar_wait(p_ready, i & 1, &g_tree_timeout);
                if (i >= 2) ok = ok && tc::mbar_wait(o_empty + 8 * b, ((i >> 1) - 1) & 1, &g_tree_timeout);
                if (!ok) break;
                tc::tc_fence_after();
                const uint32_t va = sa + sl * F::kSlot;
                // D 64: the second 64 rows of the product are not read; any
                // part of shared memory will do for them
                constexpr uint32_t kChunk = D == 128 ? kTile * 128 : 1024;
#pragma unroll
                for (int l = 0; l < 2; ++l)
#pragma unroll
                    for (int k = 0; k < kTile / 16; ++k)
                        mma_16(tm_o + b * NC, sdesc_mn_sw128(va + k * 2048, kChunk),
                               sdesc_mn_plain(pa + l * F::kP + k * 256, kTile * 16), id_o, (l | k) ? 1u : 0u);
                tc::tc_commit(kv_empty + 8 * sl);
                tc::tc_commit(p_empty);
                tc::tc_commit(o_full + 8 * b);
            }
        }
        __syncwarp();
    } else if (warp < kSW * 4) {
        // ---- softmax: thread = position, columns [c0, c0 + kCols) ----
        const int wg = warp >> 2, w4 = warp & 3, c0 = wg * kCols;
        const int jl = w4 * 32 + lane;
        const uint32_t lane_off = (uint32_t)(w4 * 32) << 16;
        float *wmax = wmax_s + wg * 4 * kCols;
        const int own = tid & 127;                    // the column this thread keeps the maximum of
        float m_own = -INFINITY;
        const float cs_own = own < kCols ? cm_s[c0 + own].x : 0.0f;
        float l[kCols];
#pragma unroll
        for (int c = 0; c < kCols; ++c) l[c] = 0.0f;

        // (after a wait that gave up, the loops run on without waiting: the
        // barriers among a warpgroup's threads have to be met by all of them)
        for (int i = 0; i < nt; ++i) {
            const int b = i & 1;
            const int t0 = (tile0 + i) * kTile, t = t0 + jl;
            if (ok) ok = tc::mbar_wait(s_full + 8 * b, (i >> 1) & 1, &g_tree_timeout);
            // what this position's columns see: all, or the bits of `see`
            const int vu = 2 * i + 1;
            const uint32_t there = *reinterpret_cast<volatile uint32_t *>(&valid_s[i & 7]);
            const bool plain = t0 + kTile <= ctx && there == (1u << (kTile / pl.box * (D / 64))) - 1u;
            uint32_t see[kWordsC];
#pragma unroll
            for (int w = 0; w < kWordsC; ++w) see[w] = ~0u;
            if (!plain) {
                const bool in = t < L && ((there >> ((jl / pl.box) * (D / 64))) & 1u);
#pragma unroll
                for (int w = 0; w < kWordsC; ++w)
                    see[w] = !in ? 0u : t < ctx ? ~0u : tmask[(t - ctx) * kWordsC + w];
                // V of positions that some row does not see: what is not finite
                // would reach every row through 0 * v; it is taken out here and added
                // to the rows that see it by the summing warps
                if (ok) ok = tc::mbar_wait(kv_full + 8 * (vu % NS), (vu / NS) & 1, &g_tree_timeout);
                if (t >= ctx || !in) {
                    unsigned char *vr = slots + (vu % NS) * F::kSlot + jl * 128;
                    bool bad = false;
                    constexpr int kPieces = D / 8 / kSW;
                    for (int e = 0; e < kPieces; ++e) {
                        const int ch = wg * kPieces + e;
                        uint4 *p = reinterpret_cast<uint4 *>(vr + (ch >> 3) * (kTile * 128) + (((ch & 7) ^ (jl & 7)) << 4));
                        if (!in) {
                            *p = make_uint4(0, 0, 0, 0);
                        } else {
                            uint4 v = *p;
                            uint32_t *x = reinterpret_cast<uint32_t *>(&v);
                            bool hit = false;
#pragma unroll
                            for (int y = 0; y < 4; ++y)
                                if (nonfinite2<C>(x[y])) {
                                    constexpr uint32_t ee = std::is_same<C, __half>::value ? 0x7c00u : 0x7f80u;
                                    hit = true;
                                    if ((x[y] & ee) == ee) x[y] &= 0xffff0000u;
                                    if (((x[y] >> 16) & ee) == ee) x[y] &= 0x0000ffffu;
                                }
                            if (hit) {
                                *p = v;
                                bad = true;
                            }
                        }
                    }
                    if (bad) atomicOr(&bad_s[(i & 3) * 4 + w4], 1u << lane);
                }
            }
            tc::tc_fence_after();

            // maxima of the columns over the tile
            float sv[kCols];
            {
                uint32_t r[kCols];
#pragma unroll
                for (int c = 0; c < kCols; c += 16)
                    tc::tmem_ld16(tm_s + b * NC + lane_off + c0 + c, *reinterpret_cast<uint32_t(*)[16]>(r + c));
                tc::tmem_wait_ld();
#pragma unroll
                for (int c = 0; c < kCols; ++c) sv[c] = __uint_as_float(r[c]);
            }
            tc::tc_fence_before();
            mbar_arrive(s_empty + 8 * b);
            float keep = -INFINITY;
            if (plain) {
#pragma unroll
                for (int c = 0; c < kCols; ++c) {
                    const float v = redux_max(sv[c]);
                    if (lane == c % 32) keep = v;
                }
            } else {
#pragma unroll
                for (int c = 0; c < kCols; ++c) {
                    const bool on = (see[(c0 + c) / 32] >> ((c0 + c) % 32)) & 1u;
                    const float v = redux_max(on ? sv[c] : -INFINITY);
                    if (lane == c % 32) keep = v;
                }
            }
            if (lane < kCols) wmax[w4 * kCols + lane] = keep;
            bar_sync(1 + wg, 128);
            if (own < kCols) {
                float v = fmaxf(fmaxf(wmax[own], wmax[kCols + own]), fmaxf(wmax[2 * kCols + own], wmax[3 * kCols + own]));
                v = v == -INFINITY ? v : v * cs_own;
                const float m = fmaxf(m_own, v);
                alpha_s[(i & 3) * NC + c0 + own] = m_own == m ? 1.0f : ex2(m_own - m);
                m_own = m;
                cm_s[c0 + own].y = m == -INFINITY ? 0.0f : m - kPBias;
            }
            bar_sync(1 + wg, 128);

            // p, its sum, and p into shared memory as hi + lo
            if (i > 0 && ok) ok = tc::mbar_wait(p_empty, (i - 1) & 1, &g_tree_timeout);
            unsigned char *pd = p_s + (c0 / 8) * (kTile * 16) + jl * 16;
#pragma unroll
            for (int c8 = 0; c8 < kCols; c8 += 8) {
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const int c = c8 + e;
                    const float4 cm = *reinterpret_cast<const float4 *>(&cm_s[c0 + c]);
                    const float2 al = *reinterpret_cast<const float2 *>(&alpha_s[(i & 3) * NC + c0 + c]);
                    float pa = ex2(fmaf(sv[c], cm.x, -cm.y)), pb = ex2(fmaf(sv[c + 1], cm.z, -cm.w));
                    if (!plain) {
                        pa = ((see[(c0 + c) / 32] >> ((c0 + c) % 32)) & 1u) ? pa : 0.0f;
                        pb = ((see[(c0 + c + 1) / 32] >> ((c0 + c + 1) % 32)) & 1u) ? pb : 0.0f;
                    }
                    l[c] = fmaf(l[c], al.x, pa);
                    l[c + 1] = fmaf(l[c + 1], al.y, pb);
                    hi[e / 2] = pack2<C>(pa, pb);
                    const float2 h = unpack2<C>(hi[e / 2]);
                    lo[e / 2] = pack2<C>(pa - h.x, pb - h.y);
                }
                *reinterpret_cast<uint4 *>(pd + (c8 / 8) * (kTile * 16)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                *reinterpret_cast<uint4 *>(pd + F::kP + (c8 / 8) * (kTile * 16)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
            fence_async_smem();
            mbar_arrive(p_ready);
        }
        // sums over the positions
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
            float v = l[c];
#pragma unroll
            for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
            if (lane == c % 32) wmax[w4 * kCols + c] = v;
        }
        bar_sync(1 + wg, 128);
        if (own < kCols) {
            const float v = (wmax[own] + wmax[kCols + own]) + (wmax[2 * kCols + own] + wmax[3 * kCols + own]);
            cm_s[c0 + own] = make_float2(v, m_own);
        }
    }
    // ---- output sums: thread = value of the head ----
    float acc[NC];
    const bool summing = warp >= kSW * 4 && warp < kSW * 4 + 4;
    if (summing) {
        const int d = tid & 127;
        const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
#pragma unroll
        for (int c = 0; c < NC; ++c) acc[c] = 0.0f;
        for (int i = 0; i < nt; ++i) {
            const int b = i & 1;
            // the factors were written before p_ready, on which the product waited
            if (ok) ok = tc::mbar_wait(o_full + 8 * b, (i >> 1) & 1, &g_tree_timeout);
            tc::tc_fence_after();
            const float *al = alpha_s + (i & 3) * NC;
#pragma unroll
            for (int c = 0; c < NC; c += 16) {
                uint32_t r[16];
                tc::tmem_ld16(tm_o + b * NC + lane_off + c, r);
                tc::tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const float4 f = *reinterpret_cast<const float4 *>(al + c + e);
                    acc[c + e] = fmaf(acc[c + e], f.x, __uint_as_float(r[e]));
                    acc[c + e + 1] = fmaf(acc[c + e + 1], f.y, __uint_as_float(r[e + 1]));
                    acc[c + e + 2] = fmaf(acc[c + e + 2], f.z, __uint_as_float(r[e + 2]));
                    acc[c + e + 3] = fmaf(acc[c + e + 3], f.w, __uint_as_float(r[e + 3]));
                }
            }
            tc::tc_fence_before();
            const int t0 = (tile0 + i) * kTile;
            if (t0 + kTile > ctx) {
                // values that were taken out of the product: infinities and NaN
                for (int w = 0; w < 4; ++w) {
                    uint32_t m = *reinterpret_cast<volatile uint32_t *>(&bad_s[(i & 3) * 4 + w]);
                    for (; m; m &= m - 1) {
                        const int t = t0 + w * 32 + __ffs(m) - 1;
                        if (t < ctx || t >= L || d >= D) continue;
                        const int pg = a.table[(size_t)s * a.maxp + t / a.P];
                        const C v = reinterpret_cast<const C *>(a.v_pages)[(((long)pg * a.NKV + kvh) * a.P + t % a.P) * D + d];
                        const float x = to_f32(v);
                        if (fabsf(x) <= 3.402823466e38f) continue;
                        const uint32_t *see = tmask + (t - ctx) * kWordsC;
#pragma unroll
                        for (int c = 0; c < NC; ++c)
                            if ((see[c / 32] >> (c % 32)) & 1u) acc[c] += x;
                    }
                }
                bar_sync(3, 128);
                if (d < 4) bad_s[(i & 3) * 4 + d] = 0;
            }
            mbar_arrive(o_empty + 8 * b);
        }
    }
    __syncwarp();
    tc::tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) tc::tmem_dealloc(tmem, F::kTmem);
    if (!ok) return;
    if (summing) {
        const int d = tid & 127;
        float *part = reinterpret_cast<float *>(a.workspace);
        const long heads = (long)a.T * a.NH;
        float2 *ml = reinterpret_cast<float2 *>(part + (size_t)pl.splits * heads * D);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            if (c < rows) {
                const int node = (r0 + c) / G;
                const long row = (long)(first + node) * a.NH + kvh * G + (r0 + c - node * G);
                const float2 st = cm_s[c];
                if (nsl == 1) {
                    if (d < D) out[row * D + d] = from_f32<T>(st.x == 0.0f ? 0.0f : acc[c] / st.x);
                } else {
                    if (d < D) part[(z * heads + row) * D + d] = acc[c];
                    if (d == 0) ml[z * heads + row] = make_float2(st.y, st.x);
                }
            }
        }
    }
}

// Joins the slices of each row: weights 2^(m_z - max m).  One warp per row and head.
template <typename T, int D>
__global__ void __launch_bounds__(256) tree_join_kernel(const __grid_constant__ TreeArgs a, const __grid_constant__ Plan pl) {
    pdl_launch_dependents();
    pdl_wait();
    const long heads = (long)a.T * a.NH;
    const long w = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (w >= heads) return;
    const int lane = threadIdx.x & 31, row = (int)(w / a.NH);
    // the request that owns the row: the last one that starts at or before it
    int lo = 0, hi = a.S;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.starts[mid] <= row) lo = mid;
        else hi = mid;
    }
    int first, ctx;
    const int n = node_count(a, lo, first);
    if (row < first || row >= first + n) return;
    const int nsl = slices(context(a, lo, n, ctx), pl);
    if (nsl == 1) return;
    const float *part = reinterpret_cast<const float *>(a.workspace);
    const float2 *ml = reinterpret_cast<const float2 *>(part + (size_t)pl.splits * heads * D);
    float m = -INFINITY;
    for (int z = lane; z < nsl; z += 32) m = fmaxf(m, ml[z * heads + w].x);
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
    constexpr int E = D / 32;
    float acc[E], l = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.0f;
    for (int z = 0; z < nsl; ++z) {
        const float2 st = ml[z * heads + w];
        const float f = st.x == m ? 1.0f : ex2(st.x - m);
        l = fmaf(st.y, f, l);
        const float *p = part + (z * heads + w) * D + lane * E;
        if constexpr (E == 4) {
            const float4 v = *reinterpret_cast<const float4 *>(p);
            acc[0] = fmaf(v.x, f, acc[0]);
            acc[1] = fmaf(v.y, f, acc[1]);
            acc[2] = fmaf(v.z, f, acc[2]);
            acc[3] = fmaf(v.w, f, acc[3]);
        } else {
            const float2 v = *reinterpret_cast<const float2 *>(p);
            acc[0] = fmaf(v.x, f, acc[0]);
            acc[1] = fmaf(v.y, f, acc[1]);
        }
    }
    T *o = reinterpret_cast<T *>(a.out) + w * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = from_f32<T>(l == 0.0f ? 0.0f : acc[e] / l);
}

// ---------------------------------------------------------------- host side
namespace {
using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                 const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_fn() {
    static const EncodeTiled fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
                       q == cudaDriverEntryPointSuccess
                   ? reinterpret_cast<EncodeTiled>(p)
                   : nullptr;
    }();
    return fn;
}

// One half of the cache as rows of D 16-bit values, boxes of 64 values x `box` rows.
bool map_cache(CUtensorMap *m, const void *base, uint64_t rows, int D, int box, bool bf16) {
    const EncodeTiled enc = encode_fn();
    if (!enc) return false;
    cuuint64_t dims[2] = {(cuuint64_t)D, rows};
    cuuint64_t strides[1] = {(cuuint64_t)D * 2};
    cuuint32_t bx[2] = {64, (cuuint32_t)box};
    cuuint32_t es[2] = {1, 1};
    return enc(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void *>(base),
               dims, strides, bx, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int columns_for(int rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : 64; }

Plan plan_for(int S, int max_ctx, int max_nodes, int NH, int NKV) {
    Plan p{};
    const int rows = max_nodes * (NH / NKV), nc = columns_for(rows);
    p.row_tiles = (rows + nc - 1) / nc;
    const long tiles = ((long)max_ctx + kTile - 1) / kTile;
    const long ctas = 148l * (nc > 32 ? 1 : 2);
    // a few slices per resident CTA even out requests of different lengths
    long chunk = (tiles * S * NKV * p.row_tiles + 4 * ctas - 1) / (4 * ctas);
    chunk = chunk < 1 ? 1 : chunk > tiles ? tiles : chunk;
    p.chunk = (int)chunk;
    p.splits = (int)((tiles + chunk - 1) / chunk);
    return p;
}

template <typename T, typename C, int D, int NC>
cudaError_t launch_nc(const TreeArgs &a, Plan pl, cudaStream_t st) {
    using F = Conf<T, D, NC>;
    pl.box = 16;
    while (pl.box < kTile && a.P % (2 * pl.box) == 0) pl.box *= 2;
    CUtensorMap mk, mv;
    const uint64_t rows = (uint64_t)a.num_pages * a.NKV * a.P;
    const bool bf = a.kv_dtype == QVL_DTYPE_BF16;
    if (!map_cache(&mk, a.k_pages, rows, D, pl.box, bf) || !map_cache(&mv, a.v_pages, rows, D, pl.box, bf))
        return cudaErrorInvalidValue;
    auto kern = tree_tc_kernel<T, C, D, NC>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, F::kSmem);
    if (e != cudaSuccess) return e;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(pl.splits * pl.row_tiles, a.NKV, a.S);
    cfg.blockDim = dim3(F::kThreads);
    cfg.dynamicSmemBytes = F::kSmem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, kern, mk, mv, a, pl);
    if (e != cudaSuccess || pl.splits == 1) return e;
    cfg.gridDim = dim3((unsigned)(((long)a.T * a.NH + 7) / 8));
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = 0;
    return cudaLaunchKernelEx(&cfg, tree_join_kernel<T, D>, a, pl);
}
template <typename T, typename C, int D>
cudaError_t launch_d(const TreeArgs &a, cudaStream_t st) {
    const Plan pl = plan_for(a.S, a.max_ctx, a.max_nodes, a.NH, a.NKV);
    switch (columns_for(a.max_nodes * (a.NH / a.NKV))) {
    case 16: return launch_nc<T, C, D, 16>(a, pl, st);
    case 32: return launch_nc<T, C, D, 32>(a, pl, st);
    default: return launch_nc<T, C, D, 64>(a, pl, st);
    }
}
template <typename T, typename C>
cudaError_t launch_t(const TreeArgs &a, cudaStream_t st) {
    return a.D == 64 ? launch_d<T, C, 64>(a, st) : launch_d<T, C, 128>(a, st);
}
}  // namespace

int *tree_timeout_word() {
    void *p = nullptr;
    return cudaGetSymbolAddress(&p, g_tree_timeout) == cudaSuccess ? static_cast<int *>(p) : nullptr;
}

size_t tree_workspace_bytes(int S, int T, int max_ctx, int max_nodes, int NH, int NKV, int D) {
    const Plan p = plan_for(S, max_ctx, max_nodes, NH, NKV);
    if (p.splits == 1) return 0;
    return ((size_t)p.splits * T * NH * (D * sizeof(float) + sizeof(float2)) + 255) & ~(size_t)255;
}

cudaError_t launch_tree_attention(const TreeArgs &a, cudaStream_t st) {
    if (a.kv_dtype == QVL_DTYPE_BF16) return launch_t<__nv_bfloat16, __nv_bfloat16>(a, st);
    if (a.dtype == QVL_DTYPE_FP16) return launch_t<__half, __half>(a, st);
    return launch_t<float, __half>(a, st);
}

}  // namespace qvl
