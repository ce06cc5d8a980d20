// Attention of a tree of drafted tokens over the paged cache.
//
// Node i of request s (row starts[s] + i of q) sees the request's cached
// positions [0, ctx) and, of the drafted ones at positions ctx + j, itself and
// its ancestors:  out = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale q.k_t - m).
// A parent is an earlier node, so a chain of parents ends by itself; an entry
// that names no earlier node counts as a root.
//
// The query rows of one request that share a key head (nodes x heads per
// key head) read the same keys and values, 512 bytes a position at D 128.  Up to 128
// such rows are one tile of the tensor cores' long side, so that the cache is
// read once; with 6.5 TB/s of memory a tile of 128 positions (64 KB) then has 1.5
// us of one SM's time, and everything else has to hide behind it.
//
// Work: a unit is a tile of 128 positions of one (request, key head, 128 rows).
// All units in a row are cut into one equal stretch per CTA, one CTA
// per SM, whatever the requests' lengths are; a stretch is a few segments,
// each a range of one pair's tiles.  A segment that is a whole pair writes its
// rows; parts of a pair go to the workspace and meet in tree_join_kernel.
//
// Warps of a CTA:
//   TMA      cuts the stretch into segments, finds the pages, fills a ring of slots for K
//            and one for V (a slot: 128 positions, 128-byte swizzle), and loads a segment's Q
//   MMA      S = Q K^T [128 rows, 128 positions], O = P V [128 rows, D], a thread each, so
//            that one has its next product ready while the other's is under way.  Q, S, P
//            (over S) and O in tensor memory, so that shared memory, whose bandwidth the
//            products would need most of otherwise, is read for K and V alone
//   softmax  two warpgroups, every other tile each, so that one's waits pass beside the
//            other's work; thread = row.  A warpgroup's reference of a row (p = 2^(score -
//            reference)) is left as it is until a score passes it by 2^5 (2^7 over bf16), which the way
//            p is held allows: almost no tile rescales anything, and scores are
//            read once.  Between segments they bring the next one's Q to tensor memory.
//            A tile of at most 32 (64) rows is there four times (twice) over, in as many
//            blocks of the 128 rows: each block takes its share of the positions and
//            has p = 0 elsewhere, so that all warps have work, and the blocks are
//            added at the end like parts of a context
//   sums     two warpgroups (half of D each) add each tile's O to fp32 registers, times what
//            its warpgroup's reference is below the largest: the tensor cores do not round
//            their sums to nearest, so no chain of them is longer than a tile
//   fixer    the nodes' ancestors as bits, and values of the drafted tile that some
//            row does not see: 0 * NaN
// fp32 queries are split q = hi + lo (fp16 each, after a power of two per row
// that keeps both in fp16's normal range), 22 bits in all, and all probabilities p = hi + lo, 23 bits
// (bf16: 17; Held): the products of 16-bit values are exact in the tensor
// cores, so fp32 outputs keep fp32 accuracy and 16-bit ones are rounded once.
// Infinities and NaN of keys and values that a row sees: 0 * inf and inf - inf of the halves, and of the
// other blocks' zeros, make NaN where the definition has an infinity or nothing at all.  They leave a sum
// that is not finite, for which a row's sums are tested; such outputs are computed
// once more in plain fp32 (fix_row), after the products or in the joining launch.
// 16-bit queries are exact as they are.
//
// Exponentials are ex2.approx (relative error 2^-22) of arguments with one fp32 rounding.
//
// Measured (16 query and 8 key heads of 128, fp16 cache, keys and values read once: 4.6 TB/s
// and 4.1 TB/s of the 6.5 that a copy reaches): 16 requests of 64 nodes over up to 32768
// positions, fp16, 270 us; 32 of 16 nodes over up to 4096, fp32, 77 us, of which
// tiles take what memory does, and a segment's beginning and end the rest.  In a long
// row of such calls the board's power limit, not a pipe, sets the time (320 to 350 and 92 us, the
// SMs at 1.4 and 1.5 GHz of 1.97): the products of p's low halves are a tenth of it, and
// at 32 rows a fifth goes to the scores' products, of which each block uses a quarter.  12 requests of
// 132 rows over up to 6000, bf16, heads of 64: 38 us, the softmax's 3400 cycles for a
// tile of 128 x 128.  One token over 452 positions 13.9 us, 27 nodes over 2011 21 us: latency,
// the kernel's beginning (5 us: finding the stretch, queries to tensor memory), one tile, and the
// join (5 us).
// Tried and not kept: 16 scores a step (4000 cycles a tile for 3000), 64 with the largest
// found first; scores a step ahead in registers (spills: 318 us for 268);
// 16-bit queries as an operand from shared memory, with a third buffer of scores at D 128 (no
// difference); rings of 3 + 3 slots (none).
//
// Every wait is bounded (2 s); one that gives up sets this kernel's timeout word,
// and while it is set the kernel computes nothing (qvl_tc_timeout_status).
#include <algorithm>
#include <atomic>
#include <type_traits>
#include "serving.cuh"
#include "tc_common.cuh"

namespace qvl {

__device__ int g_tree_timeout = 0;

namespace {
constexpr int kTile = 128;              // positions per tile
constexpr int kRows = 128;              // query rows per tile
constexpr int kSMs = 148;
// 96 registers each at launch, 61440 in all; the last four warps hand 32 of each of their
// threads to the softmax's and the sums': 512 * 104 + 128 * 64 = 61440
constexpr int kThreads = 20 * 32;
constexpr int kMoreRegs = 104, kRestRegs = 64;
constexpr int kSumWarp = 8, kTmaWarp = 16, kScoreWarp = 17, kOutWarp = 18;          // the fixer is the last one
constexpr float kLog2e = 1.4426950408889634f;
// Probabilities over an fp16 cache.  A reference moves when a score passes it by more than 2^kRise, and p is
// held times 2^(15 - kRise), so that it fits fp16; the low halves times 2^11 more, which their product
// takes back (the accumulator goes down by 2^11 before the high halves' product is added).  p is
// then off by 2^-23 of itself, or by 2^(kRise - 51) of its reference where fp16's smallest step
// is more: where the largest p meets a value of 0, and the others 2^-29 of it are the output, by
// 2^-17.  kRise 5: 16 requests of 64 nodes over 32768 positions 274 us (7: 274, 3: 293, 1: 397), with scores five
// times as far apart 418 (7: 402, 3: 440).
template <typename C> struct Held;
template <> struct Held<__half> {
    static constexpr float kRise = 5.0f, kBias = 15.0f - kRise;
    static constexpr int kLow = 11;
    static constexpr float kLowUp = 2048.0f, kLowDown = 1.0f / 2048.0f;
};
// Over a bf16 cache: fp32's exponents, 2^-17 of itself.
template <> struct Held<__nv_bfloat16> {
    static constexpr float kRise = 7.0f, kBias = 8.0f;
    static constexpr int kLow = 0;
    static constexpr float kLowUp = 1.0f, kLowDown = 1.0f;
};

// ---- tensor core helpers ----
// kind::f16, fp32 sums; B with the contraction index as its slow one if `b_mn`.
template <typename C>
__host__ __device__ constexpr uint32_t idesc_16(int n, bool b_mn) {
    const uint32_t t = std::is_same<C, __nv_bfloat16>::value ? 1u : 0u;
    return (1u << 4) | (t << 7) | (t << 10) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(kRows >> 4) << 24);
}
// Operand whose contraction index is the slow one, as TMA wrote it with
// 128-byte swizzle: rows of 64 values, 8-row atoms of 1024 bytes, `chunk`
// bytes from one block of 64 values to the next.
__device__ __forceinline__ uint64_t sdesc_mn_sw128(uint32_t addr, uint32_t chunk) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | (uint64_t)(chunk >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 |
           (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// A from tensor memory: row = lane, two 16-bit values a column.
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
// The same onto 2^-N of what is there.
template <int N> __device__ __forceinline__ void mma_ts_down(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, 1, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p, %4;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "n"(N)
        : "memory");
}
#define QVL_R8(r, o) "=r"(r[o]), "=r"(r[o + 1]), "=r"(r[o + 2]), "=r"(r[o + 3]), "=r"(r[o + 4]), "=r"(r[o + 5]), "=r"(r[o + 6]), "=r"(r[o + 7])
#define QVL_V8(r, o) "r"(r[o]), "r"(r[o + 1]), "r"(r[o + 2]), "r"(r[o + 3]), "r"(r[o + 4]), "r"(r[o + 5]), "r"(r[o + 6]), "r"(r[o + 7])
__device__ __forceinline__ void tmem_ld32(uint32_t t, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : QVL_R8(r, 0), QVL_R8(r, 8), QVL_R8(r, 16), QVL_R8(r, 24)
        : "r"(t));
}
__device__ __forceinline__ void tmem_st8(uint32_t t, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::QVL_V8(r, 0), "r"(t) : "memory");
}
__device__ __forceinline__ void tmem_ld8(uint32_t t, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];" : QVL_R8(r, 0) : "r"(t));
}
// Waits for this thread's loads; the values in r are not looked at before.
#define QVL_RW8(r, o) "+r"(r[o]), "+r"(r[o + 1]), "+r"(r[o + 2]), "+r"(r[o + 3]), "+r"(r[o + 4]), "+r"(r[o + 5]), "+r"(r[o + 6]), "+r"(r[o + 7])
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : QVL_RW8(r, 0), QVL_RW8(r, 8)::"memory");
}
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : QVL_RW8(r, 0), QVL_RW8(r, 8), QVL_RW8(r, 16), QVL_RW8(r, 24)::"memory");
}
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[8], uint32_t (&q)[8]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : QVL_RW8(r, 0), QVL_RW8(q, 0)::"memory");
}
#undef QVL_RW8
#undef QVL_R8
#undef QVL_V8
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.402823466e38f; }
// 2^(m - top) of what was held under the reference m <= top, which may be -inf both.
__device__ __forceinline__ float weight(float m, float top) { return m == top ? 1.0f : ex2(m - top); }
template <int N> __device__ __forceinline__ void regs_more() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_less() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
// A whole warp's wait: false for all lanes where one gave up.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity) {
    return __all_sync(~0u, tc::mbar_wait(bar, parity, &g_tree_timeout));
}

// Two fp32 operations in one instruction.
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
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
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
// A pair as hi + 2^-kLow lo, 16 bits each: hi rounded, what is left of it exact before its own rounding.
template <typename C> __device__ __forceinline__ void split2(float a, float b, uint32_t &hi, uint32_t &lo) {
    constexpr float up = Held<C>::kLowUp;
    hi = pack2<C>(a, b);
    const float2 h = unpack2<C>(hi);
    float2 l;
    if constexpr (up == 1.0f) l = parts(add2(two(a, b), two(-h.x, -h.y)));
    else l = parts(fma2(two(h.x, h.y), two(-up, -up), fma2(two(a, b), two(up, up), two(-0.0f, -0.0f))));
    lo = pack2<C>(l.x, l.y);
}
// Both halves of a packed pair are finite; the pair with those that are not set to 0.
template <typename C> __device__ __forceinline__ bool finite2(uint32_t v) {
    constexpr uint32_t e = std::is_same<C, __half>::value ? 0x7c00u : 0x7f80u;
    return (v & e) != e && ((v >> 16) & e) != e;
}
template <typename C> __device__ __forceinline__ uint32_t held2(uint32_t v) {
    constexpr uint32_t e = std::is_same<C, __half>::value ? 0x7c00u : 0x7f80u;
    return ((v & e) == e ? 0u : v & 0xffffu) | (((v >> 16) & e) == e ? 0u : v & 0xffff0000u);
}
template <typename T> __device__ __forceinline__ void store4(T *o, const float4 &acc, bool none, float inv) {
    const float4 x = none ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4 *>(o) = x;
    else *reinterpret_cast<uint2 *>(o) = make_uint2(pack2<T>(x.x, x.y), pack2<T>(x.z, x.w));
}
// Eight outputs acc / l (`inv` = 1 / l), rounded once.
template <typename T> __device__ __forceinline__ void store8(T *o, const float *acc, bool none, float inv) {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = none ? 0.0f : acc[e] * inv;
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4 *>(o) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4 *>(o + 4) = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        *reinterpret_cast<uint4 *>(o) = make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
    }
}

// ---- the work ----
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
struct Request {
    int first, n, ctx, L, tiles, row_tiles;
    // A pair (key head, tile of rows) has `begin` units ahead of its tiles.
    __device__ __forceinline__ long units(int NKV, int begin) const { return (long)(tiles + begin) * row_tiles * NKV; }
};
__device__ __forceinline__ Request request_of(const TreeArgs &a, int s) {
    Request r;
    r.n = node_count(a, s, r.first);
    r.L = context(a, s, r.n, r.ctx);
    r.tiles = (r.L + kTile - 1) / kTile;
    const int per = kRows / (a.NH / a.NKV);     // whole nodes of a tile of rows
    r.row_tiles = (r.n + per - 1) / per;
    return r;
}
// Where a CTA's stretch is being cut: request, units into it, and units to go.
struct Cut {
    int s, begin;
    long off, left;
};
// A range of the tiles of one pair.  part: -1 whole pair; otherwise the place in
// the CTA's half of the workspace.
struct Segment {
    int s, kvh, r0, rows, tile0, nt, ctx, L, first, n, part, pad;
};
// What the joining launch knows of a partial segment.
struct Part {
    int first, kvh, r0, rows;      // rows 0: nothing
    int behind, s;                 // the CTAs after this one that have parts of the pair too; its request
};
// The next segment of a stretch (false at its end), and the pair's units behind it.
__device__ __forceinline__ bool next_segment(const TreeArgs &a, int q_rows, Cut &c, Request &rq, Segment &g, int &behind) {
    while (c.left > 0) {
        while (c.off >= rq.units(a.NKV, c.begin)) {
            c.off -= rq.units(a.NKV, c.begin);
            rq = request_of(a, ++c.s);
        }
        // key head, then tile of rows, then the units of the pair
        const int len = rq.tiles + c.begin;
        const int pair = c.off < 1l << 31 ? (int)((uint32_t)c.off / (uint32_t)len) : (int)(c.off / len);
        const int u0 = (int)(c.off - (long)pair * len), u1 = (int)min((long)u0 + c.left, (long)len);
        c.off += u1 - u0;
        c.left -= u1 - u0;
        g.tile0 = max(u0 - c.begin, 0);
        g.nt = max(u1 - c.begin, 0) - g.tile0;
        if (g.nt <= 0) continue;                           // ended before the pair's first tile
        g.s = c.s;
        g.kvh = pair / rq.row_tiles;
        g.r0 = (pair - g.kvh * rq.row_tiles) * q_rows;
        g.rows = min(q_rows, rq.n * (a.NH / a.NKV) - g.r0);
        g.ctx = rq.ctx;
        g.L = rq.L;
        g.first = rq.first;
        g.n = rq.n;
        const bool starts = g.tile0 == 0, ends = g.tile0 + g.nt == rq.tiles;
        g.part = starts && ends ? -1 : starts ? 1 : 0;
        behind = len - u1;
        return true;
    }
    g.nt = 0;
    return false;
}

template <typename T, int D, int CAP>
struct Conf {
    static constexpr bool kSplitQ = std::is_same<T, float>::value;
    static constexpr int kQHalves = kSplitQ ? 2 : 1;
    static constexpr int kSlot = kTile * D * 2;
    static constexpr int kQBox = CAP * 128, kQBoxes = D * (int)sizeof(T) / 128;      // queries: boxes of 128 bytes a row
    static constexpr int kPitch = D / 2 * (CAP == 64 ? 1 : 2) / 2 + 4;  // floats of a row that a block hands to the others
    static constexpr int kBlocks = CAP < kRows ? 2 * kRows * kPitch * 4 : 0;
    static constexpr int kMaxRing = 4;
    // Buffers of scores.  With three a warpgroup finds its next tile's scores made when it is through
    // with a tile; with two they wait for its probabilities' product (12 requests of
    // 132 rows over 6000 positions, D 64: 38 and 42 us).  At D 128 there is no room for a third.
    static constexpr int kNS = D == 64 ? 3 : 2;
    // tensor memory columns: scores and probabilities (128 each), O, Q
    static constexpr uint32_t kTmO = kNS * kTile, kTmQ = kTmO + D;
    static_assert(kTmQ + kQHalves * D / 2 <= 512, "");
};
// Shared memory of a launch: what an SM has goes to the rings.
struct Layout {
    int nk, nv;         // slots for K and for V
    int words;          // of a node's ancestors
    int anc_bytes;
    int box, box_log2;  // positions per TMA box
    uint32_t all;       // a bit for each box of a tile (and half of D)
    int q_rows;         // query rows of a tile: whole nodes
    int smem;
};
// What does not depend on the launch.
struct Fixed {
    float ref[4][kRows];            // references, by tile
    float cs[2][kRows];             // score factors, by segment
    float l[2][2][kRows];           // sums of p, by segment and warpgroup
    float m[2][2][kRows];           // references, by segment and warpgroup
    float qmax[2][kRows];           // maxima of a query row's halves
    Segment seg[4];
    Cut cut;                        // the whole stretch
    int again;                      // some output of a whole pair is not finite
    uint64_t k_full[4], k_empty[4], v_full[4], v_empty[4], s_full[3], s_free[3], p_ready[3], o_full, o_empty, q_load, q_full,
        q_empty, anc_full[2], seg_full[4], seg_empty[4], l_bar[2], seg_done[2], qmax_bar, block_bar[2], fix_ask, fix_done;
    uint32_t valid[8];              // boxes of a tile that exist, by tile
    uint32_t bad[8][4];             // positions with values held back, by tile
    uint32_t moved[4][4];           // some reference moved, by tile and warp
    uint32_t tmem;
    int off;
};
constexpr uint32_t kTmCols = 512;       // of tensor memory: all

__host__ __device__ constexpr size_t part_floats(int D) { return (size_t)kRows * D; }
__host__ __device__ constexpr size_t part_bytes(int D) {
    return (size_t)kSMs * (2 * (part_floats(D) * sizeof(float) + kRows * sizeof(float2)) + sizeof(Part));
}
struct Workspace {
    float *acc;         // [CTA][2][row][D]
    float2 *ml;         // [CTA][2][row]: maximum, sum
    Part *part;         // [CTA]: the pair that begins in its last segment and goes on behind it
};
__device__ __forceinline__ Workspace workspace_of(void *p, int D) {
    Workspace w;
    w.acc = static_cast<float *>(p);
    w.ml = reinterpret_cast<float2 *>(w.acc + (size_t)kSMs * 2 * part_floats(D));
    w.part = reinterpret_cast<Part *>(w.ml + (size_t)kSMs * 2 * kRows);
    return w;
}

// Half of a query row from shared memory (rows of 128 bytes, 128-byte swizzle) into
// tensor memory (columns of two 16-bit values, hi and then lo) by the thread of the row,
// and the row's score factor.  False where a wait gave up.
template <typename T, typename C, int D, int CAP>
__device__ __forceinline__ bool stage_queries(const TreeArgs &a, Fixed &fx, const unsigned char *q_s, float *cs_s,
                                              uint32_t tq, int half, int row, int turn) {
    using F = Conf<T, D, CAP>;
    constexpr int H = D / 2, V = 16 / sizeof(T);             // values of 16 bytes
    const int lane = threadIdx.x & 31, src = row & (CAP - 1);
    const float qmul = a.scale * kLog2e;
    // values [c, c + V) of the half
    auto load = [&](int c, float (&x)[V]) {
        const int byte = (half * H + c) * (int)sizeof(T), chunk = byte >> 7;
        const unsigned char *p = q_s + chunk * F::kQBox;
        const uint4 v = *reinterpret_cast<const uint4 *>(p + src * 128 + ((((byte >> 4) & 7) ^ (src & 7)) << 4));
        const T *t = reinterpret_cast<const T *>(&v);
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] = to_f32(t[e]);
    };
    float f = qmul < 0.0f ? -1.0f : 1.0f, cs = fmaxf(fabsf(qmul), 1.175494351e-38f);     // (times -inf: -inf)
    if constexpr (F::kSplitQ) {
        float mx = 0.0f;
#pragma unroll 4
        for (int c = 0; c < H; c += V) {
            float x[V];
            load(c, x);
#pragma unroll
            for (int e = 0; e < V; ++e) mx = fmaxf(mx, fabsf(x[e] * qmul));
        }
        fx.qmax[half][row] = mx;
        __syncwarp();
        if (lane == 0) mbar_arrive(tc::smem_u32(&fx.qmax_bar));
        if (!warp_wait(tc::smem_u32(&fx.qmax_bar), turn & 1)) return false;
        mx = fmaxf(mx, fx.qmax[half ^ 1][row]);
        // largest value into [2^9, 2^10)
        int ex = (int)(__float_as_uint(mx) >> 23);
        if (mx == 0.0f || ex == 255) ex = 127 + 9;
        ex = max(ex, 10);
        f = __uint_as_float((uint32_t)min(254, 263 - ex) << 23);
        cs = __uint_as_float((uint32_t)(ex - 9) << 23);
    }
#pragma unroll 1
    for (int c = 0; c < H; c += 16) {
        uint32_t hi[8], lo[8];
#pragma unroll
        for (int v = 0; v < 16 / V; ++v) {
            float x[V];
            load(c + v * V, x);
#pragma unroll
            for (int e = 0; e < V; e += 2) {
                const int at = (v * V + e) / 2;
                const float y = F::kSplitQ ? x[e] * qmul * f : x[e] * f, z = F::kSplitQ ? x[e + 1] * qmul * f : x[e + 1] * f;
                hi[at] = pack2<C>(y, z);
                if constexpr (F::kSplitQ) {
                    const float2 w = unpack2<C>(hi[at]);
                    lo[at] = pack2<C>(y - w.x, z - w.y);
                }
            }
        }
        tmem_st8(tq + half * (H / 2) + c / 2, hi);
        if constexpr (F::kSplitQ) tmem_st8(tq + D / 2 + half * (H / 2) + c / 2, lo);
    }
    tmem_wait_st();
    tc::tc_fence_before();
    if (half == 0) cs_s[row] = cs;
    return true;
}
// Ancestors of every node as bits, its own among them: a node's are its parent's and itself.  One warp.
__device__ __forceinline__ void stage_ancestors(const TreeArgs &a, const Segment &g, uint32_t *anc, int words, int lane) {
    for (int i0 = 0; i0 < g.n; i0 += 32) {
        const int mine = i0 + lane < g.n ? a.parents[g.first + i0 + lane] : -1;
        for (int i = i0; i < min(i0 + 32, g.n); ++i) {
            const int p = __shfl_sync(~0u, mine, i - i0);
            if (lane < words) {
                uint32_t v = p >= 0 && p < i ? anc[p * words + lane] : 0u;
                if (lane == (i >> 5)) v |= 1u << (i & 31);
                anc[i * words + lane] = v;
            }
            __syncwarp();
        }
    }
}
// What a row sees of positions t0 .. t0 + 31, of its ancestors' bits.
__device__ __forceinline__ uint32_t seen_word(const uint32_t *anc, int words, int t0, int ctx, int L) {
    if (t0 >= L) return 0u;
    uint32_t m;
    const int off = t0 - ctx;                   // the node at t0
    if (off <= -32) {
        m = ~0u;
    } else if (off < 0) {
        m = ((1u << -off) - 1u) | (anc[0] << -off);
    } else {
        const int w = off >> 5, b = off & 31;
        const uint32_t lo = w < words ? anc[w] : 0u, hi = w + 1 < words ? anc[w + 1] : 0u;
        m = __funnelshift_r(lo, hi, b);
    }
    return L - t0 < 32 ? m & ((1u << (L - t0)) - 1u) : m;
}
// Outputs of one row (node, head h of the key head's group) that are not finite, by a warp and by
// definition in fp32: of a score that is NaN or inf, NaN; a score of -inf has no weight, every other one a
// weight above 0 (it may meet an infinite value), and a row without weights is 0.  Outputs that are finite
// stay as they are.  A lane has a position's score, 32 at a time.
// Where some outputs are finite, the weights are: the others are infinite or NaN by the values
// alone that are, which are looked for in their columns.  Measured: 16 requests of 64 nodes over 32768
// positions, every page with a NaN among its values, 12.6 ms (each row anew, two bytes of a key at a time: 326
// ms); 32 of 16 nodes over 4096, fp32, keys with -inf in them, half the rows anew, 9.1 ms.
template <typename T, typename C, int D>
__device__ __forceinline__ void fix_row(const TreeArgs &a, int s, int ctx, int L, int first, int kvh, int node, int h, int lane) {
    constexpr int E = D / 32, V = 16 / sizeof(T);
    const long at = (((long)first + node) * a.NH + (long)kvh * (a.NH / a.NKV) + h) * D;
    T *out = reinterpret_cast<T *>(a.out) + at + lane * E;
    const T *q = reinterpret_cast<const T *>(a.q) + ((long)first + node) * a.q_stride + ((long)kvh * (a.NH / a.NKV) + h) * D;
    uint32_t odd = 0;                           // of this lane's outputs
#pragma unroll
    for (int e = 0; e < E; ++e) odd |= finite(to_f32(out[e])) ? 0u : 1u << e;
    if (!__any_sync(~0u, odd)) return;
    // the node and its ancestors: lane l has nodes 32 l to 32 l + 31
    uint32_t mine = 0;
    for (int j = node; j >= 0;) {
        if (lane == (j >> 5)) mine |= 1u << (j & 31);
        const int p = a.parents[first + j];
        j = p < j ? p : -1;
    }
    // row of the cache that holds position t, or -1: not seen, or on no page
    auto row_of = [&](int t) -> long {
        const int j = t - ctx;
        const uint32_t w = __shfl_sync(~0u, mine, max(j, 0) >> 5);
        if (t >= L || (j >= 0 && !((w >> (j & 31)) & 1u))) return -1;
        const int c = t / a.P, pg = a.table[(size_t)s * a.maxp + c];
        return pg >= 0 && pg < a.num_pages ? ((long)pg * a.NKV + kvh) * a.P + (t - c * a.P) : -1;
    };
    const C *kp = reinterpret_cast<const C *>(a.k_pages), *vp = reinterpret_cast<const C *>(a.v_pages);
    auto score = [&](long r) {
        if (r < 0) return -INFINITY;
        float x = 0.0f;
#pragma unroll 4
        for (int c = 0; c < D; c += V) {
            const uint4 qv = *reinterpret_cast<const uint4 *>(q + c);
            uint32_t k[V / 2];
            if constexpr (V == 8) *reinterpret_cast<uint4 *>(k) = *reinterpret_cast<const uint4 *>(kp + r * D + c);
            else *reinterpret_cast<uint2 *>(k) = *reinterpret_cast<const uint2 *>(kp + r * D + c);
#pragma unroll
            for (int e = 0; e < V; e += 2) {
                const T *y = reinterpret_cast<const T *>(&qv) + e;
                const float2 w = unpack2<C>(k[e / 2]);
                x = fmaf(to_f32(y[1]) * a.scale, w.y, fmaf(to_f32(y[0]) * a.scale, w.x, x));
            }
        }
        return x;
    };
    bool whole = !__any_sync(~0u, odd != (1u << E) - 1u);
    for (int col = 0; col < D && !whole; ++col) {
        if (!((__shfl_sync(~0u, odd, col / E) >> (col % E)) & 1u)) continue;
        uint32_t kinds = 0;                     // 1: inf, 2: -inf, 4: NaN
        for (int t = 0; t < L; t += 128) {
            long r[4];
            float v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) r[u] = row_of(t + u * 32 + lane);
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = r[u] < 0 ? 0.0f : to_f32(vp[r[u] * D + col]);
#pragma unroll 1
            for (int u = 0; u < 4; ++u) {
                const float x = u == 0 ? v[0] : u == 1 ? v[1] : u == 2 ? v[2] : v[3];
                if (finite(x)) continue;
                if (score(u == 0 ? r[0] : u == 1 ? r[1] : u == 2 ? r[2] : r[3]) > -INFINITY) kinds |= x > 0.0f ? 1u : x < 0.0f ? 2u : 4u;
            }
        }
        kinds = __reduce_or_sync(~0u, kinds);
        whole = kinds == 0;                     // (those found have no weight)
        if (!whole && lane == col / E) out[col % E] = from_f32<T>(kinds == 1 ? INFINITY : kinds == 2 ? -INFINITY : NAN);
    }
    if (!whole) return;
    float m = -INFINITY, l = 0.0f, acc[E];
    bool none = false;                          // a score of inf or NaN
    for (int t = 0; t < L && !none; t += 32) {
        const float x = score(row_of(t + lane));
        none = __any_sync(~0u, !(x < INFINITY));
        m = fmaxf(m, x);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.0f;
    for (int t = 0; t < L && !none; t += 32) {
        const long r = row_of(t + lane);
        const float x = score(r), p = x > -INFINITY ? fmaxf(expf(x - m), 1.175494351e-38f) : 0.0f;
        l += p;
#pragma unroll 8
        for (int u = 0; u < 32; ++u) {
            const float w = __shfl_sync(~0u, p, u);
            const C *v = vp + __shfl_sync(~0u, r, u) * D + lane * E;
#pragma unroll
            for (int e = 0; e < E; e += 2) {
                const float2 y = unpack2<C>(w > 0.0f ? *reinterpret_cast<const uint32_t *>(v + e) : 0u);
                acc[e] = fmaf(w, y.x, acc[e]);
                acc[e + 1] = fmaf(w, y.y, acc[e + 1]);
            }
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(~0u, l, o);
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const float y = none ? NAN : l == 0.0f ? 0.0f : acc[e] / l;
        if (!finite(to_f32(out[e]))) out[e] = from_f32<T>(y);
    }
}
// A place in a ring of n slots: the slot, and the parity of its turn.
struct Turn {
    int slot = 0;
    uint32_t parity = 0;
    __device__ __forceinline__ void step(int n) {
        if (++slot == n) {
            slot = 0;
            parity ^= 1;
        }
    }
};
// TMA load whose lines leave L2 first: the cache is read once, and would push
// everything else out.
__device__ __forceinline__ void tma_load_once(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar, uint64_t pol) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %3}], "
        "[%4], %5;" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar), "l"(pol)
        : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap *map, int x, int y, int z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}
}  // namespace

// CAP: rows of a block (32, 64 or 128).
template <typename T, typename C, int D, int CAP>
__global__ void __launch_bounds__(kThreads, 1)
tree_tc_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
               const __grid_constant__ CUtensorMap tm_q,
               const __grid_constant__ TreeArgs a, const __grid_constant__ Layout ly) {
    using F = Conf<T, D, CAP>;
    // (addresses in it are constants, which keeps them out of the registers)
    extern __shared__ __align__(1024) unsigned char smem[];
    Fixed &fx = *reinterpret_cast<Fixed *>(smem);
    constexpr int kHead = ((int)sizeof(Fixed) + 1023) & ~1023;
    unsigned char *k_s = smem + kHead;                              // slots of K, of V
    unsigned char *v_s = k_s + ly.nk * F::kSlot;
    unsigned char *q_s = v_s + ly.nv * F::kSlot;                    // a segment's queries
    uint32_t *anc_s = reinterpret_cast<uint32_t *>(q_s + F::kQBoxes * F::kQBox);    // [2][node][words], by segment
    // the blocks' sums, to be added: [half of D][row][pitch]
    float *blocks_s = reinterpret_cast<float *>(q_s + F::kQBoxes * F::kQBox + ly.anc_bytes);
    auto bar = [](uint64_t &b) { return tc::smem_u32(&b); };

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int G = a.NH / a.NKV;

    if (tid == 0) {
        for (int i = 0; i < 4; ++i) {
            tc::mbar_init(bar(fx.k_full[i]), 1);
            tc::mbar_init(bar(fx.k_empty[i]), 1);
            tc::mbar_init(bar(fx.v_full[i]), 1);
            tc::mbar_init(bar(fx.v_empty[i]), 1);
            tc::mbar_init(bar(fx.seg_full[i]), 1);
            tc::mbar_init(bar(fx.seg_empty[i]), 19);
        }
        for (int i = 0; i < F::kNS; ++i) {
            tc::mbar_init(bar(fx.s_full[i]), 1);
            tc::mbar_init(bar(fx.s_free[i]), 1);
            tc::mbar_init(bar(fx.p_ready[i]), 128);
        }
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(bar(fx.anc_full[i]), 1);
            tc::mbar_init(bar(fx.l_bar[i]), 256);
            tc::mbar_init(bar(fx.seg_done[i]), 16);
        }
        tc::mbar_init(bar(fx.o_full), 1);
        tc::mbar_init(bar(fx.o_empty), 256);
        tc::mbar_init(bar(fx.q_load), 1);
        tc::mbar_init(bar(fx.q_full), 256);
        tc::mbar_init(bar(fx.q_empty), 1);
        tc::mbar_init(bar(fx.qmax_bar), 8);
        tc::mbar_init(bar(fx.block_bar[0]), 4);
        tc::mbar_init(bar(fx.block_bar[1]), 4);
        tc::mbar_init(bar(fx.fix_ask), 1);
        tc::mbar_init(bar(fx.fix_done), 32);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        tc::prefetch_tmap(&tm_k);
        tc::prefetch_tmap(&tm_v);
        tc::prefetch_tmap(&tm_q);
    }
    if (warp == kScoreWarp) {
        tc::tmem_alloc(tc::smem_u32(&fx.tmem), kTmCols);
        tc::tmem_relinquish();
    }
    pdl_wait();
    if (tid == 0) {
        fx.off = *reinterpret_cast<volatile int *>(&g_tree_timeout);
        fx.again = 0;
    }

    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    pdl_launch_dependents();
    const uint32_t tmem = fx.tmem;
    bool ok = fx.off == 0 && (tc::smem_u32(smem) & 1023) == 0;
    const Workspace ws = workspace_of(a.workspace, D);
    int seg = 0, i = 0;                 // segments and tiles so far, in step in all roles
    auto next = [&](const Segment *&g) {        // the segment, or false at the end
        if (!(ok = warp_wait(bar(fx.seg_full[seg & 3]), (seg >> 2) & 1))) return false;
        g = &fx.seg[seg & 3];
        return g->nt > 0;
    };
    auto done = [&] {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(fx.seg_empty[seg & 3]));
        ++seg;
    };

    if (warp == kTmaWarp) {
        regs_less<kRestRegs>();
        // ---- segments, pages and loads ----
        // this CTA's stretch of all units: [lo, hi), found among the requests 32 at a time
        // (sums over the requests up to each lane's; of up to 32 requests they stay)
        Request mine{};
        long tiles = 0, pairs = 0, tiles_to = 0, pairs_to = 0;
        auto sums = [&](int base) {
            mine = Request{};
            if (base + lane < a.S) mine = request_of(a, base + lane);
            pairs_to = mine.row_tiles * (long)a.NKV;
            tiles_to = pairs_to * mine.tiles;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long t = __shfl_up_sync(~0u, tiles_to, o), p = __shfl_up_sync(~0u, pairs_to, o);
                tiles_to += lane >= o ? t : 0;
                pairs_to += lane >= o ? p : 0;
            }
        };
        for (int base = 0; base < a.S; base += 32) {
            sums(base);
            tiles += __shfl_sync(~0u, tiles_to, 31);
            pairs += __shfl_sync(~0u, pairs_to, 31);
        }
        // What a pair costs beside its tiles, in tiles: about four where blocks have to be
        // added and tiles are quick, two otherwise (32 requests of up to 16 nodes over 4096: 82
        // us with 1, 78 with 2, 79 with 3, 76 with 4, 77 with 6; 16 of 128 rows over 32768 and 12 of
        // 132 over 6000: 269 and 43.7 with 0, 267 and 42.6 with 1, 265 and 42.7 with 2,
        // 264 and 43.0 with 3).  Where there are fewer tiles than CTAs, each tile gets its own.
        const int begin = tiles > gridDim.x ? (CAP < kRows ? 4 : 2) : 0;
        const long total = tiles + pairs * begin;
        // (fewer units than CTAs: the last CTAs have none, so that a pair's parts
        // are in consecutive CTAs)
        const long ctas = min((long)gridDim.x, max(total, 1l)), me = blockIdx.x;
        long each, more;
        if (total < 1l << 31) {
            each = (uint32_t)total / (uint32_t)ctas;
            more = (uint32_t)total % (uint32_t)ctas;
        } else {
            each = total / ctas;
            more = total % ctas;
        }
        const long lo = min(each * me + min(me, more), total), hi = min(lo + each + (me < more ? 1 : 0), total);
        int s = 0;
        long off = lo;
        Request rq{};
        for (int base = 0; ok && hi > lo; base += 32) {
            if (a.S > 32) sums(base);
            const long inc = tiles_to + pairs_to * begin;
            const uint32_t past = __ballot_sync(~0u, inc > off);
            if (past) {
                const int at = __ffs(past) - 1;
                const long before = __shfl_sync(~0u, inc, max(at - 1, 0));
                s = base + at;
                off -= at ? before : 0;
                rq.first = __shfl_sync(~0u, mine.first, at);
                rq.n = __shfl_sync(~0u, mine.n, at);
                rq.ctx = __shfl_sync(~0u, mine.ctx, at);
                rq.L = __shfl_sync(~0u, mine.L, at);
                rq.tiles = __shfl_sync(~0u, mine.tiles, at);
                rq.row_tiles = __shfl_sync(~0u, mine.row_tiles, at);
                break;
            }
            off -= __shfl_sync(~0u, inc, 31);
        }
        Cut cut{s, begin, off, ok ? hi - lo : 0};
        if (lane == 0) {
            ws.part[blockIdx.x].rows = 0;
            fx.cut = cut;
        }
        __syncwarp();
        // lane l: box l / (D / 64) of the tile's 64-value half l % (D / 64)
        const int lanes = (kTile >> ly.box_log2) * (D / 64);
        const int bx = lane / (D / 64), half = lane % (D / 64);
        const int oob = (int)(a.num_pages * a.NKV * a.P);          // past the last row: zeros
        const int to = half * (kTile * 128) + bx * ly.box * 128;
        Turn kt, vt;
        int keys = 0;                                              // loads of K so far
        int queries = 0;                                           // and of queries
        uint64_t once;
        asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(once));
        while (ok) {
            Segment g{};
            int behind = 0;                                        // the pair's units after the segment
            next_segment(a, ly.q_rows, cut, rq, g, behind);
            if (seg >= 4) ok = warp_wait(bar(fx.seg_empty[seg & 3]), ((seg >> 2) - 1) & 1);
            if (!ok) break;
            if (lane == 0) {
                fx.seg[seg & 3] = g;
                mbar_arrive(bar(fx.seg_full[seg & 3]));
            }
            ++seg;
            if (g.nt == 0) break;
            // (the place is free when the queries before are in tensor memory)
            if (seg > 1 && !(ok = warp_wait(bar(fx.q_full), seg & 1))) break;
            if (lane == 0) tc::mbar_expect_tx(bar(fx.q_load), F::kQBoxes * ly.q_rows * 128);
            __syncwarp();
            if (lane < F::kQBoxes)
                tma_load_3d(tc::smem_u32(q_s + lane * F::kQBox), &tm_q, lane * (128 / (int)sizeof(T)), g.kvh * G,
                            g.first + g.r0 / G, bar(fx.q_load));
            ++queries;
            // rows of the cache that 32 boxes start at (those of several tiles), one a lane, a
            // group ahead: behind the loads of K and V an answer takes microseconds
            const int nb = kTile >> ly.box_log2, group = 32 / nb;
            auto rows_of = [&](int k) {
                const int t = (g.tile0 + k + lane / nb) * kTile + (lane % nb << ly.box_log2);
                if (t >= g.L || k + lane / nb >= g.nt) return oob;
                const int c = t / a.P;
                const int pg = a.table[(size_t)g.s * a.maxp + c];
                return pg >= 0 && pg < a.num_pages ? (int)(((long)pg * a.NKV + g.kvh) * a.P + (t - c * a.P)) : oob;
            };
            int ahead = rows_of(0), rows_now = 0;
            for (int k = 0; k < g.nt; ++k, ++i) {
                if (k % group == 0) {
                    rows_now = ahead;
                    ahead = k + group < g.nt ? rows_of(k + group) : oob;
                }
                int y = __shfl_sync(~0u, rows_now, (k % group * nb + bx) & 31);
                if (lane >= lanes) y = oob;
                const uint32_t there = __ballot_sync(~0u, y != oob);
                if (i >= ly.nk && !(ok = warp_wait(bar(fx.k_empty[kt.slot]), kt.parity ^ 1))) break;
                if (lane == 0) {
                    // (keys are loaded at most nk + 2 tiles, six, ahead of the softmax that
                    // reads this)
                    fx.valid[i & 7] = there;
                    tc::mbar_expect_tx(bar(fx.k_full[kt.slot]), F::kSlot);
                }
                __syncwarp();
                if (lane < lanes)
                    tma_load_once(tc::smem_u32(k_s + kt.slot * F::kSlot + to), &tm_k, half * 64, y, bar(fx.k_full[kt.slot]), once);
                kt.step(ly.nk);
                ++keys;
                if (i >= ly.nv && !(ok = warp_wait(bar(fx.v_empty[vt.slot]), vt.parity ^ 1))) break;
                if (lane == 0) tc::mbar_expect_tx(bar(fx.v_full[vt.slot]), F::kSlot);
                __syncwarp();
                if (lane < lanes)
                    tma_load_once(tc::smem_u32(v_s + vt.slot * F::kSlot + to), &tm_v, half * 64, y, bar(fx.v_full[vt.slot]), once);
                vt.step(ly.nv);
            }
            if (g.part == 1 && lane == 0) {
                // the CTA that has the pair's last unit
                const long x = hi - cut.left + behind - 1, y = x - more * (each + 1);
                const long last = total < 1l << 31 ? (y < 0 ? (uint32_t)x / (uint32_t)(each + 1) : more + (uint32_t)y / (uint32_t)each)
                                                   : (y < 0 ? x / (each + 1) : more + y / each);
                ws.part[blockIdx.x] = {g.first, g.kvh, g.r0, g.rows, (int)(last - me), g.s};
            }
        }
        // after a wait that gave up: loads in flight land before the CTA ends
        // (each slot's last load; a slot never filled has nothing in flight)
        if (!ok) {
            if (queries > 0) tc::mbar_wait(bar(fx.q_load), (queries - 1) & 1, nullptr);
            for (int n = 0; n < min(keys, ly.nk); ++n) tc::mbar_wait(bar(fx.k_full[n]), (((keys - 1 - n) / ly.nk) & 1), nullptr);
            for (int n = 0; n < min(i, ly.nv); ++n) tc::mbar_wait(bar(fx.v_full[n]), (((i - 1 - n) / ly.nv) & 1), nullptr);
        }
    } else if (warp == kScoreWarp) {
        regs_less<kRestRegs>();
        // ---- scores.  Low halves first: what they add up to is small, and exact beside
        // the roundings of the high halves' sums ----
        if (lane == 0) {
            constexpr uint32_t id = idesc_16<C>(kTile, false);
            const uint64_t kd = tc::sdesc_k_sw128(tc::smem_u32(k_s));     // the address is its low end, in units of 16 bytes
            Turn kt;
            auto wait = [&](uint64_t &b, uint32_t parity) { return ok = tc::mbar_wait(bar(b), parity, &g_tree_timeout); };
            while (ok && wait(fx.seg_full[seg & 3], (seg >> 2) & 1)) {
                const int nt = *reinterpret_cast<volatile int *>(&fx.seg[seg & 3].nt);
                if (nt == 0 || !wait(fx.q_full, seg & 1)) break;
                for (int k = 0; k < nt; ++k, ++i) {
                    const int b = i % F::kNS;
                    if (i >= F::kNS && !wait(fx.s_free[b], (i / F::kNS - 1) & 1)) break;
                    if (!wait(fx.k_full[kt.slot], kt.parity)) break;
                    tc::tc_fence_after();
                    const uint64_t kb = kd + (uint32_t)(kt.slot * (F::kSlot >> 4));
                    const uint32_t d = tmem + b * kTile;
#pragma unroll
                    for (int l = F::kQHalves - 1; l >= 0; --l)
#pragma unroll
                        for (int c = 0; c < D / 16; ++c)
                            mma_ts(d, tmem + F::kTmQ + l * (D / 2) + c * 8, kb + ((c >> 2) * (kTile * 8) + (c & 3) * 2), id,
                                   l < F::kQHalves - 1 || c ? 1u : 0u);
                    tc::tc_commit(bar(fx.s_full[b]));
                    tc::tc_commit(bar(fx.k_empty[kt.slot]));
                    kt.step(ly.nk);
                }
                if (!ok) break;
                tc::tc_commit(bar(fx.q_empty));
                mbar_arrive(bar(fx.seg_empty[seg & 3]));
                ++seg;
            }
        }
    } else if (warp == kOutWarp) {
        regs_less<kRestRegs>();
        // ---- outputs ----
        if (lane == 0) {
            constexpr uint32_t id = idesc_16<C>(D, true);
            const uint64_t vd = sdesc_mn_sw128(tc::smem_u32(v_s), kTile * 128);
            Turn vt;
            auto wait = [&](uint64_t &b, uint32_t parity) { return ok = tc::mbar_wait(bar(b), parity, &g_tree_timeout); };
            int fixes = 0;
            while (ok && wait(fx.seg_full[seg & 3], (seg >> 2) & 1)) {
                const volatile Segment &sg = fx.seg[seg & 3];
                const int nt = sg.nt, plain = max(0, sg.ctx / kTile - sg.tile0);      // tiles before the drafted ones
                if (nt == 0) break;
                for (int k = 0; k < nt; ++k, ++i) {
                    const int b = i % F::kNS;
                    const bool tail = k >= plain;
                    // (the fixer is told one tile ahead: the slot of the tile's V then has its
                    // turn, and it waits for the load itself)
                    if (k == 0 && tail) mbar_arrive(bar(fx.fix_ask));
                    const bool ask = k + 1 < nt && k + 1 >= plain;
                    if (ask && !tail) mbar_arrive(bar(fx.fix_ask));
                    if (i >= 1 && !wait(fx.o_empty, (i - 1) & 1)) break;
                    if (!wait(fx.v_full[vt.slot], vt.parity)) break;
                    if (tail && !wait(fx.fix_done, fixes++ & 1)) break;
                    if (ask && tail) mbar_arrive(bar(fx.fix_ask));
                    if (!wait(fx.p_ready[b], (i / F::kNS) & 1)) break;
                    tc::tc_fence_after();
                    const uint64_t vb = vd + (uint32_t)(vt.slot * (F::kSlot >> 4));
                    const uint32_t pb = tmem + b * kTile, d = tmem + F::kTmO;
#pragma unroll
                    for (int l = 1; l >= 0; --l)
#pragma unroll
                        for (int c = 0; c < kTile / 16; ++c) {
                            if (l == 0 && c == 0) mma_ts_down<Held<C>::kLow>(d, pb, vb, id);
                            else mma_ts(d, pb + c * 16 + l * 8, vb + c * (2048 >> 4), id, l == 0 || c ? 1u : 0u);
                        }
                    tc::tc_commit(bar(fx.o_full));
                    tc::tc_commit(bar(fx.s_free[b]));
                    tc::tc_commit(bar(fx.v_empty[vt.slot]));
                    vt.step(ly.nv);
                }
                if (!ok) break;
                mbar_arrive(bar(fx.seg_empty[seg & 3]));
                ++seg;
            }
        }
    } else if (warp < kSumWarp) {
        regs_more<kMoreRegs>();
        // ---- softmax: thread = row, the tiles of this warpgroup's parity ----
        const int wg = warp >> 2, w4 = warp & 3, row = tid & 127;
        const uint32_t tr = tmem + ((uint32_t)(w4 * 32) << 16);
        const Segment *g;
        // the queries of segment n, after the products with those before them
        auto queries = [&](int n) {
            if (!(ok = warp_wait(bar(fx.seg_full[n & 3]), (n >> 2) & 1))) return;
            if (fx.seg[n & 3].nt == 0) return;
            if (n > 0 && !(ok = warp_wait(bar(fx.q_empty), (n - 1) & 1))) return;
            if (!(ok = warp_wait(bar(fx.q_load), n & 1))) return;
            tc::tc_fence_after();
            if ((ok = stage_queries<T, C, D, CAP>(a, fx, q_s, fx.cs[n & 1], tr + F::kTmQ, wg, row, n))) mbar_arrive(bar(fx.q_full));
        };
        if (ok) queries(0);
        while (ok && next(g)) {
            // (what is seldom needed is read from shared memory where it is)
            const volatile Segment &sg = fx.seg[seg & 3];
            const int nt = sg.nt;
            constexpr int cap = CAP, nc = cap / 16;     // chunks of 16 positions of a block
            const int r = row & (cap - 1);          // the row, in its block
            const bool active = (w4 * 32 & (cap - 1)) < sg.rows;
            const int c0 = row / cap * nc;          // the block's first chunk
            float m = -INFINITY, l = 0.0f;
            for (int k = 0; k < nt; ++k, ++i) {
                if ((i & 1) != wg) continue;
                const int b = i % F::kNS;
                const uint32_t sb = tr + b * kTile;
                if (!(ok = warp_wait(bar(fx.s_full[b]), (i / F::kNS) & 1))) break;
                tc::tc_fence_after();
                const int t0 = (sg.tile0 + k) * kTile, ctx = sg.ctx;
                const uint32_t there = *reinterpret_cast<volatile uint32_t *>(&fx.valid[i & 7]);
                const bool plain = t0 + kTile <= ctx && there == ly.all;
                if (t0 + kTile > ctx && !(ok = warp_wait(bar(fx.anc_full[seg & 1]), (seg >> 1) & 1))) break;
                bool moved = false;
                if (active) {
                    const float cs = fx.cs[seg & 1][row];
                    const uint64_t cs2 = two(cs, cs);
                    float mm = m == -INFINITY ? 0.0f : Held<C>::kBias - m;
                    uint64_t ls = two(0.0f, 0.0f);
                    // 32 positions at a time, enough of them to keep the pipes busy: their scores, and
                    // then the high and low halves of their p in the same columns, 16 by 16
                    auto part = [&](int c) {
                        uint32_t v[32];
                        tmem_ld32(sb + c * 16, v);
                        tmem_wait_ld(v);
                        if (!plain) {
                            // what the row sees of them
                            const uint32_t *anc = anc_s + ((seg & 1) * a.max_nodes + min((sg.r0 + r) / G, sg.n - 1)) * ly.words;
                            const uint32_t lo = (there >> ((c * 16 >> ly.box_log2) * (D / 64))) & 1u;
                            const uint32_t hi = (there >> ((c * 16 + 16 >> ly.box_log2) * (D / 64))) & 1u;
                            const uint32_t see = seen_word(anc, ly.words, t0 + c * 16, ctx, sg.L) &
                                                 ((lo ? 0xffffu : 0u) | (hi ? 0xffff0000u : 0u));
#pragma unroll
                            for (int e = 0; e < 32; ++e) v[e] = (see >> e) & 1u ? v[e] : 0xff800000u;
                        }
                        float t4[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) t4[e] = fmaxf(__uint_as_float(v[e]), __uint_as_float(v[28 + e]));
#pragma unroll
                        for (int e = 4; e < 28; e += 2)
                            t4[e / 2 % 4] = max3(t4[e / 2 % 4], __uint_as_float(v[e]), __uint_as_float(v[e + 1]));
                        const float mt = fmaxf(max3(t4[0], t4[1], t4[2]), t4[3]) * cs;
                        if (__any_sync(~0u, mt > m + Held<C>::kRise && r < sg.rows)) {
                            // a new reference, a whole power of two; what the tile has under the old one is
                            // taken down
                            moved = true;
                            float f = 1.0f;
                            if (mt > m + Held<C>::kRise && r < sg.rows) {
                                const float up = ceilf(mt);
                                f = ex2(m - up);
                                m = up;
                                mm = Held<C>::kBias - m;
                                l *= f;
                                ls = fma2(ls, two(f, f), two(-0.0f, -0.0f));
                            }
                            tmem_wait_st();
#pragma unroll 1
                            for (int x = c0; x < c; ++x) {
                                uint32_t hi[8], lo[8];
                                tmem_ld8(sb + x * 16, hi);
                                tmem_ld8(sb + x * 16 + 8, lo);
                                tmem_wait_ld(hi, lo);
#pragma unroll
                                for (int e = 0; e < 8; ++e) {
                                    const float2 h = unpack2<C>(hi[e]), w = unpack2<C>(lo[e]);
                                    constexpr float down = Held<C>::kLowDown;
                                    if (f != 1.0f) split2<C>(fmaf(w.x, down, h.x) * f, fmaf(w.y, down, h.y) * f, hi[e], lo[e]);
                                }
                                tmem_st8(sb + x * 16, hi);
                                tmem_st8(sb + x * 16 + 8, lo);
                            }
                        }
                        const uint64_t mm2 = two(mm, mm);
#pragma unroll
                        for (int b = 0; b < 2; ++b) {
                            uint32_t hi[8], lo[8];
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                const float2 x = parts(fma2(two(__uint_as_float(v[b * 16 + 2 * e]), __uint_as_float(v[b * 16 + 2 * e + 1])), cs2, mm2));
                                const float pa = ex2(x.x), pb = ex2(x.y);
                                ls = add2(ls, two(pa, pb));
                                split2<C>(pa, pb, hi[e], lo[e]);
                            }
                            tmem_st8(sb + (c + b) * 16, hi);
                            tmem_st8(sb + (c + b) * 16 + 8, lo);
                        }
                    };
#pragma unroll 1
                    for (int c = c0; c < c0 + nc; c += 2) part(c);
                    if constexpr (cap != kRows) {
                        // the other blocks' positions
                        const uint32_t none[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
                        for (int c = 0; c < 8; ++c)
                            if (c / nc != c0 / nc) {
                                tmem_st8(sb + c * 16, none);
                                tmem_st8(sb + c * 16 + 8, none);
                            }
                    }
                    l += parts(ls).x + parts(ls).y;
                    tmem_wait_st();
                }
                if (moved) fx.ref[i & 3][row] = m;
                if (lane == 0) fx.moved[i & 3][w4] = moved;
                tc::tc_fence_before();
                mbar_arrive(bar(fx.p_ready[b]));
            }
            // (one warpgroup is through with the segment a tile before the other)
            if (ok) queries(seg + 1);
            if (!ok || (seg > 1 && !(ok = warp_wait(bar(fx.seg_done[seg & 1]), ((seg >> 1) - 1) & 1)))) break;
            fx.l[seg & 1][wg][row] = l;
            fx.m[seg & 1][wg][row] = m;
            mbar_arrive(bar(fx.l_bar[seg & 1]));
            if (lane == 0) mbar_arrive(bar(fx.seg_done[seg & 1]));
            done();
        }
    } else if (warp < kTmaWarp) {
        regs_more<kMoreRegs>();
        // ---- output sums: thread = row, half of the head's values ----
        constexpr int CW = D / 2;
        const int half = (warp - kSumWarp) >> 2, w4 = warp & 3, row = tid & 127;
        const uint32_t to = tmem + ((uint32_t)(w4 * 32) << 16) + F::kTmO + half * CW;
        T *out = reinterpret_cast<T *>(a.out);
        // rows that no node owns get zeros
        for (int s = blockIdx.x; s < a.S; s += gridDim.x) {
            int first;
            const int n = node_count(a, s, first);
            auto clear = [&](long from, long to_) {
                for (long e = from * a.NH * D + (tid - kSumWarp * 32); e < to_ * a.NH * D; e += 256) out[e] = from_f32<T>(0.0f);
            };
            if (s == 0) clear(0, first);
            clear(first + n, s + 1 < a.S ? min(max(a.starts[s + 1], first), a.T) : a.T);
        }
        const Segment *g;
        int meets = 0;
        while (ok && next(g)) {
            const volatile Segment &sg = fx.seg[seg & 3];
            const int nt = sg.nt;
            constexpr int cap = CAP;
            const int r = row & (cap - 1);          // the row, in its block
            const bool active = (w4 * 32 & (cap - 1)) < sg.rows;
            uint64_t acc2[CW / 2];
#pragma unroll
            for (int c = 0; c < CW / 2; ++c) acc2[c] = two(0.0f, 0.0f);
            float top = -INFINITY, f0 = 1.0f, f1 = 1.0f;       // the larger reference; 2^(reference - top) of both
            for (int k = 0; k < nt; ++k, ++i) {
                if (!(ok = warp_wait(bar(fx.o_full), i & 1))) break;
                tc::tc_fence_after();
                // O is free for the next product as soon as it is in registers
                auto read = [&] {
                    tc::tc_fence_before();
                    mbar_arrive(bar(fx.o_empty));
                };
                if (!active) read();
                if (active) {
                    // (written before the probabilities, on which the product waited)
                    if (*reinterpret_cast<volatile uint32_t *>(&fx.moved[i & 3][w4])) {
                        const float m = fx.ref[i & 3][row];
                        if (__any_sync(~0u, m > top)) {
                            const float up = fmaxf(m, top), f = weight(top, up);
                            const uint64_t f2 = two(f, f), z = two(-0.0f, -0.0f);
#pragma unroll
                            for (int c = 0; c < CW / 2; ++c) acc2[c] = fma2(acc2[c], f2, z);
                            f0 *= f;
                            f1 *= f;
                            top = up;
                        }
                        (i & 1 ? f1 : f0) = weight(m, top);
                    }
                    const uint64_t f = i & 1 ? two(f1, f1) : two(f0, f0);
                    constexpr int step = D == 64 ? 32 : 16;         // (registers allow no more at D 128)
#pragma unroll
                    for (int c = 0; c < CW; c += step) {
                        uint32_t v[step];
                        if constexpr (step == 32) tmem_ld32(to + c, v);
                        else tc::tmem_ld16(to + c, v);
                        tmem_wait_ld(v);
                        if (c + step == CW) read();
#pragma unroll
                        for (int e = 0; e < step; e += 2)
                            acc2[(c + e) / 2] = fma2(two(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), f, acc2[(c + e) / 2]);
                    }
                    const int t0 = (sg.tile0 + k) * kTile, ctx = sg.ctx;
                    if (t0 + kTile > ctx) {
                        const uint32_t *anc = anc_s + ((seg & 1) * a.max_nodes + min((sg.r0 + r) / G, sg.n - 1)) * ly.words;
                        // values that were held back from the product: infinities and NaN
                        for (int w = 0; w < 4; ++w) {
                            const uint32_t bad = *reinterpret_cast<volatile uint32_t *>(&fx.bad[i & 7][w]);
                            if (!bad) continue;
                            // (by the block that has the position)
                            if (w * 32 / cap != row / cap) continue;
                            for (uint32_t x = bad & seen_word(anc, ly.words, t0 + 32 * w, ctx, sg.L); x; x &= x - 1) {
                                const int t = t0 + 32 * w + __ffs(x) - 1;
                                const int pg = a.table[(size_t)g->s * a.maxp + t / a.P];
                                const C *v = reinterpret_cast<const C *>(a.v_pages) +
                                             (((long)pg * a.NKV + g->kvh) * a.P + t % a.P) * D + half * CW;
#pragma unroll
                                for (int c = 0; c < CW; c += 2) {
                                    const float2 y = unpack2<C>(*reinterpret_cast<const volatile uint32_t *>(v + c));
                                    acc2[c / 2] = add2(acc2[c / 2], two(finite(y.x) ? 0.0f : y.x, finite(y.y) ? 0.0f : y.y));
                                }
                            }
                        }
                        __syncwarp();
                    }
                }
            }
            if (!ok || !(ok = warp_wait(bar(fx.l_bar[seg & 1]), (seg >> 1) & 1))) break;
            float acc[CW];
#pragma unroll
            for (int c = 0; c < CW / 2; ++c) {
                const float2 v = parts(acc2[c]);
                acc[2 * c] = v.x;
                acc[2 * c + 1] = v.y;
            }
            const float (*lp)[kRows] = fx.l[seg & 1], (*mp)[kRows] = fx.m[seg & 1];
            // reference and sum of a row of a block, of both warpgroups' tiles
            auto of_row = [&](int x, float &l) {
                const float m = fmaxf(mp[0][x], mp[1][x]);
                l = lp[0][x] * weight(mp[0][x], m) + lp[1][x] * weight(mp[1][x], m);
                return m;
            };
            const int node = (sg.r0 + r) / G, h = sg.r0 + r - node * G;
            T *o = out + ((long)(sg.first + node) * a.NH + sg.kvh * G + h) * D + half * CW;
            const int part = sg.part;
            const size_t at = ((size_t)blockIdx.x * 2 + max(part, 0)) * kRows + r;
            float m, l, odd;        // odd: a sum of all that goes out, not finite where a part of it is not
            if constexpr (cap == kRows) {
                m = of_row(r, l);
                odd = l;
                if (r < sg.rows) {
                    if (part < 0) {
                        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
                        for (int c = 0; c < CW; c += 8) store8(o + c, acc + c, l == 0.0f, inv);
#pragma unroll
                        for (int c = 0; c < CW; ++c) odd += acc[c];
                        if (!finite(odd)) fx.again = 1;
                    } else {
#pragma unroll
                        for (int c = 0; c < CW; c += 4)
                            *reinterpret_cast<float4 *>(ws.acc + at * D + half * CW + c) =
                                make_float4(acc[c], acc[c + 1], acc[c + 2], acc[c + 3]);
                    }
                }
            } else {
                // the blocks of a row are added; each of its threads has a share of the values
                constexpr int nb = kRows / cap, share = CW / nb;
                const int mine = row / cap;
                m = -INFINITY;
#pragma unroll
                for (int b = 0; b < nb; ++b) m = fmaxf(m, fmaxf(mp[0][b * cap + r], mp[1][b * cap + r]));
                l = 0.0f;
                for (int b = 0; b < nb; ++b) {
                    float lb;
                    const float mb = of_row(b * cap + r, lb);
                    l += lb * weight(mb, m);
                }
                const float f = weight(top, m), inv = l == 0.0f ? 0.0f : 1.0f / l;
                odd = l;
                auto meet = [&] {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(fx.block_bar[half]));
                    return ok = warp_wait(bar(fx.block_bar[half]), meets++ & 1);
                };
                float *mine_s = blocks_s + (half * kRows + row) * F::kPitch;
                if (!meet()) break;                 // (the segment before this one is read)
                if constexpr (nb == 2) {
                    // (each block hands over the other's share alone: there is room for no more)
#pragma unroll
                    for (int c = 0; c < share; ++c) {
                        const float keep = (mine ? acc[share + c] : acc[c]) * f;
                        acc[share + c] = (mine ? acc[c] : acc[share + c]) * f;
                        acc[c] = keep;
                    }
#pragma unroll
                    for (int c = 0; c < share; c += 4)
                        *reinterpret_cast<float4 *>(mine_s + c) = make_float4(acc[share + c], acc[share + c + 1], acc[share + c + 2], acc[share + c + 3]);
                } else {
#pragma unroll
                    for (int c = 0; c < CW; c += 4)
                        *reinterpret_cast<float4 *>(mine_s + c) = make_float4(acc[c] * f, acc[c + 1] * f, acc[c + 2] * f, acc[c + 3] * f);
                }
                if (!meet()) break;
                if (r < sg.rows) {
                    auto put = [&](int c, const float4 &v) {
                        odd += (v.x + v.y) + (v.z + v.w);
                        if (part < 0) store4(o + c, v, l == 0.0f, inv);
                        else *reinterpret_cast<float4 *>(ws.acc + at * D + half * CW + c) = v;
                    };
                    const float *from = blocks_s + (half * kRows + r) * F::kPitch;
                    if constexpr (nb == 2) {
                        from += (mine ^ 1) * cap * F::kPitch;
#pragma unroll
                        for (int c = 0; c < share; c += 4) {
                            const float4 w = *reinterpret_cast<const float4 *>(from + c);
                            put(mine * share + c, make_float4(acc[c] + w.x, acc[c + 1] + w.y, acc[c + 2] + w.z, acc[c + 3] + w.w));
                        }
                    } else {
#pragma unroll
                        for (int c = mine * share; c < (mine + 1) * share; c += 4) {
                            float4 v = *reinterpret_cast<const float4 *>(from + c);
#pragma unroll
                            for (int b = 1; b < nb; ++b) {
                                const float4 w = *reinterpret_cast<const float4 *>(from + b * cap * F::kPitch + c);
                                v = make_float4(v.x + w.x, v.y + w.y, v.z + w.z, v.w + w.w);
                            }
                            put(c, v);
                        }
                    }
                    if (!finite(odd)) fx.again = 1;
                }
                if (!ok) break;
            }
            if (part >= 0 && half == 0 && row < sg.rows) ws.ml[at] = make_float2(m, l);
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(fx.seg_done[seg & 1]));
            done();
        }
        // whole pairs' outputs that are not finite, when nobody waits for these warps any more
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (ok && *reinterpret_cast<volatile int *>(&fx.again)) {
            Cut cut = fx.cut;
            Request rq = request_of(a, cut.s);
            Segment x{};
            int behind;
            while (next_segment(a, ly.q_rows, cut, rq, x, behind)) {
                if (x.part >= 0) continue;
                for (int y = warp - kSumWarp; y < x.rows; y += 8)
                    fix_row<T, C, D>(a, x.s, x.ctx, x.L, x.first, x.kvh, (x.r0 + y) / G, (x.r0 + y) % G, lane);
            }
        }
    } else {
        regs_less<kRestRegs>();
        // ---- values of tiles that hold drafted tokens or end the context: rows past
        // the end are zeroed; of the drafted ones, which some rows do not see,
        // what is not finite would reach every row through 0 * v: it is taken out
        // here and added to the rows that see it by the summing warps.  Before
        // them, the ancestors ----
        const Segment *g;
        int fixes = 0;
        Turn vt;
        while (ok && next(g)) {
            const int nt = g->nt, tile0 = g->tile0, ctx = g->ctx, L = g->L;
            if (seg > 1 && !(ok = warp_wait(bar(fx.seg_done[seg & 1]), ((seg >> 1) - 1) & 1))) break;
            if ((tile0 + nt) * kTile > ctx) stage_ancestors(a, *g, anc_s + (seg & 1) * a.max_nodes * ly.words, ly.words, lane);
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(fx.anc_full[seg & 1]));
            for (int k = 0; k < nt; ++k, ++i, vt.step(ly.nv)) {
                const int t0 = (tile0 + k) * kTile;
                if (t0 + kTile <= ctx) continue;
                if (!(ok = warp_wait(bar(fx.fix_ask), fixes++ & 1))) break;
                if (!(ok = warp_wait(bar(fx.v_full[vt.slot]), vt.parity))) break;
#pragma unroll 1
                for (int w = 0; w < 4; ++w) {
                    const int j = w * 32 + lane, t = t0 + j;
                    unsigned char *vr = v_s + vt.slot * F::kSlot + j * 128;
                    auto piece = [&](int ch) {
                        return reinterpret_cast<uint4 *>(vr + (ch >> 3) * (kTile * 128) + (((ch & 7) ^ (j & 7)) << 4));
                    };
                    bool bad = false;
                    // (short code rather than fast: its first run waits for each line of it)
                    if (t0 + w * 32 + 31 >= ctx) {
#pragma unroll 1
                        for (int ch = 0; ch < D / 8; ++ch) {
                            const uint4 v = *piece(ch);
                            if (t >= L) {
                                *piece(ch) = make_uint4(0, 0, 0, 0);
                            } else if (t >= ctx && !(finite2<C>(v.x) & finite2<C>(v.y) & finite2<C>(v.z) & finite2<C>(v.w))) {
                                bad = true;
                                *piece(ch) = make_uint4(held2<C>(v.x), held2<C>(v.y), held2<C>(v.z), held2<C>(v.w));
                            }
                        }
                    }
                    const uint32_t x = __ballot_sync(~0u, bad);
                    if (lane == 0) fx.bad[i & 7][w] = x;
                }
                fence_async_smem();
                mbar_arrive(bar(fx.fix_done));
            }
            if (ok) done();
        }
    }
    __syncwarp();
    tc::tc_fence_before();
    __syncthreads();
    if (warp == kScoreWarp) tc::tmem_dealloc(tmem, kTmCols);
}

// Joins the parts of the pairs that more than one CTA worked on: weights
// 2^(m_part - max m).  grid (CTAs, rows / 16): block (c, y) has the pair whose
// first part is CTA c's last segment; 16 lanes a row, and four parts' reads on
// their way at a time (latency is all that counts here).
constexpr int kJoinRows = 16;
template <typename T, typename C, int D>
__global__ void __launch_bounds__(16 * kJoinRows) tree_join_kernel(const __grid_constant__ TreeArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    const Workspace ws = workspace_of(a.workspace, D);
    const int col = threadIdx.x & 15, row = blockIdx.y * kJoinRows + (threadIdx.x >> 4), c0 = blockIdx.x;
    const Part p = ws.part[c0];
    if ((row & ~1) >= p.rows) return;           // (whole warps, of two rows)
    const bool in = row < p.rows;
    constexpr int E = D / 16, U = 4;
    float acc[E], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.0f;
#pragma unroll 1
    for (int k = 0; in && k <= p.behind; k += U) {
        float2 st[U];
        float4 v[U][E / 4];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            st[u] = make_float2(-INFINITY, 0.0f);
#pragma unroll
            for (int e = 0; e < E / 4; ++e) v[u][e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (k + u > p.behind) continue;
            const size_t at = ((size_t)(c0 + k + u) * 2 + (k + u == 0)) * kRows + row;
            st[u] = ws.ml[at];
#pragma unroll
            for (int e = 0; e < E / 4; ++e) v[u][e] = *reinterpret_cast<const float4 *>(ws.acc + at * D + e * 64 + col * 4);
        }
        float up = m;
#pragma unroll
        for (int u = 0; u < U; ++u) up = fmaxf(up, st[u].x);
        const float f = weight(m, up);
        m = up;
        l *= f;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] *= f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float w = weight(st[u].x, m);
            l = fmaf(st[u].y, w, l);
#pragma unroll
            for (int e = 0; e < E / 4; ++e) {
                acc[4 * e] = fmaf(v[u][e].x, w, acc[4 * e]);
                acc[4 * e + 1] = fmaf(v[u][e].y, w, acc[4 * e + 1]);
                acc[4 * e + 2] = fmaf(v[u][e].z, w, acc[4 * e + 2]);
                acc[4 * e + 3] = fmaf(v[u][e].w, w, acc[4 * e + 3]);
            }
        }
    }
    const int G = a.NH / a.NKV, node = (p.r0 + row) / G, h = p.r0 + row - node * G;
    T *o = reinterpret_cast<T *>(a.out) + ((long)(p.first + node) * a.NH + p.kvh * G + h) * D + col * 4;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    float odd = l;              // a sum of all, not finite where a part of it is not
#pragma unroll
    for (int e = 0; e < E; ++e) odd += acc[e];
#pragma unroll
    for (int e = 0; e < E / 4; ++e)
        if (in) store4(o + e * 64, make_float4(acc[4 * e], acc[4 * e + 1], acc[4 * e + 2], acc[4 * e + 3]), l == 0.0f, inv);
    uint32_t again = __ballot_sync(~0u, in && !finite(odd));
    if (again) {
        __syncwarp();
        const Request rq = request_of(a, p.s);
        for (int u = 0; u < 2; ++u, again >>= 16)
            if (again & 0xffffu) {
                const int y = p.r0 + (row & ~1) + u;
                fix_row<T, C, D>(a, p.s, rq.ctx, rq.L, p.first, p.kvh, y / G, y % G, threadIdx.x & 31);
            }
    }
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

// The queries as [rows][heads][values]; a box is 128 bytes of each head of a key
// head's group, of as many rows as a tile takes.
bool map_queries(CUtensorMap *m, const TreeArgs &a, size_t bytes, int q_rows) {
    const EncodeTiled enc = encode_fn();
    if (!enc) return false;
    const int G = a.NH / a.NKV;
    cuuint64_t dims[3] = {(cuuint64_t)a.D, (cuuint64_t)a.NH, (cuuint64_t)a.T};
    // (of one row, the distance to the next is never used, but has to be one)
    const cuuint64_t row = (cuuint64_t)(a.T > 1 ? a.q_stride : (long)a.NH * a.D) * bytes;
    cuuint64_t strides[2] = {(cuuint64_t)a.D * bytes, row};
    cuuint32_t bx[3] = {(cuuint32_t)(128 / bytes), (cuuint32_t)G, (cuuint32_t)(q_rows / G)};
    cuuint32_t es[3] = {1, 1, 1};
    const CUtensorMapDataType t = bytes == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                  : a.dtype == QVL_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    return enc(m, t, 3, const_cast<void *>(a.q), dims, strides, bx, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D, int CAP>
Layout layout_for(const TreeArgs &a) {
    using F = Conf<T, D, CAP>;
    Layout ly{};
    ly.words = (a.max_nodes + 31) / 32;
    ly.box_log2 = 4;
    while ((1 << ly.box_log2) < kTile && a.P % (2 << ly.box_log2) == 0) ++ly.box_log2;
    ly.box = 1 << ly.box_log2;
    ly.all = (1u << ((kTile >> ly.box_log2) * (D / 64))) - 1u;
    const int G = a.NH / a.NKV;
    ly.q_rows = CAP / G * G;
    ly.anc_bytes = (2 * a.max_nodes * ly.words * 4 + 15) & ~15;
    // (3 + 3 slots where there is room measure as 2 + 2 do)
    const int rest = (((int)sizeof(Fixed) + 1023) & ~1023) + ly.anc_bytes + F::kBlocks + F::kQBoxes * F::kQBox;
    const int slots = std::min(2 * F::kMaxRing, (227 * 1024 - rest) / F::kSlot);
    ly.nk = slots / 2;
    ly.nv = slots - ly.nk;
    ly.smem = rest + slots * F::kSlot;
    return ly;
}

template <typename T, typename C, int D, int CAP>
cudaError_t launch_cap(const TreeArgs &a, cudaStream_t st) {
    const Layout ly = layout_for<T, D, CAP>(a);
    CUtensorMap mk, mv, mq;
    const uint64_t rows = (uint64_t)a.num_pages * a.NKV * a.P;
    const bool bf = a.kv_dtype == QVL_DTYPE_BF16;
    if (!map_cache(&mk, a.k_pages, rows, D, ly.box, bf) || !map_cache(&mv, a.v_pages, rows, D, ly.box, bf) ||
        !map_queries(&mq, a, sizeof(T), ly.q_rows))
        return cudaErrorInvalidValue;
    // no more CTAs than there can be units
    const long qrows = (long)a.max_nodes * (a.NH / a.NKV);
    const long units = (long)a.S * a.NKV * ((qrows + ly.q_rows - 1) / ly.q_rows) * (((long)a.max_ctx + kTile - 1) / kTile);
    const int ctas = (int)(units < kSMs ? units : kSMs);
    auto kern = tree_tc_kernel<T, C, D, CAP>;
    static std::atomic<uint64_t> allowed{0};       // devices on which the kernel may use all shared memory
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !((allowed.load(std::memory_order_relaxed) >> dev) & 1)) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
        if (e != cudaSuccess) return e;
        if (dev < 64) allowed.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = ly.smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, kern, mk, mv, mq, a, ly);
    if (e != cudaSuccess || ctas == 1) return e;
    cfg.gridDim = dim3(ctas, (unsigned)((std::min(qrows, (long)kRows) + kJoinRows - 1) / kJoinRows));
    cfg.blockDim = dim3(16 * kJoinRows);
    cfg.dynamicSmemBytes = 0;
    return cudaLaunchKernelEx(&cfg, tree_join_kernel<T, C, D>, a);
}
// Rows of a request that has max_nodes: up to 32 or 64 go in blocks.
template <typename T, typename C, int D>
cudaError_t launch_d(const TreeArgs &a, cudaStream_t st) {
    const int rows = a.max_nodes * (a.NH / a.NKV);
    return rows <= 32 ? launch_cap<T, C, D, 32>(a, st) : rows <= 64 ? launch_cap<T, C, D, 64>(a, st) : launch_cap<T, C, D, 128>(a, st);
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

size_t tree_workspace_bytes(int D) { return (part_bytes(D) + 255) & ~(size_t)255; }

cudaError_t launch_tree_attention(const TreeArgs &a, cudaStream_t st) {
    if (a.kv_dtype == QVL_DTYPE_BF16) return launch_t<__nv_bfloat16, __nv_bfloat16>(a, st);
    if (a.dtype == QVL_DTYPE_FP16) return launch_t<__half, __half>(a, st);
    return launch_t<float, __half>(a, st);
}

}  // namespace qvl
