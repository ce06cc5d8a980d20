// Page tables and slot maps from request lengths, on the GPU.
//
// With have_s = ceil(old_s / P) and need_s = ceil(new_s / P) pages of request
// s (at most maxp each):
//   released pages (need < have) go onto the free stack in request order,
//   lowest page first: released page r gets stack entry fc + r;
//   wanted pages (need > have) are taken off its top in the same order:
//   wanted page a is stack entry fc + R - 1 - a, R pages released in all.
// So a wanted page is either a free page or one released by the same step.
//   the new tokens old_s <= pos < new_s, packed in request order, get
//   slot = table[s, pos / P] * P + pos % P.
//
// Only three prefix sums over the requests connect the requests with one
// another.  Every CTA forms them for itself in shared memory (S words from
// L2), and a page's stack entry then follows from its index alone: nothing
// that one CTA writes is read by another, so that the whole plan is one
// launch without a grid barrier.  What is written: table columns at or past a
// growing request's have_s, stack entries at or past fc; what is read: columns
// before have_s and entries before fc.
//
// Bound by latency: the launch, two dependent reads (lengths, then table or stack)
// and the sums between.  So tokens, pages and totals are taken by
// CTAs of their own beside one another, and a warp looks up the requests of its
// stretch of tokens at once.  Measured: 64 requests, 2048 tokens 4.3 us (an empty
// kernel 1.0); 2048 requests, half a million tokens 10.6 us (14 with the three jobs one after
// another in every CTA and a search per token; 16 with two and three CTAs on an SM, the
// sums formed in each).
#include <algorithm>
#include <atomic>
#include "serving.cuh"

namespace qvl {
namespace {
constexpr int kThreads = 1024, kWarps = kThreads / 32;

struct Sums {
    int tok, take, give;
};

__device__ __forceinline__ Sums add(const Sums &a, const Sums &b) {
    return {a.tok + b.tok, a.take + b.take, a.give + b.give};
}

// Last index s with p[s] <= x, of a non-decreasing p[0..n] with p[0] <= x < p[n].
__device__ __forceinline__ int find(const int *p, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (p[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// The same for x in the warp's lower half and y in its upper one, by the warp together: each
// half looks at 16 places a round.
__device__ __forceinline__ int2 find_two(const int *p, int n, int x, int y) {
    const int lane = threadIdx.x & 31, mine = lane < 16 ? x : y;
    int lo = 0, len = n;
    for (int step = n; step > 1;) {
        step = (step + 15) / 16;
        const int at = lo + (lane & 15) * step;
        const unsigned hit = __ballot_sync(~0u, (lane & 15) * step < len && p[min(at, n - 1)] <= mine);
        const int k = __popc(lane < 16 ? hit & 0xffff : hit >> 16) - 1;
        lo += k * step;
        len = min(step, len - k * step);
    }
    return make_int2(__shfl_sync(~0u, lo, 0), __shfl_sync(~0u, lo, 16));
}

// x / P: with M = floor(2^64 / P) + 1, x M / 2^64 passes x / P by less than 1 / P for
// every x and P below 2^32
__device__ __forceinline__ unsigned pages_of(const PlanArgs &a, unsigned x) {
    return a.P == 1 ? x : (unsigned)__umul64hi(x, a.inv_p);
}

struct Len {
    int oldl, newl, have, need;
};
__device__ __forceinline__ Len length_of(const PlanArgs &a, int s) {
    Len l;
    l.oldl = max(a.old_len[s], 0);
    l.newl = max(a.new_len[s], 0);
    const unsigned up = (unsigned)a.P - 1;          // sums of less than 2^32
    l.have = (int)min(pages_of(a, (unsigned)l.oldl + up), (unsigned)a.maxp);
    l.need = (int)min(pages_of(a, (unsigned)l.newl + up), (unsigned)a.maxp);
    return l;
}
}  // namespace

__global__ void __launch_bounds__(kThreads) plan_pages_kernel(PlanArgs a) {
    extern __shared__ int sm[];
    int *tok0 = sm, *take0 = sm + (a.S + 1), *give0 = sm + 2 * (a.S + 1);
    __shared__ Sums wsum[kWarps];
    __shared__ int lost;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_launch_dependents();
    pdl_wait();
    const int free_count = a.free_count[0];
    const int rows = (a.S + kThreads - 1) / kThreads;       // of 32 requests, for each warp
    const int first = warp * rows * 32 + lane;

    // exclusive prefix sums over the requests
    auto up = [&](const Sums &v) {
        Sums inc = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            Sums x{__shfl_up_sync(~0u, inc.tok, o), __shfl_up_sync(~0u, inc.take, o), __shfl_up_sync(~0u, inc.give, o)};
            if (lane >= o) inc = add(inc, x);
        }
        return inc;
    };
    Sums run{0, 0, 0};
    for (int r = 0, s = first; r < rows && s - lane < a.S; ++r, s += 32) {
        Sums own{0, 0, 0};
        if (s < a.S) {
            const Len l = length_of(a, s);
            own = {max(l.newl - l.oldl, 0), max(l.need - l.have, 0), max(l.have - l.need, 0)};
        }
        const Sums inc = up(own);
        if (s < a.S) {
            tok0[s] = run.tok + inc.tok - own.tok;
            take0[s] = run.take + inc.take - own.take;
            give0[s] = run.give + inc.give - own.give;
        }
        run = add(run, {__shfl_sync(~0u, inc.tok, 31), __shfl_sync(~0u, inc.take, 31), __shfl_sync(~0u, inc.give, 31)});
    }
    if (lane == 0) wsum[warp] = run;
    if (tid == 0) lost = 0;
    __syncthreads();
    const Sums all = up(wsum[lane]);                        // by every warp for itself
    auto of_lane = [&](int l) {
        return Sums{__shfl_sync(~0u, all.tok, l), __shfl_sync(~0u, all.take, l), __shfl_sync(~0u, all.give, l)};
    };
    const Sums tot = of_lane(31);
    if (warp > 0) {
        const Sums before = of_lane(warp - 1);
        for (int r = 0, s = first; r < rows && s < a.S; ++r, s += 32) {
            tok0[s] += before.tok;
            take0[s] += before.take;
            give0[s] += before.give;
        }
    }
    if (tid == 0) {
        tok0[a.S] = tot.tok;
        take0[a.S] = tot.take;
        give0[a.S] = tot.give;
    }
    __syncthreads();

    const int fc = min(max(free_count, 0), a.capacity);
    const int avail = fc + tot.give;                    // wanted pages 0..avail-1 are there
    const int left = max(avail - tot.take, 0);

    auto released = [&](int r) {
        const int s = find(give0, a.S, r);
        return a.table[(size_t)s * a.maxp + length_of(a, s).need + (r - give0[s])];
    };
    auto wanted = [&](int x) {
        const int i = avail - 1 - x;
        return i < 0 ? -1 : i < fc ? a.free_pages[i] : released(i - fc);
    };

    // CTA 0: totals; the next a.page_ctas: tables and stack; the rest: tokens
    const int role = blockIdx.x == 0 ? 0 : (int)blockIdx.x <= a.page_ctas ? 1 : 2;
    const int gt = ((int)blockIdx.x - (role == 2 ? 1 + a.page_ctas : 1)) * kThreads + tid;
    const int gn = (role == 2 ? (int)gridDim.x - 1 - a.page_ctas : a.page_ctas) * kThreads;
    if (role == 2) {
        // a warp takes a stretch of tokens
        const int span = ((a.max_tokens + (gn >> 5) - 1) / (gn >> 5) + 31) / 32 * 32;
        const int t0 = (gt >> 5) * span, end = min(t0 + span, a.max_tokens);
        if (t0 < end) {
            // the requests of its first and last token; the others' lie between
            const int t1 = min(end, tot.tok) - 1;
            const int2 ab = t0 <= t1 ? find_two(tok0, a.S, t0, t1) : make_int2(0, 0);
#pragma unroll 2
            for (int t = t0 + lane; t < end; t += 32) {
                int s = -1, pos = -1, slot = -1;
                if (t < tot.tok) {
                    s = ab.x + find(tok0 + ab.x, ab.y - ab.x + 1, t);
                    const Len l = length_of(a, s);
                    pos = l.oldl + (t - tok0[s]);
                    const int c = (int)pages_of(a, pos);
                    if (c < a.maxp) {
                        const int page = c < l.have ? a.table[(size_t)s * a.maxp + c] : wanted(take0[s] + (c - l.have));
                        if (page >= 0) slot = page * a.P + (pos - c * a.P);
                    }
                }
                a.seq_ids[t] = s;
                a.positions[t] = pos;
                a.slots[t] = slot;
            }
        }
    } else if (role == 1) {
        for (int x = gt; x < tot.take; x += gn) {
            const int s = find(take0, a.S, x);
            a.table[(size_t)s * a.maxp + length_of(a, s).have + (x - take0[s])] = wanted(x);
        }
        for (int i = fc + gt; i < min(left, a.capacity); i += gn) a.free_pages[i] = released(i - fc);
    } else {
        for (int s = tid; s <= a.S; s += kThreads) a.starts[s] = tok0[s];
        // tokens that no page was left for: past the pool, or past the table's width
        int none = 0;
        for (int s = tid; s < a.S; s += kThreads) {
            const Len l = length_of(a, s);
            if (l.newl <= l.oldl) continue;
            const int pages = l.need <= l.have ? l.need : l.have + min(max(avail - take0[s], 0), l.need - l.have);
            const long held = (long)pages * a.P;
            none += (int)max((long)l.newl - max((long)l.oldl, held), 0l);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) none += __shfl_xor_sync(~0u, none, o);
        if (lane == 0 && none) atomicAdd(&lost, none);
        __syncthreads();
        if (tid == 0) {
            a.missing[0] = lost;
            a.free_count_out[0] = left;
        }
    }
}

cudaError_t launch_plan_pages(const PlanArgs &args, cudaStream_t st) {
    PlanArgs a = args;
    const auto smem_of = [](int S) { return (size_t)3 * (S + 1) * sizeof(int); };
    const size_t smem = smem_of(a.S);
    if (smem > 40 * 1024) {
        // what the most requests need, whatever these do: another thread's launch goes by it too
        static std::atomic<uint64_t> allowed{0};        // devices that have it
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        if (dev >= 64 || !((allowed.load(std::memory_order_relaxed) >> dev) & 1)) {
            e = cudaFuncSetAttribute(plan_pages_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_of(kPlanMaxSeqs));
            if (e != cudaSuccess) return e;
            if (dev < 64) allowed.fetch_or(1ull << dev, std::memory_order_relaxed);
        }
    }
    a.inv_p = ~0ull / (unsigned)a.P + ((a.P & (a.P - 1)) == 0) + 1;
    // a CTA an SM; the pages that may change hands are about a request's last one and a page
    // of tokens each
    a.page_ctas = (int)std::min(std::max((a.max_tokens / a.P / 2 + (long)a.S + kThreads - 1) / kThreads, 1l), 32l);
    const int tokens = (int)std::min((a.max_tokens + kThreads - 1l) / kThreads, 147l - a.page_ctas);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1 + a.page_ctas + tokens);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, plan_pages_kernel, a);
}

}  // namespace qvl
