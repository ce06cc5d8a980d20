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
#include "serving.cuh"

namespace qvl {
namespace {
constexpr int kThreads = 1024;

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

struct Len {
    int oldl, newl, have, need;
};
__device__ __forceinline__ Len length_of(const PlanArgs &a, int s) {
    Len l;
    l.oldl = max(a.old_len[s], 0);
    l.newl = max(a.new_len[s], 0);
    l.have = min((int)(((long)l.oldl + a.P - 1) / a.P), a.maxp);
    l.need = min((int)(((long)l.newl + a.P - 1) / a.P), a.maxp);
    return l;
}
}  // namespace

__global__ void __launch_bounds__(kThreads) plan_pages_kernel(PlanArgs a) {
    extern __shared__ int sm[];
    int *tok0 = sm, *take0 = sm + (a.S + 1), *give0 = sm + 2 * (a.S + 1);
    __shared__ Sums wsum[32];
    __shared__ int lost;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (a.S + kThreads - 1) / kThreads;
    const int s0 = min(tid * per, a.S), s1 = min(s0 + per, a.S);

    // exclusive prefix sums over the requests
    Sums mine{0, 0, 0};
    for (int s = s0; s < s1; ++s) {
        const Len l = length_of(a, s);
        mine = add(mine, {max(l.newl - l.oldl, 0), max(l.need - l.have, 0), max(l.have - l.need, 0)});
    }
    Sums inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        Sums up{__shfl_up_sync(~0u, inc.tok, o), __shfl_up_sync(~0u, inc.take, o), __shfl_up_sync(~0u, inc.give, o)};
        if (lane >= o) inc = add(inc, up);
    }
    if (lane == 31) wsum[warp] = inc;
    if (tid == 0) lost = 0;
    __syncthreads();
    if (warp == 0) {
        Sums w = wsum[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            Sums up{__shfl_up_sync(~0u, w.tok, o), __shfl_up_sync(~0u, w.take, o), __shfl_up_sync(~0u, w.give, o)};
            if (lane >= o) w = add(w, up);
        }
        wsum[lane] = w;
    }
    __syncthreads();
    Sums run{inc.tok - mine.tok, inc.take - mine.take, inc.give - mine.give};
    if (warp > 0) run = add(run, wsum[warp - 1]);
    for (int s = s0; s < s1; ++s) {
        const Len l = length_of(a, s);
        tok0[s] = run.tok;
        take0[s] = run.take;
        give0[s] = run.give;
        run = add(run, {max(l.newl - l.oldl, 0), max(l.need - l.have, 0), max(l.have - l.need, 0)});
    }
    const Sums tot = wsum[31];
    if (tid == 0) {
        tok0[a.S] = tot.tok;
        take0[a.S] = tot.take;
        give0[a.S] = tot.give;
    }
    __syncthreads();

    const int fc = min(max(a.free_count[0], 0), a.capacity);
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

    const int gt = blockIdx.x * kThreads + tid, gn = gridDim.x * kThreads;
    for (int t = gt; t < a.max_tokens; t += gn) {
        int s = -1, pos = -1, slot = -1;
        if (t < tot.tok) {
            s = find(tok0, a.S, t);
            const Len l = length_of(a, s);
            pos = l.oldl + (t - tok0[s]);
            const int c = pos / a.P;
            if (c < a.maxp) {
                const int page = c < l.have ? a.table[(size_t)s * a.maxp + c] : wanted(take0[s] + (c - l.have));
                if (page >= 0) slot = page * a.P + (pos - c * a.P);
            }
        }
        a.seq_ids[t] = s;
        a.positions[t] = pos;
        a.slots[t] = slot;
    }
    for (int x = gt; x < tot.take; x += gn) {
        const int s = find(take0, a.S, x);
        a.table[(size_t)s * a.maxp + length_of(a, s).have + (x - take0[s])] = wanted(x);
    }
    for (int i = fc + gt; i < min(left, a.capacity); i += gn) a.free_pages[i] = released(i - fc);
    if (blockIdx.x == 0) {
        for (int s = tid; s <= a.S; s += kThreads) a.starts[s] = tok0[s];
        // tokens that no page was left for: past the pool, or past the table's width
        int none = 0;
        for (int s = s0; s < s1; ++s) {
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

cudaError_t launch_plan_pages(const PlanArgs &a, cudaStream_t st) {
    const size_t smem = (size_t)3 * (a.S + 1) * sizeof(int);
    if (smem > 40 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(plan_pages_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
    }
    const int want = (a.max_tokens + kThreads - 1) / kThreads;
    plan_pages_kernel<<<want < 1 ? 1 : want > 148 ? 148 : want, kThreads, smem, st>>>(a);
    return cudaGetLastError();
}

}  // namespace qvl
