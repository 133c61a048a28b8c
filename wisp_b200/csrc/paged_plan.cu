// paged_plan.cu -- the row tiles of a paged attention call, found on the device: sequence
// lengths stay there, so a step needs no host synchronisation and can be captured once.
//
// One CTA per plan (the sequences' own parts; the shared prefixes).  It counts the row tiles
// of every sequence, then for each row tile the KV tiles that its mask leaves (the window's
// and the sinks'), and keeps running sums of both; the attention kernels cut the line of all
// KV tiles into equal pieces.  A sequence without cached positions keeps one (fully hidden)
// tile, so its rows are written like any others.

#include <algorithm>

#include "internal.h"
#include "paged.h"

namespace wb {
namespace {

constexpr int kPlanThreads = 1024;

// Exclusive scan of v over the block; `total` is the block's sum.
__device__ int block_scan(int v, int* total, int* warp_sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();  // the previous scan's readers are done
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    if (warp == 0) {
        int s = warp_sums[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += y;
        }
        warp_sums[lane] = s;
    }
    __syncthreads();
    *total = warp_sums[31];
    return x - v + (warp ? warp_sums[warp - 1] : 0);
}

struct Seg {
    int t0, t1;  // tokens
    int s0, s1;  // sequences
};

__device__ Seg segment(const PagedArgs& A, bool prefix, int i) {
    Seg g;
    g.s0 = prefix ? min(max(A.groups[i], 0), A.n_seq) : i;
    g.s1 = prefix ? min(max(A.groups[i + 1], g.s0), A.n_seq) : i + 1;
    g.t0 = min(max(A.q_start[g.s0], 0), A.n_tokens);
    g.t1 = min(max(A.q_start[g.s1], g.t0), A.n_tokens);
    if (g.s0 == g.s1) g.t1 = g.t0;
    return g;
}

__device__ int cached(const PagedArgs& A, int s) {
    const long long cap = (long long)A.table_stride * A.page_size;
    int n = max(A.kv_len[s], 0);
    if (n > cap) {
        n = (int)cap;
        if (blockIdx.x == 0) atomicOr(A.status, PG_BAD_LENGTH);
    }
    return n;
}

__global__ void __launch_bounds__(kPlanThreads) plan_kernel(PagedArgs A) {
    __shared__ int sums[32];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const bool prefix = blockIdx.x == 1;
    const PagedPlan& P = A.plan[blockIdx.x];
    const int n_seg = prefix ? A.n_groups : A.n_seq, tid = threadIdx.x;
    if (!prefix && tid == 0) *A.status = 0;  // the sequences' plan alone writes it here
    int carry = 0, total;
    for (int base = 0; base < n_seg; base += kPlanThreads) {
        const int i = base + tid;
        int n = 0;
        if (i < n_seg) {
            const Seg g = segment(A, prefix, i);
            n = (g.t1 - g.t0 + P.tpt - 1) / P.tpt;
        }
        const int at = carry + block_scan(n, &total, sums);
        if (i < n_seg) P.item_off[i] = at;
        carry += total;
    }
    const int n_items = min(carry, P.max_items);
    if (tid == 0) {
        P.item_off[n_seg] = n_items;
        *P.n_items = n_items;
    }
    __syncthreads();
    carry = 0;
    for (int base = 0; base < n_items; base += kPlanThreads) {
        const int i = base + tid;
        int tiles = 0;
        if (i < n_items) {
            int lo = 0, hi = n_seg;  // the last segment with item_off <= i
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (P.item_off[mid] <= i) lo = mid;
                else hi = mid;
            }
            const Seg g = segment(A, prefix, lo);
            PagedItem it;
            it.tok0 = g.t0 + (i - P.item_off[lo]) * P.tpt;
            it.ntok = min(P.tpt, g.t1 - it.tok0);
            it.seq = g.s0;
            it.mixed = prefix && g.s1 - g.s0 > 1;
            int reach;  // the most that any sequence of the segment has cached
            if (!it.mixed) {
                reach = cached(A, g.s0);
                it.pos0 = reach - (g.t1 - it.tok0);
                it.pmin = it.pos0;
                it.pmax = it.pos0 + it.ntok - 1;
            } else {
                it.pos0 = 0;
                it.pmin = 0x7fffffff;
                it.pmax = -0x7fffffff;
                reach = 0;
                int s = g.s0;
                for (int t = it.tok0; t < it.tok0 + it.ntok; ++t) {
                    while (s + 1 < g.s1 && A.q_start[s + 1] <= t) ++s;
                    const int n = cached(A, s), p = n - (A.q_start[s + 1] - t);
                    it.pmin = min(it.pmin, p);
                    it.pmax = max(it.pmax, p);
                    reach = max(reach, n);
                }
            }
            it.kv_lo = 0;
            it.kv_hi = reach;
            if (A.n_groups > 0) {
                int gr = lo;
                if (!prefix) {  // the sequence's group
                    int a = 0, b = A.n_groups;
                    while (b - a > 1) {
                        const int mid = (a + b) >> 1;
                        if (A.groups[mid] <= g.s0) a = mid;
                        else b = mid;
                    }
                    gr = A.groups[a] <= g.s0 && g.s0 < A.groups[a + 1] ? a : -1;
                }
                const int pl = gr >= 0 ? max(A.prefix_len[gr], 0) : 0;
                if (prefix) it.kv_hi = min(reach, pl);
                else it.kv_lo = min(reach, pl);
            }
            const int end = min(it.kv_hi, it.pmax + 1), begin = it.kv_lo;
            int wlo = A.window > 0 ? max(begin, it.pmin - A.window + 1) : begin;
            wlo = max(wlo, 0);
            it.sink0 = it.n_sink = 0;
            it.first = begin / P.tile;
            it.n_tiles = 1;
            if (end > begin) {
                const int last = (end + P.tile - 1) / P.tile;  // exclusive
                int f = min(wlo, end - 1) / P.tile;
                const int send = min(A.window > 0 ? A.sinks : 0, end);
                if (send > begin) {
                    it.sink0 = begin / P.tile;
                    const int se = (send + P.tile - 1) / P.tile;
                    if (se >= f) f = it.sink0;  // they meet: one list
                    else it.n_sink = se - it.sink0;
                }
                it.first = f;
                it.n_tiles = it.n_sink + last - f;
            }
            tiles = it.n_tiles;
            P.items[i] = it;
        }
        const int at = carry + block_scan(tiles, &total, sums);
        if (i < n_items) P.cum[i] = at;
        carry += total;
    }
    if (tid == 0) P.cum[n_items] = carry;
}

}  // namespace

cudaError_t launch_paged_plan(const PagedArgs& A, cudaStream_t s) {
    return launch_pdl(plan_kernel, dim3(A.n_groups > 0 ? 2 : 1), dim3(kPlanThreads), 0, s, A);
}

}  // namespace wb
