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
#include "paged_math.cuh"

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

__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const __grid_constant__ PagedArgs A) {
    __shared__ int sums[32], s_off[kPlanThreads];  // (item_off of the first segments)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const bool prefix = blockIdx.x == PLAN_PREFIX;
    const PagedPlan& P = A.plan[blockIdx.x];
    if (!P.used || P.inlined) return;
    const int n_seg = prefix ? A.n_groups : A.n_seq, tid = threadIdx.x;
    int carry = 0, total, bad = 0;
    for (int base = 0; base < n_seg; base += kPlanThreads) {
        const int i = base + tid;
        int n = 0;
        if (i < n_seg) {
            const PagedSeg g = paged_segment(A, prefix, i);
            n = (g.t1 - g.t0 + P.tpt - 1) / P.tpt;
            bad |= !prefix && (length_too_long(A, i) || left_out(A, P, g.t1 - g.t0));
        }
        const int at = carry + block_scan(n, &total, sums);
        if (i < n_seg) P.item_off[i] = at;
        if (base == 0) s_off[tid] = at;
        carry += total;
    }
    const int n_items = min(carry, P.max_items);
    bad = __syncthreads_or(bad);
    if (tid == 0) {
        P.bad[P.lanes * P.heads] = bad ? PG_BAD_LENGTH : 0;
        P.item_off[n_seg] = n_items;
        *P.n_items = n_items;
    }
    __syncthreads();
    const int* off = n_seg <= kPlanThreads ? s_off : P.item_off;
    auto segment_of = [&](int i) {  // the last segment with item_off <= i
        int lo = 0, hi = n_seg;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (off[mid] <= i) lo = mid;
            else hi = mid;
        }
        return lo;
    };
    if (prefix) {  // a group's row tile has many sequences: a warp each
        for (int i = tid / 32; i < n_items; i += kPlanThreads / 32) {
            const int seg = segment_of(i);
            const PagedItem it = make_item<true>(A, P, true, seg, i - off[seg]);
            if (tid % 32 == 0) P.items[i] = it;
        }
        __syncthreads();
    }
    carry = 0;
    for (int base = 0; base < n_items; base += kPlanThreads) {
        const int i = base + tid;
        int units = 0;
        if (i < n_items) {
            PagedItem it;
            if (prefix) {
                it = P.items[i];
            } else {
                const int seg = segment_of(i);
                it = make_item(A, P, false, seg, i - off[seg]);
            }
            units = item_units(P, it);
            if (!prefix) P.items[i] = it;
        }
        const int at = carry + block_scan(units, &total, sums);
        if (i < n_items) P.cum[i] = at;
        carry += total;
    }
    if (tid == 0) P.cum[n_items] = carry;
    if (P.redo)
        for (int i = tid; i < n_items * P.heads; i += kPlanThreads) P.redo[i] = 0;
}

}  // namespace

cudaError_t launch_paged_plan(const PagedArgs& A, cudaStream_t s) {
    return launch_pdl(plan_kernel, dim3(PLANS), dim3(kPlanThreads), 0, s, A);
}

}  // namespace wb
