// paged_tma.cuh -- bounded mbarrier waits and the TMA loads of pages, shared by the paged
// attention kernels.
#pragma once

#include <cuda.h>

#include <mutex>

#include "paged.h"
#include "paged_math.cuh"

namespace wb {
namespace {

constexpr unsigned long long kDrainNs = 2000000000ull;
// How long a wait may take, and whether one of the CTA has run out.
struct Waits {
    unsigned long long limit;  // ns
    volatile int out;
};
constexpr unsigned kAll = 0xffffffffu;

__device__ __forceinline__ uint64_t now_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
__device__ __forceinline__ void bar_init(uint64_t* b, uint32_t n) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(b)), "r"(n) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t* b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(b)) : "memory");
}
__device__ __forceinline__ void bar_expect(uint64_t* b, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(b)),
                 "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ bool bar_try(uint64_t* b, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_addr(b)), "r"(parity)
        : "memory");
    return ok != 0;
}
// Bounded wait; false when it ran out here or in another role.
__device__ __forceinline__ bool bar_wait(uint64_t* b, uint32_t parity, Waits* w) {
    if (bar_try(b, parity)) return true;
    uint64_t t0 = 0;
    for (uint32_t it = 0;; ++it) {
        if (bar_try(b, parity)) return true;
        if ((it & 63) == 3) {
            if (w->out) return false;
            const uint64_t t = now_ns();
            if (t0 == 0) t0 = t;
            if (t - t0 >= w->limit) {
                w->out = 1;
                return false;
            }
        }
    }
}
__device__ __forceinline__ bool bar_wait_warp(uint64_t* b, uint32_t parity, Waits* w) {
    return __all_sync(kAll, bar_wait(b, parity, w));
}
// For a copy or a product that has been issued and will arrive.
__device__ __forceinline__ void bar_drain(uint64_t* b, uint32_t parity) {
    const uint64_t t0 = now_ns();
    while (!bar_try(b, parity))
        if (now_ns() - t0 > kDrainNs) return;
}

__device__ __forceinline__ void tma4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2,
                                      int c3, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3),
        "r"(smem_addr(bar))
        : "memory");
}

__device__ __forceinline__ void tma3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2,
                                      uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(smem_addr(bar))
        : "memory");
}

struct KvMaps {
    CUtensorMap k, v;  // (dim, kv head, position in page, page), boxes of 64 dims
};

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                             const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                             const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encoder() {
    static EncodeFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault,
                                             &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeFn>(p);
    });
    return fn;
}

bool encode(CUtensorMap* map, const void* addr, const PagedArgs& A, bool bf16, int rows) {
    EncodeFn fn = encoder();
    if (!fn) return false;
    const cuuint64_t dims[4] = {(cuuint64_t)A.hd, (cuuint64_t)A.nkv, (cuuint64_t)A.page_size,
                                (cuuint64_t)A.n_pages};
    const cuuint64_t strides[3] = {(cuuint64_t)A.hd * 2, (cuuint64_t)A.nkv * A.hd * 2,
                                   (cuuint64_t)A.page_stride * 2};
    const cuuint32_t box[4] = {64, 1, (cuuint32_t)rows, 1}, one[4] = {1, 1, 1, 1};
    return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
              const_cast<void*>(addr), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// 16-bit rows of q, (dim, head, token), boxes of 64 dims, `heads` heads and `tokens` tokens.
bool encode_rows(CUtensorMap* map, const PagedArgs& A, bool bf16, int heads, int tokens) {
    EncodeFn fn = encoder();
    if (!fn) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)A.hd, (cuuint64_t)A.nh, (cuuint64_t)A.n_tokens};
    const cuuint64_t strides[2] = {(cuuint64_t)A.hd * 2, (cuuint64_t)A.q_stride * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)heads, (cuuint32_t)tokens}, one[3] = {1, 1, 1};
    return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
              const_cast<void*>(A.q), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Both maps for boxes of at most `most` positions; the positions of a box (they lie in one page),
// 0 on failure.
int kv_maps(KvMaps* m, const PagedArgs& A, bool bf16, int most) {
    int rows = most;
    while (A.page_size % rows) rows /= 2;
    return encode(&m->k, A.k, A, bf16, rows) && encode(&m->v, A.v, A, bf16, rows) ? rows : 0;
}

// Page and row in it of box `rb` (box_rows positions) of the KV tile that starts at position j0;
// a box that no row sees, or without a page, lies outside the pool: TMA fills it with zeros.
__device__ __forceinline__ int2 box_place(const PagedArgs& A, const PagedItem& it, int j0, int rb,
                                          int box_rows, int* bad) {
    const int any_hi = min(it.kv_hi, it.pmax + 1);
    const int any_lo = A.window > 0 ? it.pmin - A.window + 1 : INT_MIN;
    const int sinks = A.window > 0 ? A.sinks : 0;
    const int j = j0 + rb * box_rows, je = j + box_rows;
    if (j < any_hi && je > it.kv_lo && (je > any_lo || j < sinks)) {
        const int p = A.page_shift >= 0 ? j >> A.page_shift : j / A.page_size;
        const int page = __ldg(A.table + (size_t)it.seq * A.table_stride + p);
        if ((unsigned)page < (unsigned)A.n_pages) return make_int2(page, j - p * A.page_size);
        atomicOr(bad, PG_BAD_PAGE);
    }
    return make_int2(A.n_pages, 0);
}

}  // namespace
}  // namespace wb
