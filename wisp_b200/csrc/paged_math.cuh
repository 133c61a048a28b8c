// paged_math.cuh -- device helpers of the paged attention kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <limits.h>
#include <stdint.h>

#include "paged.h"

namespace wb {
namespace {

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t smem_addr(const void* p) {
    return (uint32_t)__cvta_generic_to_shared(p);
}
// 16 bytes global -> shared; zeros when !in (src is not read then, but stays a valid address)
__device__ __forceinline__ void cp16(void* dst, const void* src, bool in) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(dst)), "l"(src),
                 "r"(in ? 16 : 0)
                 : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], const void* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(smem_addr(p))
                 : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], const void* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(smem_addr(p))
                 : "memory");
}

template <typename T>
struct PMath;

template <>
struct PMath<__half> {
    static constexpr float kPShift = 15.f;
    static constexpr uint32_t kExp = 0x7c00, kMan = 0x03ff, kOne = 0x3c00;
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t v) {
        return __half22float2(*reinterpret_cast<const __half2*>(&v));
    }
    static __device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
        hi = pack(a, b);
        const float2 f = unpack(hi);
        lo = pack(a - f.x, b - f.y);
    }
    static __device__ __forceinline__ bool not_finite(uint32_t v) {
        return (v & 0x7c00u) == 0x7c00u || (v & 0x7c000000u) == 0x7c000000u;
    }
    static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                               uint32_t b1) {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
            "{%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};

template <>
struct PMath<__nv_bfloat16> {
    static constexpr float kPShift = 0.f;  // bf16 has fp32's range
    static constexpr uint32_t kExp = 0x7f80, kMan = 0x007f, kOne = 0x3f80;
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t v) {
        return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
    }
    static __device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
        hi = pack(a, b);
        const float2 f = unpack(hi);
        lo = pack(a - f.x, b - f.y);
    }
    static __device__ __forceinline__ bool not_finite(uint32_t v) {
        return (v & 0x7f80u) == 0x7f80u || (v & 0x7f800000u) == 0x7f800000u;
    }
    static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                               uint32_t b1) {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
            "{%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};

// o += (places `one` that are visible) * (infinities and NaNs of the fragment b0, b1), which
// leaves the fragment with zeros in their places: a hidden NaN times a zero weight would reach
// rows that do not see it.  By value: the accumulators stay in registers elsewhere.
struct SpecialFrag {
    float o[4];
    uint32_t b0, b1;
};
template <typename T>
__device__ __noinline__ SpecialFrag specials(SpecialFrag f, uint32_t a0, uint32_t a1, uint32_t a2,
                                             uint32_t a3) {
    using M = PMath<T>;
    uint32_t set[3][2] = {};  // +infinity, -infinity, NaN
    uint32_t b[2] = {f.b0, f.b1};
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const uint32_t h = (b[i] >> (16 * e)) & 0xffffu, one = M::kOne << (16 * e);
            if ((h & M::kExp) != M::kExp) continue;
            if (h & M::kMan) set[2][i] |= one;
            else if (h & 0x8000u) set[1][i] |= one;
            else set[0][i] |= one;
            b[i] &= ~(0xffffu << (16 * e));
        }
    f.b0 = b[0];
    f.b1 = b[1];
    const uint32_t one[4] = {a0, a1, a2, a3};
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        float c[4] = {0.f, 0.f, 0.f, 0.f};
        M::mma(c, one, set[k][0], set[k][1]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (c[i] > 0.f) f.o[i] += k == 0 ? INFINITY : k == 1 ? -INFINITY : NAN;
    }
    return f;
}

// The last i in [0, n) with a[i] <= x (0 when there is none).
__device__ __forceinline__ int last_le(const int* __restrict__ a, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ int cached_positions(const PagedArgs& A, int s) {
    const long long cap = (long long)A.table_stride * A.page_size;
    const int n = max(A.kv_len[s], 0);
    return n > cap ? (int)cap : n;
}

__device__ __forceinline__ int token_position(const PagedArgs& A, int t) {
    const int s = last_le(A.q_start, A.n_seq, t);
    return cached_positions(A, s) - (A.q_start[s + 1] - t);
}

// Element offset of position j's row for kv head h; -1 (and a status bit) where the table
// names no page of the pool.
__device__ __forceinline__ long long page_offset(const PagedArgs& A, int seq, int j, int h) {
    const int p = A.page_shift >= 0 ? j >> A.page_shift : j / A.page_size;
    const int page = __ldg(A.table + (size_t)seq * A.table_stride + p);
    if ((unsigned)page >= (unsigned)A.n_pages) {
        atomicOr(A.status, PG_BAD_PAGE);
        return -1;
    }
    return (long long)page * (long long)A.page_stride +
           ((long long)(j - p * A.page_size) * A.nkv + h) * A.hd;
}

// q rows of a tile into shared memory: row r of MMA tile wr at line wr * 16 + r, 16-byte pieces
// XORed with the line number.  SPLIT: 8 fp32 rows per MMA tile, hi parts in lines 0-7 and lo
// parts in 8-15; fp16 parts are of q / 2^e with 2^e the row's largest exponent (s_fac).
template <typename T, bool SPLIT, int HD, int RW, int THREADS>
__device__ void load_rows(const PagedArgs& A, int tok0, int n_rows, int h0, int gpb, T* qs,
                          float* s_fac) {
    constexpr int kCh = HD / 8;
    if (!SPLIT) {
        const T* q = reinterpret_cast<const T*>(A.q);
        for (int i = threadIdx.x; i < 16 * RW * kCh; i += THREADS) {
            const int r = i / kCh, c = i - r * kCh;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (r < n_rows && c * 8 < A.hd)
                v = __ldg(reinterpret_cast<const uint4*>(
                    q + (size_t)(tok0 + r / gpb) * A.q_stride + (size_t)(h0 + r % gpb) * A.hd + c * 8));
            *reinterpret_cast<uint4*>(qs + (size_t)r * HD + ((c ^ (r & 7)) * 8)) = v;
        }
    } else {
        const float* q = reinterpret_cast<const float*>(A.q);
        const int lane = threadIdx.x & 31;
        for (int i = threadIdx.x >> 5; i < 8 * RW; i += THREADS / 32) {  // real row i
            const int line = (i / 8) * 16 + (i & 7);
            const bool in = i < n_rows;
            const float* src = q + (in ? (size_t)(tok0 + i / gpb) * A.q_stride +
                                             (size_t)(h0 + i % gpb) * A.hd
                                       : 0);
            constexpr int kN = HD / 64;
            float2 v[kN];
            float mx = 0.f;
#pragma unroll
            for (int u = 0; u < kN; ++u) {
                const int d = (u * 32 + lane) * 2;
                v[u] = in && d < A.hd ? __ldg(reinterpret_cast<const float2*>(src + d))
                                      : make_float2(0.f, 0.f);
                mx = fmaxf(mx, fmaxf(fabsf(v[u].x), fabsf(v[u].y)));
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            const uint32_t e = (__float_as_uint(mx) >> 23) & 255u;
            const bool scaled = PMath<T>::kPShift != 0.f && e > 0 && e < 254;
            const float inv = scaled ? __uint_as_float((254u - e) << 23) : 1.f;
            if (lane == 0) s_fac[line] = scaled ? __uint_as_float(e << 23) : 1.f;
#pragma unroll
            for (int u = 0; u < kN; ++u) {
                const int d = (u * 32 + lane) * 2, c = d / 8;
                uint32_t hi, lo;
                PMath<T>::split2(v[u].x * inv, v[u].y * inv, hi, lo);
                const int at = ((c ^ (line & 7)) * 8) + (d & 7);  // line + 8 has the same key
                *reinterpret_cast<uint32_t*>(qs + (size_t)line * HD + at) = hi;
                *reinterpret_cast<uint32_t*>(qs + (size_t)(line + 8) * HD + at) = lo;
            }
        }
    }
}

// log-sum-exp (natural) of a row with running maximum M (log2 units) and sum L, whose
// weights carry the factor 2^shift.
__device__ __forceinline__ float row_lse(float M, float L, float shift) {
    return L == 0.f ? -INFINITY : (M + log2f(L) - shift) * 0.69314718055994531f;
}

__device__ __forceinline__ size_t part_row(const PagedPlan& P, int piece, int head_lane, int slot,
                                           int row) {
    return (((size_t)piece * P.heads + head_lane) * 2 + slot) * P.rows + row;
}

// Where one finished row of a piece goes: the output, or a partial record.
template <typename T, bool SPLIT>
struct RowOut {
    float* o32;   // partial record, or the fp32 output
    T* o16;
    float* ml;    // partial record's maximum and sum
    float* lse;
    bool final;
    __device__ RowOut(const PagedArgs& A, const PagedPlan& P, int which, const PagedItem& it,
                      int piece, int head_lane, int h0, int gpb, int row, int a, bool whole) {
        const size_t t = it.tok0 + row / gpb, h = h0 + row % gpb;
        final = whole && A.n_groups == 0;
        o32 = nullptr;
        o16 = nullptr;
        ml = lse = nullptr;
        if (final) {
            if (SPLIT) o32 = reinterpret_cast<float*>(A.out) + t * A.out_stride + h * A.hd;
            else o16 = reinterpret_cast<T*>(A.out) + t * A.out_stride + h * A.hd;
            if (A.lse) lse = A.lse + t * A.nh + h;
        } else if (whole) {
            const size_t id = (size_t)which * A.n_tokens * A.nh + t * A.nh + h;
            o32 = A.full_o + id * A.hd;
            ml = A.full_ml + id * 2;
        } else {
            const size_t id = part_row(P, piece, head_lane, a > 0 ? 0 : 1, row);
            o32 = P.part_o + id * A.hd;
            ml = P.part_ml + id * 2;
        }
    }
    __device__ __forceinline__ void put2(int d, float2 v, float L) {
        if (final) {
            const float inv = 1.f / L;
            v = L == 0.f ? make_float2(0.f, 0.f) : make_float2(v.x * inv, v.y * inv);
            if (!SPLIT) {
                *reinterpret_cast<uint32_t*>(o16 + d) = PMath<T>::pack(v.x, v.y);
                return;
            }
        }
        *reinterpret_cast<float2*>(o32 + d) = v;
    }
    __device__ __forceinline__ void put_ml(float M, float L) {
        if (final) {
            if (lse) *lse = row_lse(M, L, PMath<T>::kPShift);
        } else {
            *reinterpret_cast<float2*>(ml) = make_float2(M, L);
        }
    }
};

// A warp's join of one row's partial records, in the order of the pieces.
struct Joined {
    float M, L;
    float2 acc[4];  // dims (i * 32 + lane) * 2
    __device__ __forceinline__ void init() {
        M = -INFINITY;
        L = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = make_float2(0.f, 0.f);
    }
    __device__ __forceinline__ void rebase(float m) {
        const float base = m == -INFINITY ? 0.f : m;
        const float e = ex2(M - base);
        M = m;
        L *= e;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            acc[i].x *= e;
            acc[i].y *= e;
        }
    }
    __device__ __forceinline__ void add(const PagedArgs& A, const float* o, float2 ml) {
        const float base = M == -INFINITY ? 0.f : M;
        const float e = ex2(ml.x - base);
        L = fmaf(ml.y, e, L);
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = (i * 32 + lane) * 2;
            if (d >= A.hd) break;
            const float2 v = *reinterpret_cast<const float2*>(o + d);
            acc[i].x = fmaf(v.x, e, acc[i].x);
            acc[i].y = fmaf(v.y, e, acc[i].y);
        }
    }
    __device__ void add_full(const PagedArgs& A, int which, size_t id) {
        id += (size_t)which * A.n_tokens * A.nh;
        const float2 ml = *reinterpret_cast<const float2*>(A.full_ml + id * 2);
        rebase(fmaxf(M, ml.x));
        add(A, A.full_o + id * A.hd, ml);
    }
    __device__ void add_range(const PagedArgs& A, const PagedPlan& P, int first, int last,
                              int head_lane, int row) {
        const int lane = threadIdx.x & 31, total = P.cum[*P.n_items];
        float m = M;
        for (int p = first + lane; p <= last; p += 32)
            if (used(P, p, total))
                m = fmaxf(m, P.part_ml[part_row(P, p, head_lane, p == first, row) * 2]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        rebase(m);
#pragma unroll 4
        for (int p = first; p <= last; ++p) {
            if (!used(P, p, total)) continue;
            const size_t id = part_row(P, p, head_lane, p == first, row);
            add(A, P.part_o + id * A.hd, *reinterpret_cast<const float2*>(P.part_ml + id * 2));
        }
    }
    static __device__ __forceinline__ bool used(const PagedPlan& P, int p, int total) {
        return (long long)p * total / P.lanes < (long long)(p + 1) * total / P.lanes;
    }
    template <typename T, bool SPLIT>
    __device__ void write(const PagedArgs& A, int t, int h) {
        const int lane = threadIdx.x & 31;
        const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = (i * 32 + lane) * 2;
            if (d >= A.hd) break;
            const size_t at = (size_t)t * A.out_stride + (size_t)h * A.hd + d;
            const float2 v = L == 0.f ? make_float2(0.f, 0.f)
                                      : make_float2(acc[i].x * inv, acc[i].y * inv);
            if (SPLIT) *reinterpret_cast<float2*>(reinterpret_cast<float*>(A.out) + at) = v;
            else *reinterpret_cast<uint32_t*>(reinterpret_cast<T*>(A.out) + at) = PMath<T>::pack(v.x, v.y);
        }
        if (lane == 0 && A.lse)
            A.lse[(size_t)t * A.nh + h] = row_lse(M, L, PMath<T>::kPShift);
    }
};

}  // namespace
}  // namespace wb
