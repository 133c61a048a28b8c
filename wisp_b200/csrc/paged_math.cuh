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

template <bool B>
struct Flag {
    static constexpr bool value = B;
};

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
    // a, b in parts: two here (`third` is not written)
    static constexpr int kFrags = 1;
    static __device__ __forceinline__ void split(float a, float b, uint32_t& hi, uint32_t& lo,
                                                 uint32_t&) {
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
    static constexpr int kFrags = 2;
    static __device__ __forceinline__ void split(float a, float b, uint32_t& hi, uint32_t& mid,
                                                 uint32_t& third) {
        hi = pack(a, b);
        const float2 f = unpack(hi);
        mid = pack(a - f.x, b - f.y);
        const float2 g = unpack(mid);
        third = pack(a - f.x - g.x, b - f.y - g.y);
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

// o0, o1 += p V for 16 positions and 16 dims.  The tensor core cuts its sums off (they shrink by
// half a unit of their last place each time: 5e-7 of rows over 2668 positions, 1e-6 over 16000), so
// fp32 rows take the products by themselves and add them rounded.
template <typename T, bool SPLIT, int F>
__device__ __forceinline__ void add_products(float (&o0)[4], float (&o1)[4],
                                             const uint32_t (&p)[F][4], const uint32_t (&v)[4]) {
    float t0[4] = {0.f, 0.f, 0.f, 0.f}, t1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int n = 0; n < F; ++n) {
        PMath<T>::mma(SPLIT ? t0 : o0, p[n], v[0], v[1]);
        PMath<T>::mma(SPLIT ? t1 : o1, p[n], v[2], v[3]);
    }
    if constexpr (SPLIT) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            o0[u] += t0[u];
            o1[u] += t1[u];
        }
    }
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
    const long long cap = (long long)A.table_width * A.page_size;
    const int n = max(A.kv_len[s], 0);
    return n > cap ? (int)cap : n;
}

// Does the sequence claim more positions than its table row holds?
__device__ __forceinline__ bool length_too_long(const PagedArgs& A, int s) {
    return A.kv_len[s] > (long long)A.table_width * A.page_size;
}

// May rows of a sequence with so many tokens be left out (it has more than the call's bound)?  The
// joins of split items take used_rows of each; in prefix mode they go by tokens.
__device__ __forceinline__ bool left_out(const PagedArgs& A, const PagedPlan& P, int tokens) {
    return A.n_groups == 0 && min(tokens, P.tpt) * P.gpb > P.used_rows;
}

struct PagedSeg {
    int t0, t1;  // tokens
    int s0, s1;  // sequences
};
// Sequence i, or group i of sequences.
__device__ __forceinline__ PagedSeg paged_segment(const PagedArgs& A, bool prefix, int i) {
    PagedSeg g;
    g.s0 = prefix ? min(max(A.groups[i], 0), A.n_seq) : i;
    g.s1 = prefix ? min(max(A.groups[i + 1], g.s0), A.n_seq) : i + 1;
    g.t0 = min(max(A.q_start[g.s0], 0), A.n_tokens);
    g.t1 = min(max(A.q_start[g.s1], g.t0), A.n_tokens);
    if (g.s0 == g.s1) g.t1 = g.t0;
    return g;
}

// Row tile `nth` of segment `seg`; WARP: by a whole warp, whose lanes share the sequences.
template <bool WARP = false>
__device__ inline PagedItem make_item(const PagedArgs& A, const PagedPlan& P, bool prefix, int seg,
                                      int nth) {
    const PagedSeg g = paged_segment(A, prefix, seg);
    PagedItem it;
    it.tok0 = g.t0 + nth * P.tpt;
    it.ntok = min(P.tpt, g.t1 - it.tok0);
    it.seq = min(g.s0, A.n_seq - 1);
    it.mixed = prefix && g.s1 - g.s0 > 1;
    int reach;  // the most that any sequence of the segment has cached
    if (!it.mixed) {
        reach = cached_positions(A, it.seq);
        it.pos0 = reach - (g.t1 - it.tok0);
        it.pmin = it.pos0;
        it.pmax = it.pos0 + it.ntok - 1;
    } else {
        it.pos0 = 0;
        it.pmin = 0x7fffffff;
        it.pmax = -0x7fffffff;
        reach = 0;
#pragma unroll 4
        for (int s = g.s0 + (WARP ? (int)(threadIdx.x & 31) : 0); s < g.s1; s += WARP ? 32 : 1) {
            // the tile's tokens of each sequence
            const int end = A.q_start[s + 1], n = cached_positions(A, s);
            const int a = max(A.q_start[s], it.tok0), b = min(end, it.tok0 + it.ntok);
            if (a >= b) continue;
            it.pmin = min(it.pmin, n - (end - a));
            it.pmax = max(it.pmax, n - (end - b) - 1);
            reach = max(reach, n);
        }
        if (WARP) {
            it.pmin = __reduce_min_sync(0xffffffffu, it.pmin);
            it.pmax = __reduce_max_sync(0xffffffffu, it.pmax);
            reach = __reduce_max_sync(0xffffffffu, reach);
        }
    }
    it.kv_lo = 0;
    it.alone = 1;
    it.kv_hi = reach;
    if (A.n_groups > 0) {
        int gr = seg;
        if (!prefix) {  // the sequence's group
            gr = last_le(A.groups, A.n_groups, g.s0);
            if (g.s0 < A.groups[gr] || g.s0 >= A.groups[gr + 1]) gr = -1;
        }
        const int pl = gr >= 0 ? max(A.prefix_len[gr], 0) : 0;
        it.alone = gr < 0;
        if (prefix) it.kv_hi = min(reach, pl);
        else it.kv_lo = min(reach, pl);
        if (it.mixed && A.window == 0 && it.kv_hi <= it.pmin + 1) {
            // every row sees the whole prefix: any positions from pmin on say so (looking each
            // token's up is a search and two loads behind one another)
            it.mixed = 0;
            it.pos0 = it.pmin;
        }
    }
    const int end = min(it.kv_hi, it.pmax + 1), begin = it.kv_lo;
    const int wlo = A.window > 0 ? max(begin, it.pmin - A.window + 1) : begin;
    it.sink0 = it.n_sink = 0;
    it.first = begin / kPagedTile;
    it.n_tiles = 1;
    if (end > begin) {
        const int last = (end + kPagedTile - 1) / kPagedTile;  // exclusive
        int f = min(wlo, end - 1) / kPagedTile;
        const int send = min(A.window > 0 ? A.sinks : 0, end);
        if (send > begin) {
            it.sink0 = begin / kPagedTile;
            const int se = (send + kPagedTile - 1) / kPagedTile;
            if (se >= f) f = it.sink0;  // they meet: one list
            else it.n_sink = se - it.sink0;
        }
        it.first = f;
        it.n_tiles = it.n_sink + last - f;
    }
    if (it.ntok <= 0) it.n_tiles = 0;
    return it;
}

__device__ __forceinline__ int token_position(const PagedArgs& A, int t) {
    const int s = last_le(A.q_start, A.n_seq, t);
    return cached_positions(A, s) - (A.q_start[s + 1] - t);
}

// Element offset of position j's row for kv head h; -1 (and a status bit in shared memory) where
// the table names no page of the pool.
__device__ __forceinline__ long long page_offset(const PagedArgs& A, int seq, int j, int h,
                                                 int* bad) {
    const int p = A.page_shift >= 0 ? j >> A.page_shift : j / A.page_size;
    const int page = __ldg(A.table + (size_t)seq * A.table_stride + p);
    if ((unsigned)page >= (unsigned)A.n_pages) {
        atomicOr(bad, PG_BAD_PAGE);
        return -1;
    }
    return (long long)page * (long long)A.page_stride +
           ((long long)(j - p * A.page_size) * A.nkv + h) * A.hd;
}

// q rows of a tile into shared memory: row r of MMA tile wr at line wr * 16 + r, 16-byte pieces
// XORed with the line number.  SPLIT: 8 fp32 rows per MMA tile, first parts in lines 0-7 and
// second ones in 8-15 (third ones in lines 0-7 of a second set of tiles); fp16 parts are of q / 2^e with 2^e the row's largest exponent (s_fac).
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
                uint32_t hi, lo, third = 0;
                PMath<T>::split(v[u].x * inv, v[u].y * inv, hi, lo, third);
                const int at = ((c ^ (line & 7)) * 8) + (d & 7);  // line + 8 has the same key
                *reinterpret_cast<uint32_t*>(qs + (size_t)line * HD + at) = hi;
                *reinterpret_cast<uint32_t*>(qs + (size_t)(line + 8) * HD + at) = lo;
                if (PMath<T>::kFrags == 2) {
                    T* q2 = qs + (size_t)16 * RW * HD;
                    *reinterpret_cast<uint32_t*>(q2 + (size_t)line * HD + at) = third;
                    *reinterpret_cast<uint32_t*>(q2 + (size_t)(line + 8) * HD + at) = 0;
                }
            }
        }
    }
}

// The same from up to 8 fp32 rows that lie in shared memory ([row][HD]), by a block of 128
// threads: parts into `out` ([fragment][16][HD], swizzled), factors by row.
template <typename T, int HD>
__device__ __forceinline__ void split_rows(const PagedArgs& A, const float* rows, int n_rows, T* out,
                                           float* s_fac) {
    const int lane = threadIdx.x & 31;
    constexpr int kN = HD / 64;
    for (int r = threadIdx.x >> 5; r < 8; r += 4) {
        float2 v[kN];
        float mx = 0.f;
#pragma unroll
        for (int u = 0; u < kN; ++u) {
            v[u] = r < n_rows ? *reinterpret_cast<const float2*>(rows + r * HD + (u * 32 + lane) * 2)
                              : make_float2(0.f, 0.f);
            mx = fmaxf(mx, fmaxf(fabsf(v[u].x), fabsf(v[u].y)));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const uint32_t e = (__float_as_uint(mx) >> 23) & 255u;
        const bool scaled = PMath<T>::kPShift != 0.f && e > 0 && e < 254;
        const float inv = scaled ? __uint_as_float((254u - e) << 23) : 1.f;
        if (lane == 0) s_fac[r] = scaled ? __uint_as_float(e << 23) : 1.f;
#pragma unroll
        for (int u = 0; u < kN; ++u) {
            const int d = (u * 32 + lane) * 2;
            uint32_t p[3] = {0, 0, 0};
            PMath<T>::split(v[u].x * inv, v[u].y * inv, p[0], p[1], p[2]);
            T* to = out + ((((d / 8) ^ (r & 7)) * 8) + (d & 7));  // rows r and r + 8 share the key
            *reinterpret_cast<uint32_t*>(to + r * HD) = p[0];
            *reinterpret_cast<uint32_t*>(to + (r + 8) * HD) = p[1];
            if (PMath<T>::kFrags == 2) {
                *reinterpret_cast<uint32_t*>(to + (16 + r) * HD) = p[2];
                *reinterpret_cast<uint32_t*>(to + (24 + r) * HD) = 0;
            }
        }
    }
}

// log-sum-exp (natural) of a row whose weights 2^(score - M), score in log2 units, sum to L.
__device__ __forceinline__ float row_lse(float M, float L) {
    return L == 0.f ? -INFINITY : (M + log2f(L)) * 0.69314718055994531f;
}

// The status word of the call: the CTAs' and the plans' bits, gathered by the last kernel's
// first CTA.
__device__ __forceinline__ void gather_status(const PagedArgs& A) {
    int bits = 0;
    for (int w = 0; w < PLANS; ++w) {
        const PagedPlan& P = A.plan[w];
        if (!P.used) continue;
        for (int i = threadIdx.x; i <= P.lanes * P.heads; i += blockDim.x) bits |= P.bad[i];
    }
    const int any = __syncthreads_or(bits & PG_BAD_PAGE) ? PG_BAD_PAGE : 0;
    const int len = __syncthreads_or(bits & PG_BAD_LENGTH) ? PG_BAD_LENGTH : 0;
    const int late = __syncthreads_or(bits & PG_TIMEOUT) ? PG_TIMEOUT : 0;
    if (threadIdx.x == 0) {
        *A.status = any | len | late;
        if (A.all_status && (any | len | late)) atomicOr(A.all_status, any | len | late);
    }
}

// A KV tile of the item is 2^item_shift units.
__device__ __forceinline__ int item_shift(const PagedPlan& P, const PagedItem& it) {
    return P.grain > 1 && it.ntok * P.gpb > kPagedHalf;
}
__device__ __forceinline__ int item_units(const PagedPlan& P, const PagedItem& it) {
    return it.n_tiles ? (it.n_tiles << item_shift(P, it)) + P.lead : 0;
}

// The last i in [0, n) with cum[i] <= x (cum[0] <= x), by the whole block.
__device__ __forceinline__ int block_last_le(const int* cum, int n, int x) {
    int lo = 0, span = n;
    while (span > 1) {
        const int step = (span + (int)blockDim.x - 1) / (int)blockDim.x;
        const int at = (int)threadIdx.x * step;
        const int hit = __syncthreads_count(at < span && cum[lo + min(at, span - 1)] <= x) - 1;
        lo += hit * step;
        span = min(step, span - hit * step);
    }
    return lo;
}

// The line of `total` units in pieces: as many as there are lanes, each with a unit at least.
// Piece p starts at unit start(p); unit x lies in piece of(x).
struct Pieces {
    int total, n;
    __device__ Pieces(const PagedPlan& P, int total_) : total(total_) {
        n = min(P.lanes, P.grain > 1 ? max(total_ / P.grain, 1) : total_);
    }
    __device__ __forceinline__ int start(int p) const {
        if (total <= 1 << 20) return (int)((unsigned)p * (unsigned)total / (unsigned)n);
        return (int)((unsigned long long)p * total / n);
    }
    __device__ __forceinline__ int of(int x) const {
        if (total <= 1 << 20)
            return (int)((((unsigned)x + 1) * (unsigned)n - 1) / (unsigned)total);
        return (int)((((unsigned long long)x + 1) * n - 1) / total);
    }
};

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
            const size_t id = (size_t)(which == PLAN_PREFIX) * A.n_tokens * A.nh + t * A.nh + h;
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
            if (lse) *lse = row_lse(M, L);
        } else {
            *reinterpret_cast<float2*>(ml) = make_float2(M, L);
        }
    }
};

// The join of one row's partial records by W warps.
constexpr int kJoinThreads = 256;
template <int VECS>
struct JoinShared {
    float2 acc[8][32 * VECS];
    float m[8], l[8];
};
// A lane holds dims (i * 32 + lane) * 2 and the next for i < VECS: heads of up to 64 VECS dims.
template <int VECS>
struct Joined {
    float M, L;
    float2 acc[VECS];
    __device__ __forceinline__ void init() {
        M = -INFINITY;
        L = 0.f;
#pragma unroll
        for (int i = 0; i < VECS; ++i) acc[i] = make_float2(0.f, 0.f);
    }
    __device__ __forceinline__ void rebase(float m) {
        const float base = m == -INFINITY ? 0.f : m;
        const float e = ex2(M - base);
        M = m;
        L *= e;
#pragma unroll
        for (int i = 0; i < VECS; ++i) {
            acc[i].x *= e;
            acc[i].y *= e;
        }
    }
    // kBatch records whose loads are issued together; `ok` marks those that exist
    template <int N>
    __device__ __forceinline__ void add(const PagedArgs& A, const float* const (&o)[N],
                                        const float* const (&ml)[N], int n) {
        const int lane = threadIdx.x & 31;
        float2 v[N][VECS], w[N];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            w[k] = k < n ? __ldcg(reinterpret_cast<const float2*>(ml[k]))
                         : make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int i = 0; i < VECS; ++i) {
                const int d = (i * 32 + lane) * 2;
                v[k][i] = k < n && d < A.hd ? __ldcg(reinterpret_cast<const float2*>(o[k] + d))
                                            : make_float2(0.f, 0.f);
            }
        }
        float m = M;
#pragma unroll
        for (int k = 0; k < N; ++k) m = fmaxf(m, w[k].x);
        rebase(m);
        const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            if (k >= n) break;
            const float e = ex2(w[k].x - base);
            L = fmaf(w[k].y, e, L);
#pragma unroll
            for (int i = 0; i < VECS; ++i) {
                acc[i].x = fmaf(v[k][i].x, e, acc[i].x);
                acc[i].y = fmaf(v[k][i].y, e, acc[i].y);
            }
        }
    }
    __device__ __forceinline__ void add_range(const PagedArgs& A, const PagedPlan& P, int first,
                                              int last, int head_lane, int row, int warp,
                                              int warps) {
        constexpr int kBatch = 4;
        for (int p = first + warp; p <= last; p += kBatch * warps) {
            const float *o[kBatch], *ml[kBatch];
            int n = 0;
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const int pp = min(p + k * warps, last);
                const size_t id = part_row(P, pp, head_lane, pp == first, row);
                o[k] = P.part_o + id * A.hd;
                ml[k] = P.part_ml + id * 2;
                n += p + k * warps <= last;
            }
            add<kBatch>(A, o, ml, n);
        }
    }
    // All warps of the block: a row's warps (consecutive ones) hand their sums to the first.
    __device__ __forceinline__ void meet(JoinShared<VECS>& S, int warp, int warps) {
        if (warps == 1) return;
        const int lane = threadIdx.x & 31, me = threadIdx.x / 32;
#pragma unroll
        for (int i = 0; i < VECS; ++i) S.acc[me][i * 32 + lane] = acc[i];
        if (lane == 0) {
            S.m[me] = M;
            S.l[me] = L;
        }
        __syncthreads();
        if (warp != 0) return;
        for (int w = me + 1; w < me + warps; ++w) {
            const float m = S.m[w];
            rebase(fmaxf(M, m));
            const float e = ex2(m - (M == -INFINITY ? 0.f : M));
            L = fmaf(S.l[w], e, L);
#pragma unroll
            for (int i = 0; i < VECS; ++i) {
                const float2 v = S.acc[w][i * 32 + lane];
                acc[i].x = fmaf(v.x, e, acc[i].x);
                acc[i].y = fmaf(v.y, e, acc[i].y);
            }
        }
    }
    // One row without tiles, position by position: what it does not see is never touched.
    template <typename T, bool SPLIT>
    __device__ __noinline__ void restate(const PagedArgs& A, int t, int h) {
        init();
        const int lane = threadIdx.x & 31;
        const int s = last_le(A.q_start, A.n_seq, t);
        const int pos = cached_positions(A, s) - (A.q_start[s + 1] - t), kvh = h / A.group;
        const int sinks = A.window > 0 ? A.sinks : 0;
        const int lo = A.window > 0 ? max(0, pos - A.window + 1) : 0;
        const size_t at = (size_t)t * A.q_stride + (size_t)h * A.hd;
        float2 q[VECS];
#pragma unroll
        for (int i = 0; i < VECS; ++i) {
            const int d = (i * 32 + lane) * 2;
            q[i] = make_float2(0.f, 0.f);
            if (d >= A.hd) continue;
            q[i] = SPLIT ? *reinterpret_cast<const float2*>(reinterpret_cast<const float*>(A.q) + at + d)
                         : PMath<T>::unpack(*reinterpret_cast<const uint32_t*>(
                               reinterpret_cast<const T*>(A.q) + at + d));
        }
        for (int j = min(sinks, lo) > 0 ? 0 : lo; j <= pos; ++j) {
            if (j >= sinks && j < lo) j = lo;
            const int p = A.page_shift >= 0 ? j >> A.page_shift : j / A.page_size;
            const int page = A.table[(size_t)s * A.table_stride + p];
            const bool in = (unsigned)page < (unsigned)A.n_pages;  // (else: zeros)
            const size_t row = (size_t)(in ? page : 0) * A.page_stride +
                               ((size_t)(j - p * A.page_size) * A.nkv + kvh) * A.hd;
            float dot = 0.f;
            float2 v[VECS];
#pragma unroll
            for (int i = 0; i < VECS; ++i) {
                const int d = (i * 32 + lane) * 2;
                v[i] = make_float2(0.f, 0.f);
                if (d >= A.hd || !in) continue;
                const float2 k = PMath<T>::unpack(*reinterpret_cast<const uint32_t*>(
                    reinterpret_cast<const T*>(A.k) + row + d));
                v[i] = PMath<T>::unpack(*reinterpret_cast<const uint32_t*>(
                    reinterpret_cast<const T*>(A.v) + row + d));
                dot = fmaf(q[i].x, k.x, fmaf(q[i].y, k.y, dot));
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
            const float x = dot * A.scale_log2;
            rebase(fmaxf(M, x));
            const float e = ex2(x - (M == -INFINITY ? 0.f : M));
            L += e;
#pragma unroll
            for (int i = 0; i < VECS; ++i) {
                acc[i].x = fmaf(v[i].x, e, acc[i].x);
                acc[i].y = fmaf(v[i].y, e, acc[i].y);
            }
        }
    }
    template <typename T, bool SPLIT>
    __device__ void write(const PagedArgs& A, int t, int h) {
        const int lane = threadIdx.x & 31;
        const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
        for (int i = 0; i < VECS; ++i) {
            const int d = (i * 32 + lane) * 2;
            if (d >= A.hd) break;
            const size_t at = (size_t)t * A.out_stride + (size_t)h * A.hd + d;
            const float2 v = L == 0.f ? make_float2(0.f, 0.f)
                                      : make_float2(acc[i].x * inv, acc[i].y * inv);
            if (SPLIT) *reinterpret_cast<float2*>(reinterpret_cast<float*>(A.out) + at) = v;
            else *reinterpret_cast<uint32_t*>(reinterpret_cast<T*>(A.out) + at) = PMath<T>::pack(v.x, v.y);
        }
        if (lane == 0 && A.lse)
            A.lse[(size_t)t * A.nh + h] = row_lse(M, L);
    }
};

}  // namespace
}  // namespace wb
