// paged.cu -- the paged cache's entry points: rotary positions with the append of k and v,
// page copies, and the attention calls (argument checks, workspace, choice of kernels; the
// kernels are in paged_plan.cu and paged_attn.cu).

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include <algorithm>
#include <atomic>
#include <new>
#include <vector>

#include "internal.h"
#include "paged.h"
#include "paged_math.cuh"

namespace wb {

cudaError_t launch_paged_plan(const PagedArgs& A, cudaStream_t s);
cudaError_t launch_paged_few(const PagedArgs& A, int which, bool both, bool behind, int q_dtype,
                             int kv_dtype, cudaStream_t s);
int paged_few_ctas(int hd);
cudaError_t launch_paged_attn(const PagedArgs& A, int which, int rw, int q_dtype, int kv_dtype,
                              cudaStream_t s);
cudaError_t launch_paged_mma(const PagedArgs& A, int which, int q_dtype, int kv_dtype,
                             cudaStream_t s);
bool paged_mma_takes(int hd);
int paged_mma_rows(bool split);
cudaError_t launch_paged_join(const PagedArgs& A, int q_dtype, int kv_dtype, cudaStream_t s);
int paged_attn_rw(int rows, bool split);
int paged_attn_ctas();

namespace {

// ------------------------------------------------------------------------
// Rotary positions and append.
//
// Bound by HBM: every row is read once and written once.  A head is units of two pieces of eight
// dims: the pairs that turn together, or what passes through.  A CTA takes a block of at most 384
// units through every gridDim.x-th token; where a thread's units lie is worked out once.  Finding
// a token's place is three loads behind one another and the sines and cosines of its position, so
// a warp of its own does that one token ahead of the four that turn the rows.  (A CTA per token
// with the chain in front of its rows: 114 us for 10,838 tokens of 48 heads of 128 in bf16; with
// the rows' loads in front of the chain: 86 us.)  The angle in turns is reduced in 64 bits, then
// sin and cos are taken in 32.
// ------------------------------------------------------------------------
constexpr int kRopeWork = 128;                  // threads that turn rows
constexpr int kRopeThreads = kRopeWork + 32;  // and the warp that finds their places
constexpr int kRopeUnits = 3;                 // of a thread, in flight together
constexpr int kRopeCtas = 8;                  // of an SM

struct RopeArgs {
    const void *q, *k, *v;
    void* q_out;
    void *kp, *vp;
    const int *q_start, *kv_len, *table, *positions;
    const double* freq;
    int* status;
    size_t qs, ks, vs, qos, page_stride;
    int n_seq, n_tokens, table_stride, table_width, n_pages, page_size, nh, nkv, hd;
    int dim, off, interleaved, per_head, units_per_cta;
    float gain;
};

// Eight values as they lie in memory.
template <typename T>
struct Raw8 {
    uint4 w[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = *(reinterpret_cast<const uint4*>(p) + i);
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
            const uint32_t u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (sizeof(T) == 4) {
                    v[i * 4 + e] = __uint_as_float(u[e]);
                } else {
                    const float2 f = PMath<T>::unpack(u[e]);
                    v[2 * e] = f.x;
                    v[2 * e + 1] = f.y;
                }
            }
        }
    }
};
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
        *(reinterpret_cast<float4*>(p) + 1) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        *reinterpret_cast<uint4*>(p) =
            make_uint4(PMath<T>::pack(v[0], v[1]), PMath<T>::pack(v[2], v[3]),
                       PMath<T>::pack(v[4], v[5]), PMath<T>::pack(v[6], v[7]));
    }
}

// A thread's unit: which row it is in and where its pieces start (d1 < 0: there is one only).
struct RopeUnit {
    int kind;  // 0: q, 1: k, 2: v
    int h, d0, d1;
    int turn;  // first of its eight pairs, -1: it passes through
    __device__ __forceinline__ RopeUnit() {}
    __device__ __forceinline__ RopeUnit(const RopeArgs& A, int i) {
        h = i / A.per_head;
        const int u = i - h * A.per_head, pairs = A.dim / 16;
        kind = h < A.nh ? 0 : h < A.nh + A.nkv ? 1 : 2;
        h -= kind == 0 ? 0 : kind == 1 ? A.nh : A.nh + A.nkv;
        turn = u < pairs && kind < 2 ? u * 8 : -1;
        if (u < pairs) {
            d0 = A.interleaved ? A.off + u * 16 : A.off + u * 8;
            d1 = A.interleaved ? d0 + 8 : d0 + A.dim / 2;
        } else {
            d0 = (u - pairs) * 16;
            d1 = d0 + 8 < A.hd - A.dim ? d0 + 8 : -1;
            if (d1 >= A.off) d1 += A.dim;
            if (d0 >= A.off) d0 += A.dim;
        }
    }
};

template <typename TI, typename TC, typename TQ>
__global__ void __launch_bounds__(kRopeThreads) rope_append_kernel(const __grid_constant__ RopeArgs A) {
    __shared__ float2 cs[2][128];   // (cos, sin) * gain of each pair of this and the next token
    __shared__ long long s_row[2];  // the token's row in the pages, -1: it has none
    const int tid = threadIdx.x, half = A.dim / 2, step = gridDim.x;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (tid >= kRopeWork) {
        const int lane = tid & 31;
        double freq[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) freq[k] = lane + 32 * k < half ? A.freq[lane + 32 * k] : 0.0;
        int b = 0;
        for (int t = blockIdx.x; t < A.n_tokens; t += step, b ^= 1) {
            int seq = -1;
            for (int s = lane; s < A.n_seq; s += 32)
                if (A.q_start[s] <= t && t < A.q_start[s + 1]) seq = s;
            seq = __reduce_max_sync(0xffffffffu, seq);
            int pos = -1, page = -1;
            if (seq >= 0) {
                pos = A.kv_len[seq] - (A.q_start[seq + 1] - t);
                if (pos >= 0 && pos < (long long)A.table_width * A.page_size) {
                    page = A.table[(size_t)seq * A.table_stride + pos / A.page_size];
                    if ((unsigned)page >= (unsigned)A.n_pages) page = -1;
                }
                if (page < 0 && pos >= 0 && lane == 0 && A.status) atomicOr(A.status, PG_BAD_PAGE);
            }
            const double at = (double)(A.positions ? A.positions[t] : pos) * 0.15915494309189533577;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (lane + 32 * k >= half) break;
                const double turns = at * freq[k];
                float s, c;
                sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
                cs[b][lane + 32 * k] = make_float2(c * A.gain, s * A.gain);
            }
            if (lane == 0)
                s_row[b] = page < 0 ? -1
                                    : (long long)page * (long long)A.page_stride +
                                          (long long)(pos % A.page_size) * A.nkv * A.hd;
            __syncthreads();
        }
        return;
    }
    const int first = blockIdx.y * A.units_per_cta + tid;
    const int end = min((A.nh + 2 * A.nkv) * A.per_head, (int)(blockIdx.y + 1) * A.units_per_cta);
    RopeUnit U[kRopeUnits];
    const TI* src[kRopeUnits];
    size_t stride[kRopeUnits];
    int n = 0;
#pragma unroll
    for (int k = 0; k < kRopeUnits; ++k) {
        if (first + k * kRopeWork >= end) break;
        U[k] = RopeUnit(A, first + k * kRopeWork);
        src[k] = reinterpret_cast<const TI*>(U[k].kind == 0 ? A.q : U[k].kind == 1 ? A.k : A.v) +
                 (size_t)U[k].h * A.hd;
        stride[k] = U[k].kind == 0 ? A.qs : U[k].kind == 1 ? A.ks : A.vs;
        n = k + 1;
    }
    int b = 0;
    for (int t = blockIdx.x; t < A.n_tokens; t += step, b ^= 1) {
        Raw8<TI> x[kRopeUnits], y[kRopeUnits];
#pragma unroll
        for (int k = 0; k < kRopeUnits; ++k) {
            if (k >= n) break;
            const TI* from = src[k] + (size_t)t * stride[k];
            x[k].load(from + U[k].d0);
            if (U[k].d1 >= 0) y[k].load(from + U[k].d1);
        }
        __syncthreads();
        const long long row = s_row[b];
#pragma unroll
        for (int k = 0; k < kRopeUnits; ++k) {
            if (k >= n) break;
            if (row < 0 && U[k].kind > 0) continue;
            float a[8], c[8];
            x[k].get(a);
            y[k].get(c);
            if (row < 0) {
#pragma unroll
                for (int e = 0; e < 8; ++e) a[e] = c[e] = 0.f;
            } else if (U[k].turn >= 0) {
                const float2* w = cs[b] + U[k].turn;
                if (A.interleaved) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 p = w[e], q = w[4 + e];
                        const float a0 = a[2 * e], a1 = a[2 * e + 1], c0 = c[2 * e], c1 = c[2 * e + 1];
                        a[2 * e] = a0 * p.x - a1 * p.y;
                        a[2 * e + 1] = a1 * p.x + a0 * p.y;
                        c[2 * e] = c0 * q.x - c1 * q.y;
                        c[2 * e + 1] = c1 * q.x + c0 * q.y;
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float2 p = w[e];
                        const float a0 = a[e], c0 = c[e];
                        a[e] = a0 * p.x - c0 * p.y;
                        c[e] = c0 * p.x + a0 * p.y;
                    }
                }
            }
            if (U[k].kind == 0) {
                TQ* to = reinterpret_cast<TQ*>(A.q_out) + (size_t)t * A.qos + (size_t)U[k].h * A.hd;
                store8(to + U[k].d0, a);
                if (U[k].d1 >= 0) store8(to + U[k].d1, c);
            } else {
                TC* to = reinterpret_cast<TC*>(U[k].kind == 1 ? A.kp : A.vp) + row +
                         (size_t)U[k].h * A.hd;
                store8(to + U[k].d0, a);
                if (U[k].d1 >= 0) store8(to + U[k].d1, c);
            }
        }
    }
}

template <typename TI, typename TC>
cudaError_t launch_rope(const RopeArgs& A, bool q_as_cache, cudaStream_t s) {
    RopeArgs B = A;
    B.per_head = A.dim / 16 + (A.hd - A.dim + 15) / 16;
    // blocks of units that a CTA's threads hold at once; few tokens: smaller ones on more SMs
    const int units = (A.nh + 2 * A.nkv) * B.per_head;
    const int fit = (units + kRopeUnits * kRopeWork - 1) / (kRopeUnits * kRopeWork);
    const int spread = std::min((units + kRopeWork - 1) / kRopeWork,
                                2 * sm_count() / std::max(1, A.n_tokens));
    const int parts = std::max(fit, spread);
    B.units_per_cta = (units + parts - 1) / parts;
    const dim3 grid(std::min(A.n_tokens, std::max(1, kRopeCtas * sm_count() / parts)), parts);
    if (q_as_cache)
        return launch_pdl(rope_append_kernel<TI, TC, TC>, grid, dim3(kRopeThreads), 0, s, B);
    return launch_pdl(rope_append_kernel<TI, TC, TI>, grid, dim3(kRopeThreads), 0, s, B);
}

// ------------------------------------------------------------------------
// Page copies: CTA (piece of a page, layer and K / V, move); the moves travel in the launch's
// parameters, so nothing is copied to the device and nothing is waited for.  Bound by HBM: 512
// pages of 32 KB in 32 layers 338 us = 6.35 TB/s read and written (98% of the measured copy);
// four pages 4 us.
// ------------------------------------------------------------------------
constexpr int kCopyThreads = 256;
constexpr int kCopyVec = 8;  // 16-byte loads in flight per thread
constexpr size_t kCopyPiece = (size_t)kCopyThreads * kCopyVec * 16;

template <int N>
struct CopyArgs {
    char *k, *v;
    size_t layer_bytes, page_stride_bytes, page_bytes;
    int n_layers;
    int2 move[N];
};

template <int N>
__global__ void __launch_bounds__(kCopyThreads) pages_copy_kernel(const __grid_constant__ CopyArgs<N> A) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int2 mv = A.move[blockIdx.z];
    const int l = blockIdx.y >> 1;
    char* base = (blockIdx.y & 1 ? A.v : A.k) + (size_t)l * A.layer_bytes;
    const uint4* src = reinterpret_cast<const uint4*>(base + (size_t)mv.x * A.page_stride_bytes);
    uint4* dst = reinterpret_cast<uint4*>(base + (size_t)mv.y * A.page_stride_bytes);
    const size_t n = A.page_bytes / 16;
    const size_t at = (size_t)blockIdx.x * kCopyThreads * kCopyVec + threadIdx.x;
    uint4 r[kCopyVec];
#pragma unroll
    for (int i = 0; i < kCopyVec; ++i)
        if (at + i * kCopyThreads < n) r[i] = __ldcs(src + at + i * kCopyThreads);
#pragma unroll
    for (int i = 0; i < kCopyVec; ++i)
        if (at + i * kCopyThreads < n) __stcs(dst + at + i * kCopyThreads, r[i]);
}

template <int N>
cudaError_t launch_copy(const WispKvPages* P, int n_layers, size_t layer_stride, const int* src,
                        const int* dst, int n, cudaStream_t s) {
    CopyArgs<N> A;
    A.k = static_cast<char*>(P->k);
    A.v = static_cast<char*>(P->v);
    A.layer_bytes = layer_stride * 2;
    A.page_stride_bytes = P->page_stride * 2;
    A.page_bytes = (size_t)P->page_size * P->n_kv_heads * P->head_dim * 2;
    A.n_layers = n_layers;
    for (int i = 0; i < n; ++i) A.move[i] = make_int2(src[i], dst[i]);
    const unsigned pieces = (unsigned)((A.page_bytes + kCopyPiece - 1) / kCopyPiece);
    return launch_pdl(pages_copy_kernel<N>, dim3(pieces, 2 * n_layers, n), dim3(kCopyThreads), 0, s,
                      A);
}

// ------------------------------------------------------------------------
// Argument checks
// ------------------------------------------------------------------------
bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool known(int d) { return d == WISP_DTYPE_F32 || d == WISP_DTYPE_F16 || d == WISP_DTYPE_BF16; }

#define PG_REFUSE(...)                                      \
    do {                                                    \
        WB_SET_ERR(err, WISP_ERR_INVALID_ARG, __VA_ARGS__); \
        return WISP_ERR_INVALID_ARG;                        \
    } while (0)

WispError check_pages(const char* who, const WispKvPages* P, WispErrCtx* err) {
    if (!P || !P->k || !P->v || !al16(P->k) || !al16(P->v))
        PG_REFUSE("%s: pages NULL or not 16-byte aligned", who);
    if (P->dtype != WISP_DTYPE_F16 && P->dtype != WISP_DTYPE_BF16)
        PG_REFUSE("%s: pages of dtype %d (fp16 or bf16)", who, P->dtype);
    if (P->n_pages <= 0 || P->page_size <= 0 || P->page_size % 8 || P->page_size > 65536 ||
        P->n_kv_heads <= 0 || P->n_kv_heads > 1024 || P->head_dim <= 0 || P->head_dim % 8 ||
        P->head_dim > 256)
        PG_REFUSE("%s: unsupported pages: %d of %d positions, %d heads of %d (page_size a multiple "
                  "of 8, head_dim a multiple of 8 up to 256)",
                  who, P->n_pages, P->page_size, P->n_kv_heads, P->head_dim);
    if (P->page_stride % 8 ||
        P->page_stride < (size_t)P->page_size * P->n_kv_heads * P->head_dim)
        PG_REFUSE("%s: page_stride %zu (a multiple of 8, at least a page)", who, P->page_stride);
    return WISP_OK;
}

WispError check_batch(const char* who, const WispTokenBatch* B, WispErrCtx* err) {
    if (!B || B->n_seq < 0 || B->n_tokens < 0 || B->max_q < 0 || B->table_stride < 0 ||
        B->table_width < 0 || B->table_width > B->table_stride)
        PG_REFUSE("%s: batch NULL or negative", who);
    if (B->n_tokens > 0 &&
        (B->n_seq == 0 || !B->q_start || !B->kv_len || !B->table || B->table_stride == 0 ||
         B->max_q == 0))
        PG_REFUSE("%s: a batch of %d tokens without sequences, table or max_q", who, B->n_tokens);
    return WISP_OK;
}

WispError check_rows(const char* who, const char* name, const WispRows* R, int hd, WispErrCtx* err) {
    if (!R || !R->base || !al16(R->base) || !known(R->dtype))
        PG_REFUSE("%s: %s NULL, not 16-byte aligned or of unknown dtype", who, name);
    if (R->n_heads <= 0 || R->n_heads > 65535 || R->stride % 8 ||
        R->stride < (size_t)R->n_heads * hd)
        PG_REFUSE("%s: %s has %d heads and stride %zu (a multiple of 8, at least its heads)", who,
                  name, R->n_heads, R->stride);
    return WISP_OK;
}

// Do the rows of n tokens (the same number of heads and dtype) share memory?
bool overlap(const WispRows& a, const WispRows& b, int n, int hd) {
    const long long size = a.dtype == WISP_DTYPE_F32 ? 4 : 2, w = (long long)a.n_heads * hd * size;
    const long long sa = (long long)a.stride * size, sb = (long long)b.stride * size;
    const long long d = static_cast<char*>(b.base) - static_cast<char*>(a.base);
    if (d >= (n - 1) * sa + w || -d >= (n - 1) * sb + w) return false;
    for (long long t = 0; t < n; ++t) {
        // the first row of b that ends behind the begin of row t of a
        const long long gap = t * sa - d - w;
        const long long u = gap < 0 ? 0 : gap / sb + 1;
        if (u < n && d + u * sb < t * sa + w) return true;
    }
    return false;
}

// ------------------------------------------------------------------------
// Attention: what runs, and its workspace
// ------------------------------------------------------------------------
// What a row tile costs before its first KV tile, in KV tiles (a prompt of 8192 tokens took 816 us
// with 0 and 694 us with 4, later 560 us with 4 and 540 us with 6, where a KV tile took 0.94 us
// and a beginning 5.4 us; fp32 rows, which are split first: 2048 tokens 280 us with 3, 212 with 6,
// 179 with 12 (205 when measured again), 191 with 16, and 3 x 500 tokens behind 4000 116 us with 3 and 118 with 12; 14 single
// tokens behind up to 4096 positions 32.6 us with 0 and 30.9 us with 2).
constexpr int kLeadMma = 6, kLeadMma32 = 12, kLeadFew = 2;
// Up to so many 16-row tiles stay with paged_few_kernel, where all that they read again (for wide
// heads: all that the tables can name) is at most so large.
constexpr int kFewTiles = 4, kFewTilesWide = 8;
constexpr double kFewBytes = 50e6, kFewBytesWide = 100e6;

struct AttnShape {
    int rw[PLANS];  // 16-row tiles of the plan's row tiles; 0: the tensor-core kernel
    size_t bytes;
    double units;  // no plan's line of work is longer
};

// Fills the geometry, plans and (with a workspace) pointers of a call.
//
// Which kernel: a sequence (or group) whose rows for one kv head fit one 16-row tile of
// mma.sync (8 rows in fp32) goes through paged_few_kernel, whose CTAs are bound by HBM; more
// rows go to tcgen05 where it takes the head dim, else to paged_attn_kernel's row tiles of two
// or four 16-row tiles.  A batch goes by its longest sequence: single tokens beside a prompt
// take its kernel too (they read the cache at 80% of HBM there instead of 95%; a second pair of
// launches for them cost 12 us a call).  A few 16-row tiles stay with paged_few_kernel where they are
// few enough to read the cache again out of L2: it needs no plan kernel before it.  The lengths
// are not known here, so what a batch reads again is bounded by its table's width: a table wider
// than its sequences need (a captured step's) leaves this choice early.  Measured with tables as
// wide as the longest sequence (B200, 8 kv heads; paged_few_kernel against the other):
//   128 dims, 4 sequences of 1024: 32 rows 19.6 and 22.2 us, 64 rows 25.0 and 20.4 us
//             2 of 4096: 32 rows 23.2 and 23.1 us, 64 rows 31.1 and 24.5 us
//             8 of 8192: 32 rows 98 and 67 us
//     64 rows behind a shared prefix of 2048: 27.5 and 31.4 us, of 8192: 50.2 and 36.9 us
//   256 dims, 4 of 1024: 32 rows 24.0 and 31.2 us, 128 rows 51 and 59 us
//             2 of 4096: 32 rows 30.7 and 38.5 us, 128 rows 80 and 92 us
//             8 of 8192: 32 rows 170 and 153 us, 128 rows 624 and 437 to 460 us
AttnShape attention_layout(PagedArgs& A, int q_dtype, int max_q, char* ws) {
    const bool split = q_dtype == WISP_DTYPE_F32;
    const int per = split ? 8 : 16;
    AttnShape S{};
    size_t at = 256;
    auto take = [&](size_t bytes) {
        char* p = ws ? ws + at : nullptr;
        at += (bytes + 255) / 256 * 256;
        return p;
    };
    A.status = reinterpret_cast<int*>(ws);
    A.group = A.nh / A.nkv;
    const bool mma = paged_mma_takes(A.hd);
    const int few_tok = std::max(1, per / A.group);  // tokens of a 16-row tile
    const double row_bytes = (double)A.table_width * A.page_size * A.nkv * A.hd * 4;
    for (int w = 0; w < PLANS; ++w) {
        PagedPlan& P = A.plan[w];
        P = PagedPlan{};
        const int n_seg = w == PLAN_PREFIX ? A.n_groups : A.n_seq;
        if (n_seg == 0) continue;
        // tokens of the plan's largest segment (a guess for a prefix, which may have all)
        const int tokens = w == PLAN_PREFIX ? (A.n_tokens + n_seg - 1) / n_seg : max_q;
        const int most_tokens = w == PLAN_PREFIX ? A.n_tokens : max_q;
        const long long tiles16 = (long long)((A.group + per - 1) / per) *
                                  ((tokens + few_tok - 1) / few_tok);
        const double bytes = n_seg * row_bytes;  // no more lies behind the segments' table rows
        const bool is_few =
            (long long)tokens * A.group <= per ||
            (mma ? tiles16 <= kFewTiles && tiles16 * bytes <= kFewBytes
                 : tiles16 <= kFewTilesWide && bytes <= kFewBytesWide);
        const bool on_mma = !is_few && mma;
        if (w != PLAN_PREFIX && on_mma != (w == PLAN_MANY)) continue;
        P.used = 1;
        const int most = on_mma ? paged_mma_rows(split) : is_few ? per : 4 * per;
        P.gpb = std::min(A.group, most);
        P.hblocks = (A.group + P.gpb - 1) / P.gpb;
        P.heads = A.nkv * P.hblocks;
        const int rows = (int)std::min<long long>((long long)tokens * P.gpb, most);
        S.rw[w] = on_mma ? 0 : is_few ? 1 : paged_attn_rw(rows, split);
        P.rows = on_mma ? most : S.rw[w] * per;
        P.tpt = std::max(1, P.rows / P.gpb);
        P.used_rows = w == PLAN_PREFIX ? P.rows : std::min(rows, P.rows);
        const int ctas =
            (on_mma ? 1 : is_few ? paged_few_ctas(A.hd) : paged_attn_ctas()) * sm_count();
        P.grain = on_mma && !split ? 2 : 1;
        P.lead = on_mma ? (split ? kLeadMma32 : kLeadMma * P.grain) : kLeadFew;
        P.lanes = std::min(4095, std::max(1, ctas / P.heads));
        if (is_few && w == PLAN_PREFIX && A.plan[PLAN_FEW].used) {  // they share one launch
            A.plan[PLAN_FEW].lanes = std::max(1, A.plan[PLAN_FEW].lanes / 2);
            P.lanes = std::max(1, P.lanes / 2);
        }
        P.max_items = A.n_tokens / P.tpt + n_seg;
        P.per_seg = (most_tokens + P.tpt - 1) / P.tpt;
        P.inlined = is_few && (long long)n_seg * P.per_seg <= kPagedInline;
        if (P.inlined) P.max_items = n_seg * P.per_seg;
        // KV tiles of a row tile: of the positions that a table row holds or, of consecutive tokens
        // with a window, of the window and the sinks
        double tiles = (double)A.table_width * A.page_size / kPagedTile + 1;
        if (A.window > 0 && w != PLAN_PREFIX)
            tiles = std::min(tiles, ((double)A.window + P.tpt + A.sinks) / kPagedTile + 4);
        S.units = std::max(S.units, P.max_items * (tiles * P.grain + P.lead));
        P.n_items = reinterpret_cast<int*>(take(4));
        P.bad = reinterpret_cast<int*>(take(((size_t)P.lanes * P.heads + 1) * 4));
        P.item_off = reinterpret_cast<int*>(take((size_t)(n_seg + 1) * 4));
        P.cum = reinterpret_cast<int*>(take((size_t)(P.max_items + 1) * 4));
        P.items = reinterpret_cast<PagedItem*>(take((size_t)P.max_items * sizeof(PagedItem)));
        const size_t recs = (size_t)P.lanes * P.heads * 2 * P.rows;
        P.part_o = reinterpret_cast<float*>(take(recs * A.hd * 4));
        P.part_ml = reinterpret_cast<float*>(take(recs * 8));
        P.split = reinterpret_cast<PagedSplit*>(take((size_t)P.lanes * sizeof(PagedSplit)));
        if (on_mma) P.redo = reinterpret_cast<int*>(take((size_t)P.max_items * P.heads * 4));
        if (A.n_groups > 0)
            P.where = reinterpret_cast<PagedWhere*>(take((size_t)A.n_tokens * sizeof(PagedWhere)));
    }
    if (A.n_groups > 0) {
        const size_t recs = (size_t)2 * A.n_tokens * A.nh;
        A.full_o = reinterpret_cast<float*>(take(recs * A.hd * 4));
        A.full_ml = reinterpret_cast<float*>(take(recs * 8));
    }
    S.bytes = at;
    return S;
}

cudaError_t launch_plan_kernel(const PagedArgs& A, const AttnShape& S, int which, bool both,
                               bool behind, int q_dtype, int kv_dtype, cudaStream_t s) {
    return S.rw[which] == 0   ? launch_paged_mma(A, which, q_dtype, kv_dtype, s)
           : S.rw[which] == 1 ? launch_paged_few(A, which, both, behind, q_dtype, kv_dtype, s)
                              : launch_paged_attn(A, which, S.rw[which], q_dtype, kv_dtype, s);
}

std::atomic<unsigned long long> g_wait_ns{2000000000ull};

PagedArgs attention_args(const WispKvPages* P, const WispTokenBatch* B, int n_heads, int n_groups) {
    PagedArgs A{};
    A.k = P->k;
    A.v = P->v;
    A.q_start = B->q_start;
    A.kv_len = B->kv_len;
    A.table = B->table;
    A.all_status = B->status;
    A.page_stride = P->page_stride;
    A.n_seq = B->n_seq;
    A.n_tokens = B->n_tokens;
    A.n_groups = n_groups;
    A.table_stride = B->table_stride;
    A.table_width = B->table_width ? B->table_width : B->table_stride;
    A.n_pages = P->n_pages;
    A.page_size = P->page_size;
    A.page_shift = (P->page_size & (P->page_size - 1)) ? -1 : __builtin_ctz(P->page_size);
    A.nh = n_heads;
    A.nkv = P->n_kv_heads;
    A.hd = P->head_dim;
    A.wait_ns = g_wait_ns.load(std::memory_order_relaxed);
    return A;
}

WispError attention_call(const char* who, const WispRows* q, const WispRows* out, float* lse,
                         const WispKvPages* P, const WispTokenBatch* B, const int* groups,
                         const int* prefix_len, int n_groups, float scale, int window, int sinks,
                         void* ws, size_t ws_bytes, cudaStream_t s, WispErrCtx* err) {
    WispError rc;
    if ((rc = check_pages(who, P, err)) || (rc = check_batch(who, B, err))) return rc;
    if (B->n_tokens == 0) {  // nothing can go wrong: the status word says so
        if (ws && al16(ws) && ws_bytes >= 4)
            WB_CUDA_RET(launch_zero_words(static_cast<int*>(ws), 1, s), err);
        return WISP_OK;
    }
    if ((rc = check_rows(who, "q", q, P->head_dim, err)) ||
        (rc = check_rows(who, "out", out, P->head_dim, err)))
        return rc;
    if (q->dtype != out->dtype || (q->dtype != WISP_DTYPE_F32 && q->dtype != P->dtype))
        PG_REFUSE("%s: q of dtype %d, out of %d (fp32 or the pages' %d, both the same)", who,
                  q->dtype, out->dtype, P->dtype);
    if (q->n_heads != out->n_heads || q->n_heads % P->n_kv_heads)
        PG_REFUSE("%s: %d heads of q, %d of out (a multiple of the %d kv heads, both the same)", who,
                  q->n_heads, out->n_heads, P->n_kv_heads);
    if (overlap(*q, *out, B->n_tokens, P->head_dim))
        PG_REFUSE("%s: out overlaps q, whose rows may be read again behind the results", who);
    if (!(fabsf(scale) <= 3e38f) || window < 0 || sinks < 0)
        PG_REFUSE("%s: scale %g, window %d, sinks %d (finite; not negative)", who, (double)scale,
                  window, sinks);
    if (n_groups < 0 || (n_groups > 0 && (!groups || !prefix_len)))
        PG_REFUSE("%s: %d groups without their arrays", who, n_groups);
    PagedArgs A = attention_args(P, B, q->n_heads, n_groups);
    A.q = q->base;
    A.out = out->base;
    A.lse = lse;
    A.groups = groups;
    A.prefix_len = prefix_len;
    A.q_stride = q->stride;
    A.out_stride = out->stride;
    A.window = window >= (1 << 30) ? 0 : window;  // longer than any cache: none
    A.sinks = sinks;
    A.scale_log2 = scale * 1.4426950408889634f;
    const AttnShape S = attention_layout(A, q->dtype, std::min(B->max_q, B->n_tokens),
                                         static_cast<char*>(ws));
    if (S.units >= 2147483648.0)  // (they are counted in 32 bits)
        PG_REFUSE("%s: up to %.2g KV tiles in one call, the limit is 2^31: fewer tokens at a time or a "
                  "narrower table", who, S.units);
    if (!ws || !al16(ws) || ws_bytes < S.bytes)
        PG_REFUSE("%s: workspace of %zu bytes, need %zu (16-byte aligned)", who, ws ? ws_bytes : 0,
                  S.bytes);
    bool plan = false;
    for (int w = 0; w < PLANS; ++w) plan |= A.plan[w].used && !A.plan[w].inlined;
    if (plan) WB_CUDA_RET(launch_paged_plan(A, s), err);
    // the shared prefixes go with the sequences' own parts where one kernel takes both
    const bool both = A.plan[PLAN_PREFIX].used && A.plan[PLAN_FEW].used &&
                      S.rw[PLAN_PREFIX] == 1 && S.rw[PLAN_FEW] == 1;
    const int order[PLANS] = {PLAN_PREFIX, PLAN_MANY, PLAN_FEW};
    bool behind = false;
    for (int w : order) {
        if (!A.plan[w].used || (w == PLAN_PREFIX && both)) continue;
        WB_CUDA_RET(launch_plan_kernel(A, S, w, both && w == PLAN_FEW, behind, q->dtype, P->dtype, s),
                    err);
        behind = true;
    }
    WB_CUDA_RET(launch_paged_join(A, q->dtype, P->dtype, s), err);
    return WISP_OK;
}

}  // namespace
}  // namespace wb

using namespace wb;

extern "C" unsigned long long wisp_paged_wait_limit(unsigned long long ns) {
    return g_wait_ns.exchange(ns, std::memory_order_relaxed);
}

extern "C" size_t wisp_paged_attention_workspace_bytes(const WispKvPages* P, const WispTokenBatch* B,
                                                       int n_heads, int q_dtype, int n_groups) {
    if (check_pages("paged_attention", P, nullptr) || check_batch("paged_attention", B, nullptr) ||
        n_heads <= 0 || n_heads % P->n_kv_heads || n_groups < 0 || B->n_tokens == 0)
        return 0;
    PagedArgs A = attention_args(P, B, n_heads, n_groups);
    return attention_layout(A, q_dtype, std::min(B->max_q, B->n_tokens), nullptr).bytes;
}

extern "C" WispError wisp_paged_attention(const WispRows* q, const WispRows* out, float* lse,
                                          const WispKvPages* pages, const WispTokenBatch* batch,
                                          float scale, int window, int sinks, void* workspace,
                                          size_t workspace_bytes, cudaStream_t stream,
                                          WispErrCtx* err) {
    return attention_call("paged_attention", q, out, lse, pages, batch, nullptr, nullptr, 0, scale,
                          window, sinks, workspace, workspace_bytes, stream, err);
}

extern "C" WispError wisp_prefix_attention(const WispRows* q, const WispRows* out, float* lse,
                                           const WispKvPages* pages, const WispTokenBatch* batch,
                                           const int* groups, const int* prefix_len, int n_groups,
                                           float scale, int window, int sinks, void* workspace,
                                           size_t workspace_bytes, cudaStream_t stream,
                                           WispErrCtx* err) {
    return attention_call("prefix_attention", q, out, lse, pages, batch, groups, prefix_len,
                          n_groups, scale, window, sinks, workspace, workspace_bytes, stream, err);
}

extern "C" WispError wisp_rope_append(const WispRows* q, const WispRows* k, const WispRows* v,
                                      const WispRows* q_out, const WispKvPages* P,
                                      const WispTokenBatch* B, const WispRope* rope, int* status,
                                      cudaStream_t s, WispErrCtx* err) {
    const char* who = "rope_append";
    WispError rc;
    if ((rc = check_pages(who, P, err)) || (rc = check_batch(who, B, err))) return rc;
    if (B->n_tokens == 0) return WISP_OK;
    const int hd = P->head_dim;
    if ((rc = check_rows(who, "q", q, hd, err)) || (rc = check_rows(who, "k", k, hd, err)) ||
        (rc = check_rows(who, "v", v, hd, err)) || (rc = check_rows(who, "q_out", q_out, hd, err)))
        return rc;
    if (q->dtype != k->dtype || q->dtype != v->dtype ||
        (q_out->dtype != q->dtype && q_out->dtype != P->dtype))
        PG_REFUSE("%s: q, k, v of dtypes %d, %d, %d and q_out of %d (the first three the same, q_out "
                  "theirs or the pages' %d)",
                  who, q->dtype, k->dtype, v->dtype, q_out->dtype, P->dtype);
    if (q_out->n_heads != q->n_heads || k->n_heads != P->n_kv_heads || v->n_heads != P->n_kv_heads)
        PG_REFUSE("%s: %d heads of q, %d of q_out, %d of k, %d of v for %d kv heads", who, q->n_heads,
                  q_out->n_heads, k->n_heads, v->n_heads, P->n_kv_heads);
    if (!rope || rope->dim < 0 || rope->dim % 16 || rope->offset < 0 || rope->offset % 8 ||
        rope->offset + rope->dim > hd || (rope->dim > 0 && !rope->inv_freq))
        PG_REFUSE("%s: a window of %d at %d in heads of %d (a multiple of 16 at one of 8, with "
                  "frequencies)",
                  who, rope ? rope->dim : 0, rope ? rope->offset : 0, hd);
    RopeArgs A{};
    A.q = q->base;
    A.k = k->base;
    A.v = v->base;
    A.q_out = q_out->base;
    A.kp = P->k;
    A.vp = P->v;
    A.q_start = B->q_start;
    A.kv_len = B->kv_len;
    A.table = B->table;
    A.positions = rope->positions;
    A.freq = rope->inv_freq;
    A.status = status;
    A.qs = q->stride;
    A.ks = k->stride;
    A.vs = v->stride;
    A.qos = q_out->stride;
    A.page_stride = P->page_stride;
    A.n_seq = B->n_seq;
    A.n_tokens = B->n_tokens;
    A.table_stride = B->table_stride;
    A.table_width = B->table_width ? B->table_width : B->table_stride;
    A.n_pages = P->n_pages;
    A.page_size = P->page_size;
    A.nh = q->n_heads;
    A.nkv = P->n_kv_heads;
    A.hd = hd;
    A.dim = rope->dim;
    A.off = rope->offset;
    A.interleaved = rope->interleaved != 0;
    A.gain = rope->gain;
    const bool h = P->dtype == WISP_DTYPE_F16, as_cache = q_out->dtype != q->dtype;
    cudaError_t e;
    if (q->dtype == WISP_DTYPE_F32)
        e = h ? launch_rope<float, __half>(A, as_cache, s)
              : launch_rope<float, __nv_bfloat16>(A, as_cache, s);
    else if (q->dtype == WISP_DTYPE_F16)
        e = h ? launch_rope<__half, __half>(A, as_cache, s)
              : launch_rope<__half, __nv_bfloat16>(A, as_cache, s);
    else
        e = h ? launch_rope<__nv_bfloat16, __half>(A, as_cache, s)
              : launch_rope<__nv_bfloat16, __nv_bfloat16>(A, as_cache, s);
    WB_CUDA_RET(e, err);
    return WISP_OK;
}

extern "C" WispError wisp_pages_copy(const WispKvPages* P, int n_layers, size_t layer_stride,
                                     const int* src, const int* dst, int n, cudaStream_t s,
                                     WispErrCtx* err) {
    const char* who = "pages_copy";
    WispError rc;
    if ((rc = check_pages(who, P, err))) return rc;
    if (n < 0 || (n > 0 && (!src || !dst)) || n_layers <= 0 || n_layers > 32767 || layer_stride % 8)
        PG_REFUSE("%s: %d moves, %d layers, layer_stride %zu (a multiple of 8)", who, n, n_layers,
                  layer_stride);
    if (n == 0) return WISP_OK;
    try {
        // 1: a source, 2: a destination
        std::vector<unsigned char> seen(P->n_pages, 0);
        for (int i = 0; i < n; ++i) {
            if (src[i] < 0 || src[i] >= P->n_pages || dst[i] < 0 || dst[i] >= P->n_pages)
                PG_REFUSE("%s: move %d (%d -> %d) outside a pool of %d pages", who, i, src[i], dst[i],
                          P->n_pages);
            seen[src[i]] |= 1;
        }
        for (int i = 0; i < n; ++i) {
            if (seen[dst[i]])
                PG_REFUSE("%s: page %d is %s", who, dst[i],
                          seen[dst[i]] & 1 ? "a source and a destination" : "twice a destination");
            seen[dst[i]] |= 2;
        }
    } catch (const std::bad_alloc&) {
        WB_SET_ERR(err, WISP_ERR_OOM, "%s: no host memory", who);
        return WISP_ERR_OOM;
    }
    constexpr int kFew = 64, kMany = 1024;  // moves in a launch's parameters
    for (int at = 0; at < n; at += kMany) {
        const int m = std::min(kMany, n - at);
        WB_CUDA_RET(m <= kFew ? launch_copy<kFew>(P, n_layers, layer_stride, src + at, dst + at, m, s)
                              : launch_copy<kMany>(P, n_layers, layer_stride, src + at, dst + at, m, s),
                    err);
    }
    return WISP_OK;
}
