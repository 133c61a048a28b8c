// paged_attn.cu -- causal attention of a batch's tokens over a paged fp16 / bf16 cache: the kernel
// for many rows of heads wider than 128, and the join of what pieces share for all kernels.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i . k_j)
//   over cached j <= i with (window == 0 or i - j < window or j < sinks)
//
// A row tile holds the rows (token, query head) of consecutive tokens that read one kv head;
// it passes over the positions once with a running maximum and sum per row.  The line of all
// (row tile, KV tile) pairs of the batch is cut into equal pieces (paged_plan.cu), one CTA
// per piece and kv head: ragged batches balance by themselves, long sequences are split over
// many CTAs, and at most two row tiles of a piece are shared with its neighbours, whose
// partial results a second kernel joins in a fixed order (results do not depend on timing).
//
// Products run on mma.sync m16n8k16 with fp32 accumulators.  32-bit rows are split into two
// 16-bit parts (x ~= hi + lo, 22 bits in fp16) that fill the two halves of a
// 16-row tile, so 8 rows cost one instruction and their two sums meet in one thread; the
// weights p are split the same way.  bf16 parts hold 8 bits each, so there it takes three and a
// second instruction (two parts left the results 2.8e-6 off, ten times the fp32 rounding).  In
// fp16, p is scaled by 2^kPShift so that small weights of long contexts stay above the subnormals
// (the factor cancels in the quotient).
//
// The join reads each split row tile's partial sums (fp32) and their maxima; with its loads in
// flight together it takes 4 us for a row over 37 pieces (21 us one piece after another).

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "internal.h"
#include "paged.h"
#include "paged_math.cuh"

namespace wb {
namespace {

constexpr int kThreads = 128;
constexpr int kTile = kPagedTile;  // positions of a KV tile

constexpr int HD = 256;   // dims in shared memory; narrower heads are filled up with zeros
constexpr int kStages = 2;
constexpr int kStage = 2 * kTile * HD;  // elements: K then V

template <int RW, int FRAGS>
constexpr size_t attn_smem_bytes() {
    return (size_t)kStages * kStage * 2 + (size_t)16 * RW * HD * 2 * FRAGS;
}

// ------------------------------------------------------------------------
// Row tile of 16 * RW MMA rows: warp w owns rows 16 * (w % RW) .. and the positions
// (w / RW) * kTile * RW / 4 .. of every KV tile.
// ------------------------------------------------------------------------
template <typename T, bool SPLIT, int RW>
__global__ void __launch_bounds__(kThreads)
paged_attn_kernel(const __grid_constant__ PagedArgs A, int which) {
    constexpr int kS = kStages;
    constexpr int kNP = kTile * RW / 4;       // positions per warp and tile
    constexpr int kNT = kNP / 8;              // score tiles of 8 positions
    constexpr int kRows = SPLIT ? 8 : 16;     // real rows per warp
    constexpr int kF = SPLIT ? PMath<T>::kFrags : 1;  // 16-row fragments that hold a row's parts
    extern __shared__ __align__(128) char smem[];
    T* ring = reinterpret_cast<T*>(smem);
    T* qs = ring + (size_t)kS * kStage;    // [kF][16 * RW][HD], swizzled like the cache rows
    __shared__ int s_pos[16 * RW];            // position of each real row (INT_MIN: no row)
    __shared__ float s_fac[16 * RW];          // SPLIT: the row's power-of-two factor
    __shared__ int s_bad;
    const PagedPlan& P = A.plan[which];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c4 = lane & 3;
    const int rw = warp % RW, pw = warp / RW;
    const int head_lane = blockIdx.x % P.heads, piece = blockIdx.x / P.heads;
    const int kvh = head_lane / P.hblocks, hb = head_lane - kvh * P.hblocks;
    const int h0 = kvh * A.group + hb * P.gpb;             // first query head
    const int gpb = min(P.gpb, A.group - hb * P.gpb);      // query heads of this block

    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    if (tid == 0) {
        s_bad = 0;
        P.bad[blockIdx.x] = 0;
        if (head_lane == 0) P.split[piece] = PagedSplit{0, 0, 0, 0, 0, 0};
    }
    const int n_items = *P.n_items;
    if (n_items == 0) return;
    const int* cum = P.cum;
    const int total = cum[n_items];
    const Pieces pieces(P, total);
    if (piece >= pieces.n) return;
    int x = pieces.start(piece);
    const int x_end = pieces.start(piece + 1);
    int item = block_last_le(cum, n_items, x);  // the item of unit x

    const T* __restrict__ Kc = reinterpret_cast<const T*>(A.k);
    const T* __restrict__ Vc = reinterpret_cast<const T*>(A.v);
    const float sl2 = A.scale_log2;
    constexpr float kShift = PMath<T>::kPShift;

    for (; x < x_end; ++item) {
        const PagedItem it = P.items[item];
        const int c0 = cum[item] + P.lead;
        if (it.n_tiles == 0) continue;
        const int a = max(0, x - c0), b = min(it.n_tiles, x_end - c0);  // KV tiles [a, b)
        x = c0 + max(b, 0);
        if (b <= 0) break;  // the piece ends before the item's first tile
        const bool whole = a == 0 && b == it.n_tiles;
        const int n_rows = it.ntok * gpb;
        if (a == 0 && head_lane == 0) {  // what the join kernels need to know
            if (A.n_groups > 0) {
                const int last = pieces.of(c0 + it.n_tiles - 1);
                for (int i = tid; i < it.ntok; i += kThreads)
                    P.where[it.tok0 + i] = PagedWhere{piece, last, i * P.gpb, it.alone, which, item};
            } else if (!whole && tid == 0) {
                P.split[piece] = PagedSplit{it.tok0, it.ntok * P.gpb,
                                            pieces.of(c0 + it.n_tiles - 1), item, 0, 0};
            }
        }

        __syncthreads();  // the previous item's readers of s_pos / qs / ring are done
        // what some row of the tile sees / what every row sees
        const int any_hi = min(it.kv_hi, it.pmax + 1);
        const int any_lo = A.window > 0 ? it.pmin - A.window + 1 : INT_MIN;
        const int all_hi = min(it.kv_hi, it.pmin + 1);
        const int all_lo = A.window > 0 ? it.pmax - A.window + 1 : INT_MIN;
        const int sinks = A.window > 0 ? A.sinks : 0;

        auto tile_at = [&](int i) { return i < it.n_sink ? it.sink0 + i : it.first + i - it.n_sink; };
        // Where the 16 rows [16 * (warp)) of KV tile i start in the cache, one lane each
        // (elements; -1: no row of the tile sees the position).
        auto row_offset = [&](int i) -> long long {
            const int j = tile_at(i) * kTile + warp * 16 + (lane & 15);
            const bool seen = j >= it.kv_lo && j < any_hi && (j >= any_lo || j < sinks);
            return seen ? page_offset(A, it.seq, j, kvh, &s_bad) : -1;
        };
        auto load_tile = [&](int st, long long off) {
            T* kd = ring + (size_t)st * kStage;
            T* vd = kd + kTile * HD;
#pragma unroll
            for (int rr = 0; rr < 16; ++rr) {  // a row a pass: 32 lanes of 16 bytes
                const long long at = __shfl_sync(0xffffffffu, off, rr);
                const int row = warp * 16 + rr;
                const bool in = at >= 0 && lane * 8 < A.hd;
                const size_t src = in ? (size_t)at + lane * 8 : 0;
                const int dst = row * HD + ((lane ^ (row & 7)) * 8);
                cp16(kd + dst, Kc + src, in);
                cp16(vd + dst, Vc + src, in);
            }
        };

        // ring: kS - 1 tiles ahead; the page of the next tile to load is looked up one
        // iteration before its copies are issued
        long long off = -1;
        for (int u = 0; u < kS - 1; ++u) {
            if (a + u < b) load_tile(u, row_offset(a + u));
            cp_commit();
        }
        if (a + kS - 1 < b) off = row_offset(a + kS - 1);
        // rows of this tile: positions, and q as swizzled 16-bit rows in shared memory
        for (int r = tid; r < 16 * RW; r += kThreads) {
            const int wr = r / 16, rr = r & 15;
            const int row = wr * kRows + rr;
            int pos = INT_MIN;
            if (rr < kRows && row < n_rows) {
                const int t = it.tok0 + row / gpb;
                pos = it.mixed ? token_position(A, t) : it.pos0 + row / gpb;
            }
            s_pos[r] = pos;
        }
        load_rows<T, SPLIT, HD, RW, kThreads>(A, it.tok0, n_rows, h0, gpb, qs, s_fac);
        __syncthreads();

        const int prow[2] = {s_pos[rw * 16 + g], SPLIT ? INT_MIN : s_pos[rw * 16 + g + 8]};
        int hi_row[2], lo_row[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            hi_row[u] = prow[u] == INT_MIN ? 0 : min(it.kv_hi, prow[u] + 1);
            lo_row[u] = A.window > 0 && prow[u] != INT_MIN ? prow[u] - A.window + 1 : INT_MIN;
        }
        const float fac = SPLIT ? s_fac[rw * 16 + g] * sl2 : sl2;
        auto load_q = [&](int n, int kk, uint32_t (&f)[4]) {
            const int r = rw * 16 + (lane & 15), c = kk * 2 + (lane >> 4);
            ldsm4(f, qs + (size_t)(n * 16 * RW + r) * HD + ((c ^ (r & 7)) * 8));
        };
        float o[HD / 8][4];
#pragma unroll
        for (int i = 0; i < HD / 8; ++i)
#pragma unroll
            for (int u = 0; u < 4; ++u) o[i][u] = 0.f;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

        int st = 0;
        for (int i = a; i < b; ++i) {
            cp_wait<kS - 2>();
            __syncthreads();
            {
                const int ld = st == 0 ? kS - 1 : st - 1;
                if (i + kS - 1 < b) load_tile(ld, off);
                cp_commit();
                if (i + kS < b) off = row_offset(i + kS);
            }
            const T* kd = ring + (size_t)st * kStage;
            const T* vd = kd + kTile * HD;
            st = st + 1 == kS ? 0 : st + 1;
            const int j0 = tile_at(i) * kTile, jw = j0 + pw * kNP;
            const bool full = jw >= it.kv_lo && jw + kNP <= all_hi &&
                              (jw >= all_lo || jw + kNP <= sinks);

            float s[kNT][4];
#pragma unroll
            for (int t = 0; t < kNT; ++t)
#pragma unroll
                for (int u = 0; u < 4; ++u) s[t][u] = 0.f;
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk) {
                uint32_t qv[kF][4];
#pragma unroll
                for (int n = 0; n < kF; ++n) load_q(n, kk, qv[n]);
#pragma unroll
                for (int t = 0; t < kNT; t += 2) {
                    const int r = pw * kNP + t * 8 + ((lane >> 4) & 1) * 8 + (lane & 7);
                    const int c = kk * 2 + ((lane >> 3) & 1);
                    uint32_t kf[4];
                    ldsm4(kf, kd + (size_t)r * HD + ((c ^ (r & 7)) * 8));
#pragma unroll
                    for (int n = 0; n < kF; ++n) {
                        PMath<T>::mma(s[t], qv[n], kf[0], kf[1]);
                        PMath<T>::mma(s[t + 1], qv[n], kf[2], kf[3]);
                    }
                }
            }
            // scores in log2 units, masked; the row maxima
            float mx[2] = {m[0], m[1]};
#pragma unroll
            for (int t = 0; t < kNT; ++t)
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    if (SPLIT && u >= 2) continue;
                    float v = SPLIT ? (s[t][u] + s[t][u + 2 < 4 ? u + 2 : u]) * fac : s[t][u] * sl2;
                    if (!full) {
                        const int j = jw + t * 8 + c4 * 2 + (u & 1);
                        if (!(j >= it.kv_lo && j < hi_row[u >> 1] &&
                              (j >= lo_row[u >> 1] || j < sinks)))
                            v = -INFINITY;
                    }
                    s[t][u] = v;
                    mx[u >> 1] = fmaxf(mx[u >> 1], v);
                }
            float al[2], mb[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                mx[u] = fmaxf(mx[u], __shfl_xor_sync(0xffffffffu, mx[u], 1));
                mx[u] = fmaxf(mx[u], __shfl_xor_sync(0xffffffffu, mx[u], 2));
                const float base = mx[u] == -INFINITY ? 0.f : mx[u];
                al[u] = ex2(m[u] - base);
                mb[u] = base - kShift;
                m[u] = mx[u];
                l[u] *= al[u];
            }
#pragma unroll
            for (int t = 0; t < kNT; ++t)
#pragma unroll
                for (int u = 0; u < (SPLIT ? 2 : 4); ++u) {
                    s[t][u] = ex2(s[t][u] - mb[u >> 1]);
                    l[u >> 1] += s[t][u];
                }
            if (al[0] != 1.f || (!SPLIT && al[1] != 1.f)) {
#pragma unroll
                for (int d = 0; d < HD / 8; ++d)
#pragma unroll
                    for (int u = 0; u < 4; ++u) o[d][u] *= SPLIT ? al[0] : al[u >> 1];
            }
            // Rows that see different positions of one tile: what is hidden from one may be an
            // infinity or a NaN that another sees.  Such values are looked for first (rare), so
            // that the usual loop stays short.
            bool odd = false;
            if (!full && it.pmin != it.pmax) {
                for (int i = lane; i < kNP * HD / 8; i += 32) {
                    const uint4 w = *reinterpret_cast<const uint4*>(vd + (size_t)pw * kNP * HD + i * 8);
                    odd |= PMath<T>::not_finite(w.x) || PMath<T>::not_finite(w.y) ||
                           PMath<T>::not_finite(w.z) || PMath<T>::not_finite(w.w);
                }
                odd = __any_sync(0xffffffffu, odd);
            }
            auto weigh = [&](auto special) {
#pragma unroll
                for (int kk = 0; kk < kNP / 16; ++kk) {
                    uint32_t pf[kF][4];
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        float(&w)[4] = s[2 * kk + t];
                        if (!SPLIT) {
                            pf[0][2 * t] = PMath<T>::pack(w[0], w[1]);
                            pf[0][2 * t + 1] = PMath<T>::pack(w[2], w[3]);
                        } else {
                            PMath<T>::split(w[0], w[1], pf[0][2 * t], pf[0][2 * t + 1],
                                            pf[kF - 1][2 * t]);
                            if (kF == 2) pf[kF - 1][2 * t + 1] = 0;
                        }
                    }
                    uint32_t one[4];  // visible places of the 16 x 16 block of weights as ones
                    if (decltype(special)::value) {
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            one[u] = 0;
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const int j = jw + kk * 16 + (u >> 1) * 8 + c4 * 2 + e;
                                if (j >= it.kv_lo && j < hi_row[u & 1] &&
                                    (j >= lo_row[u & 1] || j < sinks))
                                    one[u] |= PMath<T>::kOne << (16 * e);
                            }
                        }
                    }
#pragma unroll
                    for (int d = 0; d < HD / 8; d += 2) {
                        const int r = pw * kNP + kk * 16 + ((lane >> 3) & 1) * 8 + (lane & 7);
                        const int c = d + (lane >> 4);
                        uint32_t vf[4];
                        ldsm4t(vf, vd + (size_t)r * HD + ((c ^ (r & 7)) * 8));
                        if (decltype(special)::value) {
#pragma unroll
                            for (int n = 0; n < 2; ++n) {
                                SpecialFrag f{{o[d + n][0], o[d + n][1], o[d + n][2], o[d + n][3]},
                                              vf[2 * n], vf[2 * n + 1]};
                                f = specials<T>(f, one[0], one[1], one[2], one[3]);
#pragma unroll
                                for (int u = 0; u < 4; ++u) o[d + n][u] = f.o[u];
                                vf[2 * n] = f.b0;
                                vf[2 * n + 1] = f.b1;
                            }
                        }
                        add_products<T, SPLIT, kF>(o[d], o[d + 1], pf, vf);
                    }
                }
            };
            if (odd) weigh(Flag<true>());
            else weigh(Flag<false>());
        }
        cp_wait<0>();
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            l[u] += __shfl_xor_sync(0xffffffffu, l[u], 1);
            l[u] += __shfl_xor_sync(0xffffffffu, l[u], 2);
        }

        // join the warps that read other positions of the same rows (shared memory, fp32)
        if (RW < 4) {
            __syncthreads();
            float* xo = reinterpret_cast<float*>(smem);           // [4 / RW][16 * RW][HD]
            float* xm = xo + (size_t)(4 / RW) * 16 * RW * HD;     // [4 / RW][16 * RW][2]
#pragma unroll
            for (int u = 0; u < (SPLIT ? 1 : 2); ++u) {
                const int r = rw * 16 + g + 8 * u;
                float* dst = xo + ((size_t)pw * 16 * RW + r) * HD;
#pragma unroll
                for (int d = 0; d < HD / 8; ++d) {
                    const float2 v = SPLIT ? make_float2(o[d][0] + o[d][2], o[d][1] + o[d][3])
                                           : make_float2(o[d][2 * u], o[d][2 * u + 1]);
                    *reinterpret_cast<float2*>(dst + d * 8 + c4 * 2) = v;
                }
                if (c4 == 0) {
                    xm[(pw * 16 * RW + r) * 2] = m[u];
                    xm[(pw * 16 * RW + r) * 2 + 1] = l[u];
                }
            }
            __syncthreads();
            // warp w joins rows w, w + 4, ...
            for (int r = warp; r < 16 * RW; r += 4) {
                const int row = (r / 16) * kRows + (r & 15);
                if ((r & 15) >= kRows || row >= n_rows) continue;
                float M = -INFINITY;
#pragma unroll
                for (int w = 0; w < 4 / RW; ++w) M = fmaxf(M, xm[(w * 16 * RW + r) * 2]);
                const float base = M == -INFINITY ? 0.f : M;
                float e[4 / RW], L = 0.f;
#pragma unroll
                for (int w = 0; w < 4 / RW; ++w) {
                    e[w] = ex2(xm[(w * 16 * RW + r) * 2] - base);
                    L += xm[(w * 16 * RW + r) * 2 + 1] * e[w];
                }
                RowOut<T, SPLIT> R(A, P, which, it, piece, head_lane, h0, gpb, row, a, whole);
                for (int d = lane * 2; d < A.hd; d += 64) {
                    float2 acc = make_float2(0.f, 0.f);
#pragma unroll
                    for (int w = 0; w < 4 / RW; ++w) {
                        const float2 v = *reinterpret_cast<const float2*>(
                            xo + ((size_t)w * 16 * RW + r) * HD + d);
                        acc.x = fmaf(v.x, e[w], acc.x);
                        acc.y = fmaf(v.y, e[w], acc.y);
                    }
                    R.put2(d, acc, L);
                }
                if (lane == 0) R.put_ml(M - kShift, L);
            }
        } else {
#pragma unroll
            for (int u = 0; u < (SPLIT ? 1 : 2); ++u) {
                const int row = rw * kRows + g + 8 * u;
                if (row >= n_rows) continue;
                RowOut<T, SPLIT> R(A, P, which, it, piece, head_lane, h0, gpb, row, a, whole);
#pragma unroll
                for (int d = 0; d < HD / 8; ++d) {
                    if (d * 8 >= A.hd) break;
                    const float2 v = SPLIT ? make_float2(o[d][0] + o[d][2], o[d][1] + o[d][3])
                                           : make_float2(o[d][2 * u], o[d][2 * u + 1]);
                    R.put2(d * 8 + c4 * 2, v, l[u]);
                }
                if (c4 == 0) R.put_ml(m[u] - kShift, l[u]);
            }
        }
    }
    __syncthreads();
    if (tid == 0 && s_bad) P.bad[blockIdx.x] = s_bad;
}

// ------------------------------------------------------------------------
// Joins the pieces of split items.  CTA (piece, block of heads, ...): the item that begins in the
// piece and ends after it.  Items that the tensor-core kernel marked are worked out here without
// tiles.
// ------------------------------------------------------------------------
struct JoinPlace {
    int piece, head_lane, h0, gpb;
    __device__ __forceinline__ JoinPlace(const PagedArgs& A, const PagedPlan& P) {
        head_lane = blockIdx.x % P.heads;
        piece = blockIdx.x / P.heads;
        const int kvh = head_lane / P.hblocks, hb = head_lane - kvh * P.hblocks;
        h0 = kvh * A.group + hb * P.gpb;
        gpb = min(P.gpb, A.group - hb * P.gpb);
    }
};

// By the whole CTA: the marked ones of the items whose first KV tile lies in the piece.
template <typename T, bool SPLIT>
__device__ __forceinline__ void join_marked(const PagedArgs& A, const PagedPlan& P,
                                            const PagedSplit& sp, const JoinPlace& at) {
    int marked = 0;
    for (int i = sp.item0 + (int)threadIdx.x; i < sp.item1; i += kJoinThreads)
        marked |= P.redo[(size_t)i * P.heads + at.head_lane];
    if (!__syncthreads_or(marked)) return;
    for (int i = sp.item0; i < sp.item1; ++i) {
        if (!P.redo[(size_t)i * P.heads + at.head_lane]) continue;
        const PagedItem it = P.items[i];
        for (int r = threadIdx.x / 32; r < it.ntok * at.gpb; r += kJoinThreads / 32) {
            Joined<4> J;
            J.restate<T, SPLIT>(A, it.tok0 + r / at.gpb, at.h0 + r % at.gpb);
            J.write<T, SPLIT>(A, it.tok0 + r / at.gpb, at.h0 + r % at.gpb);
        }
    }
}

// Rows of tokens that no sequence owns, as of rows that see nothing: [0, lo) and [hi, n_tokens), by
// the CTAs of the first row.
struct Owned {
    int lo, hi;
    __device__ __forceinline__ explicit Owned(const PagedArgs& A) {
        lo = min(max(A.q_start[0], 0), A.n_tokens);
        hi = min(max(A.q_start[A.n_seq], lo), A.n_tokens);
    }
};
template <bool SPLIT>
__device__ __forceinline__ void clear_rest(const PagedArgs& A, const Owned& own) {
    const int rest = A.n_tokens - (own.hi - own.lo), size = SPLIT ? 4 : 2;
    for (int i = blockIdx.x; i < rest; i += gridDim.x) {
        const size_t t = i < own.lo ? i : own.hi + (i - own.lo);
        uint4* row = reinterpret_cast<uint4*>(static_cast<char*>(A.out) + t * A.out_stride * size);
        for (int d = threadIdx.x; d < A.nh * A.hd * size / 16; d += kJoinThreads)
            row[d] = make_uint4(0, 0, 0, 0);
        for (int h = threadIdx.x; A.lse && h < A.nh; h += kJoinThreads)
            A.lse[t * A.nh + h] = -INFINITY;
    }
}

// Items of few rows, usually in many pieces: two rows a CTA, four warps per row take every fourth
// piece, in batches whose loads are in flight together, and meet in shared memory in their order.
template <typename T, bool SPLIT, int VECS>
__global__ void __launch_bounds__(kJoinThreads)
paged_join_kernel(const __grid_constant__ PagedArgs A, int which) {
    __shared__ JoinShared<VECS> S;
    constexpr int kWarps = 4, kRows = 2;
    const PagedPlan& P = A.plan[which];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (blockIdx.x == 0 && blockIdx.y == 0) gather_status(A);
    const JoinPlace at(A, P);
    const Owned own(A);
    const PagedSplit sp = P.split[at.piece];
    if (blockIdx.y == 0) clear_rest<SPLIT>(A, own);
    if (P.redo && blockIdx.y == 0) join_marked<T, SPLIT>(A, P, sp, at);
    const int n_rows = sp.n_rows / P.gpb * at.gpb;  // (counted with full blocks of heads)
    if ((int)blockIdx.y * kRows >= n_rows) return;
    if (P.redo && P.redo[(size_t)sp.item * P.heads + at.head_lane]) return;
    const int warp = threadIdx.x / 32, row = blockIdx.y * kRows + warp / kWarps;
    Joined<VECS> J;
    J.init();
    if (row < n_rows) J.add_range(A, P, at.piece, sp.last, at.head_lane, row, warp % kWarps, kWarps);
    J.meet(S, warp % kWarps, kWarps);
    if (row < n_rows && warp % kWarps == 0)
        J.template write<T, SPLIT>(A, sp.tok0 + row / at.gpb, at.h0 + row % at.gpb);
}

// Items of many rows, mostly in two pieces: a thread takes four dims of two rows and two pieces at a
// time, so that all lanes load whatever the head's size.  Measured (B200): ragged chunks of 7652
// tokens, 16 heads of 64, 121 us a call against 133 us with a warp per row and four pieces in
// flight (80 registers, eight rows a CTA); four rows or four pieces at a time 124 to 125 us.
constexpr int kJoinRows = 2, kJoinBatch = 2;
template <typename T, bool SPLIT>
__global__ void __launch_bounds__(kJoinThreads)
paged_join_rows_kernel(const __grid_constant__ PagedArgs A, int which) {
    const PagedPlan& P = A.plan[which];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (blockIdx.x == 0 && blockIdx.y == 0) gather_status(A);
    const JoinPlace at(A, P);
    const Owned own(A);
    const PagedSplit sp = P.split[at.piece];
    if (blockIdx.y == 0) clear_rest<SPLIT>(A, own);
    if (P.redo && blockIdx.y == 0) join_marked<T, SPLIT>(A, P, sp, at);
    const int n_rows = sp.n_rows / P.gpb * at.gpb, quads = A.hd / 4;
    const int e0 = blockIdx.y * (kJoinRows * kJoinThreads) + threadIdx.x;
    if (e0 >= n_rows * quads) return;
    if (P.redo && P.redo[(size_t)sp.item * P.heads + at.head_lane]) return;
    int row[kJoinRows], d[kJoinRows];
    float M[kJoinRows], L[kJoinRows];
    float4 acc[kJoinRows];
#pragma unroll
    for (int u = 0; u < kJoinRows; ++u) {
        const int e = min(e0 + u * kJoinThreads, n_rows * quads - 1);
        row[u] = e / quads;
        d[u] = (e - row[u] * quads) * 4;
        M[u] = -INFINITY;
        L[u] = 0.f;
        acc[u] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (int p = at.piece; p <= sp.last; p += kJoinBatch) {
        float4 v[kJoinRows][kJoinBatch];
        float2 w[kJoinRows][kJoinBatch];
#pragma unroll
        for (int u = 0; u < kJoinRows; ++u)
#pragma unroll
            for (int k = 0; k < kJoinBatch; ++k) {
                v[u][k] = make_float4(0.f, 0.f, 0.f, 0.f);
                w[u][k] = make_float2(-INFINITY, 0.f);
                if (p + k > sp.last) continue;
                const size_t id = part_row(P, p + k, at.head_lane, p + k == at.piece, row[u]);
                v[u][k] = __ldcg(reinterpret_cast<const float4*>(P.part_o + id * A.hd + d[u]));
                w[u][k] = __ldcg(reinterpret_cast<const float2*>(P.part_ml + id * 2));
            }
#pragma unroll
        for (int u = 0; u < kJoinRows; ++u) {
            float to = M[u];
#pragma unroll
            for (int k = 0; k < kJoinBatch; ++k) to = fmaxf(to, w[u][k].x);
            const float base = to == -INFINITY ? 0.f : to, old = ex2(M[u] - base);
            M[u] = to;
            L[u] *= old;
            acc[u].x *= old, acc[u].y *= old, acc[u].z *= old, acc[u].w *= old;
#pragma unroll
            for (int k = 0; k < kJoinBatch; ++k) {
                if (p + k > sp.last) break;
                const float e = ex2(w[u][k].x - base);
                L[u] = fmaf(w[u][k].y, e, L[u]);
                acc[u].x = fmaf(v[u][k].x, e, acc[u].x);
                acc[u].y = fmaf(v[u][k].y, e, acc[u].y);
                acc[u].z = fmaf(v[u][k].z, e, acc[u].z);
                acc[u].w = fmaf(v[u][k].w, e, acc[u].w);
            }
        }
    }
#pragma unroll
    for (int u = 0; u < kJoinRows; ++u) {
        if (e0 + u * kJoinThreads >= n_rows * quads) break;
        const int t = sp.tok0 + row[u] / at.gpb, h = at.h0 + row[u] % at.gpb;
        const size_t to = (size_t)t * A.out_stride + (size_t)h * A.hd + d[u];
        const float inv = 1.f / L[u];
        const float4 o = L[u] == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f)
                                     : make_float4(acc[u].x * inv, acc[u].y * inv, acc[u].z * inv,
                                                   acc[u].w * inv);
        if (SPLIT)
            *reinterpret_cast<float4*>(reinterpret_cast<float*>(A.out) + to) = o;
        else
            *reinterpret_cast<uint2*>(reinterpret_cast<T*>(A.out) + to) =
                make_uint2(PMath<T>::pack(o.x, o.y), PMath<T>::pack(o.z, o.w));
        if (d[u] == 0 && A.lse) A.lse[(size_t)t * A.nh + h] = row_lse(M[u], L[u]);
    }
}

// Prefix mode: CTA (token, two of its heads), over the records of the shared prefix and of the
// sequence's own part: pieces, or one whole record.
// (Both parts' records in one batch of loads: 64 sequences behind 32768 and 16384 positions 102 us a
// call, one part after the other with room for 256 dims 107 us.)
template <typename T, bool SPLIT, int VECS>
__global__ void __launch_bounds__(kJoinThreads)
paged_join2_kernel(const __grid_constant__ PagedArgs A) {
    __shared__ JoinShared<VECS> S;
    constexpr int kWarps = 4, kRows = 2, kBatch = 4;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (blockIdx.x == 0 && blockIdx.y == 0) gather_status(A);
    const int t = blockIdx.x, warp = threadIdx.x / 32 % kWarps;
    const int h = blockIdx.y * kRows + threadIdx.x / 32 / kWarps;
    const bool owned = t >= A.q_start[0] && t < A.q_start[A.n_seq];  // (else: zeros)
    Joined<VECS> J;
    J.init();
    bool redo = false;
    if (h < A.nh && owned) {
        PagedWhere w[2] = {A.plan[A.plan[PLAN_FEW].used ? PLAN_FEW : PLAN_MANY].where[t],
                           A.plan[PLAN_PREFIX].where[t]};
        const int kvh = h / A.group, hg = h - kvh * A.group;
        int n[2], lane[2], row[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            n[k] = 0;
            if ((k && w[0].alone) || w[k].plan < 0 || w[k].plan >= PLANS) continue;
            const PagedPlan& P = A.plan[w[k].plan];
            const int hb = hg / P.gpb, gpb = min(P.gpb, A.group - hb * P.gpb);
            lane[k] = kvh * P.hblocks + hb;
            row[k] = w[k].row0 / P.gpb * gpb + hg - hb * P.gpb;
            // (a malformed q_start leaves tokens without a record)
            if (w[k].first < 0 || w[k].last < w[k].first || w[k].last >= P.lanes || row[k] < 0 ||
                row[k] >= P.rows || w[k].item < 0 || w[k].item >= P.max_items)
                continue;
            if (P.redo && P.redo[(size_t)w[k].item * P.heads + lane[k]]) redo = true;
            n[k] = w[k].last - w[k].first + 1;
        }
        for (int i = warp; i < n[0] + n[1]; i += kBatch * kWarps) {
            const float *o[kBatch], *ml[kBatch];
            int have = 0;
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const int j = min(i + b * kWarps, n[0] + n[1] - 1), k = j >= n[0];
                const PagedPlan& P = A.plan[k ? w[1].plan : w[0].plan];
                const int c = k ? n[1] : n[0], first = k ? w[1].first : w[0].first;
                const int p = first + (k ? j - n[0] : j);
                const size_t id =
                    c == 1 ? (size_t)k * A.n_tokens * A.nh + (size_t)t * A.nh + h
                           : part_row(P, p, k ? lane[1] : lane[0], p == first, k ? row[1] : row[0]);
                o[b] = (c == 1 ? A.full_o : P.part_o) + id * A.hd;
                ml[b] = (c == 1 ? A.full_ml : P.part_ml) + id * 2;
                have += i + b * kWarps < n[0] + n[1];
            }
            J.template add<kBatch>(A, o, ml, have);
        }
    }
    J.meet(S, warp, kWarps);
    if (h < A.nh && warp == 0) {
        if (redo) J.template restate<T, SPLIT>(A, t, h);
        J.template write<T, SPLIT>(A, t, h);
    }
}

template <typename T, bool SPLIT, int RW>
cudaError_t launch_one(const PagedArgs& A, int which, cudaStream_t s) {
    auto kern = paged_attn_kernel<T, SPLIT, RW>;
    constexpr size_t smem = attn_smem_bytes<RW, SPLIT ? PMath<T>::kFrags : 1>();
    static std::atomic<uint64_t> done{0};
    cudaError_t e = smem_opt_in(reinterpret_cast<const void*>(kern), smem, done);
    if (e != cudaSuccess) return e;
    const PagedPlan& P = A.plan[which];
    return launch_pdl(kern, dim3(P.heads * P.lanes), dim3(kThreads), smem, s, A, which);
}

template <typename T, bool SPLIT>
cudaError_t launch_rw(const PagedArgs& A, int which, int rw, cudaStream_t s) {
    return rw == 2 ? launch_one<T, SPLIT, 2>(A, which, s) : launch_one<T, SPLIT, 4>(A, which, s);
}

template <typename T, bool SPLIT, int VECS>
cudaError_t launch_join(const PagedArgs& A, cudaStream_t s) {
    if (A.n_groups > 0)
        return launch_pdl(paged_join2_kernel<T, SPLIT, VECS>, dim3(A.n_tokens, (A.nh + 1) / 2),
                          dim3(kJoinThreads), 0, s, A);
    const int w = A.plan[PLAN_FEW].used ? PLAN_FEW : PLAN_MANY;
    const PagedPlan& P = A.plan[w];
    if (P.used_rows <= 32)
        return launch_pdl(paged_join_kernel<T, SPLIT, VECS>,
                          dim3(P.heads * P.lanes, (P.used_rows + 1) / 2), dim3(kJoinThreads), 0, s, A,
                          w);
    constexpr int kPer = kJoinRows * kJoinThreads;
    return launch_pdl(paged_join_rows_kernel<T, SPLIT>,
                      dim3(P.heads * P.lanes, (P.used_rows * (A.hd / 4) + kPer - 1) / kPer),
                      dim3(kJoinThreads), 0, s, A, w);
}

}  // namespace

// 16-row MMA tiles of a row tile with `rows` rows: two take half the registers and the sums, four
// read the cache half as often.  Measured (B200, 8 sequences of 8192, 8 kv heads of 256): 32 rows
// 153 us with two and 235 us with four, 64 rows 272 and 246 us, 128 rows 512 and 437 us.
int paged_attn_rw(int rows, bool split) { return rows <= (split ? 16 : 32) ? 2 : 4; }

// CTAs of one SM: what the ring leaves room for.
int paged_attn_ctas() { return 1; }

cudaError_t launch_paged_attn(const PagedArgs& A, int which, int rw, int q_dtype, int kv_dtype,
                              cudaStream_t s) {
    const bool split = q_dtype == WISP_DTYPE_F32;
    if (kv_dtype == WISP_DTYPE_F16)
        return split ? launch_rw<__half, true>(A, which, rw, s)
                     : launch_rw<__half, false>(A, which, rw, s);
    return split ? launch_rw<__nv_bfloat16, true>(A, which, rw, s)
                 : launch_rw<__nv_bfloat16, false>(A, which, rw, s);
}

cudaError_t launch_paged_join(const PagedArgs& A, int q_dtype, int kv_dtype, cudaStream_t s) {
    const bool split = q_dtype == WISP_DTYPE_F32, wide = A.hd > 128;
    auto go = [&](auto t) {
        using T = decltype(t);
        return split ? (wide ? launch_join<T, true, 4>(A, s) : launch_join<T, true, 2>(A, s))
                     : (wide ? launch_join<T, false, 4>(A, s) : launch_join<T, false, 2>(A, s));
    };
    return kv_dtype == WISP_DTYPE_F16 ? go(__half{}) : go(__nv_bfloat16{});
}

}  // namespace wb
