// paged_few.cu -- attention of row tiles with few rows (single tokens, a few drafted ones, few
// sequences behind a prefix): one 16-row tile of mma.sync per kv head, bound by the cache's HBM
// reads.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = 2^(log2(e) scale q_i . k_j - m_i)
//
// A CTA streams its piece of the line of KV tiles (64 positions, one kv head) through a ring of
// cp.async stages that does not stop at the end of a row tile: the next one's rows of q and its
// first positions are on their way while the last tiles of this one are worked on.  Per tile,
// each of the four warps scores 16 of the positions; the row maxima and the weights go through
// shared memory, and then each warp adds all 64 weighted positions to a quarter of the head's
// dims.  (The first form had each warp keep all dims for its own positions: 64 accumulators a
// thread, a join of four 16 x head_dim tiles per row tile, and a ring that drained there.)
//
// 32-bit rows are split into 16-bit parts (two in fp16, 22 bits, three in bf16) that share the
// 16 rows of a fragment, 8 rows each; their sums meet in one thread.  The weights are split the
// same way.  In fp16 they carry 2^kPShift, which cancels, so that small weights of long caches
// stay above the subnormals.

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "internal.h"
#include "paged.h"
#include "paged_math.cuh"

namespace wb {
namespace {

constexpr int kThreads = 128;
constexpr int kTile = 64;
constexpr int kRecs = 16;

template <typename T, bool SPLIT, int HD>
struct FCfg {
    static constexpr int kF = SPLIT ? PMath<T>::kFrags : 1;  // 16-row fragments of a row's parts
    static constexpr int kStages = HD == 64 ? 4 : HD == 128 && kF == 1 ? 3 : 2;
    static constexpr int kCtas = HD == 64 ? 3 : HD == 128 ? 2 : 1;
    static constexpr int kStage = 2 * kTile * HD;                  // elements: K then V
    static constexpr int kQBytes = SPLIT ? 8 * HD * 4 : 16 * HD * 2;  // a row tile's q as it is
    // converted q (fp32 rows only) or the tile's weights
    static constexpr int kWork = std::max(kF * 16 * kTile, SPLIT ? kF * 16 * HD : 0);
    static constexpr size_t kSmem = (size_t)kStages * kStage * 2 + 2 * kQBytes + (size_t)kWork * 2;
};

struct Rec {  // a row tile of this piece and its KV tiles [a, b); b < 0: there are no more
    PagedItem it;
    int a, b;
    int item, c0;
};

template <typename T, bool SPLIT, int HD>
__global__ void __launch_bounds__(kThreads, (FCfg<T, SPLIT, HD>::kCtas))
paged_few_kernel(const __grid_constant__ PagedArgs A, int which0) {
    using C = FCfg<T, SPLIT, HD>;
    constexpr int kF = C::kF, kS = C::kStages, kCh = HD / 8, kRows = SPLIT ? 8 : 16;
    constexpr int kDW = HD / 4;  // dims of a warp
    constexpr float kShift = PMath<T>::kPShift;
    extern __shared__ __align__(128) char smem[];
    T* ring = reinterpret_cast<T*>(smem);
    char* qraw = smem + (size_t)kS * C::kStage * 2;
    T* work = reinterpret_cast<T*>(qraw + 2 * C::kQBytes);
    __shared__ Rec s_rec[kRecs], s_cur[2];
    __shared__ int s_cum[kPagedInline + 1];
    __shared__ int s_sum[4], s_bad, s_pos[16];
    __shared__ float s_fac[16], s_max[4][16], s_l[4][16];
    const int which = blockIdx.y ? PLAN_PREFIX : which0;
    const PagedPlan& P = A.plan[which];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c4 = lane & 3;
    const int head_lane = blockIdx.x % P.heads, piece = blockIdx.x / P.heads;
    const int kvh = head_lane / P.hblocks, hb = head_lane - kvh * P.hblocks;
    const int h0 = kvh * A.group + hb * P.gpb, gpb = min(P.gpb, A.group - hb * P.gpb);

    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    const bool inlined = P.inlined != 0, prefix = which == PLAN_PREFIX;
    if (tid == 0) {
        s_bad = 0;
        P.bad[blockIdx.x] = 0;
        if (head_lane == 0) P.split[piece] = PagedSplit{0, 0, 0, 0, 0, 0};
        if (inlined && blockIdx.x == 0) P.bad[P.lanes * P.heads] = 0;
    }
    const int n_items = inlined ? (prefix ? A.n_groups : A.n_seq) : *P.n_items;
    if (n_items == 0) return;
    const int* cum = inlined ? s_cum : P.cum;
    if (inlined) {
        // one row tile per segment: every CTA counts the units itself, which is shorter than a
        // kernel of its own before this one
        __syncthreads();  // the words above are cleared
        int carry = 0;
        for (int base = 0; base < n_items; base += kThreads) {
            const int i = base + tid;
            int n = 0;
            if (i < n_items) {
                n = item_units(P, make_item(A, P, prefix, i, 0).n_tiles);
                if (blockIdx.x == 0 && !prefix) {
                    const int t = A.q_start[i + 1] - A.q_start[i];
                    if (length_too_long(A, i) || (t > P.tpt && t <= P.max_tok))
                        P.bad[P.lanes * P.heads] = PG_BAD_LENGTH;
                }
            }
            int v = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v += y;
            }
            if (lane == 31) s_sum[warp] = v;
            __syncthreads();
            int before = carry;
            for (int w = 0; w < 4; ++w) {
                if (w < warp) before += s_sum[w];
                carry += s_sum[w];
            }
            if (i < n_items) s_cum[i] = before + v - n;
            __syncthreads();
        }
        if (tid == 0) s_cum[n_items] = carry;
        __syncthreads();
    }
    const int total = cum[n_items];
    const Pieces pieces(P, max(total, 1));
    if (total == 0 || piece >= pieces.n) return;
    const int x0 = pieces.start(piece), x_end = pieces.start(piece + 1);
    const int item0 = block_last_le(cum, n_items, x0);

    const T* __restrict__ Kc = reinterpret_cast<const T*>(A.k);
    const T* __restrict__ Vc = reinterpret_cast<const T*>(A.v);
    const int sinks = A.window > 0 ? A.sinks : 0;

    // ---------------------------------------------------------------- what comes next
    // Records of this piece, kRecs at a time; the loading side walks them (all threads alike).
    int lk = 0, li = 0, lq = 0;  // record, next tile of it, row tiles begun
    int issued = 0;              // tiles whose copies were issued
    bool have = false;           // there is a next tile, with
    long long off = -1;          // the cache offset of this lane's row of it (-1: unseen)
    auto fill = [&]() {
        if (tid < kRecs) {
            Rec r;
            r.b = -1;
            r.a = 0;
            r.item = item0 + lk + tid;
            if (r.item < n_items && cum[r.item] < x_end) {
                r.it = inlined ? make_item(A, P, prefix, r.item, 0) : P.items[r.item];
                r.c0 = cum[r.item] + P.lead;
                r.a = max(0, x0 - r.c0);
                r.b = max(0, min(r.it.n_tiles, x_end - r.c0));
            }
            s_rec[tid] = r;
        }
        __syncthreads();
    };
    auto look = [&]() {  // to the next tile that exists
        const Rec* r = &s_rec[lk % kRecs];
        while (r->b >= 0 && li >= r->b) {
            ++lk;
            if (lk % kRecs == 0) {
                __syncthreads();
                fill();
            }
            r = &s_rec[lk % kRecs];
            li = r->a;
            if (r->b > r->a) ++lq;
        }
        have = r->b >= 0;
        if (!have) return;
        const PagedItem& it = r->it;
        const int t = li < it.n_sink ? it.sink0 + li : it.first + li - it.n_sink;
        const int j = t * kTile + warp * 16 + (lane & 15);
        const int any_hi = min(it.kv_hi, it.pmax + 1);
        const int any_lo = A.window > 0 ? it.pmin - A.window + 1 : INT_MIN;
        const bool seen = j >= it.kv_lo && j < any_hi && (j >= any_lo || j < sinks);
        off = seen ? page_offset(A, it.seq, j, kvh, &s_bad) : -1;
    };
    auto issue = [&]() {
        const Rec& r = s_rec[lk % kRecs];
        if (li == r.a) {  // the row tile's record and rows travel with its first positions
            if (tid == 0) s_cur[lq & 1] = r;
            char* dst = qraw + (lq & 1) * C::kQBytes;
            constexpr int kPer = SPLIT ? HD / 4 : HD / 8;  // 16-byte pieces of a row
            const int n_rows = r.it.ntok * gpb;
            for (int i = tid; i < n_rows * kPer; i += kThreads) {
                const int row = i / kPer, c = i - row * kPer;
                const size_t at = (size_t)(r.it.tok0 + row / gpb) * A.q_stride +
                                  (size_t)(h0 + row % gpb) * A.hd;
                if (SPLIT) {
                    const bool in = c * 4 < A.hd;
                    cp16(dst + row * HD * 4 + c * 16,
                         reinterpret_cast<const float*>(A.q) + (in ? at + c * 4 : 0), in);
                } else {
                    const bool in = c * 8 < A.hd;
                    cp16(dst + row * HD * 2 + ((c ^ (row & 7)) * 16),
                         reinterpret_cast<const T*>(A.q) + (in ? at + c * 8 : 0), in);
                }
            }
        }
        T* kd = ring + (size_t)(issued % kS) * C::kStage;
        T* vd = kd + kTile * HD;
        constexpr int kPer = kCh >= 32 ? 1 : 32 / kCh;  // rows per pass of the warp
#pragma unroll
        for (int p = 0; p < 16 / kPer; ++p) {
            const int rr = p * kPer + (kCh >= 32 ? 0 : lane / kCh);
            const long long o = __shfl_sync(0xffffffffu, off, rr);
            const int row = warp * 16 + rr, c = kCh >= 32 ? lane : lane % kCh;
            const bool in = o >= 0 && c * 8 < A.hd;
            const size_t src = in ? (size_t)o + c * 8 : 0;
            const int to = row * HD + ((c ^ (row & 7)) * 8);
            cp16(kd + to, Kc + src, in);
            cp16(vd + to, Vc + src, in);
        }
        ++issued;
        ++li;
        look();
    };

    fill();
    li = s_rec[0].a;
    if (s_rec[0].b > s_rec[0].a) lq = 1;
    look();
    int cq = 0, done = 0, end = 0;  // row tiles begun, tiles worked on, tile that ends this one
    // Copy group c holds tile c while one tile is issued per iteration; where it was not (at most
    // one row tile is fetched ahead), the next `loose` iterations wait for all groups.
    int loose = 0;
#pragma unroll
    for (int u = 0; u < kS - 1; ++u) {
        if (have && lq <= cq + 1) issue();
        else if (have) loose = kS;
        cp_commit();
    }

    Rec cur;
    int hi_row[2] = {0, 0}, lo_row[2] = {INT_MIN, INT_MIN};
    int all_hi = 0, all_lo = 0, n_rows = 0;
    float fac = A.scale_log2;
    uint32_t qf[kF][HD / 16][4];
    float o[kDW / 8][4], m[2], l[2];
    int ci = 0;  // tile of the current row tile

    while (done < issued || have) {
        if (loose > 0) {
            cp_wait<0>();
            --loose;
        } else {
            cp_wait<kS - 2>();
        }
        __syncthreads();  // this tile is here, the last one's stage, weights and maxima are free
        const bool begins = done == end;
        if (begins) {
            ++cq;
            cur = s_cur[cq & 1];
            end = done + cur.b - cur.a;
            ci = cur.a;
        }
        {
            int n = 0;
            for (; have && lq <= cq + 1 && issued < done + kS; ++n) issue();
            if (n > 1 || (n == 0 && have)) loose = kS;
            cp_commit();
        }
        const PagedItem& it = cur.it;
        if (begins) {
            n_rows = it.ntok * gpb;
            all_hi = min(it.kv_hi, it.pmin + 1);
            all_lo = A.window > 0 ? it.pmax - A.window + 1 : INT_MIN;
            if (tid < 16) {
                int pos = INT_MIN;
                if (tid < kRows && tid < n_rows)
                    pos = it.mixed ? token_position(A, it.tok0 + tid / gpb) : it.pos0 + tid / gpb;
                s_pos[tid] = pos;
            }
            const T* q = reinterpret_cast<const T*>(qraw + (cq & 1) * C::kQBytes);
            if (SPLIT) {
                split_rows<T, HD>(A, reinterpret_cast<const float*>(q), n_rows, work, s_fac);
                q = work;
            }
            __syncthreads();
#pragma unroll
            for (int n = 0; n < kF; ++n)
#pragma unroll
                for (int kk = 0; kk < HD / 16; ++kk) {
                    const int r = lane & 15, c = kk * 2 + (lane >> 4);
                    ldsm4(qf[n][kk], q + (size_t)(n * 16 + r) * HD + ((c ^ (r & 7)) * 8));
                }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int pos = SPLIT && u ? INT_MIN : s_pos[g + 8 * u];
                hi_row[u] = pos == INT_MIN ? 0 : min(it.kv_hi, pos + 1);
                lo_row[u] = A.window > 0 && pos != INT_MIN ? pos - A.window + 1 : INT_MIN;
                m[u] = -INFINITY;
                l[u] = 0.f;
            }
            fac = SPLIT ? s_fac[g] * A.scale_log2 : A.scale_log2;
#pragma unroll
            for (int d = 0; d < kDW / 8; ++d)
#pragma unroll
                for (int u = 0; u < 4; ++u) o[d][u] = 0.f;
        }

        const T* kd = ring + (size_t)(done % kS) * C::kStage;
        const T* vd = kd + kTile * HD;
        const int j0 = (ci < it.n_sink ? it.sink0 + ci : it.first + ci - it.n_sink) * kTile;
        const bool full = j0 >= it.kv_lo && j0 + kTile <= all_hi &&
                          (j0 >= all_lo || j0 + kTile <= sinks);
        const int jw = j0 + warp * 16;
        auto sees = [&](int u, int j) {
            return j >= it.kv_lo && j < hi_row[u] && (j >= lo_row[u] || j < sinks);
        };

        // scores of this warp's 16 positions
        float s[2][4];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int u = 0; u < 4; ++u) s[t][u] = 0.f;
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
            const int r = warp * 16 + ((lane >> 4) & 1) * 8 + (lane & 7);
            const int c = kk * 2 + ((lane >> 3) & 1);
            uint32_t kf[4];
            ldsm4(kf, kd + (size_t)r * HD + ((c ^ (r & 7)) * 8));
#pragma unroll
            for (int n = 0; n < kF; ++n) {
                PMath<T>::mma(s[0], qf[n][kk], kf[0], kf[1]);
                PMath<T>::mma(s[1], qf[n][kk], kf[2], kf[3]);
            }
        }
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int u = 0; u < (SPLIT ? 2 : 4); ++u) {
                float v = SPLIT ? (s[t][u] + s[t][(u + 2) & 3]) * fac : s[t][u] * fac;
                if (!full && !sees(u >> 1, jw + t * 8 + c4 * 2 + (u & 1))) v = -INFINITY;
                s[t][u] = v;
                mx[u >> 1] = fmaxf(mx[u >> 1], v);
            }
#pragma unroll
        for (int u = 0; u < (SPLIT ? 1 : 2); ++u) {
            mx[u] = fmaxf(mx[u], __shfl_xor_sync(0xffffffffu, mx[u], 1));
            mx[u] = fmaxf(mx[u], __shfl_xor_sync(0xffffffffu, mx[u], 2));
            if (c4 == 0) s_max[warp][g + 8 * u] = mx[u];
        }
        __syncthreads();
        float al[2] = {1.f, 1.f};
#pragma unroll
        for (int u = 0; u < (SPLIT ? 1 : 2); ++u) {
            float to = m[u];
#pragma unroll
            for (int w = 0; w < 4; ++w) to = fmaxf(to, s_max[w][g + 8 * u]);
            const float base = to == -INFINITY ? 0.f : to;
            al[u] = ex2(m[u] - base);
            m[u] = to;
            l[u] *= al[u];
            const float mb = base - kShift;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    s[t][2 * u + e] = ex2(s[t][2 * u + e] - mb);
                    l[u] += s[t][2 * u + e];
                }
        }
        // the weights, 16 (or 8, in parts) rows x 64 positions
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int c = warp * 2 + t;
            auto put = [&](int n, int r, uint32_t v) {
                *reinterpret_cast<uint32_t*>(work + (n * 16 + r) * kTile + ((c ^ (r & 7)) * 8) +
                                             c4 * 2) = v;
            };
            if (!SPLIT) {
                put(0, g, PMath<T>::pack(s[t][0], s[t][1]));
                put(0, g + 8, PMath<T>::pack(s[t][2], s[t][3]));
            } else {
                uint32_t p0, p1, p2 = 0;
                PMath<T>::split(s[t][0], s[t][1], p0, p1, p2);
                put(0, g, p0);
                put(0, g + 8, p1);
                if (kF == 2) {
                    put(kF - 1, g, p2);
                    put(kF - 1, g + 8, 0);
                }
            }
        }
        if (al[0] != 1.f || al[1] != 1.f) {
#pragma unroll
            for (int d = 0; d < kDW / 8; ++d)
#pragma unroll
                for (int u = 0; u < 4; ++u) o[d][u] *= SPLIT ? al[0] : al[u >> 1];
        }
        // Rows that see different positions of one tile: what is hidden from one may be an
        // infinity or a NaN that another sees.  Looked for first (rare), so that the usual loop
        // stays short.
        bool odd = false;
        if (!full && it.pmin != it.pmax) {
            for (int i = lane; i < kTile * kDW / 8; i += 32) {
                const int r = i / (kDW / 8), c = warp * (kDW / 8) + i % (kDW / 8);
                const uint4 w = *reinterpret_cast<const uint4*>(vd + (size_t)r * HD + ((c ^ (r & 7)) * 8));
                odd |= PMath<T>::not_finite(w.x) || PMath<T>::not_finite(w.y) ||
                       PMath<T>::not_finite(w.z) || PMath<T>::not_finite(w.w);
            }
            odd = __any_sync(0xffffffffu, odd);
        }
        __syncthreads();  // the weights are there
        auto weigh = [&](auto special) {
#pragma unroll
            for (int kk = 0; kk < kTile / 16; ++kk) {
                uint32_t pf[kF][4], one[4];
#pragma unroll
                for (int n = 0; n < kF; ++n) {
                    const int r = lane & 15, c = kk * 2 + (lane >> 4);
                    ldsm4(pf[n], work + (n * 16 + r) * kTile + ((c ^ (r & 7)) * 8));
                }
                if (decltype(special)::value) {  // visible places as ones
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        one[u] = 0;
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            if (sees(u & 1, j0 + kk * 16 + (u >> 1) * 8 + c4 * 2 + e))
                                one[u] |= PMath<T>::kOne << (16 * e);
                    }
                }
#pragma unroll
                for (int d = 0; d < kDW / 8; d += 2) {
                    const int r = kk * 16 + ((lane >> 3) & 1) * 8 + (lane & 7);
                    const int c = warp * (kDW / 8) + d + (lane >> 4);
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
#pragma unroll
                    for (int n = 0; n < kF; ++n) {
                        PMath<T>::mma(o[d], pf[n], vf[0], vf[1]);
                        PMath<T>::mma(o[d + 1], pf[n], vf[2], vf[3]);
                    }
                }
            }
        };
        if (odd) weigh(Flag<true>());
        else weigh(Flag<false>());
        ++done;
        ++ci;
        if (done != end) continue;

        // ------------------------------------------------------------ the row tile's piece ends
        const bool whole = cur.a == 0 && cur.b == it.n_tiles;
        if (cur.a == 0 && head_lane == 0) {  // what the join kernels need to know
            const int last = pieces.of(cur.c0 + it.n_tiles - 1);
            if (A.n_groups > 0) {
                for (int i = tid; i < it.ntok; i += kThreads)
                    P.where[it.tok0 + i] =
                        PagedWhere{piece, last, i * P.gpb, it.alone, which, cur.item};
            } else if (!whole && tid == 0) {
                P.split[piece] = PagedSplit{it.tok0, it.ntok * P.gpb, last, cur.item, 0, 0};
            }
        }
#pragma unroll
        for (int u = 0; u < (SPLIT ? 1 : 2); ++u) {
            l[u] += __shfl_xor_sync(0xffffffffu, l[u], 1);
            l[u] += __shfl_xor_sync(0xffffffffu, l[u], 2);
            if (c4 == 0) s_l[warp][g + 8 * u] = l[u];
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < (SPLIT ? 1 : 2); ++u) {
            const int row = g + 8 * u;
            if (row >= n_rows) continue;
            const float L = (s_l[0][row] + s_l[1][row]) + (s_l[2][row] + s_l[3][row]);
            RowOut<T, SPLIT> R(A, P, which, it, piece, head_lane, h0, gpb, row, cur.a, whole);
#pragma unroll
            for (int d = 0; d < kDW / 8; ++d) {
                const int at = warp * kDW + d * 8 + c4 * 2;
                if (at >= A.hd) break;
                R.put2(at, SPLIT ? make_float2(o[d][0] + o[d][2], o[d][1] + o[d][3])
                                 : make_float2(o[d][2 * u], o[d][2 * u + 1]), L);
            }
            if (warp == 0 && c4 == 0) R.put_ml(m[u] - kShift, L);
        }
    }
    cp_wait<0>();
    __syncthreads();
    if (tid == 0 && s_bad) P.bad[blockIdx.x] = s_bad;
}

template <typename T, bool SPLIT, int HD>
cudaError_t launch_one(const PagedArgs& A, int which, bool with_prefix, cudaStream_t s) {
    auto kern = paged_few_kernel<T, SPLIT, HD>;
    constexpr size_t smem = FCfg<T, SPLIT, HD>::kSmem;
    cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(kern),
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    const PagedPlan& P = A.plan[which];
    return launch_pdl(kern, dim3(P.heads * P.lanes, with_prefix ? 2 : 1), dim3(kThreads), smem, s, A,
                      which);
}

template <typename T, bool SPLIT>
cudaError_t launch_t(const PagedArgs& A, int which, bool both, cudaStream_t s) {
    return A.hd <= 64    ? launch_one<T, SPLIT, 64>(A, which, both, s)
           : A.hd <= 128 ? launch_one<T, SPLIT, 128>(A, which, both, s)
                         : launch_one<T, SPLIT, 256>(A, which, both, s);
}

}  // namespace

int paged_few_tile() { return kTile; }
int paged_few_ctas(int hd) {
    return hd <= 64 ? FCfg<__half, false, 64>::kCtas : hd <= 128 ? FCfg<__half, false, 128>::kCtas : 1;
}

// both: the shared prefixes' plan in the same launch.
cudaError_t launch_paged_few(const PagedArgs& A, int which, bool both, int q_dtype, int kv_dtype,
                             cudaStream_t s) {
    const bool split = q_dtype == WISP_DTYPE_F32;
    if (kv_dtype == WISP_DTYPE_F16)
        return split ? launch_t<__half, true>(A, which, both, s)
                     : launch_t<__half, false>(A, which, both, s);
    return split ? launch_t<__nv_bfloat16, true>(A, which, both, s)
                 : launch_t<__nv_bfloat16, false>(A, which, both, s);
}

}  // namespace wb
