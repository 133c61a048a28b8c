// paged_few.cu -- attention of row tiles with few rows (single tokens, a few drafted ones, few
// sequences behind a prefix): one 16-row tile of mma.sync per kv head, bound by the cache's HBM
// reads.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = 2^(log2(e) scale q_i . k_j - m_i)
//
// A CTA streams its piece of the line of KV tiles (64 positions, one kv head).  A loading warp
// walks the piece's row tiles, looks their pages up and issues the TMA boxes (128-byte swizzle)
// and the rows of q into rings that do not stop at the end of a row tile.  Four warps work: each
// scores 16 of a tile's positions; the row maxima and the weights go through shared memory, and
// then each warp adds all 64 weighted positions to a quarter of the head's dims.
//
// Measured (B200): 64 sequences with a window of 4096 and four sinks, 32 heads of 128 over 8 kv
// heads, 171 us = 6.3 TB/s (97% of the measured copy); 14 ragged sequences of up to 4096 positions
// 30 us (63%: the first tile is there after 5 us, the join takes 4.5 us); one sequence of 1024
// 10.6 us (11.9 us with the row tiles of a piece worked out twice and shared memory for one CTA
// an SM where two were counted on).  Before: each warp kept all dims for its own positions (64
// accumulators a thread, a join of four 16 x head_dim tiles and an empty ring at the end of every
// row tile: 39.7 us for 14 ragged sequences of up to 4096 positions); the same split with cp.async
// issued by the working warps (486 instructions a warp and tile: 35.7 us, but long windows fell
// from 6.4 to 5.6 TB/s).
//
// 32-bit rows are split into 16-bit parts (two in fp16, 22 bits, three in bf16) that share the
// 16 rows of a fragment, 8 rows each; their sums meet in one thread.  The weights are split the
// same way.  In fp16 they carry 2^kPShift, which cancels, so that small weights of long caches
// stay above the subnormals.

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "internal.h"
#include "paged.h"
#include "paged_math.cuh"
#include "paged_tma.cuh"

namespace wb {
namespace {

constexpr int kWork = 128;             // working threads
constexpr int kThreads = kWork + 32;  // and the loading warp
constexpr int kTile = kPagedTile;
constexpr int kRecs = 16;
static_assert(kPagedInline <= kThreads, "a thread per row tile");

template <typename T, bool SPLIT, int HD>
struct FCfg {
    static constexpr int kF = SPLIT ? PMath<T>::kFrags : 1;  // 16-row fragments of a row's parts
    static constexpr int kStages = HD == 64 ? (kF == 1 ? 4 : 3) : HD == 128 && kF == 1 ? 3 : 2;
    static constexpr int kCtas = HD == 64 ? 3 : HD == 128 ? 2 : 1;
    static constexpr int kHalves = HD / 64;
    static constexpr int kTen = kTile * HD * 2;      // bytes of a K or V tile
    static constexpr int kQBytes = SPLIT ? 8 * HD * 4 : 16 * HD * 2;  // a row tile's q as it is
    // converted q (fp32 rows only) or the tile's weights, elements
    static constexpr int kBuf = std::max(kF * 16 * kTile, SPLIT ? kF * 16 * HD : 0);
    static constexpr size_t kSmem = 1024 + (size_t)kStages * 2 * kTen + 2 * kQBytes + kBuf * 2;
    // (4 KB for what is declared in the kernel, 1 KB of the system's for each CTA of the SM's 228)
    static_assert((kSmem + 4096 + 1024) * kCtas <= 228 * 1024, "kCtas do not fit");
};

struct Rec {  // a row tile of this piece and its KV tiles [a, b); b < 0: there are no more
    PagedItem it;
    int a, b;
    int item, c0;
};
__device__ __forceinline__ Rec make_rec(const PagedPlan& P, const PagedItem& it, int item, int cum,
                                        int x0, int x_end) {
    const int c0 = cum + P.lead;
    return Rec{it, max(0, x0 - c0), max(0, min(it.n_tiles, x_end - c0)), item, c0};
}

__device__ __forceinline__ void work_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
// The same; whether any thread has `x` set.
__device__ __forceinline__ bool work_any(bool x) {
    uint32_t any;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\tbar.red.or.pred p, 1, 128, q;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(any)
        : "r"((uint32_t)x)
        : "memory");
    return any != 0;
}

template <typename T, bool SPLIT, int HD>
__global__ void __launch_bounds__(kThreads, (FCfg<T, SPLIT, HD>::kCtas))
paged_few_kernel(const __grid_constant__ PagedArgs A, const __grid_constant__ KvMaps maps, int which0,
                 int box_rows, int behind) {
    using C = FCfg<T, SPLIT, HD>;
    constexpr int kF = C::kF, kS = C::kStages, kRows = SPLIT ? 8 : 16;
    constexpr int kDW = HD / 4;  // dims of a warp
    constexpr float kShift = PMath<T>::kPShift;
    extern __shared__ char raw[];
    char* ring = reinterpret_cast<char*>(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    char* qraw = ring + kS * 2 * C::kTen;  // [2] rows of q as they are
    T* work = reinterpret_cast<T*>(qraw + 2 * C::kQBytes);
    __shared__ uint64_t full[kS], empty[kS], q_full[2], q_empty[2];
    __shared__ Waits s_wait;
    __shared__ Rec s_rec[kRecs], s_cur[2];
    __shared__ int s_cum[kPagedInline + 1];
    __shared__ int s_sum[kThreads / 32], s_bad, s_item0, s_pos[16];
    __shared__ float s_fac[16], s_max[4][16], s_l[4][16];
    const int which = blockIdx.y ? PLAN_PREFIX : which0;
    const PagedPlan& P = A.plan[which];
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(kAll, tid >> 5, 0);
    const int g = lane >> 2, c4 = lane & 3;
    const int head_lane = blockIdx.x % P.heads, piece = blockIdx.x / P.heads;
    const int kvh = head_lane / P.hblocks, hb = head_lane - kvh * P.hblocks;
    const int h0 = kvh * A.group + hb * P.gpb, gpb = min(P.gpb, A.group - hb * P.gpb);

    if (tid == 0) {
        for (int i = 0; i < kS; ++i) {
            bar_init(&full[i], 1);
            bar_init(&empty[i], 4);
        }
        for (int i = 0; i < 2; ++i) {
            bar_init(&q_full[i], 33);
            bar_init(&q_empty[i], 4);
        }
        s_wait.out = 0;
        s_wait.limit = A.wait_ns;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // Behind the shared prefixes' kernel of this call, which has waited for all that is read here,
    // the SMs that it leaves start on this one: only the end waits for it (for the join's sake).
    // (64 sequences behind two long prefixes: 98 us a call, 102 us with the wait here.)
    auto wait_before = [&]() { asm volatile("griddepcontrol.wait;" ::: "memory"); };
    if (!behind) wait_before();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    const bool inlined = P.inlined != 0, prefix = which == PLAN_PREFIX;
    if (tid == 0) {
        s_bad = 0;
        P.bad[blockIdx.x] = 0;
        if (head_lane == 0) P.split[piece] = PagedSplit{0, 0, 0, 0, 0, 0};
        if (inlined && blockIdx.x == 0) P.bad[P.lanes * P.heads] = 0;
    }
    const int n_items = inlined ? (prefix ? A.n_groups : A.n_seq) * P.per_seg : *P.n_items;
    if (n_items == 0) {
        if (behind) wait_before();
        return;
    }
    const int* cum = inlined ? s_cum : P.cum;
    PagedItem mine;
    int units = 0, before = 0, total = 0;
    if (inlined) {
        // few row tiles: every CTA counts the units itself, a thread per row tile, which is shorter
        // than a kernel of its own before this one
        if (tid < kRecs) s_rec[tid].a = 0, s_rec[tid].b = -1;
        __syncthreads();  // the words above are cleared
        if (tid < n_items) {
            const int seg = P.per_seg == 1 ? tid : tid / P.per_seg;
            mine = make_item(A, P, prefix, seg, tid - seg * P.per_seg);
            units = item_units(P, mine);
            if (blockIdx.x == 0 && !prefix && tid == seg * P.per_seg) {
                const int t = A.q_start[seg + 1] - A.q_start[seg];
                if (length_too_long(A, seg) || t > P.tpt * P.per_seg || left_out(A, P, t))
                    P.bad[P.lanes * P.heads] = PG_BAD_LENGTH;
            }
        }
        int v = units;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += y;
        }
        if (lane == 31) s_sum[warp] = v;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kThreads / 32; ++w) {
            if (w < warp) before += s_sum[w];
            total += s_sum[w];
        }
        before += v - units;
        if (tid < n_items) s_cum[tid] = before;
        if (tid == 0) s_cum[n_items] = total;
    } else {
        total = P.cum[n_items];
    }
    const Pieces pieces(P, max(total, 1));
    if (total == 0 || piece >= pieces.n) {
        if (behind) wait_before();
        return;
    }
    const int x0 = pieces.start(piece), x_end = pieces.start(piece + 1);
    int item0;
    if (inlined) {  // the first records of this piece are at hand
        if (before <= x0 && x0 < before + units) s_item0 = tid;
        __syncthreads();
        item0 = s_item0;
        if (tid >= item0 && tid < item0 + kRecs && tid < n_items && before < x_end)
            s_rec[tid - item0] = make_rec(P, mine, tid, before, x0, x_end);
    } else {
        item0 = block_last_le(cum, n_items, x0);
    }

    __syncthreads();  // the barriers are there (a plan that is not inlined had no barrier yet)
    const int sinks = A.window > 0 ? A.sinks : 0;

    if (warp == kWork / 32) {
        // ------------------------------------------------------------ loads
        const int per_half = kTile / box_rows, boxes = per_half * C::kHalves;
        uint32_t tiles = 0, rows = 0;  // KV tiles and row tiles so far
        bool ok = true;
        // hands a record (and with it the rows of q) over
        auto hand = [&](const Rec& r) {
            const int b = rows & 1;
            if (!bar_wait_warp(&q_empty[b], ((rows >> 1) & 1) ^ 1, &s_wait)) return false;
            ++rows;
            if (lane == 0) {
                s_cur[b] = r;
                bar_arrive(&q_full[b]);
            }
            char* dst = qraw + b * C::kQBytes;
            constexpr int kPer = SPLIT ? HD / 4 : HD / 8;  // 16-byte pieces of a row
            const int n = r.b < 0 ? 0 : r.it.ntok * gpb * kPer;
            for (int i = lane; i < n; i += 32) {
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
            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(
                             smem_addr(&q_full[b]))
                         : "memory");
            return true;
        };
        for (int k = 0; ok; ++k) {
            if (k % kRecs == 0 && !(inlined && k == 0)) {  // the next records, one a lane
                __syncwarp();
                const int i = item0 + k + lane;
                if (lane < kRecs) {
                    s_rec[lane].a = 0;
                    s_rec[lane].b = -1;
                    if (i < n_items && cum[i] < x_end)
                        s_rec[lane] =
                            make_rec(P, inlined ? make_item(A, P, prefix, i / P.per_seg, i % P.per_seg)
                                                : P.items[i],
                                     i, cum[i], x0, x_end);
                }
                __syncwarp();
            }
            const Rec& r = s_rec[k % kRecs];
            if (r.b >= 0 && r.a >= r.b) continue;
            auto place = [&](int i) {
                const int t = i < r.it.n_sink ? r.it.sink0 + i : r.it.first + i - r.it.n_sink;
                return lane < boxes
                           ? box_place(A, r.it, t * kTile, lane % per_half, box_rows, &s_bad)
                           : make_int2(0, 0);
            };
            int2 at = r.b < 0 ? make_int2(0, 0) : place(r.a);
            for (int i = r.a; ok && i < r.b; ++i, ++tiles) {
                const int2 cur = at;
                if (i + 1 < r.b) at = place(i + 1);
                const int st = tiles % kS;
                ok = bar_wait_warp(&empty[st], ((tiles / kS) & 1) ^ 1, &s_wait);
                if (!ok) break;
                if (lane == 0) bar_expect(&full[st], 2 * C::kTen);
                __syncwarp();
                const uint32_t dst = smem_addr(ring + st * 2 * C::kTen);
                if (lane < boxes) {
                    const int half = lane / per_half, rb = lane % per_half;
                    const uint32_t to = dst + half * (kTile * 128) + rb * box_rows * 128;
                    tma4d(to, &maps.k, half * 64, kvh, cur.y, cur.x, &full[st]);
                    tma4d(to + C::kTen, &maps.v, half * 64, kvh, cur.y, cur.x, &full[st]);
                }
                if (i == r.a) ok = hand(r);
            }
            if (r.b < 0) {  // the end
                if (ok) hand(r);
                break;
            }
        }
        cp_commit();
        cp_wait<0>();
        __syncwarp();
        if (lane == 0)  // (only after a timeout can some of these still be in flight)
            for (uint32_t i = tiles > (uint32_t)kS ? tiles - kS : 0; i < tiles; ++i)
                bar_drain(&full[i % kS], (i / kS) & 1);
    } else {
    // ---------------------------------------------------------------- work
    Rec cur{};
    int hi_row[2] = {0, 0}, lo_row[2] = {INT_MIN, INT_MIN};
    int all_hi = 0, all_lo = 0, n_rows = 0;
    float fac = A.scale_log2;
    uint32_t qf[kF][HD / 16][4];
    float o[kDW / 8][4], m[2], l[2];
    uint32_t done = 0, rows = 0;  // KV tiles, row tiles so far
    int ci = 0;                   // tile of the current row tile
    bool begins = true;

    for (;;) {
        // A warp whose wait ran out goes on to the next barrier of the four, where all leave together:
        // one that left alone would keep the others there.
        bool late = false;
        if (begins) {
            const int b = rows & 1;
            late = !bar_wait_warp(&q_full[b], (rows >> 1) & 1, &s_wait);
            if (!late) cur = s_cur[b];
            ci = cur.a;
        }
        if (!late && !(begins && cur.b < 0))
            late = !bar_wait_warp(&full[done % kS], (done / kS) & 1, &s_wait);
        const PagedItem& it = cur.it;
        if (begins) {
            if (tid < 16 && !late && cur.b >= 0) {
                int pos = INT_MIN;
                if (tid < kRows && tid < it.ntok * gpb)
                    pos = it.mixed ? token_position(A, it.tok0 + tid / gpb) : it.pos0 + tid / gpb;
                s_pos[tid] = pos;
            }
            // (behind it the last tile's weights have been read, too)
            if (work_any(late) || cur.b < 0) break;
            n_rows = it.ntok * gpb;
            all_hi = min(it.kv_hi, it.pmin + 1);
            all_lo = A.window > 0 ? it.pmax - A.window + 1 : INT_MIN;
            const T* q = reinterpret_cast<const T*>(qraw + (rows & 1) * C::kQBytes);
            if (SPLIT) {
                split_rows<T, HD>(A, reinterpret_cast<const float*>(q), n_rows, work, s_fac);
                q = work;
                work_sync();
            }
#pragma unroll
            for (int n = 0; n < kF; ++n)
#pragma unroll
                for (int kk = 0; kk < HD / 16; ++kk) {
                    const int r = lane & 15, c = kk * 2 + (lane >> 4);
                    ldsm4(qf[n][kk], q + (size_t)(n * 16 + r) * HD + ((c ^ (r & 7)) * 8));
                }
            __syncwarp();
            if (lane == 0) bar_arrive(&q_empty[rows & 1]);
            ++rows;
            begins = false;
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

        // [half][position][64 dims], 16-byte pieces XORed with the position's low bits
        const char* kd = ring + (done % kS) * 2 * C::kTen;
        const char* vd = kd + C::kTen;
        auto piece_at = [&](const char* tile, int row, int c) {
            return tile + (c / 8) * (kTile * 128) + row * 128 + (((c & 7) ^ (row & 7)) * 16);
        };
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
            ldsm4(kf, piece_at(kd, r, c));
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
        if (work_any(late)) break;
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
        // What a partly hidden tile hides (a page's end that nobody wrote, another row's future)
        // may hold infinities and NaNs.  They are looked for first (rare), so that the usual loop
        // stays short.
        bool odd = false;
        if (!full) {
            for (int i = lane; i < kTile * kDW / 8; i += 32) {
                const int r = i / (kDW / 8), c = warp * (kDW / 8) + i % (kDW / 8);
                const uint4 w = *reinterpret_cast<const uint4*>(piece_at(vd, r, c));
                odd |= PMath<T>::not_finite(w.x) || PMath<T>::not_finite(w.y) ||
                       PMath<T>::not_finite(w.z) || PMath<T>::not_finite(w.w);
            }
            odd = __any_sync(0xffffffffu, odd);
        }
        work_sync();  // the weights are there
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
                    ldsm4t(vf, piece_at(vd, r, c));
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
        __syncwarp();
        if (lane == 0) bar_arrive(&empty[done % kS]);
        ++done;
        if (++ci < cur.b) continue;
        begins = true;

        // ------------------------------------------------------------ the row tile's piece ends
        const bool whole = cur.a == 0 && cur.b == it.n_tiles;
        if (cur.a == 0 && head_lane == 0) {  // what the join kernels need to know
            const int last = pieces.of(cur.c0 + it.n_tiles - 1);
            if (A.n_groups > 0) {
                for (int i = tid; i < it.ntok; i += kWork)
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
        work_sync();
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
    }
    __syncthreads();
    if (tid == 0 && (s_bad || s_wait.out)) P.bad[blockIdx.x] = s_bad | (s_wait.out ? PG_TIMEOUT : 0);
    if (behind) wait_before();
}

template <typename T, bool SPLIT, int HD>
cudaError_t launch_one(const PagedArgs& A, int which, bool with_prefix, bool behind,
                       cudaStream_t s) {
    auto kern = paged_few_kernel<T, SPLIT, HD>;
    constexpr size_t smem = FCfg<T, SPLIT, HD>::kSmem;
    static std::atomic<uint64_t> done{0};
    cudaError_t e = smem_opt_in(reinterpret_cast<const void*>(kern), smem, done);
    if (e != cudaSuccess) return e;
    KvMaps maps;
    const int rows = kv_maps(&maps, A, std::is_same<T, __nv_bfloat16>::value,
                             kTile);
    if (rows == 0) return cudaErrorInvalidValue;
    const PagedPlan& P = A.plan[which];
    return launch_pdl(kern, dim3(P.heads * P.lanes, with_prefix ? 2 : 1), dim3(kThreads), smem, s, A,
                      maps, which, rows, (int)behind);
}

template <typename T, bool SPLIT>
cudaError_t launch_t(const PagedArgs& A, int which, bool both, bool behind, cudaStream_t s) {
    return A.hd <= 64    ? launch_one<T, SPLIT, 64>(A, which, both, behind, s)
           : A.hd <= 128 ? launch_one<T, SPLIT, 128>(A, which, both, behind, s)
                         : launch_one<T, SPLIT, 256>(A, which, both, behind, s);
}

}  // namespace

int paged_few_ctas(int hd) {
    return hd <= 64 ? FCfg<__half, false, 64>::kCtas : hd <= 128 ? FCfg<__half, false, 128>::kCtas : 1;
}

// both: the shared prefixes' plan in the same launch.  behind: the launch before it on the stream
// is another attention kernel of this call.
cudaError_t launch_paged_few(const PagedArgs& A, int which, bool both, bool behind, int q_dtype,
                             int kv_dtype, cudaStream_t s) {
    const bool split = q_dtype == WISP_DTYPE_F32;
    if (kv_dtype == WISP_DTYPE_F16)
        return split ? launch_t<__half, true>(A, which, both, behind, s)
                     : launch_t<__half, false>(A, which, both, behind, s);
    return split ? launch_t<__nv_bfloat16, true>(A, which, both, behind, s)
                 : launch_t<__nv_bfloat16, false>(A, which, both, behind, s);
}

}  // namespace wb
