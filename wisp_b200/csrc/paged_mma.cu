// paged_mma.cu -- attention of row tiles with many rows (prompts, chunks, drafted tokens, the
// sequences of a shared prefix) on tcgen05, over the pages.
//
// One persistent CTA per SM takes a piece of the line of (row tile, KV tile) pairs for one kv
// head.  Per KV tile of 64 positions and 128 rows:
//   S = Q K^T   tcgen05.mma M=128 N=64, Q and K from shared memory, S in tensor memory
//   P = 2^(S fac - m)  one thread per row; P back to tensor memory as 16-bit pairs
//   O += P V    tcgen05.mma M=128 N=head_dim, P from tensor memory, V from shared memory
// Two tiles of 128 rows share each K / V tile; an item with at most 128 rows (drafted tokens, a
// group behind a prefix) takes both for itself, one for its even and one for its odd KV tiles,
// and joins them at the end (each thread reads both O's: one tile's softmax alone kept such
// items at 75% of HBM).  S is double buffered, so the tensor core works on tile j + 1 while the
// softmax warps work on tile j.  Roles:
//   warps 0-3 (and 4-7)  softmax of row tile 0 (and 1): rows 32 * (warp & 3) + lane
//   warps 8 and 9        issue the MMAs of one row tile each (an elected thread)
//   warp 10              loads K and V: TMA boxes of up to 64 positions out of one page, lane
//                        per box, 128-byte swizzle, ring of 16-KB slots
//   warp 11              loads the rows of Q (TMA where a row tile is whole tokens) as soon as the
//                        last product that reads the previous ones is done; 32-bit rows, which
//                        have one row tile, are loaded and split by warps 4-7 (one prompt of 2048
//                        fp32 tokens 222 us at that step, 641 us with one warp).  It also looks V of partly
//                        hidden tiles through for infinities and NaNs, for both row tiles: their
//                        products with V wait for it
// A row's running maximum is only moved when a score passes it by more than 2^8 (the weights
// then still fit 16 bits and the sums are fp32), so that O is rarely rescaled; the warp that
// needs it does so itself, behind the previous product.
//
// 32-bit rows: q and p are split into PARTS 16-bit parts (two in fp16, three in bf16) with one
// product each into the same accumulator; one tile of 128 rows then.
//
// Hidden values.  A box outside what the tile's rows see is loaded from outside the tensor map
// (zeros).  In tiles that are partly hidden V is looked through for infinities and NaNs before
// the product: those that no row sees are zeroed in shared memory; where some row sees one, the
// row tile is marked and the join kernel works it out again without tiles.
//
// Measured (B200; ranges: the best and the middle of long replays, under the power limit): a
// prompt of 8192 tokens, 32 heads of 128 over 8 kv heads, 515 to 590 us = 1.07 to 0.93 PFLOP/s of
// the visible pairs (63 to 55% of the measured bf16 rate), tensor pipe and exponential unit 56%
// busy each at 1.66 GHz; chunks of 7652 tokens behind up to 9000 positions, 16 heads of 64, window
// 1024, 117 us; four drafted tokens behind 64K to 128K positions, 64 heads, 302 to 345 us = 6.0 to
// 5.2 TB/s (92 to 81% of the measured copy); 2048 fp32 tokens 205 us.  Steps of the prompt, at
// their best: mma.sync row tiles
// of 64 rows 4.57 ms; this kernel with one thread issuing all products 1.15 ms (it was bound by
// 80 to 115 cycles an instruction); a warp per row tile with warp-uniform operands 816 us; pieces
// that count what beginning a row tile costs 694 us; Q by TMA behind the last product 551 us;
// pieces balanced by what a row tile costs to begin (six KV tiles) and by its rows 540 us.
// Measured and not kept: Q double buffered with a ring of three KV tiles (817 us), registers moved
// to the softmax warps (no gain), one softmax warp of a pair waiting for the other's exponentials
// (no gain), skipping hidden tiles warp by warp inside the loop (prompts 10% slower), a quarter to
// a half of the exponentials as polynomials (no gain; with five eighths 8% slower), deciding per
// 128 rows what is hidden (chunks 3% faster, prompts 2 to 5% slower).
//
// TMEM (512 columns): S buffers of 64 columns, P over them (or beside them when it has several
// parts), O of head_dim columns per row tile.  Every wait is bounded; on a timeout all roles
// leave, copies and products in flight are drained and TMEM is freed.

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "internal.h"
#include "paged.h"
#include "paged_math.cuh"
#include "paged_tma.cuh"

namespace wb {
namespace {

constexpr int kN = kPagedTile;          // positions of a KV tile
constexpr int kM = kPagedHalf;  // rows of a row tile
constexpr int kThreads = 384;
// fp32 rows: O is added to a rounded sum after so many KV tiles.  The tensor core cuts its sums off,
// which shrinks a long row by half a unit of the last place an instruction: 40 tokens behind 16000
// positions were 3.6e-6 off (plain fp32 0.7e-6), with 8 tiles 1.7e-6, with 4 1.25e-6, with 1 0.9e-6;
// 3 x 500 tokens behind 4000, 16 heads of 64, took 109, 112, 116 and 131 us.
constexpr int kFlush = 4;
constexpr int kMmaWarp = 8, kLoadWarp = 10, kRowWarp = 11;

template <int HD, int PARTS>
struct MCfg {
    static constexpr int kRT = PARTS == 1 ? 2 : 1;       // row tiles
    static constexpr int kHalves = HD / 64;
    static constexpr int kSlot = kN * HD * 2;            // bytes of a K or V tile
    static constexpr int kQ = kM * HD * 2;               // bytes of one part of Q
    // Q of this and the next row tile where the ring keeps four KV tiles beside them (with 128
    // dims it does not: a ring of three tiles cost more than Q's early loads gave)
    static constexpr int kQBufs = HD == 64 ? 2 : 1;
    static constexpr int kSlots = HD == 64 ? (PARTS == 3 ? 8 : 12) : PARTS == 3 ? 7 : 9;
    static constexpr int kSmem = 1024 + kQBufs * kRT * PARTS * kQ + kSlots * kSlot;
    // TMEM columns: S in two buffers, part p of P over them or (two parts, and the third) behind
    static __host__ __device__ constexpr int s_col(int x, int b) { return (x * 2 + b) * 64; }
    static __host__ __device__ constexpr int p_col(int x, int b, int p) {
        return PARTS == 1   ? s_col(x, b)
               : PARTS == 2 ? 128 + b * 64 + p * 32
               : p < 2      ? s_col(x, b) + p * 32
                            : 128 + b * 32;
    }
    static __host__ __device__ constexpr int o_col(int x) { return 512 - (kRT - x) * HD; }
    // fp32 rows: what O held every kFlush KV tiles, added rounded
    static constexpr int kSumCol = 512 - 2 * HD;
};

// Shared-memory descriptors, 128-byte swizzle.  K-major (Q, K): 64 elements per row of 128 B,
// atoms of 8 rows 1024 B apart.  MN-major (V: positions are K, head dims N): blocks of 64 dims
// `lead` bytes apart, groups of 8 positions 1024 B apart.
// (Both as the low word of `addr` with a constant high word: an address step is one addition.)
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_k(uint32_t addr) { return (addr >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_mn(uint32_t addr, uint32_t lead) {
    return (addr >> 4) | ((lead >> 4) << 16);
}
// Instruction descriptor of kind::f16: A and B fp16 (0) or bf16 (1), fp32 accumulator, M = 128,
// N = n, A K-major, B K-major or (b_mn) MN-major.
__host__ __device__ constexpr uint32_t idesc(int type, int n, int b_mn) {
    return (1u << 4) | ((uint32_t)type << 7) | ((uint32_t)type << 10) | ((uint32_t)b_mn << 16) |
           ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kM >> 4) << 24);
}
// By the whole warp with the same operands; the thread with `leader` set issues.
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t id, uint32_t acc,
                                       uint32_t leader) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 da, db;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
        "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(id), "r"(acc), "r"(kDescHi), "r"(leader)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t id, uint32_t acc,
                                       uint32_t leader) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 db;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
        "mov.b64 db, {%2, %5};\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(id), "r"(acc), "r"(kDescHi), "r"(leader)
        : "memory");
}
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t is;
    asm volatile(
        "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(is));
    return is;
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
    asm volatile(
        "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
            smem_addr(bar))
        : "memory");
}
__device__ __forceinline__ void tc_before() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_after() {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void async_fence() {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
// 32 or 64 columns of this thread's TMEM lane.  The wait is part of the statement: the
// registers are not valid before it, and nothing may be scheduled in between that reads them.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float* v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
        "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31"
        "}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]),
          "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]),
          "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]),
          "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
          "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]),
          "=f"(v[31])
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tmem_ld64(uint32_t addr, float* v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
        "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32,%33,%34,%35,%36,"
        "%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,"
        "%54,%55,%56,%57,%58,%59,%60,%61,%62,%63"
        "}, [%64];\n\ttcgen05.wait::ld.sync.aligned;"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]),
          "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]),
          "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]),
          "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
          "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]),
          "=f"(v[31]), "=f"(v[32]), "=f"(v[33]), "=f"(v[34]), "=f"(v[35]), "=f"(v[36]),
          "=f"(v[37]), "=f"(v[38]), "=f"(v[39]), "=f"(v[40]), "=f"(v[41]), "=f"(v[42]),
          "=f"(v[43]), "=f"(v[44]), "=f"(v[45]), "=f"(v[46]), "=f"(v[47]), "=f"(v[48]),
          "=f"(v[49]), "=f"(v[50]), "=f"(v[51]), "=f"(v[52]), "=f"(v[53]), "=f"(v[54]),
          "=f"(v[55]), "=f"(v[56]), "=f"(v[57]), "=f"(v[58]), "=f"(v[59]), "=f"(v[60]),
          "=f"(v[61]), "=f"(v[62]), "=f"(v[63])
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,"
        "%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(
            addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
        "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
        "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
        "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// Weights of 16-bit pairs stay below 2^15 with the maximum up to 2^8 behind (fp16).
template <typename T>
struct MShift {
    static constexpr float value = std::is_same<T, __half>::value ? 6.f : 0.f;
};

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    return v;
}
__device__ __forceinline__ void unpair(uint64_t v, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// 32 bytes to a 32-byte boundary.
__device__ __forceinline__ void store32(void* to, const uint32_t* w) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(to), "r"(w[0]), "r"(w[1]),
                 "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}

// The low n bits (none for n <= 0, all for n >= 64).
__device__ __forceinline__ uint64_t below(int n) {
    return n <= 0 ? 0 : n >= 64 ? ~0ull : (1ull << n) - 1;
}
// Nonzero when a half of v is an infinity or a NaN: adding one to a full exponent carries.
template <typename T>
__device__ __forceinline__ uint32_t odd_halves(uint32_t v) {
    constexpr uint32_t e = PMath<T>::kExp * 0x10001u;
    constexpr uint32_t one = (PMath<T>::kExp & (0u - PMath<T>::kExp)) * 0x10001u;
    return ((v & e) + one) & 0x80008000u;
}

// The shared state of a piece's walk: which item and tiles come next.  Every role walks alike.
struct Walk {
    int item, x, x_end;
    int a, b;  // KV tiles [a, b) of the item
    int c0;    // the item's first KV tile on the line
    int sh;    // its KV tiles are 2^sh units
    int all_hi, all_lo;  // every row sees the positions between (and the sinks)
    int w0, w1;          // of the KV tiles behind the sinks' the ones that every row sees whole
    PagedItem it;
    __device__ __forceinline__ bool next(const PagedArgs& A, const PagedPlan& P) {
        while (x < x_end) {
            it = P.items[item];
            c0 = P.cum[item] + P.lead;
            sh = item_shift(P, it);
            ++item;
            if (it.n_tiles == 0) continue;
            all_hi = min(it.kv_hi, it.pmin + 1);
            all_lo = A.window > 0 ? it.pmax - A.window + 1 : INT_MIN;
            w0 = it.n_sink + max(0, (max(it.kv_lo, all_lo) + kN - 1) / kN - it.first);
            w1 = it.n_sink + all_hi / kN - it.first;
            a = (max(0, x - c0) + sh) >> sh;
            b = min(it.n_tiles, (max(0, x_end - c0) + sh) >> sh);
            x = min(c0 + (it.n_tiles << sh), x_end);
            if (a < b) return true;  // (else: the piece has none of the item's tiles)
        }
        return false;
    }
    // The piece of the item's last KV tile.
    __device__ __forceinline__ static int last_piece(const Pieces& pieces, int c0, int sh, int n_tiles) {
        return pieces.of(c0 + ((n_tiles - 1) << sh));
    }
    __device__ __forceinline__ int tile(int i) const {
        return i < it.n_sink ? it.sink0 + i : it.first + i - it.n_sink;
    }
};

// n rows of Q from row `row0` of the item on into a 128-row tile (zeros below them): all of it by
// one warp, of fp32 rows 32 from row `part` on.
template <typename T, int PARTS, int HD>
__device__ __forceinline__ void load_q_tile(const PagedArgs& A, int tok0, int row0, int n, int h0,
                                            int gpb, bool flip, char* tile, float* s_fac, int part) {
    const int lane = threadIdx.x & 31;
    using C = MCfg<HD, PARTS>;
    auto source = [&](int r) {
        const int row = row0 + r, t = row / gpb;
        return (size_t)(tok0 + t) * A.q_stride + (size_t)(h0 + row - t * gpb) * A.hd;
    };
    if constexpr (PARTS == 1) {
        constexpr int kCh = HD / 8, kPer = 32 / kCh;  // rows per pass
        const int c = lane % kCh;
        const T* q = reinterpret_cast<const T*>(A.q) + c * 8;
        char* dst = tile + (c / 8) * (kM * 128);
        const bool in_row = c * 8 < A.hd;
#pragma unroll 8
        for (int r = lane / kCh; r < kM; r += kPer) {
            const bool in = r < n && in_row;
            char* to = dst + r * 128 + (((c & 7) ^ (r & 7)) * 16);
            const T* from = in ? q + source(r) : reinterpret_cast<const T*>(A.q);
            if (!flip) {
                cp16(to, from, in);
            } else {
                uint4 w = in ? __ldg(reinterpret_cast<const uint4*>(from)) : make_uint4(0, 0, 0, 0);
                w.x ^= 0x80008000u, w.y ^= 0x80008000u, w.z ^= 0x80008000u, w.w ^= 0x80008000u;
                *reinterpret_cast<uint4*>(to) = w;
            }
        }
        cp_commit();
        cp_wait<0>();
    } else {
        // fp32 rows, HD / 32 floats a lane: parts of 16 bits, in fp16 of q / 2^e with 2^e the row's
        // largest exponent
        constexpr int kV = HD / 32;  // 2 or 4
        const int d = lane * kV, c = d / 8;
#pragma unroll 8
        for (int r = part; r < part + 32; ++r) {
            const bool in = r < n && d < A.hd;
            const float* from = reinterpret_cast<const float*>(A.q) + (in ? source(r) + d : 0);
            float v[kV], mx = 0.f;
            if constexpr (kV == 4) {
                const float4 w = in ? __ldg(reinterpret_cast<const float4*>(from))
                                    : make_float4(0.f, 0.f, 0.f, 0.f);
                v[0] = w.x, v[1] = w.y, v[2] = w.z, v[3] = w.w;
            } else {
                const float2 w = in ? __ldg(reinterpret_cast<const float2*>(from))
                                    : make_float2(0.f, 0.f);
                v[0] = w.x, v[1] = w.y;
            }
#pragma unroll
            for (int i = 0; i < kV; ++i) mx = fmaxf(mx, fabsf(v[i]));
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(kAll, mx, o));
            const uint32_t e = (__float_as_uint(mx) >> 23) & 255u;
            const bool scaled = std::is_same<T, __half>::value && e > 0 && e < 254;
            const float inv = (scaled ? __uint_as_float((254u - e) << 23) : 1.f) * (flip ? -1.f : 1.f);
            if (lane == 0) s_fac[r] = scaled ? __uint_as_float(e << 23) : 1.f;
            char* to = tile + (c / 8) * (kM * 128) + r * 128 + (((c & 7) ^ (r & 7)) * 16) + (d & 7) * 2;
#pragma unroll
            for (int i = 0; i < kV; ++i) v[i] *= inv;
#pragma unroll
            for (int p = 0; p < PARTS; ++p) {
                uint32_t w[kV / 2];
#pragma unroll
                for (int i = 0; i < kV / 2; ++i) {
                    w[i] = PMath<T>::pack(v[2 * i], v[2 * i + 1]);
                    const float2 f = PMath<T>::unpack(w[i]);
                    v[2 * i] -= f.x;
                    v[2 * i + 1] -= f.y;
                }
                if constexpr (kV == 4)
                    *reinterpret_cast<uint2*>(to + p * C::kQ) = make_uint2(w[0], w[1]);
                else
                    *reinterpret_cast<uint32_t*>(to + p * C::kQ) = w[0];
            }
        }
    }
}

template <typename T, int PARTS, int HD>
__global__ void __launch_bounds__(kThreads, 1)
paged_mma_kernel(const __grid_constant__ PagedArgs A, const __grid_constant__ KvMaps maps,
                 const __grid_constant__ CUtensorMap q_map, int which, int box_rows, int q_boxes) {
    using C = MCfg<HD, PARTS>;
    constexpr int kRT = C::kRT, kSlots = C::kSlots, kH = C::kHalves;
    constexpr bool SPLIT = PARTS > 1;
    constexpr int kType = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
    extern __shared__ char raw[];
    char* base = reinterpret_cast<char*>(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    constexpr int kQB = C::kQBufs;
    char* sQ = base;                                // [kQB][kRT][PARTS][kH][128 rows][128 B]
    char* sKV = base + kQB * kRT * PARTS * C::kQ;   // [kSlots][kH][64 rows][128 B]
    __shared__ uint64_t full[kSlots], empty[kSlots], v_load[kSlots], v_seen[kSlots];
    __shared__ uint64_t q_full[kRT][kQB], q_empty[kRT][kQB], s_full[kRT][2], p_full[kRT][2], o_done[kRT][2], drain[kRT];
    __shared__ uint32_t s_tmem;
    __shared__ uint64_t x_done[2], x_read[2];  // both halves of an item: sums there, O read
    __shared__ float2 s_ml[2][kM];
    __shared__ float s_fac[kRT][kQB][kM];  // fp32 rows: score factors
    __shared__ Waits s_wait;
    __shared__ int s_bad;
    // (the shuffle tells the compiler that the warp number is the same for all lanes)
    const int tid = threadIdx.x, warp = __shfl_sync(kAll, tid >> 5, 0), lane = tid & 31;
    const PagedPlan& P = A.plan[which];
    const int head_lane = blockIdx.x % P.heads, piece = blockIdx.x / P.heads;
    const int kvh = head_lane / P.hblocks, hb = head_lane - kvh * P.hblocks;
    const int h0 = kvh * A.group + hb * P.gpb, gpb = min(P.gpb, A.group - hb * P.gpb);

    if (tid == 0) {
        for (int i = 0; i < kSlots; ++i) {
            bar_init(&full[i], 1);
            bar_init(&empty[i], kRT);
            bar_init(&v_load[i], 1);
            bar_init(&v_seen[i], 1);
        }
        for (int x = 0; x < kRT; ++x) {
            for (int b = 0; b < kQB; ++b) {
                bar_init(&q_full[x][b], SPLIT ? 4 : 1);
                bar_init(&q_empty[x][b], SPLIT ? 5 : 1);
            }
            for (int b = 0; b < 2; ++b) {
                bar_init(&o_done[x][b], 1);
                bar_init(&s_full[x][b], 1);
                bar_init(&p_full[x][b], 4);
            }
        }
        for (int x = 0; x < kRT; ++x) bar_init(&drain[x], 1);
        for (int x = 0; x < 2; ++x) {
            bar_init(&x_done[x], 4);
            bar_init(&x_read[x], 4);
        }
        s_wait.out = 0;
        s_wait.limit = A.wait_ns;
        s_bad = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                         smem_addr(&s_tmem))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = s_tmem;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    Walk W;
    {
        const int n_items = *P.n_items, total = n_items ? P.cum[n_items] : 0;
        const Pieces pieces(P, max(total, 1));
        W.x = W.x_end = 0;
        if (total > 0 && piece < pieces.n) {
            W.x = pieces.start(piece);
            W.x_end = pieces.start(piece + 1);
        }
        W.item = n_items ? block_last_le(P.cum, n_items, W.x) : 0;
        if (tid == 0) {
            P.bad[blockIdx.x] = 0;
            if (head_lane == 0) {
                PagedSplit sp{0, 0, 0, -1, 0, 0};
                // the items whose first KV tile lies in this piece
                sp.item0 = W.item + (n_items && W.x < W.x_end && P.cum[W.item] + P.lead < W.x);
                sp.item1 = sp.item0;
                if (W.x < W.x_end) {
                    int last = last_le(P.cum, n_items, W.x_end - 1);
                    last -= P.cum[last] + P.lead >= W.x_end;
                    sp.item1 = max(sp.item0, last + 1);
                    if (last >= sp.item0 && P.cum[last + 1] > W.x_end && A.n_groups == 0) {
                        const PagedItem it = P.items[last];
                        const int to = Walk::last_piece(pieces, P.cum[last] + P.lead,
                                                        item_shift(P, it), it.n_tiles);
                        if (to > piece) {
                            sp.tok0 = it.tok0;
                            sp.n_rows = it.ntok * P.gpb;
                            sp.last = to;
                            sp.item = last;
                        }
                    }
                }
                P.split[piece] = sp;
            }
        }
    }

    // The product with V of row tile x's c-th KV tile is done.  (A barrier for odd and one for
    // even tiles: a waiter may be two tiles ahead, where one barrier's parity would repeat.)
    auto pv_done = [&](int x, uint32_t c) {
        return bar_wait(&o_done[x][c & 1], (c >> 1) & 1, &s_wait);
    };
    // Whether both row tiles' roles work on one item of at most kM rows (even and odd KV tiles).
    auto halved = [&]() { return kRT == 2 && W.it.ntok * gpb <= kM && W.b - W.a >= 2; };
    uint32_t ring = 0;  // K / V tiles so far: slot ring % kSlots, phase (ring / kSlots) & 1
    // Is some of KV tile i of the item hidden from some row?  V of these tiles is looked through.  The
    // c-th such tile of the piece has its load behind it with v_load[c % kSlots] (a wait for `full`
    // any earlier could meet an older phase of its parity) and its look with v_seen[c % kSlots].
    // Its slot is released only behind both, and the tile kSlots before has been when it is loaded.
    const int sinks = A.window > 0 ? A.sinks : 0;
    auto hides = [&](int i) {
        const int j0 = W.tile(i) * kN;
        return !(j0 >= W.it.kv_lo && j0 + kN <= W.all_hi && (j0 >= W.all_lo || j0 + kN <= sinks));
    };
    // (the same for the warps that move and multiply tiles: with the rule in full for each tile four
    // drafted tokens behind 64K to 128K positions took 2 to 4% longer)
    auto hides_some = [&](int i) { return !(i >= W.w0 && i < W.w1) && hides(i); };
    uint32_t looks = 0;  // such tiles so far
    auto looked = [&]() {
        return bar_wait_warp(&v_seen[looks % kSlots], (looks / kSlots) & 1, &s_wait);
    };
    if (warp == kLoadWarp) {
        // ------------------------------------------------------------- K / V tiles
        const int per_half = kN / box_rows, boxes = per_half * kH;
        const int half = lane / per_half, rb = lane - half * per_half;
        bool ok = true;
        while (ok && W.next(A, P)) {
            // this lane's page and row of a tile's box
            auto place = [&](int i) {
                return lane < boxes
                           ? box_place(A, W.it, W.tile(i) * kN, rb, box_rows, &s_bad)
                           : make_int2(0, 0);
            };
            int2 at = place(W.a);
            for (int i = W.a; ok && i < W.b; ++i) {
                const int2 cur = at;
                if (i + 1 < W.b) at = place(i + 1);
#pragma unroll
                for (int kv = 0; kv < 2; ++kv, ++ring) {
                    const int s = ring % kSlots;
                    if (!bar_wait_warp(&empty[s], ((ring / kSlots) & 1) ^ 1, &s_wait)) {
                        ok = false;
                        break;
                    }
                    if (lane == 0) bar_expect(&full[s], C::kSlot);
                    __syncwarp();
                    if (lane < boxes)
                        tma4d(smem_addr(sKV + s * C::kSlot + half * (kN * 128) + rb * box_rows * 128),
                              kv ? &maps.v : &maps.k, half * 64, kvh, cur.y, cur.x, &full[s]);
                }
                if (ok && hides_some(i)) {
                    if (lane == 0) bar_arrive(&v_load[looks % kSlots]);
                    ++looks;
                }
            }
        }
        __syncwarp();
        // (only after a timeout can some of these still be in flight)
        if (lane == 0)
            for (uint32_t i = ring > kSlots ? ring - kSlots : 0; i < ring; ++i)
                bar_drain(&full[i % kSlots], (i / kSlots) & 1);
    } else if (warp >= kMmaWarp && warp < kMmaWarp + kRT) {
        // ------------------------------------------------------------- products of a row tile
        const int x = warp - kMmaWarp;
        const uint32_t leader = elect_one();
        const uint32_t qd0 = desc_k(smem_addr(sQ) + x * PARTS * C::kQ);
        const uint32_t kd = desc_k(smem_addr(sKV)), vd = desc_mn(smem_addr(sKV), kN * 128);
        bool ok = true;
        uint32_t seg = 0, cnt = 0;  // segments, KV tiles of this row tile so far
        auto arrive_full = [&](uint32_t i) {
            return bar_wait_warp(&full[i % kSlots], (i / kSlots) & 1, &s_wait);
        };
        auto commit = [&](uint64_t* bar) {
            if (leader) mma_commit(bar);
            __syncwarp();
        };
        auto issue_s = [&](uint32_t slot, uint32_t c, uint32_t qb) {
            const uint32_t qd = qd0 + qb * (kRT * PARTS * C::kQ >> 4);
            const uint32_t d = tmem + C::s_col(x, c & 1), k0 = kd + slot * (C::kSlot >> 4);
#pragma unroll
            for (int p = 0; p < PARTS; ++p)
#pragma unroll
                for (int k = 0; k < HD / 16; ++k)
                    mma_ss(d, qd + ((p * C::kQ + (k / 4) * (kM * 128) + (k % 4) * 32) >> 4),
                           k0 + (((k / 4) * (kN * 128) + (k % 4) * 32) >> 4), idesc(kType, kN, 0),
                           (p | k) ? 1u : 0u, leader);
            commit(&s_full[x][c & 1]);
        };
        auto release = [&](uint32_t first, uint32_t slots) {  // what the other row tile reads
            for (uint32_t i = first; i < first + slots; ++i) {
                if (!arrive_full(i)) return false;
                if (lane == 0) bar_arrive(&empty[i % kSlots]);
            }
            return true;
        };
        for (; ok && W.next(A, P); ring += 2 * (W.b - W.a)) {
            const int n = W.b - W.a;
            const bool half = halved();
            if (!half && x * kM >= W.it.ntok * gpb) {  // no rows here
                for (int i = W.a; i < W.b; ++i) looks += hides_some(i);
                ok = release(ring, 2 * n);
                continue;
            }
            const int step = half ? 2 : 1, first = half ? x : 0, own = half ? (n - x + 1) / 2 : n;
            const uint32_t qb = seg % kQB, r0 = ring + 2 * first;
            // S of tile c takes the buffer of tile c - 2's P
            ok = (first == 0 || release(ring, 2)) &&
                 bar_wait_warp(&q_full[x][qb], (seg / kQB) & 1, &s_wait) && arrive_full(r0) &&
                 (cnt < 2 || __all_sync(kAll, pv_done(x, cnt - 2)));
            if (!ok) break;
            ++seg;
            if (first) looks += hides_some(W.a);
            tc_after();
            issue_s(r0 % kSlots, cnt, qb);
            commit(&empty[r0 % kSlots]);
            if (own == 1) commit(&q_empty[x][qb]);
            for (int j = 0; j < own; ++j, ++cnt) {
                const uint32_t rv = r0 + 2 * j * step + 1, rk = rv + 2 * step - 1;
                if (j + 1 < own) {
                    ok = (cnt == 0 || __all_sync(kAll, pv_done(x, cnt - 1))) &&
                         (!half || release(rv + 1, 2)) && arrive_full(rk);
                    if (!ok) break;
                    tc_after();
                    issue_s(rk % kSlots, cnt + 1, qb);
                    commit(&empty[rk % kSlots]);
                    if (j + 2 == own) commit(&q_empty[x][qb]);
                }
                const int i = W.a + first + j * step;
                const bool hidden = hides_some(i);
                ok = bar_wait_warp(&p_full[x][cnt & 1], (cnt >> 1) & 1, &s_wait) &&
                     arrive_full(rv) && (!hidden || looked());
                if (!ok) break;
                looks += hidden + (half && i + 1 < W.b && hides_some(i + 1));
                tc_after();
                const uint32_t d = tmem + C::o_col(x);
                const uint32_t v0 = vd + (rv % kSlots) * (C::kSlot >> 4);
#pragma unroll
                for (int p = 0; p < PARTS; ++p) {
                    const uint32_t a0 = tmem + C::p_col(x, 0, p) +
                                        (cnt & 1) * (C::p_col(x, 1, p) - C::p_col(x, 0, p));
#pragma unroll
                    for (int k = 0; k < kN / 16; ++k)
                        mma_ts(d, a0 + k * 8, v0 + ((k * 16 * 128) >> 4), idesc(kType, HD, 1),
                               p || k ? 1u : (uint32_t)(SPLIT ? j % kFlush > 0 : j > 0), leader);
                }
                commit(&o_done[x][cnt & 1]);
                commit(&empty[rv % kSlots]);
            }
            if (ok && half && (first + own * 2 - 1) < n) ok = release(ring + 2 * (first + own * 2 - 1), 2);
        }
        commit(&drain[x]);
        if (lane == 0) bar_drain(&drain[x], 0);
        __syncwarp();
    } else if (warp == kRowWarp || (SPLIT && warp >= 4 && warp < 8)) {
        // ------------------------------------------------------------- rows of Q, a look at V
        const bool rows = !SPLIT || warp < 8;
        const bool flip = A.scale_log2 < 0.f;  // q takes the sign, so that the factor is >= 0
        uint32_t seg[kRT] = {};
        bool ok = true;
        for (; ok && W.next(A, P); ring += 2 * (W.b - W.a)) {
            const PagedItem& it = W.it;
            const int n_rows = it.ntok * gpb;
#pragma unroll
            for (int x = 0; x < kRT; ++x) {
                const int row0 = halved() ? 0 : x * kM;
                if (!ok || !rows || row0 >= n_rows) continue;
                const uint32_t qb = seg[x] % kQB;
                ok = bar_wait_warp(&q_empty[x][qb], ((seg[x] / kQB) & 1) ^ 1, &s_wait);
                if (!ok) continue;
                ++seg[x];
                if (q_boxes) {
                    if (lane == 0) {
                        bar_expect(&q_full[x][qb], C::kQ);
#pragma unroll
                        for (int h = 0; h < kH; ++h)
                            tma3d(smem_addr(sQ + (qb * kRT + x) * C::kQ + h * (kM * 128)), &q_map,
                                  h * 64, h0, it.tok0 + row0 / gpb, &q_full[x][qb]);
                    }
                    continue;
                }
                const int n = min(kM, n_rows - row0);
                load_q_tile<T, PARTS, HD>(A, it.tok0, row0, n, h0, gpb, flip,
                                          sQ + (qb * kRT + x) * PARTS * C::kQ, s_fac[x][qb],
                                          SPLIT ? (warp - 4) * 32 : 0);
                async_fence();
                __syncwarp();
                if (lane == 0) bar_arrive(&q_full[x][qb]);
            }
            if (warp != kRowWarp) continue;
            // No infinity or NaN of a partly hidden tile may meet a zero weight: zeros take their
            // places, and where some row sees one the join works the item out again without tiles.
            // (One warp for both row tiles: with each of them looking for itself nothing ordered the
            // zeros that one had written before the other's product.)
            const int any_hi = min(it.kv_hi, it.pmax + 1);
            const int any_lo = A.window > 0 ? it.pmin - A.window + 1 : INT_MIN;
            for (int i = W.a; i < W.b; ++i) {
                if (!hides_some(i)) continue;
                const uint32_t rv = ring + 2 * (i - W.a) + 1;
                ok = bar_wait_warp(&v_load[looks % kSlots], (looks / kSlots) & 1, &s_wait) &&
                     bar_wait_warp(&full[rv % kSlots], (rv / kSlots) & 1, &s_wait);
                if (!ok) break;
                const int j0 = W.tile(i) * kN;
                char* vt = sKV + (rv % kSlots) * C::kSlot;
                uint32_t found = 0;
#pragma unroll 8
                for (int c = lane; c < kN * HD / 8; c += 32) {
                    const uint4 v = *reinterpret_cast<const uint4*>(vt + c * 16);
                    found |= odd_halves<T>(v.x) | odd_halves<T>(v.y) | odd_halves<T>(v.z) |
                             odd_halves<T>(v.w);
                }
                if (found) {
                    for (int c = lane; c < kN * HD / 8; c += 32) {
                        uint4* at = reinterpret_cast<uint4*>(vt + c * 16);
                        const uint4 v = *at;
                        if (!(odd_halves<T>(v.x) | odd_halves<T>(v.y) | odd_halves<T>(v.z) |
                              odd_halves<T>(v.w)))
                            continue;
                        const int p = j0 + ((c / 8) & (kN - 1));
                        if (p >= it.kv_lo && p < any_hi && (p >= any_lo || p < sinks))
                            P.redo[(size_t)(W.item - 1) * P.heads + head_lane] = 1;
                        *at = make_uint4(0, 0, 0, 0);
                    }
                    async_fence();
                }
                __syncwarp();
                if (lane == 0) bar_arrive(&v_seen[looks % kSlots]);
                ++looks;
            }
        }
        if (q_boxes && lane == 0)  // (only after a timeout can some of these still be in flight)
#pragma unroll
            for (int x = 0; x < kRT; ++x)
                for (uint32_t i = seg[x] > (uint32_t)kQB ? seg[x] - kQB : 0; i < seg[x]; ++i)
                    bar_drain(&q_full[x][i % kQB], (i / kQB) & 1);
        __syncwarp();
    } else if (warp < 4 * kRT) {
        // ------------------------------------------------------------- softmax of a row tile
        const int x = warp >> 2, r = (warp & 3) * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        constexpr float kShift = MShift<T>::value;
        uint32_t cnt = 0, seg = 0, pairs = 0;
        bool ok = true;
        while (ok && W.next(A, P)) {
            const PagedItem& it = W.it;
            const int n_rows = it.ntok * gpb, n = W.b - W.a;
            const bool half = halved();
            if (!half && x * kM >= n_rows) continue;
            const int step = half ? 2 : 1, first = half ? x : 0, own = half ? (n - x + 1) / 2 : n;
            const int row0 = half ? 0 : x * kM, row = row0 + r;
            const bool real = row < n_rows;
            const int tok = it.tok0 + row / gpb, h = h0 + row % gpb;
            int pos = INT_MIN;
            if (real) pos = it.mixed ? token_position(A, tok) : it.pos0 + row / gpb;
            float fac = fabsf(A.scale_log2);
            if (SPLIT) {
                const uint32_t qb = seg % kQB;
                if (!bar_wait_warp(&q_full[x][qb], (seg / kQB) & 1, &s_wait)) {
                    ok = false;
                    break;
                }
                fac *= s_fac[x][qb][r];
                __syncwarp();
                if (lane == 0) bar_arrive(&q_empty[x][qb]);
            }
            ++seg;
            fac = fmaxf(fac, 1e-37f);  // (0 would make NaNs of hidden scores)
            const int hi_row = real ? min(it.kv_hi, pos + 1) : 0;
            const int lo_row = real && A.window > 0 ? pos - A.window + 1 : INT_MIN;
            float m = -INFINITY, l = 0.f;
            // A warp without rows only keeps step: what P holds for it reaches no row that is read.
            // (In a loop of its own: as a branch of the next one it cost prompts 5%.)
            const bool idle = row0 + (warp & 3) * 32 >= n_rows;
            for (int j = 0; idle && j < own; ++j, ++cnt) {
                const int b = cnt & 1;
                ok = bar_wait_warp(&s_full[x][b], (cnt >> 1) & 1, &s_wait);
                if (!ok) break;
                __syncwarp();
                if (lane == 0) bar_arrive(&p_full[x][b]);
            }
            for (int j = 0; !idle && j < own; ++j, ++cnt) {
                const int b = cnt & 1, i0 = W.a + first + j * step, j0 = W.tile(i0) * kN;
                const bool whole = !hides(i0);
                if (!bar_wait_warp(&s_full[x][b], (cnt >> 1) & 1, &s_wait)) {
                    ok = false;
                    break;
                }
                tc_after();
                float s[kN];
                tmem_ld64(lanes + C::s_col(x, b), s);
                if (!whole) {
                    // this row's visible places as bits
                    uint64_t seen = below(hi_row - j0) & ~below(lo_row == INT_MIN ? 0 : lo_row - j0);
                    if (sinks) seen |= below(min(sinks, hi_row) - j0);
                    seen &= ~below(it.kv_lo - j0);
                    const uint32_t w[2] = {(uint32_t)seen, (uint32_t)(seen >> 32)};
#pragma unroll
                    for (int i = 0; i < kN; ++i)
                        if (!((w[i / 32] >> (i % 32)) & 1u)) s[i] = -INFINITY;
                }
                float mx4[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) mx4[i] = max3(s[i], s[i + 4], s[i + 8]);
#pragma unroll
                for (int i = 12; i < kN - 4; i += 8)
#pragma unroll
                    for (int u = 0; u < 4; ++u) mx4[u] = max3(mx4[u], s[i + u], s[i + 4 + u]);
                const float mx =
                    max3(max3(mx4[0], s[kN - 4], s[kN - 3]), max3(mx4[1], s[kN - 2], s[kN - 1]),
                         fmaxf(mx4[2], mx4[3])) * fac;
                const bool flush = SPLIT && j > 0 && j % kFlush == 0;
                if (flush || __any_sync(kAll, mx > m + 8.f)) {
                    const float to = fmaxf(m, mx);
                    const float al = ex2(m - (to == -INFINITY ? 0.f : to));
                    m = to;
                    l *= al;
                    if (j > 0) {
                        if (!__all_sync(kAll, pv_done(x, cnt - 1))) {
                            ok = false;
                            break;
                        }
                        tc_after();
#pragma unroll 1
                        for (int c = 0; c < HD; c += 32) {
                            float o[32];
                            tmem_ld32(lanes + C::o_col(x) + c, o);
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] *= al;
                            if (!flush)
                                tmem_st32(lanes + C::o_col(x) + c, reinterpret_cast<uint32_t*>(o));
                            if (SPLIT && (flush || j > kFlush)) {
                                // the sums up to the last multiple of kFlush, and O at the next
                                float sum[32];
                                if (j > kFlush) tmem_ld32(lanes + C::kSumCol + c, sum);
#pragma unroll
                                for (int i = 0; i < 32; ++i)
                                    sum[i] = (j > kFlush ? sum[i] * al : 0.f) + (flush ? o[i] : 0.f);
                                tmem_st32(lanes + C::kSumCol + c, reinterpret_cast<uint32_t*>(sum));
                            }
                        }
                    }
                }
                const float mb = (m == -INFINITY ? 0.f : m) - kShift;
                // (pairs of fp32 in one instruction: these warps are short of issue slots)
                const uint64_t fac2 = pair(fac, fac), mb2 = pair(-mb, -mb);
                uint64_t l2[2] = {0, 0};
#pragma unroll
                for (int i = 0; i < kN; i += 2) {
                    unpair(fma2(pair(s[i], s[i + 1]), fac2, mb2), s[i], s[i + 1]);
                    s[i] = ex2(s[i]);
                    s[i + 1] = ex2(s[i + 1]);
                    l2[(i / 2) & 1] = add2(l2[(i / 2) & 1], pair(s[i], s[i + 1]));
                }
                {
                    float a, b;
                    unpair(add2(l2[0], l2[1]), a, b);
                    l += a + b;
                }
#pragma unroll
                for (int p = 0; p < PARTS; ++p) {
                    uint32_t w[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        w[i] = PMath<T>::pack(s[2 * i], s[2 * i + 1]);
                        if (p + 1 < PARTS) {
                            const float2 f = PMath<T>::unpack(w[i]);
                            s[2 * i] -= f.x;
                            s[2 * i + 1] -= f.y;
                        }
                    }
                    tmem_st32(lanes + C::p_col(x, b, p), w);
                }
                tmem_wait_st();
                tc_before();
                __syncwarp();
                if (lane == 0) bar_arrive(&p_full[x][b]);
            }
            if (!ok) break;
            // the rows of this piece of the item
            if (!__all_sync(kAll, pv_done(x, cnt - 1))) {
                ok = false;
                break;
            }
            tc_after();
            const bool complete = W.a == 0 && W.b == it.n_tiles;
            const bool last_word = complete && A.n_groups == 0;
            float mine = 1.f, other = 0.f;  // factors of this row tile's O and of the other one's
            if (half) {
                s_ml[x][r] = make_float2(m, l);
                tc_before();
                __syncwarp();
                if (lane == 0) bar_arrive(&x_done[x]);
                if (!bar_wait_warp(&x_done[1 - x], pairs & 1, &s_wait)) {
                    ok = false;
                    break;
                }
                tc_after();
                const float2 o = s_ml[1 - x][r];
                const float to = fmaxf(m, o.x), base = to == -INFINITY ? 0.f : to;
                mine = ex2(m - base);
                other = ex2(o.x - base);
                m = to;
                l = l * mine + o.y * other;
            }
            const float inv = l == 0.f ? 0.f : 1.f / l;
            const float M = m - kShift;
            const bool tells = !half || x == 0;  // one of two halves writes what is per row
            char* dst;  // this row's place
            if (last_word) {
                const size_t at = (size_t)tok * A.out_stride + (size_t)h * A.hd;
                dst = reinterpret_cast<char*>(A.out) + at * (SPLIT ? 4 : 2);
                if (real && tells && A.lse) A.lse[(size_t)tok * A.nh + h] = row_lse(M, l);
            } else {
                const size_t id = complete ? (size_t)(which == PLAN_PREFIX) * A.n_tokens * A.nh +
                                                 (size_t)tok * A.nh + h
                                           : part_row(P, piece, head_lane, W.a > 0 ? 0 : 1, row);
                dst = reinterpret_cast<char*>((complete ? A.full_o : P.part_o) + id * A.hd);
                if (real && tells)
                    *reinterpret_cast<float2*>((complete ? A.full_ml : P.part_ml) + id * 2) =
                        make_float2(M, l);
            }
            if (A.n_groups > 0 && W.a == 0 && head_lane == 0 && real && tells && h == h0) {
                const int last =
                    Walk::last_piece(Pieces(P, P.cum[*P.n_items]), W.c0, W.sh, it.n_tiles);
                P.where[tok] = PagedWhere{piece, last, row, it.alone, which, W.item - 1};
            }
            // A lane writes whole sectors of its own row (32 bytes in one store: 3350 cycles an item
            // of 256 rows of 128, 4850 through shared memory with two lanes to a sector).
            const bool halves = !SPLIT && last_word;
            const bool wide = (reinterpret_cast<uintptr_t>(dst) & 31) == 0;
            auto send = [&](int d, const uint32_t* w) {  // 8 words of this row from dim d on
                if (!real || d >= A.hd) return;
                char* to = dst + d * (halves ? 2 : 4);
                if (wide && d + (halves ? 16 : 8) <= A.hd) {
                    store32(to, w);
                } else {
                    *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
                    if (!halves || d + 8 < A.hd)
                        *reinterpret_cast<uint4*>(to + 16) = make_uint4(w[4], w[5], w[6], w[7]);
                }
            };
#pragma unroll 1
            for (int c = half ? x * (HD / 2) : 0; c < (half ? (x + 1) * (HD / 2) : HD); c += 32) {
                float o[32];
                tmem_ld32(lanes + C::o_col(x) + c, o);
                if (SPLIT && own > kFlush) {
                    float sum[32];
                    tmem_ld32(lanes + C::kSumCol + c, sum);
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] += sum[i];
                }
                if (half) {
                    float p[32];
                    tmem_ld32(lanes + C::o_col(kRT - 1 - x) + c, p);
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = fmaf(o[i], mine, p[i] * other);
                }
                if (last_word) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = l == 0.f ? 0.f : o[i] * inv;
                }
                if (halves) {
                    uint32_t w[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) w[i] = PMath<T>::pack(o[2 * i], o[2 * i + 1]);
                    send(c, w);
                    send(c + 16, w + 8);
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        send(c + 8 * k, reinterpret_cast<const uint32_t*>(o + 8 * k));
                }
            }
            tc_before();
            if (half) {  // neither O is written again before both have been read
                __syncwarp();
                if (lane == 0) bar_arrive(&x_read[x]);
                if (!bar_wait_warp(&x_read[1 - x], pairs & 1, &s_wait)) {
                    ok = false;
                    break;
                }
                ++pairs;
            }
        }
    }

    tc_before();
    __syncthreads();
    if (tid == 0 && (s_bad || s_wait.out)) P.bad[blockIdx.x] = s_bad | (s_wait.out ? PG_TIMEOUT : 0);
    if (warp == kMmaWarp) {
        tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem)
                     : "memory");
    }
}

template <typename T, int PARTS, int HD>
cudaError_t launch_one(const PagedArgs& A, int which, cudaStream_t s) {
    auto kern = paged_mma_kernel<T, PARTS, HD>;
    constexpr int smem = MCfg<HD, PARTS>::kSmem;
    static std::atomic<uint64_t> done{0};
    cudaError_t e = smem_opt_in(reinterpret_cast<const void*>(kern), smem, done);
    if (e != cudaSuccess) return e;
    KvMaps maps;
    const bool bf16 = std::is_same<T, __nv_bfloat16>::value;
    const int rows = kv_maps(&maps, A, bf16, kN);
    if (rows == 0) return cudaErrorInvalidValue;
    const PagedPlan& P = A.plan[which];
    // Q by TMA where a row tile is whole tokens of whole blocks of heads
    const bool q_boxes = PARTS == 1 && kM % P.gpb == 0 && A.group % P.gpb == 0 && A.scale_log2 >= 0.f;
    CUtensorMap q_map = maps.k;
    if (q_boxes && !encode_rows(&q_map, A, bf16, P.gpb, kM / P.gpb)) return cudaErrorInvalidValue;
    return launch_pdl(kern, dim3(P.heads * P.lanes), dim3(kThreads), (size_t)smem, s, A, maps, q_map,
                      which, rows, (int)q_boxes);
}

template <typename T, int PARTS>
cudaError_t launch_hd(const PagedArgs& A, int which, cudaStream_t s) {
    return A.hd <= 64 ? launch_one<T, PARTS, 64>(A, which, s) : launch_one<T, PARTS, 128>(A, which, s);
}

}  // namespace

// Head dims that the tensor-core kernel takes: one or two boxes of 64, the last possibly cut.
bool paged_mma_takes(int hd) { return hd <= 128; }
int paged_mma_rows(bool split) { return split ? kM : 2 * kM; }

cudaError_t launch_paged_mma(const PagedArgs& A, int which, int q_dtype, int kv_dtype,
                             cudaStream_t s) {
    const bool split = q_dtype == WISP_DTYPE_F32;
    if (kv_dtype == WISP_DTYPE_F16)
        return split ? launch_hd<__half, 2>(A, which, s) : launch_hd<__half, 1>(A, which, s);
    return split ? launch_hd<__nv_bfloat16, 3>(A, which, s)
                 : launch_hd<__nv_bfloat16, 1>(A, which, s);
}

}  // namespace wb
