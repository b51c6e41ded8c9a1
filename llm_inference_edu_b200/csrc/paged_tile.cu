// Attention of many rows (prompt chunks) over the paged cache on the
// tcgen05 tensor cores, one CTA an item.
//
// The packed rows of one sequence and KV head (token-major, the group's
// query heads innermost) are the M = 128 of the MMAs, so a group of seven
// heads fills the tile and the causal edge of 128 rows is only 18 tokens
// long.  Two softmax streams alternate on the tensor cores: while one
// exponentiates its scores, the products of the other run.
//   rows > 128 (BF16 values): each stream has its own 128 rows and both use
//     every key tile, so a key tile is loaded once for 256 rows;
//   otherwise: both streams have the same rows and take every other key tile;
//     their results are joined at the end.
// Per key tile of a stream: S = Q K^T into tensor memory; each thread of the
// stream's warpgroup owns a row, finds the maximum (which may lag by 2^8, so
// O is rarely rescaled), writes the weights back over S as the bf16 A
// operand of O += P V, and keeps the row's sum in FP32.
// BF16 caches.  FP32 values: Q and the weights are three bf16 planes (exact
// to 2^-24) and a key tile has 64 keys, so that three planes fit beside S.
// BF16 values: one plane each; the weights' single rounding (2^-8 of each at
// most) is of the size of the result's own.
// INT8 caches: pages are copied raw and widened to f16 by a warpgroup; two
// planes of FP32 values, one of BF16 values (paged_attn.cuh).  Their scales
// multiply scores and weights in the softmax.  509 tokens behind 2,999 and 23
// single ones, 28/4 heads of 128, FP32: 132 us, 8 of them for looking at each
// key's own weight and V row where a base rises (once a stream as a rule).
// Such rare code waits for its instructions: a warp stands two cycles without
// one for each that it issues, so it is kept short.
// FP32 values: each tile's product is gathered in FP32 by a warpgroup.
// K tiles are K-major operands as TMA leaves them (128-byte swizzle, a box a
// page); V tiles are the MN-major operand in the same layout.
// 4,096 tokens behind 4,096, 28/4 heads of 128, BF16: 370 us, 975 TFLOP/s.
// A stream's softmax takes 1.7 k cycles a tile and its products 1.1 k, with
// the other stream's in between: neither pipe is full.
// Every wait is bounded: a role that gives up raises the abort flag, copies
// and MMAs in flight are drained, TMEM is freed and the item's rows are NaN.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <atomic>
#include <mutex>

#include "paged_attn.cuh"

namespace qb {
namespace paged {
namespace {

constexpr unsigned long long kWaitNs = 2000000000ull;

template <typename TV, typename TC, int HD_>
struct Tile {
    static constexpr bool kInt8 = sizeof(TC) == 1;
    static constexpr int HD = HD_;
    static constexpr bool kWide = sizeof(TV) == 4;
    static constexpr int NP = kWide ? (kInt8 ? 2 : 3) : 1;  // planes of Q and of the weights
    static constexpr int KT = NP == 3 ? 64 : 128;           // keys a tile
    static constexpr int QT = kWide ? 1 : 2;                // row tiles an item may have
    static constexpr int PN = HD / 64;                  // 64-element panels of a row
    static constexpr int kTileBytes = KT * HD * 2;
    static constexpr int kQBytes = QT * NP * PN * 128 * 128;
    // Operand stages of each ring, raw INT8 pieces of 64 keys, scale slots.
    static constexpr int NS = kTileBytes == 32768 ? 2 : kWide && HD == 128 ? 3 : 4;
    static constexpr int kPiece = 64 * HD;
    static constexpr int RS = kInt8 ? (HD == 128 ? 3 : 4) : 0;
    static constexpr int D = kInt8 ? 4 : 0;
    // Warps: 8 softmax, K producer, MMA issuer, scale producer, TMEM and V producer;
    // 4 that gather O (FP32 values); 4 INT8 converters.
    static constexpr int kGather = 12, kConvert = kWide ? 16 : 12;
    static constexpr int kThreads = 384 + (kWide ? 128 : 0) + (kInt8 ? 128 : 0);
    // The launch's registers, split among the roles: the softmax holds its
    // scores (BF16 caches) and the gathering warps O.
    static constexpr int kLaunchRegs = 65536 / kThreads / 8 * 8;
    static constexpr int kSoftRegs = kWide ? (kInt8 ? 112 : 120) : kInt8 ? 168 : 216, kGatherRegs = kInt8 ? 168 : 176,
                         kOtherRegs = kWide ? (kInt8 ? 40 : 88) : kInt8 ? 88 : 72;
    static_assert(256 * kSoftRegs + (kWide ? 128 * kGatherRegs : 0) + (kThreads - (kWide ? 384 : 256)) * kOtherRegs <=
                      kThreads * kLaunchRegs,
                  "register split");
    // Columns of a stream: scores from 0 (KT of them), O from 128.  The
    // weights' operand starts over the scores.  Up to two planes: chunk ch of
    // 32 scores leaves 16 columns a plane where it was or before.  Three
    // planes (64 scores, all read before): 1 and 2 from column 64.
    static __host__ __device__ constexpr int chunk_col(int pl, int ch) {
        return NP == 3 ? (pl == 0 ? 0 : 32 + 32 * pl) + 16 * ch : 16 * (NP * ch + pl);
    }
    static __host__ __device__ constexpr int plane_col(int pl, int kb) { return chunk_col(pl, kb / 2) + kb % 2 * 8; }
    // Scores held between the maximum and the weights, where they fit.
    static constexpr bool kHold = !kInt8;
    static constexpr float kAbove = kInt8 ? kAboveBase : 0.0f;  // of the base the weights are taken against
    static constexpr size_t kv_off = kQBytes, raw_off = kv_off + (size_t)2 * NS * kTileBytes,
                            scl_off = raw_off + (size_t)RS * kPiece, max_off = scl_off + (size_t)D * 2 * KT * 4,
                            ctl_off = max_off + (kWide ? 2048 : 0);
    // The results' way out, behind what the streams leave each other.
    static constexpr int stage_off = HD == 128 ? 72 * 1024 : 40 * 1024;
    static_assert(128 * (HD + 4) * 4 + 2048 <= stage_off && stage_off + (kWide ? 4 : 8) * 4608 <= 2 * NS * kTileBytes, "stage");
    static constexpr size_t bytes = ctl_off + 2048 + 1024;
    static_assert(bytes <= 232448, "shared memory of a CTA");
};

// Barriers and flags, after the tiles.
struct Ctl {
    uint64_t q_full, done;
    uint64_t s_full[2], p_full[2][2], o_full[2], o_empty[2];
    uint64_t k_full[4], k_empty[4], v_full[4], v_empty[4];
    uint64_t raw_full[4], raw_empty[4], scl_full[4], scl_empty[4];
    uint32_t tmem;
    int abort_;
    uint8_t bad[256];
    float c[256];  // scale * log2(e) over the row's own scale (INT8 caches)
};
static_assert(sizeof(Ctl) <= 2048, "control block");

__device__ __forceinline__ bool wait_slow(uint64_t *bar, uint32_t parity, volatile int *abort_) {
    const uint64_t t0 = globaltimer_ns();
#pragma unroll 1
    for (unsigned it = 1;; ++it) {
        if (mbar_try_wait_suspend(bar, parity, 1000)) return true;
        if ((it & 15u) == 0 && (*abort_ || globaltimer_ns() - t0 > kWaitNs)) {
            *abort_ = 1;
            return false;
        }
    }
}
__device__ __forceinline__ bool wait(uint64_t *bar, uint32_t parity, Ctl *ctl) {
    return mbar_try_wait(bar, parity) || wait_slow(bar, parity, &ctl->abort_);
}
// Copies and MMAs already issued: bounded by time alone.
__device__ __forceinline__ bool wait_issued(uint64_t *bar, uint32_t parity) {
    const uint64_t t0 = globaltimer_ns();
#pragma unroll 1
    while (!mbar_try_wait_suspend(bar, parity, 1000))
        if (globaltimer_ns() - t0 > kWaitNs) return false;
    return true;
}

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// Issued by the elected lane of a converged warp: the whole warp walks the
// issue loop, so that the operands stay in uniform registers (in a one-lane
// branch each MMA cost 100 cycles to issue, twice its execution).
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r;
}
__device__ __forceinline__ void commit(uint64_t *bar, uint32_t leader) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_addr(bar)),
        "r"(leader)
        : "memory");
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc, uint32_t leader) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc), "r"(leader)
        : "memory");
}
// A from tensor memory (bf16 pairs along the columns).
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc, uint32_t leader) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc), "r"(leader)
        : "memory");
}
// By the elected lane of a converged warp, as the MMAs.
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap *m, int x, int y, uint32_t bar, uint32_t leader) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
        "\n\t}" ::"r"(dst),
        "l"((uint64_t)m), "r"(x), "r"(y), "r"(bar), "r"(leader)
        : "memory");
}

// All panels of a page at once (V).
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap *m, int y, uint32_t bar, uint32_t leader) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %4, 0;\n\t"
        "@q cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%5, %2, %5}], [%3];"
        "\n\t}" ::"r"(dst),
        "l"((uint64_t)m), "r"(y), "r"(bar), "r"(leader), "r"(0)
        : "memory");
}

#define QB_R8(v, o) "=r"(v[o]), "=r"(v[o + 1]), "=r"(v[o + 2]), "=r"(v[o + 3]), "=r"(v[o + 4]), "=r"(v[o + 5]), "=r"(v[o + 6]), "=r"(v[o + 7])
// 32 columns of this warp's 32 lanes; valid after wait_ld.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : QB_R8(v, 0), QB_R8(v, 8), QB_R8(v, 16), QB_R8(v, 24)
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
        "[%16];"
        : QB_R8(v, 0), QB_R8(v, 8)
        : "r"(taddr));
}
#undef QB_R8
#define QB_R8(v, o) "r"(v[o]), "r"(v[o + 1]), "r"(v[o + 2]), "r"(v[o + 3]), "r"(v[o + 4]), "r"(v[o + 5]), "r"(v[o + 6]), "r"(v[o + 7])
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16};" ::"r"(taddr),
        QB_R8(v, 0), QB_R8(v, 8)
        : "memory");
}
#undef QB_R8
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Shared-memory operand descriptors, 128-byte swizzle.  K-major: 8-row
// groups 1024 bytes apart.  MN-major: 64-element panels `panel` bytes apart,
// groups of 8 reduction rows 1024 bytes apart (16 rows, a page, a step).
__device__ __forceinline__ uint64_t desc_k(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ uint64_t desc_mn(uint32_t saddr, uint32_t panel) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(panel >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// BF16 or f16 operands, FP32 result, M = 128; b_mn: B is MN-major.
__host__ __device__ constexpr uint32_t idesc(int n, bool b_mn, bool f16) {
    return (1u << 4) | (f16 ? 0u : (1u << 7) | (1u << 10)) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}

// (a0, a1) * (b0, b1) + (c0, c1) in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
        "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
        "mul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
        "add.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

// The largest of three, NaN if one is.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// Two parts of a row's softmax: maximum, sum, and the parts' factors.
struct Join {
    float m, l, f0, f1;
};
__device__ __forceinline__ Join join(float m0, float l0, float m1, float l1) {
    Join j;
    j.m = fmaxf(m0, m1);
    const float base = j.m == -INFINITY ? 0.0f : j.m;
    const float h0 = m0 == base ? 1.0f : ex2_half(m0 - base), h1 = m1 == base ? 1.0f : ex2_half(m1 - base);
    j.f0 = h0 * h0;
    j.f1 = h1 * h1;
    j.l = l0 * h0 * h0 + l1 * h1 * h1;
    return j;
}

// 128 bytes of results (CB dimensions from d on) of this warp's 32 rows, a
// row a lane: as the item's part with its maximum and sum, or divided by the
// sum.  Results go through shared memory (`stage`, 32 rows 144 bytes apart),
// so that eight lanes write a row's 128 bytes (a lane a row: 80 against 75 us
// on 2,001 tokens under a window of 1,001, with Q's loads four at a time).
// An item that gave up (`fin` unset) leaves NaN, and not through shared
// memory, where copies may still be landing.
template <typename TV, int HD>
__device__ __forceinline__ void put_rows(const Args &a, const Item &it, const SeqRec &sq, int r, int d,
                                         float (&v)[128 / sizeof(TV)], float m, float l, bool fin, uint8_t *stage, int lane) {
    constexpr int CB = 128 / (int)sizeof(TV);
    if (!fin) l = __uint_as_float(0x7fffffffu);
    if (it.slot >= 0) {
        if (r >= it.rows) return;
#pragma unroll
        for (int e = 0; e < CB; e += 4)
            *(float4 *)(a.ws + it.slot + part_at(it.rows, HD, r, d + e, true)) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
        if (d == 0) {
            a.ws[it.slot + (size_t)it.rows * HD + r] = m;
            a.ws[it.slot + (size_t)it.rows * (HD + 1) + r] = l;
        }
        return;
    }
    const size_t at = row_at(a, sq, it.kvh, it.row0 + r, (size_t)a.H * HD) + d;
    const float inv = __fdiv_rn(1.0f, l);
#pragma unroll
    for (int e = 0; e < CB; ++e) v[e] *= inv;
    if (!fin || ((uintptr_t)a.y & 15)) {
        if (r < it.rows)
#pragma unroll
            for (int e = 0; e < CB; ++e) store_value((TV *)a.y, at + e, v[e]);
        return;
    }
    uint4 *mine = (uint4 *)(stage + lane * 144);
    __syncwarp();
#pragma unroll
    for (int x = 0; x < 8; ++x) {
        if constexpr (sizeof(TV) == 4)
            mine[x] = make_uint4(__float_as_uint(v[4 * x]), __float_as_uint(v[4 * x + 1]), __float_as_uint(v[4 * x + 2]),
                                 __float_as_uint(v[4 * x + 3]));
        else
            mine[x] = make_uint4(pack_bf16(v[8 * x], v[8 * x + 1]), pack_bf16(v[8 * x + 2], v[8 * x + 3]),
                                 pack_bf16(v[8 * x + 4], v[8 * x + 5]), pack_bf16(v[8 * x + 6], v[8 * x + 7]));
    }
    __syncwarp();
#pragma unroll
    for (int x = 0; x < 8; ++x) {
        const int from = x * 4 + lane / 8;
        const size_t to = __shfl_sync(0xffffffffu, (unsigned long long)at, from);
        if (r - lane + from < it.rows)
            *(uint4 *)((TV *)a.y + to + (lane & 7) * (16 / sizeof(TV))) = *(uint4 *)(stage + from * 144 + (lane & 7) * 16);
    }
}

// The order in which the tiles of both operands are produced: K one tile
// ahead of V.  Position x: K 0, K 1, V 0, K 2, V 1, ..., V n-1.
__device__ __forceinline__ void nth(int x, int n, bool &is_k, int &tile) {
    if (x == 0) {
        is_k = true;
        tile = 0;
    } else if (x < 2 * n - 1) {
        is_k = x & 1;
        tile = is_k ? (x + 1) / 2 : x / 2 - 1;
    } else {
        is_k = false;
        tile = n - 1;
    }
}

template <typename TV, typename TC, int HD>
__global__ void __launch_bounds__(Tile<TV, TC, HD>::kThreads, 1)
    attend_tile(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv, const __grid_constant__ Args a) {
    using T = Tile<TV, TC, HD>;
    constexpr int NP = T::NP, KT = T::KT, NS = T::NS, PN = T::PN, RS = T::RS, D = T::D, CH = 32;
    constexpr int kPages = KT / kPage;
    extern __shared__ uint8_t raw_[];
    uint8_t *sm = (uint8_t *)(((uintptr_t)raw_ + 1023) & ~(uintptr_t)1023);
    uint8_t *s_q = sm, *s_k = sm + T::kv_off, *s_v = s_k + (size_t)NS * T::kTileBytes;
    uint8_t *s_raw = sm + T::raw_off;
    float *s_scl = (float *)(sm + T::scl_off);  // [D][k, v][KT]
    float *s_max = (float *)(sm + T::max_off);  // [stream][step & 1][row]
    Ctl *ctl = (Ctl *)(sm + T::ctl_off);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Item *item = (const Item *)(a.words + a.off_items + (size_t)blockIdx.x * 12);
    const Item it = *item;
    const SeqRec sq = *(const SeqRec *)(a.words + a.off_seqs + it.seq * 4);
    const int32_t *table = a.words + sq.table;
    const int nk = it.i1 - it.i0;
    const bool shared = it.rows > 128;
    const int steps = shared ? 2 * nk : nk;
    auto key0 = [&](int i) {  // first key of the item's i-th tile
        const int u = it.i0 + i;
        return (u < it.ns ? u : it.u0 + u - it.ns) * KT;
    };
    auto none = [&](int j) { return j >= it.hi || (j < it.w0 && j >= a.sinks); };  // hidden from every row
    // Some row sees a key of page j (in units of pages).
    auto page_seen = [&](int j) { return j * kPage < it.hi && ((j + 1) * kPage > it.w0 || j * kPage < a.sinks); };

    if (threadIdx.x == 0) {
        mbar_init(&ctl->q_full, 256);
        mbar_init(&ctl->done, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&ctl->s_full[i], 1);
            mbar_init(&ctl->p_full[i][0], 128);
            mbar_init(&ctl->p_full[i][1], 128);
            mbar_init(&ctl->o_full[i], 1);
            mbar_init(&ctl->o_empty[i], 128);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(&ctl->k_full[i], T::kInt8 ? 4 : 1);
            mbar_init(&ctl->v_full[i], T::kInt8 ? 4 : 1);
            mbar_init(&ctl->k_empty[i], 1);
            mbar_init(&ctl->v_empty[i], 1);
            mbar_init(&ctl->raw_full[i], 1);
            mbar_init(&ctl->raw_empty[i], T::kInt8 ? 4 : 1);
            mbar_init(&ctl->scl_full[i], 1);
            mbar_init(&ctl->scl_empty[i], shared ? 8 : 4);
        }
        ctl->abort_ = 0;
        fence_mbar_init();
    }
    if (threadIdx.x < 256) ctl->bad[threadIdx.x] = 0;
    if (warp == 11) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&ctl->tmem))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = ctl->tmem;
    depend_trigger();

    // Loads every tile of one operand (BF16): a box a page (V) or a page's
    // panel (K).  A copy takes its warp about 110 cycles to issue, so K and V
    // have a warp each.  (K by two warps was slower: 421 against 402 us on
    // 4,096 tokens behind 4,096 at the 7B shape.)
    auto produce = [&](bool is_k) {
        uint64_t *full = is_k ? ctl->k_full : ctl->v_full, *empty = is_k ? ctl->k_empty : ctl->v_empty;
        const uint32_t base = smem_addr(is_k ? s_k : s_v), leader = elect_one();
        // A tile's pages (as pool rows) are looked up one tile ahead: the
        // table's latency would otherwise come on top of the copy's.
        auto page = [&](int i) {
            if (i >= nk) return -1;
            const int pj = key0(i) / kPage + lane;
            return lane < kPages && page_seen(pj) ? (table[pj] * a.KV + it.kvh) * kPage : -1;
        };
        int i = 0, next = page(0);
#pragma unroll 1
        for (; i < nk; ++i) {
            const int st = i % NS;
            int row[kPages];
#pragma unroll
            for (int g = 0; g < kPages; ++g) row[g] = __shfl_sync(0xffffffffu, next, g);
            const int pages = __popc(__ballot_sync(0xffffffffu, next >= 0));
            next = page(i + 1);
            if (i >= NS && !__all_sync(0xffffffffu, wait(empty + st, (uint32_t)((i / NS - 1) & 1), ctl))) break;
            if (lane == 0) mbar_arrive_expect_tx(full + st, (uint32_t)pages * (kPage * HD * 2));
            __syncwarp();
            const uint32_t dst = base + st * T::kTileBytes, bar = smem_addr(full + st);
#pragma unroll
            for (int g = 0; g < kPages; ++g) {
                const uint32_t go = row[g] >= 0 ? leader : 0u;
                if (is_k) {
#pragma unroll
                    for (int p = 0; p < PN; ++p)
                        tma_2d(dst + p * (KT * 128) + g * (kPage * 128), &mk, p * 64, row[g], bar, go);
                } else {
                    tma_3d(dst + g * (PN * kPage * 128), &mv, row[g], bar, go);
                }
            }
            __syncwarp();
        }
        // Every copy issued must land before the CTA can exit.
        for (int y = i > NS ? i - NS : 0; y < i; ++y) wait_issued(full + y % NS, (uint32_t)((y / NS) & 1));
    };
    if (warp < 8) {
        if constexpr (T::kSoftRegs > T::kLaunchRegs) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(T::kSoftRegs));
        if constexpr (T::kSoftRegs < T::kLaunchRegs) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(T::kSoftRegs));
        // ---- Q into its planes, then this stream's softmax ----
        const int s = warp >> 2;
        {
            const int nrows = shared ? 256 : 128;
            const bool vec = (((uintptr_t)a.q | (a.q_stride * sizeof(TV))) & 15) == 0;
            // Four pieces of eight elements under way at once.
            constexpr int kRun = 4, kWords = T::kWide ? 2 : 1;
#pragma unroll 1
            for (int u0 = threadIdx.x; u0 < nrows * (HD / 8); u0 += 256 * kRun) {
                uint4 raw[kRun][kWords];
#pragma unroll
                for (int x = 0; x < kRun; ++x) {
                    const int u = u0 + 256 * x, r = u / (HD / 8), ch = u % (HD / 8), row = it.row0 + r;
#pragma unroll
                    for (int y = 0; y < kWords; ++y) raw[x][y] = make_uint4(0u, 0u, 0u, 0u);
                    if (r >= it.rows) continue;
                    const TV *q = (const TV *)a.q + row_at(a, sq, it.kvh, row, a.q_stride) + ch * 8;
                    if (vec) {
#pragma unroll
                        for (int y = 0; y < kWords; ++y) raw[x][y] = ((const uint4 *)q)[y];
                    } else {
                        TV *e = (TV *)raw[x];
#pragma unroll
                        for (int y = 0; y < 8; ++y) e[y] = q[y];
                    }
                }
#pragma unroll
                for (int x = 0; x < kRun; ++x) {
                    const int u = u0 + 256 * x, r = u / (HD / 8), ch = u % (HD / 8);
                    if constexpr (!T::kWide && !T::kInt8) {
                        *(uint4 *)(s_q + ((r >> 7) * PN + ch / 8) * 16384 + (r & 127) * 128 + (((ch & 7) ^ (r & 7)) << 4)) = raw[x][0];
                    } else {
                        float v[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] = load_value((const TV *)raw[x], e);
                        const int rr = r & 127;
                        if constexpr (T::kInt8) {
                            // The row's HD / 8 pieces are neighbouring lanes.
                            uint32_t mb = 0;
#pragma unroll
                            for (int e = 0; e < 8; ++e) mb = max(mb, __float_as_uint(v[e]) & 0x7fffffffu);
#pragma unroll
                            for (int off = HD / 16; off; off >>= 1) mb = max(mb, __shfl_xor_sync(0xffffffffu, mb, off));
                            const float up = row_scale(mb);
#pragma unroll
                            for (int e = 0; e < 8; ++e) v[e] *= up;
                            if (ch == 0) ctl->c[r] = __fdiv_rn(a.c, up);
                        }
#pragma unroll
                        for (int pl = 0; pl < NP; ++pl) {
                            uint32_t w[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                if constexpr (T::kInt8) {
                                    w[e] = pack_f16(v[2 * e], v[2 * e + 1]);
                                    const float2 x = unpack_f16(w[e]);
                                    v[2 * e] -= x.x;
                                    v[2 * e + 1] -= x.y;
                                } else {
                                    w[e] = pack_bf16(v[2 * e], v[2 * e + 1]);
                                    v[2 * e] -= bf16_lo(w[e]);
                                    v[2 * e + 1] -= bf16_hi(w[e]);
                                }
                            }
                            uint8_t *dst = s_q + ((r >> 7) * PN + pl * PN + ch / 8) * 16384 + rr * 128 + (((ch & 7) ^ (rr & 7)) << 4);
                            *(uint4 *)dst = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    }
                }
            }
            if (T::kInt8) asm volatile("bar.sync 2, 256;" ::: "memory");
            fence_proxy_async_smem();
            mbar_arrive(&ctl->q_full);
        }
        const int r_in = (warp & 3) * 32 + lane;               // row of the tile
        const int r = (shared ? s * 128 : 0) + r_in;           // row of the item
        const int rmax = it.row0 + it.rows - 1;
        const int pos = sq.start + token_of(a, min(it.row0 + r, rmax));
        const int rb = it.row0 + (shared ? s * 128 : 0);
        const int p_lo = sq.start + token_of(a, min(rb, rmax)), p_hi = sq.start + token_of(a, min(rb + 127, rmax));
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + s * 256 + lanes, to = ts + 128;
        const int n_steps = shared ? nk : (nk - s + 1) / 2;
        const float c = T::kInt8 ? ctl->c[r] : a.c;
        float m = -INFINITY;   // in units of log2
        float2 l2[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
        bool ok = true, wild = false;
#pragma unroll 1
        for (int n = 0; n < n_steps; ++n) {
            const int i = shared ? n : 2 * n + s, j0 = key0(i);
            const bool whole = j0 + KT - 1 <= p_lo && (a.window == 0 || j0 > p_hi - a.window || j0 + KT <= a.sinks);
            // The products issued before these scores are then done too.
            if (!(ok = __all_sync(0xffffffffu, wait(&ctl->s_full[s], (uint32_t)(n & 1), ctl)))) break;
            fence_after();
            const float *ks = nullptr;
            float *vs = nullptr;
            if constexpr (T::kInt8) {
                if (!(ok = __all_sync(0xffffffffu, wait(&ctl->scl_full[i % D], (uint32_t)((i / D) & 1), ctl)))) break;
                ks = s_scl + (i % D * 2) * KT;
                vs = s_scl + (i % D * 2 + 1) * KT;
            }
            // Key e of the tile is visible up to e_hi, and then above e_lo or below e_sk.
            const int e_hi = pos - j0, e_lo = a.window ? pos - a.window - j0 : -1, e_sk = a.window ? a.sinks - j0 : 0;
            // A chunk of scores: scaled by the keys' scales, hidden ones -inf.
            auto finish = [&](uint32_t (&x)[CH], int ch) {
                if constexpr (T::kInt8) {
#pragma unroll
                    for (int e = 0; e < CH; e += 4) {
                        const float4 f = *(const float4 *)(ks + ch * CH + e);
                        float2 u = mul2(make_float2(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), make_float2(f.x, f.y));
                        float2 w = mul2(make_float2(__uint_as_float(x[e + 2]), __uint_as_float(x[e + 3])), make_float2(f.z, f.w));
                        x[e] = __float_as_uint(u.x);
                        x[e + 1] = __float_as_uint(u.y);
                        x[e + 2] = __float_as_uint(w.x);
                        x[e + 3] = __float_as_uint(w.y);
                    }
                }
                if (!whole) {
                    const int hi = e_hi - ch * CH, lo = e_lo - ch * CH, sk = e_sk - ch * CH;
#pragma unroll
                    for (int e = 0; e < CH; ++e) x[e] = (e <= hi) & ((e > lo) | (e < sk)) ? x[e] : 0xff800000u;
                }
            };
            auto largest = [&](const uint32_t (&x)[CH]) {
                float q[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) q[e] = __uint_as_float(x[e]);
#pragma unroll
                for (int e = 4; e < CH; e += 8)
#pragma unroll
                    for (int y = 0; y < 4; ++y)
                        q[y] = max3(q[y], __uint_as_float(x[e + y]), __uint_as_float(x[(e + 4 + y) % CH]));
                return max3(max3(q[0], q[1], q[2]), q[3], q[3]);
            };
            float bm = -INFINITY;
            uint32_t hold[T::kHold ? KT / CH : 1][CH];
            if constexpr (T::kHold) {
#pragma unroll
                for (int ch = 0; ch < KT / CH; ++ch) tmem_ld32(ts + ch * CH, hold[ch]);
                wait_ld();
            }
#pragma unroll
            for (int ch = 0; ch < KT / CH; ++ch) {
                uint32_t(&x)[CH] = hold[T::kHold ? ch : 0];
                if constexpr (!T::kHold) {
                    tmem_ld32(ts + ch * CH, x);
                    wait_ld();
                }
                finish(x, ch);
                bm = max3(bm, largest(x), bm);
            }
            bm *= c;
            // A NaN among the visible scores is the row's result.
            if (bm != bm) l2[0].x = bm;
            if constexpr (T::kInt8) {
                // The weights carry the V scales: score and largest scale of
                // the tile together bound every key's, so the base stays as
                // it is unless they pass it (after a stream's first tile they
                // seldom do).  Only then each key's own product is looked at:
                // the largest scale may be of a key that the row does not see
                // or hardly weighs, and f16 would drop the others' weights.
                float vm = 0.0f;
#pragma unroll
                for (int e = 0; e < KT; e += 32)
                    if (!none(j0 + e + lane)) {
                        vm = fmaxf(vm, fabsf(vs[e + lane]));
                        wild |= wild_scale(ks[e + lane]);
                    }
#pragma unroll
                for (int off = 16; off; off >>= 1) vm = fmaxf(vm, __shfl_xor_sync(0xffffffffu, vm, off));
                const float top = m + (8.0f + T::kAbove);
                const bool pass = bm + scale_log2(vm) > top;
                bm = -INFINITY;
                if (__any_sync(0xffffffffu, pass)) {
#pragma unroll 1
                    for (bool first = true;; first = false) {
                        bm = -INFINITY;
#pragma unroll 1
                        for (int ch = 0; ch < KT / CH; ++ch) {
                            const float lv = scale_log2(vs[ch * CH + lane]);
                            uint32_t x[CH];
                            tmem_ld32(ts + ch * CH, x);
                            wait_ld();
                            finish(x, ch);
#pragma unroll
                            for (int e = 0; e < CH; ++e)
                                bm = fmaxf(bm, fmaf(__uint_as_float(x[e]), c, __shfl_sync(0xffffffffu, lv, e)));
                        }
                        if (!first || !__any_sync(0xffffffffu, bm > top)) break;
                        // Nor may a V row of zeros set the base, whose scale
                        // says nothing.  The tile's V rows are widened
                        // without these weights; each lane looks at four.
                        if (!(ok = __all_sync(0xffffffffu, wait(&ctl->v_full[i % NS], (uint32_t)((i / NS) & 1), ctl)))) break;
                        const uint8_t *v = s_v + (size_t)(i % NS) * T::kTileBytes;
                        uint32_t zero = 0u;
#pragma unroll
                        for (int ch = 0; ch < KT / CH; ++ch) {
                            // (One 16-byte piece of the row nearly always says it.)
                            const int key = ch * CH + lane;
                            const uint4 w = *(const uint4 *)(v + key / kPage * (PN * kPage * 128) + key % kPage * 128 + (lane & 7) * 16);
                            zero |= (w.x | w.y | w.z | w.w) == 0u ? 1u << ch : 0u;
                        }
                        if (!__any_sync(0xffffffffu, zero)) break;
#pragma unroll 1
                        for (int ch = 0; ch < KT / CH; ++ch) {
                            const int key = ch * CH + lane;
                            uint32_t any = 0u;
#pragma unroll 1
                            for (int y = 0; y < PN * 8; ++y) {
                                const uint4 w = *(const uint4 *)(v + (key / kPage * PN + y / 8) * (kPage * 128) + key % kPage * 128 + ((y + lane) & 7) * 16);
                                any |= w.x | w.y | w.z | w.w;
                            }
                            // Taken as 0 the scale counts as the smallest,
                            // which keeps the row's sum in range; one that is
                            // not finite makes the result NaN and stays.  (The
                            // other warps of this tile may read either.)
                            if (!any && isfinite(vs[key])) vs[key] = 0.0f;
                        }
                        // The slot's next copy comes through the async proxy.
                        fence_proxy_async_smem();
                        __syncwarp();
                    }
                    if (!ok) break;
                }
            }
            if (__any_sync(0xffffffffu, bm > m + (8.0f + T::kAbove))) {
                const float mn = fmaxf(m, bm - T::kAbove), h = m == mn ? 1.0f : ex2_half(m - mn), f = h * h;
                m = mn;
#pragma unroll
                for (int e = 0; e < 2; ++e) l2[e] = mul2(mul2(l2[e], make_float2(h, h)), make_float2(h, h));
                if (!T::kWide && n > 0) {
#pragma unroll 1
                    for (int d = 0; d < HD; d += 16) {
                        uint32_t x[16];
                        tmem_ld16(to + d, x);
                        wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * f);
                        tmem_st16(to + d, x);
                    }
                }
            }
            if constexpr (T::kWide) s_max[(s * 2 + (n & 1)) * 128 + r_in] = m;
            const float base = m == -INFINITY ? 0.0f : m;
            const float2 c2 = make_float2(c, c), b2 = make_float2(-base, -base);
#pragma unroll
            for (int ch = 0; ch < KT / CH; ++ch) {
                uint32_t(&x)[CH] = hold[T::kHold ? ch : 0];
                if constexpr (!T::kHold) {
                    tmem_ld32(ts + ch * CH, x);
                    wait_ld();
                    finish(x, ch);
                }
                float2 p[CH / 2];
#pragma unroll
                for (int e = 0; e < CH / 2; ++e) {
                    p[e] = fma2(make_float2(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1])), c2, b2);
                    // (A quarter of them by polynomial on the FMA pipe made no
                    // difference, half was slower: the special functions are
                    // not what the tile waits for.)
                    p[e].x = ex2(p[e].x);
                    p[e].y = ex2(p[e].y);
                    l2[e & 1] = add2(l2[e & 1], p[e]);
                    if constexpr (T::kInt8) {
                        p[e] = mul2(p[e], *(const float2 *)(vs + ch * CH + 2 * e));
                        if (!whole) {
                            // A hidden key's scale may be anything.  (A visible
                            // one's NaN is the result's, whatever the weight.)
                            p[e].x = x[2 * e] == 0xff800000u ? 0.0f : p[e].x;
                            p[e].y = x[2 * e + 1] == 0xff800000u ? 0.0f : p[e].y;
                        }
                    }
                }
#pragma unroll
                for (int pl = 0; pl < NP; ++pl) {
                    uint32_t w[CH / 2];
#pragma unroll
                    for (int e = 0; e < CH / 2; ++e) {
                        if constexpr (T::kInt8) {
                            w[e] = pack_f16(p[e].x, p[e].y);
                            if (pl + 1 < NP) {
                                const float2 x = unpack_f16(w[e]);
                                p[e] = add2(p[e], make_float2(-x.x, -x.y));
                            }
                        } else if constexpr (NP == 1) {
                            w[e] = pack_bf16(p[e].x, p[e].y);
                        } else {
                            // Planes by truncation: 8 bits of the significand
                            // each, exact in three.
                            const uint32_t x0 = __float_as_uint(p[e].x), x1 = __float_as_uint(p[e].y);
                            w[e] = __byte_perm(x0, x1, 0x7632u);
                            if (pl + 1 < NP)
                                p[e] = fma2(make_float2(__uint_as_float(x0 & 0xffff0000u), __uint_as_float(x1 & 0xffff0000u)),
                                            make_float2(-1.0f, -1.0f), p[e]);
                        }
                    }
                    tmem_st16(ts + T::chunk_col(pl, ch), w);
                }
                if (ch == KT / CH / 2 - 1 || ch == KT / CH - 1) {
                    wait_st();
                    fence_before();
                    mbar_arrive(&ctl->p_full[s][ch == KT / CH - 1]);
                }
            }
            if constexpr (T::kInt8) {
                __syncwarp();
                if (lane == 0) mbar_arrive(&ctl->scl_empty[i % D]);
            }
        }
        const float2 lsum = add2(l2[0], l2[1]);
        const float l = lsum.x + lsum.y;
        bool fin = __all_sync(0xffffffffu, wait_issued(&ctl->done, 0u) && ok && !ctl->abort_);
        if (T::kInt8 && __any_sync(0xffffffffu, wild) && fin && r < it.rows) ctl->bad[r] = 1;
        fence_after();
        // Every copy and product has ended: stream 1's sums (and, where O is
        // not gathered, its O) for whoever writes the rows both streams had.
        float *s_o = (float *)s_k, *s_ml = s_o + 128 * (HD + 4);  // [stream][maximum, sum][row]
        if (!shared) {
            s_ml[s * 256 + r_in] = m;
            s_ml[s * 256 + 128 + r_in] = fin ? l : __uint_as_float(0x7fffffffu);
            if (!T::kWide && s == 1 && nk > 1) {
#pragma unroll 1
                for (int d = 0; d < HD; d += 32) {
                    uint32_t x[32];
                    tmem_ld32(to + d, x);
                    wait_ld();
#pragma unroll
                    for (int e = 0; e < 32; e += 4)
                        *(uint4 *)(s_o + r_in * (HD + 4) + d + e) = make_uint4(x[e], x[e + 1], x[e + 2], x[e + 3]);
                }
            }
            asm volatile("bar.sync 1, %0;" ::"n"(T::kWide ? 384 : 256) : "memory");
            // The other stream may have given up: what it left is not read.
            fin = __all_sync(0xffffffffu, fin && !ctl->abort_);
        }
        if constexpr (!T::kWide) if (shared || s == 0) {
            Join j = {m, l, 1.0f, 0.0f};
            if (!shared && nk > 1) j = join(m, l, s_ml[256 + r_in], s_ml[384 + r_in]);
            bool bad = false;
#pragma unroll 1
            for (int d = 0; d < HD; d += 64) {
                float v[64];
#pragma unroll
                for (int h = 0; h < 64; h += 32) {
                    uint32_t x[32];
                    tmem_ld32(to + d + h, x);
                    wait_ld();
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        v[h + e] = __uint_as_float(x[e]) * j.f0;
                        if (j.f1 != 0.0f) v[h + e] = fmaf(j.f1, s_o[r_in * (HD + 4) + d + h + e], v[h + e]);
                        bad |= !isfinite(v[h + e]);
                    }
                }
                put_rows<uint16_t, HD>(a, it, sq, r, d, v, j.m, j.l, fin, s_k + T::stage_off + warp * 4608, lane);
            }
            if (bad && fin && r < it.rows) ctl->bad[r] = 1;
        }
    } else if (T::kWide && warp >= T::kGather && warp < T::kGather + 4) {
        // O of both streams, in registers.  Each tile's product starts from
        // zero and is added here: the tensor cores cut their sums instead of
        // rounding them, and over a long row that adds up (5e-6 of the result
        // at 3,000 keys).
        if constexpr (T::kWide) {
            asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(T::kGatherRegs));
            const int r = (warp & 3) * 32 + lane;
            const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
            float2 o[HD / 2];
#pragma unroll
            for (int d = 0; d < HD / 2; ++d) o[d] = make_float2(0.0f, 0.0f);
            float m = -INFINITY;
            bool ok = true;
#pragma unroll 1
            for (int t = 0; t < steps; ++t) {
                const int s = t & 1;
                if (!(ok = __all_sync(0xffffffffu, wait(&ctl->o_full[s], (uint32_t)((t >> 1) & 1), ctl)))) break;
                fence_after();
                const float mt = s_max[(s * 2 + ((t >> 1) & 1)) * 128 + r];
                if (__any_sync(0xffffffffu, mt > m)) {
                    const float mn = fmaxf(m, mt), f = m == mn ? 1.0f : ex2(m - mn);
                    m = mn;
#pragma unroll
                    for (int d = 0; d < HD / 2; ++d) o[d] = mul2(o[d], make_float2(f, f));
                }
                const float w = mt == m ? 1.0f : ex2(mt - m);
#pragma unroll
                for (int d = 0; d < HD; d += 16) {
                    uint32_t x[16];
                    tmem_ld16(tmem + s * 256 + 128 + lanes + d, x);
                    wait_ld();
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        o[d / 2 + e] = fma2(make_float2(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1])),
                                            make_float2(w, w), o[d / 2 + e]);
                }
                fence_before();
                mbar_arrive(&ctl->o_empty[s]);
            }
            asm volatile("bar.sync 1, 384;" ::: "memory");
            const bool fin = __all_sync(0xffffffffu, ok && !ctl->abort_);
            const float *s_ml = (const float *)s_k + 128 * (HD + 4);
            const Join j = join(s_ml[r], s_ml[128 + r], s_ml[256 + r], s_ml[384 + r]);
            bool bad = false;
#pragma unroll
            for (int d = 0; d < HD; d += 32) {
                float v[32];
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                    v[e] = o[(d + e) / 2].x;
                    v[e + 1] = o[(d + e) / 2].y;
                    bad |= !isfinite(v[e]) | !isfinite(v[e + 1]);
                }
                put_rows<float, HD>(a, it, sq, r, d, v, j.m, j.l, fin, s_k + T::stage_off + (warp - T::kGather) * 4608, lane);
            }
            if (bad && fin && r < it.rows) ctl->bad[r] = 1;
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(T::kOtherRegs));
        if (warp == 8) {
            // Producers: BF16 boxes straight into the operand stages (K by this
            // warp, V by warp 11), INT8 pages raw into the pieces.
            if constexpr (!T::kInt8) {
                produce(true);
            } else {
                constexpr int per = KT / 64;
                auto page = [&](int z) {
                    bool is_k;
                    int i;
                    nth(z / per, nk, is_k, i);
                    const int pj = key0(i) / kPage + z % per * 4 + lane;
                    return z < 2 * nk * per && lane < 4 && page_seen(pj) ? table[pj] : -1;
                };
                int z = 0, next = page(0);  // pieces issued
#pragma unroll 1
                for (; z < 2 * nk * per; ++z) {
                    bool is_k;
                    int i;
                    nth(z / per, nk, is_k, i);
                    const int st = z % RS, pid = next;
                    next = page(z + 1);
                    if (z >= RS && !__all_sync(0xffffffffu, wait(&ctl->raw_empty[st], (uint32_t)((z / RS - 1) & 1), ctl))) break;
                    const bool on = pid >= 0;
                    const int pages = __popc(__ballot_sync(0xffffffffu, on));
                    if (lane == 0) mbar_arrive_expect_tx(&ctl->raw_full[st], (uint32_t)pages * (kPage * HD));
                    __syncwarp();
                    if (on)
                        bulk_copy_g2s(s_raw + (size_t)st * T::kPiece + lane * (kPage * HD),
                                      (is_k ? a.k : a.v) + ((size_t)pid * a.KV + it.kvh) * (kPage * HD), kPage * HD,
                                      &ctl->raw_full[st]);
                    __syncwarp();
                }
                for (int y = z > RS ? z - RS : 0; y < z; ++y) wait_issued(&ctl->raw_full[y % RS], (uint32_t)((y / RS) & 1));
            }
        } else if (warp == 9) {
            constexpr uint32_t is = idesc(KT, false, T::kInt8), io = idesc(HD, true, T::kInt8);
            const uint32_t leader = elect_one();
            const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
            const bool two = __shfl_sync(0xffffffffu, it.rows, 0) > 128;
            const int total = __shfl_sync(0xffffffffu, steps, 0);
            const uint32_t q_at = __shfl_sync(0xffffffffu, smem_addr(s_q), 0), k_at = q_at + (uint32_t)T::kv_off,
                           v_at = k_at + (uint32_t)(NS * T::kTileBytes);
            auto await = [&](uint64_t *bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity, ctl)); };
            auto k_ready = [&](int t) {
                const int i = two ? t >> 1 : t;
                return (two && (t & 1)) || await(&ctl->k_full[i % NS], (uint32_t)((i / NS) & 1));
            };
            auto scores = [&](int t) {
                const int i = two ? t >> 1 : t, st = i % NS, s = t & 1;
                const uint32_t q = q_at + (two ? s : 0) * (PN * 16384), k = k_at + st * T::kTileBytes;
#pragma unroll
                for (int pl = NP - 1; pl >= 0; --pl)
#pragma unroll
                    for (int ks = 0; ks < HD / 16; ++ks)
                        mma_ss(tm + s * 256, desc_k(q + (pl * PN + ks / 4) * 16384) + 2 * (ks % 4),
                               desc_k(k + ks / 4 * (KT * 128)) + 2 * (ks % 4), is, pl != NP - 1 || ks != 0, leader);
                commit(&ctl->s_full[s], leader);
                if (!two || s == 1) commit(&ctl->k_empty[st], leader);
            };
            bool ok = await(&ctl->q_full, 0u);
#pragma unroll 1
            for (int t = 0; t < 2 && t < total && (ok = ok && k_ready(t)); ++t) {
                fence_after();
                scores(t);
            }
#pragma unroll 1
            for (int t = 0; ok && t < total; ++t) {
                const int i = two ? t >> 1 : t, st = i % NS, s = t & 1;
                // The tiles of these products and of the next scores are there
                // long before the weights: looked at first.
                if ((!two || s == 0) && !await(&ctl->v_full[st], (uint32_t)((i / NS) & 1))) break;
                if (!T::kInt8 && (!two || s == 0)) {
                    // V rows that no row sees may hold anything (0 * inf is
                    // not 0; INT8 values are always finite).  Here and not in
                    // a warp of its own: one more waiting warp cost 5 %.
                    const int j0 = key0(i);
                    if (j0 + KT > it.hi || (j0 < it.w0 && j0 + KT > a.sinks)) {
                        // 16 bytes a lane, in the order they lie in: page,
                        // panel, row, piece.
                        uint4 *v = (uint4 *)(s_v + (size_t)st * T::kTileBytes);
#pragma unroll 4
                        for (int e = lane; e < KT * PN * 8; e += 32)
                            if (none(j0 + e / (PN * kPage * 8) * kPage + e / 8 % kPage)) v[e] = make_uint4(0, 0, 0, 0);
                        fence_proxy_async_smem();
                        __syncwarp();
                    }
                }
                if (t + 2 < total && !k_ready(t + 2)) break;
                if (T::kWide && t > 1 && !await(&ctl->o_empty[s], (uint32_t)(((t >> 1) - 1) & 1))) break;
                const uint32_t v = v_at + st * T::kTileBytes;
                // The first half of the keys while the second's weights are
                // still being computed.
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (!(ok = await(&ctl->p_full[s][h], (uint32_t)((t >> 1) & 1)))) break;
                    fence_after();
#pragma unroll
                    for (int pl = NP - 1; pl >= 0; --pl)
#pragma unroll
                        for (int kb = h * (KT / 32); kb < (h + 1) * (KT / 32); ++kb)
                            mma_ts(tm + s * 256 + 128, tm + s * 256 + T::plane_col(pl, kb),
                                   desc_mn(v + kb * (PN * 2048), 2048), io,
                                   (!T::kWide && t > 1) || h || pl != NP - 1 || kb != 0, leader);
                }
                if (!ok) break;
                if (T::kWide) commit(&ctl->o_full[s], leader);
                if (!two || s == 1) commit(&ctl->v_empty[st], leader);
                if (t + 2 < total) scores(t + 2);
            }
            // Whoever sees `done` sees that this warp gave up.
            __threadfence_block();
            __syncwarp();
            commit(&ctl->done, leader);
            __syncwarp();
        } else if (warp == 10) {
            if constexpr (T::kInt8) {
                // The scales of every tile's keys, a 64-byte copy a page and pool.
                auto page = [&](int i) {
                    if (i >= nk) return -1;
                    const int pj = key0(i) / kPage + lane;
                    return lane < kPages && page_seen(pj) ? table[pj] : -1;
                };
                int i = 0, next = page(0);
#pragma unroll 1
                for (; i < nk; ++i) {
                    const int st = i % D, pid = next;
                    next = page(i + 1);
                    if (i >= D && !__all_sync(0xffffffffu, wait(&ctl->scl_empty[st], (uint32_t)((i / D - 1) & 1), ctl))) break;
                    const bool on = pid >= 0;
                    const int pages = __popc(__ballot_sync(0xffffffffu, on));
                    if (lane == 0) mbar_arrive_expect_tx(&ctl->scl_full[st], (uint32_t)pages * 128u);
                    __syncwarp();
                    if (on) {
                        const size_t at = ((size_t)pid * a.KV + it.kvh) * kPage;
                        bulk_copy_g2s(s_scl + (st * 2) * KT + lane * kPage, a.ks + at, 64, &ctl->scl_full[st]);
                        bulk_copy_g2s(s_scl + (st * 2 + 1) * KT + lane * kPage, a.vs + at, 64, &ctl->scl_full[st]);
                    }
                    __syncwarp();
                }
                for (int y = i > D ? i - D : 0; y < i; ++y) wait_issued(&ctl->scl_full[y % D], (uint32_t)((y / D) & 1));
            }
        } else if (warp == 11) {
            if constexpr (!T::kInt8) produce(false);
        } else if (warp >= T::kConvert) {
            if constexpr (T::kInt8) {
                // INT8 -> f16 (exact), 64 keys a piece, into the operand layout.
                constexpr int per = KT / 64, units = T::kPiece / 16 / 128;
                const int ct = threadIdx.x - T::kConvert * 32;
                // Unit u of this thread: 16 values of key u * step + key_t.
                constexpr int step = 2048 / HD;
                const int key_t = ct / (HD / 16), q = ct % (HD / 16), c0 = q % 4 * 2, sw = key_t & 7;
                const int at_k = q / 4 * (KT * 128) + key_t * 128,
                          at_v = (key_t / kPage * PN + q / 4) * (kPage * 128) + key_t % kPage * 128;
                bool ok = true;
#pragma unroll 1
                for (int z = 0; ok && z < 2 * nk * per; ++z) {
                    bool is_k;
                    int i;
                    nth(z / per, nk, is_k, i);
                    const int rs = z % RS, st = i % NS, half = z % per;
                    ok = half != 0 || i < NS ||
                         wait(is_k ? &ctl->k_empty[st] : &ctl->v_empty[st], (uint32_t)((i / NS - 1) & 1), ctl);
                    ok = __all_sync(0xffffffffu, ok && wait(&ctl->raw_full[rs], (uint32_t)((z / RS) & 1), ctl));
                    if (!ok) break;
                    const uint8_t *src = s_raw + (size_t)rs * T::kPiece;
                    // K: panels of all the tile's keys; V: a page's panels together.
                    uint8_t *dst = (is_k ? s_k : s_v) + (size_t)st * T::kTileBytes + half * (is_k ? 64 * 128 : 64 * HD * 2);
                    uint4 w[units];
#pragma unroll
                    for (int u = 0; u < units; ++u) w[u] = *(const uint4 *)(src + (u * 128 + ct) * 16);
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&ctl->raw_empty[rs]);
#pragma unroll
                    for (int u = 0; u < units; ++u) {
                        uint4 o0, o1;
                        o0.x = s8x2_to_f16x2(__byte_perm(w[u].x, 0u, 0x4140u));
                        o0.y = s8x2_to_f16x2(__byte_perm(w[u].x, 0u, 0x4342u));
                        o0.z = s8x2_to_f16x2(__byte_perm(w[u].y, 0u, 0x4140u));
                        o0.w = s8x2_to_f16x2(__byte_perm(w[u].y, 0u, 0x4342u));
                        o1.x = s8x2_to_f16x2(__byte_perm(w[u].z, 0u, 0x4140u));
                        o1.y = s8x2_to_f16x2(__byte_perm(w[u].z, 0u, 0x4342u));
                        o1.z = s8x2_to_f16x2(__byte_perm(w[u].w, 0u, 0x4140u));
                        o1.w = s8x2_to_f16x2(__byte_perm(w[u].w, 0u, 0x4342u));
                        uint8_t *r = dst + (is_k ? at_k + u * (step * 128) : at_v + u * (step / kPage * PN * kPage * 128));
                        *(uint4 *)(r + ((c0 ^ sw) << 4)) = o0;
                        *(uint4 *)(r + (((c0 + 1) ^ sw) << 4)) = o1;
                    }
                    fence_proxy_async_smem();
                    if (half == per - 1) {
                        __syncwarp();
                        if (lane == 0) mbar_arrive(is_k ? &ctl->k_full[st] : &ctl->v_full[st]);
                    }
                }
            }
        }
    }
    fence_before();
    __syncthreads();
    const int redo = __syncthreads_or(warp < 8 && ctl->bad[threadIdx.x & 255]);
    fence_after();
    if (warp == 11)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    if (redo && warp < 8)
        for (int r = warp; r < it.rows; r += 8)
            if (ctl->bad[r]) attend_row<TV, TC>(a, item, r, KT, lane, true);
}

// ------------------------------------------------------------------ host ----

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = (PFN_cuTensorMapEncodeTiled_v12000)p;
    });
    return fn;
}

// A pool as rows of HD bf16 elements: boxes of one page's 64-element panel
// (K), or of all its panels, one after the other (V).
bool encode_pool(CUtensorMap &m, const void *base, int hd, size_t rows, bool panels) {
    auto fn = encode_fn();
    if (!fn) return false;
    const cuuint32_t pn = (cuuint32_t)hd / 64;
    cuuint64_t dims[3] = {(cuuint64_t)(panels ? 64 : hd), (cuuint64_t)rows, pn};
    cuuint64_t strides[2] = {(cuuint64_t)hd * 2, 128};
    cuuint32_t box[3] = {64, kPage, pn}, es[3] = {1, 1, 1};
    return fn(&m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, panels ? 3 : 2, (void *)base, dims, strides, box, es,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename TV, typename TC, int HD>
cudaError_t launch_tile(const Args &a, size_t pool_rows, cudaStream_t st) {
    using T = Tile<TV, TC, HD>;
    // At least what keeps one CTA on an SM: an item takes all of its TMEM.
    const int smem = (int)(T::bytes > 120 * 1024 ? T::bytes : 120 * 1024);
    static std::atomic<bool> configured[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!configured[dev].load()) {
        e = cudaFuncSetAttribute(attend_tile<TV, TC, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        // The split of the registers counts on what the launch allots: with
        // fewer a warpgroup would wait for its share forever, so a build that
        // comes out otherwise is refused here.
        cudaFuncAttributes fa;
        e = cudaFuncGetAttributes(&fa, attend_tile<TV, TC, HD>);
        if (e != cudaSuccess) return e;
        if (fa.numRegs != T::kLaunchRegs) return cudaErrorInvalidConfiguration;
        configured[dev].store(true);
    }
    alignas(64) CUtensorMap mk = {}, mv = {};
    if (!T::kInt8 && (!encode_pool(mk, a.k, HD, pool_rows, false) || !encode_pool(mv, a.v, HD, pool_rows, true)))
        return cudaErrorInvalidValue;
    return paged::launch(attend_tile<TV, TC, HD>, dim3(a.items), T::kThreads, smem, st, false, mk, mv, a);
}

template <typename TV>
cudaError_t launch_tv(const Args &a, int cache, size_t rows, cudaStream_t st) {
    if (cache == QB_PAGED_BF16)
        return a.hd == 64 ? launch_tile<TV, uint16_t, 64>(a, rows, st) : launch_tile<TV, uint16_t, 128>(a, rows, st);
    return a.hd == 64 ? launch_tile<TV, int8_t, 64>(a, rows, st) : launch_tile<TV, int8_t, 128>(a, rows, st);
}

}  // namespace

cudaError_t tile_attention(const Args &a, bool wide, int cache, size_t pool_rows, cudaStream_t st) {
    return wide ? launch_tv<float>(a, cache, pool_rows, st) : launch_tv<uint16_t>(a, cache, pool_rows, st);
}

}  // namespace paged
}  // namespace qb
