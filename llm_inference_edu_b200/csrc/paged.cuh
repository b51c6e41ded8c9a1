// Paged cache operators: the plan of one step (built on the host, read by the
// kernels) and the row-by-row attention that every shape can fall back on.
//
// A plan is an array of 32-bit words with five parts: one SeqRec a sequence,
// the page tables, two words a token (its cache slot, page * 16 + row, and
// its sequence), the attention items of the two kernels, the merges.  An item
// is a run of packed rows (row r of a sequence and KV head = token r / G,
// query head r % G of the head's group of G) over a run of key units; a row
// block whose units are cut among several items gets one partial result
// (maximum, sum, unnormalised context) per item and one merge.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>
#include <stddef.h>

#include "common.cuh"

namespace qb {
namespace paged {

constexpr int kPage = QB_PAGE_TOKENS;
constexpr int kMaxHeadDim = 256;

struct SeqRec {
    int32_t tok0, count, start, table;  // first packed token, new tokens, position of the first, word offset of the table
};

struct Item {
    int32_t seq, kvh, row0, rows;
    // Units [i0, i1) of the row block's list: the first `ns` are units
    // 0 .. ns - 1 of the sequence (sinks), the others start at unit u0.
    int32_t i0, i1, ns, u0;
    int32_t w0, hi;      // keys visible to some row: [w0, hi), and below the sinks
    int32_t slot;        // float offset of the partial result, or -1: the item covers all its units
    int32_t cost;
};

struct Merge {
    int32_t seq, kvh, row0, rows, slot, parts, stride, quads;
};

// Where a partial result keeps element d of row r.  The tile kernel has a
// thread a row: in quads of four dimensions, rows side by side, its lanes
// write 512 bytes at once (row by row an item of 256 rows took 6 us
// longer).  The others have lanes along a row.
__device__ __forceinline__ size_t part_at(int rows, int hd, int r, int d, bool quads) {
    return quads ? ((size_t)(d >> 2) * rows + r) * 4 + (d & 3) : (size_t)r * hd + d;
}

// A sequence goes to the step kernel (mma.sync, 8 rows an n8 tile) up to this
// many packed rows: with more, the step kernel would read the cache more than
// once.  Others go to the tile kernel (tcgen05, 128 rows an MMA).
constexpr int kStepRows = 16;
// The merge kernel's warps a CTA, and the parts up to which one takes a row.
constexpr int kMergeWarps = 4, kMergeFew = 8;

struct Args {
    const int32_t *words;
    uint32_t off_seqs, off_items, off_merges;
    int items, merges;
    int H, KV, G, hd;
    int window, sinks;
    float c;              // scale * log2(e)
    const void *q;
    size_t q_stride;      // elements between tokens
    void *y;
    const uint8_t *k, *v;
    const float *ks, *vs;
    float *ws;
    int dependent;        // launched behind another kernel of the same call
    uint32_t g_mul, g_shift;  // row / G = (mulhi(row, g_mul) + row) >> g_shift, row < 2^31
};

// Byte element types of values and caches.
__device__ __forceinline__ float load_value(const float *p, size_t i) { return p[i]; }
__device__ __forceinline__ float load_value(const uint16_t *p, size_t i) { return bf16_to_f32(p[i]); }
__device__ __forceinline__ float load_value(const int8_t *p, size_t i) { return (float)p[i]; }

__device__ __forceinline__ uint16_t bf16_bits(float x) {
    uint16_t r;
    asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ void store_value(float *p, size_t i, float v) { p[i] = v; }
__device__ __forceinline__ void store_value(uint16_t *p, size_t i, float v) { p[i] = bf16_bits(v); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The square root of 2^x.  Sums of weights are brought to another base by its
// two factors: over INT8 pages a base holds a V row's scale, so two may lie
// further apart than a float reaches while both sums count.  (A context under
// the lower base is then nothing next to the other's.)
__device__ __forceinline__ float ex2_half(float x) { return ex2(0.5f * x); }

// The kernels of one call follow each other by programmatic dependent launch:
// a kernel may start while the one before it still runs.  depend_wait waits
// for everything before to be complete; a kernel that writes only its own
// results calls it last, so that its own end means theirs too.
__device__ __forceinline__ void depend_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void depend_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename... KArgs, typename... Args_>
cudaError_t launch(void (*kernel)(KArgs...), dim3 grid, int threads, size_t smem, cudaStream_t st, bool dependent,
                   const Args_ &...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = dependent ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Multiplier and shift of a division by d of numbers below 2^31.
inline void divide_by(uint32_t d, uint32_t &mul, uint32_t &shift) {
    shift = 0;
    while ((1ull << shift) < d) ++shift;
    mul = (uint32_t)(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
}

// Packed row `row` of a sequence and KV head: its token and query head.
__device__ __forceinline__ int token_of(const Args &a, int row) {
    return (int)((__umulhi((uint32_t)row, a.g_mul) + (uint32_t)row) >> a.g_shift);
}
// Element offset of packed row `row` in Q (stride a token) or Y (a.H * a.hd).
__device__ __forceinline__ size_t row_at(const Args &a, const SeqRec &sq, int kvh, int row, size_t stride) {
    const int t = token_of(a, row);
    return (size_t)(sq.tok0 + t) * stride + (size_t)(kvh * a.G + row - t * a.G) * a.hd;
}

// Position p sees position j of its sequence.
__device__ __forceinline__ bool sees(int p, int j, int window, int sinks) {
    return j <= p && (window == 0 || j > p - window || j < sinks);
}

// One row by one warp over the item's units of `unit` keys: 32 keys at a
// time, one lane a key for the scores, one lane for every 32nd dimension of
// the context.  Reads only what the row sees, so nothing hidden (a stale
// page, a NaN of a later token) can reach the result.  Writes the finished
// row, or its partial result.  Used where no tensor-core variant fits
// (head widths other than 64 and 128, FP32 caches) and, by those variants,
// for items whose partly hidden units hold values that are not finite.
template <typename TV, typename TC>
__device__ __noinline__ void attend_row(const Args &a, const Item *item, int r, int unit, int lane, bool quads = false) {
    const Item it = *item;
    const SeqRec sq = *(const SeqRec *)(a.words + a.off_seqs + it.seq * 4);
    const int32_t *table = a.words + sq.table;
    const int row = it.row0 + r, p = sq.start + row / a.G;
    const size_t qh = (size_t)it.kvh * a.G + row % a.G, tok = (size_t)sq.tok0 + row / a.G;
    const TV *q = (const TV *)a.q + tok * a.q_stride + qh * a.hd;
    const TC *kc = (const TC *)a.k, *vc = (const TC *)a.v;
    float m = -INFINITY, l = 0.0f, o[kMaxHeadDim / 32];
#pragma unroll
    for (int i = 0; i < kMaxHeadDim / 32; ++i) o[i] = 0.0f;
    for (int i = it.i0; i < it.i1; ++i) {
        const int j0 = (i < it.ns ? i : it.u0 + i - it.ns) * unit;
        for (int b = j0; b < j0 + unit; b += 32) {
            const int j = b + lane;
            const bool ok = j < j0 + unit && sees(p, j, a.window, a.sinks);
            if (!__any_sync(0xffffffffu, ok)) continue;
            size_t at = 0;
            float t = -INFINITY, vsc = 1.0f;
            if (ok) {
                at = ((size_t)table[j / kPage] * a.KV + it.kvh) * kPage + j % kPage;
                const TC *kr = kc + at * a.hd;
                float s = 0.0f;
                for (int d = 0; d < a.hd; ++d) s = fmaf(load_value(q, d), load_value(kr, d), s);
                if (a.ks) s = s * a.ks[at];
                t = s * a.c;
                if (a.vs) vsc = a.vs[at];
            }
            // A NaN score must not vanish in the maximum.
            float bm = t;
            bool nan = ok && t != t;
#pragma unroll
            for (int off = 16; off; off >>= 1) bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, off));
            nan = __any_sync(0xffffffffu, nan);
            float mn = fmaxf(m, bm);
            if (nan) mn = __uint_as_float(0x7fffffffu);
            const float base = mn == -INFINITY ? 0.0f : mn;
            const float f = exp2f(m - base), e = ok ? exp2f(t - base) : 0.0f;
            m = mn;
            float se = e;
#pragma unroll
            for (int off = 16; off; off >>= 1) se += __shfl_xor_sync(0xffffffffu, se, off);
            l = fmaf(l, f, se);
#pragma unroll
            for (int i2 = 0; i2 < kMaxHeadDim / 32; ++i2) o[i2] *= f;
            const float pe = e * vsc;
            for (int x = 0; x < 32; ++x) {
                if (!__shfl_sync(0xffffffffu, (int)ok, x)) continue;
                const float pw = __shfl_sync(0xffffffffu, pe, x);
                const size_t vat = __shfl_sync(0xffffffffu, (unsigned long long)at, x) * (size_t)a.hd;
#pragma unroll
                for (int i2 = 0; i2 < kMaxHeadDim / 32; ++i2)
                    if (lane + 32 * i2 < a.hd) o[i2] = fmaf(pw, load_value(vc, vat + lane + 32 * i2), o[i2]);
            }
        }
    }
    if (it.slot >= 0) {
        float *w = a.ws + it.slot;
#pragma unroll
        for (int i2 = 0; i2 < kMaxHeadDim / 32; ++i2)
            if (lane + 32 * i2 < a.hd) w[part_at(it.rows, a.hd, r, lane + 32 * i2, quads)] = o[i2];
        if (lane == 0) {
            w[(size_t)it.rows * a.hd + r] = m;
            w[(size_t)it.rows * (a.hd + 1) + r] = l;
        }
    } else {
        TV *y = (TV *)a.y + (tok * a.H + qh) * a.hd;
#pragma unroll
        for (int i2 = 0; i2 < kMaxHeadDim / 32; ++i2)
            if (lane + 32 * i2 < a.hd) store_value(y, lane + 32 * i2, __fdiv_rn(o[i2], l));
    }
}

}  // namespace paged
}  // namespace qb
