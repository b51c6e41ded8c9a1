// The tensor-core kernels of the paged attention and what they share.
#pragma once
#include "paged.cuh"

namespace qb {
namespace paged {

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// INT8 caches are widened to f16, which holds a byte exactly at one addition
// a pair (1024 + 128 + q is the f16 with bits 0x6480 ^ q), and holds more of
// Q and of the weights than bf16: two planes of an FP32 value to 2^-22, one
// of a bf16 value exactly.  f16 lacks range.  So each row of Q is scaled by a
// power of two to a largest element in 2^13 .. 2^14, and the weights, which
// carry the V rows' scales, are taken against a base that keeps the largest
// between 2^7 and 2^15: what f16 drops is below 2^-31 of it.  The largest is
// over the keys that the row sees and whose V row has a nonzero byte: a stored
// row of zeros has scale 1 whatever the others' are.  (Scales under 2^-90, and
// what is that far below the weight of a row of zeros, lose precision; where
// one over 2^90 overflows, the row is done again by attend_row.)
constexpr float kAboveBase = 7.0f, kScaleSpan = 90.0f;

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float2 unpack_f16(uint32_t w) {
    float2 r;
    asm("{\n\t.reg .b16 x, y;\n\tmov.b32 {x, y}, %2;\n\tcvt.f32.f16 %0, x;\n\tcvt.f32.f16 %1, y;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "r"(w));
    return r;
}
// Two int8 values in the low bytes of t's halves as f16, exactly.
__device__ __forceinline__ uint32_t s8x2_to_f16x2(uint32_t t) {
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"((t & 0x00ff00ffu) ^ 0x64806480u), "r"(0x64806480u));
    return r;
}
__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Whether a K row's scale may take a score out of a float's range (a product of
// scaled Q and bytes is below 2^28).  Rows that see one are done again by
// attend_row; elsewhere a score of -inf means a hidden key.
__device__ __forceinline__ bool wild_scale(float scale) { return !(fabsf(scale) <= 0x1p99f); }

// log2 of a V row's scale as the base counts it: finite whatever the scale.
__device__ __forceinline__ float scale_log2(float scale) {
    return fminf(fmaxf(lg2(fabsf(scale)), -kScaleSpan), kScaleSpan);
}

// The power of two for a row of Q whose largest magnitude has bits mb.
__device__ __forceinline__ float row_scale(uint32_t mb) {
    return __uint_as_float((267u - min(max(mb >> 23, 27u), 250u)) << 23);
}

// One CTA an item; nt: n8 tiles of an item's rows.
cudaError_t step_attention(const Args &a, bool wide, int cache, int nt, cudaStream_t st);
// One CTA an item; pool_rows: rows of a pool (pages * kv_heads * 16).
cudaError_t tile_attention(const Args &a, bool wide, int cache, size_t pool_rows, cudaStream_t st);

}  // namespace paged
}  // namespace qb
