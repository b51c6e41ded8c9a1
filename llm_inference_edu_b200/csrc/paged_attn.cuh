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

// Two int8 values, in the low bytes of `t`'s halves (the high bytes are
// ignored), as bf16, exactly: with the low 7 bits u as the mantissa of 128,
// 128 + u - (128 or 256 by the sign bit) is the value.
__device__ __forceinline__ uint32_t s8x2_to_bf16x2(uint32_t t) {
    const uint32_t x = (t & 0x007f007fu) | 0x43004300u, y = (t & 0x00800080u) | 0x43004300u;
    uint32_t r;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y));
    return r;
}

// One CTA an item; nt: n8 tiles of an item's rows.
cudaError_t step_attention(const Args &a, bool wide, int cache, int nt, cudaStream_t st);
// One CTA an item; pool_rows: rows of a pool (pages * kv_heads * 16).
cudaError_t tile_attention(const Args &a, bool wide, int cache, size_t pool_rows, cudaStream_t st);

}  // namespace paged
}  // namespace qb
