// Cache rows of the paged operators: stored (INT8: round(x / scale), halves
// away from zero, one scale a row) and read back.
#include <math.h>

#include "paged.cuh"

namespace qb {
namespace paged {
namespace {

struct RowArgs {
    const int32_t *slots;
    size_t rows;      // tokens * kv_heads; the grid's y picks K or V
    int KV, hd;
    const void *x[2];
    void *out[2];
    size_t stride[2];
    void *pool[2];
    float *scales[2];
    uint32_t mul, shift;  // row / KV = (mulhi(row, mul) + row) >> shift, row < 2^31
};

constexpr int kRowWarps = 8;

// A row's scale is its largest magnitude times this.  Next to the quotient by
// 127 (qb_quantize_int8's) it differs in the last place for 4 % of rows, and a
// byte may differ where x / scale is that close to a half; either is within
// half a scale of x.
constexpr float kStep = 1.0f / 127.0f;

// One warp a row, in any alignment: the row sits in registers between the
// maximum and the encode.
template <typename TV, typename TC>
__global__ void __launch_bounds__(kRowWarps * 32) kv_write_rows(const __grid_constant__ RowArgs a) {
    const size_t row = (size_t)blockIdx.x * kRowWarps + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31, z = blockIdx.y;
    if (row >= a.rows) return;
    const size_t tok = row / a.KV;
    const int g = (int)(row % a.KV), slot = a.slots[tok];
    const size_t at = ((size_t)(slot / kPage) * a.KV + g) * kPage + slot % kPage;
    const TV *x = (const TV *)a.x[z] + tok * a.stride[z] + (size_t)g * a.hd;
    TC *y = (TC *)a.pool[z] + at * a.hd;
    float v[kMaxHeadDim / 32];
    float m = 0.0f;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < kMaxHeadDim / 32; ++i) {
        const int d = lane + 32 * i;
        v[i] = d < a.hd ? load_value(x, d) : 0.0f;
        m = fmaxf(m, fabsf(v[i]));
        bad |= !isfinite(v[i]);
    }
    if constexpr (sizeof(TC) == 1) {
#pragma unroll
        for (int off = 16; off; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
        bad = __any_sync(0xffffffffu, bad);
        float scale = __fmul_rn(m, kStep);
        if (scale == 0.0f) scale = 1.0f;
        if (lane == 0) a.scales[z][at] = bad ? __uint_as_float(0x7fffffffu) : scale;
#pragma unroll
        for (int i = 0; i < kMaxHeadDim / 32; ++i) {
            const int d = lane + 32 * i;
            const float r = fminf(fmaxf(roundf(__fdiv_rn(v[i], scale)), -127.0f), 127.0f);
            if (d < a.hd) y[d] = bad ? (int8_t)0 : (int8_t)r;
        }
    } else {
#pragma unroll
        for (int i = 0; i < kMaxHeadDim / 32; ++i)
            if (lane + 32 * i < a.hd) store_value(y, lane + 32 * i, v[i]);
    }
}

template <typename TV, typename TC>
__global__ void __launch_bounds__(kRowWarps * 32) kv_read_rows(const __grid_constant__ RowArgs a) {
    const size_t row = (size_t)blockIdx.x * kRowWarps + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31, z = blockIdx.y;
    if (row >= a.rows) return;
    const size_t tok = row / a.KV;
    const int g = (int)(row % a.KV), slot = a.slots[tok];
    const size_t at = ((size_t)(slot / kPage) * a.KV + g) * kPage + slot % kPage;
    const TC *x = (const TC *)a.pool[z] + at * a.hd;
    TV *y = (TV *)a.out[z] + tok * a.stride[z] + (size_t)g * a.hd;
    const float scale = sizeof(TC) == 1 ? a.scales[z][at] : 1.0f;
#pragma unroll
    for (int i = 0; i < kMaxHeadDim / 32; ++i)
        if (lane + 32 * i < a.hd) store_value(y, lane + 32 * i, __fmul_rn(load_value(x, lane + 32 * i), scale));
}

// The same in 16-byte pieces of the values, where widths and alignment allow
// (lanes: pieces a row, a power of two up to 32).  Each thread has kRun rows
// under way, a block's worth apart.  8,192 tokens of 4 heads of 128 from FP32
// to INT8: 18 us for K and V (42 MB; HBM alone: 6.4), bound by issue, 38
// instructions a piece of four values; back: 15 us, the latency of the slot
// and then of the row.
constexpr int kRun = 4;

template <typename TV>
struct Piece {
    static constexpr int E = 16 / (int)sizeof(TV);
    __device__ static void unpack(const uint4 &w, float (&v)[E]) {
        if constexpr (sizeof(TV) == 4) {
            v[0] = __uint_as_float(w.x); v[1] = __uint_as_float(w.y);
            v[2] = __uint_as_float(w.z); v[3] = __uint_as_float(w.w);
        } else {
            v[0] = bf16_lo(w.x); v[1] = bf16_hi(w.x); v[2] = bf16_lo(w.y); v[3] = bf16_hi(w.y);
            v[4] = bf16_lo(w.z); v[5] = bf16_hi(w.z); v[6] = bf16_lo(w.w); v[7] = bf16_hi(w.w);
        }
    }
};

// E elements of the row as FP32 or BF16.
template <typename TC, int E>
__device__ __forceinline__ void store_piece(TC *p, const float (&v)[E]) {
    if constexpr (sizeof(TC) == 4) {
#pragma unroll
        for (int e = 0; e < E; e += 4) *(float4 *)(p + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
    } else if constexpr (sizeof(TC) == 2) {
        uint32_t w[E / 2];
#pragma unroll
        for (int e = 0; e < E / 2; ++e) w[e] = bf16_bits(v[2 * e]) | (uint32_t)bf16_bits(v[2 * e + 1]) << 16;
#pragma unroll
        for (int e = 0; e < E / 2; e += 2) *(uint2 *)((uint32_t *)p + e) = make_uint2(w[e], w[e + 1]);
    }
}

template <typename TC, int E>
__device__ __forceinline__ void load_piece(const TC *p, float (&v)[E]) {
    if constexpr (sizeof(TC) == 4) {
#pragma unroll
        for (int e = 0; e < E; e += 4) {
            const float4 w = *(const float4 *)(p + e);
            v[e] = w.x; v[e + 1] = w.y; v[e + 2] = w.z; v[e + 3] = w.w;
        }
    } else if constexpr (sizeof(TC) == 2) {
#pragma unroll
        for (int e = 0; e < E; e += 4) {
            const uint2 w = *(const uint2 *)(p + e);
            v[e] = bf16_lo(w.x); v[e + 1] = bf16_hi(w.x); v[e + 2] = bf16_lo(w.y); v[e + 3] = bf16_hi(w.y);
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; e += 4) {
            const uint32_t w = *(const uint32_t *)(p + e);
#pragma unroll
            for (int x = 0; x < 4; ++x) v[e + x] = (float)(int8_t)(w >> (8 * x));
        }
    }
}

// A row of the grid: its token, KV head and cache row.
struct RowAt {
    uint32_t tok, g;
    __device__ RowAt(const RowArgs &a, uint32_t row) {
        tok = (__umulhi(row, a.mul) + row) >> a.shift;
        g = row - tok * (uint32_t)a.KV;
    }
    __device__ size_t cache_row(const RowArgs &a, int slot) const {
        return ((size_t)((uint32_t)slot / kPage) * (uint32_t)a.KV + g) * kPage + (uint32_t)slot % kPage;
    }
};

// One row's E elements as INT8 with the row's scale (mb: the largest bit
// pattern of the row's magnitudes).  x / scale rounded, halves away from
// zero: added to 1.5 * 2^23 the product x * (1 / scale) rounds to the
// integer that then lies in the low byte.  The product is within 2^-23 of
// the FP32 quotient (relative: one rounding each; so 1.6e-5 here) and rounds
// alike unless it lies that close to a half; there (taken as 1e-4), and where
// it is no number, the quotient itself decides.
template <int E>
__device__ __forceinline__ float encode_row(const float (&v)[E], uint32_t mb, uint32_t (&out)[E / 4]) {
    const bool bad = mb >= 0x7f800000u;
    float scale = __fmul_rn(__uint_as_float(mb), kStep);
    if (scale == 0.0f) scale = 1.0f;
    const float inv = __fdiv_rn(1.0f, scale), big = 12582912.0f;
    bool exact = bad;
    uint32_t q[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const float h = fmaf(v[e], inv, big);
        q[e] = __float_as_uint(h);
        exact |= !(fabsf(fmaf(v[e], inv, -(h - big))) <= 0.4999f);
    }
    if (exact)
#pragma unroll
        for (int e = 0; e < E; ++e)
            q[e] = bad ? 0u : (uint32_t)(int)fminf(fmaxf(roundf(__fdiv_rn(v[e], scale)), -127.0f), 127.0f);
#pragma unroll
    for (int e = 0; e < E; e += 4)
        out[e / 4] = __byte_perm(__byte_perm(q[e], q[e + 1], 0x0040u), __byte_perm(q[e + 2], q[e + 3], 0x0040u), 0x5410u);
    return bad ? __uint_as_float(0x7fffffffu) : scale;
}

template <typename TV, typename TC>
__global__ void __launch_bounds__(256) kv_write_pieces(const __grid_constant__ RowArgs a, int lanes) {
    constexpr int E = Piece<TV>::E;
    const int per = 256 / lanes, lane = threadIdx.x & (lanes - 1), z = blockIdx.y;
    const uint32_t rows = (uint32_t)a.rows, row0 = blockIdx.x * per * kRun + threadIdx.x / lanes;
    const TV *x = (const TV *)a.x[z] + lane * E;
    TC *pool = (TC *)a.pool[z] + lane * E;
    uint4 w[kRun];
    size_t at[kRun];
#pragma unroll
    for (int r = 0; r < kRun; ++r) {
        const uint32_t row = row0 + r * per;
        w[r] = make_uint4(0u, 0u, 0u, 0u);
        if (row < rows) {
            const RowAt p(a, row);
            w[r] = ld_stream_u4(x + p.tok * a.stride[z] + p.g * (uint32_t)a.hd);
            at[r] = p.cache_row(a, a.slots[p.tok]);
        }
    }
#pragma unroll
    for (int r = 0; r < kRun; ++r) {
        float v[E];
        Piece<TV>::unpack(w[r], v);
        if constexpr (sizeof(TC) == 1) {
            uint32_t mb = 0, q[E / 4];
#pragma unroll
            for (int e = 0; e < E; ++e) mb = max(mb, __float_as_uint(v[e]) & 0x7fffffffu);
            for (int off = lanes >> 1; off; off >>= 1) mb = max(mb, __shfl_xor_sync(0xffffffffu, mb, off));
            const float scale = encode_row<E>(v, mb, q);
            if (row0 + r * per >= rows) continue;
            uint32_t *y = (uint32_t *)(pool + at[r] * (uint32_t)a.hd);
            if constexpr (E == 8)
                *(uint2 *)y = make_uint2(q[0], q[1]);
            else
                *y = q[0];
            if (lane == 0) a.scales[z][at[r]] = scale;
        } else {
            if (row0 + r * per < rows) store_piece<TC, E>(pool + at[r] * (uint32_t)a.hd, v);
        }
    }
}

template <typename TV, typename TC>
__global__ void __launch_bounds__(256) kv_read_pieces(const __grid_constant__ RowArgs a, int lanes) {
    constexpr int E = Piece<TV>::E;
    const int per = 256 / lanes, lane = threadIdx.x & (lanes - 1), z = blockIdx.y;
    const uint32_t rows = (uint32_t)a.rows, row0 = blockIdx.x * per * kRun + threadIdx.x / lanes;
    const TC *pool = (const TC *)a.pool[z] + lane * E;
    TV *out = (TV *)a.out[z] + lane * E;
    int slot[kRun];
    float v[kRun][E], scale[kRun];
#pragma unroll
    for (int r = 0; r < kRun; ++r)
        slot[r] = row0 + r * per < rows ? a.slots[RowAt(a, row0 + r * per).tok] : 0;
#pragma unroll
    for (int r = 0; r < kRun; ++r)
        if (row0 + r * per < rows) {
            const size_t at = RowAt(a, row0 + r * per).cache_row(a, slot[r]);
            load_piece<TC, E>(pool + at * (uint32_t)a.hd, v[r]);
            scale[r] = sizeof(TC) == 1 ? a.scales[z][at] : 1.0f;
        }
#pragma unroll
    for (int r = 0; r < kRun; ++r)
        if (row0 + r * per < rows) {
            const RowAt p(a, row0 + r * per);
#pragma unroll
            for (int e = 0; e < E; ++e) v[r][e] = __fmul_rn(v[r][e], scale[r]);
            store_piece<TV, E>(out + p.tok * a.stride[z] + p.g * (uint32_t)a.hd, v[r]);
        }
}

template <typename TV, typename TC>
uint32_t launch_rows(const RowArgs &a, bool write, cudaStream_t st) {
    constexpr int E = Piece<TV>::E;
    const int lanes = a.hd / E;
    uintptr_t all = 0;
    for (int z = 0; z < 2; ++z) all |= (uintptr_t)a.x[z] | (uintptr_t)a.out[z] | a.stride[z] * sizeof(TV);
    // 8,192 tokens of 4 heads of 128, FP32 into INT8 and back: 31 us in
    // pieces, 74 us a row at a time.
    if (a.hd % E == 0 && lanes <= 32 && (lanes & (lanes - 1)) == 0 && !(all & 15)) {
        const size_t per = (size_t)(256 / lanes) * kRun;
        const dim3 grid((unsigned)((a.rows + per - 1) / per), 2);
        if (write)
            kv_write_pieces<TV, TC><<<grid, 256, 0, st>>>(a, lanes);
        else
            kv_read_pieces<TV, TC><<<grid, 256, 0, st>>>(a, lanes);
        QB_CUDA(cudaGetLastError());
        return QB_OK;
    }
    const dim3 grid((unsigned)((a.rows + kRowWarps - 1) / kRowWarps), 2);
    if (write)
        kv_write_rows<TV, TC><<<grid, kRowWarps * 32, 0, st>>>(a);
    else
        kv_read_rows<TV, TC><<<grid, kRowWarps * 32, 0, st>>>(a);
    QB_CUDA(cudaGetLastError());
    return QB_OK;
}

uint32_t run_rows(RowArgs a, uint32_t vt, uint32_t ct, bool write, cudaStream_t st) {
    divide_by((uint32_t)a.KV, a.mul, a.shift);
    if (vt == QB_PAGED_F32) {
        if (ct == QB_PAGED_F32) return launch_rows<float, float>(a, write, st);
        if (ct == QB_PAGED_BF16) return launch_rows<float, uint16_t>(a, write, st);
        return launch_rows<float, int8_t>(a, write, st);
    }
    if (ct == QB_PAGED_F32) return launch_rows<uint16_t, float>(a, write, st);
    if (ct == QB_PAGED_BF16) return launch_rows<uint16_t, uint16_t>(a, write, st);
    return launch_rows<uint16_t, int8_t>(a, write, st);
}

}  // namespace

uint32_t admit(const qb_paged_cache *c, const qb_paged_plan *p, const int32_t *words) {
    if (!c || !p || !words || !c->k || !c->v) return QB_INVALID_PARAMETERS;
    if (c->pages != p->pages || c->kv_heads != p->kv_heads || c->head_dim != p->head_dim ||
        c->dtype != p->cache_dtype)
        return QB_INVALID_SHAPE;
    if (c->dtype == QB_PAGED_INT8 && (!c->k_scales || !c->v_scales)) return QB_INVALID_PARAMETERS;
    const uintptr_t all = (uintptr_t)c->k | (uintptr_t)c->v | (uintptr_t)c->k_scales | (uintptr_t)c->v_scales |
                          (uintptr_t)words;
    return all & 15 ? QB_INVALID_PARAMETERS : QB_OK;
}

// Rows of `width` elements, `stride` apart: the length must reach exactly
// from the first to the last.
uint32_t admit_rows(size_t buffer, size_t len, size_t stride, size_t width, size_t tokens) {
    size_t need;
    if (tokens > 1 && stride < width) {
        set_detail(buffer, width, stride);
        return QB_INVALID_SHAPE;
    }
    if (mul_ovf(tokens - 1, stride, &need) || need > SIZE_MAX - width) return QB_DIMENSION_OVERFLOW;
    need += width;
    if (len != need) {
        set_detail(buffer, need, len);
        return QB_INVALID_LENGTH;
    }
    return QB_OK;
}

// Whether two sets of rows (`tokens` rows of `width` elements of `size`
// bytes, `stride` elements apart) share memory.  Rows of one buffer with the
// same stride may lie side by side; with other strides any overlap of the
// whole ranges counts.
bool rows_meet(const void *p, size_t p_stride, const void *q, size_t q_stride, size_t width, size_t tokens, size_t size) {
    const uintptr_t a = (uintptr_t)p, b = (uintptr_t)q;
    const uintptr_t a_end = a + ((tokens - 1) * p_stride + width) * size, b_end = b + ((tokens - 1) * q_stride + width) * size;
    if (a >= b_end || b >= a_end) return false;
    if (tokens == 1 || p_stride != q_stride) return true;
    const size_t step = p_stride * size, off = (a > b ? a - b : b - a) % step, w = width * size;
    return off < w || step - off < w;
}

// Whether bytes [p, p + n) and [q, q + m) share memory.
static bool meet(const void *p, size_t n, const void *q, size_t m) {
    return (uintptr_t)p < (uintptr_t)q + m && (uintptr_t)q < (uintptr_t)p + n;
}

// Whether the range of `tokens` rows shares memory with a pool of the cache
// or its scales.
bool rows_in_cache(const void *p, size_t stride, size_t width, size_t tokens, size_t size, const qb_paged_cache *c) {
    const size_t n = ((tokens - 1) * stride + width) * size, rows = c->pages * c->kv_heads * kPage;
    const size_t pool = rows * c->head_dim * (c->dtype == QB_PAGED_F32 ? 4 : c->dtype == QB_PAGED_BF16 ? 2 : 1);
    if (meet(p, n, c->k, pool) || meet(p, n, c->v, pool)) return true;
    return c->dtype == QB_PAGED_INT8 && (meet(p, n, c->k_scales, rows * 4) || meet(p, n, c->v_scales, rows * 4));
}

// Whether K's and V's rows would be stored over each other.
static bool pools_meet(const qb_paged_cache *c) {
    const size_t rows = c->pages * c->kv_heads * kPage;
    const size_t pool = rows * c->head_dim * (c->dtype == QB_PAGED_F32 ? 4 : c->dtype == QB_PAGED_BF16 ? 2 : 1);
    return meet(c->k, pool, c->v, pool) || (c->dtype == QB_PAGED_INT8 && meet(c->k_scales, rows * 4, c->v_scales, rows * 4));
}

}  // namespace paged
}  // namespace qb

using namespace qb;
using namespace qb::paged;

extern "C" {

uint32_t qb_kv_write(const void *k, size_t k_len, size_t k_stride, const void *v, size_t v_len, size_t v_stride,
                     const qb_paged_cache *cache, const qb_paged_plan *plan, const int32_t *words, void *stream) {
    clear_detail();
    uint32_t s = admit(cache, plan, words);
    if (s) return s;
    const size_t width = plan->kv_heads * plan->head_dim;
    if ((s = admit_rows(0, k_len, k_stride, width, plan->tokens))) return s;
    if ((s = admit_rows(1, v_len, v_stride, width, plan->tokens))) return s;
    if (!k || !v) return QB_INVALID_PARAMETERS;
    const size_t size = plan->value_dtype == QB_PAGED_F32 ? 4 : 2;
    if (pools_meet(cache) || rows_in_cache(k, k_stride, width, plan->tokens, size, cache) ||
        rows_in_cache(v, v_stride, width, plan->tokens, size, cache))
        return QB_INVALID_PARAMETERS;
    if (plan->shared_rows) return QB_INVALID_STATE;
    RowArgs a{words + plan->off_slots, plan->tokens * plan->kv_heads, (int)plan->kv_heads, (int)plan->head_dim,
              {k, v}, {nullptr, nullptr}, {k_stride, v_stride}, {cache->k, cache->v},
              {cache->k_scales, cache->v_scales}};
    return run_rows(a, plan->value_dtype, plan->cache_dtype, true, (cudaStream_t)stream);
}

uint32_t qb_kv_read(const qb_paged_cache *cache, const qb_paged_plan *plan, const int32_t *words, void *k,
                    size_t k_len, size_t k_stride, void *v, size_t v_len, size_t v_stride, void *stream) {
    clear_detail();
    uint32_t s = admit(cache, plan, words);
    if (s) return s;
    const size_t width = plan->kv_heads * plan->head_dim;
    if ((s = admit_rows(0, k_len, k_stride, width, plan->tokens))) return s;
    if ((s = admit_rows(1, v_len, v_stride, width, plan->tokens))) return s;
    if (!k || !v) return QB_INVALID_PARAMETERS;
    const size_t size = plan->value_dtype == QB_PAGED_F32 ? 4 : 2;
    if (rows_meet(k, k_stride, v, v_stride, width, plan->tokens, size) ||
        rows_in_cache(k, k_stride, width, plan->tokens, size, cache) ||
        rows_in_cache(v, v_stride, width, plan->tokens, size, cache))
        return QB_INVALID_PARAMETERS;
    RowArgs a{words + plan->off_slots, plan->tokens * plan->kv_heads, (int)plan->kv_heads, (int)plan->head_dim,
              {nullptr, nullptr}, {k, v}, {k_stride, v_stride}, {cache->k, cache->v},
              {cache->k_scales, cache->v_scales}};
    return run_rows(a, plan->value_dtype, plan->cache_dtype, false, (cudaStream_t)stream);
}

}  // extern "C"
