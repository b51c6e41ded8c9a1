// Cache rows of the paged operators: stored (with the INT8 encode of
// ops.cu's quant_kernel, one group a row) and read back.
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
};

constexpr int kRowWarps = 8;

// One warp a row, in any alignment: the row sits in registers between the
// maximum and the encode.
template <typename TV, typename TC>
__global__ void __launch_bounds__(kRowWarps * 32) kv_write_rows(const RowArgs a) {
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
        float scale = __fdiv_rn(m, 127.0f);
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
__global__ void __launch_bounds__(kRowWarps * 32) kv_read_rows(const RowArgs a) {
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

template <typename TV, typename TC>
uint32_t launch_rows(const RowArgs &a, bool write, cudaStream_t st) {
    const size_t blocks = (a.rows + kRowWarps - 1) / kRowWarps;
    const dim3 grid((unsigned)blocks, 2);
    if (write)
        kv_write_rows<TV, TC><<<grid, kRowWarps * 32, 0, st>>>(a);
    else
        kv_read_rows<TV, TC><<<grid, kRowWarps * 32, 0, st>>>(a);
    QB_CUDA(cudaGetLastError());
    return QB_OK;
}

uint32_t run_rows(const RowArgs &a, uint32_t vt, uint32_t ct, bool write, cudaStream_t st) {
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
    RowArgs a{words + plan->off_slots, plan->tokens * plan->kv_heads, (int)plan->kv_heads, (int)plan->head_dim,
              {nullptr, nullptr}, {k, v}, {k_stride, v_stride}, {cache->k, cache->v},
              {cache->k_scales, cache->v_scales}};
    return run_rows(a, plan->value_dtype, plan->cache_dtype, false, (cudaStream_t)stream);
}

}  // extern "C"
