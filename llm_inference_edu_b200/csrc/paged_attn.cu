// Attention over the paged cache: the entry point, the row-by-row kernel and
// the merge of partial results.
#include <math.h>

#include "paged_attn.cuh"

namespace qb {
namespace paged {
namespace {

constexpr int kRowsWarps = 4;

// One CTA an item, its rows dealt to the warps.
template <typename TV, typename TC>
__global__ void __launch_bounds__(kRowsWarps * 32) attend_rows(const __grid_constant__ Args a) {
    depend_trigger();
    const Item *it = (const Item *)(a.words + a.off_items + (size_t)blockIdx.x * 12);
    for (int r = threadIdx.x >> 5; r < it->rows; r += kRowsWarps) attend_row<TV, TC>(a, it, r, 64, threadIdx.x & 31);
}

// Joins the partial results: M = max m_z, y = sum_z o_z 2^(m_z - M) /
// sum_z l_z 2^(m_z - M).  Few parts: a warp a row, kMergeWarps rows a CTA.
// Many (kMergeFew): a CTA a row, the parts dealt to the warps and the warps'
// sums joined in order.  Either way the order is fixed, so the result does
// not depend on timing.  Bound by the latency of the parts' loads: eight
// parts' are under way at once, before their maximum is known (a pass for
// the maximum first and four at a time took 2 us longer, 80 drafted tokens
// 22.9 -> 21.0 us; CTAs of two or eight warps were slower).

// Parts z0, z0 + dz, ... of row r: o (V dimensions a lane) and l against
// their maximum m.  A part that is NaN leaves l or o NaN.
template <int V>
__device__ __forceinline__ void merge_parts(const float *w, const Merge &mg, int hd, int r, int z0, int dz, int lane, float (&o)[V],
                                            float &m, float &l) {
    constexpr int N = kMergeFew;
    const float *wm = w + (size_t)mg.rows * hd + r, *wl = wm + mg.rows;
    m = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = 0.0f;
#pragma unroll 1
    for (int z = z0; z < mg.parts; z += N * dz) {
        float mz[N], lz[N], oz[N][V], mn = m;
#pragma unroll
        for (int x = 0; x < N; ++x) {
            const bool on = z + x * dz < mg.parts;
            const size_t at = (size_t)(on ? z + x * dz : z) * mg.stride;
            mz[x] = on ? wm[at] : -INFINITY;
            lz[x] = on ? wl[at] : 0.0f;
#pragma unroll
            for (int i = 0; i < V; ++i)
                oz[x][i] = on && lane + 32 * i < hd ? w[at + part_at(mg.rows, hd, r, lane + 32 * i, mg.quads)] : 0.0f;
        }
#pragma unroll
        for (int x = 0; x < N; ++x) mn = fmaxf(mn, mz[x]);
        // (In two factors: ex2_half.)
        const float base = mn == -INFINITY ? 0.0f : mn, h = exp2f(0.5f * (m - base)), f = h * h;
        m = mn;
        l = l * h * h;
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] *= f;
#pragma unroll
        for (int x = 0; x < N; ++x) {
            const float hx = exp2f(0.5f * (mz[x] - base)), e = hx * hx;
            l = fmaf(lz[x] * hx, hx, l);
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] = fmaf(e, oz[x][i], o[i]);
        }
    }
}

template <typename TV, int V>
__global__ void __launch_bounds__(kMergeWarps * 32) merge_rows(const __grid_constant__ Args a) {
    __shared__ float s_o[kMergeWarps][32 * V], s_m[kMergeWarps], s_l[kMergeWarps];
    const Merge mg = *(const Merge *)(a.words + a.off_merges + (size_t)blockIdx.x * 8);
    const bool few = mg.parts <= kMergeFew;
    const int r0 = few ? blockIdx.y * kMergeWarps : blockIdx.y;
    if (r0 >= mg.rows) return;  // (other CTAs of this grid wait for the parts)
    const SeqRec sq = *(const SeqRec *)(a.words + a.off_seqs + mg.seq * 4);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hd = a.hd;
    auto out = [&](int r) { return (TV *)a.y + row_at(a, sq, mg.kvh, mg.row0 + r, (size_t)a.H * hd); };
    depend_wait();
    const float *w = a.ws + mg.slot;
    float o[V], m, l;
    if (few) {
        const int r = r0 + warp;
        if (r >= mg.rows) return;
        merge_parts<V>(w, mg, hd, r, 0, 1, lane, o, m, l);
        TV *y = out(r);
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (lane + 32 * i < hd) store_value(y, lane + 32 * i, __fdiv_rn(o[i], l));
        return;
    }
    merge_parts<V>(w, mg, hd, r0, warp, kMergeWarps, lane, o, m, l);
#pragma unroll
    for (int i = 0; i < V; ++i) s_o[warp][lane + 32 * i] = o[i];
    if (lane == 0) {
        s_m[warp] = m;
        s_l[warp] = l;
    }
    __syncthreads();
    m = s_m[0];
#pragma unroll
    for (int x = 1; x < kMergeWarps; ++x) m = fmaxf(m, s_m[x]);
    const float base = m == -INFINITY ? 0.0f : m;
    TV *y = out(r0);
    for (int d = threadIdx.x; d < hd; d += kMergeWarps * 32) {
        float v = 0.0f, ll = 0.0f;
#pragma unroll
        for (int x = 0; x < kMergeWarps; ++x) {
            const float h = exp2f(0.5f * (s_m[x] - base));
            v = fmaf(h * h, s_o[x][d], v);
            ll = fmaf(s_l[x] * h, h, ll);
        }
        store_value(y, d, __fdiv_rn(v, ll));
    }
}

template <typename TV>
cudaError_t launch_merge(const Args &a, int blocks, cudaStream_t st) {
    auto kern = a.hd <= 64 ? merge_rows<TV, 2> : a.hd <= 128 ? merge_rows<TV, 4> : merge_rows<TV, 8>;
    return launch(kern, dim3(a.merges, blocks), kMergeWarps * 32, 0, st, true, a);
}

template <typename TV>
uint32_t run_rows(const Args &a, uint32_t ct, cudaStream_t st) {
    auto kern = ct == QB_PAGED_F32 ? attend_rows<TV, float> : ct == QB_PAGED_BF16 ? attend_rows<TV, uint16_t> : attend_rows<TV, int8_t>;
    QB_CUDA(launch(kern, dim3(a.items), kRowsWarps * 32, 0, st, false, a));
    return QB_OK;
}

}  // namespace

uint32_t admit(const qb_paged_cache *c, const qb_paged_plan *p, const int32_t *words);
uint32_t admit_rows(size_t buffer, size_t len, size_t stride, size_t width, size_t tokens);
bool rows_meet(const void *p, size_t p_stride, const void *q, size_t q_stride, size_t width, size_t tokens, size_t size);
bool rows_in_cache(const void *p, size_t stride, size_t width, size_t tokens, size_t size, const qb_paged_cache *c);

}  // namespace paged
}  // namespace qb

using namespace qb;
using namespace qb::paged;

extern "C" {

uint32_t qb_paged_attention(const void *q, size_t q_len, size_t q_stride, const qb_paged_cache *cache,
                            const qb_paged_plan *plan, const int32_t *words, void *y, size_t y_len, float scale,
                            void *workspace, size_t workspace_bytes, void *stream) {
    clear_detail();
    uint32_t s = admit(cache, plan, words);
    if (s) return s;
    const size_t width = plan->query_heads * plan->head_dim;
    if ((s = admit_rows(0, q_len, q_stride, width, plan->tokens))) return s;
    if ((s = admit_rows(2, y_len, width, width, plan->tokens))) return s;
    // Scores are taken in units of log2.
    const float c = (float)((double)scale * 1.4426950408889634);
    if (!q || !y || !(isfinite(c) && scale > 0.0f)) return QB_INVALID_PARAMETERS;
    const size_t size = plan->value_dtype == QB_PAGED_F32 ? 4 : 2;
    if (rows_meet(q, q_stride, y, width, width, plan->tokens, size) ||
        rows_in_cache(y, width, width, plan->tokens, size, cache))
        return QB_INVALID_PARAMETERS;
    if (workspace_bytes < plan->workspace_bytes) {
        set_detail(3, plan->workspace_bytes, workspace_bytes);
        return QB_INVALID_LENGTH;
    }
    if (plan->workspace_bytes && (!workspace || ((uintptr_t)workspace & 15))) return QB_INVALID_PARAMETERS;
    Args a{};
    a.words = words;
    a.off_seqs = plan->off_seqs;
    a.off_merges = plan->off_merges;
    a.merges = (int)plan->merges;
    a.H = (int)plan->query_heads;
    a.KV = (int)plan->kv_heads;
    a.G = a.H / a.KV;
    divide_by((uint32_t)a.G, a.g_mul, a.g_shift);
    a.hd = (int)plan->head_dim;
    // A window as long as a table row hides nothing.
    a.window = plan->window < plan->pages_per_sequence * kPage ? (int)plan->window : 0;
    a.sinks = (int)(plan->sinks < 0x7fffffffu ? plan->sinks : 0x7fffffffu);
    a.c = c;
    a.q = q;
    a.q_stride = q_stride;
    a.y = y;
    a.k = (const uint8_t *)cache->k;
    a.v = (const uint8_t *)cache->v;
    a.ks = cache->dtype == QB_PAGED_INT8 ? cache->k_scales : nullptr;
    a.vs = cache->dtype == QB_PAGED_INT8 ? cache->v_scales : nullptr;
    a.ws = (float *)workspace;
    cudaStream_t st = (cudaStream_t)stream;
    const bool wide = plan->value_dtype == QB_PAGED_F32;
    // The tile kernel first: the step kernel's CTAs fill the SMs as its
    // last ones leave.  Both only read what was there before the call.
    if (plan->tile_items) {
        a.off_items = plan->off_tile;
        a.items = (int)plan->tile_items;
        QB_CUDA(tile_attention(a, wide, (int)plan->cache_dtype, plan->pages * plan->kv_heads * kPage, st));
    }
    if (plan->small_items) {
        a.off_items = plan->off_small;
        a.items = (int)plan->small_items;
        a.dependent = plan->tile_items != 0;
        if (plan->small_kind)
            QB_CUDA(step_attention(a, wide, (int)plan->cache_dtype, (int)plan->small_kind, st));
        else if ((s = wide ? run_rows<float>(a, plan->cache_dtype, st) : run_rows<uint16_t>(a, plan->cache_dtype, st)))
            return s;
    }
    if (plan->merges)
        QB_CUDA(wide ? launch_merge<float>(a, (int)plan->merge_blocks, st)
                     : launch_merge<uint16_t>(a, (int)plan->merge_blocks, st));
    return QB_OK;
}

}  // extern "C"
