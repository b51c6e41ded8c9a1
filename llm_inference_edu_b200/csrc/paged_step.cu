// Attention of few rows over the paged cache (single tokens, a few drafted
// ones): bound by the bytes of the cache, so the work is arranged around
// loading each page once, straight into registers.
//
// Scores are taken transposed, S^T [16 keys][8 rows] = K Q^T: a page's 16
// keys are the M of one m16n8k16 and eight packed rows (the query heads of
// one KV head, or several tokens') its N, so a group of seven heads wastes
// one row, not nine.  The reduction index may be permuted freely as long as
// K and Q agree, so a thread's K operand is whole 16-byte pieces of its two
// keys' rows; O^T [head_dim][8 rows] = V^T P^T likewise takes whole pieces of
// four keys' rows, two byte permutes an operand word pairing the keys.  The
// weights cross from accumulator to operand layout by two 8x8 transposes.
// Nothing goes through shared memory but Q (fragments) and the end result.
//
// BF16 caches.  FP32 values: Q is three bf16 planes (q = p0 + p1 + p2 to
// 2^-24) and so are the weights, which keeps FP32 precision over exact
// operands at three products each.  BF16 values: one plane of Q, two of the
// weights (one would double the error of the result's own rounding, and the
// products are not what this kernel waits for).
//
// INT8 caches: what bounds them is the widening of the bytes on the integer
// pipe, so they are widened to f16 (paged_attn.cuh).  64 sequences of 100 to
// 8,191 positions at the 7B shape: 63 us widened to bf16, 48 us so (38 us as
// the plan now cuts them and with the merge: 3.4 TB/s, 14.8 M instructions).
#include "paged_attn.cuh"

namespace qb {
namespace paged {
namespace {

constexpr int kStepWarps = 4;

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma16816h(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// 16 or 8 bytes of the cache, read once.
__device__ __forceinline__ void load_piece(const uint8_t *p, uint32_t (&r)[4]) {
    const uint4 v = ld_stream_u4(p);
    r[0] = v.x; r[1] = v.y; r[2] = v.z; r[3] = v.w;
}
__device__ __forceinline__ void load_piece(const uint8_t *p, uint32_t (&r)[2]) {
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "l"(p));
}

template <typename TV, typename TC, int HD, int NT>
struct StepShape {
    static constexpr bool kInt8 = sizeof(TC) == 1;
    static constexpr int NQ = sizeof(TV) == 4 ? (kInt8 ? 2 : 3) : 1;   // planes of Q
    static constexpr int NPV = sizeof(TV) == 4 ? (kInt8 ? 2 : 3) : kInt8 ? 1 : 2;  // planes of the weights
    static constexpr float kAbove = kInt8 ? kAboveBase : 0.0f;  // of the base the weights are taken against
    static constexpr int KS = HD / 16;                   // k-steps of the scores
    static constexpr int MT = HD / 16;                   // m16 tiles of O^T
    static constexpr int PG = 8192 / (2 * 16 * HD * (int)sizeof(TC));  // pages a warp holds: 8 KB of K and V
    static constexpr int KL = HD * (int)sizeof(TC) / 64; // 16-byte pieces of a key's row a thread
    static constexpr int VW = HD * (int)sizeof(TC) / 8 / 4;            // words of a V row a thread
    static constexpr int VP = VW >= 4 ? 4 : VW;          // words a load
    static constexpr int EPL = VP * 4 / (int)sizeof(TC); // elements a load
    static constexpr size_t q_bytes = (size_t)NQ * NT * KS * 32 * 8;
    static constexpr int OS = HD + 8;                    // row stride of the joined context
    static constexpr size_t o_bytes = (size_t)kStepWarps * 8 * NT * OS * 4;
    // The head dimension a thread's i-th V element has (lane group g).
    static __device__ __forceinline__ int dim_of(int g, int i) { return i / EPL * (8 * EPL) + g * EPL + i % EPL; }
};

template <typename TV, typename TC, int HD, int NT>
__global__ void __launch_bounds__(kStepWarps * 32, 3) attend_step(const __grid_constant__ Args a) {
    using S = StepShape<TV, TC, HD, NT>;
    constexpr int NQ = S::NQ, NPV = S::NPV, KS = S::KS, MT = S::MT, PG = S::PG, KL = S::KL, VP = S::VP, VW = S::VW;
    __shared__ __align__(16) uint8_t s_raw[S::q_bytes > S::o_bytes ? S::q_bytes : S::o_bytes];
    __shared__ float s_m[kStepWarps][8 * NT], s_l[kStepWarps][8 * NT], s_c[8 * NT];
    uint2 *s_q = (uint2 *)s_raw;  // [plane][n tile][k-step][lane]

    depend_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const Item *item = (const Item *)(a.words + a.off_items + (size_t)blockIdx.x * 12);
    const Item it = *item;
    const SeqRec sq = *(const SeqRec *)(a.words + a.off_seqs + it.seq * 4);
    const int32_t *table = a.words + sq.table;
    const int p_lo = sq.start + token_of(a, it.row0), p_hi = it.hi - 1;
    auto page_of = [&](int i) { return i < it.ns ? i : it.u0 + i - it.ns; };

    // The pages of this warp's next group: table entries one group ahead of
    // the loads, the loads one group ahead of their use.
    int32_t pid[PG];
    auto ids = [&](int i) {
#pragma unroll
        for (int x = 0; x < PG; ++x) pid[x] = i + x < it.i1 ? table[page_of(i + x)] : -1;
    };
    uint32_t kr[PG][2][KL][4], vr[PG][4][VW / VP][VP];
    float ksc[PG][2], vsc[PG][2];
    auto load_k = [&]() {
#pragma unroll
        for (int x = 0; x < PG; ++x) {
            if (pid[x] < 0) continue;
            const size_t blk = (size_t)pid[x] * a.KV + it.kvh;
            const uint8_t *p = a.k + blk * (kPage * HD * sizeof(TC)) + g * (HD * sizeof(TC)) + c * 16;
#pragma unroll
            for (int y = 0; y < 2; ++y)
#pragma unroll
                for (int j = 0; j < KL; ++j) load_piece(p + y * (8 * HD * sizeof(TC)) + j * 64, kr[x][y][j]);
            if constexpr (S::kInt8) {
                ksc[x][0] = a.ks[blk * kPage + g];
                ksc[x][1] = a.ks[blk * kPage + g + 8];
            }
        }
    };
    auto load_v = [&]() {
#pragma unroll
        for (int x = 0; x < PG; ++x) {
            if (pid[x] < 0) {
                // Weights of absent keys are 0: their operand must be finite.
#pragma unroll
                for (int y = 0; y < 4; ++y)
#pragma unroll
                    for (int j = 0; j < VW / VP; ++j)
#pragma unroll
                        for (int z = 0; z < VP; ++z) vr[x][y][j][z] = 0u;
                continue;
            }
            const size_t blk = (size_t)pid[x] * a.KV + it.kvh;
            const uint8_t *p = a.v + blk * (kPage * HD * sizeof(TC)) + g * (VP * 4);
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const int key = 2 * c + (y & 1) + (y >> 1) * 8;
#pragma unroll
                for (int j = 0; j < VW / VP; ++j)
                    load_piece(p + key * (HD * sizeof(TC)) + j * (8 * VP * 4), vr[x][y][j]);
            }
            if constexpr (S::kInt8) {
                vsc[x][0] = a.vs[blk * kPage + g];
                vsc[x][1] = a.vs[blk * kPage + g + 8];
            }
        }
    };

    const int step = kStepWarps * PG;
    int i = it.i0 + warp * PG;
    ids(i);
    load_k();
    load_v();

    // Q fragments, a row a warp and four elements a lane: k-step ks of a
    // thread is elements 4 h .. 4 h + 3 of its 8 (bf16) or 16 (int8) in a
    // stretch of 32 or 64.
    for (int r = warp; r < 8 * NT; r += kStepWarps) {
        constexpr int per = S::kInt8 ? 4 : 2, run = S::kInt8 ? 16 : 8;
        const int d = lane * 4, ks = d / (4 * run) * per + d % run / 4, fl = (r & 7) * 4 + d % (4 * run) / run;
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (r < it.rows && d < HD) {
            const TV *q = (const TV *)a.q + row_at(a, sq, it.kvh, it.row0 + r, a.q_stride) + d;
#pragma unroll
            for (int x = 0; x < 4; ++x) v[x] = load_value(q, x);
        }
        if constexpr (S::kInt8) {
            uint32_t mb = 0;
#pragma unroll
            for (int x = 0; x < 4; ++x) mb = max(mb, __float_as_uint(v[x]) & 0x7fffffffu);
#pragma unroll
            for (int off = 16; off; off >>= 1) mb = max(mb, __shfl_xor_sync(0xffffffffu, mb, off));
            const float up = row_scale(mb);
#pragma unroll
            for (int x = 0; x < 4; ++x) v[x] *= up;
            if (lane == 0) s_c[r] = __fdiv_rn(a.c, up);
        } else if (lane == 0) {
            s_c[r] = a.c;
        }
        if (d < HD) {
#pragma unroll
            for (int pl = 0; pl < NQ; ++pl) {
                uint2 w;
                if constexpr (S::kInt8) {
                    w.x = pack_f16(v[0], v[1]);
                    w.y = pack_f16(v[2], v[3]);
                    const float2 x = unpack_f16(w.x), y = unpack_f16(w.y);
                    v[0] -= x.x;
                    v[1] -= x.y;
                    v[2] -= y.x;
                    v[3] -= y.y;
                } else {
                    w.x = pack_bf16(v[0], v[1]);
                    w.y = pack_bf16(v[2], v[3]);
                    v[0] -= bf16_lo(w.x);
                    v[1] -= bf16_hi(w.x);
                    v[2] -= bf16_lo(w.y);
                    v[3] -= bf16_hi(w.y);
                }
                s_q[((pl * NT + (r >> 3)) * KS + ks) * 32 + fl] = w;
            }
        }
    }
    __syncthreads();

    // Positions of this thread's rows (2 c, 2 c + 1 of each n tile).
    int pos[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int y = 0; y < 2; ++y) pos[nt][y] = sq.start + token_of(a, min(it.row0 + nt * 8 + 2 * c + y, it.row0 + it.rows - 1));

    // m: what the weights are taken against, at least the running maximum
    // less kAbove.
    float m[NT][2], l[NT][2], o[NT][MT][4], cr[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        m[nt][0] = m[nt][1] = -INFINITY;
        cr[nt][0] = s_c[nt * 8 + 2 * c];
        cr[nt][1] = s_c[nt * 8 + 2 * c + 1];
        l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[nt][t][e] = 0.0f;
    }

    bool bad = false;
#pragma unroll 1
    for (; i < it.i1; i += step) {
        float s[PG][NT][4];
#pragma unroll
        for (int x = 0; x < PG; ++x)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[x][nt][e] = 0.0f;
        // Small planes first: the tensor cores cut each sum to its own size,
        // and only the last KS sums are of the score's.  (INT8 bytes are
        // widened once for both planes.)
        constexpr int kTurns = S::kInt8 ? 1 : NQ;
#pragma unroll
        for (int turn = kTurns - 1; turn >= 0; --turn)
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                constexpr int here = NQ / kTurns;
                uint2 b[here][NT];
#pragma unroll
                for (int pl = 0; pl < here; ++pl)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) b[pl][nt] = s_q[(((turn + pl) * NT + nt) * KS + ks) * 32 + lane];
#pragma unroll
                for (int x = 0; x < PG; ++x) {
                    uint32_t w[2][2];
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        if constexpr (S::kInt8) {
                            const uint32_t q4 = kr[x][y][ks / 4][ks % 4];
                            w[y][0] = s8x2_to_f16x2(__byte_perm(q4, 0u, 0x4140u));
                            w[y][1] = s8x2_to_f16x2(__byte_perm(q4, 0u, 0x4342u));
                        } else {
                            w[y][0] = kr[x][y][ks / 2][ks % 2 * 2];
                            w[y][1] = kr[x][y][ks / 2][ks % 2 * 2 + 1];
                        }
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int pl = here - 1; pl >= 0; --pl)
                            if constexpr (S::kInt8)
                                mma16816h(s[x][nt], w[0][0], w[1][0], w[0][1], w[1][1], b[pl][nt].x, b[pl][nt].y);
                            else
                                mma16816(s[x][nt], w[0][0], w[1][0], w[0][1], w[1][1], b[pl][nt].x, b[pl][nt].y);
                }
            }
        // Scores, masked.
        bool whole[PG], all = true;
#pragma unroll
        for (int x = 0; x < PG; ++x) {
            const int j0 = page_of(i + x) * kPage;
            whole[x] = i + x < it.i1 && j0 + kPage - 1 <= p_lo &&
                       (a.window == 0 || j0 > p_hi - a.window || j0 + kPage <= a.sinks);
            all &= whole[x];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float t = s[x][nt][e];
                    if constexpr (S::kInt8) t *= ksc[x][e >> 1];
                    if (!whole[x]) {
                        // A visible key's -inf would pass for a hidden key.
                        if (i + x < it.i1 && sees(pos[nt][e & 1], j0 + g + (e >> 1) * 8, a.window, a.sinks))
                            bad |= S::kInt8 && t == -INFINITY;
                        else
                            t = -INFINITY;
                    }
                    s[x][nt][e] = t;
                }
            if (!S::kInt8 && !whole[x]) {
                // V rows that no row sees may hold anything: 0 * inf is not
                // 0 (INT8 values are always finite).
                const bool here = i + x < it.i1;
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    const int j = j0 + 2 * c + (y & 1) + (y >> 1) * 8;
                    if (!here || j >= it.hi || (j < it.w0 && j >= a.sinks))
#pragma unroll
                        for (int jj = 0; jj < VW / VP; ++jj)
#pragma unroll
                            for (int z = 0; z < VP; ++z) vr[x][y][jj][z] = 0u;
                }
            }
        }
        // This group's maximum of score * log2(e) (the row's factor c), with
        // log2 of the V row's scale added for INT8, and whether it passes the
        // base.
        float bm[NT][2];
        auto passes = [&]() {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) bm[nt][0] = bm[nt][1] = -INFINITY;
#pragma unroll
            for (int x = 0; x < PG; ++x) {
                float lv[2] = {0.0f, 0.0f};
                if constexpr (S::kInt8) {
                    lv[0] = scale_log2(vsc[x][0]);
                    lv[1] = scale_log2(vsc[x][1]);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float t = s[x][nt][e], f = cr[nt][e & 1];
                        bm[nt][e & 1] = fmaxf(bm[nt][e & 1], S::kInt8 ? fmaf(t, f, lv[e >> 1]) : t * f);
                    }
            }
            bool grow = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
#pragma unroll
                    for (int off = 4; off < 32; off <<= 1)
                        bm[nt][y] = fmaxf(bm[nt][y], __shfl_xor_sync(0xffffffffu, bm[nt][y], off));
                    grow |= bm[nt][y] > m[nt][y] + (8.0f + S::kAbove);
                }
            return (bool)__any_sync(0xffffffffu, grow);
        };
        const int nxt = i + step;
        ids(nxt);
        load_k();
        // The maximum may lag by a factor 2^8 (weights up to 256 are no less
        // exact): the rescaling of O is then rare.
        bool grow = passes();
        if constexpr (S::kInt8)
            if (grow) {
                // A V row of zeros must not set the base, whose scale says
                // nothing: taken as 0 it counts as the smallest, which keeps
                // the row's sum in range (a scale that is not finite makes
                // the result NaN and stays).  V is there only now: where the
                // base stays, nothing waits for it before the products.
#pragma unroll
                for (int x = 0; x < PG; ++x) {
                    uint32_t full[4];
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        uint32_t any = 0u;
#pragma unroll
                        for (int j = 0; j < VW / VP; ++j)
#pragma unroll
                            for (int z = 0; z < VP; ++z) any |= vr[x][y][j][z];
                        full[y] = __ballot_sync(0xffffffffu, any != 0u);
                    }
                    // Key 2 c + (y & 1) + (y >> 1) * 8 is row y of the lanes
                    // with that c; this thread's scales are of g and g + 8.
                    const uint32_t lanes = 0x11111111u << (g >> 1);
#pragma unroll
                    for (int y = 0; y < 2; ++y)
                        if (!((g & 1 ? full[2 * y + 1] : full[2 * y]) & lanes) && isfinite(vsc[x][y])) vsc[x][y] = 0.0f;
                }
                grow = passes();
            }
        if (grow) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const float mn = fmaxf(m[nt][y], bm[nt][y] - S::kAbove);
                    const float h = m[nt][y] == mn ? 1.0f : ex2_half(m[nt][y] - mn), f = h * h;
                    m[nt][y] = mn;
                    l[nt][y] = l[nt][y] * h * h;
#pragma unroll
                    for (int t = 0; t < MT; ++t) {
                        o[nt][t][y] *= f;
                        o[nt][t][2 + y] *= f;
                    }
                }
        }
#pragma unroll
        for (int x = 0; x < PG; ++x) {
            uint32_t pb[NT][NPV][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float p[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float t = s[x][nt][e];
                    // One rounding of the difference: score * c alone would
                    // carry one of its own size.
                    p[e] = ex2(fmaf(t, cr[nt][e & 1], -m[nt][e & 1]));
                    // Nothing seen so far leaves m at -inf; a hidden key's
                    // scale may be anything.
                    if (!all && t == -INFINITY) p[e] = 0.0f;
                    l[nt][e & 1] += p[e];
                    if constexpr (S::kInt8) {
                        p[e] *= vsc[x][e >> 1];
                        if (!all && t == -INFINITY) p[e] = 0.0f;
                    }
                }
#pragma unroll
                for (int pl = 0; pl < NPV; ++pl) {
                    uint32_t lo, hi;
                    if constexpr (S::kInt8) {
                        lo = pack_f16(p[0], p[1]);
                        hi = pack_f16(p[2], p[3]);
                    } else {
                        lo = pack_bf16(p[0], p[1]);
                        hi = pack_bf16(p[2], p[3]);
                    }
                    pb[nt][pl][0] = transpose8x8(lo);
                    pb[nt][pl][1] = transpose8x8(hi);
                    if (pl + 1 == NPV) break;
                    if constexpr (S::kInt8) {
                        const float2 u = unpack_f16(lo), v = unpack_f16(hi);
                        p[0] -= u.x;
                        p[1] -= u.y;
                        p[2] -= v.x;
                        p[3] -= v.y;
                    } else {
                        p[0] -= bf16_lo(lo);
                        p[1] -= bf16_hi(lo);
                        p[2] -= bf16_lo(hi);
                        p[3] -= bf16_hi(hi);
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                uint32_t w[4];
                if constexpr (S::kInt8) {
                    // Elements 2 t, 2 t + 1 of the thread: half a word.
                    const int jj = 2 * t / S::EPL, z = 2 * t % S::EPL / 4, hi = t & 1;
                    const uint32_t *k0 = vr[x][0][jj], *k1 = vr[x][1][jj], *k2 = vr[x][2][jj], *k3 = vr[x][3][jj];
                    const uint32_t sel0 = hi ? 0x0602u : 0x0400u, sel1 = hi ? 0x0703u : 0x0501u;
                    w[0] = s8x2_to_f16x2(__byte_perm(k0[z], k1[z], sel0));
                    w[1] = s8x2_to_f16x2(__byte_perm(k0[z], k1[z], sel1));
                    w[2] = s8x2_to_f16x2(__byte_perm(k2[z], k3[z], sel0));
                    w[3] = s8x2_to_f16x2(__byte_perm(k2[z], k3[z], sel1));
                } else {
                    const int jj = t / VP, z = t % VP;
                    w[0] = __byte_perm(vr[x][0][jj][z], vr[x][1][jj][z], 0x5410u);
                    w[1] = __byte_perm(vr[x][0][jj][z], vr[x][1][jj][z], 0x7632u);
                    w[2] = __byte_perm(vr[x][2][jj][z], vr[x][3][jj][z], 0x5410u);
                    w[3] = __byte_perm(vr[x][2][jj][z], vr[x][3][jj][z], 0x7632u);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int pl = NPV - 1; pl >= 0; --pl)
                        if constexpr (S::kInt8)
                            mma16816h(o[nt][t], w[0], w[1], w[2], w[3], pb[nt][pl][0], pb[nt][pl][1]);
                        else
                            mma16816(o[nt][t], w[0], w[1], w[2], w[3], pb[nt][pl][0], pb[nt][pl][1]);
            }
        }
        load_v();
    }

    // A result that is not finite may be a hidden value's doing (a key that
    // only some of the rows see, with weight 0 in the others) or the planes'
    // (an infinity times planes of both signs): such items go row by row.
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) bad |= !isfinite(o[nt][t][e]);
    if (__syncthreads_or(bad)) {
        for (int r = warp; r < it.rows; r += kStepWarps) attend_row<TV, TC>(a, item, r, kPage, lane);
        if (a.dependent) depend_wait();
        return;
    }

    // Join the warps: their maxima and sums, then the contexts in warp order.
    float *s_o = (float *)s_raw;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) l[nt][y] += __shfl_xor_sync(0xffffffffu, l[nt][y], off);
            if (g == 0) {
                s_m[warp][nt * 8 + 2 * c + y] = m[nt][y];
                s_l[warp][nt * 8 + 2 * c + y] = l[nt][y];
            }
        }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                float2 w = make_float2(o[nt][t][y], o[nt][t][2 + y]);
                *(float2 *)(s_o + ((size_t)warp * 8 * NT + nt * 8 + 2 * c + y) * S::OS + S::dim_of(g, 2 * t)) = w;
            }
    __syncthreads();
    for (int r = warp; r < it.rows; r += kStepWarps) {
        float mm = s_m[0][r];
#pragma unroll
        for (int w = 1; w < kStepWarps; ++w) mm = fmaxf(mm, s_m[w][r]);
        const float base = mm == -INFINITY ? 0.0f : mm;
        float f[kStepWarps], ll = 0.0f;
#pragma unroll
        for (int w = 0; w < kStepWarps; ++w) {
            const float h = s_m[w][r] == base ? 1.0f : ex2_half(s_m[w][r] - base);
            f[w] = h * h;
            ll = fmaf(s_l[w][r] * h, h, ll);
        }
        if (S::kInt8 && ll == 0.0f) {
            // It sees no key of these, or all scores left a float's range.
            attend_row<TV, TC>(a, item, r, kPage, lane);
            continue;
        }
        const size_t at = row_at(a, sq, it.kvh, it.row0 + r, (size_t)a.H * HD);
#pragma unroll
        for (int d0 = 0; d0 < HD; d0 += 32) {
            const int d = d0 + lane;
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < kStepWarps; ++w) v = fmaf(f[w], s_o[((size_t)w * 8 * NT + r) * S::OS + d], v);
            if (it.slot >= 0)
                a.ws[it.slot + (size_t)r * HD + d] = v;
            else
                store_value((TV *)a.y, at + d, __fdiv_rn(v, ll));
        }
        if (it.slot >= 0 && lane == 0) {
            a.ws[it.slot + (size_t)it.rows * HD + r] = mm;
            a.ws[it.slot + (size_t)it.rows * (HD + 1) + r] = ll;
        }
    }
    if (a.dependent) depend_wait();
}

template <typename TV, typename TC, int HD>
cudaError_t launch_nt(const Args &a, int nt, cudaStream_t st) {
    return launch(nt == 1 ? attend_step<TV, TC, HD, 1> : attend_step<TV, TC, HD, 2>, dim3(a.items), kStepWarps * 32, 0, st,
                  a.dependent != 0, a);
}

template <typename TV>
cudaError_t launch_tv(const Args &a, int cache, int nt, cudaStream_t st) {
    if (cache == QB_PAGED_BF16)
        return a.hd == 64 ? launch_nt<TV, uint16_t, 64>(a, nt, st) : launch_nt<TV, uint16_t, 128>(a, nt, st);
    return a.hd == 64 ? launch_nt<TV, int8_t, 64>(a, nt, st) : launch_nt<TV, int8_t, 128>(a, nt, st);
}

}  // namespace

cudaError_t step_attention(const Args &a, bool wide, int cache, int nt, cudaStream_t st) {
    return wide ? launch_tv<float>(a, cache, nt, st) : launch_tv<uint16_t>(a, cache, nt, st);
}

}  // namespace paged
}  // namespace qb
