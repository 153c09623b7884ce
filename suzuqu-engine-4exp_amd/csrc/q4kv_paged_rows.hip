/*
 * q4kv_paged_rows.hip -- paged attention of few columns (new tokens x query
 * heads of a KV head): 16 columns a tile, one token per request above all.
 *
 * A wave takes 16 positions at a time, their K and V rows straight from
 * global memory into registers in the layouts that the matrix products take
 * (no staging, no barrier in the loop):
 *  - scores: lane (c, g) holds K[position c][32 b + 8 g .. + 7], the A operand
 *    of S^T = K Q^T (v_mfma_f32_16x16x32_f16), the query columns in two fp16
 *    parts, each divided by the power of two that brings its largest
 *    magnitude into [0.5, 1); q8_0: exact int8 values in fp16, the block
 *    scales applied in fp32 to each block's product; f32: 16x16x4 products of
 *    fp32 operands;
 *  - online softmax in base 2, the running maximum raised only when a score
 *    passes it by 2^RAISE;
 *  - O^T += V^T P^T (16x16x16): the weights leave the score tile in the B
 *    layout; lane (c, g) holds U = hd / 16 consecutive dims U c .. of
 *    positions 4 g + i, regrouped in the lane into the A operands of U tiles
 *    (tile u, row r: dim U r + u); q8_0: v x scale in two fp16 parts, exact
 *    (VScale).
 * A buffer of K (of V) is filled again as soon as its products are issued, D
 * buffers deep, so that rows are in flight while other rows are computed. The
 * four waves of a workgroup take every fourth pass and are joined in LDS; the
 * runs of the workgroups are joined by a second launch (Share).
 *
 * What bounds it: the rows' bytes in large batches (64 requests, 8 KV heads of
 * 128 dims, f16: 1.43 GB in 284 us; 32 of 2 KV heads of 256 dims, q8_0: 1.57
 * GB in 359), the chain of dependent loads in small ones (lengths, page
 * numbers, rows, partials: one token over 1500 positions 17 us).
 */
#include <algorithm>

#include "q4kv_paged_attn.h"

namespace {

typedef uint32_t u2a_t __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u4a_t __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u1a_t __attribute__((aligned(2)));

constexpr uint32_t PASS = 16; /* positions of a wave's pass, and its columns */
/* in positions: a tile's start, what cuts keep from its ends, runs (Share) */
constexpr uint32_t START = 64, SNAP = 64, MIN_RUN = 64, MAX_RUN = 256;
constexpr float RAISE = 6.f;

/* K and V of a pass in registers */
template <int KIND, int HD> struct Rows {
    static constexpr uint32_t NB = HD / 32, U = HD / 16;
    u2_t kq[KIND == Q4KV_Q8 ? NB : 1];
    uint16_t ks[KIND == Q4KV_Q8 ? (NB + 3) / 4 : 1]; /* scale of blocks jg, 4 + jg of row c */
    u4_t kh[KIND == Q4KV_F16 ? NB : 1];
    f4_t kf[KIND == Q4KV_F32 ? HD / 16 : 1]; /* dims 16 x + 4 jg .. */
    uint32_t v[4][KIND == Q4KV_Q8 ? U / 4 : KIND == Q4KV_F16 ? U / 2 : U]; /* dims U c .. of positions 4 jg + i */
    uint16_t vs[KIND == Q4KV_Q8 ? 4 : 1];
    uint32_t slot;  /* of position c */
    uint32_t mask;  /* positions that exist */
};

template <int N> __device__ inline void load_words(uint32_t (&d)[N], const uint8_t *p) {
    if constexpr (N == 1) {
        d[0] = *(const GLOBAL u1a_t *)p;
    } else if constexpr (N == 2) {
        const u2_t x = *(const GLOBAL u2a_t *)p;
        d[0] = x[0];
        d[1] = x[1];
    } else {
#pragma unroll
        for (int k = 0; k < N; k += 4) {
            const u4_t x = *(const GLOBAL u4a_t *)(p + 4 * k);
#pragma unroll
            for (int e = 0; e < 4; e++) d[k + e] = x[e];
        }
    }
}

/* CG column groups of 16: the waves of a group take every NS-th pass, the
 * groups the same rows (one fetch of them from memory, not two).
 * FULL: the head has HD dims, not fewer. */
template <int KIND, int HD, int D, int CG, bool FULL>
__global__ __launch_bounds__(256, 2) void paged_rows_k(PagedArgs a) {
    constexpr uint32_t NB = HD / 32, U = HD / 16, MROW = HD + 4;
    constexpr uint32_t NC = 16 * CG, NS = 4 / CG, STEP = PASS * NS; /* positions of a workgroup's pass */
    typedef Share<NC, START, SNAP, MIN_RUN, MAX_RUN, 256> Runs;
    /* the query operands while a tile runs (the waves share them: 64 registers
     * a lane at 256 dims), the waves' sums after it */
    constexpr uint32_t QW = 2 * NB; /* 16-byte words a lane */
    __shared__ __attribute__((aligned(16))) float mrg[4 * 16 * MROW];
    static_assert(sizeof(mrg) >= CG * QW * 64 * 16, "query operands fit");
    __shared__ __attribute__((aligned(16))) float s_ks[4][KIND == Q4KV_Q8 ? NB * 16 : 4];
    __shared__ float s_m[4][16], s_l[4][16];
    __shared__ uint16_t s_odd[4][PASS * 16]; /* [position][lane c]: values that are not finite */
    __shared__ typename Runs::Lds lds;

    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = uni(tid >> 6);
    const uint32_t c = lane & 15u, jg = lane >> 4, group = wave % CG, part = wave / CG;
    u4_t *const s_q = (u4_t *)mrg + group * QW * 64u;
    const uint32_t hd = FULL ? (uint32_t)HD : a.hd, nb = hd / 32u;
    const size_t slot_b = (size_t)a.n_kvh * a.rowb;
    Cut *const cuts = (Cut *)a.part;
    float *const parts = a.part + gridDim.x * (sizeof(Cut) / 4u);

    Runs run;
    const bool any = run.find(a, lds);
    Cut cut = {};
    while (any) {
        const Req &r = run.req;
        const uint32_t seq = run.seq, kh = run.kh;
        const uint32_t col = run.tile * NC + 16u * group + c;
        const bool live = col < run.tiles.cols;
        const uint32_t t = live ? col / a.gqa : 0u, h = live ? col - t * a.gqa : 0u;
        /* the positions that the tile's last, its first and this lane's column see */
        const uint32_t n_all = uni(seen_by(r, (min((run.tile + 1u) * NC, run.tiles.cols) - 1u) / a.gqa));
        const uint32_t n_min = uni(seen_by(r, run.tile * NC / a.gqa));
        const uint32_t n_c = live ? seen_by(r, t) : 0u;
        uint32_t q0, q1;
        bool begins, ends;
        run.piece(a, (n_all + STEP - 1u) / STEP, q0, q1, begins, ends);
        const uint32_t j0 = q0 * STEP, j1 = min(q1 * STEP, n_all);
        /* passes of this wave: none without a column */
        const uint32_t nk = j1 > j0 && run.tile * NC + 16u * group < run.tiles.cols ? (j1 - j0 + STEP - 1u) / STEP : 0u;
        const int32_t *const trow = a.table + (size_t)seq * a.stride;
        const uint8_t *const kb = a.kp + (size_t)kh * a.rowb, *const vb = a.vp + (size_t)kh * a.rowb;

        /* page number of position c of pass k; past the end the last one's */
        auto entry = [&](uint32_t k) -> int32_t {
            const uint32_t p = min(j0 + STEP * k + PASS * part + c, j1 - 1u);
            return ldg(trow + q4kv_page_of(a.page, p));
        };
        auto resolve = [&](uint32_t k, int32_t number, uint32_t &slot, uint32_t &mask) {
            const uint32_t e = j0 + STEP * k + PASS * part + c, p = min(e, j1 - 1u);
            const bool ok = e < j1 && (uint32_t)number < a.n_pages;
            mask = (uint32_t)__ballot(ok) & 0xFFFFu;
            const uint32_t s = (uint32_t)number * a.page.d + (p - q4kv_page_of(a.page, p) * a.page.d);
            /* positions that do not exist read the first one that does (slot 0 without one) */
            const uint32_t first = mask ? (uint32_t)__builtin_amdgcn_readlane(s, __builtin_ctz(mask)) : 0u;
            slot = ok ? s : first;
        };
        typedef Rows<KIND, HD> R;
        auto load_k = [&](R &b) {
            const uint8_t *kr = kb + (size_t)b.slot * slot_b;
            if constexpr (KIND == Q4KV_Q8) {
#pragma unroll
                for (uint32_t x = 0; x < (NB + 3u) / 4u; x++)
                    b.ks[x] = ldg((const uint16_t *)(kr + 34u * min(4u * x + jg, nb - 1u)));
#pragma unroll
                for (uint32_t x = 0; x < NB; x++) b.kq[x] = *(const GLOBAL u2a_t *)(kr + 34u * min(x, nb - 1u) + 2u + 8u * jg);
            } else if constexpr (KIND == Q4KV_F16) {
#pragma unroll
                for (uint32_t x = 0; x < NB; x++) b.kh[x] = ldg((const u4_t *)(kr + 64u * min(x, nb - 1u) + 16u * jg));
            } else {
#pragma unroll
                for (uint32_t x = 0; x < HD / 16u; x++)
                    b.kf[x] = ldg((const f4_t *)(kr + 64u * min(x, 2u * nb - 1u) + 16u * jg));
            }
        };
        const uint32_t vdim = U * c < hd ? U * c : 0u; /* dims past the head read its first ones */
        auto load_v = [&](R &b) {
#pragma unroll
            for (uint32_t i = 0; i < 4u; i++) {
                const uint32_t s = (uint32_t)__builtin_amdgcn_ds_bpermute((int)((4u * jg + i) * 4u), (int)b.slot);
                const uint8_t *vr = vb + (size_t)s * slot_b;
                if constexpr (KIND == Q4KV_Q8) {
                    const uint8_t *blk = vr + 34u * (vdim / 32u);
                    b.vs[i] = ldg((const uint16_t *)blk);
                    load_words(b.v[i], blk + 2u + (vdim & 31u));
                } else {
                    load_words(b.v[i], vr + vdim * (KIND == Q4KV_F16 ? 2u : 4u));
                }
            }
        };

        R buf[D];
        int32_t number[D];
        if (nk) {
#pragma unroll
            for (int d = 0; d < D; d++) number[d] = entry(d);
        }
        /* ---- Q^T operands of column c: words [x][lane], the fp16 parts of
         * block b at 2 b and 2 b + 1; every wave writes its share ---- */
        float qmul = 1.f;
        {
            /* the loads of q ahead of those of the first rows */
            constexpr uint32_t MB = (NB + NS - 1u) / NS; /* blocks part, part + NS, .. */
            const float *qr = a.q + ((size_t)(r.t0 + t) * a.n_head + kh * a.gqa + h) * hd;
            float x[MB][8];
#pragma unroll
            for (uint32_t m = 0; m < MB; m++)
#pragma unroll
                for (uint32_t i = 0; i < 8u; i++) {
                    /* f32: words 2 b and 2 b + 1 of block b, four dims each */
                    const uint32_t b = min(NS * m + part, nb - 1u);
                    x[m][i] = ldg(qr + 32u * b + (KIND == Q4KV_F32 ? 16u * (i / 4u) + 4u * jg + (i & 3u) : 8u * jg + i));
                }
            if (nk) {
#pragma unroll
                for (int d = 0; d < D; d++) {
                    resolve(d, number[d], buf[d].slot, buf[d].mask);
                    load_k(buf[d]);
                    load_v(buf[d]);
                }
#pragma unroll
                for (int d = 0; d < D; d++) number[d] = entry(D + d);
            }

            float am = 0.f;
#pragma unroll
            for (uint32_t m = 0; m < MB; m++)
#pragma unroll
                for (uint32_t i = 0; i < 8u; i++) {
                    x[m][i] = live && NS * m + part < nb ? x[m][i] : 0.f;
                    am = fmaxf(am, fabsf(x[m][i]));
                }
            float qs = a.scale_log2;
            if constexpr (KIND != Q4KV_F32) {
                am = max32(max16(am));
                s_m[wave][c] = am;
                __syncthreads();
                #pragma unroll
                for (uint32_t p = 0; p < NS; p++) am = fmaxf(am, s_m[CG * p + group][c]);
                am *= fabsf(a.scale_log2);
                const int e = (am > 0.f && am <= 3.4e38f) ? __builtin_amdgcn_frexp_expf(am) : 0;
                qmul = __builtin_ldexpf(1.f, e);
                qs = __builtin_ldexpf(a.scale_log2, -e);
            }
#pragma unroll
            for (uint32_t m = 0; m < MB; m++) {
                const uint32_t b = NS * m + part;
                if (b >= NB) continue;
                u4_t wh, wl;
#pragma unroll
                for (uint32_t i = 0; i < 4u; i++) {
                    if constexpr (KIND == Q4KV_F32) {
                        wh[i] = __float_as_uint(x[m][i] * qs);
                        wl[i] = __float_as_uint(x[m][4u + i] * qs);
                    } else {
                        const float y0 = x[m][2u * i] * qs, y1 = x[m][2u * i + 1u] * qs;
                        wh[i] = pk(y0, y1);
                        wl[i] = pk(y0 - h2lo(wh[i]), y1 - h2hi(wh[i]));
                    }
                }
                s_q[(2u * b) * 64u + lane] = wh;
                s_q[(2u * b + 1u) * 64u + lane] = wl;
            }
        }
        __syncthreads(); /* s_q is written */

        float m_run = -INFINITY, l_run = 0.f;
        f4_t acc[U];
#pragma unroll
        for (uint32_t u = 0; u < U; u++) acc[u] = (f4_t){0.f, 0.f, 0.f, 0.f};
        VScale vq;
        uint64_t nan_out = 0u; /* bit U i + u: acc[u][i] sums a value that is not finite */

        auto pass = [&](uint32_t k, R &b, int32_t &next) {
            const uint32_t base = j0 + STEP * k + PASS * part;
            const uint32_t mask = b.mask;
            /* ---- S^T = K Q^T ---- */
            f4_t S = {0.f, 0.f, 0.f, 0.f};
            if constexpr (KIND == Q4KV_Q8) {
                /* the rows' scales, to the lanes that hold their positions */
#pragma unroll
                for (uint32_t x = 0; x < (NB + 3u) / 4u; x++)
                    if (4u * x + jg < NB) s_ks[wave][16u * (4u * x + jg) + c] = (float)__builtin_bit_cast(_Float16, b.ks[x]);
                __builtin_amdgcn_wave_barrier();
                /* two blocks at a time, their scales applied one stage late */
                f4_t C[NB];
                auto scaled = [&](uint32_t x) {
                    const f4_t ks = *(const f4_t *)&s_ks[wave][16u * x + 4u * jg];
#pragma unroll
                    for (uint32_t i = 0; i < 4u; i++) S[i] = fmaf(ks[i], C[x][i], S[i]);
                };
#pragma unroll
                for (uint32_t x0 = 0; x0 < NB; x0 += 2u) {
                    u4_t w[2];
                    h8_t qh[2], ql[2];
#pragma unroll
                    for (uint32_t j = 0; j < 2u; j++) {
                        const uint32_t x = x0 + j;
                        qh[j] = __builtin_bit_cast(h8_t, s_q[(2u * x) * 64u + lane]);
                        ql[j] = __builtin_bit_cast(h8_t, s_q[(2u * x + 1u) * 64u + lane]);
                        h2_t y[4];
                        biased_h4(b.kq[x][0], y[0], y[1]);
                        biased_h4(b.kq[x][1], y[2], y[3]);
#pragma unroll
                        for (uint32_t i = 0; i < 4u; i++)
                            w[j][i] = __builtin_bit_cast(uint32_t, y[i] - (h2_t)((_Float16)1152.f));
                    }
#pragma unroll
                    for (uint32_t j = 0; j < 2u; j++)
                        C[x0 + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, w[j]), ql[j],
                                                                          (f4_t){0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
                    for (uint32_t j = 0; j < 2u; j++)
                        C[x0 + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, w[j]), qh[j], C[x0 + j], 0, 0, 0);
                    if (x0) {
                        scaled(x0 - 2u);
                        scaled(x0 - 1u);
                    }
                }
                scaled(NB - 2u);
                scaled(NB - 1u);
                __builtin_amdgcn_wave_barrier();
            } else if constexpr (KIND == Q4KV_F16) {
                f4_t Sl = {0.f, 0.f, 0.f, 0.f}; /* the small parts apart: fewer roundings at the sum's size */
#pragma unroll
                for (uint32_t x = 0; x < NB; x++) {
                    const h8_t qh = __builtin_bit_cast(h8_t, s_q[(2u * x) * 64u + lane]);
                    const h8_t ql = __builtin_bit_cast(h8_t, s_q[(2u * x + 1u) * 64u + lane]);
                    Sl = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, b.kh[x]), ql, Sl, 0, 0, 0);
                    S = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, b.kh[x]), qh, S, 0, 0, 0);
                    if (x & 1u) __builtin_amdgcn_sched_barrier(0);
                }
                S += Sl;
            } else {
                /* sums of 8 products at 64 dims, 32 at 128: each is rounded at the
                 * size of the sum so far, one large product makes all that
                 * follow coarse (24 / 2 heads of 64 dims: 1.4e-6 in norm with
                 * sums of 32, now 8.4e-7; the registers for more are not there at 256) */
                constexpr uint32_t NA = HD == 64 ? 8 : HD == 128 ? 4 : 2;
                f4_t Sx[NA];
#pragma unroll
                for (uint32_t x = 0; x < NA; x++) Sx[x] = (f4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (uint32_t x = 0; x < HD / 16u; x++) {
                    const f4_t qf = __builtin_bit_cast(f4_t, s_q[x * 64u + lane]);
#pragma unroll
                    for (uint32_t e = 0; e < 4u; e++) {
                        f4_t &s = Sx[(4u * x + e) % NA];
                        s = __builtin_amdgcn_mfma_f32_16x16x4f32(b.kf[x][e], qf[e], s, 0, 0, 0);
                    }
                    if (x & 1u) __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (uint32_t n = NA / 2u; n; n /= 2u)
#pragma unroll
                    for (uint32_t x = 0; x < n; x++) Sx[x] += Sx[x + n];
                S = Sx[0];
            }
            uint32_t slot_next, mask_next;
            resolve(k + D, next, slot_next, mask_next);
            next = entry(k + 2 * D);
            /* V of this pass is regrouped from the old slots' rows, which are
             * in flight already */
            b.slot = slot_next;
            load_k(b);
            __builtin_amdgcn_sched_barrier(0);
            /* ---- online softmax ---- */
            float T[4];
#pragma unroll
            for (uint32_t i = 0; i < 4u; i++) {
                const uint32_t p = 4u * jg + i;
                T[i] = ((mask >> p) & 1u) && base + p < n_c ? S[i] * qmul : -INFINITY;
            }
            const float mx = fmax2(fmax2(T[0], T[1]), fmax2(T[2], T[3]));
            uint32_t vs[4], vtop = 0u;
            if constexpr (KIND == Q4KV_Q8) {
#pragma unroll
                for (uint32_t i = 0; i < 4u; i++) /* a stand-in row may hold inf or NaN */
                    vs[i] = (mask >> (4u * jg + i)) & 1u ? b.vs[i] : 0u;
                vtop = max(max(vs[0], vs[1]), max(vs[2], vs[3]));
            }
            /* one branch for the maximum and for large scales (negative ones,
             * which the quantiser never writes, and infinities come here too) */
            if (__ballot(mx > m_run + RAISE || (KIND == Q4KV_Q8 && vtop >= 0x6000u)) != 0u) {
                float f = 1.f;
                if (KIND == Q4KV_Q8 && !vq.big() &&
                    __ballot(q4kv_big_scale(vs[0]) || q4kv_big_scale(vs[1]) || q4kv_big_scale(vs[2]) ||
                             q4kv_big_scale(vs[3])) != 0u) {
                    vq.divide();
                    f = VSCALE_STEP;
                }
                const float mn = fmax2(m_run, max32(max16(mx)));
                const float alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run - mn);
                l_run *= alpha;
                f *= alpha;
#pragma unroll
                for (uint32_t u = 0; u < U; u++) acc[u] *= f;
                m_run = mn;
            }
            const float ms = m_run == -INFINITY ? 0.f : m_run;
#pragma unroll
            for (uint32_t i = 0; i < 4u; i++) T[i] = __builtin_amdgcn_exp2f(T[i] - ms);
            l_run += (T[0] + T[1]) + (T[2] + T[3]);
            /* a stand-in row may hold inf or NaN */
            if (KIND == Q4KV_F16 && mask != 0xFFFFu) {
#pragma unroll
                for (uint32_t i = 0; i < 4u; i++)
#pragma unroll
                    for (uint32_t u = 0; u < sizeof(b.v[0]) / 4u; u++)
                        b.v[i][u] = (mask >> (4u * jg + i)) & 1u ? b.v[i][u] : 0u;
            }
            /* ---- rows that some columns do not see yet may hold inf or NaN,
             * which a weight of zero would turn into NaN there: they are taken
             * out of the operands, and the columns that see them get NaN ---- */
            uint32_t odd[4] = {0u, 0u, 0u, 0u};
            bool odd_seen = false;
            if (base + PASS > n_min) {
#pragma unroll
                for (uint32_t i = 0; i < 4u; i++) {
                    if constexpr (KIND == Q4KV_Q8) {
                        odd[i] = (vs[i] & 0x7C00u) == 0x7C00u ? (1u << U) - 1u : 0u;
                    } else {
#pragma unroll
                        for (uint32_t u = 0; u < U; u++) {
                            const bool bad = KIND == Q4KV_F16 ? ((b.v[i][u / 2u] >> (16u * (u & 1u))) & 0x7C00u) == 0x7C00u
                                                              : (b.v[i][u] & 0x7F800000u) == 0x7F800000u;
                            odd[i] |= bad ? 1u << u : 0u;
                        }
                        if (!((mask >> (4u * jg + i)) & 1u)) odd[i] = 0u;
                    }
                }
                odd_seen = __ballot((odd[0] | odd[1] | odd[2] | odd[3]) != 0u) != 0u;
            }
            if (odd_seen) {
                uint16_t *const bits = s_odd[wave];
#pragma unroll
                for (uint32_t i = 0; i < 4u; i++) {
                    bits[(4u * jg + i) * 16u + c] = (uint16_t)odd[i];
                    if (KIND == Q4KV_Q8) {
                        if (odd[i]) vs[i] = 0u;
                    } else {
#pragma unroll
                        for (uint32_t u = 0; u < U; u++)
                            if (odd[i] >> u & 1u) {
                                if (KIND == Q4KV_F16)
                                    b.v[i][u / 2u] &= u & 1u ? 0x0000FFFFu : 0xFFFF0000u;
                                else
                                    b.v[i][u] = 0u;
                            }
                    }
                }
                __builtin_amdgcn_wave_barrier();
#pragma unroll 1
                for (uint32_t p = 0; p < PASS; p++) {
                    if (!((mask >> p) & 1u) || base + p >= n_c) continue;
#pragma unroll
                    for (uint32_t i = 0; i < 4u; i++) {
                        const uint32_t w = bits[p * 16u + 4u * jg + i];
                        nan_out |= (uint64_t)w << (U * i);
                    }
                }
                __builtin_amdgcn_wave_barrier();
            }
            /* ---- O^T += V^T P^T ---- */
            if constexpr (KIND == Q4KV_F32) {
#pragma unroll
                for (uint32_t i = 0; i < 4u; i++)
#pragma unroll
                    for (uint32_t u = 0; u < U; u++)
                        acc[u] = __builtin_amdgcn_mfma_f32_16x16x4f32((mask >> (4u * jg + i)) & 1u ? __uint_as_float(b.v[i][u]) : 0.f,
                                                                      T[i], acc[u], 0, 0, 0);
            } else {
                constexpr uint32_t NV = KIND == Q4KV_Q8 ? 2 : 1;
                const uint32_t h0 = pk(T[0], T[1]), h1 = pk(T[2], T[3]);
                const h4_t Bh = __builtin_bit_cast(h4_t, (u2_t){h0, h1});
                const h4_t Bl = __builtin_bit_cast(h4_t, (u2_t){pk(T[0] - h2lo(h0), T[1] - h2hi(h0)), pk(T[2] - h2lo(h1), T[3] - h2hi(h1))});
                h2_t sc[2];
                if constexpr (KIND == Q4KV_Q8) {
                    sc[0] = __builtin_bit_cast(h2_t, vs[0] | vs[1] << 16);
                    sc[1] = __builtin_bit_cast(h2_t, vs[2] | vs[3] << 16);
                }
                /* V^T of four tiles, dims U c + 4 d .. + 3: [tile][part], two
                 * words of the four positions */
                auto regroup = [&](uint32_t d, u2_t (&A)[4][NV]) {
#pragma unroll
                    for (uint32_t o = 0; o < 4u; o++)
#pragma unroll
                        for (uint32_t p = 0; p < 2u; p++) {
                            if constexpr (KIND == Q4KV_F16) {
                                A[o][0][p] = __builtin_amdgcn_perm(b.v[2u * p + 1u][2u * d + (o >> 1)], b.v[2u * p][2u * d + (o >> 1)],
                                                                   o & 1u ? 0x07060302u : 0x05040100u);
                            } else {
                                /* byte o of both rows under fp16's 1024, v from that, its
                                 * product with the scale rounded once, what that left */
                                const uint32_t w = __builtin_amdgcn_perm(b.v[2u * p + 1u][d], b.v[2u * p][d], 0x0C040C00u + 0x00010001u * o);
                                const h2_t f = vq.value(__builtin_bit_cast(h2_t, w ^ 0x64806480u));
                                const h2_t hi = f * sc[p];
                                A[o][0][p] = __builtin_bit_cast(uint32_t, hi);
                                A[o][NV - 1u][p] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(f, sc[p], -hi));
                            }
                        }
                };
                u2_t A[2][4][NV];
                regroup(0u, A[0]);
#pragma unroll
                for (uint32_t d = 0; d < U / 4u; d++) {
                    __builtin_amdgcn_sched_barrier(0);
                    /* the next tiles' operands between this one's products */
                    if (d + 1u < U / 4u) regroup(d + 1u, A[(d + 1u) & 1u]);
                    if constexpr (NV == 2) {
#pragma unroll
                        for (uint32_t o = 0; o < 4u; o++)
                            acc[4u * d + o] = __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(h4_t, A[d & 1u][o][1]), Bh, acc[4u * d + o], 0, 0, 0);
                    }
#pragma unroll
                    for (uint32_t o = 0; o < 4u; o++)
                        acc[4u * d + o] = __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(h4_t, A[d & 1u][o][0]), Bl, acc[4u * d + o], 0, 0, 0);
#pragma unroll
                    for (uint32_t o = 0; o < 4u; o++)
                        acc[4u * d + o] = __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(h4_t, A[d & 1u][o][0]), Bh, acc[4u * d + o], 0, 0, 0);
#pragma unroll
                    for (uint32_t k = 0; k < 8u + 4u * (NV - 1u); k++) {
                        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x002, NV == 2 ? 4 : 2, 0);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            b.mask = mask_next;
            load_v(b);
            __builtin_amdgcn_sched_barrier(0);
        };
        for (uint32_t k = 0; k < nk; k += D) {
#pragma unroll
            for (int d = 0; d < D; d++) pass(k + d, buf[d], number[d]);
        }

        /* ---- the waves' sums, then the rows or the run's partial. A thread
         * has up to TASKS times four dims of a column; their gates are on the
         * way while the sums are joined, or four at a time (one after the other
         * they took 10 us of a launch of whole tiles) ---- */
        constexpr uint32_t TASKS = NC * (HD / 4) / 256;
        constexpr bool AHEAD = CG == 1 && !(KIND == Q4KV_F32 && HD == 256); /* registers for it */
        constexpr uint32_t WAYS = AHEAD ? TASKS : KIND == Q4KV_F32 ? 1 : TASKS < 4 ? TASKS : 4;
        constexpr bool GATES = AHEAD || KIND != Q4KV_F32;
        static_assert(TASKS % WAYS == 0, "whole trips");
        const uint32_t n_col = min(NC, run.tiles.cols - run.tile * NC);
        const bool whole = begins && ends;
        auto out_at = [&](uint32_t task) {
            const uint32_t cj = run.tile * NC + task / (HD / 4u), tj = cj / a.gqa;
            return ((size_t)(r.t0 + tj) * a.n_head + kh * a.gqa + (cj - tj * a.gqa)) * hd + 4u * (task % (HD / 4u));
        };
        f4_t gate[WAYS];
        auto load_gates = [&](uint32_t k0) {
            if (!whole || !a.gate) return;
#pragma unroll
            for (uint32_t k = 0; k < WAYS; k++) {
                const uint32_t task = tid + 256u * (k0 + k);
                const float *g = a.gate + (task < n_col * (HD / 4u) && 4u * (task % (HD / 4u)) < hd ? out_at(task) : 0u);
#pragma unroll
                for (uint32_t i = 0; i < 4u; i++) gate[k][i] = ldg(g + i);
            }
        };
        if (AHEAD) load_gates(0u);
        __syncthreads(); /* s_q is read */
        {
            const float lw = pair32_sum(sum16(l_run));
            if (jg == 0u) {
                s_m[wave][c] = m_run;
                s_l[wave][c] = lw;
            }
            const float vmul = vq.undo();
            if (nan_out) {
#pragma unroll
                for (uint32_t i = 0; i < 4u; i++)
#pragma unroll
                    for (uint32_t u = 0; u < U; u++)
                        if ((nan_out >> (U * i + u)) & 1u) acc[u][i] = __builtin_nanf("");
            }
#pragma unroll
            for (uint32_t i = 0; i < 4u; i++) {
                float *d = mrg + (wave * 16u + c) * MROW + U * (4u * jg + i);
#pragma unroll
                for (uint32_t u = 0; u < U; u += 4u)
                    *(f4_t *)(d + u) = (f4_t){acc[u][i], acc[u + 1u][i], acc[u + 2u][i], acc[u + 3u][i]} * vmul;
            }
        }
        __syncthreads();
        float *const slot = parts + (size_t)(2u * (run.g * a.n_kvh + kh) + (begins ? 1u : 0u)) * (NC * (HD + PAGED_PHEAD));
#pragma unroll 1
        for (uint32_t k0 = 0; k0 < TASKS && tid + 256u * k0 < n_col * (HD / 4u); k0 += WAYS) {
            if (GATES && !AHEAD) load_gates(k0);
#pragma unroll
            for (uint32_t k = 0; k < WAYS; k++) {
                const uint32_t task = tid + 256u * (k0 + k);
                if (task >= n_col * (HD / 4u)) break;
                const uint32_t j = task / (HD / 4u), d = 4u * (task % (HD / 4u));
                const uint32_t w0 = j / 16u, i = j & 15u; /* the group's waves: w0, w0 + CG, .. */
                float M = -INFINITY, L = 0.f;
#pragma unroll
                for (uint32_t p = 0; p < NS; p++) M = fmax2(M, s_m[w0 + CG * p][i]);
                f4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (uint32_t p = 0; p < NS; p++) {
                    const uint32_t w = w0 + CG * p;
                    const float lw = s_l[w][i];
                    if (lw == 0.f) continue; /* nothing seen; a NaN takes part */
                    const float f = s_m[w][i] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(s_m[w][i] - M);
                    L = fmaf(f, lw, L);
                    v += f * *(const f4_t *)(mrg + (w * 16u + i) * MROW + d);
                }
                if (whole) {
                    if (d >= hd) continue;
                    const size_t ro = out_at(task);
                    const float inv = L != 0.f ? 1.f / L : 0.f;
#pragma unroll
                    for (uint32_t i = 0; i < 4u; i++) {
                        float o = v[i] * inv;
                        if (a.gate) o *= q4kv_sigmoid(GATES ? gate[k][i] : ldg(a.gate + ro + i));
                        stg(a.out + ro + i, o);
                    }
                } else {
                    float *pr = slot + j * (HD + PAGED_PHEAD);
                    if (d == 0u) stg((f2_t *)pr, (f2_t){M, L});
                    stg((f4_t *)(pr + PAGED_PHEAD + d), v);
                }
            }
        }
        if (begins && !ends) cut = Cut{run.pieces(a), run.g, kh, run.tile, r.t0, run.tiles.cols, {}};
        run.advance(a);
        if (run.u >= run.end) break;
        __syncthreads(); /* mrg is read */
    }
    if (tid == 0u) {
        uint32_t *const cw = (uint32_t *)(cuts + blockIdx.x);
        stg((u4_t *)cw, (u4_t){cut.pieces, cut.g, cut.kh, cut.tile});
        stg((u2_t *)(cw + 4), (u2_t){cut.t0, cut.cols});
    }
}

template <int KIND, int HD, int D, int CG> bool launch(PagedArgs a) {
    /* two workgroups a CU */
    constexpr uint32_t G = 512, NC = 16 * CG;
    static_assert(paged_part_floats(G, NC, HD) <= (CG == 1 ? (size_t)8 << 20 : Q4KV_TILE_FLOATS),
                  "the scratch holds the partials");
    a.unit = q4kv_paged_unit(a, NC, START);
    a.runs = q4kv_paged_runs(G, a.n_kvh);
    const uint32_t grid = a.runs * a.n_kvh;
    const bool prof = q4kv_prof_open();
    if (a.hd == HD)
        paged_rows_k<KIND, HD, D, CG, true><<<grid, 256, 0, q4kv_stream>>>(a);
    else
        paged_rows_k<KIND, HD, D, CG, false><<<grid, 256, 0, q4kv_stream>>>(a);
    q4kv_prof_close(prof);
    paged_merge_k<HD, NC><<<dim3(grid, NC), 256, 0, q4kv_stream>>>(a);
    return q4kv_launch_ok("paged attention, few columns");
}

template <int KIND, int CG> bool launch_hd(const PagedArgs &a) {
    if (a.hd <= 64u) return launch<KIND, 64, 2, CG>(a);
    if (a.hd <= 128u) return launch<KIND, 128, 2, CG>(a);
    return launch<KIND, 256, 1, CG>(a);
}
template <int KIND> bool launch_cols(const PagedArgs &a, uint32_t cols) {
    return cols == 32u ? launch_hd<KIND, 2>(a) : launch_hd<KIND, 1>(a);
}

} // namespace

bool q4kv_paged_rows_launch(int kind, const PagedArgs &a, uint32_t cols) {
    return kind == Q4KV_Q8    ? launch_cols<Q4KV_Q8>(a, cols)
           : kind == Q4KV_F16 ? launch_cols<Q4KV_F16>(a, cols)
                              : launch_cols<Q4KV_F32>(a, cols);
}
