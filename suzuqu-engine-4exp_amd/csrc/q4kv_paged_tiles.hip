/*
 * q4kv_paged_tiles.hip -- paged attention of many columns (new tokens x query
 * heads of a KV head): chunks of prompts, q8_0 and f16 caches.
 *
 * Tiles of 128 columns, 16 to each of 8 waves. The positions stream through
 * LDS once per tile, PT = 8192 / HD at a time: the next pass's rows are
 * loaded into registers, through the block table, while this one computes,
 * converted once for all columns and stored to the other LDS buffer (one
 * barrier a pass). q8_0: K as its exact int8 values in fp16 beside the block
 * scales, V as v * scale in two fp16 parts, exact (VScale); f16: as stored.
 *  - S^T = K Q^T on v_mfma_f32_16x16x32_f16, Q in two fp16 parts (each
 *    column's q divided by the power of two that brings its largest magnitude
 *    into [0.5, 1)), q8_0 block scales in fp32 on each block's product;
 *  - online softmax in base 2, the running maximum raised only when a score
 *    passes it by 2^RAISE;
 *  - O^T += V^T P^T: the weights leave the score tile in the product's layout
 *    (slot 8 g + i of a k-group is position 4 g + i, or 16 + 4 g + i - 4) and
 *    are split into two fp16 parts in the lane; V^T comes from the row-major
 *    tile by ds_read_b64_tr_b16.
 * An fp32 result takes two parts of q and of the weights (and of q8_0's V x
 * scale): 2 (f16) or 2.5 (q8_0) products for each of the plain contraction.
 *
 * What bounds it: the matrix pipe, shared with the conversions and softmax of
 * the other wave of a SIMD. One workgroup fills a CU's LDS; 256 of them run
 * equal shares of the batch (Share), so causal tiles and ragged requests end
 * together. 4096 tokens of 16 / 2 heads of 256 dims after 8192, f16: 1280 to
 * 1360 us by the card, 1.0 to 1.07 PFLOP/s of products issued; the pipe is busy
 * 47 % of the time, as it is in a large library product (51 %).
 */
#include "q4kv_paged_attn.h"

namespace {

constexpr uint32_t NWAVE = 8, NTHR = 64 * NWAVE, COLS = 16 * NWAVE;
constexpr float RAISE = 6.f;

template <int KIND, int HD> struct Geo {
    static constexpr uint32_t NB = HD / 32, PT = 8192 / HD, NT = PT / 16, KG = PT / 32;
    static constexpr uint32_t KS = HD * 2 + 32; /* K row bytes in LDS: 16-row reads without conflicts */
    static constexpr uint32_t VS = HD * 2;      /* V row bytes (vaddr) */
    static constexpr uint32_t NV = KIND == Q4KV_Q8 ? 2 : 1;
    /* What a tile costs beside its passes: queries, first rows, gates and
     * outputs take 33 thousand cycles at 256 dims, where a pass takes 6. (At 4
     * passes instead of 7 the runs of short tiles are the last: 3 chunks of 701
     * tokens beside 40 decode tokens 545 us, now 462; 2048 tokens 236, 209; but
     * 8 requests of 48 columns 85, 90.) Cuts stay as far from a tile's ends, and
     * a run is as long: a short tile does not follow another one in it (two of
     * 30 tokens 38.1 us, now 23.6). */
    static constexpr uint32_t START = PT * (1 + HD / 42);
    typedef Share<COLS, START, START, START, 12 * PT, NTHR> Runs;
};

typedef uint32_t u4a_t __attribute__((ext_vector_type(4), aligned(2)));

template <int KIND, int HD> __global__ __launch_bounds__(512, 2) void paged_tiles_k(PagedArgs a) {
    using G = Geo<KIND, HD>;
    constexpr uint32_t NB = G::NB, PT = G::PT, NT = G::NT, KG = G::KG, KS = G::KS, VS = G::VS;
    constexpr uint32_t TD = HD / 16; /* output tiles of 16 dims */
    constexpr uint32_t NR = KIND == Q4KV_Q8 ? 1 : 2; /* rows of a pass that a thread loads pieces of */
    __shared__ __attribute__((aligned(16))) uint8_t s_k[2][PT * KS];
    __shared__ __attribute__((aligned(16))) uint8_t s_v[2][G::NV][PT * VS];
    /* K block scales, in the order the score stages read them: [tile pair]
     * [block][k-group][tile][position], 16 bytes per lane and stage */
    __shared__ __attribute__((aligned(16))) uint16_t s_ks[KIND == Q4KV_Q8 ? 2 : 1][KIND == Q4KV_Q8 ? NB * PT : 8];
    /* 1 + the last pass (mod 2^16) with a V value that is not finite, with a V
     * scale that VScale divides for, and with a position on no page: what
     * they lead to is right, if not needed, at any pass */
    __shared__ __attribute__((aligned(8))) uint16_t s_flag[2][4];
    __shared__ uint32_t s_nan[PT * NB]; /* a pass's values that are not finite, one bit each */
    __shared__ uint8_t s_none[2][PT];   /* positions on no page */
    __shared__ typename G::Runs::Lds lds;

    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = uni(tid >> 6);
    const uint32_t c = lane & 15u, jg = lane >> 4;
    const uint32_t hd = a.hd, nb = hd / 32u;
    Cut *const cuts = (Cut *)a.part;
    float *const parts = a.part + gridDim.x * (sizeof(Cut) / 4u);
    const size_t slot_b = (size_t)a.n_kvh * a.rowb;

    typename G::Runs run;
    const bool any = run.find(a, lds);
    Cut cut = {};
    while (any) {
        const Req &r = run.req;
        const uint32_t seq = run.seq, kh = run.kh, gqa = a.gqa;
        const uint32_t lc = wave * 16u + c, col = run.tile * COLS + lc;
        const uint32_t n_col = min(COLS, run.tiles.cols - run.tile * COLS);
        const bool live = lc < n_col, wave_live = wave * 16u < n_col;
        const uint32_t t = live ? col / gqa : 0u, h = live ? col - t * gqa : 0u;
        const uint32_t n_c = live ? seen_by(r, t) : 0u;
        const uint32_t n_all = uni(seen_by(r, (run.tile * COLS + n_col - 1u) / gqa));
        const uint32_t n_min = uni(seen_by(r, run.tile * COLS / gqa));
        uint32_t p0, p1;
        bool begins, ends;
        run.piece(a, (n_all + PT - 1u) / PT, p0, p1, begins, ends);
        const int32_t *const trow = a.table + (size_t)seq * a.stride;
        const uint8_t *const kb = a.kp + (size_t)kh * a.rowb, *const vb = a.vp + (size_t)kh * a.rowb;
        if (tid < 8u) s_flag[tid >> 2][tid & 3u] = 0u;
        VScale vq;

        /* ---- this thread's share of a pass's rows. q8_0: threads 0-255 one
         * block of K, 256-511 one of V; 16 rows x 4 blocks per wave ---- */
        const bool late = wave >= NWAVE / 2u, is_v = late;
        const uint32_t u = tid & 255u;
        const uint32_t bp = (u & 15u) + 16u * (u / (16u * NB)), bb = (u >> 4) % NB;
        auto row_of = [&](uint32_t pass, uint32_t i) {
            return min(pass * PT + (KIND == Q4KV_Q8 ? bp : (tid + NTHR * i) / (HD / 8u)), n_all - 1u);
        };
        int32_t number[NR];
        auto look = [&](uint32_t pass) {
#pragma unroll
            for (uint32_t i = 0; i < NR; i++) number[i] = ldg(trow + q4kv_page_of(a.page, row_of(pass, i)));
        };
        u4_t r0, r1;
        uint16_t rs;
        u4_t rk[NR], rv[NR];
        bool none[NR]; /* no page: the rows read are slot 0's */
        auto load = [&](uint32_t pass) {
#pragma unroll
            for (uint32_t i = 0; i < NR; i++) {
                const uint32_t p = row_of(pass, i);
                none[i] = (uint32_t)number[i] >= a.n_pages;
                const uint32_t slot = none[i] ? 0u : (uint32_t)number[i] * a.page.d + (p - q4kv_page_of(a.page, p) * a.page.d);
                const size_t at = (size_t)slot * slot_b;
                if constexpr (KIND == Q4KV_Q8) {
                    const uint8_t *src = (is_v ? vb : kb) + at + 34u * min(bb, nb - 1u);
                    rs = ldg((const uint16_t *)src);
                    r0 = *(const GLOBAL u4a_t *)(src + 2);
                    r1 = *(const GLOBAL u4a_t *)(src + 18);
                } else {
                    const uint32_t pc = min((tid + NTHR * i) % (HD / 8u), hd / 8u - 1u);
                    rk[i] = ldg((const u4_t *)(kb + at) + pc);
                    rv[i] = ldg((const u4_t *)(vb + at) + pc);
                }
            }
            look(pass + 1u);
        };
        auto partly = [&](uint32_t pass) { return (pass + 1u) * PT > n_min; }; /* some column does not see all of it */
        auto store = [&](uint32_t pass) {
            const uint32_t buf = pass & 1u;
            const bool masked = partly(pass);
            const uint16_t tag = (uint16_t)(pass + 1u);
            if constexpr (KIND == Q4KV_Q8) {
                const uint32_t d[8] = {r0[0], r0[1], r0[2], r0[3], r1[0], r1[1], r1[2], r1[3]};
                if (!is_v) {
                    uint8_t *dst = s_k[buf] + bp * KS + 64u * bb;
#pragma unroll
                    for (uint32_t k = 0; k < 4u; k++) {
                        h2_t x[4];
                        biased_h4(d[2u * k], x[0], x[1]);
                        biased_h4(d[2u * k + 1u], x[2], x[3]);
                        u4_t w;
#pragma unroll
                        for (uint32_t i = 0; i < 4u; i++) w[i] = __builtin_bit_cast(uint32_t, x[i] - (h2_t)((_Float16)1152.f));
                        *(u4_t *)(dst + 16u * k) = w;
                    }
                    s_ks[buf][(((bp >> 5) * NB + bb) * 4u + ((bp >> 2) & 3u)) * 8u + ((bp >> 4) & 1u) * 4u + (bp & 3u)] = rs;
                    if (bb == 0u) {
                        s_none[buf][bp] = none[0];
                        if (none[0]) s_flag[buf][2] = tag;
                    }
                } else {
                    const uint16_t sb = none[0] ? (uint16_t)0u : rs;
                    const h2_t vs = (h2_t)(__builtin_bit_cast(_Float16, sb));
#pragma unroll
                    for (uint32_t k = 0; k < 4u; k++) {
                        h2_t x[4];
                        biased_h4(d[2u * k], x[0], x[1]);
                        biased_h4(d[2u * k + 1u], x[2], x[3]);
                        u4_t wh, wl;
#pragma unroll
                        for (uint32_t i = 0; i < 4u; i++) {
                            /* v, exact; its product with the scale rounded once,
                             * and what the rounding left */
                            const h2_t f = vq.value(x[i]);
                            const h2_t hi = f * vs;
                            wh[i] = __builtin_bit_cast(uint32_t, hi);
                            wl[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(f, vs, -hi));
                        }
                        const uint32_t at = vaddr<VS>(bp, 4u * bb + k);
                        *(u4_t *)(s_v[buf][0] + at) = wh;
                        *(u4_t *)(s_v[buf][G::NV - 1u] + at) = wl;
                    }
                    if (masked && (sb & 0x7C00u) == 0x7C00u) s_flag[buf][0] = tag;
                    if (q4kv_big_scale(sb)) s_flag[buf][1] = tag;
                }
            } else {
#pragma unroll
                for (uint32_t i = 0; i < NR; i++) {
                    const uint32_t e = tid + NTHR * i, pc = e % (HD / 8u), p = e / (HD / 8u);
                    *(u4_t *)(s_k[buf] + p * KS + 16u * pc) = rk[i];
                    const u4_t v = none[i] ? (u4_t){0u, 0u, 0u, 0u} : rv[i];
                    *(u4_t *)(s_v[buf][0] + vaddr<VS>(p, pc)) = v;
                    if (pc == 0u) {
                        s_none[buf][p] = none[i];
                        if (none[i]) s_flag[buf][2] = tag;
                    }
                    if (masked) {
                        bool bad = false;
#pragma unroll
                        for (uint32_t k = 0; k < 4u; k++)
                            bad = bad || (v[k] & 0x7C00u) == 0x7C00u || (v[k] & 0x7C000000u) == 0x7C000000u;
                        if (bad) s_flag[buf][0] = tag;
                    }
                }
            }
        };
        if (p0 < p1) {
            look(p0);
            load(p0);
        }

        /* ---- this wave's Q^T operands: column c, dims 32 b + 8 jg .. + 7, q x
         * scale / ln 2 divided by the column's power of two, in two parts ---- */
        h8_t qh[NB], ql[NB];
        float qmul;
        {
            const float *qr = a.q + ((size_t)(r.t0 + t) * a.n_head + kh * gqa + h) * hd + 8u * jg;
            float x[NB][8], am = 0.f;
#pragma unroll
            for (uint32_t b = 0; b < NB; b++)
#pragma unroll
                for (uint32_t i = 0; i < 8u; i++) x[b][i] = ldg(qr + 32u * min(b, nb - 1u) + i);
#pragma unroll
            for (uint32_t b = 0; b < NB; b++)
#pragma unroll
                for (uint32_t i = 0; i < 8u; i++) {
                    x[b][i] = live && b < nb ? x[b][i] : 0.f;
                    am = fmaxf(am, fabsf(x[b][i]));
                }
            am = fmaxf(am, __shfl_xor(am, 16));
            am = fmaxf(am, __shfl_xor(am, 32));
            am *= fabsf(a.scale_log2);
            const int e = (am > 0.f && am <= 3.4e38f) ? __builtin_amdgcn_frexp_expf(am) : 0;
            qmul = __builtin_ldexpf(1.f, e);
            const float qs = __builtin_ldexpf(a.scale_log2, -e);
#pragma unroll
            for (uint32_t b = 0; b < NB; b++) {
                u4_t wh, wl;
#pragma unroll
                for (uint32_t i = 0; i < 4u; i++) {
                    const float y0 = x[b][2u * i] * qs, y1 = x[b][2u * i + 1u] * qs;
                    wh[i] = pk(y0, y1);
                    wl[i] = pk(y0 - h2lo(wh[i]), y1 - h2hi(wh[i]));
                }
                qh[b] = __builtin_bit_cast(h8_t, wh);
                ql[b] = __builtin_bit_cast(h8_t, wl);
            }
        }

        float m_run = -INFINITY, l_run = 0.f;
        uint64_t nan_out = 0u; /* bit 4 T + i: acc[T][i] sums a value that is not finite */
        f4_t acc[TD];
#pragma unroll
        for (uint32_t T = 0; T < TD; T++) acc[T] = (f4_t){0.f, 0.f, 0.f, 0.f};

        __syncthreads(); /* s_flag cleared */
        if (p0 < p1) {
            store(p0);
            if (p0 + 1u < p1) load(p0 + 1u);
        }
        __syncthreads();

        for (uint32_t pass = p0; pass < p1; pass++) {
            const uint32_t buf = pass & 1u, base = pass * PT;
            const bool masked = partly(pass);
            const u2_t flag_at = *(const u2_t *)s_flag[buf];
            /* ---- what the rows of this pass ask of the whole workgroup ---- */
            const uint32_t flag = uni(flag_at[0]);
            const bool bad = masked && (flag & 0xFFFFu) == ((pass + 1u) & 0xFFFFu);
            const bool grow = KIND == Q4KV_Q8 && !vq.big() && flag >> 16 == ((pass + 1u) & 0xFFFFu);
            if (bad || grow) { /* the whole workgroup */
                __syncthreads();
                if (grow) {
                    /* V over 128 from this pass on: its rows once more */
                    vq.divide();
#pragma unroll
                    for (uint32_t T = 0; T < TD; T++) acc[T] *= VSCALE_STEP;
#pragma unroll 1
                    for (uint32_t i = tid; i < PT * (HD / 8u); i += NTHR) {
                        const uint32_t p = i / (HD / 8u), pc = i % (HD / 8u), b = min(pc / 4u, nb - 1u);
                        const uint32_t q = min(base + p, n_all - 1u), pg = q4kv_page_of(a.page, q);
                        const int32_t num = ldg(trow + pg);
                        const bool no = (uint32_t)num >= a.n_pages;
                        const uint32_t slot = no ? 0u : (uint32_t)num * a.page.d + (q - pg * a.page.d);
                        const uint8_t *blk = vb + (size_t)slot * slot_b + 34u * b;
                        const uint16_t sb = no ? (uint16_t)0u : ldg((const uint16_t *)blk);
                        const h2_t vs = (h2_t)(__builtin_bit_cast(_Float16, sb));
                        u4_t wh, wl;
#pragma unroll
                        for (uint32_t e = 0; e < 4u; e++) {
                            const uint32_t w = ldg((const uint16_t *)(blk + 2u + 8u * (pc & 3u)) + e) ^ 0x8080u;
                            const h2_t f = vq.value(__builtin_bit_cast(h2_t, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)));
                            const h2_t hi = f * vs;
                            wh[e] = __builtin_bit_cast(uint32_t, hi);
                            wl[e] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(f, vs, -hi));
                        }
                        *(u4_t *)(s_v[buf][0] + vaddr<VS>(p, pc)) = wh;
                        *(u4_t *)(s_v[buf][G::NV - 1u] + vaddr<VS>(p, pc)) = wl;
                    }
                    __syncthreads();
                }
                if (bad) {
                    /* Rows that not every column sees hold inf or NaN, which a
                     * zero weight would turn into NaN. They are taken out of
                     * the tile, and the outputs of the columns that do see
                     * them become NaN at the end. */
                    for (uint32_t i = tid; i < PT * NB; i += NTHR) s_nan[i] = 0u;
                    __syncthreads();
                    for (uint32_t i = tid; i < PT * (HD / 8u); i += NTHR) {
                        const uint32_t p = i / (HD / 8u), pc = i % (HD / 8u), at = vaddr<VS>(p, pc);
                        uint32_t bits = 0u;
                        for (uint32_t e = 0; e < 8u; e++) {
                            uint16_t *v = (uint16_t *)(s_v[buf][0] + at) + e;
                            if ((*v & 0x7C00u) != 0x7C00u) continue;
                            bits |= 1u << e;
                            *v = 0u;
                            if (G::NV == 2) ((uint16_t *)(s_v[buf][G::NV - 1u] + at))[e] = 0u;
                        }
                        if (bits) atomicOr(&s_nan[p * NB + pc / 4u], bits << (8u * (pc & 3u)));
                    }
                    __syncthreads();
                    for (uint32_t p = 0; p < PT && base + p < n_c; p++)
                        for (uint32_t b = 0; b < NB; b++) {
                            const uint32_t w = s_nan[p * NB + b] >> (4u * jg);
                            nan_out |= ((uint64_t)(w & 15u) | (uint64_t)((w >> 16) & 15u) << 4) << (8u * b);
                        }
                }
                __syncthreads();
            }
            /* Waves 4-7 convert the next pass's rows at its start, waves 0-3 at
             * its end: the two waves of a SIMD are then in different stages, one
             * with products while the other has vector work. */
            if (late && pass + 1u < p1) {
                store(pass + 1u);
                if (pass + 2u < p1) load(pass + 2u);
            }
            /* ---- scores: tile tt holds positions base + 16 tt + 4 jg + i of
             * column c. Eight stages of two tiles and one block; the operands
             * of the stage after next are in flight, and the scales are
             * applied one stage late ---- */
            f4_t S[NT], Sl[KIND == Q4KV_Q8 ? 1 : NT];
            h8_t VA[8][2][G::NV];
            const uint32_t at0 = vaddr<VS>(4u * jg + (c >> 2), (c >> 1) & 1u) + 8u * (c & 1u);
            auto vfetch = [&](uint32_t st) {
                const uint32_t kg = st / (TD / 2u), T0 = 2u * (st % (TD / 2u));
#pragma unroll
                for (uint32_t k = 0; k < 2u; k++) {
                    /* vaddr(row, 2 T + ..): T enters by the window's xor */
                    const uint32_t at = (at0 ^ ((T0 + k) << 5)) + kg * 32u * VS;
#pragma unroll
                    for (uint32_t v = 0; v < G::NV; v++) {
                        const s4_t a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LOCAL s4_t *)(s_v[buf][v] + at));
                        const s4_t a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LOCAL s4_t *)(s_v[buf][v] + at + 16u * VS));
                        VA[st][k][v] = __builtin_bit_cast(h8_t, __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7));
                    }
                }
            };
            float mx = -INFINITY;
            const bool gone = (uni(flag_at[1]) & 0xFFFFu) == ((pass + 1u) & 0xFFFFu);
            if (wave_live) {
#pragma unroll
                for (uint32_t tt = 0; tt < NT; tt++) S[tt] = (f4_t){0.f, 0.f, 0.f, 0.f};
                if constexpr (KIND != Q4KV_Q8) {
#pragma unroll
                    for (uint32_t tt = 0; tt < NT; tt++) Sl[tt] = (f4_t){0.f, 0.f, 0.f, 0.f};
                }
                const uint8_t *kr = s_k[buf] + c * KS + 16u * jg;
                const uint16_t *ksr = s_ks[KIND == Q4KV_Q8 ? buf : 0u] + 8u * jg;
                h8_t A[8][2], ks[8];
                auto fetch = [&](uint32_t st) {
                    const uint32_t b = st % NB, tp = st / NB;
#pragma unroll
                    for (uint32_t k = 0; k < 2u; k++)
                        A[st][k] = *(const h8_t *)(kr + (2u * tp + k) * 16u * KS + 64u * b);
                    if constexpr (KIND == Q4KV_Q8) ks[st] = *(const h8_t *)(ksr + st * 32u);
                };
                f4_t C[8][2];
                auto scale = [&](uint32_t st) {
                    const uint32_t tp = st / NB;
#pragma unroll
                    for (uint32_t k = 0; k < 2u; k++)
#pragma unroll
                        for (uint32_t i = 0; i < 4u; i++)
                            S[2u * tp + k][i] = fmaf((float)ks[st][4u * k + i], C[st][k][i], S[2u * tp + k][i]);
                };
                fetch(0u);
                fetch(1u);
                __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (uint32_t st = 0; st < 8u; st++) {
                    const uint32_t b = st % NB, tp = st / NB;
                    if (st + 2u < 8u) fetch(st + 2u);
                    if constexpr (KIND == Q4KV_Q8) {
#pragma unroll
                        for (uint32_t k = 0; k < 2u; k++)
                            C[st][k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A[st][k], ql[b], (f4_t){0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
                        for (uint32_t k = 0; k < 2u; k++)
                            C[st][k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A[st][k], qh[b], C[st][k], 0, 0, 0);
                        if (st) scale(st - 1u);
                    } else {
#pragma unroll
                        for (uint32_t k = 0; k < 2u; k++)
                            Sl[2u * tp + k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A[st][k], ql[b], Sl[2u * tp + k], 0, 0, 0);
#pragma unroll
                        for (uint32_t k = 0; k < 2u; k++)
                            S[2u * tp + k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A[st][k], qh[b], S[2u * tp + k], 0, 0, 0);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                if constexpr (KIND == Q4KV_Q8) {
                    scale(7u);
                } else {
                    /* the small parts summed apart: half the roundings at the sum's size */
#pragma unroll
                    for (uint32_t tt = 0; tt < NT; tt++) S[tt] += Sl[tt];
                }
                __builtin_amdgcn_s_setprio(0);
                vfetch(0u); /* ahead of the softmax */
                if (masked || gone) {
#pragma unroll
                    for (uint32_t tt = 0; tt < NT; tt++)
#pragma unroll
                        for (uint32_t i = 0; i < 4u; i++) {
                            const uint32_t p = 16u * tt + 4u * jg + i;
                            S[tt][i] = base + p < n_c && !(gone && s_none[buf][p]) ? S[tt][i] : -INFINITY;
                        }
                }
#pragma unroll
                for (uint32_t tt = 0; tt < NT; tt++) mx = max3(max3(mx, S[tt][0], S[tt][1]), S[tt][2], S[tt][3]);
                mx *= qmul;
            }
            /* this lane's positions only: the column's maximum is formed when a
             * lane passes the limit */
            const bool up = __ballot(mx > m_run + RAISE) != 0u;
            if (up) {
                const float mn = max2(m_run, col_max(mx));
                const float alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run - mn);
                m_run = mn;
                l_run *= alpha;
#pragma unroll
                for (uint32_t T = 0; T < TD; T++) acc[T] *= alpha;
            }
            if (wave_live) {
                const float ms = m_run == -INFINITY ? 0.f : m_run;
#pragma unroll
                for (uint32_t tt = 0; tt < NT; tt++) {
#pragma unroll
                    for (uint32_t i = 0; i < 4u; i++) S[tt][i] = __builtin_amdgcn_exp2f(fmaf(S[tt][i], qmul, -ms));
                    l_run += (S[tt][0] + S[tt][1]) + (S[tt][2] + S[tt][3]);
                }
                /* ---- O^T += V^T P^T ---- */
                h8_t Ph[KG], Pl[KG];
#pragma unroll
                for (uint32_t kg = 0; kg < KG; kg++) {
                    u4_t wh, wl;
#pragma unroll
                    for (uint32_t i = 0; i < 4u; i++) {
                        const f4_t &P = S[2u * kg + (i >> 1)];
                        const float x0 = P[2u * (i & 1u)], x1 = P[2u * (i & 1u) + 1u];
                        wh[i] = pk(x0, x1);
                        wl[i] = pk(x0 - h2lo(wh[i]), x1 - h2hi(wh[i]));
                    }
                    Ph[kg] = __builtin_bit_cast(h8_t, wh);
                    Pl[kg] = __builtin_bit_cast(h8_t, wl);
                }
                __builtin_amdgcn_s_setprio(1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (uint32_t st = 0; st < 8u; st++) {
                    const uint32_t kg = st / (TD / 2u), T0 = 2u * (st % (TD / 2u));
                    if (st + 1u < 8u) vfetch(st + 1u);
                    if constexpr (G::NV == 2) {
#pragma unroll
                        for (uint32_t k = 0; k < 2u; k++)
                            acc[T0 + k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(VA[st][k][1], Ph[kg], acc[T0 + k], 0, 0, 0);
                    }
#pragma unroll
                    for (uint32_t k = 0; k < 2u; k++)
                        acc[T0 + k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(VA[st][k][0], Pl[kg], acc[T0 + k], 0, 0, 0);
#pragma unroll
                    for (uint32_t k = 0; k < 2u; k++)
                        acc[T0 + k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(VA[st][k][0], Ph[kg], acc[T0 + k], 0, 0, 0);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            __builtin_amdgcn_s_setprio(0);
            if (!late && pass + 1u < p1) {
                store(pass + 1u);
                if (pass + 2u < p1) load(pass + 2u);
            }
            __syncthreads();
        }

        /* ---- the columns' rows: finished, or the run's partial ---- */
        const float l = col_sum(l_run);
        if (live) {
            if (nan_out) {
#pragma unroll
                for (uint32_t T = 0; T < TD; T++)
#pragma unroll
                    for (uint32_t i = 0; i < 4u; i++)
                        if ((nan_out >> (4u * T + i)) & 1u) acc[T][i] = __builtin_nanf("");
            }
            const float vmul = vq.undo();
            if (!(begins && ends)) {
                float *pb = parts + ((size_t)(2u * (run.g * a.n_kvh + kh) + (begins ? 1u : 0u)) * COLS + lc) * (HD + PAGED_PHEAD);
                if (jg == 0u) stg((f2_t *)pb, (f2_t){m_run, l});
#pragma unroll
                for (uint32_t T = 0; T < TD; T++) stg((f4_t *)(pb + PAGED_PHEAD + 16u * T + 4u * jg), acc[T] * vmul);
            } else {
                const float inv = l != 0.f ? vmul / l : 0.f;
                const size_t ro = ((size_t)(r.t0 + t) * a.n_head + kh * gqa + h) * hd + 4u * jg;
                const bool al = (((uintptr_t)a.out | (uintptr_t)a.gate) & 15u) == 0u;
                if (al && hd == HD) {
                    /* four gates a trip: one after the other they took half of a
                     * short tile's time, all at once the loop's registers */
#pragma unroll
                    for (uint32_t T0 = 0; T0 < TD; T0 += 4u) {
                        f4_t g[4];
                        if (a.gate) {
#pragma unroll
                            for (uint32_t k = 0; k < 4u; k++) g[k] = ldg((const f4_t *)(a.gate + ro + 16u * (T0 + k)));
                        }
#pragma unroll
                        for (uint32_t k = 0; k < 4u; k++) {
                            f4_t o = acc[T0 + k] * inv;
                            if (a.gate) {
#pragma unroll
                                for (uint32_t i = 0; i < 4u; i++) o[i] *= q4kv_sigmoid(g[k][i]);
                            }
                            stg((f4_t *)(a.out + ro + 16u * (T0 + k)), o);
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                } else {
#pragma unroll
                    for (uint32_t T = 0; T < TD; T++) {
                        if (16u * T >= hd) continue;
#pragma unroll
                        for (uint32_t i = 0; i < 4u; i++) {
                            float o = acc[T][i] * inv;
                            if (a.gate) o *= q4kv_sigmoid(ldg(a.gate + ro + 16u * T + i));
                            stg(a.out + ro + 16u * T + i, o);
                        }
                    }
                }
            }
        }
        if (begins && !ends) cut = Cut{run.pieces(a), run.g, kh, run.tile, r.t0, run.tiles.cols, {}};
        run.advance(a);
        if (run.u >= run.end) break;
        __syncthreads();
    }
    if (tid == 0u) {
        uint32_t *const cw = (uint32_t *)(cuts + blockIdx.x);
        stg((u4_t *)cw, (u4_t){cut.pieces, cut.g, cut.kh, cut.tile});
        stg((u2_t *)(cw + 4), (u2_t){cut.t0, cut.cols});
    }
}

template <int KIND, int HD> bool launch(PagedArgs a) {
    a.unit = q4kv_paged_unit(a, COLS, Geo<KIND, HD>::START);
    constexpr uint32_t N_CU = 256;
    static_assert(paged_part_floats(N_CU, COLS, HD) <= Q4KV_TILE_FLOATS, "the scratch holds the partials");
    a.runs = q4kv_paged_runs(N_CU, a.n_kvh);
    const uint32_t grid = a.runs * a.n_kvh;
    const bool prof = q4kv_prof_open();
    paged_tiles_k<KIND, HD><<<grid, NTHR, 0, q4kv_stream>>>(a);
    q4kv_prof_close(prof);
    paged_merge_k<HD, COLS><<<dim3(grid, 16), 256, 0, q4kv_stream>>>(a);
    return q4kv_launch_ok("paged attention, tiles");
}

} // namespace

bool q4kv_paged_tiles_launch(int kind, const PagedArgs &a) {
    if (kind == Q4KV_Q8)
        return a.hd <= 64u ? launch<Q4KV_Q8, 64>(a) : a.hd <= 128u ? launch<Q4KV_Q8, 128>(a) : launch<Q4KV_Q8, 256>(a);
    return a.hd <= 64u ? launch<Q4KV_F16, 64>(a) : a.hd <= 128u ? launch<Q4KV_F16, 128>(a) : launch<Q4KV_F16, 256>(a);
}
