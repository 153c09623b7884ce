/*
 * q4kv_paged_attn.hip -- causal attention of a ragged batch's new tokens over
 * a paged cache.
 */
#include <hip/hip_runtime.h>
#include <hip/hip_fp16.h>
#include <math.h>
#include <algorithm>

#include "q4kv_paged_attn.h"

namespace {

/* ---- any shape: a workgroup per (token, query head) ----
 * Each wave takes 64 positions at a time: a lane forms the score of one, then
 * the lanes share the dims of the weighted sum. Plain fp32 arithmetic, one
 * pass with a running maximum; for shapes that the matrix kernels do not take
 * (head dims off 32, unaligned pools). Bound by its scalar row loads. */

template <int KIND> __device__ inline float cache_value(const uint8_t *row, uint32_t d) {
    if (KIND == Q4KV_F32) return ldg((const float *)row + d);
    if (KIND == Q4KV_F16) return __half2float(__ushort_as_half(ldg((const uint16_t *)row + d)));
    const uint8_t *blk = row + 34u * (d >> 5);
    return (float)(int8_t)ldg(blk + 2u + (d & 31u)) * __half2float(__ushort_as_half(ldg((const uint16_t *)blk)));
}

template <int KIND> __global__ __launch_bounds__(256) void paged_any_k(PagedArgs a) {
    __shared__ float s_q[256], s_acc[4][256], s_m[4], s_l[4];
    const uint32_t t = blockIdx.x / a.n_head, h = blockIdx.x - t * a.n_head, kh = h / a.gqa;
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    /* the last request that starts at or before token t */
    uint32_t lo = 0u, hi = a.n_seq;
    while (hi - lo > 1u) {
        const uint32_t mid = (lo + hi) / 2u;
        if (ldg(a.q_start + mid) <= (int32_t)t)
            lo = mid;
        else
            hi = mid;
    }
    const Req r = req_of(a, lo);
    if (t < r.t0 || t - r.t0 >= r.n_q) return; /* nobody's row */
    const uint32_t n = seen_by(r, t - r.t0);
    const size_t ro = ((size_t)t * a.n_head + h) * a.hd;
    if (threadIdx.x < a.hd) s_q[threadIdx.x] = ldg(a.q + ro + threadIdx.x) * a.scale_log2;
    __syncthreads();
    const size_t slot_b = (size_t)a.n_kvh * a.rowb;
    const uint8_t *const kb = a.kp + (size_t)kh * a.rowb, *const vb = a.vp + (size_t)kh * a.rowb;
    float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t p0 = 64u * wave; p0 < n; p0 += 256u) {
        const uint32_t p = p0 + lane;
        const int32_t slot = p < n ? slot_at(a, lo, p) : -1;
        float s = -INFINITY;
        if (slot >= 0) {
            const uint8_t *row = kb + (size_t)slot * slot_b;
            s = 0.f;
            for (uint32_t d = 0; d < a.hd; d++) s = fmaf(s_q[d], cache_value<KIND>(row, d), s);
        }
        /* a score that is not a number makes the row one, as it does l */
        float mx = s == s ? s : -INFINITY;
        for (uint32_t d = 1; d < 64u; d *= 2u) mx = fmaxf(mx, __shfl_xor(mx, d));
        const float mn = fmaxf(m, mx), base = mn == -INFINITY ? 0.f : mn;
        const float f = m == -INFINITY ? 0.f : exp2f(m - mn);
        const float w = slot >= 0 ? exp2f(s - base) : 0.f;
        m = mn;
        l *= f;
#pragma unroll
        for (uint32_t i = 0; i < 4u; i++) acc[i] *= f;
        l += w;
        for (uint64_t todo = __ballot(slot >= 0); todo; todo &= todo - 1u) {
            const int j = __builtin_ctzll(todo);
            const uint8_t *row = vb + (size_t)__shfl(slot, j) * slot_b;
            const float wj = __shfl(w, j);
#pragma unroll
            for (uint32_t i = 0; i < 4u; i++)
                if (lane + 64u * i < a.hd) acc[i] = fmaf(wj, cache_value<KIND>(row, lane + 64u * i), acc[i]);
        }
    }
    for (uint32_t d = 1; d < 64u; d *= 2u) l += __shfl_xor(l, d);
    if (lane == 0u) {
        s_m[wave] = m;
        s_l[wave] = l;
    }
#pragma unroll
    for (uint32_t i = 0; i < 4u; i++) s_acc[wave][lane + 64u * i] = acc[i];
    __syncthreads();
    if (threadIdx.x >= a.hd) return;
    const float M = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
    float L = 0.f, o = 0.f;
    for (uint32_t w = 0; w < 4u; w++) {
        if (s_l[w] == 0.f) continue;
        const float f = s_m[w] == -INFINITY ? 1.f : exp2f(s_m[w] - M);
        L = fmaf(f, s_l[w], L);
        o = fmaf(f, s_acc[w][threadIdx.x], o);
    }
    o = L != 0.f ? o / L : 0.f;
    if (a.gate) o *= q4kv_sigmoid(ldg(a.gate + ro + threadIdx.x));
    stg(a.out + ro + threadIdx.x, o);
}

/* Columns (new tokens x query heads of a KV head) past which a request runs
 * on the tiles. None does where those of all KV heads of a launch are no more
 * than tiles_from: a few tiles leave the chip idle, each takes 25 us beside
 * its passes, and decode tokens beside them need a launch of their own. (us,
 * rows / tiles. 256 dims, q8_0, one request of 10 thousand positions: 256
 * columns 49 / 87, 1024 83 / 95, 2048 142 / 92; 20 tokens and 10 decodes of 2
 * thousand positions 36 / 82, of 16 thousand 108 / 155. 128 dims, f16: 512
 * columns 33 / 39, 1024 45 / 44, 2048 76 / 46; 20 tokens and 4 decodes 32 / 48
 * and 118 / 110, 10 decodes 42 / 57 and 209 / 185.) */
constexpr uint32_t TILE_COLS = 32;
static inline uint32_t tiles_from(uint32_t hd) { return hd > 128u ? 1024u : 768u; }

template <int KIND> bool any_launch(const PagedArgs &a) {
    paged_any_k<KIND><<<a.n_tok * a.n_head, 256, 0, q4kv_stream>>>(a);
    return q4kv_launch_ok("paged attention");
}

} // namespace

extern "C" bool q4_hip_qsa_paged_attend(const float *q, const void *kpool, const void *vpool,
                                        const float *gate, float *out, const q4kv_paged_batch *b,
                                        uint32_t n_tok, uint32_t max_q, uint32_t n_head,
                                        uint32_t n_kvh, uint32_t hd, float scale, int kind) {
    Q4KV_FLUSH_OR_FAIL();
    if (!q4kv_ok || !q || !kpool || !vpool || !out || !q4kv_batch_ok(b) || !b->q_start) return false;
    if (out == q || out == gate) return false; /* a tile's columns are read by several workgroups */
    if (!n_tok || !max_q || !n_head || !n_kvh || n_head % n_kvh || !hd || hd > 256u) return false;
    if (kind < Q4KV_F32 || kind > Q4KV_Q8 || (kind == Q4KV_Q8 && hd % 32u)) return false;
    if ((uint64_t)n_tok * n_head > 0x7fffffffull) return false;
    if (((uintptr_t)kpool | (uintptr_t)vpool) & (kind == Q4KV_F32 ? 3u : 1u)) return false;
    (void)hipGetLastError();
    PagedArgs a = {};
    a.q = q;
    a.gate = gate;
    a.kp = (const uint8_t *)kpool;
    a.vp = (const uint8_t *)vpool;
    a.out = out;
    a.table = b->table;
    a.q_start = b->q_start;
    a.kv_len = b->kv_len;
    a.n_seq = b->n_seq;
    a.stride = b->table_stride;
    a.n_pages = b->n_pages;
    a.n_tok = n_tok;
    a.n_head = n_head;
    a.n_kvh = n_kvh;
    a.gqa = n_head / n_kvh;
    a.hd = hd;
    a.rowb = kind == Q4KV_Q8 ? hd / 32u * 34u : hd * (kind == Q4KV_F16 ? 2u : 4u);
    a.page = q4kv_page_div(b->page);
    a.scale_log2 = scale * 1.44269504f;
    if (hd % 32u == 0u && n_kvh <= PAGED_KVH && (((uintptr_t)kpool | (uintptr_t)vpool) & 15u) == 0u) {
        if (!q4kv_part) {
            Q4KV_ERR("paged attention: no scratch");
            return false;
        }
        /* Few columns run on the rows kernel, many on the tiles (q8_0, f16).
         * Which requests are which is known on the device only; the host knows
         * when all of them are alike. */
        const uint64_t most = (uint64_t)max_q * a.gqa;
        const bool alike = b->n_seq == 1u || n_tok == (uint64_t)b->n_seq * max_q;
        const bool tiles = kind != Q4KV_F32 && q4kv_tile_part && most > TILE_COLS &&
                           (uint64_t)n_tok * n_head > tiles_from(hd);
        a.min_cols = 1u;
        a.max_cols = ~0u;
        if (tiles) {
            PagedArgs t = a;
            t.part = q4kv_tile_part;
            if (!alike) t.min_cols = (a.max_cols = TILE_COLS) + 1u;
            if (!q4kv_paged_tiles_launch(kind, t)) return false;
            if (alike) return true;
        }
        const bool wide = most > 16u && !tiles && q4kv_tile_part;
        a.part = wide ? q4kv_tile_part : q4kv_part;
        return q4kv_paged_rows_launch(kind, a, wide ? 32u : 16u);
    }
    if (kind == Q4KV_Q8) return any_launch<Q4KV_Q8>(a);
    if (kind == Q4KV_F16) return any_launch<Q4KV_F16>(a);
    return any_launch<Q4KV_F32>(a);
}
