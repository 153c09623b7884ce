/*
 * q4kv_paged.hip -- the paged cache around its attention: pages given back
 * and handed out, block tables and slot maps from the requests' lengths, rows
 * written to and read from slots, position lists as lists of slots.
 *
 * All of it is integer bookkeeping or a copy: the table calls are bound by
 * the latency of a launch and of a few dependent loads, the row calls by the
 * bytes they move.
 */
#include <hip/hip_runtime.h>
#include <algorithm>

#include "q4kv_paged.h"

namespace {

constexpr uint32_t SCAN_T = 1024; /* threads of a scan's workgroup */

__device__ inline int64_t shfl_up64(int64_t v, uint32_t d) {
    const int lo = __shfl_up((int)(uint32_t)v, d), hi = __shfl_up((int)(v >> 32), d);
    return ((int64_t)hi << 32) | (uint32_t)lo;
}

/* Inclusive prefix sums of two values over a workgroup of SCAN_T threads. */
__device__ inline void scan2(int64_t &a, int64_t &b, int64_t (*tot)[2]) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
#pragma unroll
    for (uint32_t d = 1; d < 64u; d *= 2u) {
        const int64_t x = shfl_up64(a, d), y = shfl_up64(b, d);
        if (lane >= d) {
            a += x;
            b += y;
        }
    }
    __syncthreads(); /* tot of the scan before is read */
    if (lane == 63u) {
        tot[wave][0] = a;
        tot[wave][1] = b;
    }
    __syncthreads();
    for (uint32_t w = 0; w < wave; w++) {
        a += tot[w][0];
        b += tot[w][1];
    }
}

__device__ inline int64_t clamp_count(int32_t n, uint32_t n_pages) {
    return n < 0 ? 0 : (uint32_t)n > n_pages ? (int64_t)n_pages : n;
}

/* ---- pages given back ---- */

struct ReleaseArgs {
    const int32_t *table, *lens, *rows;
    int32_t *free_pages;
    const int32_t *n_free;
    int32_t *left, *base;
    uint32_t stride, n, n_pages;
    PageDiv page;
};

__device__ inline uint32_t pages_of(const PageDiv &page, int64_t len) {
    return len <= 0 ? 0u : q4kv_page_of(page, (uint32_t)(len - 1)) + 1u;
}
/* the table row of request r and the pages that it holds */
__device__ inline uint32_t release_row(const ReleaseArgs &a, uint32_t r, int32_t &row) {
    row = a.rows ? ldg(a.rows + r) : (int32_t)r;
    return row < 0 ? 0u : min(pages_of(a.page, ldg(a.lens + row)), a.stride);
}

__global__ __launch_bounds__(SCAN_T) void release_scan_k(ReleaseArgs a) {
    __shared__ int64_t tot[SCAN_T / 64][2];
    const int64_t have = clamp_count(ldg(a.n_free), a.n_pages);
    int64_t before = have;
    for (uint32_t r0 = 0; r0 < a.n; r0 += SCAN_T) {
        const uint32_t r = r0 + threadIdx.x;
        int32_t row;
        const int64_t held = r < a.n ? release_row(a, r, row) : 0;
        int64_t upto = held, unused = 0;
        scan2(upto, unused, tot);
        if (r < a.n) stg(a.base + r, (int32_t)min(before + upto - held, (int64_t)a.n_pages));
        int64_t sum = 0;
        for (uint32_t w = 0; w < SCAN_T / 64u; w++) sum += tot[w][0];
        before += sum;
    }
    if (threadIdx.x == 0u) stg(a.left, (int32_t)min(before, (int64_t)a.n_pages));
}

/* a wave per request */
__global__ __launch_bounds__(256) void release_fill_k(ReleaseArgs a) {
    const uint32_t r = blockIdx.x * 4u + (threadIdx.x >> 6), lane = threadIdx.x & 63u;
    if (r >= a.n) return;
    int32_t row;
    const uint32_t held = release_row(a, r, row), at = (uint32_t)ldg(a.base + r);
    for (uint32_t j = lane; j < held && at + j < a.n_pages; j += 64u)
        stg(a.free_pages + at + j, ldg(a.table + (size_t)row * a.stride + j));
}

/* ---- tables and slots of a step ---- */

struct PlanArgs {
    const int32_t *ctx, *n_new, *free_pages;
    const int32_t *n_free;
    int32_t *table, *left, *q_start, *kv_len, *slot, *tok_seq, *tok_pos, *top;
    uint32_t n_seq, stride, n_pages, max_tok;
    PageDiv page;
};

/* A request's tokens, whether its lengths are sound (but for the tokens
 * before it), the pages that it holds and lacks. */
struct Ask {
    int64_t ctx, add;
    bool fits;
    uint32_t held, need;
};
__device__ inline Ask ask_of(const PlanArgs &a, uint32_t i) {
    Ask r;
    r.ctx = ldg(a.ctx + i);
    r.add = max(ldg(a.n_new + i), 0);
    r.fits = r.ctx >= 0 && r.ctx + r.add <= (int64_t)a.stride * a.page.d;
    r.held = r.fits ? pages_of(a.page, r.ctx) : 0u;
    r.need = r.fits ? pages_of(a.page, r.ctx + r.add) - r.held : 0u;
    return r;
}

__global__ __launch_bounds__(SCAN_T) void plan_scan_k(PlanArgs a) {
    __shared__ int64_t tot[SCAN_T / 64][2];
    __shared__ int64_t s_tok[SCAN_T / 64];
    __shared__ uint32_t s_taken, s_refused;
    const int64_t avail = clamp_count(ldg(a.n_free), a.n_pages);
    if (threadIdx.x == 0u) s_taken = s_refused = 0u;
    int64_t tok0 = 0, need0 = 0;
    for (uint32_t i0 = 0; i0 < a.n_seq; i0 += SCAN_T) {
        const uint32_t i = i0 + threadIdx.x;
        Ask q = {0, 0, true, 0u, 0u};
        if (i < a.n_seq) q = ask_of(a, i);
        /* tokens first: a request whose tokens end past max_tok asks for no page */
        int64_t tok = q.add, unused = 0;
        scan2(tok, unused, tot);
        tok += tok0;
        const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
        if (lane == 63u) s_tok[wave] = tok;
        if (tok > (int64_t)a.max_tok && q.add) {
            q.fits = false;
            q.need = 0u;
        }
        int64_t need = q.need;
        scan2(need, unused, tot);
        need += need0;
        int64_t sum = 0;
        for (uint32_t w = 0; w < SCAN_T / 64u; w++) sum += tot[w][0];
        if (i < a.n_seq) {
            const bool granted = q.fits && (q.need == 0u || need <= avail);
            stg(a.q_start + i, (int32_t)min(tok - q.add, (int64_t)a.max_tok));
            if (i + 1u == a.n_seq) stg(a.q_start + i + 1u, (int32_t)min(tok, (int64_t)a.max_tok));
            stg(a.kv_len + i, granted ? (int32_t)(q.ctx + q.add) : 0);
            /* one past the stack entry that is taken first */
            stg(a.top + i, (int32_t)(avail - (need - q.need)));
            if (granted && q.need) atomicMax(&s_taken, (uint32_t)need);
            if (!granted) atomicAdd(&s_refused, 1u);
        }
        tok0 = s_tok[SCAN_T / 64u - 1u];
        need0 += sum;
        __syncthreads(); /* s_tok is read */
    }
    __syncthreads();
    if (threadIdx.x == 0u) {
        stg(a.left, (int32_t)(avail - s_taken));
        stg(a.left + 1, (int32_t)s_refused);
    }
}

/* A wave per request (grid.y of them share its tokens and pages), then the
 * tokens behind the last request. */
__global__ __launch_bounds__(256) void plan_fill_k(PlanArgs a) {
    const uint32_t lane = (threadIdx.x & 63u) + 64u * blockIdx.y, step = 64u * gridDim.y;
    const uint32_t i = blockIdx.x * 4u + (threadIdx.x >> 6);
    if (i > a.n_seq) return;
    if (i == a.n_seq) {
        for (uint32_t t = (uint32_t)ldg(a.q_start + i) + lane; t < a.max_tok; t += step) {
            stg(a.slot + t, -1);
            if (a.tok_seq) stg(a.tok_seq + t, -1);
            if (a.tok_pos) stg(a.tok_pos + t, -1);
        }
        return;
    }
    const Ask q = ask_of(a, i);
    const uint32_t t0 = (uint32_t)ldg(a.q_start + i), t1 = (uint32_t)ldg(a.q_start + i + 1u);
    const int32_t len = ldg(a.kv_len + i), top = ldg(a.top + i);
    const bool granted = q.fits && (int64_t)len == q.ctx + q.add && t1 - t0 == (uint32_t)q.add;
    int32_t *const row = a.table + (size_t)i * a.stride;
    if (granted)
        for (uint32_t j = lane; j < q.need; j += step) stg(row + q.held + j, ldg(a.free_pages + top - 1 - (int32_t)j));
    for (uint32_t t = t0 + lane; t < t1; t += step) {
        const int64_t p = q.ctx + (t - t0);
        int32_t s = -1;
        if (granted) {
            const uint32_t pg = q4kv_page_of(a.page, (uint32_t)p);
            const int32_t number =
                pg < q.held ? ldg(row + pg) : ldg(a.free_pages + top - 1 - (int32_t)(pg - q.held));
            if ((uint32_t)number < a.n_pages)
                s = (int32_t)((uint32_t)number * a.page.d + ((uint32_t)p - pg * a.page.d));
        }
        stg(a.slot + t, s);
        if (a.tok_seq) stg(a.tok_seq + t, (int32_t)i);
        if (a.tok_pos) stg(a.tok_pos + t, (int32_t)min(max(p, (int64_t)INT32_MIN), (int64_t)INT32_MAX));
    }
}

/* ---- rows ---- */

struct RowsArgs {
    uint8_t *kp, *vp;
    const float *k, *v;
    float *ko, *vo;
    const int32_t *slot;
    uint64_t k_stride, v_stride;
    uint32_t n_tok, n, bpt, n_slots;
};

/* Eight lanes per 32 values, four each, of K (grid.y 0) or V. */
template <int KIND> __global__ __launch_bounds__(256) void paged_append_k(RowsArgs a) {
    const uint64_t quad = (uint64_t)blockIdx.x * 256u + threadIdx.x;
    const uint32_t nq = (a.n + 3u) / 4u;
    const uint64_t t = quad / nq;
    const uint32_t at = 4u * (uint32_t)(quad - t * nq);
    const int32_t slot = t < a.n_tok ? ldg(a.slot + t) : -1;
    const bool live = slot >= 0 && (uint32_t)slot < a.n_slots;
    const float *src = blockIdx.y ? a.v + t * a.v_stride : a.k + t * a.k_stride;
    uint8_t *dst = (blockIdx.y ? a.vp : a.kp) + (size_t)(live ? slot : 0) * a.bpt;
    float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (uint32_t i = 0; i < 4u; i++)
        if (live && at + i < a.n) x[i] = ldg(src + at + i);
    if constexpr (KIND == Q4KV_Q8) {
        int q[4]; /* the eight lanes of a block are of one token: n % 32 == 0 */
        const float d = q8_lane_quant(x[0], x[1], x[2], x[3], q);
        if (live) q8_lane_store(dst + (size_t)(at / 32u) * 34u, (at / 4u) & 7u, d, q);
    } else if (live) {
#pragma unroll
        for (uint32_t i = 0; i < 4u; i++) {
            if (at + i >= a.n) continue;
            if (KIND == Q4KV_F16)
                stg((uint16_t *)dst + at + i, __half_as_ushort(__float2half_rn(x[i])));
            else
                stg((float *)dst + at + i, x[i]);
        }
    }
}

template <int KIND> __global__ __launch_bounds__(256) void paged_read_k(RowsArgs a) {
    const uint64_t quad = (uint64_t)blockIdx.x * 256u + threadIdx.x;
    const uint32_t nq = (a.n + 3u) / 4u;
    const uint64_t t = quad / nq;
    if (t >= a.n_tok) return;
    const uint32_t at = 4u * (uint32_t)(quad - t * nq);
    const int32_t slot = ldg(a.slot + t);
    const bool live = slot >= 0 && (uint32_t)slot < a.n_slots;
    const uint8_t *src = (blockIdx.y ? a.vp : a.kp) + (size_t)(live ? slot : 0) * a.bpt;
    float *dst = (blockIdx.y ? a.vo : a.ko) + t * a.n;
#pragma unroll
    for (uint32_t i = 0; i < 4u; i++) {
        const uint32_t e = at + i;
        if (e >= a.n) continue;
        float x = 0.f;
        if (live) {
            if (KIND == Q4KV_Q8) {
                const uint8_t *blk = src + (size_t)(e / 32u) * 34u;
                x = (float)(int8_t)ldg(blk + 2u + (e & 31u)) *
                    __half2float(__ushort_as_half(ldg((const uint16_t *)blk)));
            } else if (KIND == Q4KV_F16) {
                x = __half2float(__ushort_as_half(ldg((const uint16_t *)src + e)));
            } else {
                x = ldg((const float *)src + e);
            }
        }
        stg(dst + e, x);
    }
}

/* ---- position lists as slots ---- */

struct SlotsArgs {
    const int32_t *idx, *tok_seq, *table, *kv_len;
    int32_t *out;
    uint64_t n;
    uint32_t width, n_list, n_seq, stride, n_pages;
    PageDiv page;
};

__global__ __launch_bounds__(256) void paged_slots_k(SlotsArgs a) {
    const uint64_t e = (uint64_t)blockIdx.x * 256u + threadIdx.x;
    if (e >= a.n) return;
    const int32_t p = ldg(a.idx + e), seq = ldg(a.tok_seq + e / a.width / a.n_list);
    int32_t s = -1;
    if (seq >= 0 && (uint32_t)seq < a.n_seq && p >= 0 && p < ldg(a.kv_len + seq)) {
        const uint32_t pg = q4kv_page_of(a.page, (uint32_t)p);
        const int32_t number = pg < a.stride ? ldg(a.table + (size_t)seq * a.stride + pg) : -1;
        if ((uint32_t)number < a.n_pages) s = (int32_t)((uint32_t)number * a.page.d + ((uint32_t)p - pg * a.page.d));
    }
    stg(a.out + e, s);
}

bool rows_ok(const void *kp, const void *vp, const void *k, const void *v, const int32_t *slot,
             uint32_t n_tok, uint32_t n, uint32_t bpt, uint32_t n_slots, int kind) {
    if (!q4kv_ok || !kp || !vp || !k || !v || !slot || !n_tok || !n || !bpt || !n_slots) return false;
    if (n_slots > 0x7fffffffu || kind < Q4KV_F32 || kind > Q4KV_Q8) return false;
    if (kind == Q4KV_Q8 && (n % 32u || bpt % 2u)) return false;
    /* a row's bytes fit its slot, and its values lie where they can be stored */
    const uint64_t row = kind == Q4KV_Q8 ? (uint64_t)n / 32u * 34u : (uint64_t)n * (kind == Q4KV_F16 ? 2u : 4u);
    const uintptr_t al = kind == Q4KV_F32 ? 3u : 1u;
    return row <= bpt && (((uintptr_t)kp | (uintptr_t)vp | bpt) & al) == 0;
}

/* workgroups of 256 threads with four values each; 0 where the grid has no room */
uint32_t quads_grid(uint32_t n_tok, uint32_t n) {
    const uint64_t wg = ((uint64_t)n_tok * ((n + 3u) / 4u) + 255u) / 256u;
    return wg <= 0x7fffffu ? (uint32_t)wg : 0u;
}

} // namespace

extern "C" bool q4_hip_paged_release(const int32_t *table, uint32_t table_stride, const int32_t *lens,
                                     const int32_t *rows, uint32_t n, uint32_t page,
                                     int32_t *free_pages, uint32_t n_pages, const int32_t *n_free,
                                     int32_t *left) {
    Q4KV_FLUSH_OR_FAIL();
    if (!q4kv_ok || !table || !lens || !free_pages || !n_free || !left) return false;
    if (!q4kv_pages_ok(n, table_stride, page, n_pages)) return false;
    if (!q4kv_part || q4kv_part_cap < n) {
        Q4KV_ERR("paged release: no scratch");
        return false;
    }
    (void)hipGetLastError();
    const ReleaseArgs a = {table,        lens, rows,    free_pages,           n_free, left, (int32_t *)q4kv_part,
                           table_stride, n,    n_pages, q4kv_page_div(page)};
    release_scan_k<<<1, SCAN_T, 0, q4kv_stream>>>(a);
    release_fill_k<<<(n + 3u) / 4u, 256, 0, q4kv_stream>>>(a);
    return q4kv_launch_ok("paged release");
}

extern "C" bool q4_hip_paged_plan(const int32_t *ctx_len, const int32_t *n_new, uint32_t n_seq,
                                  uint32_t page, int32_t *table, uint32_t table_stride,
                                  const int32_t *free_pages, uint32_t n_pages, const int32_t *n_free,
                                  int32_t *left, int32_t *q_start, int32_t *kv_len, uint32_t max_tok,
                                  int32_t *slot, int32_t *tok_seq, int32_t *tok_pos) {
    Q4KV_FLUSH_OR_FAIL();
    if (!q4kv_ok || !ctx_len || !n_new || !table || !free_pages || !n_free || !left || !q_start ||
        !kv_len || !slot || !max_tok || max_tok > 0x7fffffffu)
        return false;
    if (!q4kv_pages_ok(n_seq, table_stride, page, n_pages)) return false;
    if (!q4kv_part || q4kv_part_cap < n_seq) {
        Q4KV_ERR("paged plan: no scratch");
        return false;
    }
    (void)hipGetLastError();
    const PlanArgs a = {ctx_len, n_new, free_pages, n_free, table,        left,    q_start, kv_len,
                        slot,    tok_seq, tok_pos, (int32_t *)q4kv_part, n_seq, table_stride, n_pages, max_tok,
                        q4kv_page_div(page)};
    plan_scan_k<<<1, SCAN_T, 0, q4kv_stream>>>(a);
    const uint32_t y = std::min(64u, std::max(1u, max_tok / 1024u));
    plan_fill_k<<<dim3(n_seq / 4u + 1u, y), 256, 0, q4kv_stream>>>(a);
    return q4kv_launch_ok("paged plan");
}

extern "C" bool q4_hip_paged_append(void *kpool, void *vpool, const float *k, const float *v,
                                    uint64_t k_stride, uint64_t v_stride, const int32_t *slot,
                                    uint32_t n_tok, uint32_t n, uint32_t bpt, uint32_t n_slots,
                                    int kind) {
    Q4KV_FLUSH_OR_FAIL();
    if (!rows_ok(kpool, vpool, k, v, slot, n_tok, n, bpt, n_slots, kind) || k_stride < n || v_stride < n)
        return false;
    const uint32_t grid = quads_grid(n_tok, n);
    if (!grid) return false;
    (void)hipGetLastError();
    const RowsArgs a = {(uint8_t *)kpool, (uint8_t *)vpool, k,        v,     nullptr, nullptr,
                        slot,             k_stride,         v_stride, n_tok, n,       bpt,
                        n_slots};
    if (kind == Q4KV_Q8)
        paged_append_k<Q4KV_Q8><<<dim3(grid, 2), 256, 0, q4kv_stream>>>(a);
    else if (kind == Q4KV_F16)
        paged_append_k<Q4KV_F16><<<dim3(grid, 2), 256, 0, q4kv_stream>>>(a);
    else
        paged_append_k<Q4KV_F32><<<dim3(grid, 2), 256, 0, q4kv_stream>>>(a);
    return q4kv_launch_ok("paged append");
}

extern "C" bool q4_hip_paged_read(const void *kpool, const void *vpool, float *k, float *v,
                                  const int32_t *slot, uint32_t n_tok, uint32_t n, uint32_t bpt,
                                  uint32_t n_slots, int kind) {
    Q4KV_FLUSH_OR_FAIL();
    if (!rows_ok(kpool, vpool, k, v, slot, n_tok, n, bpt, n_slots, kind)) return false;
    const uint32_t grid = quads_grid(n_tok, n);
    if (!grid) return false;
    (void)hipGetLastError();
    const RowsArgs a = {(uint8_t *)kpool, (uint8_t *)vpool, nullptr, nullptr, k, v,  slot,
                        n,                n,                n_tok,   n,       bpt, n_slots};
    if (kind == Q4KV_Q8)
        paged_read_k<Q4KV_Q8><<<dim3(grid, 2), 256, 0, q4kv_stream>>>(a);
    else if (kind == Q4KV_F16)
        paged_read_k<Q4KV_F16><<<dim3(grid, 2), 256, 0, q4kv_stream>>>(a);
    else
        paged_read_k<Q4KV_F32><<<dim3(grid, 2), 256, 0, q4kv_stream>>>(a);
    return q4kv_launch_ok("paged read");
}

extern "C" bool q4_hip_paged_slots(const int32_t *idx, int32_t *out, const int32_t *tok_seq,
                                   uint32_t n_tok, uint32_t n_list, uint32_t width,
                                   const q4kv_paged_batch *b) {
    Q4KV_FLUSH_OR_FAIL();
    if (!q4kv_ok || !idx || !out || !tok_seq || !n_tok || !n_list || !width || !q4kv_batch_ok(b)) return false;
    const uint64_t n = (uint64_t)n_tok * n_list;
    if (n > 0x7fffffffu || n * width > 0x7fffff00ull * 256u) return false;
    (void)hipGetLastError();
    const SlotsArgs a = {idx,   tok_seq, b->table, b->kv_len,       out,        n * width,
                         width, n_list,  b->n_seq, b->table_stride, b->n_pages, q4kv_page_div(b->page)};
    paged_slots_k<<<(uint32_t)((a.n + 255u) / 256u), 256, 0, q4kv_stream>>>(a);
    return q4kv_launch_ok("paged slots");
}
