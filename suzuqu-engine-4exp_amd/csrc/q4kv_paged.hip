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

/* The last of n ascending values that is <= v (at[0] <= v). */
__device__ inline uint32_t last_at(const int32_t *at, uint32_t n, int32_t v) {
    uint32_t lo = 0u, hi = n;
    while (hi - lo > 1u) {
        const uint32_t mid = (lo + hi) / 2u;
        if (at[mid] <= v)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
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

/* Up to SCAN_T requests in one launch (a second one costs 4 us, as much as
 * all of this): every workgroup scans all of them and copies its share of the
 * pages, a thread each, whose requests it finds in LDS. With more than one
 * workgroup left is not n_free, which the others may still read. 40 requests
 * of 380 pages: 4.2 us (a wave per request, by one workgroup: 5.9). */
__global__ __launch_bounds__(SCAN_T) void release_one_k(ReleaseArgs a) {
    __shared__ int64_t tot[SCAN_T / 64][2];
    __shared__ int32_t s_page[SCAN_T], s_row[SCAN_T];
    __shared__ uint32_t s_all;
    const uint32_t i = threadIdx.x, step = SCAN_T * gridDim.x;
    const int64_t have = clamp_count(ldg(a.n_free), a.n_pages), room = a.n_pages - have;
    int32_t row = 0;
    const int64_t held = i < a.n ? release_row(a, i, row) : 0;
    int64_t upto = held, unused = 0;
    scan2(upto, unused, tot);
    if (i < a.n) {
        s_page[i] = (int32_t)min(upto - held, room);
        s_row[i] = row;
    }
    if (i == SCAN_T - 1u) {
        s_all = (uint32_t)min(upto, room);
        if (blockIdx.x == 0u) stg(a.left, (int32_t)(have + s_all));
    }
    __syncthreads();
    const uint32_t all = s_all;
    for (uint32_t f = blockIdx.x * SCAN_T + i; f < all; f += step) {
        const uint32_t r = last_at(s_page, a.n, (int32_t)f);
        stg(a.free_pages + have + f, ldg(a.table + (size_t)s_row[r] * a.stride + (f - (uint32_t)s_page[r])));
    }
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

/* Up to SCAN_T requests in one launch: every workgroup scans all of them (a
 * second launch costs more) and takes its share of the tokens and of the new
 * pages, a thread each, whose requests it finds in LDS. Workgroup 0 writes
 * what the requests have; with more than one, left is not n_free, which the
 * others may still read. 64 decodes 5.1 us; 16 prompt chunks of 1000 tokens
 * beside 368 decodes 6.3 (four tokens a thread: 9.1). */
__global__ __launch_bounds__(SCAN_T) void plan_one_k(PlanArgs a) {
    __shared__ int64_t tot[SCAN_T / 64][2];
    __shared__ int32_t s_start[SCAN_T + 1], s_page[SCAN_T + 1]; /* tokens and lacking pages before a request */
    __shared__ int32_t s_ctx[SCAN_T];
    __shared__ uint32_t s_held[SCAN_T]; /* refused: ~0 */
    __shared__ uint32_t s_taken, s_refused;
    const uint32_t i = threadIdx.x, step = SCAN_T * gridDim.x;
    const int64_t avail = clamp_count(ldg(a.n_free), a.n_pages);
    if (i == 0u) s_taken = s_refused = 0u;
    Ask q = {0, 0, true, 0u, 0u};
    if (i < a.n_seq) q = ask_of(a, i);
    int64_t tok = q.add, need = q.need;
    scan2(tok, need, tot);
    /* a request whose tokens end past max_tok asks for no page */
    const bool past = tok > (int64_t)a.max_tok && q.add;
    if (__syncthreads_or(past)) {
        if (past) {
            q.fits = false;
            q.need = 0u;
        }
        int64_t unused = 0;
        need = q.need;
        scan2(need, unused, tot);
    }
    const bool granted = q.fits && (q.need == 0u || need <= avail);
    const int32_t t0 = (int32_t)min(tok - q.add, (int64_t)a.max_tok), t1 = (int32_t)min(tok, (int64_t)a.max_tok);
    if (i < a.n_seq) {
        s_start[i] = t0;
        s_page[i] = (int32_t)min(need - q.need, avail);
        s_ctx[i] = (int32_t)q.ctx;
        s_held[i] = granted ? q.held : ~0u;
        if (granted && q.need) atomicMax(&s_taken, (uint32_t)need);
        if (!granted) atomicAdd(&s_refused, 1u);
        if (i + 1u == a.n_seq) s_start[a.n_seq] = t1;
        if (blockIdx.x == 0u) {
            stg(a.q_start + i, t0);
            if (i + 1u == a.n_seq) stg(a.q_start + i + 1u, t1);
            stg(a.kv_len + i, granted ? (int32_t)(q.ctx + q.add) : 0);
        }
    }
    __syncthreads();
    const uint32_t taken = s_taken;
    if (blockIdx.x == 0u && i == 0u) {
        stg(a.left, (int32_t)(avail - taken));
        stg(a.left + 1, (int32_t)s_refused);
    }
    const int32_t *const top = a.free_pages + avail; /* page f of all new ones is top[-1 - f] */
    for (uint32_t f = blockIdx.x * SCAN_T + i; f < taken; f += step) {
        const uint32_t r = last_at(s_page, a.n_seq, (int32_t)f), held = s_held[r];
        /* pages below `taken` are of granted requests that lack some */
        stg(a.table + (size_t)r * a.stride + held + (f - (uint32_t)s_page[r]), ldg(top - 1 - (int32_t)f));
    }
    const uint32_t n_tok = (uint32_t)s_start[a.n_seq];
    for (uint32_t t = blockIdx.x * SCAN_T + i; t < a.max_tok; t += step) {
        int32_t s = -1, seq = -1, pos = -1;
        if (t < n_tok) {
            const uint32_t r = last_at(s_start, a.n_seq, (int32_t)t);
            const int64_t p = (int64_t)s_ctx[r] + (t - (uint32_t)s_start[r]);
            seq = (int32_t)r;
            pos = (int32_t)min(p, (int64_t)INT32_MAX);
            if (s_held[r] != ~0u) {
                const uint32_t pg = q4kv_page_of(a.page, (uint32_t)p);
                const int32_t number = pg < s_held[r] ? ldg(a.table + (size_t)r * a.stride + pg)
                                                      : ldg(top - 1 - s_page[r] - (int32_t)(pg - s_held[r]));
                if ((uint32_t)number < a.n_pages)
                    s = (int32_t)((uint32_t)number * a.page.d + ((uint32_t)p - pg * a.page.d));
            }
        }
        stg(a.slot + t, s);
        if (a.tok_seq) stg(a.tok_seq + t, seq);
        if (a.tok_pos) stg(a.tok_pos + t, pos);
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
    PageDiv quads; /* of a token */
    bool rows16;   /* q8_0: slots of whole 256-value groups, 16-byte aligned */
};

typedef float f4a_t __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u2a_t __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u1a_t __attribute__((aligned(2)));

/* This thread's four values: token t, the first value's index. Whether its
 * token is one, the row that its slot names and whether there is one. */
struct Quad {
    uint32_t t, at, slot;
    bool in, live, whole;
    __device__ explicit Quad(const RowsArgs &a) {
        const uint32_t quad = blockIdx.x * 256u + threadIdx.x;
        t = q4kv_page_of(a.quads, quad);
        at = 4u * (quad - t * a.quads.d);
        in = t < a.n_tok;
        const int32_t s = in ? ldg(a.slot + t) : -1;
        live = s >= 0 && (uint32_t)s < a.n_slots;
        slot = live ? (uint32_t)s : 0u;
        whole = at + 4u <= a.n;
    }
};

/* Eight lanes per 32 values, four each, of K (grid.y 0) or V. Bound by the
 * bytes: 8192 tokens of 512 values, q8_0, read 33.6 MB and write 8.9 in 10.5 us
 * (q8_0 blocks written from LDS, 17 stores of 16 bytes per 8 of them; two bytes
 * a store took 13.8). */
template <int KIND> __global__ __launch_bounds__(256) void paged_append_k(RowsArgs a) {
    __shared__ __attribute__((aligned(16))) uint8_t s_row[KIND == Q4KV_Q8 ? 4 : 1][272];
    const Quad q(a);
    const float *src = (blockIdx.y ? a.v + q.t * a.v_stride : a.k + q.t * a.k_stride) + q.at;
    uint8_t *dst = (blockIdx.y ? a.vp : a.kp) + (size_t)q.slot * a.bpt;
    q4kv_f4 x = {0.f, 0.f, 0.f, 0.f};
    if (q.live) {
        if (q.whole) {
            x = *(const GLOBAL f4a_t *)src;
        } else {
            for (uint32_t i = 0; q.at + i < a.n; i++) x[i] = ldg(src + i);
        }
    }
    if constexpr (KIND == Q4KV_Q8) {
        int v[4]; /* the eight lanes of a block are of one token: n % 32 == 0 */
        const float d = q8_lane_quant(x[0], x[1], x[2], x[3], v);
        const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
        if (a.rows16) {
            /* a wave's eight blocks are of one row, 272 bytes from a multiple
             * of 16: written as 16-byte pieces */
            q8_lane_store(s_row[wave] + 34u * (lane >> 3), lane & 7u, d, v);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            if (q.live && lane < 17u)
                stg((q4kv_u4 *)(dst + (size_t)((q.at & ~255u) / 32u) * 34u) + lane, ((const q4kv_u4 *)s_row[wave])[lane]);
        } else if (q.live) {
            q8_lane_store(dst + (size_t)(q.at / 32u) * 34u, lane & 7u, d, v);
        }
    } else if (q.live && KIND == Q4KV_F16) {
        const uint32_t h[4] = {__half_as_ushort(__float2half_rn(x[0])), __half_as_ushort(__float2half_rn(x[1])),
                               __half_as_ushort(__float2half_rn(x[2])), __half_as_ushort(__float2half_rn(x[3]))};
        if (q.whole) {
            *(GLOBAL u2a_t *)((uint16_t *)dst + q.at) = (u2a_t){h[0] | h[1] << 16, h[2] | h[3] << 16};
        } else {
            for (uint32_t i = 0; q.at + i < a.n; i++) stg((uint16_t *)dst + q.at + i, (uint16_t)h[i]);
        }
    } else if (q.live) {
        if (q.whole) {
            *(GLOBAL f4a_t *)((float *)dst + q.at) = x;
        } else {
            for (uint32_t i = 0; q.at + i < a.n; i++) stg((float *)dst + q.at + i, x[i]);
        }
    }
}

/* As many threads and bytes as paged_append_k: 9.1 us for its 8192 tokens. */
template <int KIND> __global__ __launch_bounds__(256) void paged_read_k(RowsArgs a) {
    const Quad q(a);
    if (!q.in) return;
    const uint8_t *src = (blockIdx.y ? a.vp : a.kp) + (size_t)q.slot * a.bpt;
    float *dst = (blockIdx.y ? a.vo : a.ko) + (size_t)q.t * a.n + q.at;
    q4kv_f4 x = {0.f, 0.f, 0.f, 0.f};
    if (q.live) {
        if constexpr (KIND == Q4KV_Q8) {
            const uint8_t *blk = src + (size_t)(q.at / 32u) * 34u;
            const float d = __half2float(__ushort_as_half(ldg((const uint16_t *)blk)));
            const uint32_t w = *(const GLOBAL u1a_t *)(blk + 2u + (q.at & 31u));
#pragma unroll
            for (uint32_t i = 0; i < 4u; i++) x[i] = (float)(int8_t)(w >> (8u * i)) * d;
        } else if constexpr (KIND == Q4KV_F16) {
            uint32_t h[4] = {0u, 0u, 0u, 0u};
            if (q.whole) {
                const u2a_t w = *(const GLOBAL u2a_t *)((const uint16_t *)src + q.at);
                h[0] = w[0] & 0xFFFFu;
                h[1] = w[0] >> 16;
                h[2] = w[1] & 0xFFFFu;
                h[3] = w[1] >> 16;
            } else {
                for (uint32_t i = 0; q.at + i < a.n; i++) h[i] = ldg((const uint16_t *)src + q.at + i);
            }
#pragma unroll
            for (uint32_t i = 0; i < 4u; i++) x[i] = __half2float(__ushort_as_half((unsigned short)h[i]));
        } else if (q.whole) {
            x = *(const GLOBAL f4a_t *)((const float *)src + q.at);
        } else {
            for (uint32_t i = 0; q.at + i < a.n; i++) x[i] = ldg((const float *)src + q.at + i);
        }
    }
    if (q.whole) {
        *(GLOBAL f4a_t *)dst = x;
    } else {
        for (uint32_t i = 0; q.at + i < a.n; i++) stg(dst + i, x[i]);
    }
}

/* ---- position lists as slots ---- */

struct SlotsArgs {
    const int32_t *idx, *tok_seq, *table, *kv_len;
    int32_t *out;
    uint32_t rows, width, n_list, n_seq, stride, n_pages;
    PageDiv page;
};

/* A row's request is the workgroup's; four entries a thread, SLOT_W apart, so
 * that their table entries are on the way together: 3.1 us for 64 lists of
 * 2051, 4.2 for 512, a launch and three dependent loads. */
constexpr uint32_t SLOT_W = 256;
__global__ __launch_bounds__(SLOT_W) void paged_slots_k(SlotsArgs a) {
    for (uint32_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const int32_t seq = ldg(a.tok_seq + row / a.n_list);
        const bool some = seq >= 0 && (uint32_t)seq < a.n_seq;
        const int32_t n = some ? (int32_t)min((uint64_t)(uint32_t)max(ldg(a.kv_len + seq), 0), (uint64_t)a.stride * a.page.d) : 0;
        const int32_t *const trow = a.table + (some ? (size_t)seq * a.stride : 0u);
        for (uint32_t j0 = blockIdx.x * 4u * SLOT_W + threadIdx.x; j0 < a.width; j0 += gridDim.x * 4u * SLOT_W) {
            const size_t at = (size_t)row * a.width + j0;
            int32_t p[4], number[4];
#pragma unroll
            for (uint32_t k = 0; k < 4u; k++) p[k] = j0 + k * SLOT_W < a.width ? ldg(a.idx + at + k * SLOT_W) : -1;
#pragma unroll
            for (uint32_t k = 0; k < 4u; k++)
                number[k] = p[k] >= 0 && p[k] < n ? ldg(trow + q4kv_page_of(a.page, (uint32_t)p[k])) : -1;
#pragma unroll
            for (uint32_t k = 0; k < 4u; k++) {
                if (j0 + k * SLOT_W >= a.width) continue;
                const uint32_t pg = q4kv_page_of(a.page, (uint32_t)p[k]);
                stg(a.out + at + k * SLOT_W, (uint32_t)number[k] < a.n_pages
                                                 ? (int32_t)((uint32_t)number[k] * a.page.d + ((uint32_t)p[k] - pg * a.page.d))
                                                 : -1);
            }
        }
    }
}

/* workgroups of SCAN_T threads for n entries, one a thread up to a chipful */
uint32_t share_of(uint64_t n) { return (uint32_t)std::min((n + SCAN_T - 1u) / SCAN_T, (uint64_t)256u); }

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

/* Launches f(args, workgroups) over all tokens, 2^30 quads at a time. */
template <class F> bool each_quads(RowsArgs a, const char *what, F f) {
    const uint32_t nq = (a.n + 3u) / 4u, most = std::max(1u, (1u << 30) / nq);
    if (nq > 1u << 30) return false;
    a.quads = q4kv_page_div(nq);
    a.rows16 = a.n % 256u == 0u && (((uintptr_t)a.kp | (uintptr_t)a.vp | a.bpt) & 15u) == 0u;
    (void)hipGetLastError();
    for (uint32_t left = a.n_tok; left;) {
        a.n_tok = std::min(left, most);
        f(a, (uint32_t)(((uint64_t)a.n_tok * nq + 255u) / 256u));
        left -= a.n_tok;
        a.slot += a.n_tok;
        if (a.k) a.k += a.n_tok * a.k_stride;
        if (a.v) a.v += a.n_tok * a.v_stride;
        if (a.ko) a.ko += (uint64_t)a.n_tok * a.n;
        if (a.vo) a.vo += (uint64_t)a.n_tok * a.n;
    }
    return q4kv_launch_ok(what);
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
    const uint32_t wgs = share_of((uint64_t)n * table_stride);
    if (n <= SCAN_T && (wgs == 1u || left != n_free)) {
        release_one_k<<<wgs, SCAN_T, 0, q4kv_stream>>>(a);
    } else {
        release_scan_k<<<1, SCAN_T, 0, q4kv_stream>>>(a);
        release_fill_k<<<(n + 3u) / 4u, 256, 0, q4kv_stream>>>(a);
    }
    return q4kv_launch_ok("paged release");
}

extern "C" bool q4_hip_paged_plan(const int32_t *ctx_len, const int32_t *n_new, uint32_t n_seq,
                                  uint32_t page, int32_t *table, uint32_t table_stride,
                                  const int32_t *free_pages, uint32_t n_pages, const int32_t *n_free,
                                  int32_t *left, int32_t *q_start, int32_t *kv_len, uint32_t max_tok,
                                  int32_t *slot, int32_t *tok_seq, int32_t *tok_pos) {
    Q4KV_FLUSH_OR_FAIL();
    if (!q4kv_ok || !ctx_len || !n_new || !table || !free_pages || !n_free || !left || !q_start ||
        !kv_len || !slot || !max_tok || max_tok > 0x7fffffffu || kv_len == ctx_len || kv_len == n_new ||
        q_start == ctx_len || q_start == n_new)
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
    const uint32_t wgs = share_of(max_tok);
    if (n_seq <= SCAN_T && (wgs == 1u || (n_free != left && n_free != left + 1))) {
        plan_one_k<<<wgs, SCAN_T, 0, q4kv_stream>>>(a);
        return q4kv_launch_ok("paged plan");
    }
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
    const RowsArgs a = {(uint8_t *)kpool, (uint8_t *)vpool, k,       v,       nullptr, nullptr, slot, k_stride,
                        v_stride,         n_tok,            n,       bpt,     n_slots, {},      false};
    return each_quads(a, "paged append", [&](const RowsArgs &r, uint32_t grid) {
        if (kind == Q4KV_Q8)
            paged_append_k<Q4KV_Q8><<<dim3(grid, 2), 256, 0, q4kv_stream>>>(r);
        else if (kind == Q4KV_F16)
            paged_append_k<Q4KV_F16><<<dim3(grid, 2), 256, 0, q4kv_stream>>>(r);
        else
            paged_append_k<Q4KV_F32><<<dim3(grid, 2), 256, 0, q4kv_stream>>>(r);
    });
}

extern "C" bool q4_hip_paged_read(const void *kpool, const void *vpool, float *k, float *v,
                                  const int32_t *slot, uint32_t n_tok, uint32_t n, uint32_t bpt,
                                  uint32_t n_slots, int kind) {
    Q4KV_FLUSH_OR_FAIL();
    if (!rows_ok(kpool, vpool, k, v, slot, n_tok, n, bpt, n_slots, kind)) return false;
    const RowsArgs a = {(uint8_t *)kpool, (uint8_t *)vpool, nullptr, nullptr, k,       v,  slot, n,
                        n,                n_tok,            n,       bpt,     n_slots, {}, false};
    return each_quads(a, "paged read", [&](const RowsArgs &r, uint32_t grid) {
        if (kind == Q4KV_Q8)
            paged_read_k<Q4KV_Q8><<<dim3(grid, 2), 256, 0, q4kv_stream>>>(r);
        else if (kind == Q4KV_F16)
            paged_read_k<Q4KV_F16><<<dim3(grid, 2), 256, 0, q4kv_stream>>>(r);
        else
            paged_read_k<Q4KV_F32><<<dim3(grid, 2), 256, 0, q4kv_stream>>>(r);
    });
}

extern "C" bool q4_hip_paged_slots(const int32_t *idx, int32_t *out, const int32_t *tok_seq,
                                   uint32_t n_tok, uint32_t n_list, uint32_t width,
                                   const q4kv_paged_batch *b) {
    Q4KV_FLUSH_OR_FAIL();
    if (!q4kv_ok || !idx || !out || !tok_seq || !n_tok || !n_list || !width || !q4kv_batch_ok(b)) return false;
    const uint64_t rows = (uint64_t)n_tok * n_list;
    if (rows > 0x7fffffffu || width > 0x7fffffffu) return false;
    (void)hipGetLastError();
    const SlotsArgs a = {idx,   tok_seq, b->table, b->kv_len,       out,        (uint32_t)rows,
                         width, n_list,  b->n_seq, b->table_stride, b->n_pages, q4kv_page_div(b->page)};
    const uint32_t x = std::min((width + 4u * SLOT_W - 1u) / (4u * SLOT_W), 65535u);
    paged_slots_k<<<dim3(x, std::min((uint32_t)rows, 65535u)), SLOT_W, 0, q4kv_stream>>>(a);
    return q4kv_launch_ok("paged slots");
}
