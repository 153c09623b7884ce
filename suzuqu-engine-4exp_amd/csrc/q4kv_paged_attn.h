/*
 * q4kv_paged_attn.h -- what the paged attention kernels share: a launch's
 * arguments, requests, and the division of a ragged batch's work.
 *
 * The division. A request's new tokens times the query heads of a KV head are
 * columns, NC of them a tile; a tile streams the positions that its last
 * token sees. The lengths are on the device, so a launch has a fixed number
 * of workgroups and each finds its share itself: the costs of all tiles of
 * all requests and KV heads, laid end to end, are cut into equal runs, one per
 * workgroup, wherever the cuts fall (but not within SNAP of a tile's ends).
 * A batch of any mix of lengths fills the chip evenly, and a tile is only cut
 * where a run ends: at most one begins and one ends inside a workgroup's run,
 * so two partial slots per workgroup hold all that a second launch merges.
 */
#ifndef Q4KV_PAGED_ATTN_H
#define Q4KV_PAGED_ATTN_H
#include <hip/hip_runtime.h>
#include <math.h>

#include "q4kv_tile.h"
#include "q4kv_paged.h"

struct PagedArgs {
    const float *q, *gate;
    const uint8_t *kp, *vp;
    float *out;
    const int32_t *table, *q_start, *kv_len;
    uint32_t n_seq, stride, n_pages, n_tok;
    uint32_t n_head, n_kvh, gqa, hd, rowb; /* rowb: bytes of one KV head's row */
    PageDiv page;
    float scale_log2;
    /* the division: requests of min_cols .. max_cols columns per KV head take
     * part; partials and the records of cut tiles */
    uint32_t min_cols, max_cols;
    float *part;
};

/* One request: its first token and how many (those below n_tok), the position
 * of the first one, and the positions that its table row can hold. */
struct Req {
    uint32_t t0, n_q, cap;
    int64_t pos0;
};
__device__ inline Req req_of(const PagedArgs &a, uint32_t i) {
    const int32_t s0 = ldg(a.q_start + i), s1 = ldg(a.q_start + i + 1u), len = ldg(a.kv_len + i);
    Req r;
    r.cap = a.stride * a.page.d;
    r.t0 = (uint32_t)max(s0, 0);
    const int64_t n = (int64_t)s1 - r.t0;
    r.pos0 = (int64_t)len - max(n, (int64_t)0);
    r.n_q = n <= 0 || r.t0 >= a.n_tok ? 0u : min((uint32_t)n, a.n_tok - r.t0);
    return r;
}
/* positions that token t of the request sees */
__device__ inline uint32_t seen_by(const Req &r, uint32_t t) {
    const int64_t n = r.pos0 + t + 1;
    return n <= 0 ? 0u : n < r.cap ? (uint32_t)n : r.cap;
}
/* the slot of position p of request i, or < 0 where its table names no page */
__device__ inline int32_t slot_at(const PagedArgs &a, uint32_t i, uint32_t p) {
    const uint32_t pg = q4kv_page_of(a.page, p);
    const int32_t number = ldg(a.table + (size_t)i * a.stride + pg);
    return (uint32_t)number < a.n_pages ? (int32_t)((uint32_t)number * a.page.d + (p - pg * a.page.d)) : -1;
}


/* ---- the division of the work ---- */

/* a quotient of whole numbers below 2^53 */
__device__ inline uint64_t div53(uint64_t x, uint64_t y) {
    uint64_t q = (uint64_t)((double)x / (double)y);
    if (q * y > x) q--;
    if ((q + 1u) * y <= x) q++;
    return q;
}
__device__ inline uint32_t uni(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }
__device__ inline uint64_t uni64(uint64_t v) { return ((uint64_t)uni((uint32_t)(v >> 32)) << 32) | uni((uint32_t)v); }

/* A request's tiles of NC columns. Costs in sixteenths of a position: tile k
 * costs first + k * step (what it starts with, and the positions that it
 * sees, which grow evenly from the first tile to the last). */
template <uint32_t NC, uint32_t START> struct Tiles {
    uint32_t n, cols;
    uint64_t first, step;
    __device__ uint64_t before(uint64_t k) const { return k * first + step * (k * (k - 1u) / 2u); }
    __device__ uint64_t cost(uint64_t k) const { return first + step * k; }
    __device__ static Tiles of(const PagedArgs &a, const Req &r) {
        Tiles t;
        t.cols = r.n_q * a.gqa;
        t.n = (t.cols + NC - 1u) / NC;
        if (t.cols < a.min_cols || t.cols > a.max_cols) t.n = 0u;
        t.first = t.step = 0u;
        if (t.n) {
            const uint32_t lo = seen_by(r, (min(NC, t.cols) - 1u) / a.gqa), hi = seen_by(r, r.n_q - 1u);
            t.first = 16u * ((uint64_t)START + lo);
            t.step = t.n > 1u ? 16u * (uint64_t)(hi - lo) / (t.n - 1u) : 0u;
        }
        return t;
    }
};

/* a place in the work: tile `tile` of KV head kh of request seq, `x` into it */
struct Place {
    uint32_t seq, kh, tile;
    uint64_t x;
};
/* what the merge of a cut tile reads, one per workgroup: the tile that begins
 * in its run and does not end there, and in how many runs it lies */
struct Cut {
    uint32_t pieces, g, seq, kh, tile, unused[3];
};

template <uint32_t NC, uint32_t START, uint32_t SNAP, uint32_t NTHR> struct Share {
    typedef Tiles<NC, START> T;
    uint64_t u, end; /* what is left of the run */
    uint64_t all;
    uint32_t g, n_g;
    Place at;
    Req req;
    T tiles;

    struct Lds {
        uint64_t wave[NTHR / 64], upto[NTHR];
        uint32_t seq[2];
        uint64_t before[2];
    };

    /* the costs of requests i0 .. i0 + NTHR - 1: their sum; upto holds the running sums */
    __device__ static uint64_t scan(const PagedArgs &a, uint32_t i0, Lds &s) {
        const uint32_t i = i0 + threadIdx.x, lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
        uint64_t c = 0u;
        if (i < a.n_seq) {
            const T t = T::of(a, req_of(a, i));
            if (t.n) c = t.before(t.n) * a.n_kvh;
        }
#pragma unroll
        for (uint32_t d = 1; d < 64u; d *= 2u) {
            const uint64_t lo = (uint32_t)__shfl_up((int)(uint32_t)c, d), hi = (uint32_t)__shfl_up((int)(c >> 32), d);
            if (lane >= d) c += hi << 32 | lo;
        }
        __syncthreads();
        if (lane == 63u) s.wave[wave] = c;
        __syncthreads();
        uint64_t sum = 0u;
#pragma unroll
        for (uint32_t w = 0; w < NTHR / 64u; w++) {
            if (w == wave) c += sum;
            sum += s.wave[w];
        }
        s.upto[threadIdx.x] = c;
        return uni64(sum);
    }

    /* tile and offset of cost r (of one request, all its KV heads) */
    __device__ static void within(const PagedArgs &a, const T &t, uint64_t r, Place &p) {
        const uint64_t w = t.before(t.n);
        p.kh = (uint32_t)div53(r, w);
        r -= p.kh * w;
        uint64_t k = 0u;
        if (t.n == 1u) {
            p.tile = 0u;
            p.x = r;
            return;
        }
        if (t.step) {
            const double b = (double)t.first - 0.5 * (double)t.step;
            k = (uint64_t)fmax(0.0, (sqrt(b * b + 2.0 * (double)t.step * (double)r) - b) / (double)t.step);
            if (k >= t.n) k = t.n - 1u;
        } else {
            k = div53(r, t.first);
        }
        while (t.before(k) > r) k--;
        while (k + 1u < t.n && t.before(k + 1u) <= r) k++;
        p.tile = (uint32_t)k;
        p.x = r - t.before(k);
    }
    /* cuts keep SNAP away from a tile's ends */
    __device__ static uint64_t snapped(uint64_t u, const Place &p, uint64_t cost) {
        return p.x < SNAP ? u - p.x : cost - p.x < SNAP ? u + (cost - p.x) : u;
    }

    /* Finds the run of workgroup blockIdx.x. min_run: costs that are worth a
     * workgroup. False: nothing for this one. */
    __device__ bool find(const PagedArgs &a, Lds &s, uint64_t min_run) {
        all = scan(a, 0u, s);
        for (uint32_t i0 = NTHR; i0 < a.n_seq; i0 += NTHR) all += scan(a, i0, s);
        n_g = gridDim.x;
        if (all < min_run * n_g) n_g = (uint32_t)max((uint64_t)1u, div53(all, min_run));
        /* consecutive runs on one XCD (workgroup L runs on XCD L mod 8): tiles
         * of a request share its rows in one L2 */
        const uint32_t per = (n_g + 7u) / 8u;
        g = (blockIdx.x & 7u) * per + (blockIdx.x >> 3);
        if ((blockIdx.x >> 3) >= per || g >= n_g || !all) return false;
        const uint64_t r[2] = {div53(all * g, n_g), div53(all * (g + 1u), n_g)};
        uint64_t base = 0u;
        uint32_t found = 0u;
        for (uint32_t i0 = 0; i0 < a.n_seq && found < 2u; i0 += NTHR) {
            const uint64_t sum = i0 || a.n_seq > NTHR ? scan(a, i0, s) : all;
            __syncthreads();
            const uint64_t hi = base + s.upto[threadIdx.x], lo = threadIdx.x ? base + s.upto[threadIdx.x - 1u] : base;
#pragma unroll
            for (uint32_t k = 0; k < 2u; k++) {
                if (lo <= r[k] && r[k] < hi) {
                    s.seq[k] = i0 + threadIdx.x;
                    s.before[k] = lo;
                }
            }
            base += sum;
            found = (r[0] < base ? 1u : 0u) + (r[1] < base || r[1] == all ? 1u : 0u);
            __syncthreads();
        }
        uint64_t edge[2] = {0u, all};
#pragma unroll
        for (int k = 1; k >= 0; k--) {
            if (k && r[1] == all) continue;
            at.seq = uni(s.seq[k]);
            req = req_of(a, at.seq);
            tiles = T::of(a, req);
            within(a, tiles, r[k] - s.before[k], at);
            edge[k] = snapped(r[k], at, tiles.cost(at.tile));
        }
        u = uni64(edge[0]);
        end = uni64(edge[1]);
        at.kh = uni(at.kh);
        at.tile = uni(at.tile);
        const uint64_t u0 = uni64(r[0] - at.x); /* the tile's start */
        at.x = u - u0;
        if (u >= end) return false;
        if (at.x == tiles.cost(at.tile)) {
            at.x = 0u;
            next(a);
        }
        return true;
    }
    /* the tile after this one */
    __device__ void next(const PagedArgs &a) {
        if (++at.tile < tiles.n) return;
        at.tile = 0u;
        if (++at.kh < a.n_kvh) return;
        at.kh = 0u;
        do {
            at.seq++;
            if (at.seq >= a.n_seq) { /* not reached: costs are left */
                end = u;
                return;
            }
            req = req_of(a, at.seq);
            tiles = T::of(a, req);
            tiles.n = uni(tiles.n);
        } while (!tiles.n);
    }
    /* The part of the current tile that lies in the run: of its n_pass passes
     * the first and one past the last; whether the tile begins and ends here. */
    __device__ void piece(uint32_t n_pass, uint32_t &p0, uint32_t &p1, bool &begins, bool &ends) const {
        const uint64_t c = tiles.cost(at.tile), x1 = min(c, at.x + (end - u));
        auto pass = [&](uint64_t x) {
            const uint64_t s16 = 16u * START;
            return x <= s16 ? 0u : (uint32_t)div53((x - s16) * n_pass, c - s16);
        };
        begins = at.x == 0u;
        ends = x1 == c;
        p0 = uni(begins ? 0u : pass(at.x));
        p1 = uni(ends ? n_pass : pass(x1));
    }
    /* in how many runs the tile lies that begins in this one */
    __device__ uint32_t pieces() const {
        const uint64_t te = u - at.x + tiles.cost(at.tile);
        uint64_t last = div53(te * n_g - 1u, all); /* the last run whose start is below te */
        if (te - div53(all * last, n_g) < SNAP) last--;
        return uni((uint32_t)(last - g) + 1u);
    }
    __device__ void advance(const PagedArgs &a) {
        const uint64_t c = tiles.cost(at.tile), x1 = min(c, at.x + (end - u));
        u += x1 - at.x;
        at.x = 0u;
        if (u < end) next(a);
    }
};

/* A launch of G workgroups leaves G records of cut tiles, then two partial
 * slots per run: 2 g + 1 for the tile that begins in run g, 2 g for the one
 * that run g continues or ends. A partial row: m, l, two unused, HD sums. */
constexpr uint32_t PAGED_PHEAD = 4;
constexpr size_t paged_part_floats(uint32_t G, uint32_t nc, uint32_t HD) {
    return (size_t)G * (sizeof(Cut) / 4u) + 2u * (size_t)G * nc * (HD + PAGED_PHEAD);
}

/* Merges the cut tiles: workgroup (x, y) takes columns y, y + grid.y, .. of
 * the tile that begins in the run of workgroup x of the launch before: HD / 4
 * lanes of four dims each, lane groups with every NG-th piece, eight of them
 * in flight per group. A piece that saw nothing has l = 0; one with l = NaN
 * (scores that are not finite) takes part. */
template <int HD, uint32_t NC>
__global__ __launch_bounds__(256) static void paged_merge_k(PagedArgs a) {
    constexpr uint32_t LPH = HD / 4, NG = 256 / LPH, ROW = HD + PAGED_PHEAD;
    __shared__ __attribute__((aligned(16))) f4_t s_acc[256];
    __shared__ float s_m[NG], s_l[NG];
    const uint32_t *const cw = (const uint32_t *)((const Cut *)a.part + blockIdx.x);
    const Cut cut = {ldg(cw), ldg(cw + 1), ldg(cw + 2), ldg(cw + 3), ldg(cw + 4), {}};
    if (!cut.pieces) return;
    const uint32_t grp = threadIdx.x / LPH, dl = threadIdx.x % LPH, d = 4u * dl;
    const Req r = req_of(a, cut.seq);
    const uint32_t cols = r.n_q * a.gqa;
    const float *const parts = a.part + gridDim.x * (sizeof(Cut) / 4u);
    for (uint32_t j = blockIdx.y; j < NC && cut.tile * NC + j < cols; j += gridDim.y) {
        const uint32_t col = cut.tile * NC + j, t = col / a.gqa;
        const size_t ro = ((size_t)(r.t0 + t) * a.n_head + cut.kh * a.gqa + (col - t * a.gqa)) * a.hd + d;
        float gt[4] = {0.f, 0.f, 0.f, 0.f};
        if (a.gate && d < a.hd) {
#pragma unroll
            for (uint32_t k = 0; k < 4u; k++) gt[k] = ldg(a.gate + ro + k);
        }
        float M = -INFINITY, L = 0.f;
        f4_t acc = {0.f, 0.f, 0.f, 0.f};
        for (uint32_t s0 = grp; s0 < cut.pieces; s0 += 8u * NG) {
            float ml[8][2];
            f4_t v[8];
#pragma unroll
            for (uint32_t k = 0; k < 8u; k++) {
                const uint32_t s = min(s0 + k * NG, cut.pieces - 1u);
                const float *p = parts + ((size_t)(2u * (cut.g + s) + (s ? 0u : 1u)) * NC + j) * ROW;
                const u2_t x = ldg((const u2_t *)p);
                ml[k][0] = __uint_as_float(x[0]);
                ml[k][1] = s0 + k * NG < cut.pieces ? __uint_as_float(x[1]) : 0.f;
                v[k] = ldg((const f4_t *)(p + PAGED_PHEAD + d));
            }
            float mn = M;
#pragma unroll
            for (uint32_t k = 0; k < 8u; k++)
                if (ml[k][1] != 0.f) mn = fmax2(mn, ml[k][0]);
            const float f = M == -INFINITY ? (L != 0.f ? 1.f : 0.f) : __builtin_amdgcn_exp2f(M - mn);
            L *= f;
            acc *= f;
            M = mn;
#pragma unroll
            for (uint32_t k = 0; k < 8u; k++)
                if (ml[k][1] != 0.f) {
                    const float w = ml[k][0] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ml[k][0] - mn);
                    L += w * ml[k][1];
                    acc += w * v[k];
                }
        }
        s_acc[threadIdx.x] = acc;
        if (dl == 0u) {
            s_m[grp] = M;
            s_l[grp] = L;
        }
        __syncthreads();
        if (grp == 0u && d < a.hd) {
            M = -INFINITY;
#pragma unroll
            for (uint32_t k = 0; k < NG; k++)
                if (s_l[k] != 0.f) M = fmax2(M, s_m[k]);
            L = 0.f;
            acc = (f4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (uint32_t k = 0; k < NG; k++) {
                if (s_l[k] == 0.f) continue;
                const float w = s_m[k] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(s_m[k] - M);
                L += w * s_l[k];
                acc += w * s_acc[k * LPH + dl];
            }
            const float inv = L != 0.f ? 1.f / L : 0.f;
#pragma unroll
            for (uint32_t k = 0; k < 4u; k++) {
                float o = acc[k] * inv;
                if (a.gate) o *= q4kv_sigmoid(gt[k]);
                stg(a.out + ro + k, o);
            }
        }
        __syncthreads();
    }
}

/* The launches (q4kv_paged_rows.hip, q4kv_paged_tiles.hip): requests of
 * min_cols .. max_cols columns per KV head. */
bool q4kv_paged_rows_launch(int kind, const PagedArgs &a);
bool q4kv_paged_tiles_launch(int kind, const PagedArgs &a);

#endif
