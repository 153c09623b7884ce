/*
 * q4kv_paged_attn.h -- what the paged attention kernels share: a launch's
 * arguments, requests, and the division of a ragged batch's work.
 *
 * The division. A request's new tokens times the query heads of a KV head are
 * columns, NC of them a tile; a tile streams the positions that its last
 * token sees. The lengths are on the device, so a launch has a fixed number
 * of workgroups and each finds its share itself: the costs of all tiles of
 * all requests, laid end to end, are cut into equal runs wherever the cuts
 * fall (but not within SNAP of a tile's ends), and a workgroup per KV head
 * walks each run. A batch of any mix of lengths fills the chip evenly, and a
 * tile is only cut where a run ends: at most one begins and one ends inside a
 * run, so two partial slots per workgroup hold all that a second launch
 * merges. The KV heads of a run are neighbours on one XCD and in step: their
 * rows of a position share cache lines (q8_0 rows of 272 bytes: 4.25 lines
 * for two heads together, 3 each apart).
 */
#ifndef Q4KV_PAGED_ATTN_H
#define Q4KV_PAGED_ATTN_H
#include <hip/hip_runtime.h>
#include <math.h>
#include <type_traits>

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
    uint32_t unit; /* of the costs: 2^unit positions */
    uint32_t runs; /* most runs of the division */
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

__device__ inline uint32_t uni(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }

/* A request's tiles of NC columns. A tile costs what it starts with and the
 * positions that its last token sees, in units of 2^unit positions that keep
 * all sums below 2^31; from the first tile to the last they grow evenly by
 * step / 256. (All of this is executed once per workgroup, from cold
 * instruction lines: with 64-bit sums, quotients in double and a square root
 * it took 20 KB of code and 3 us.) */
template <uint32_t NC, uint32_t START> struct Tiles {
    uint32_t n, cols, first, step;
    __device__ uint32_t before(uint32_t k) const {
        return k * first + (uint32_t)(((uint64_t)step * ((uint64_t)k * (k - 1u) / 2u)) >> 8);
    }
    __device__ uint32_t cost(uint32_t k) const { return before(k + 1u) - before(k); }
    __device__ static Tiles of(const PagedArgs &a, const Req &r) {
        Tiles t;
        t.cols = r.n_q * a.gqa;
        t.n = (t.cols + NC - 1u) / NC;
        if (t.cols < a.min_cols || t.cols > a.max_cols) t.n = 0u;
        t.first = t.step = 0u;
        if (t.n) {
            const uint32_t lo = seen_by(r, min((NC - 1u) / a.gqa, r.n_q - 1u)), hi = seen_by(r, r.n_q - 1u);
            t.first = max((START + lo) >> a.unit, 1u);
            if (t.n > 1u) t.step = (uint32_t)((float)(hi - lo) * 256.f / (float)(t.n - 1u)) >> a.unit;
        }
        return t;
    }
};

/* what the merge of a cut tile reads, one per workgroup: the tile that begins
 * in its run and does not end there, and the runs that it lies in */
struct Cut {
    uint32_t pieces, g, kh, tile;
    uint32_t t0, cols, unused[2]; /* the request's first token and columns */
};

template <uint32_t NC, uint32_t START, uint32_t SNAP, uint32_t MIN_RUN, uint32_t MAX_RUN, uint32_t NTHR> struct Share {
    static_assert(START <= SNAP && SNAP <= MIN_RUN, "a cut falls past a tile's start, and on a tile at most once");
    typedef Tiles<NC, START> T;
    uint32_t u, end;        /* what is left of the run */
    uint32_t each, more;    /* run g starts at g * each + min(g, more) */
    uint32_t g, n_g;
    uint32_t seq, kh, tile, x; /* where u is: x into the tile */
    Req req;
    T tiles;

    struct Lds {
        uint32_t wave[NTHR / 64], upto[NTHR];
        struct {
            uint32_t seq, before;
            Req req;
        } at[2];
    };

    /* the costs of requests i0 .. i0 + NTHR - 1: their sum; upto holds the
     * running sums, r this thread's request */
    __device__ static uint32_t scan(const PagedArgs &a, uint32_t i0, Lds &s, Req &r) {
        const uint32_t i = i0 + threadIdx.x, lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
        uint32_t c = 0u;
        if (i < a.n_seq) {
            r = req_of(a, i);
            const T t = T::of(a, r);
            if (t.n) c = t.before(t.n);
        }
#pragma unroll
        for (uint32_t d = 1; d < 64u; d *= 2u) {
            const uint32_t v = (uint32_t)__shfl_up((int)c, d);
            if (lane >= d) c += v;
        }
        __syncthreads();
        if (lane == 63u) s.wave[wave] = c;
        __syncthreads();
        uint32_t sum = 0u;
#pragma unroll
        for (uint32_t w = 0; w < NTHR / 64u; w++) {
            if (w == wave) c += sum;
            sum += s.wave[w];
        }
        s.upto[threadIdx.x] = c;
        return uni(sum);
    }

    __device__ uint32_t starts(uint32_t k) const { return k * each + min(k, more); }
    /* tile and x of cost v of the request in req and tiles */
    __device__ void place(uint32_t v) {
        uint32_t lo = 0u, hi = tiles.n;
        while (hi - lo > 1u) {
            const uint32_t mid = (lo + hi) / 2u;
            if (tiles.before(mid) <= v)
                lo = mid;
            else
                hi = mid;
        }
        tile = uni(lo);
        x = uni(v - tiles.before(lo));
    }
    __device__ void take(const PagedArgs &a, const Req &r) {
        req.t0 = uni(r.t0);
        req.n_q = uni(r.n_q);
        req.cap = a.stride * a.page.d;
        req.pos0 = (int64_t)((uint64_t)uni((uint32_t)((uint64_t)r.pos0 >> 32)) << 32 | uni((uint32_t)r.pos0));
        tiles = T::of(a, req);
        tiles.first = uni(tiles.first);
        tiles.step = uni(tiles.step);
    }

    /* Finds the run of workgroup blockIdx.x. False: nothing for this one. */
    __device__ bool find(const PagedArgs &a, Lds &s) {
        Req r = {};
        if (threadIdx.x < 2u) s.at[threadIdx.x] = {}; /* q_start that does not ascend finds no request */
        uint32_t all = scan(a, 0u, s, r);
        for (uint32_t i0 = NTHR; i0 < a.n_seq; i0 += NTHR) all += scan(a, i0, s, r);
        const uint32_t snap = max(SNAP >> a.unit, 1u);
        /* what is worth a run: more where there is more, so that the pieces of
         * one long request stay few (16-column tiles, one request: 1500
         * positions 22.1 us in runs of 256, 17.2 of 64; 20 thousand 24.0 of
         * 256, 32.4 of 96), and at least a short tile, which would follow
         * another one in its run (30 tokens of 16 heads 38.0 us, now 20.0) */
        const uint32_t least = max(min(max(MIN_RUN >> a.unit, all >> 6), MAX_RUN >> a.unit), snap);
        n_g = min(a.runs, max(uni(all / least), 1u));
        /* a run's KV heads on one XCD (workgroup L runs on XCD L mod 8), and
         * consecutive runs: tiles of a request share its rows in one L2 */
        const uint32_t per = (n_g + 7u) / 8u, at = uni((blockIdx.x >> 3) / a.n_kvh);
        kh = (blockIdx.x >> 3) - at * a.n_kvh;
        g = (blockIdx.x & 7u) * per + at;
        if (at >= per || g >= n_g || !all) return false;
        each = uni(all / n_g);
        more = all - each * n_g;
        const uint32_t v[2] = {starts(g), starts(g + 1u)};
        uint32_t base = 0u;
        for (uint32_t i0 = 0; i0 < a.n_seq; i0 += NTHR) {
            const uint32_t sum = a.n_seq > NTHR ? scan(a, i0, s, r) : all;
            __syncthreads();
            const uint32_t hi = base + s.upto[threadIdx.x], lo = threadIdx.x ? base + s.upto[threadIdx.x - 1u] : base;
#pragma unroll
            for (uint32_t k = 0; k < 2u; k++)
                if (lo <= v[k] && v[k] < hi) {
                    s.at[k].seq = i0 + threadIdx.x;
                    s.at[k].before = lo;
                    s.at[k].req = r;
                }
            base += sum;
            __syncthreads();
            if (v[1] < base) break;
        }
        /* cuts keep snap away from a tile's ends */
        end = all;
        for (uint32_t k = v[1] < all ? 2u : 1u; k-- > 0u;) {
            seq = uni(s.at[k].seq);
            take(a, s.at[k].req);
            place(v[k] - uni(s.at[k].before));
            const uint32_t c = tiles.cost(tile);
            u = x < snap ? v[k] - x : c - x < snap ? v[k] + (c - x) : v[k];
            if (k) end = u;
        }
        if (u >= end) return false;
        x += u - v[0];
        if (x == tiles.cost(tile)) {
            x = 0u;
            next(a);
        }
        return true;
    }
    /* the tile after this one */
    __device__ void next(const PagedArgs &a) {
        if (++tile < tiles.n) return;
        tile = 0u;
        do {
            if (++seq >= a.n_seq) { /* not reached: costs are left */
                end = u;
                return;
            }
            take(a, req_of(a, seq));
        } while (!tiles.n);
    }
    /* The part of the current tile that lies in the run: of its n_pass passes
     * the first and one past the last; whether the tile begins and ends here.
     * Both runs at a cut find the same pass for it. */
    __device__ void piece(const PagedArgs &a, uint32_t n_pass, uint32_t &p0, uint32_t &p1, bool &begins, bool &ends) const {
        const uint32_t c = tiles.cost(tile), x1 = min(c, x + (end - u)), s = START >> a.unit;
        auto pass = [&](uint32_t y) {
            return min(n_pass, (uint32_t)((float)(y - min(y, s)) / (float)(c - s) * (float)n_pass));
        };
        begins = x == 0u;
        ends = x1 == c;
        p0 = begins ? 0u : uni(pass(x));
        p1 = ends ? n_pass : uni(pass(x1));
    }
    /* in how many runs the tile lies that begins in this one */
    __device__ uint32_t pieces(const PagedArgs &a) const {
        const uint32_t te = u - x + tiles.cost(tile), v = te - 1u, long_ones = more * (each + 1u);
        /* the last run that starts at or before v, if not close enough to te to start there */
        uint32_t last = uni(v < long_ones ? v / (each + 1u) : more + (v - long_ones) / each);
        if (te - starts(last) < max(SNAP >> a.unit, 1u)) last--;
        return last - g + 1u;
    }
    __device__ void advance(const PagedArgs &a) {
        const uint32_t c = tiles.cost(tile), x1 = min(c, x + (end - u));
        u += x1 - x;
        x = 0u;
        if (u < end) next(a);
    }
};

/* The unit of the costs (Tiles): what the batch can cost at most, from the
 * sizes that the host knows, stays below 2^31. */
static inline uint32_t q4kv_paged_unit(const PagedArgs &a, uint32_t nc, uint32_t start) {
    const double tiles = (double)a.n_tok * a.gqa / nc + a.n_seq;
    double most = tiles * ((double)start + 2.0 + (double)a.stride * a.page.d);
    uint32_t unit = 0u;
    for (; most >= 1.8e9; most = 0.5 * most + tiles) unit++;
    return unit;
}

/* Runs for G workgroups that are resident at once, each XCD its share. The
 * launch has runs x n_kvh workgroups: at most G for up to PAGED_KVH KV heads. */
constexpr uint32_t PAGED_KVH = 32;
static inline uint32_t q4kv_paged_runs(uint32_t G, uint32_t n_kvh) { return 8u * (G / 8u / n_kvh ? G / 8u / n_kvh : 1u); }

/* A launch of G workgroups leaves G records of cut tiles, then two partial
 * slots for each (run g, KV head): 2 (g n_kvh + kh) + 1 for the tile that
 * begins in the run, the one before for the tile that it continues or ends. A
 * partial row: m, l, two unused, HD sums. */
constexpr uint32_t PAGED_PHEAD = 4;
constexpr size_t paged_part_floats(uint32_t G, uint32_t nc, uint32_t HD) {
    return (size_t)G * (sizeof(Cut) / 4u) + 2u * (size_t)G * nc * (HD + PAGED_PHEAD);
}

/* What a lane has merged of one row: four of its sums */
struct Merged {
    float M, L;
    f4_t acc;
    __device__ Merged() : M(-INFINITY), L(0.f), acc((f4_t){0.f, 0.f, 0.f, 0.f}) {}
    /* N pieces; one that saw nothing has l = 0, one with l = NaN (scores that
     * are not finite) takes part */
    template <int N> __device__ void add(const float (&m)[N], const float (&l)[N], const f4_t (&v)[N]) {
        float mn = M;
#pragma unroll
        for (int k = 0; k < N; k++)
            if (l[k] != 0.f) mn = fmax2(mn, m[k]);
        const float f = M == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(M - mn); /* M of nothing: L and acc are 0 */
        L *= f;
        acc *= f;
        M = mn;
#pragma unroll
        for (int k = 0; k < N; k++)
            if (l[k] != 0.f) {
                const float w = m[k] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[k] - mn);
                L += w * l[k];
                acc += w * v[k];
            }
    }
};

/* Merges the cut tiles, those that begin in the run of workgroup x of the
 * launch before: HD / 4 lanes of four dims each to a column. Few columns:
 * a workgroup per column, its lane groups take every NG-th piece.
 * Many: a lane group per column, which is most often of two pieces (43
 * requests with 3 chunks of 701 tokens: 134 MB of partials, gates and outputs
 * in 25 us, the memory's rate). */
template <int HD, uint32_t NC>
__global__ __launch_bounds__(256) static void paged_merge_k(PagedArgs a) {
    constexpr bool FEW = NC <= 32;
    constexpr uint32_t LPH = HD / 4, NG = 256 / LPH, ROW = HD + PAGED_PHEAD, N = FEW ? 8 : 2;
    __shared__ __attribute__((aligned(16))) f4_t s_acc[FEW ? 256 : 1];
    __shared__ float s_m[NG], s_l[NG];
    const uint32_t *const cw = (const uint32_t *)((const Cut *)a.part + blockIdx.x);
    const Cut cut = {ldg(cw), ldg(cw + 1), ldg(cw + 2), ldg(cw + 3), ldg(cw + 4), ldg(cw + 5), {}};
    if (!cut.pieces) return;
    const uint32_t grp = threadIdx.x / LPH, dl = threadIdx.x % LPH, d = 4u * dl;
    const float *const parts = a.part + gridDim.x * (sizeof(Cut) / 4u);
    for (uint32_t j = FEW ? blockIdx.y : blockIdx.y * NG + grp; j < NC && cut.tile * NC + j < cut.cols;
         j += gridDim.y * (FEW ? 1u : NG)) {
        const uint32_t col = cut.tile * NC + j, t = col / a.gqa;
        const size_t ro = ((size_t)(cut.t0 + t) * a.n_head + cut.kh * a.gqa + (col - t * a.gqa)) * a.hd + d;
        float gt[4] = {0.f, 0.f, 0.f, 0.f};
        if (a.gate && d < a.hd) {
#pragma unroll
            for (uint32_t k = 0; k < 4u; k++) gt[k] = ldg(a.gate + ro + k);
        }
        Merged s;
        auto take = [&](uint32_t s0, auto n) {
            constexpr uint32_t M = decltype(n)::value;
            float m[M], l[M];
            f4_t v[M];
#pragma unroll
            for (uint32_t k = 0; k < M; k++) {
                const uint32_t at = s0 + k * (FEW ? NG : 1u), i = min(at, cut.pieces - 1u);
                const float *p = parts + ((size_t)(2u * ((cut.g + i) * a.n_kvh + cut.kh) + (i ? 0u : 1u)) * NC + j) * ROW;
                const u2_t x = ldg((const u2_t *)p);
                m[k] = __uint_as_float(x[0]);
                l[k] = at < cut.pieces ? __uint_as_float(x[1]) : 0.f;
                v[k] = ldg((const f4_t *)(p + PAGED_PHEAD + d));
            }
            s.add(m, l, v);
        };
        /* eight pieces a trip where there are many; past the end the last one
         * is read again (64 requests of two to nine pieces: 38.0 us, 35.4 with
         * two) */
        if (FEW && cut.pieces <= 2u * NG) {
            take(grp, std::integral_constant<uint32_t, 2>());
        } else {
            for (uint32_t s0 = FEW ? grp : 0u; s0 < cut.pieces; s0 += N * (FEW ? NG : 1u))
                take(s0, std::integral_constant<uint32_t, N>());
        }
        if constexpr (FEW) {
            s_acc[threadIdx.x] = s.acc;
            if (dl == 0u) {
                s_m[grp] = s.M;
                s_l[grp] = s.L;
            }
            __syncthreads();
            if (grp == 0u) {
                float m[NG], l[NG];
                f4_t v[NG];
#pragma unroll
                for (uint32_t k = 0; k < NG; k++) {
                    m[k] = s_m[k];
                    l[k] = s_l[k];
                    v[k] = s_acc[k * LPH + dl];
                }
                s = Merged();
                s.add(m, l, v);
            }
            __syncthreads();
        }
        if ((FEW && grp) || d >= a.hd) continue;
        const float inv = s.L != 0.f ? 1.f / s.L : 0.f;
#pragma unroll
        for (uint32_t k = 0; k < 4u; k++) {
            float o = s.acc[k] * inv;
            if (a.gate) o *= q4kv_sigmoid(gt[k]);
            stg(a.out + ro + k, o);
        }
    }
}

/* The launches (q4kv_paged_rows.hip, q4kv_paged_tiles.hip): requests of
 * min_cols .. max_cols columns per KV head. */
bool q4kv_paged_rows_launch(int kind, const PagedArgs &a, uint32_t cols); /* tiles of 16 or 32 columns */
bool q4kv_paged_tiles_launch(int kind, const PagedArgs &a);

#endif
