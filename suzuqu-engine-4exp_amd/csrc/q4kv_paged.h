/*
 * q4kv_paged.h -- what the paged cache's translation units share.
 */
#ifndef Q4KV_PAGED_H
#define Q4KV_PAGED_H
#include <stdint.h>

#include "q4kv_internal.h"

extern "C" {
#include "q4kv.h"
}

constexpr uint32_t Q4KV_PAGED_SEQS = 65536; /* most requests of a step */

/* p / d for 0 <= p < 2^31 and any d >= 1: with L = ceil(log2 d), m = ceil(2^(31
 * + L) / d) is below 2^32 and its excess over the quotient below d <= 2^L, so
 * p * excess < 2^(31 + L) never reaches the next whole number. */
struct PageDiv {
    uint32_t d, m, sh;
};
static inline PageDiv q4kv_page_div(uint32_t d) {
    uint32_t L = 0;
    while (L < 31u && (1u << L) < d) L++;
    return PageDiv{d, (uint32_t)(((1ull << (31u + L)) + d - 1u) / d), 31u + L};
}
__host__ __device__ static inline uint32_t q4kv_page_of(const PageDiv &v, uint32_t p) {
    return (uint32_t)(((uint64_t)p * v.m) >> v.sh);
}

/* Whether a batch's sizes are sound: slots and positions fit 31 bits. */
static inline bool q4kv_pages_ok(uint32_t n_seq, uint32_t table_stride, uint32_t page,
                                 uint32_t n_pages) {
    return n_seq && n_seq <= Q4KV_PAGED_SEQS && table_stride && page && n_pages &&
           (uint64_t)table_stride * page <= 0x7fffffffull && (uint64_t)n_pages * page <= 0x7fffffffull;
}
static inline bool q4kv_batch_ok(const q4kv_paged_batch *b) {
    return b && b->table && b->kv_len && q4kv_pages_ok(b->n_seq, b->table_stride, b->page, b->n_pages);
}

#endif
