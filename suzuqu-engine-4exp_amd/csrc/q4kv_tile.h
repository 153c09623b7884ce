/*
 * q4kv_tile.h -- lane arithmetic and LDS addressing that the kernels with
 * tiles of 128 columns (dense and paged prefill) share.
 */
#ifndef Q4KV_TILE_H
#define Q4KV_TILE_H
#include "q4kv_attn_item.h"

typedef short s4_t __attribute__((ext_vector_type(4)));
typedef float f2_t __attribute__((ext_vector_type(2)));

/* x, y -> two fp16, rounded to nearest (v_cvt_pk_f16_f32) */
__device__ static inline uint32_t pk(float x, float y) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2_t){x, y}, h2_t));
}
/* max of non-NaN operands, without fmaxf's canonicalisations */
__device__ static inline float max2(float a, float b) { return __builtin_amdgcn_fmed3f(a, b, INFINITY); }

__device__ static inline float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
/* Maximum and sum over the four lanes of a column (16 apart). */
__device__ static inline float col_max(float v) {
    v = max2(v, __shfl_xor(v, 16));
    return max2(v, __shfl_xor(v, 32));
}
__device__ static inline float col_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

/* Four biased bytes (w ^ 0x80..) -> 1024 + u in four fp16. */
__device__ static inline void biased_h4(uint32_t w, h2_t &lo, h2_t &hi) {
    w ^= 0x80808080u;
    lo = __builtin_bit_cast(h2_t, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u));
    hi = __builtin_bit_cast(h2_t, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u));
}

/* Byte offset of the 16-byte piece `pc` of V row p. The transposing read of
 * 16 dims takes 32 bytes of each of 8 rows per half wave: rows are rotated
 * by 32-byte windows (xor p mod 8 over 8 windows), which puts them on
 * distinct banks; the two pieces of a window trade places every 8 rows so
 * that the conversion's stores (16 rows of one piece) are conflict-free
 * too. A row of 128 bytes holds four windows, two rows cover the banks. */
template <uint32_t VS> __device__ static inline uint32_t vaddr(uint32_t p, uint32_t pc) {
    const uint32_t x = VS >= 256 ? p & 7u : (p >> 1) & 3u;
    return p * VS + (((pc >> 1) ^ x) << 5) + (((pc ^ (p >> 3)) & 1u) << 4);
}

#endif
