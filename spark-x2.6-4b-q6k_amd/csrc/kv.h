/* kv.h — the paged 8-bit cache as its kernels see it, and the launchers that
 * the model's paged step shares with the entry points. */
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/sparkmv.h"
#include "common.h"

namespace sparkmv {

constexpr int kKvPage = SPARKMV_KV_PAGE;
constexpr int kKvMaxSeq = 4096;      /* sequences of one call */
constexpr int kKvMaxGroup = 16;      /* query heads per kv head */
constexpr long kKvThreads = 0xffffffffl;   /* threads of a launch along one axis */

/* A page's codes of one kv head. Keys: [head_dim / 64][position][64 bytes], so
 * that a wave's 16-byte loads of 16 positions (lane = position + 16 * quarter)
 * are one contiguous kilobyte. Values: [g][head_dim][t][i] for position
 * 16 t + 4 g + i, so that 16 bytes of one element hold the positions whose
 * scores one lane group of a 16 x 16 score tile holds (rows 4 g + i of tiles
 * t = 0..3): the product with the weights then needs no exchange of lanes. */
__host__ __device__ inline int kv_key_at(int pos, int d) { return (d >> 6) * (kKvPage * 64) + pos * 64 + (d & 63); }
__host__ __device__ inline int kv_value_at(int pos, int d, int hd) {
    return (((pos >> 2 & 3) * hd + d) * 4 + (pos >> 4)) * 4 + (pos & 3);
}

/* One sequence of a batch as a kernel reads it: its slot, the position of its
 * first new token and its rows of the call's tokens. count is 0 for a
 * sequence that the call leaves out: a negative position, a slot outside the
 * table, rows outside the call's, or that end before they begin. Tokens past max_q
 * are left out, and so are positions past the page table. */
struct KvSeq {
    int slot, pos, row, count;
};

__device__ __forceinline__ KvSeq kv_seq(const sparkmv_kv_batch & b, int i, int nslots, int max_pages) {
    KvSeq s;
    s.slot = b.slot ? b.slot[i] : i;
    s.pos = b.pos[i];
    s.row = b.qstart ? b.qstart[i] : i;
    int end = b.qstart ? b.qstart[i + 1] : i + 1;
    /* the last test keeps the difference below from wrapping */
    if (s.slot < 0 || s.slot >= nslots || s.pos < 0 || s.row < 0 || end > b.ntok || end < s.row) end = s.row;
    s.count = max(0, min(min(end - s.row, b.max_q), max_pages * kKvPage - s.pos));
    return s;
}

__device__ __forceinline__ float kv_load(const float * p) { return *p; }
__device__ __forceinline__ float kv_load(const uint16_t * p) { return __uint_as_float((uint32_t) *p << 16); }
/* to nearest even, a NaN stays one: one instruction for two (in integer
 * arithmetic fourteen, which a call that runs them once also has to fetch) */
__device__ __forceinline__ uint32_t kv_bf16x2(float a, float b) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{a, b}), b2));
}
__device__ __forceinline__ uint16_t kv_bf16(float f) { return (uint16_t) kv_bf16x2(f, f); }

/* the host's checks: 0, or -1 with the message set. kv_check_rows: nrows rows of
 * n values at stride ld, each starting 16-byte aligned */
bool kv_aligned(const void * p, size_t n);
int kv_check_dtype(const char * what, int dtype);
int kv_check_rows(const char * what, const void * p, int ld, long n, int dtype, int nrows);
int kv_check_cache(const sparkmv_kv_cache * c);
int kv_check_batch(const sparkmv_kv_batch * b);
int kv_check_launch(const char * what);

}  // namespace sparkmv
