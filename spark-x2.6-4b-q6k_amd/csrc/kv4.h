/* kv4.h — the paged 4-bit cache as its kernels see it. */
#pragma once

#include <hip/hip_runtime.h>

#include "kv.h"

namespace sparkmv {

constexpr int kKv4Low = 7;       /* scale bytes that an append writes: 2^-120 .. 2^125, or 255; */
constexpr int kKv4High = 252;    /* any above this one is not a number */

/* A page's kv head: codes of keys and of values (32 hd bytes each), scales of keys
 * and of values (2 hd bytes each). The codes lie as the lanes of the 16 x 16 x 32
 * matrix instruction take them once they are converted, a load of a wave being one
 * contiguous piece: lane 16 g + c holds
 *   keys of position 16 t + c: the elements of one block (head_dim 64: half of one),
 *     so one scale serves 16 bytes; which elements an instruction adds up is of no
 *     consequence as long as the queries lie alike;
 *   values of positions 32 u + 16 a + 4 g + b (the ones whose scores such a lane
 *     holds) and of head_dim / 16 neighbouring elements, all of one block, so that
 *     16 scales serve a page and the lane of an output has 4 head_dim / 16 in a row.
 * The even element of a pair is the low half of its byte. */
__host__ __device__ inline int kv4_head_bytes(int hd) { return 68 * hd; }
__host__ __device__ inline int kv4_key_at(int pos, int d, int hd) {
    const int t = pos >> 4, c = pos & 15;
    if (hd == 64) return ((t * 4 + (d >> 4)) * 16 + c) * 8 + (d & 15) / 2;
    const int b = d >> 5;
    return (((t * (hd >> 7) + (b >> 2)) * 4 + (b & 3)) * 16 + c) * 16 + (d & 31) / 2;
}
__host__ __device__ inline int kv4_value_at(int pos, int d, int hd) {
    const int sh = hd == 256 ? 4 : (hd == 128 ? 3 : 2), n = 1 << sh, c = d >> sh;
    const int byte = ((pos >> 4 & 1) * 4 + (pos & 3)) * (n / 2) + (d & (n - 1)) / 2;
    return 32 * hd + ((((pos >> 5) * (n / 4) + (byte >> 4)) * 4 + (pos >> 2 & 3)) * 16 + c) * 16 + (byte & 15);
}
__host__ __device__ inline int kv4_key_scale_at(int pos, int d, int hd) {
    const int t = pos >> 4, c = pos & 15, b = d >> 5;
    return 64 * hd + (hd == 64 ? (b * 16 + c) * 4 + t : (((b & 3) * 16 + c) * 4 + t) * (hd >> 7) + (b >> 2));
}
__host__ __device__ inline int kv4_value_scale_at(int pos, int d, int hd) {
    return 66 * hd + ((pos >> 2 & 3) * (hd >> 5) + (d >> 5)) * 16 + (pos >> 5) * 8 + (pos >> 4 & 1) * 4 + (pos & 3);
}

typedef __bf16 kv4_b8 __attribute__((ext_vector_type(8)));

/* byte B of four pairs of codes as bf16 with their scale, exactly (two significant
 * bits and a power of two). The instruction looks at a scale's exponent alone, so a
 * byte of scales needs no more than a shift to its place */
template <int B>
__device__ __forceinline__ uint32_t kv4_pair(uint32_t codes, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, B));
}
template <int B>
__device__ __forceinline__ float kv4_scale(uint32_t bytes) {
    return __uint_as_float(B == 3 ? bytes >> 1 : bytes << (23 - 8 * B));
}

int kv4_check_cache(const sparkmv_kv4_cache * c);

}  // namespace sparkmv
