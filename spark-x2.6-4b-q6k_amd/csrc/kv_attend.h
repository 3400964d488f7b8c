/* kv_attend.h — what the attention kernels over the paged caches share: the pages
 * that a sequence's tokens see, exchanges within a wave, writing a row out, finding
 * a tile of the batch and joining the partial results of a column. */
#pragma once

#include <hip/hip_runtime.h>

#include <math.h>

#include "kv.h"

namespace sparkmv {

namespace {

constexpr float kKvLag = 16.0f;
constexpr float kKvLog2e = 1.44269504088896340736f;

typedef int kv_i4 __attribute__((ext_vector_type(4)));
typedef float kv_f4 __attribute__((ext_vector_type(4)));

/* the pages that tokens t0 .. t1 - 1 of a sequence see: the first and how many */
__device__ __forceinline__ int kv_span(const KvSeq & s, int t0, int t1, int window, int & first) {
    const int p = s.pos + t0;
    first = (window > 0 && p + 1 > window ? p + 1 - window : 0) / kKvPage;
    return (s.pos + t1 - 1) / kKvPage - first + 1;
}

template <int CTRL>
__device__ __forceinline__ int kv_quad(int v) { return __builtin_amdgcn_mov_dpp(v, CTRL, 0xf, 0xf, true); }
template <int CTRL>
__device__ __forceinline__ float kv_quad(float v) { return __int_as_float(kv_quad<CTRL>(__float_as_int(v))); }
constexpr int kKvXor1 = 0xb1, kKvXor2 = 0x4e;   /* quad permutations: lanes 1 0 3 2, 2 3 0 1 */

/* the largest of a wave, in each lane */
__device__ __forceinline__ uint32_t kv_wave_max(uint32_t v) {
    v = max(v, (uint32_t) kv_quad<kKvXor1>((int) v));
    v = max(v, (uint32_t) kv_quad<kKvXor2>((int) v));
    v = max(v, (uint32_t) kv_quad<0x141>((int) v));   /* lane 7 - i of eight */
    v = max(v, (uint32_t) kv_quad<0x140>((int) v));   /* lane 15 - i of sixteen */
    auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max((uint32_t) a[0], (uint32_t) a[1]);
    a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return max((uint32_t) a[0], (uint32_t) a[1]);
}

/* the largest, or the sum, of the four lanes 16 apart, in each of them */
__device__ __forceinline__ float kv_rows_max(float v) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float kv_rows_sum(float v) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

/* out[row][head][d ..] = o / l, gated, N neighbours; no weight at all gives 0 */
template <int N>
__device__ __forceinline__ void kv_write(const sparkmv_kv_query & q, int row, int head, int hd, int d, const float * o, float l) {
    typedef float fn __attribute__((ext_vector_type(N)));
    float f = l == 0.0f ? 0.0f : 1.0f / l;
    if (q.gate) f *= 1.0f / (1.0f + expf(-q.gate[(size_t) row * q.ldg + head]));
    const size_t at = (size_t) row * q.ldo + (size_t) head * hd + d;
    fn v;
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = l == 0.0f ? 0.0f : o[i] * f;
    if (q.out_dtype == SPARKMV_X_F32) {
        *(fn *) ((float *) q.out + at) = v;
    } else {
        if constexpr (N == 1) {
            ((uint16_t *) q.out)[at] = kv_bf16(v[0]);
        } else {
            typedef uint32_t un __attribute__((ext_vector_type(N / 2)));
            un w;
#pragma unroll
            for (int i = 0; i < N / 2; i++) w[i] = kv_bf16x2(v[2 * i], v[2 * i + 1]);
            *(un *) ((uint16_t *) q.out + at) = w;
        }
    }
}

/* The join of one column's n partials by W waves: weights e^(m - M) in LDS, then
 * each wave adds every W-th row with eight of them in flight, and the waves' sums
 * add up in order. at(k) is the k-th partial's index. Returns the sum of weights;
 * o has this lane's HD / 64 elements, complete in wave 0. */
template <int HD, int W, class At>
__device__ __forceinline__ float kv_join(const float * po, const float * pml, int n, At at, float * wts, float * acc, int wave,
                                         int lane, float (&o)[HD / 64]) {
    constexpr int E = HD / 64;
    typedef float fe __attribute__((ext_vector_type(E)));
    /* the first results are requested before their weights are known (joining 128 of
     * each of 16 columns of 256: 6.7 us, now 5.9) */
    fe v[8];
    auto load = [&](int k0) {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = *(const fe *) (po + at(min(k0 + W * j, n - 1)) * HD + E * lane);
    };
    constexpr int C = 2;
    float2 ml[C];
#pragma unroll
    for (int c = 0; c < C; c++) ml[c] = *(const float2 *) (pml + 2 * at(min(lane + 64 * c, n - 1)));
    load(wave);
    float M = fmaxf(ml[0].x, ml[1].x);
    for (int k = lane + 64 * C; k < n; k += 64) M = fmaxf(M, pml[2 * at(k)]);
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) M = fmaxf(M, __shfl_xor(M, s, 64));
    float L = 0.0f;
    auto take = [&](int k, float m, float l) {
        const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - M);
        L += m == -INFINITY ? l : f * l;
        if (wave == 0) wts[k] = f;
    };
#pragma unroll
    for (int c = 0; c < C; c++)
        if (lane + 64 * c < n) take(lane + 64 * c, ml[c].x, ml[c].y);
    for (int k = lane + 64 * C; k < n; k += 64) take(k, pml[2 * at(k)], pml[2 * at(k) + 1]);
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) L += __shfl_xor(L, s, 64);
    __syncthreads();
    fe sum = (fe) 0.0f;
    for (int k0 = wave; k0 < n; k0 += 8 * W) {
        if (k0 > wave) load(k0);
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (k0 + W * j < n) sum += wts[k0 + W * j] * v[j];
    }
    if (wave) *(fe *) (acc + (wave - 1) * HD + E * lane) = sum;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < W - 1; j++) sum += *(const fe *) (acc + j * HD + E * lane);
#pragma unroll
    for (int e = 0; e < E; e++) o[e] = sum[e];
    return L;
}

/* tile number `tile` of the batch, tiles of `cols` columns: its sequence and its
 * place there, a sequence's last (longest) first: the other way 4096 tokens from
 * position 0 took 278 us, not 238; false past the last one. Every thread of the workgroup calls it. */
template <typename Cache>
__device__ __forceinline__ bool kv_find_tile(const sparkmv_kv_batch & b, const Cache & c, int G, int cols, int tile,
                                             int * lds, KvSeq & s, int & place) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, nw = blockDim.x >> 6;
    if (tid == 0) lds[0] = -1;
    int before = 0;
    for (int i0 = 0; i0 < b.nseq; i0 += blockDim.x) {
        KvSeq mine = {0, 0, 0, 0};
        if (i0 + tid < b.nseq) mine = kv_seq(b, i0 + tid, c.nslots, c.max_pages);
        const int n = (int) (((long) mine.count * G + cols - 1) / cols);
        int scan = n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(scan, o, 64);
            if (lane >= o) scan += v;
        }
        __syncthreads();
        if (lane == 63) lds[2 + wave] = scan;
        __syncthreads();
        int at = before + scan - n;
        for (int w = 0; w < nw; w++) {
            if (w < wave) at += lds[2 + w];
            before += lds[2 + w];
        }
        if (tile >= at && tile < at + n) {
            lds[0] = i0 + tid;
            lds[1] = n - 1 - (tile - at);
        }
        if (tile < before) break;
    }
    __syncthreads();
    if (lds[0] < 0) return false;
    s = kv_seq(b, lds[0], c.nslots, c.max_pages);
    place = lds[1];
    return true;
}

}  // namespace

}  // namespace sparkmv
