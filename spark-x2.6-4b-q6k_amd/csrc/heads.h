/* heads.h — a head's RMS norm and position rotation in one pass, as the kernels of
 * rope.hip and kv4.hip run them: four neighbouring elements a lane, a head within
 * one wave.
 *
 * An element e of the turned part becomes y_e c + y_p s, p the element it turns
 * with, c and s the cosine and the sine of the pair (the sine with its sign), y the
 * normed values. Sums, norm and rotation are in 64 bits, rounded once, so that a
 * result does not depend on the order of a sum: a product of two f32 is exact there
 * and gfx950 runs f64 at f32's rate. p's value is read from memory again (it was
 * just fetched), which costs one load of cached data and serves any pairing. */
#pragma once

#include <hip/hip_runtime.h>

#include "kv.h"

namespace sparkmv {

constexpr int kHeadMax = 256;   /* elements of a head, at most: four a lane */

/* lanes of a head, as a shift: the smallest power of two of at least n / 4 */
inline int head_lane_shift(int n) {
    int s = 0;
    while ((4 << s) < n) s++;
    return s;
}

/* 0, or -1 with the message set; nrow: positions that the table has to cover */
int check_turn(const char * what, const sparkmv_head_turn * t, int head_dim, long nrow);

namespace {

struct HeadLane {
    int e0;             /* its first element */
    int pe[4];          /* the element that each one turns with, or itself */
    float c[4], s[4];   /* 1 and 0 where it does not turn */
    float w[4], pw[4];  /* the norm's weights of both */
};

__device__ __forceinline__ void head_load4(const float * p, float * x) {
    const float4 v = *(const float4 *) p;
    x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
}
__device__ __forceinline__ void head_load4(const uint16_t * p, float * x) {
    const uint2 v = *(const uint2 *) p;
    x[0] = __uint_as_float(v.x << 16); x[1] = __uint_as_float(v.x & 0xffff0000u);
    x[2] = __uint_as_float(v.y << 16); x[3] = __uint_as_float(v.y & 0xffff0000u);
}

/* which elements turn together: halves of the turned part, or neighbours */
__device__ __forceinline__ void head_pairs(HeadLane & h, int e0, int half, int inter) {
    h.e0 = e0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int e = e0 + i;
        h.pe[i] = e >= 2 * half ? e : (inter ? e ^ 1 : (e < half ? e + half : e - half));
    }
}

/* the cosines and sines of a row of the table (row null: nothing turns) */
__device__ __forceinline__ void head_angles(HeadLane & h, const float * row, int half, int inter) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int e = h.e0 + i;
        const bool turn = row && e < 2 * half;
        const int j = turn ? (inter ? e >> 1 : (e < half ? e : e - half)) : 0;
        h.c[i] = turn ? row[j] : 1.0f;
        const float s = turn ? row[half + j] : 0.0f;
        h.s[i] = h.pe[i] > e ? -s : s;
    }
}

__device__ __forceinline__ void head_weights(HeadLane & h, const float * w, int hd) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        h.w[i] = w ? w[min(h.e0 + i, hd - 1)] : 1.0f;
        h.pw[i] = w ? w[min(h.pe[i], hd - 1)] : 1.0f;
    }
}

/* the elements and those they turn with; a lane past the head gives zeros */
template <typename X>
__device__ __forceinline__ void head_fetch(const HeadLane & h, const X * row, int hd, int half, int inter, float * x, float * y) {
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = y[i] = 0.0f;
    if (h.e0 >= hd) return;
    head_load4(row + h.e0, x);
    if (inter) {
#pragma unroll
        for (int i = 0; i < 4; i++) y[i] = x[i ^ 1];
    } else if (half % 4 == 0) {
        if (h.e0 < 2 * half) head_load4(row + h.pe[0], y);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) y[i] = kv_load(row + h.pe[i]);
    }
}

/* x normed (norm) and turned, in 64 bits */
__device__ __forceinline__ void head_turn(const HeadLane & h, const float * x, const float * y, bool norm, float eps, int hd,
                                          int lanes, double * out) {
    double inv = 1.0;
    if (norm) {
        double ss = 0.0;
#pragma unroll
        for (int i = 0; i < 4; i++) ss += (double) x[i] * (double) x[i];
        for (int o = lanes >> 1; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
        inv = 1.0 / sqrt(ss / (double) hd + (double) eps);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        double a = (double) x[i], b = (double) y[i];
        if (norm) {
            a = a * inv * (double) h.w[i];
            b = b * inv * (double) h.pw[i];
        }
        out[i] = h.s[i] == 0.0f && h.pe[i] == h.e0 + i ? a : a * (double) h.c[i] + b * (double) h.s[i];
    }
}

}  // namespace

}  // namespace sparkmv
