/* heads.h — a head's RMS norm and position rotation in one pass, as the kernels of
 * rope.hip and kv4.hip run them: EL neighbouring elements a lane, a head within one
 * wave.
 *
 * An element e of the turned part becomes (x_e C_e + x_p S_e) r, p the element it turns
 * with, r the norm's 1 / sqrt(mean x^2 + eps), C and S the cosine and the sine of the
 * pair (the sine with its sign) times the norm's weights of e and p: C and S are the
 * same for all heads of a token. p's value is read from memory again (it was just
 * fetched), which costs one load of cached data and serves any pairing.
 *
 * The sum of squares and its root are in 64 bits, which no f32 overflows. The rest is in
 * T: 64 bits where the result is an f32 (a product of two f32 is exact there, so the
 * one rounding that counts is the last), f32 where it is a bf16, 2^-21 of the terms
 * beside its half step of 2^-8. */
#pragma once

#include <hip/hip_runtime.h>

#include "kv.h"

namespace sparkmv {

constexpr int kHeadMax = 256;   /* elements of a head, at most */

/* lanes of a head, as a shift: the smallest power of two of at least n / el */
inline int head_lane_shift(int n, int el) {
    int s = 0;
    while ((el << s) < n) s++;
    return s;
}

/* 0, or -1 with the message set; nrow: positions that the table has to cover */
int check_turn(const char * what, const sparkmv_head_turn * t, int head_dim, long nrow);

/* what a launch knows of the alignment of a turn's arrays, for EL elements a lane */
struct HeadVec {
    int table, weights;   /* their pieces can be loaded whole */
};
inline HeadVec head_vec(const sparkmv_head_turn & t, int el) {
    HeadVec v;
    const int half = t.rope_dim / 2;
    v.table = ((uintptr_t) t.rope & 15) == 0 && half % 4 == 0 && (t.interleaved ? t.rope_dim : half) % el == 0;
    v.weights = (((uintptr_t) t.q_norm | (uintptr_t) t.k_norm) & 15) == 0;
    return v;
}

namespace {

template <int N>
__device__ __forceinline__ void head_load(const float * p, float * x) {
    if constexpr (N == 2) {
        const float2 v = *(const float2 *) p;
        x[0] = v.x; x[1] = v.y;
    } else {
#pragma unroll
        for (int k = 0; k < N; k += 4) {
            const float4 v = *(const float4 *) (p + k);
            x[k] = v.x; x[k + 1] = v.y; x[k + 2] = v.z; x[k + 3] = v.w;
        }
    }
}
template <int N>
__device__ __forceinline__ void head_load(const uint16_t * p, float * x) {
    uint32_t v[N / 2];
    if constexpr (N == 4) {
        const uint2 w = *(const uint2 *) p;
        v[0] = w.x; v[1] = w.y;
    } else {
        const uint4 w = *(const uint4 *) p;
        v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
    }
#pragma unroll
    for (int k = 0; k < N / 2; k++) {
        x[2 * k] = __uint_as_float(v[k] << 16);
        x[2 * k + 1] = __uint_as_float(v[k] & 0xffff0000u);
    }
}

/* the element that e turns with, or e itself */
__device__ __forceinline__ int head_pair(int e, int half, int inter) {
    return e >= 2 * half ? e : (inter ? e ^ 1 : (e < half ? e + half : e - half));
}

/* C and S of elements e0 .. of a head of hd. row: the token's row of the table (half
 * 0: nothing turns); w: the norm's weights, or null */
template <int EL, typename T>
__device__ __forceinline__ void head_coef(T * C, T * S, int e0, int hd, const float * row, int half, int inter, const float * w,
                                          const HeadVec & vec) {
    float c[EL], s[EL], we[EL], wp[EL];
#pragma unroll
    for (int i = 0; i < EL; i++) {
        c[i] = we[i] = wp[i] = 1.0f;
        s[i] = -0.0f;   /* with y = 0: adds nothing, and keeps the sign of a zero */
    }
    if (e0 < hd && w) {
        if (vec.weights) head_load<EL>(w + e0, we);
        else
#pragma unroll
            for (int i = 0; i < EL; i++) we[i] = w[min(e0 + i, hd - 1)];
    }
    if (e0 < 2 * half) {
        if (vec.table) {   /* all of the lane's elements turn */
            if (inter) {
                float a[EL / 2], b[EL / 2];
                head_load<EL / 2>(row + e0 / 2, a);
                head_load<EL / 2>(row + half + e0 / 2, b);
#pragma unroll
                for (int i = 0; i < EL; i++) {
                    c[i] = a[i / 2];
                    s[i] = i & 1 ? b[i / 2] : -b[i / 2];
                    wp[i] = we[i ^ 1];
                }
            } else {
                const bool up = e0 >= half;
                head_load<EL>(row + (up ? e0 - half : e0), c);
                head_load<EL>(row + half + (up ? e0 - half : e0), s);
                if (w) {
                    const float * q = w + (up ? e0 - half : e0 + half);
                    if (vec.weights) head_load<EL>(q, wp);
                    else
#pragma unroll
                        for (int i = 0; i < EL; i++) wp[i] = q[i];
                }
#pragma unroll
                for (int i = 0; i < EL; i++) s[i] = up ? s[i] : -s[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < EL; i++) {
                const int e = e0 + i, p = head_pair(e, half, inter);
                if (p == e) continue;
                const int j = inter ? e >> 1 : (e < half ? e : e - half);
                c[i] = row[j];
                s[i] = p > e ? -row[half + j] : row[half + j];
                if (w) wp[i] = w[p];
            }
        }
    }
#pragma unroll
    for (int i = 0; i < EL; i++) {
        C[i] = (T) c[i] * (T) we[i];
        S[i] = (T) s[i] * (T) wp[i];
    }
}

/* the elements and those they turn with (0 where they do not); a lane past the head gives zeros */
template <int EL, typename X>
__device__ __forceinline__ void head_fetch(const X * row, int e0, int hd, int half, int inter, const HeadVec & vec, float * x, float * y) {
#pragma unroll
    for (int i = 0; i < EL; i++) x[i] = y[i] = 0.0f;
    if (e0 >= hd) return;
    head_load<EL>(row + e0, x);
    if (e0 >= 2 * half) return;
    if (inter) {
#pragma unroll
        for (int i = 0; i < EL; i++) y[i] = e0 + i < 2 * half ? x[i ^ 1] : 0.0f;
    } else if (vec.table) {
        head_load<EL>(row + (e0 >= half ? e0 - half : e0 + half), y);
    } else {
#pragma unroll
        for (int i = 0; i < EL; i++) {
            const int p = head_pair(e0 + i, half, 0);
            if (p != e0 + i) y[i] = kv_load(row + p);
        }
    }
}

template <int CTRL>
__device__ __forceinline__ double head_dpp(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t) __builtin_amdgcn_mov_dpp((int) (uint32_t) u, CTRL, 0xf, 0xf, true);
    const uint32_t hi = (uint32_t) __builtin_amdgcn_mov_dpp((int) (u >> 32), CTRL, 0xf, 0xf, true);
    return __builtin_bit_cast(double, (uint64_t) hi << 32 | lo);
}

/* the sum over the 1 << sh lanes of a head, in each of them */
__device__ __forceinline__ double head_sum(double v, int sh) {
    if (sh > 0) v += head_dpp<0xb1>(v);    /* lane ^ 1 */
    if (sh > 1) v += head_dpp<0x4e>(v);    /* lane ^ 2 */
    if (sh > 2) v += head_dpp<0x141>(v);   /* lane 7 - i of eight */
    if (sh > 3) v += head_dpp<0x140>(v);   /* lane 15 - i of sixteen */
    if (sh > 4) v += __shfl_xor(v, 16, 64);
    if (sh > 5) v += __shfl_xor(v, 32, 64);
    return v;
}

/* 1 / sqrt(mean x^2 + eps) of a head; 1 without a norm */
template <int EL>
__device__ __forceinline__ double head_norm(const float * x, bool norm, float eps, double inv_hd, int sh) {
    if (!norm) return 1.0;
    double ss = 0.0;
#pragma unroll
    for (int i = 0; i < EL; i++) ss = fma((double) x[i], (double) x[i], ss);
    const double a = fma(head_sum(ss, sh), inv_hd, (double) eps);
    /* the instruction is good to 2^-26 or so; two steps of Newton's iteration */
    double r = __builtin_amdgcn_rsq(a);
#pragma unroll
    for (int k = 0; k < 2; k++) r = fma(0.5 * r, fma(-a * r, r, 1.0), r);
    return a < INFINITY ? r : 1.0 / sqrt(a);
}

/* x normed and turned, in T; with f32, where that could leave its range, in 64 bits */
template <int EL>
__device__ __forceinline__ void head_turn(const double * C, const double * S, const float * x, const float * y, double r, double * out) {
#pragma unroll
    for (int i = 0; i < EL; i++) out[i] = fma((double) x[i], C[i], (double) y[i] * S[i]) * r;
}
template <int EL>
__device__ __forceinline__ void head_turn(const float * C, const float * S, const float * x, const float * y, double r, float * out) {
    if (__any(!(r > 0x1p-60 && r < 0x1p60))) {
#pragma unroll
        for (int i = 0; i < EL; i++) out[i] = (float) (fma((double) x[i], (double) C[i], (double) y[i] * (double) S[i]) * r);
    } else {
        const float rf = (float) r;
#pragma unroll
        for (int i = 0; i < EL; i++) out[i] = fmaf(x[i], C[i], y[i] * S[i]) * rf;
    }
}

/* EL neighbours, aligned to them (to 16 bytes) */
template <int EL>
__device__ __forceinline__ void head_store(float * p, const double * v) {
#pragma unroll
    for (int k = 0; k < EL; k += 4) *(float4 *) (p + k) = float4{(float) v[k], (float) v[k + 1], (float) v[k + 2], (float) v[k + 3]};
}
template <int EL>
__device__ __forceinline__ void head_store(uint16_t * p, const float * v) {
    if constexpr (EL == 4) *(uint2 *) p = uint2{kv_bf16x2(v[0], v[1]), kv_bf16x2(v[2], v[3])};
    else *(uint4 *) p = uint4{kv_bf16x2(v[0], v[1]), kv_bf16x2(v[2], v[3]), kv_bf16x2(v[4], v[5]), kv_bf16x2(v[6], v[7])};
}

/* the arithmetic of an output's type */
template <typename X> struct HeadArith { typedef double T; };
template <> struct HeadArith<uint16_t> { typedef float T; };

}  // namespace

}  // namespace sparkmv
