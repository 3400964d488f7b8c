/* heads.h — a head's RMS norm and position rotation in one pass, as the kernels of
 * rope.hip and kv4.hip run them: EL neighbouring elements a lane, a head within one
 * wave.
 *
 * An element e of the turned part becomes (x_e C_e + x_p S_e) r, p the element it turns
 * with, r the norm's 1 / sqrt(mean x^2 + eps), C and S the cosine and the sine of the
 * pair (the sine with its sign) times the norm's weights of e and p: C and S are the
 * same for all heads of a token.
 *
 * The arithmetic is in T: 64 bits where the result is an f32 (a product of two f32 is
 * exact there, and no sum of squares overflows, so the one rounding that counts is the
 * last), f32 where it is a bf16: 2^-24 of the terms for each of 4 roundings in the turn,
 * 2 of the root and half of the sum's 9, with two terms of sqrt 2 of the head's largest
 * normed element together less than 2^-20 of it, beside a half step of 2^-8.
 * A head whose squares leave f32's range takes 64 bits. */
#pragma once

#include <hip/hip_runtime.h>

#include <math.h>

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

namespace {

/* EL neighbours as they lie in memory */
template <typename X, int EL> struct HeadRaw { uint32_t v[EL * sizeof(X) / 4]; };

template <int EL>
__device__ __forceinline__ void head_load(const float * p, HeadRaw<float, EL> & x) {
    const uint4 w = *(const uint4 *) p;
    x.v[0] = w.x; x.v[1] = w.y; x.v[2] = w.z; x.v[3] = w.w;
}
template <int EL>
__device__ __forceinline__ void head_load(const uint16_t * p, HeadRaw<uint16_t, EL> & x) {
    if constexpr (EL == 4) {
        const uint2 w = *(const uint2 *) p;
        x.v[0] = w.x; x.v[1] = w.y;
    } else {
        const uint4 w = *(const uint4 *) p;
        x.v[0] = w.x; x.v[1] = w.y; x.v[2] = w.z; x.v[3] = w.w;
    }
}

/* the element that e turns with, or e itself */
__device__ __forceinline__ int head_pair(int e, int half, int inter) {
    return e >= 2 * half ? e : (inter ? e ^ 1 : (e < half ? e + half : e - half));
}

/* one element's part in a turn: its norm's weight and its partner's, and where its
 * cosine and sine stand in a row of the table */
struct HeadFactor {
    float we, wp;
    int at;      /* -1: it does not turn */
    bool first;  /* of its pair */
};
/* w: the norm's weights, or null */
__device__ __forceinline__ HeadFactor head_factor(int e, int half, int inter, const float * w) {
    const int p = head_pair(e, half, inter);
    return {w ? w[e] : 1.0f, w ? w[p] : 1.0f, p == e ? -1 : (inter ? e >> 1 : min(e, p)), p > e};
}
template <typename T>
__device__ __forceinline__ void head_coef(const HeadFactor & f, float c, float s, T & C, T & S) {
    C = f.at < 0 ? (T) f.we : (T) c * (T) f.we;
    /* -0: with a partner of 0 it adds nothing, and keeps the sign of a zero */
    S = f.at < 0 ? (T) -0.0 : (T) (f.first ? -s : s) * (T) f.wp;
}

template <int EL>
__device__ __forceinline__ void head_widen(const HeadRaw<float, EL> & x, float * a) {
#pragma unroll
    for (int i = 0; i < EL; i++) a[i] = __uint_as_float(x.v[i]);
}
template <int EL>
__device__ __forceinline__ void head_widen(const HeadRaw<uint16_t, EL> & x, float * a) {
#pragma unroll
    for (int i = 0; i < EL / 2; i++) {
        a[2 * i] = __uint_as_float(x.v[i] << 16);
        a[2 * i + 1] = __uint_as_float(x.v[i] & 0xffff0000u);
    }
}

/* Elements e0 .. (in x) and those that they turn with as f32: a partner in another lane
 * is asked of that lane, or read from the row where halves are no whole pieces (vec 0).
 * Zeros where an element does not turn, and in a lane past the head. */
template <int EL, typename X>
__device__ __forceinline__ void head_wide(const HeadRaw<X, EL> & x, const X * row, int e0, int hd, int half, int inter, int vec,
                                          float * a, float * b) {
    head_widen<EL>(x, a);
#pragma unroll
    for (int i = 0; i < EL; i++) a[i] = e0 < hd ? a[i] : 0.0f;
    if (inter) {
#pragma unroll
        for (int i = 0; i < EL; i++) b[i] = a[i ^ 1];
    } else if (vec) {
        HeadRaw<X, EL> y;
        const int other = 4 * ((int) __lane_id() + (e0 < half ? half / EL : -(half / EL)));
#pragma unroll
        for (int i = 0; i < (int) (EL * sizeof(X) / 4); i++) y.v[i] = (uint32_t) __builtin_amdgcn_ds_bpermute(other, (int) x.v[i]);
        head_widen<EL>(y, b);
    } else {
#pragma unroll
        for (int i = 0; i < EL; i++) b[i] = e0 + i < 2 * half ? kv_load(row + head_pair(e0 + i, half, 0)) : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < EL; i++) b[i] = e0 + i < 2 * half ? b[i] : 0.0f;
}

template <int CTRL>
__device__ __forceinline__ float head_dpp(float v) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int CTRL>
__device__ __forceinline__ double head_dpp(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t) __builtin_amdgcn_mov_dpp((int) (uint32_t) u, CTRL, 0xf, 0xf, true);
    const uint32_t hi = (uint32_t) __builtin_amdgcn_mov_dpp((int) (u >> 32), CTRL, 0xf, 0xf, true);
    return __builtin_bit_cast(double, (uint64_t) hi << 32 | lo);
}

/* the sum over the 1 << sh lanes of a head, in each of them */
template <typename T>
__device__ __forceinline__ T head_sum(T v, int sh) {
    if (sh > 0) v += head_dpp<0xb1>(v);    /* lane ^ 1 */
    if (sh > 1) v += head_dpp<0x4e>(v);    /* lane ^ 2 */
    if (sh > 2) v += head_dpp<0x141>(v);   /* lane 7 - i of eight */
    if (sh > 3) v += head_dpp<0x140>(v);   /* lane 15 - i of sixteen */
    if (sh > 4) v += __shfl_xor(v, 16, 64);
    if (sh > 5) v += __shfl_xor(v, 32, 64);
    return v;
}

/* 1 / sqrt(mean x^2 + eps) of a head, for arithmetic in T; 1 without a norm */
template <int EL, typename T>
__device__ __forceinline__ double head_norm(const float * x, bool norm, float eps, double inv_hd, int sh) {
    if (!norm) return 1.0;
    if constexpr (sizeof(T) == 4) {
        /* a bf16's square is exact in f32 within its range */
        float s0 = x[0] * x[0], s1 = x[1] * x[1];
#pragma unroll
        for (int i = 2; i < EL; i += 2) {
            s0 = fmaf(x[i], x[i], s0);
            s1 = fmaf(x[i + 1], x[i + 1], s1);
        }
        const float ss = head_sum(s0 + s1, sh);
        if (!__any(!(ss > 0x1p-90f && ss < 0x1p120f)))
            return __builtin_amdgcn_rsq(fma((double) ss, inv_hd, (double) eps));   /* off by 2^-24 or so */
    }
    double ss = 0.0;
#pragma unroll
    for (int i = 0; i < EL; i++) ss = fma((double) x[i], (double) x[i], ss);
    const double a = fma(head_sum(ss, sh), inv_hd, (double) eps);
    /* two steps of Newton's iteration on the instruction's root */
    double r = __builtin_amdgcn_rsq(a);
#pragma unroll
    for (int k = 0; k < 2; k++) r = fma(0.5 * r, fma(-a * r, r, 1.0), r);
    return a < INFINITY ? r : 1.0 / sqrt(a);
}

/* x normed and turned, in T. In f32 x takes the norm's factor first, so that no product with
 * large or small weights leaves f32 where the result does not; a factor that could leave it
 * takes 64 bits */
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
        for (int i = 0; i < EL; i++) out[i] = fmaf(x[i] * rf, C[i], y[i] * rf * S[i]);
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
