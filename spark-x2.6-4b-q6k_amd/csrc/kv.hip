/* kv.hip — the paged 8-bit cache: the append with the position rotation on the
 * way, reading positions back, and attention over it (include/sparkmv.h has
 * the cache's layout and its rules; kv.h the offsets of a code). */
#include "kv.h"

#include <math.h>

namespace sparkmv {

namespace {

__device__ __forceinline__ float kv_load(const float * p) { return *p; }
__device__ __forceinline__ float kv_load(const uint16_t * p) { return __uint_as_float((uint32_t) *p << 16); }
__device__ __forceinline__ uint16_t kv_bf16(float f) {
    uint32_t u = __float_as_uint(f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t) ((u >> 16) | 0x40u);
    return (uint16_t) ((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}
__device__ __forceinline__ void kv_store(float * p, float v) { *p = v; }
__device__ __forceinline__ void kv_store(uint16_t * p, float v) { *p = kv_bf16(v); }

/* 64 bits to bf16 with one rounding: to f32 toward zero with the lost bits kept
 * in the last one (an odd value cannot lie between two bf16 values), then to
 * nearest even */
__device__ __forceinline__ void kv_store_wide(float * p, double v) { *p = (float) v; }
__device__ __forceinline__ void kv_store_wide(uint16_t * p, double v) {
    const float f = (float) v;
    uint32_t u = __float_as_uint(f);
    const double back = (double) f;
    if (back != v && __builtin_isfinite(f)) {
        if (fabs(back) > fabs(v)) u--;   /* rounded away from zero: step back */
        u |= 1u;
    }
    *p = kv_bf16(__uint_as_float(u));
}

/* ---------------------------------------------------------------- rope table */

__global__ __launch_bounds__(256) void kv_rope_table_kernel(float * tab, int rows, int half, float theta) {
    const size_t i = (size_t) blockIdx.x * 256 + threadIdx.x;
    if (i >= (size_t) rows * half) return;
    const int pos = (int) (i / half), j = (int) (i - (size_t) pos * half);
    const float freq = 1.0f / powf(theta, (float) (2 * j) / (float) (2 * half));
    const float a = (float) pos * freq;
    float * r = tab + (size_t) pos * 2 * half;
    r[j] = cosf(a);
    r[half + j] = sinf(a);
}

/* -------------------------------------------------------------------- append
 *
 * Workgroups 0 .. nkv - 1 take one (sequence, touched page, kv head, keys or
 * values) each, the others four query heads of one token.
 *
 * A page's workgroup turns the new rows into f32 in LDS (at most 64 x hd),
 * takes their largest magnitude, settles the scale, and writes the codes in 16
 * byte pieces of the layout; pieces that also hold older positions are read
 * first. Nothing else writes the page's head during the launch.
 *
 * The arithmetic is fixed to the bit, so that a code does not depend on how a
 * compiler orders a sum: the rotation in 64 bits (products of f32 are exact
 * there), the scale from 64 bits, the code as the nearest integer of the exact
 * quotient. That one is found in f32: n0 = rint(x * (1 / s)) is off by one at
 * most, and x - s n0, one fma, is exact (its bits lie between the last place
 * of s or x and s), so comparing it with s / 2 settles the rounding. */
struct KvAppend {
    sparkmv_kv_cache c;
    sparkmv_kv_batch b;
    sparkmv_kv_new n;
    int nb;          /* pages a sequence's new tokens may touch */
    int nkv;         /* workgroups of pages */
    int qparts;      /* workgroups of one token's queries */
    int half;
};

/* element pair j of a head: (j, j + half) turned, or two elements past them */
__device__ __forceinline__ int kv_pair(int j, int half, int & second) {
    if (j < half) {
        second = j + half;
        return j;
    }
    second = 2 * j + 1;
    return 2 * j;
}

template <typename X>
__device__ __forceinline__ void kv_turn(const X * row, int e0, int e1, const float * rope, int j, int half, double & a,
                                        double & b) {
    a = (double) kv_load(row + e0);
    b = (double) kv_load(row + e1);
    if (j < half && rope) {
        const double c = (double) rope[j], s = (double) rope[half + j], x = a;
        a = x * c - b * s;
        b = b * c + x * s;
    }
}

/* nearest integer of x / s (ties to even), |x / s| <= 127.5 */
__device__ __forceinline__ float kv_code(float x, float s, float r, bool tiny) {
    if (tiny) return (float) rint((double) x / (double) s);
    float n = rintf(x * r);
    const float e = fmaf(-s, n, x), e2 = 2.0f * fabsf(e);
    if (e2 > s || (e2 == s && ((int) n & 1))) n += e > 0.0f ? 1.0f : -1.0f;
    return n;
}

template <typename X>
__global__ __launch_bounds__(256) void kv_append_kernel(const KvAppend A) {
    extern __shared__ __attribute__((aligned(16))) float lrow[];   /* [rows][hd] */
    __shared__ uint32_t lmax[4];
    const int tid = threadIdx.x, hd = A.c.head_dim, kvh = A.c.kv_heads, half = A.half;
    if ((int) blockIdx.x >= A.nkv) {
        /* queries */
        const int w = (int) blockIdx.x - A.nkv, t = w / A.qparts, h0 = 4 * (w - t * A.qparts);
        __shared__ int lpos;
        if (tid == 0) lpos = -1;
        __syncthreads();
        for (int i = tid; i < A.b.nseq; i += 256) {
            const KvSeq s = kv_seq(A.b, i, A.c.nslots, A.c.max_pages);
            if (t >= s.row && t - s.row < s.count) lpos = s.pos + t - s.row;
        }
        __syncthreads();
        const int pos = lpos;
        if (pos < 0) return;
        const float * rope = half ? A.n.rope + (size_t) pos * 2 * half : nullptr;
        const X * src = (const X *) A.n.q + (size_t) t * A.n.ldq;
        X * dst = (X *) A.n.q_out + (size_t) t * A.n.ldqo;
        const int pairs = hd / 2, n = min(4, A.n.heads - h0) * pairs;
        for (int i = tid; i < n; i += 256) {
            const int h = h0 + i / pairs, j = i % pairs;
            int e1;
            const int e0 = kv_pair(j, half, e1);
            double a, b;
            kv_turn(src + (size_t) h * hd, e0, e1, rope, j, half, a, b);
            kv_store_wide(dst + (size_t) h * hd + e0, a);
            kv_store_wide(dst + (size_t) h * hd + e1, b);
        }
        return;
    }
    int w = blockIdx.x;
    const int which = w & 1;
    w >>= 1;
    const int h = w % kvh;
    w /= kvh;
    const int i = w / A.nb;
    const KvSeq s = kv_seq(A.b, i, A.c.nslots, A.c.max_pages);
    if (s.count <= 0) return;
    const int blk = s.pos / kKvPage + (w - i * A.nb), p0 = blk * kKvPage, end = s.pos + s.count;
    if (p0 >= end) return;
    const int page = A.c.pages[(size_t) s.slot * A.c.max_pages + blk];
    if (page < 0 || page >= A.c.npages) return;
    const int lo = max(s.pos, p0), hi = min(end, p0 + kKvPage), held = lo - p0, rows = hi - lo;
    const X * src = (const X *) (which ? A.n.v : A.n.k);
    const int ld = which ? A.n.ldv : A.n.ldk;
    float * scale = (which ? A.c.v_scale : A.c.k_scale) + (size_t) page * kvh + h;
    int8_t * codes = (which ? A.c.v : A.c.k) + ((size_t) page * kvh + h) * (size_t) (kKvPage * hd);
    const float was = held ? *scale : 0.0f;
    uint32_t big = 0;
    const int pairs = hd / 2;
    for (int k = tid; k < rows * pairs; k += 256) {
        const int r = k / pairs, j = k - r * pairs, p = lo + r;
        int e1;
        const int e0 = kv_pair(j, half, e1);
        double a, b;
        kv_turn(src + (size_t) (s.row + p - s.pos) * ld + (size_t) h * hd, e0, e1,
                which || !half ? nullptr : A.n.rope + (size_t) p * 2 * half, j, half, a, b);
        const float x = (float) a, y = (float) b;
        lrow[r * hd + e0] = x;
        lrow[r * hd + e1] = y;
        big = max(big, max(__float_as_uint(x) & 0x7fffffffu, __float_as_uint(y) & 0x7fffffffu));
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) big = max(big, (uint32_t) __shfl_xor((int) big, o, 64));
    if ((tid & 63) == 0) lmax[tid >> 6] = big;
    __syncthreads();
    big = max(max(lmax[0], lmax[1]), max(lmax[2], lmax[3]));
    const double need = (double) __uint_as_float(big);
    const bool bad = big >= 0x7f800000u || was != was;
    const bool keep = held && need <= 127.0 * (double) was;
    const float now = bad ? __uint_as_float(0x7fc00000u)
                          : (keep ? was : (float) (need * (hi == p0 + kKvPage ? 1.0 : 1.25) / 127.0));
    if (!keep || bad) {
        if (tid == 0) *scale = now;
    }
    /* below 2^-100 the reciprocal or the remainder could leave f32's range */
    const bool none = bad || !(now > 0.0f), tiny = now < 7.9e-31f;
    const float inv = none ? 0.0f : 1.0f / now;
    const bool again = held && !keep && !bad;   /* older codes rounded anew */
    auto code = [&](int old, int r) -> int {    /* position p0 + r's code; old is what is there */
        if (r < held) return again ? (none ? 0 : (int) rint((double) old * (double) was / (double) now)) : old;
        return 0;
    };
    if (which == 0) {
        const int per = hd / 16;   /* pieces of a position */
        const int first = again ? 0 : held;
        for (int k = tid; k < (held + rows - first) * per; k += 256) {
            const int r = first + k / per, d = 16 * (k % per);
            int8_t * at = codes + kv_key_at(r, d);
            union { int4 v; int8_t c[16]; } u;
            if (r < held) {
                u.v = *(const int4 *) at;
#pragma unroll
                for (int e = 0; e < 16; e++) u.c[e] = (int8_t) code(u.c[e], r);
            } else {
                const float * x = lrow + (r - held) * hd + d;
#pragma unroll
                for (int e = 0; e < 16; e++) u.c[e] = none ? 0 : (int8_t) (int) kv_code(x[e], now, inv, tiny);
            }
            *(int4 *) at = u.v;
        }
    } else {
        const int upto = held + rows;
        for (int k = tid; k < 4 * hd; k += 256) {
            const int g = k / hd, d = k - g * hd;
            /* positions 16 t + 4 g + i of this piece */
            bool any = false, all = true;
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const int r = 16 * (e >> 2) + 4 * g + (e & 3);
                const bool in = r >= (again ? 0 : held) && r < upto;
                any = any || in;
                all = all && r >= held && r < upto;
            }
            if (!any) continue;
            int8_t * at = codes + (size_t) k * 16;
            union { int4 v; int8_t c[16]; } u;
            if (!all) u.v = *(const int4 *) at;
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const int r = 16 * (e >> 2) + 4 * g + (e & 3);
                if (r < held) u.c[e] = (int8_t) code(u.c[e], r);
                else if (r < upto) u.c[e] = none ? 0 : (int8_t) (int) kv_code(lrow[(r - held) * hd + d], now, inv, tiny);
            }
            *(int4 *) at = u.v;
        }
    }
}

/* ---------------------------------------------------------------------- read
 * One workgroup per (sequence, page its positions touch, kv head, keys or
 * values). */
template <typename X>
__global__ __launch_bounds__(256) void kv_read_kernel(const sparkmv_kv_cache c, const int * slots, const int * from,
                                                      int n, int nb, X * ko, X * vo) {
    const int tid = threadIdx.x, hd = c.head_dim, kvh = c.kv_heads;
    const int i = blockIdx.x / nb, h = blockIdx.y, which = blockIdx.z;
    X * out = which ? vo : ko;
    if (!out) return;
    const int slot = slots ? slots[i] : i, f = from[i];
    /* the page's positions of [f, f + n); before 0 and past the table: zeros */
    const long blk = (f >= 0 ? f / kKvPage : -((-(long) f + kKvPage - 1) / kKvPage)) + ((int) blockIdx.x - i * nb);
    const long p0 = blk * kKvPage, lo = max((long) f, p0), hi = min((long) f + n, p0 + kKvPage);
    if (lo >= hi) return;
    int page = -1;
    if (slot >= 0 && slot < c.nslots && blk >= 0 && blk < c.max_pages) page = c.pages[(size_t) slot * c.max_pages + blk];
    const bool have = page >= 0 && page < c.npages;
    const size_t head = have ? (size_t) page * kvh + h : 0;
    const float s = have ? (which ? c.v_scale : c.k_scale)[head] : 0.0f;
    const int8_t * codes = (which ? c.v : c.k) + head * (size_t) (kKvPage * hd);
    out += ((size_t) i * n * kvh + h) * hd;
    const size_t row = (size_t) kvh * hd;
    if (!which || !have) {
        for (int k = tid; k < (int) (hi - lo) * hd; k += 256) {
            const int r = (int) (lo - p0) + k / hd, d = k % hd;
            kv_store(out + (size_t) (p0 + r - f) * row + d, have ? (float) codes[kv_key_at(r, d)] * s : 0.0f);
        }
    } else {
        for (int k = tid; k < 4 * hd; k += 256) {
            const int g = k / hd, d = k - g * hd;
            union { int4 v; int8_t c[16]; } u;
            u.v = *(const int4 *) (codes + (size_t) k * 16);
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const long p = p0 + 16 * (e >> 2) + 4 * g + (e & 3);
                if (p >= lo && p < hi) kv_store(out + (size_t) (p - f) * row + d, (float) u.c[e] * s);
            }
        }
    }
}

/* ----------------------------------------------------------------- attention
 * One wave per (token, query head): a lane takes one position of a page for
 * the scores and hd / 64 elements for the weighted values. */
struct KvAttend {
    sparkmv_kv_cache c;
    sparkmv_kv_batch b;
    sparkmv_kv_query q;
};

__device__ __forceinline__ float kv_wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}
__device__ __forceinline__ float kv_wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

template <typename X, typename O, int HD>
__global__ __launch_bounds__(64) void kv_attend_kernel(const KvAttend A) {
    constexpr int E = HD / 64;
    __shared__ float lq[HD];
    __shared__ float lp[64];
    const int lane = threadIdx.x, t = blockIdx.x, head = blockIdx.y;
    const int h = head / (A.q.heads / A.c.kv_heads);
    int pos = -1, slot = 0;
    for (int i = lane; i < A.b.nseq; i += 64) {
        const KvSeq s = kv_seq(A.b, i, A.c.nslots, A.c.max_pages);
        if (t >= s.row && t - s.row < s.count) {
            pos = s.pos + t - s.row;
            slot = s.slot;
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const int op = __shfl_xor(pos, o, 64), os = __shfl_xor(slot, o, 64);
        if (op > pos) {
            pos = op;
            slot = os;
        }
    }
    if (pos < 0) return;
    const X * q = (const X *) A.q.q + (size_t) t * A.q.ldq + (size_t) head * HD;
    for (int e = lane; e < HD; e += 64) lq[e] = kv_load(q + e) * A.q.scale;
    __syncthreads();
    const int first = A.q.window > 0 && pos + 1 > A.q.window ? pos + 1 - A.q.window : 0;
    float m = -INFINITY, l = 0.0f, o[E];
#pragma unroll
    for (int e = 0; e < E; e++) o[e] = 0.0f;
    for (int blk = first / kKvPage; blk <= pos / kKvPage; blk++) {
        const int page = A.c.pages[(size_t) slot * A.c.max_pages + blk];
        if (page < 0 || page >= A.c.npages) continue;
        const size_t at = (size_t) page * A.c.kv_heads + h;
        const int8_t * kc = A.c.k + at * (size_t) (kKvPage * HD), * vc = A.c.v + at * (size_t) (kKvPage * HD);
        const float ks = A.c.k_scale[at], vs = A.c.v_scale[at];
        float s = 0.0f;
        for (int c = 0; c < HD / 16; c++) {
            union { int4 v; int8_t b[16]; } u;
            u.v = *(const int4 *) (kc + kv_key_at(lane, 16 * c));
#pragma unroll
            for (int e = 0; e < 16; e++) s += (float) u.b[e] * lq[16 * c + e];
        }
        s *= ks;
        const int p = blk * kKvPage + lane;
        const bool seen = p >= first && p <= pos;
        if (!seen) s = -INFINITY;
        const float mn = fmaxf(m, kv_wave_max(s));
        const float a = mn == -INFINITY ? 1.0f : expf(m - mn);
        const float w = seen ? expf(s - mn) : 0.0f;
        m = mn;
        l = l * a + kv_wave_sum(w);
        __syncthreads();
        lp[lane] = w * vs;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < E; e++) {
            const int d = lane + 64 * e;
            float acc = 0.0f;
#pragma unroll
            for (int g = 0; g < 4; g++) {
                union { int4 v; int8_t b[16]; } u;
                u.v = *(const int4 *) (vc + (size_t) (g * HD + d) * 16);
#pragma unroll
                for (int k = 0; k < 16; k++) acc += (float) u.b[k] * lp[16 * (k >> 2) + 4 * g + (k & 3)];
            }
            o[e] = o[e] * a + acc;
        }
    }
    float f = l == 0.0f ? 0.0f : 1.0f / l;
    if (A.q.gate) f *= 1.0f / (1.0f + expf(-A.q.gate[(size_t) t * A.q.ldg + head]));
    O * out = (O *) A.q.out + (size_t) t * A.q.ldo + (size_t) head * HD;
#pragma unroll
    for (int e = 0; e < E; e++) kv_store(out + lane + 64 * e, l == 0.0f ? 0.0f : o[e] * f);
}

/* ----------------------------------------------------- attention, few columns
 *
 * Up to four columns (token, query head) of a kv head: a decode step of up to
 * four query heads per kv head. The kernel is bound by reading the codes once,
 * so everything else is made to fit behind the loads:
 *
 *   S = K q  and  O = P V  run on the 8-bit integer matrix instructions,
 *   16 x 16 x 64, with the codes as they lie in memory: no conversion. What
 *   meets them is an f32 query element or weight written as four signed 7-bit
 *   digits, and the sixteen columns of a tile are the four columns times those
 *   four digits: all of f32's precision costs no further instruction. Sums are
 *   exact in i32 (64 * 127 * 256 < 2^21), and a column's value is the sum of
 *   its four digits' sums, two cross-lane additions in a quad.
 *
 *   A query element is an integer of 28 bits at a power of two chosen by the
 *   head's largest element (no rounding but the integer's, 2^-28 of the
 *   largest). A weight e^(s - m) takes the page's own largest score as m, so
 *   it is rounded to 2^-28 of the page's largest weight, whatever the rest of
 *   the sequence holds; the page's sum then enters the f32 output with the
 *   factor value scale * e^(m - M), M a running reference that moves only when
 *   a page passes it by 2^kKvLag.
 *
 * Workgroups take equal shares of all (sequence, kv head, page) in that order,
 * so lengths may differ by any amount. A share's pages of one kv head go to
 * the four waves in turn, whose results meet in LDS; a kv head's pages that lie
 * in one share are written out at once, others as a partial result that a
 * second launch joins. */
constexpr float kKvLag = 16.0f;

struct KvFlat {
    sparkmv_kv_cache c;
    sparkmv_kv_batch b;
    sparkmv_kv_query q;
    int least;       /* pages of a share, at least */
    int * pre;       /* [nseq + 2]: pages of one kv head before each sequence; the share */
    float * po;      /* [workgroups][2][4][HD] */
    float * pml;     /* [workgroups][2][4][2] */
};

typedef int kv_i4 __attribute__((ext_vector_type(4)));
typedef float kv_f4 __attribute__((ext_vector_type(4)));

/* the pages that a sequence's tokens see: first and how many */
__device__ __forceinline__ int kv_span(const KvSeq & s, int window, int & first) {
    if (s.count <= 0) {
        first = 0;
        return 0;
    }
    first = (window > 0 && s.pos + 1 > window ? s.pos + 1 - window : 0) / kKvPage;
    return (s.pos + s.count - 1) / kKvPage - first + 1;
}

template <int CTRL>
__device__ __forceinline__ float kv_quad(float v) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true));
}
/* the sum over the four lanes of a quad, the same bits in each */
__device__ __forceinline__ float kv_quad_sum(float v) {
    v += kv_quad<0xb1>(v);          /* lanes 1 0 3 2 */
    return v + kv_quad<0x4e>(v);    /* lanes 2 3 0 1 */
}

/* 16 values of a row as f32 */
__device__ __forceinline__ void kv_load16(const float * p, float * x) {
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const kv_f4 v = *(const kv_f4 *) (p + 4 * k);
#pragma unroll
        for (int i = 0; i < 4; i++) x[4 * k + i] = v[i];
    }
}
__device__ __forceinline__ void kv_load16(const uint16_t * p, float * x) {
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const kv_i4 v = *(const kv_i4 *) (p + 8 * k);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[8 * k + 2 * i] = __uint_as_float((uint32_t) v[i] << 16);
            x[8 * k + 2 * i + 1] = __uint_as_float((uint32_t) v[i] & 0xffff0000u);
        }
    }
}

template <typename O>
__device__ __forceinline__ void kv_write(const sparkmv_kv_query & q, int row, int head, int hd, int d, float o, float l) {
    float f = l == 0.0f ? 0.0f : 1.0f / l;
    if (q.gate) f *= 1.0f / (1.0f + expf(-q.gate[(size_t) row * q.ldg + head]));
    kv_store((O *) q.out + (size_t) row * q.ldo + (size_t) head * hd + d, l == 0.0f ? 0.0f : o * f);
}

template <typename X, typename O, int HD>
__global__ __launch_bounds__(256, 2) void kv_decode_kernel(const KvFlat A) {
    constexpr int NC = HD / 64, ND = HD / 16;
    extern __shared__ int lpre[];                     /* [nseq + 1] */
    __shared__ int lsum[4];
    __shared__ __attribute__((aligned(16))) float lo[4][4][HD];
    __shared__ float lm[4][4], ll[4][4];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, g = lane >> 4, c16 = lane & 15, col = c16 >> 2, dg = c16 & 3;
    const int kvh = A.c.kv_heads, G = A.q.heads / kvh, nseq = A.b.nseq;
    /* pages before each sequence */
    {
        const int per = (nseq + 255) / 256, i0 = min(nseq, tid * per), i1 = min(nseq, i0 + per);
        int sum = 0;
        for (int i = i0; i < i1; i++) {
            int first;
            lpre[i] = sum;
            sum += kv_span(kv_seq(A.b, i, A.c.nslots, A.c.max_pages), A.q.window, first);
        }
        int scan = sum;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(scan, o, 64);
            if (lane >= o) scan += v;
        }
        if (lane == 63) lsum[wave] = scan;
        __syncthreads();
        int before = scan - sum;
        for (int w = 0; w < wave; w++) before += lsum[w];
        for (int i = i0; i < i1; i++) lpre[i] += before;
        if (tid == 255) lpre[nseq] = before + sum;
        __syncthreads();
    }
    const int total = lpre[nseq] * kvh, share = max((total + (int) gridDim.x - 1) / (int) gridDim.x, A.least);
    if (blockIdx.x == 0) {
        for (int i = tid; i <= nseq; i += 256) A.pre[i] = lpre[i];
        if (tid == 0) A.pre[nseq + 1] = share;
    }
    const int ubeg = (int) blockIdx.x * share, uend = min(total, ubeg + share);
    const float wdig = (float) (1 << (7 * (3 - dg)));
    const int sh = 7 * (3 - dg);
    for (int u = ubeg; u < uend;) {
        /* the sequence: the last one that begins at or before u */
        int i = 0;
        for (int a = 0, b = nseq; b - a > 1;) {
            const int mid = (a + b) >> 1;
            if (lpre[mid] * kvh <= u) a = mid;
            else b = mid;
            i = a;
        }
        const int n = lpre[i + 1] - lpre[i], in = u - lpre[i] * kvh, h = in / n, off = in - h * n, seg = min(n - off, uend - u);
        const KvSeq s = kv_seq(A.b, i, A.c.nslots, A.c.max_pages);
        int first;
        kv_span(s, A.q.window, first);
        const int ncol = s.count * G, tok = min(col / G, s.count - 1), head = h * G + col % G;
        const int pos_c = s.pos + tok, beg_c = A.q.window > 0 && pos_c + 1 > A.q.window ? pos_c + 1 - A.q.window : 0;
        /* positions that every column sees */
        const int all_lo = A.q.window > 0 && s.pos + s.count > A.q.window ? s.pos + s.count - A.q.window : 0, all_hi = s.pos;
        /* the columns' digits */
        kv_i4 qd[NC];
        float cs;
        bool qbad;
        {
            float x[NC][16];
            const X * qp = (const X *) A.q.q + (size_t) (s.row + tok) * A.q.ldq + (size_t) head * HD + 16 * g;
            uint32_t big = 0;
#pragma unroll
            for (int c = 0; c < NC; c++) kv_load16(qp + 64 * c, x[c]);
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int e = 0; e < 16; e++) big = max(big, __float_as_uint(x[c][e]) & 0x7fffffffu);
            big = max(big, (uint32_t) __shfl_xor((int) big, 16, 64));
            big = max(big, (uint32_t) __shfl_xor((int) big, 32, 64));
            qbad = big >= 0x7f800000u;
            int ex = 0;
            (void) frexpf(__uint_as_float(qbad ? 0u : big), &ex);
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    uint32_t packed = 0;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int v = (int) rintf(ldexpf(qbad ? 0.0f : x[c][4 * w + e], 27 - ex)) + ((64 << 14) | (64 << 7) | 64);
                        const int d = dg == 0 ? v >> 21 : ((v >> sh) & 127) - 64;
                        packed |= (uint32_t) (d & 255) << (8 * e);
                    }
                    qd[c][w] = col < ncol ? (int) packed : 0;
                }
            cs = ldexpf(A.q.scale * 1.44269504088896340736f, ex - 27);
        }
        float m = -INFINITY, l = 0.0f;
        kv_f4 o[ND];
#pragma unroll
        for (int d = 0; d < ND; d++) o[d] = kv_f4{0.f, 0.f, 0.f, 0.f};
        const int * table = A.c.pages + (size_t) s.slot * A.c.max_pages + first + off;
        /* 64 pages of this wave at a time: their numbers and scales are held one a lane */
        for (int base = wave; base < seg; base += 256) {
            const int mine = min((seg - base + 3) / 4, 64);
            int id = 0;
            float ks = 0.0f, vs = 0.0f;
            bool have = false;
            if (lane < mine) {
                id = table[base + 4 * lane];
                have = id >= 0 && id < A.c.npages;
                id = have ? id : 0;
                ks = A.c.k_scale[(size_t) id * kvh + h];
                vs = A.c.v_scale[(size_t) id * kvh + h];
            }
            const uint64_t there = __ballot(have);
            kv_i4 kr[NC][4], vr[ND];
            auto fetch_k = [&](int j) {
                const int8_t * p = A.c.k + ((size_t) __builtin_amdgcn_readlane(id, j) * kvh + h) * (size_t) (kKvPage * HD) + c16 * 64 + 16 * g;
#pragma unroll
                for (int c = 0; c < NC; c++)
#pragma unroll
                    for (int t = 0; t < 4; t++) kr[c][t] = *(const kv_i4 *) (p + c * 4096 + t * 1024);
            };
            auto fetch_v = [&](int j) {
                const int8_t * p = A.c.v + ((size_t) __builtin_amdgcn_readlane(id, j) * kvh + h) * (size_t) (kKvPage * HD) + (g * HD + c16) * 16;
#pragma unroll
                for (int d = 0; d < ND; d++) vr[d] = *(const kv_i4 *) (p + d * 256);
            };
            fetch_k(0);
            fetch_v(0);
            __builtin_amdgcn_sched_barrier(0);
            for (int j = 0; j < mine; j++) {
                const int nx = min(j + 1, mine - 1);
                float x[4][4];
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    kv_i4 acc = kv_i4{0, 0, 0, 0};
#pragma unroll
                    for (int c = 0; c < NC; c++) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(kr[c][t], qd[c], acc, 0, 0, 0);
#pragma unroll
                    for (int e = 0; e < 4; e++) x[t][e] = (float) acc[e] * wdig;
                }
                __builtin_amdgcn_sched_barrier(0);
                fetch_k(nx);
                __builtin_amdgcn_sched_barrier(0);
                const float kscale = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(ks), j));
                const float vscale = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(vs), j));
                const float f = cs * kscale;
                const int p0 = (first + off + base + 4 * j) * kKvPage;
                const bool ok = there >> j & 1;
                float mp = -INFINITY;
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++) x[t][e] = kv_quad_sum(x[t][e]) * f;
                if (!ok || p0 < all_lo || p0 + kKvPage - 1 > all_hi || kscale != kscale) {
                    bool any = false;
#pragma unroll
                    for (int t = 0; t < 4; t++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const int p = p0 + 16 * t + 4 * g + e;
                            const bool seen = ok && p >= beg_c && p <= pos_c;
                            any = any || seen;
                            x[t][e] = seen ? x[t][e] : -INFINITY;
                        }
                    if (kscale != kscale) {
                        if (any) l = kscale;   /* NaN to the end for a column that sees some of it */
#pragma unroll
                        for (int t = 0; t < 4; t++)
#pragma unroll
                            for (int e = 0; e < 4; e++) x[t][e] = -INFINITY;
                    }
                }
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++) mp = fmaxf(mp, x[t][e]);
                mp = fmaxf(mp, __shfl_xor(mp, 16, 64));
                mp = fmaxf(mp, __shfl_xor(mp, 32, 64));
                if (__any(mp > m + kKvLag)) {
                    const float mn = fmaxf(m, mp);
                    const float a = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
                    l *= a;
#pragma unroll
                    for (int d = 0; d < ND; d++) o[d] *= a;
                    m = mn;
                }
                const float mref = mp == -INFINITY ? 0.0f : mp;
                kv_i4 P;
                float sum = 0.0f;
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    uint32_t packed = 0;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float p = __builtin_amdgcn_exp2f(x[t][e] - mref);
                        sum += p;
                        const uint32_t v = (uint32_t) (p * 134217728.0f + 0.5f);
                        packed |= ((v >> sh) & 127u) << (8 * e);
                    }
                    P[t] = (int) packed;
                }
                const float step = mp == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mp - m);
                l += sum * step;
                const float w = mp == -INFINITY ? 0.0f : step * vscale;
#pragma unroll
                for (int d = 0; d < ND; d++) {
                    const kv_i4 acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(vr[d], P, kv_i4{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
                    for (int e = 0; e < 4; e++) o[d][e] += w * (float) acc[e];
                }
                __builtin_amdgcn_sched_barrier(0);
                fetch_v(nx);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
        if (qbad) l = __uint_as_float(0x7fc00000u);
        /* the digits of a column, then the waves */
        const float down = wdig * 7.450580596923828e-9f;   /* 2^-27 */
#pragma unroll
        for (int d = 0; d < ND; d++) {
            kv_f4 v;
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = kv_quad_sum(o[d][e] * down);
            if ((d & 3) == dg) *(kv_f4 *) &lo[wave][col][16 * d + 4 * g] = v;
        }
        if (g == 0 && dg == 0) {
            lm[wave][col] = m;
            ll[wave][col] = l;
        }
        __syncthreads();
        const bool whole = seg == n;
        const size_t at = 2 * (size_t) blockIdx.x + (off == 0 ? 1 : 0);
        for (int k = tid; k < ncol * HD; k += 256) {
            const int cc = k / HD, d = k - cc * HD;
            float M = lm[0][cc];
#pragma unroll
            for (int w = 1; w < 4; w++) M = fmaxf(M, lm[w][cc]);
            float L = 0.0f, v = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const float a = lm[w][cc] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(lm[w][cc] - M);
                L += lm[w][cc] == -INFINITY ? ll[w][cc] : a * ll[w][cc];
                v += a * lo[w][cc][d];
            }
            if (whole) {
                kv_write<O>(A.q, s.row + cc / G, h * G + cc % G, HD, d, v, L);
            } else {
                A.po[(at * 4 + cc) * HD + d] = v;
                if (d == 0) {
                    A.pml[(at * 4 + cc) * 2] = M;
                    A.pml[(at * 4 + cc) * 2 + 1] = L;
                }
            }
        }
        __syncthreads();
        u += seg;
    }
}

/* Joins the partial results of one (sequence, kv head), in the order of its
 * pages: its first share wrote slot 1, the later ones slot 0. */
template <typename O, int HD>
__global__ __launch_bounds__(256) void kv_decode_join_kernel(const KvFlat A) {
    const int i = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
    const int kvh = A.c.kv_heads, G = A.q.heads / kvh;
    const int before = A.pre[i], n = A.pre[i + 1] - before, share = A.pre[A.b.nseq + 1];
    if (n == 0) return;
    const int a = before * kvh + h * n, w0 = a / share, w1 = (a + n - 1) / share;
    if (w0 == w1) return;
    const KvSeq s = kv_seq(A.b, i, A.c.nslots, A.c.max_pages);
    const int ncol = s.count * G;
    for (int k = tid; k < ncol * HD; k += 256) {
        const int cc = k / HD, d = k - cc * HD;
        float M = -INFINITY;
        for (int w = w0; w <= w1; w++) M = fmaxf(M, A.pml[((2 * (size_t) w + (w == w0)) * 4 + cc) * 2]);
        float L = 0.0f, v = 0.0f;
        for (int w = w0; w <= w1; w++) {
            const size_t at = (2 * (size_t) w + (w == w0)) * 4 + cc;
            const float m = A.pml[2 * at], l = A.pml[2 * at + 1], f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - M);
            L += m == -INFINITY ? l : f * l;
            v += f * A.po[at * HD + d];
        }
        kv_write<O>(A.q, s.row + cc / G, h * G + cc % G, HD, d, v, L);
    }
}

/* ------------------------------------------------------------------ checks */

bool aligned(const void * p, size_t n) { return ((uintptr_t) p & (n - 1)) == 0; }

int elem(int dtype) { return dtype == SPARKMV_X_F32 ? 4 : 2; }

int check_dtype(const char * what, int dtype) {
    if (dtype == SPARKMV_X_F32 || dtype == SPARKMV_X_BF16) return 0;
    set_error("%s: unknown type %d", what, dtype);
    return -1;
}

/* rows of n values at stride ld, each starting 16-byte aligned */
int check_rows(const char * what, const void * p, int ld, long n, int dtype, int nrows) {
    if (!p) { set_error("%s is null", what); return -1; }
    if (nrows > 1 && ld < n) { set_error("%s: a row stride of %d holds no %ld values", what, ld, n); return -1; }
    if (!aligned(p, 16) || (nrows > 1 && (size_t) ld * elem(dtype) % 16)) {
        set_error("%s: rows do not start 16-byte aligned", what);
        return -1;
    }
    return 0;
}

int check_launch(const char * what) {
    hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : fail_hip(what, e);
}

/* workgroups of the few-column kernel: two a CU, no more than there can be pages */
int flat_groups(const sparkmv_kv_cache * c, const sparkmv_kv_batch * b, int window) {
    const int most = 2 * cu_count();
    long len = b->max_len > 0 ? b->max_len : (long) c->max_pages * kKvPage;
    if (window > 0 && len > window + kKvPage) len = window + kKvPage;
    const long pages = (len + kKvPage - 1) / kKvPage * b->nseq * c->kv_heads;
    return pages < 1 ? 1 : (pages < most ? (int) pages : most);
}

/* the workspace's bytes, and its parts where f is given */
size_t flat_work(const sparkmv_kv_cache * c, const sparkmv_kv_batch * b, KvFlat * f) {
    const size_t w = 2 * (size_t) cu_count(), hd = (size_t) c->head_dim;
    size_t off = 0;
    auto take = [&](size_t bytes) { const size_t o = off; off += (bytes + 255) & ~(size_t) 255; return o; };
    const size_t pre = take(((size_t) b->nseq + 2) * 4), po = take(w * 2 * 4 * hd * 4), pml = take(w * 2 * 4 * 2 * 4);
    if (f) {
        uint8_t * m = (uint8_t *) f->q.work;
        f->pre = (int *) (m + pre);
        f->po = (float *) (m + po);
        f->pml = (float *) (m + pml);
    }
    return off;
}

}  // namespace

int kv_check_cache(const sparkmv_kv_cache * c) {
    if (!c) { set_error("kv cache is null"); return -1; }
    if (c->kv_heads < 1 || c->kv_heads > 1024) { set_error("kv_heads %d is outside 1..1024", c->kv_heads); return -1; }
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) {
        set_error("head_dim %d is not 64, 128 or 256", c->head_dim);
        return -1;
    }
    if (c->npages < 1 || c->nslots < 1 || c->max_pages < 1) {
        set_error("kv cache of %d pages, %d slots of %d pages", c->npages, c->nslots, c->max_pages);
        return -1;
    }
    if (c->max_pages > (1 << 24)) { set_error("max_pages %d is above %d", c->max_pages, 1 << 24); return -1; }
    if (!c->k || !c->v || !c->k_scale || !c->v_scale || !c->pages) { set_error("kv cache has a null array"); return -1; }
    if (!aligned(c->k, 16) || !aligned(c->v, 16)) { set_error("kv cache codes are not 16-byte aligned"); return -1; }
    return 0;
}

int kv_check_batch(const sparkmv_kv_batch * b) {
    if (!b) { set_error("kv batch is null"); return -1; }
    if (b->nseq < 0 || b->nseq > kKvMaxSeq) { set_error("%d sequences are outside 0..%d", b->nseq, kKvMaxSeq); return -1; }
    if (b->ntok < 0) { set_error("%d tokens", b->ntok); return -1; }
    if (b->nseq && !b->pos) { set_error("kv batch has no positions"); return -1; }
    if (b->max_q < 1) { set_error("max_q %d is below 1", b->max_q); return -1; }
    if (!b->qstart && b->ntok < b->nseq) {
        set_error("%d sequences of one token each, but %d rows", b->nseq, b->ntok);
        return -1;
    }
    return 0;
}

}  // namespace sparkmv

using namespace sparkmv;

extern "C" {

int sparkmv_rope_table(float * table, int rows, int rope_dim, double theta, void * stream) {
    if (!table) { set_error("rope table is null"); return -1; }
    if (rows < 1 || rope_dim < 2 || rope_dim % 2) {
        set_error("rope table of %d rows and %d values", rows, rope_dim);
        return -1;
    }
    if (!(theta > 0.0)) { set_error("theta must be positive"); return -1; }
    const size_t n = (size_t) rows * (rope_dim / 2), wg = (n + 255) / 256;
    if (wg > 0x7fffffffu) { set_error("rope table of %d rows and %d values is too large", rows, rope_dim); return -1; }
    hipLaunchKernelGGL(kv_rope_table_kernel, dim3((unsigned) wg), dim3(256), 0, (hipStream_t) stream, table, rows,
                       rope_dim / 2, (float) theta);
    return check_launch("rope table launch");
}

int sparkmv_kv_append(const sparkmv_kv_cache * cache, const sparkmv_kv_batch * batch, const sparkmv_kv_new * rows,
                      void * stream) {
    if (kv_check_cache(cache) || kv_check_batch(batch)) return -1;
    if (!rows) { set_error("kv rows are null"); return -1; }
    const sparkmv_kv_new & n = *rows;
    const int hd = cache->head_dim;
    if (check_dtype("kv rows", n.x_dtype)) return -1;
    if (n.heads < 0 || (n.heads > 0) != (n.q != nullptr) || (n.heads > 0) != (n.q_out != nullptr)) {
        set_error("%d query heads, queries and their output do not agree", n.heads);
        return -1;
    }
    if (n.heads > 65536) { set_error("%d query heads are above 65536", n.heads); return -1; }
    if (n.rope_dim < 0 || n.rope_dim % 2 || n.rope_dim > hd) {
        set_error("rope_dim %d is not even within 0..%d", n.rope_dim, hd);
        return -1;
    }
    if (n.rope_dim && !n.rope) { set_error("rope table is null"); return -1; }
    if (n.rope_dim && (long) n.rope_rows < (long) cache->max_pages * kKvPage) {
        set_error("a rope table of %d rows does not cover %ld positions", n.rope_rows, (long) cache->max_pages * kKvPage);
        return -1;
    }
    if (batch->nseq == 0 || batch->ntok == 0) return 0;
    const long kvd = (long) cache->kv_heads * hd, qd = (long) n.heads * hd;
    if (check_rows("keys", n.k, n.ldk, kvd, n.x_dtype, batch->ntok) ||
        check_rows("values", n.v, n.ldv, kvd, n.x_dtype, batch->ntok))
        return -1;
    if (n.heads && (check_rows("queries", n.q, n.ldq, qd, n.x_dtype, batch->ntok) ||
                    check_rows("rotated queries", n.q_out, n.ldqo, qd, n.x_dtype, batch->ntok)))
        return -1;
    const int max_q = batch->max_q < batch->ntok ? batch->max_q : batch->ntok;
    KvAppend a;
    a.c = *cache; a.b = *batch; a.n = n;
    a.b.max_q = batch->qstart ? max_q : 1;
    a.half = n.rope_dim / 2;
    a.nb = (a.b.max_q + kKvPage - 2) / kKvPage + 1;
    if (a.nb > cache->max_pages) a.nb = cache->max_pages;
    a.qparts = (n.heads + 3) / 4;
    const long nkv = (long) batch->nseq * a.nb * cache->kv_heads * 2, wgs = nkv + (long) batch->ntok * a.qparts;
    if (wgs > 0x7fffffffl) { set_error("an append of %ld workgroups", wgs); return -1; }
    a.nkv = (int) nkv;
    const int lrows = a.b.max_q < kKvPage ? a.b.max_q : kKvPage;
    const uint32_t lds = (uint32_t) (lrows * hd * 4);
    const bool f32 = n.x_dtype == SPARKMV_X_F32;
    static LdsAllowed allowed[2];
    /* a full page of 256 elements takes 64 KB beside the kernel's own words */
    if (lds_allow(allowed[f32], f32 ? (const void *) kv_append_kernel<float> : (const void *) kv_append_kernel<uint16_t>,
                  lds + 1024, "LDS opt-in for the kv append"))
        return -1;
    const dim3 grid((unsigned) wgs), block(256);
    hipStream_t s = (hipStream_t) stream;
    if (f32) hipLaunchKernelGGL(kv_append_kernel<float>, grid, block, lds, s, a);
    else hipLaunchKernelGGL(kv_append_kernel<uint16_t>, grid, block, lds, s, a);
    return check_launch("kv append launch");
}

int sparkmv_kv_read(const sparkmv_kv_cache * cache, int nseq, const int * slot, const int * from, int n, void * k_out,
                    void * v_out, int out_dtype, void * stream) {
    if (kv_check_cache(cache) || check_dtype("kv read", out_dtype)) return -1;
    if (nseq < 0 || nseq > kKvMaxSeq) { set_error("%d sequences are outside 0..%d", nseq, kKvMaxSeq); return -1; }
    if (n < 0) { set_error("%d positions", n); return -1; }
    if (nseq == 0 || n == 0 || (!k_out && !v_out)) return 0;
    if (!from) { set_error("kv read has no positions"); return -1; }
    const long nb = (n + kKvPage - 2) / kKvPage + 1, wgs = (long) nseq * nb;
    if (wgs > 0x7fffffffl) { set_error("a read of %ld pages", wgs); return -1; }
    const dim3 grid((unsigned) wgs, (unsigned) cache->kv_heads, 2), block(256);
    hipStream_t s = (hipStream_t) stream;
    if (out_dtype == SPARKMV_X_F32)
        hipLaunchKernelGGL(kv_read_kernel<float>, grid, block, 0, s, *cache, slot, from, n, (int) nb, (float *) k_out,
                           (float *) v_out);
    else
        hipLaunchKernelGGL(kv_read_kernel<uint16_t>, grid, block, 0, s, *cache, slot, from, n, (int) nb,
                           (uint16_t *) k_out, (uint16_t *) v_out);
    return check_launch("kv read launch");
}

size_t sparkmv_kv_attend_work(const sparkmv_kv_cache * cache, const sparkmv_kv_batch * batch, int heads) {
    if (kv_check_cache(cache) || kv_check_batch(batch)) return 0;
    return flat_work(cache, batch, nullptr);
}

int sparkmv_kv_attend(const sparkmv_kv_cache * cache, const sparkmv_kv_batch * batch, const sparkmv_kv_query * query,
                      void * stream) {
    if (kv_check_cache(cache) || kv_check_batch(batch)) return -1;
    if (!query) { set_error("kv query is null"); return -1; }
    const sparkmv_kv_query & q = *query;
    if (check_dtype("queries", q.q_dtype) || check_dtype("attention output", q.out_dtype)) return -1;
    if (q.heads < 1 || q.heads % cache->kv_heads || q.heads / cache->kv_heads > kKvMaxGroup) {
        set_error("%d query heads are not 1..%d times %d kv heads", q.heads, kKvMaxGroup, cache->kv_heads);
        return -1;
    }
    if (q.window < 0) { set_error("window %d is negative", q.window); return -1; }
    if (!(fabsf(q.scale) < INFINITY)) { set_error("the scale of the scores is not finite"); return -1; }
    if (batch->nseq == 0 || batch->ntok == 0) return 0;
    const long qd = (long) q.heads * cache->head_dim;
    if (check_rows("queries", q.q, q.ldq, qd, q.q_dtype, batch->ntok) ||
        check_rows("attention output", q.out, q.ldo, qd, q.out_dtype, batch->ntok))
        return -1;
    if (q.gate && batch->ntok > 1 && q.ldg < q.heads) { set_error("gate: a row stride of %d holds no %d heads", q.ldg, q.heads); return -1; }
    const size_t need = sparkmv_kv_attend_work(cache, batch, q.heads);
    if (need && (!q.work || !aligned(q.work, 256) || q.work_bytes < need)) {
        set_error("attention needs %zu bytes of 256-byte aligned workspace, not %zu", need, q.work ? q.work_bytes : 0);
        return -1;
    }
    hipStream_t s = (hipStream_t) stream;
    const bool xf = q.q_dtype == SPARKMV_X_F32, of = q.out_dtype == SPARKMV_X_F32;
    const int max_q = batch->qstart ? batch->max_q : 1;
#define KV_TYPES(CALL)                                                                                               \
    do {                                                                                                             \
        if (xf && of) KV_DIMS(CALL, float, float);                                                                   \
        else if (xf) KV_DIMS(CALL, float, uint16_t);                                                                 \
        else if (of) KV_DIMS(CALL, uint16_t, float);                                                                 \
        else KV_DIMS(CALL, uint16_t, uint16_t);                                                                      \
    } while (0)
#define KV_DIMS(CALL, X, O)                                                                                          \
    do {                                                                                                             \
        if (cache->head_dim == 64) CALL(X, O, 64);                                                                   \
        else if (cache->head_dim == 128) CALL(X, O, 128);                                                            \
        else CALL(X, O, 256);                                                                                        \
    } while (0)
    if ((long) max_q * (q.heads / cache->kv_heads) <= 4) {
        KvFlat f;
        f.c = *cache; f.b = *batch; f.q = q;
        f.b.max_q = max_q;
        f.least = 1;
        flat_work(cache, batch, &f);
        const dim3 grid((unsigned) flat_groups(cache, batch, q.window)), join((unsigned) batch->nseq, (unsigned) cache->kv_heads);
        const uint32_t lds = ((uint32_t) batch->nseq + 1) * 4;
#define KV_FLAT(X, O, H)                                                                                             \
    do {                                                                                                             \
        hipLaunchKernelGGL((kv_decode_kernel<X, O, H>), grid, dim3(256), lds, s, f);                                 \
        hipLaunchKernelGGL((kv_decode_join_kernel<O, H>), join, dim3(256), 0, s, f);                                 \
    } while (0)
        KV_TYPES(KV_FLAT);
#undef KV_FLAT
        return check_launch("kv attention launch");
    }
    KvAttend a;
    a.c = *cache; a.b = *batch; a.q = q;
    a.b.max_q = max_q;
    const dim3 grid((unsigned) batch->ntok, (unsigned) q.heads), block(64);
#define KV_ATTEND(X, O, H) hipLaunchKernelGGL((kv_attend_kernel<X, O, H>), grid, block, 0, s, a)
    KV_TYPES(KV_ATTEND);
#undef KV_ATTEND
#undef KV_DIMS
#undef KV_TYPES
    return check_launch("kv attention launch");
}

}  // extern "C"
