/* kv.hip — the paged 8-bit cache: the append with the position rotation on the
 * way, reading positions back, and attention over it (include/sparkmv.h has
 * the cache's layout and its rules; kv.h the offsets of a code). */
#include "kv.h"

#include <math.h>

namespace sparkmv {

namespace {

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
 * values) each, the others a few query heads of one token.
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

/* n pairs over NT threads, four of a thread's in flight: at(i, row, table) gives
 * pair i's place in its head, its row and its table row (NULL: not turned), and
 * put(i, e0, e1, a, b) takes the two results */
template <typename X, int NT, typename At, typename Put>
__device__ __forceinline__ void kv_turn_all(int n, At at, int half, Put put) {
    for (int i0 = threadIdx.x; i0 < n; i0 += 4 * NT) {
        int e0[4], e1[4];
        float x[4], y[4], c[4], s[4];
        bool turn[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int i = min(i0 + u * NT, n - 1);
            const X * row;
            const float * tab;
            const int j = at(i, row, tab);
            e0[u] = kv_pair(j, half, e1[u]);
            x[u] = kv_load(row + e0[u]);
            y[u] = kv_load(row + e1[u]);
            turn[u] = j < half && tab;
            c[u] = turn[u] ? tab[j] : 1.0f;
            s[u] = turn[u] ? tab[half + j] : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < 4; u++) {
            if (i0 + u * NT >= n) continue;
            double a = (double) x[u], b = (double) y[u];
            if (turn[u]) {
                const double p = a, cc = (double) c[u], ss = (double) s[u];
                a = p * cc - b * ss;
                b = b * cc + p * ss;
            }
            put(i0 + u * NT, e0[u], e1[u], a, b);
        }
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

template <typename X, int NT>
__global__ __launch_bounds__(NT) void kv_append_kernel(const KvAppend A) {
    constexpr int QH = NT / 64;      /* query heads of a workgroup */
    extern __shared__ __attribute__((aligned(16))) float lrow[];   /* [rows][hd] */
    __shared__ uint32_t lmax[NT / 64];
    const int tid = threadIdx.x, hd = A.c.head_dim, kvh = A.c.kv_heads, half = A.half;
    const int sh = 31 - __clz(hd / 2), pairs = 1 << sh;   /* head_dim is a power of two */
    if ((int) blockIdx.x >= A.nkv) {
        /* queries */
        const int w = (int) blockIdx.x - A.nkv, t = w / A.qparts, h0 = QH * (w - t * A.qparts);
        __shared__ int lpos;
        if (tid == 0) lpos = -1;
        __syncthreads();
        for (int i = tid; i < A.b.nseq; i += NT) {
            const KvSeq s = kv_seq(A.b, i, A.c.nslots, A.c.max_pages);
            if (t >= s.row && t - s.row < s.count) lpos = s.pos + t - s.row;
        }
        __syncthreads();
        const int pos = lpos;
        if (pos < 0) return;
        const float * rope = half ? A.n.rope + (size_t) pos * 2 * half : nullptr;
        const X * src = (const X *) A.n.q + (size_t) t * A.n.ldq + (size_t) h0 * hd;
        X * dst = (X *) A.n.q_out + (size_t) t * A.n.ldqo + (size_t) h0 * hd;
        const int n = min(QH, A.n.heads - h0) << sh;
        kv_turn_all<X, NT>(n, [&](int i, const X *& row, const float *& tab) {
            row = src + (size_t) (i >> sh) * hd;
            tab = rope;
            return i & (pairs - 1);
        }, half, [&](int i, int e0, int e1, double a, double b) {
            X * to = dst + (size_t) (i >> sh) * hd;
            kv_store_wide(to + e0, a);
            kv_store_wide(to + e1, b);
        });
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
    const X * base = src + (size_t) (s.row + lo - s.pos) * ld + (size_t) h * hd;
    kv_turn_all<X, NT>(rows << sh, [&](int i, const X *& row, const float *& tab) {
        const int r = i >> sh;
        row = base + (size_t) r * ld;
        tab = which || !half ? nullptr : A.n.rope + (size_t) (lo + r) * 2 * half;
        return i & (pairs - 1);
    }, half, [&](int i, int e0, int e1, double a, double b) {
        const float x = (float) a, y = (float) b;
        float * to = lrow + (i >> sh) * hd;
        to[e0] = x;
        to[e1] = y;
        big = max(big, max(__float_as_uint(x) & 0x7fffffffu, __float_as_uint(y) & 0x7fffffffu));
    });
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) big = max(big, (uint32_t) __shfl_xor((int) big, o, 64));
    if ((tid & 63) == 0) lmax[tid >> 6] = big;
    __syncthreads();
#pragma unroll
    for (int w2 = 0; w2 < NT / 64; w2++) big = max(big, lmax[w2]);
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
        for (int k = tid; k < (held + rows - first) * per; k += NT) {
            const int r = first + (k >> (sh - 3)), d = 16 * (k & (per - 1));
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
        for (int k = tid; k < 4 * hd; k += NT) {
            const int g = k >> (sh + 1), d = k & (hd - 1);
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

/* N neighbouring values, N a multiple of 4, aligned to four of them */
template <int N>
__device__ __forceinline__ void kv_store4(float * p, const float * x) {
#pragma unroll
    for (int k = 0; k < N; k += 4) *(float4 *) (p + k) = float4{x[k], x[k + 1], x[k + 2], x[k + 3]};
}
template <int N>
__device__ __forceinline__ void kv_store4(uint16_t * p, const float * x) {
#pragma unroll
    for (int k = 0; k < N; k += 4)
        *(uint2 *) (p + k) = uint2{(uint32_t) kv_bf16(x[k]) | (uint32_t) kv_bf16(x[k + 1]) << 16,
                                   (uint32_t) kv_bf16(x[k + 2]) | (uint32_t) kv_bf16(x[k + 3]) << 16};
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
    if (!which) {
        const int per = hd / 16, cnt = (int) (hi - lo) * per;
        for (int k = tid; k < cnt; k += 256) {
            const int r = (int) (lo - p0) + k / per, d = 16 * (k % per);
            union { int4 v; int8_t c[16]; } u;
            u.v = have ? *(const int4 *) (codes + kv_key_at(r, d)) : int4{0, 0, 0, 0};
            float x[16];
#pragma unroll
            for (int e = 0; e < 16; e++) x[e] = (float) u.c[e] * s;
            kv_store4<16>(out + (size_t) (p0 + r - f) * row + d, x);
        }
    } else {
        /* four elements of 16 positions a thread */
        for (int k = tid; k < hd; k += 256) {
            const int g = k / (hd / 4), d = 4 * (k % (hd / 4));
            union { int4 v; int8_t c[16]; } u[4];
#pragma unroll
            for (int w = 0; w < 4; w++) u[w].v = have ? *(const int4 *) (codes + (size_t) (g * hd + d + w) * 16) : int4{0, 0, 0, 0};
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const long p = p0 + 16 * (e >> 2) + 4 * g + (e & 3);
                float x[4];
#pragma unroll
                for (int w = 0; w < 4; w++) x[w] = (float) u[w].c[e] * s;
                if (p >= lo && p < hi) kv_store4<4>(out + (size_t) (p - f) * row + d, x);
            }
        }
    }
}

}  // namespace

/* ------------------------------------------------------------------ checks */

bool kv_aligned(const void * p, size_t n) { return ((uintptr_t) p & (n - 1)) == 0; }

int kv_check_dtype(const char * what, int dtype) {
    if (dtype == SPARKMV_X_F32 || dtype == SPARKMV_X_BF16) return 0;
    set_error("%s: unknown type %d", what, dtype);
    return -1;
}

/* rows of n values at stride ld, each starting 16-byte aligned */
int kv_check_rows(const char * what, const void * p, int ld, long n, int dtype, int nrows) {
    if (!p) { set_error("%s is null", what); return -1; }
    if (nrows > 1 && ld < n) { set_error("%s: a row stride of %d holds no %ld values", what, ld, n); return -1; }
    if (!kv_aligned(p, 16) || (nrows > 1 && (size_t) ld * (dtype == SPARKMV_X_F32 ? 4 : 2) % 16)) {
        set_error("%s: rows do not start 16-byte aligned", what);
        return -1;
    }
    return 0;
}

int kv_check_launch(const char * what) {
    hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : fail_hip(what, e);
}

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
    if (!kv_aligned(c->k, 16) || !kv_aligned(c->v, 16)) { set_error("kv cache codes are not 16-byte aligned"); return -1; }
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
    return kv_check_launch("rope table launch");
}

int sparkmv_kv_append(const sparkmv_kv_cache * cache, const sparkmv_kv_batch * batch, const sparkmv_kv_new * rows,
                      void * stream) {
    if (kv_check_cache(cache) || kv_check_batch(batch)) return -1;
    if (!rows) { set_error("kv rows are null"); return -1; }
    const sparkmv_kv_new & n = *rows;
    const int hd = cache->head_dim;
    if (kv_check_dtype("kv rows", n.x_dtype)) return -1;
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
    if (kv_check_rows("keys", n.k, n.ldk, kvd, n.x_dtype, batch->ntok) ||
        kv_check_rows("values", n.v, n.ldv, kvd, n.x_dtype, batch->ntok))
        return -1;
    if (n.heads && (kv_check_rows("queries", n.q, n.ldq, qd, n.x_dtype, batch->ntok) ||
                    kv_check_rows("rotated queries", n.q_out, n.ldqo, qd, n.x_dtype, batch->ntok)))
        return -1;
    const int max_q = batch->max_q < batch->ntok ? batch->max_q : batch->ntok;
    KvAppend a;
    a.c = *cache; a.b = *batch; a.n = n;
    a.b.max_q = batch->qstart ? max_q : 1;
    a.half = n.rope_dim / 2;
    a.nb = (a.b.max_q + kKvPage - 2) / kKvPage + 1;
    if (a.nb > cache->max_pages) a.nb = cache->max_pages;
    /* 1024 threads from 9 rows a page on: 64 rows x 256 elements are 8192 pairs,
     * of which 256 threads took 32 each (a chunk of 512 tokens 33 us); one row
     * gives 256 threads no work for more */
    const bool wide = a.b.max_q > 8;
    const int nt = wide ? 1024 : 256;
    a.qparts = (n.heads + nt / 64 - 1) / (nt / 64);
    const long nkv = (long) batch->nseq * a.nb * cache->kv_heads * 2, wgs = nkv + (long) batch->ntok * a.qparts;
    if (wgs > 0x7fffffffl) { set_error("an append of %ld workgroups", wgs); return -1; }
    a.nkv = (int) nkv;
    const int lrows = a.b.max_q < kKvPage ? a.b.max_q : kKvPage;
    const uint32_t lds = (uint32_t) (lrows * hd * 4);
    const dim3 grid((unsigned) wgs), block((unsigned) nt);
    hipStream_t s = (hipStream_t) stream;
    /* a full page of 256 elements takes 64 KB beside the kernel's own words */
#define KV_APPEND(X, NT)                                                                                             \
    do {                                                                                                             \
        static LdsAllowed allowed;                                                                                   \
        if (lds_allow(allowed, (const void *) kv_append_kernel<X, NT>, lds + 1024, "LDS opt-in for the kv append"))  \
            return -1;                                                                                               \
        hipLaunchKernelGGL((kv_append_kernel<X, NT>), grid, block, lds, s, a);                                       \
    } while (0)
    if (n.x_dtype == SPARKMV_X_F32) {
        if (wide) KV_APPEND(float, 1024);
        else KV_APPEND(float, 256);
    } else {
        if (wide) KV_APPEND(uint16_t, 1024);
        else KV_APPEND(uint16_t, 256);
    }
#undef KV_APPEND
    return kv_check_launch("kv append launch");
}

int sparkmv_kv_read(const sparkmv_kv_cache * cache, int nseq, const int * slot, const int * from, int n, void * k_out,
                    void * v_out, int out_dtype, void * stream) {
    if (kv_check_cache(cache) || kv_check_dtype("kv read", out_dtype)) return -1;
    if (nseq < 0 || nseq > kKvMaxSeq) { set_error("%d sequences are outside 0..%d", nseq, kKvMaxSeq); return -1; }
    if (n < 0) { set_error("%d positions", n); return -1; }
    if (nseq == 0 || n == 0 || (!k_out && !v_out)) return 0;
    if (!from) { set_error("kv read has no positions"); return -1; }
    if (!kv_aligned(k_out, 16) || !kv_aligned(v_out, 16)) { set_error("kv read: rows do not start 16-byte aligned"); return -1; }
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
    return kv_check_launch("kv read launch");
}

}  // extern "C"
