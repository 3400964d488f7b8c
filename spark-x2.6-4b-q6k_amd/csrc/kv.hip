/* kv.hip — the paged 8-bit cache: the append with the position rotation on the
 * way, reading positions back, and the checks of its calls (include/sparkmv.h
 * has the cache's layout and its rules; kv.h the offsets of a code; kv_attend.hip
 * attention over it). */
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
    const double back = (double) f;
    const uint32_t off = (uint32_t) (back != v) & (uint32_t) (fabsf(f) < INFINITY);
    /* one step back where it was rounded away from zero */
    const uint32_t u = __float_as_uint(f) - (off & (uint32_t) (fabs(back) > fabs(v)));
    *p = kv_bf16(__uint_as_float(u | off));
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
 * values) each, the others some of the tokens' queries.
 *
 * A page's workgroup holds its new rows in registers (a thread up to kKvPairs
 * pairs of elements), takes their largest magnitude, settles the scale, puts the
 * codes in LDS and writes them in 16 byte pieces of the layout; pieces that also
 * hold older positions are read first, as soon as the page is known. Nothing
 * else writes the page's head during the launch. One token is bound by its chain
 * of reads (position, page, scale and piece), a chunk by its rows.
 *
 * The arithmetic is fixed to the bit, so that a code does not depend on how a
 * compiler orders a sum: the rotation in 64 bits (products of f32 are exact
 * there), the scale from 64 bits, the code as the nearest integer of the exact
 * quotient. That one is found in f32: n0 = rint(x * (1 / s)) is off by one at
 * most, and x - s n0, one fma, is exact (its bits lie between the last place
 * of s or x and s, and s is not below 2^-126), so comparing it with s / 2
 * settles the rounding. */
struct KvAppend {
    sparkmv_kv_cache c;
    sparkmv_kv_batch b;
    sparkmv_kv_new n;
    int nb;              /* pages a sequence's new tokens may touch */
    int nkv;             /* workgroups of pages */
    int qtok, qparts;    /* tokens of a workgroup of queries, or workgroups of a token */
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

/* up to four pairs and their turns, requested together and then turned: at(u, row,
 * tab) gives the u-th pair's place in its head, its row and its table row (used
 * with rot, a uniform truth, only). Only `live` of them, a uniform count, are
 * there: a call of one token steps over the others' instructions, which it would
 * otherwise fetch */
constexpr int kKvPairs = 4;
template <typename X, typename At>
__device__ __forceinline__ void kv_turn(At at, int live, bool rot, int half, double * a, double * b) {
    float x[kKvPairs], y[kKvPairs], c[kKvPairs], s[kKvPairs];
    bool turn[kKvPairs];
#pragma unroll
    for (int u = 0; u < kKvPairs; u++) {
        if (u >= live) break;
        const X * row;
        const float * tab = nullptr;
        const int j = at(u, row, tab);
        int e1;
        const int e0 = kv_pair(j, half, e1);
        x[u] = kv_load(row + e0);
        y[u] = kv_load(row + e1);
        turn[u] = rot & (j < half);
        c[u] = 1.0f;
        s[u] = 0.0f;
        if (rot) {
            c[u] = tab[min(j, half - 1)];
            s[u] = tab[half + min(j, half - 1)];
        }
    }
#pragma unroll
    for (int u = 0; u < kKvPairs; u++) {
        if (u >= live) break;
        const double p = (double) x[u], q = (double) y[u], cc = (double) c[u], ss = (double) s[u];
        a[u] = turn[u] ? p * cc - q * ss : p;
        b[u] = turn[u] ? q * cc + p * ss : q;
    }
}

/* nearest integer of x / s (ties to even), |x / s| <= 127.5; r is f32(1 / s). Without
 * branches: sixteen of them a thread were half of the kernel's instructions */
__device__ __forceinline__ int kv_code(float x, float s, float r) {
    const float n = rintf(x * r), e = fmaf(-s, n, x), e2 = 2.0f * fabsf(e);
    const int i = (int) n, off = (int) (e2 > s) | ((int) (e2 == s) & i);
    return i + (off & 1) * (e > 0.0f ? 1 : -1);
}
/* the same of a product of a code and its old scale, exact in 64 bits */
__device__ __forceinline__ int kv_code(double x, double s, float r) {
    const double n = rint(x * (double) r), e = fma(-s, n, x), e2 = 2.0 * fabs(e);
    const int i = (int) n, off = (int) (e2 > s) | ((int) (e2 == s) & i);
    return i + (off & 1) * (e > 0.0 ? 1 : -1);
}

constexpr int kv_append_rows(int nt) { return nt == 256 ? 8 : kKvPage; }   /* new rows of a page, at most */

/* 256 threads: 8 rows of up to 256 elements; 512: 64 rows of up to 128; 1024: 64 of 256 */
template <typename X, int NT>
__global__ __launch_bounds__(NT, NT == 256 ? 1 : 8) void kv_append_kernel(const KvAppend A) {
    constexpr int U = NT == 256 ? 4 : 8, NP = NT == 256 ? 4 : 1;   /* pairs and pieces a thread, at most */
    __shared__ __attribute__((aligned(16))) int8_t lcode[kKvPage * 256];
    __shared__ uint32_t lmax[NT / 64];
    const int tid = threadIdx.x, hd = A.c.head_dim, kvh = A.c.kv_heads, half = A.half;
    const int sh = 31 - __clz(hd / 2), pairs = 1 << sh;   /* head_dim is a power of two */
    if ((int) blockIdx.x >= A.nkv) {
        /* queries */
        int * lpos = (int *) lcode;                        /* [qtok], at most NT * kKvPairs / 32 */
        const int w = (int) blockIdx.x - A.nkv, t0 = w / A.qparts * A.qtok, per = A.n.heads << sh;
        const int first = w % A.qparts * (NT * kKvPairs);   /* 0 where a workgroup takes whole tokens */
        const int n = A.qparts > 1 ? min(per, first + NT * kKvPairs) : min(A.qtok, A.b.ntok - t0) * per;
#pragma unroll 1
        for (int i = tid; i < A.qtok; i += NT) lpos[i] = -1;
        __syncthreads();
#pragma unroll 1
        for (int i = tid; i < A.b.nseq; i += NT) {
            const KvSeq s = kv_seq(A.b, i, A.c.nslots, A.c.max_pages);
#pragma unroll 1
            for (int t = max(s.row, t0); t < min(s.row + s.count, t0 + A.qtok); t++) lpos[t - t0] = s.pos + t - s.row;
        }
        __syncthreads();
#pragma unroll 1
        for (int j0 = first; j0 < n; j0 += NT * kKvPairs) {
            const int i0 = j0 + tid, live = (n - j0 + NT - 1) / NT;
            double a[kKvPairs], b[kKvPairs];
            kv_turn<X>([&](int u, const X *& row, const float *& tab) {
                const int k = min(i0 + u * NT, n - 1), t = A.qparts > 1 ? 0 : k / per, e = k - t * per, pos = lpos[t];
                row = (const X *) A.n.q + (size_t) (t0 + t) * A.n.ldq + (size_t) (e >> sh) * hd;
                tab = A.n.rope + (size_t) max(pos, 0) * 2 * half;
                return e & (pairs - 1);
            }, live, half > 0, half, a, b);
#pragma unroll
            for (int u = 0; u < kKvPairs; u++) {
                if (u >= live) break;
                const int k = i0 + u * NT;
                if (k >= n) continue;
                const int t = A.qparts > 1 ? 0 : k / per, e = k - t * per;
                if (lpos[t] < 0) continue;
                X * to = (X *) A.n.q_out + (size_t) (t0 + t) * A.n.ldqo + (size_t) (e >> sh) * hd;
                int e1;
                const int e0 = kv_pair(e & (pairs - 1), half, e1);
                kv_store_wide(to + e0, a[u]);
                kv_store_wide(to + e1, b[u]);
            }
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
    const int lo = max(s.pos, p0), hi = min(end, p0 + kKvPage), held = lo - p0, rows = hi - lo, upto = held + rows;
    /* the rows' pairs, requested before the page is looked at */
    const X * src = (const X *) (which ? A.n.v : A.n.k) + (size_t) h * hd;
    const int ld = which ? A.n.ldv : A.n.ldk, np = rows << sh;
    float x[U], y[U];
    uint32_t big = 0;
    const int live = (np + NT - 1) / NT;
#pragma unroll
    for (int v = 0; v < U; v += kKvPairs) {
        if (v >= live) break;
        double a[kKvPairs], b[kKvPairs];
        kv_turn<X>([&](int u, const X *& row, const float *& tab) {
            const int k = min(tid + (v + u) * NT, np - 1), r = k >> sh;
            row = src + (size_t) (s.row + lo + r - s.pos) * ld;
            tab = A.n.rope + (size_t) (lo + r) * 2 * half;
            return k & (pairs - 1);
        }, live - v, !which && half > 0, half, a, b);
#pragma unroll
        for (int u = 0; u < kKvPairs; u++) {
            if (v + u >= live) break;
            x[v + u] = (float) a[u];
            y[v + u] = (float) b[u];
            big = max(big, max(__float_as_uint(x[v + u]) & 0x7fffffffu, __float_as_uint(y[v + u]) & 0x7fffffffu));
        }
    }
    if (page < 0 || page >= A.c.npages) return;
    float * scale = (which ? A.c.v_scale : A.c.k_scale) + (size_t) page * kvh + h;
    int8_t * codes = (which ? A.c.v : A.c.k) + ((size_t) page * kvh + h) * (size_t) (kKvPage * hd);
    const float was = held ? *scale : 0.0f;
    /* the values' pieces that hold older positions beside new ones: piece u of a
     * thread is of group gu; only groups with a new position are touched */
    union Piece { int4 v; uint32_t w[4]; int8_t c[16]; };
    Piece piece[NP];
    auto group = [&](int u) { return (tid + u * NT) >> (sh + 1); };
    auto touched = [&](int g, int from) {   /* whether one of from .. upto - 1 is in group g */
        return ((g - (from >> 2)) & 3) <= ((upto - 1) >> 2) - (from >> 2);
    };
    if (which && (held > 0 || upto < kKvPage)) {
#pragma unroll
        for (int u = 0; u < NP; u++)
            if (group(u) < 4 && touched(group(u), held)) piece[u].v = *(const int4 *) (codes + (size_t) (tid + u * NT) * 16);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) big = max(big, (uint32_t) __shfl_xor((int) big, o, 64));
    if ((tid & 63) == 0) lmax[tid >> 6] = big;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NT / 64; k++) big = max(big, lmax[k]);
    const double need = (double) __uint_as_float(big);
    const bool bad = big >= 0x7f800000u || was != was;
    const bool keep = held && was > 0.0f && need <= 127.0 * (double) was;
    const float now = bad ? __uint_as_float(0x7fc00000u)
                          : (keep ? was : fmaxf((float) (need * (hi == p0 + kKvPage ? 1.0 : 1.25) / 127.0), 1.17549435e-38f));
    if ((!keep || bad) && tid == 0) *scale = now;
    const float inv = 1.0f / now;
    const bool again = held && !keep && !bad;   /* older codes rounded anew */
    auto old_code = [&](int c) -> int8_t { return (int8_t) kv_code((double) c * (double) was, (double) now, inv); };
    /* codes to LDS: keys by row, values as they lie in a page */
#pragma unroll
    for (int u = 0; u < U; u++) {
        if (u >= live) break;
        const int k = tid + u * NT, r = k >> sh;
        if (k >= np) continue;
        int e1;
        const int e0 = kv_pair(k & (pairs - 1), half, e1);
        const int a = bad ? 0 : kv_code(x[u], now, inv), b = bad ? 0 : kv_code(y[u], now, inv);
        lcode[which ? kv_value_at(held + r, e0, hd) : r * hd + e0] = (int8_t) a;
        lcode[which ? kv_value_at(held + r, e1, hd) : r * hd + e1] = (int8_t) b;
    }
    __syncthreads();
    if (!which) {
        const int per = hd / 16;   /* pieces of a position */
#pragma unroll 1
        for (int k = tid; k < rows * per; k += NT) {
            const int r = k >> (sh - 3), d = 16 * (k & (per - 1));
            *(int4 *) (codes + kv_key_at(held + r, d)) = *(const int4 *) (lcode + r * hd + d);
        }
        if (again)
#pragma unroll 1
            for (int k = tid; k < held * per; k += NT) {
                Piece q;
                int4 * at = (int4 *) (codes + kv_key_at(k >> (sh - 3), 16 * (k & (per - 1))));
                q.v = *at;
#pragma unroll
                for (int e = 0; e < 16; e++) q.c[e] = old_code(q.c[e]);
                *at = q.v;
            }
        return;
    }
    /* positions from .. upto - 1 of a page come from LDS, the others stay */
    const int from = again ? 0 : held;
    if (again) {
#pragma unroll 1
        for (int k = tid; k < 4 * hd; k += NT) {
            Piece q;
            q.v = *(const int4 *) (codes + (size_t) k * 16);
#pragma unroll
            for (int e = 0; e < 16; e++)
                if (16 * (e >> 2) + 4 * (k >> (sh + 1)) + (e & 3) < held) lcode[16 * k + e] = old_code(q.c[e]);
        }
    }
#pragma unroll
    for (int u = 0; u < NP; u++) {
        const int k = tid + u * NT, g = group(u);
        if (g >= 4 || !touched(g, from)) continue;
        Piece q;
        q.v = *(const int4 *) (lcode + 16 * k);
        if (from > 0 || upto < kKvPage) {
            if (again) piece[u].v = *(const int4 *) (codes + (size_t) k * 16);
#pragma unroll
            for (int t = 0; t < 4; t++) {
                /* bytes lo4 .. hi4 - 1 of the word */
                const int b = 16 * t + 4 * g, lo4 = min(max(from - b, 0), 4), hi4 = min(max(upto - b, 0), 4);
                const uint32_t m = (uint32_t) ((1ull << (8 * hi4)) - (1ull << (8 * lo4)));
                q.w[t] = hi4 > lo4 ? (q.w[t] & m) | (piece[u].w[t] & ~m) : piece[u].w[t];
            }
        }
        *(int4 *) (codes + (size_t) k * 16) = q.v;
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
        *(uint2 *) (p + k) = uint2{kv_bf16x2(x[k], x[k + 1]), kv_bf16x2(x[k + 2], x[k + 3])};
}

/* ---------------------------------------------------------------------- read
 * One workgroup per (sequence, page its positions touch, kv head, keys or
 * values). Bound by its chain (position, page number, codes, stores): one page of
 * 4 heads 4.9 us, 64 pages 10.6 (8.4 MB in, 16.8 out). */
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
        /* 64 positions of 256 elements are four pieces a thread, requested together:
         * one after another they took 2 us more */
        const int lg = 31 - __clz(hd / 16), cnt = (int) (hi - lo) << lg, r0 = (int) (lo - p0);
        union { int4 v; int8_t c[16]; } u[4];
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const int k = tid + 256 * w;
            if (256 * w < cnt && have) u[w].v = *(const int4 *) (codes + kv_key_at(r0 + (min(k, cnt - 1) >> lg), 16 * (k & ((1 << lg) - 1))));
            else u[w].v = int4{0, 0, 0, 0};
        }
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const int k = tid + 256 * w, r = r0 + (k >> lg), d = 16 * (k & ((1 << lg) - 1));
            if (k >= cnt) continue;
            float x[16];
#pragma unroll
            for (int e = 0; e < 16; e++) x[e] = (float) u[w].c[e] * s;
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
    if (wg > kKvThreads / 256) { set_error("rope table of %d rows and %d values is too large", rows, rope_dim); return -1; }
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
    /* an array of no rows may be null */
    const bool any = batch->nseq > 0 && batch->ntok > 0;
    if (n.heads < 0 || (any && ((n.heads > 0) != (n.q != nullptr) || (n.heads > 0) != (n.q_out != nullptr)))) {
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
    if (n.heads && n.q == n.q_out && n.ldq != n.ldqo && batch->ntok > 1) {
        set_error("queries rotated in place with two row strides, %d and %d", n.ldq, n.ldqo);
        return -1;
    }
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
    const long nb = ((long) a.b.max_q + kKvPage - 2) / kKvPage + 1;
    a.nb = (int) (nb < cache->max_pages ? nb : cache->max_pages);
    /* 256 threads hold eight rows of a page, 512 all 64 of up to 128 elements, 1024
     * of 256: with 256 threads the rows of a chunk of 512 tokens came in 32 turns, 33
     * us, with 1024 it takes 13.6; one row gives no more than 128 threads a pair (64
     * tokens of 64 sequences 7.6 us, one 4.3) */
    const int nt = a.b.max_q <= kv_append_rows(256) ? 256 : (hd <= 128 ? 512 : 1024);
    const int qpairs = nt * kKvPairs, per = n.heads * (hd / 2);
    a.qtok = per && per <= qpairs ? qpairs / per : 1;
    a.qparts = per > qpairs ? (per + qpairs - 1) / qpairs : 1;
    const long nkv = (long) batch->nseq * a.nb * cache->kv_heads * 2;
    const long wgs = nkv + (n.heads ? ((long) batch->ntok + a.qtok - 1) / a.qtok * a.qparts : 0);
    if (wgs > kKvThreads / nt) { set_error("an append of %ld workgroups is too much for one call", wgs); return -1; }
    a.nkv = (int) nkv;
    const dim3 grid((unsigned) wgs), block((unsigned) nt);
    hipStream_t s = (hipStream_t) stream;
#define KV_APPEND(X, NT) hipLaunchKernelGGL((kv_append_kernel<X, NT>), grid, block, 0, s, a)
#define KV_APPEND_NT(X)                                                                                              \
    do {                                                                                                             \
        if (nt == 256) KV_APPEND(X, 256);                                                                            \
        else if (nt == 512) KV_APPEND(X, 512);                                                                       \
        else KV_APPEND(X, 1024);                                                                                     \
    } while (0)
    if (n.x_dtype == SPARKMV_X_F32) KV_APPEND_NT(float);
    else KV_APPEND_NT(uint16_t);
#undef KV_APPEND_NT
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
    const long nb = ((long) n + kKvPage - 2) / kKvPage + 1, wgs = (long) nseq * nb;
    if (wgs > kKvThreads / 256) { set_error("a read of %ld pages is too much for one call", wgs); return -1; }
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
