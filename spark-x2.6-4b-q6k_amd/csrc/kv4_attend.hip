/* kv4_attend.hip — attention over the paged 4-bit cache (include/sparkmv.h):
 *   out = sum_p softmax_p(scale * q . k_p) v_p (* sigmoid(gate))
 * over the positions p that a token sees.
 *
 * Codes become bf16 with their scale in one instruction a pair, exactly, and both
 * products run on the bf16 matrix instruction, 16 x 16 x 32, which keeps an f32 sum.
 * What meets the codes is an f32 query element or weight as a sum of bf16 numbers:
 *
 *   a query element as three, each the leading 8 bits of what the ones before left
 *   out, which is all of f32; bf16 queries need one;
 *
 *   a weight e^(s - m) as three for f32 outputs, again all of it, and as two for
 *   bf16 ones, 2^-17 of it at most being lost.
 *
 * m is a running reference of the column that moves only when a page passes it by
 * 2^kKvLag. Scores, statistics and sums are f32. */
#include <math.h>

#include "kv4.h"
#include "kv_attend.h"

namespace sparkmv {

namespace {

typedef uint32_t kv4_u2 __attribute__((ext_vector_type(2)));
typedef uint32_t kv4_u4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ kv4_b8 kv4_operand(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_bit_cast(kv4_b8, kv4_u4{a, b, c, d});
}

/* eight query elements as D bf16 operands */
template <int D>
__device__ __forceinline__ void kv4_split8(const float * x, kv4_u4 * out) {
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; i++) r[i] = x[i];
#pragma unroll
    for (int d = 0; d < D; d++)
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const uint32_t a = __float_as_uint(r[2 * k]), b = __float_as_uint(r[2 * k + 1]);
            out[d][k] = __builtin_amdgcn_perm(b, a, 0x07060302u);
            r[2 * k] -= __uint_as_float(a & 0xffff0000u);
            r[2 * k + 1] -= __uint_as_float(b & 0xffff0000u);
        }
}

/* which of four scale bytes are not a number (kKv4High): bit 7 of each */
__device__ __forceinline__ uint32_t kv4_bad(uint32_t x) { return ((x & 0x7f7f7f7fu) + 0x03030303u) & x & 0x80808080u; }

constexpr int kKv4Cols = 16;      /* columns (token, query head) of a tile */
constexpr int kKv4Item = 8;       /* pages that beginning a tile's kv head counts */
constexpr int kKv4Most = 1024;    /* workgroups of shares, at most */

struct Kv4Flat {
    sparkmv_kv4_cache c;
    sparkmv_kv_batch b;
    sparkmv_kv_query q;
    int cmax;        /* columns of a tile, at most */
    int * pre;       /* [nseq + 2]: what one kv head of the sequences before counts; the share */
    float * po;      /* [workgroups][2][cmax][HD] */
    float * pml;     /* [workgroups][2][cmax][2] */
};

/* what a kv head of a sequence counts: its tiles, each with the pages of all of the
 * sequence's tokens (exact where there is one tile) and what beginning it costs */
__device__ __forceinline__ int kv4_cost(const KvSeq & s, int G, int window, int & tiles) {
    int first;
    tiles = (int) (((long) s.count * G + kKv4Cols - 1) / kKv4Cols);
    return s.count > 0 ? kv_span(s, 0, s.count, window, first) + kKv4Item : 0;
}

constexpr int kv4_lds(int hd, int dq, int waves, int cmax) {
    const int q = dq * (hd / 32) * 1024, o = waves * cmax * (hd + 4) * 4;
    return q > o ? q : o;
}

/* ------------------------------------------------------------- few columns
 *
 * A workgroup takes tiles of up to 16 columns of a kv head; its waves take pages in
 * turn and their results meet in LDS. WAVES 4: equal shares of all (sequence, tile,
 * kv head, page); 8: a whole tile and kv head, nothing to join. */
template <int HD, int DQ, int DP, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void kv4_flat_kernel(const Kv4Flat A) {
    constexpr int NW = HD / 32, ND = HD / 16, NB = HD / 32, NT = 64 * WAVES, LO = HD + 4;
    constexpr int KB = HD / 8;                       /* bytes of keys a lane and 16 positions */
    constexpr int NJ = HD >= 128 ? HD / 128 : 1;     /* scales of keys a lane and 16 positions */
    constexpr int NL = ND / 4;                       /* 16-byte pieces of values a lane and 32 positions */
    constexpr bool WHOLE = WAVES == 8;
    extern __shared__ __attribute__((aligned(16))) uint8_t ldyn[];
    float * lo = (float *) ldyn;                     /* [WAVES][cmax][LO]: a wave's output */
    kv4_u4 * lq = (kv4_u4 *) ldyn;                   /* [DQ][NW][64]: the queries as the lanes take them */
    __shared__ int lsum[8];
    __shared__ float lm[WAVES][16], ll[WAVES][16];
    int * lpre = (int *) (ldyn + kv4_lds(HD, DQ, WAVES, A.cmax));   /* [nseq + 1] */
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 4, c16 = lane & 15;
    const int kvh = A.c.kv_heads, G = A.q.heads / kvh, nseq = A.b.nseq;
    int ubeg = blockIdx.x, uend = ubeg + 1;
    if constexpr (!WHOLE) {
        const int per = (nseq + NT - 1) / NT, i0 = min(nseq, tid * per), i1 = min(nseq, i0 + per);
        int sum = 0;
        for (int i = i0; i < i1; i++) {
            int tiles;
            lpre[i] = sum;
            const int cost = kv4_cost(kv_seq(A.b, i, A.c.nslots, A.c.max_pages), G, A.q.window, tiles);
            sum += cost * tiles;
        }
        int scan = sum;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(scan, o, 64);
            if (lane >= o) scan += v;
        }
        if (lane == 63) lsum[wave] = scan;
        __syncthreads();
        int base = scan - sum;
        for (int w = 0; w < wave; w++) base += lsum[w];
        for (int i = i0; i < i1; i++) lpre[i] += base;
        if (tid == NT - 1) lpre[nseq] = base + sum;
        __syncthreads();
        const int total = __builtin_amdgcn_readfirstlane(lpre[nseq]);
        const int share = max((int) (((long) total * kvh + gridDim.x - 1) / gridDim.x), 1);
        if (blockIdx.x == 0) {
            for (int i = tid; i <= nseq; i += NT) A.pre[i] = lpre[i];
            if (tid == 0) A.pre[nseq + 1] = share;
        }
        ubeg = (int) min((long) blockIdx.x * share, (long) total * kvh);
        uend = (int) min((long) ubeg + share, (long) total * kvh);
    }
    for (int u = ubeg; u < uend;) {
        int h, off = 0, n, seg, first, place = 0, i;
        KvSeq s;
        if constexpr (WHOLE) {
            i = u / kvh;
            h = u - i * kvh;
        } else {
            i = 0;
            for (int b = nseq; b - i > 1;) {
                const int mid = (i + b) >> 1;
                if ((long) __builtin_amdgcn_readfirstlane(lpre[mid]) * kvh <= u) i = mid;
                else b = mid;
            }
        }
        s = kv_seq(A.b, i, A.c.nslots, A.c.max_pages);
        s.slot = __builtin_amdgcn_readfirstlane(s.slot);
        s.pos = __builtin_amdgcn_readfirstlane(s.pos);
        s.row = __builtin_amdgcn_readfirstlane(s.row);
        s.count = __builtin_amdgcn_readfirstlane(s.count);
        if constexpr (WHOLE) {
            if (s.count <= 0) return;
        } else {
            int tiles;
            const int in = u - __builtin_amdgcn_readfirstlane(lpre[i]) * kvh, cost = kv4_cost(s, G, A.q.window, tiles);
            const int item = in / cost;
            h = item / tiles;
            place = item - h * tiles;
            off = in - item * cost;
        }
        const int ncols = s.count * G, col0 = place * kKv4Cols, ncol = min(kKv4Cols, ncols - col0);
        const int t0 = col0 / G, t1 = (col0 + ncol - 1) / G + 1;
        n = kv_span(s, t0, t1, A.q.window, first);
        if constexpr (WHOLE) {
            seg = n;
        } else {
            if (off >= n) {
                int tiles;
                u += kv4_cost(s, G, A.q.window, tiles) - off;
                continue;
            }
            seg = min(n - off, uend - u);
        }
        /* the queries: eight elements of a column a thread */
        for (int k = tid; k < NW * 64; k += NT) {
            const int w = k >> 6, ql = k & 63, qc = ql & 15, qg = ql >> 4;
            const int d = HD >= 128 ? 32 * (4 * (w >> 2) + qg) + 8 * (w & 3) : 16 * qg + 8 * w;
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = 0.0f;
            if (qc < ncol) {
                const int t = (col0 + qc) / G, head = h * G + (col0 + qc) - t * G;
                const size_t at = (size_t) (s.row + t) * A.q.ldq + (size_t) head * HD + d;
                if (DQ == 3) {
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const kv_f4 v = *(const kv_f4 *) ((const float *) A.q.q + at + 4 * e);
#pragma unroll
                        for (int f = 0; f < 4; f++) x[4 * e + f] = v[f];
                    }
                } else {
                    const kv4_u4 v = *(const kv4_u4 *) ((const uint16_t *) A.q.q + at);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        x[2 * e] = __uint_as_float(v[e] << 16);
                        x[2 * e + 1] = __uint_as_float(v[e] & 0xffff0000u);
                    }
                }
            }
            kv4_u4 o[DQ];
            kv4_split8<DQ>(x, o);
#pragma unroll
            for (int d2 = 0; d2 < DQ; d2++) lq[(d2 * NW + w) * 64 + ql] = o[d2];
        }
        __syncthreads();
        const int col = min(c16, ncol - 1), tok = (col0 + col) / G, pos_c = s.pos + tok;
        const int beg_c = A.q.window > 0 && pos_c + 1 > A.q.window ? pos_c + 1 - A.q.window : 0;
        /* positions that every column sees */
        const int all_lo = A.q.window > 0 && s.pos + t1 > A.q.window ? s.pos + t1 - A.q.window : 0, all_hi = s.pos + t0;
        const int * table = A.c.pages + (size_t) s.slot * A.c.max_pages + first + off;
        const float f = A.q.scale * kKvLog2e;
        float m = -INFINITY, l = 0.0f;
        kv_f4 o[ND];
#pragma unroll
        for (int d = 0; d < ND; d++) o[d] = kv_f4{0.f, 0.f, 0.f, 0.f};
        for (int j = wave; j < seg; j += WAVES) {
            int id = __builtin_amdgcn_readfirstlane(table[j]);
            const bool ok = id >= 0 && id < A.c.npages;
            const uint8_t * page = A.c.data + ((size_t) (ok ? id : 0) * kvh + h) * (size_t) kv4_head_bytes(HD);
            uint32_t kr[4][KB / 4], ks[(4 * NJ + 3) / 4], vs[4];
            kv4_u4 vr[2][NL];
#pragma unroll
            for (int t = 0; t < 4; t++) {
                if constexpr (HD >= 128) {
#pragma unroll
                    for (int jj = 0; jj < NJ; jj++) {
                        const kv4_u4 v = *(const kv4_u4 *) (page + ((t * NJ + jj) * 64 + lane) * 16);
#pragma unroll
                        for (int e = 0; e < 4; e++) kr[t][4 * jj + e] = v[e];
                    }
                } else {
                    const kv4_u2 v = *(const kv4_u2 *) (page + (t * 64 + lane) * 8);
                    kr[t][0] = v[0];
                    kr[t][1] = v[1];
                }
            }
#pragma unroll
            for (int w = 0; w < NJ; w++)
                ks[w] = *(const uint32_t *) (page + 64 * HD + ((HD == 64 ? g >> 1 : g) * 16 + c16) * 4 * NJ + 4 * w);
#pragma unroll
            for (int w = 0; w < 2; w++)
#pragma unroll
                for (int k = 0; k < NL; k++) vr[w][k] = *(const kv4_u4 *) (page + 32 * HD + ((w * NL + k) * 64 + lane) * 16);
            {
                const kv4_u4 v = *(const kv4_u4 *) (page + 66 * HD + (g * NB + (c16 * ND) / 32) * 16);
#pragma unroll
                for (int e = 0; e < 4; e++) vs[e] = v[e];
            }
#pragma unroll
            for (int w = 0; w < NJ; w++) ks[w] |= (kv4_bad(ks[w]) >> 7) * 0xffu;
            /* scores: tile t's positions 4 g + e of this lane's column */
            float x[4][4];
#pragma unroll
            for (int t = 0; t < 4; t++) {
                kv_f4 acc = kv_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < NW; w++) {
                    const int k = t * NJ + w / 4;   /* its scale: byte k of ks */
                    const float sc = k % 4 == 0 ? kv4_scale<0>(ks[k / 4]) : (k % 4 == 1 ? kv4_scale<1>(ks[k / 4]) :
                                     (k % 4 == 2 ? kv4_scale<2>(ks[k / 4]) : kv4_scale<3>(ks[k / 4])));
                    const uint32_t c = kr[t][w];
                    const kv4_b8 a = kv4_operand(kv4_pair<0>(c, sc), kv4_pair<1>(c, sc), kv4_pair<2>(c, sc), kv4_pair<3>(c, sc));
#pragma unroll
                    for (int d = DQ - 1; d >= 0; d--)
                        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, __builtin_bit_cast(kv4_b8, lq[(d * NW + w) * 64 + lane]), acc, 0, 0, 0);
                }
#pragma unroll
                for (int e = 0; e < 4; e++) x[t][e] = acc[e] * f;
            }
            const int p0 = (first + off + j) * kKvPage;
            if (!ok || p0 < all_lo || p0 + kKvPage - 1 > all_hi) {
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int p = p0 + 16 * t + 4 * g + e;
                        x[t][e] = ok && p >= beg_c && p <= pos_c ? x[t][e] : -INFINITY;
                    }
            }
            /* values that are not numbers count as zero, and make the columns that see them so */
            if (__any((kv4_bad(vs[0]) | kv4_bad(vs[1]) | kv4_bad(vs[2]) | kv4_bad(vs[3])) != 0)) {
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const uint32_t b = kv4_bad(vs[k]);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const bool here = __ballot(b >> (8 * e + 7) & 1) >> (16 * g) & 0xffff;
                        if (here && x[k][e] != -INFINITY) l = __uint_as_float(0x7fc00000u);
                    }
                    vs[k] &= ~((b >> 7) * 0xffu);
                }
            }
            float mp = -INFINITY;
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) mp = fmaxf(mp, x[t][e]);
            mp = kv_rows_max(mp);
            if (__any(mp > m + kKvLag)) {
                const float mn = fmaxf(m, mp);
                const float r = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
                l *= r;
#pragma unroll
                for (int d = 0; d < ND; d++) o[d] *= r;
                m = mn;
            }
            const float mref = m == -INFINITY ? 0.0f : m;
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    x[t][e] = __builtin_amdgcn_exp2f(x[t][e] - mref);
                    l += x[t][e];
                }
            kv4_u4 P[2][DP];
#pragma unroll
            for (int w = 0; w < 2; w++)
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    float a = x[2 * w + (k >> 1)][2 * (k & 1)], b = x[2 * w + (k >> 1)][2 * (k & 1) + 1];
#pragma unroll
                    for (int d = 0; d < DP; d++) {
                        P[w][d][k] = kv_bf16x2(a, b);
                        a -= __uint_as_float(P[w][d][k] << 16);
                        b -= __uint_as_float(P[w][d][k] & 0xffff0000u);
                    }
                }
#pragma unroll
            for (int w = 0; w < 2; w++) {
#pragma unroll
                for (int k = 0; k < ND / 2; k++) {
                    uint32_t r[8];
#pragma unroll
                    for (int sl = 0; sl < 8; sl++) {
                        const uint32_t sb = vs[2 * w + sl / 4];
                        const float sc = sl % 4 == 0 ? kv4_scale<0>(sb) : (sl % 4 == 1 ? kv4_scale<1>(sb) :
                                         (sl % 4 == 2 ? kv4_scale<2>(sb) : kv4_scale<3>(sb)));
                        const int byte = sl * (ND / 2) + k;   /* of the lane's values */
                        const uint32_t v = vr[w][byte / 16][byte / 4 % 4];
                        r[sl] = byte % 4 == 0 ? kv4_pair<0>(v, sc) : (byte % 4 == 1 ? kv4_pair<1>(v, sc) :
                                (byte % 4 == 2 ? kv4_pair<2>(v, sc) : kv4_pair<3>(v, sc)));
                    }
                    uint32_t a[4], b[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        a[e] = __builtin_amdgcn_perm(r[2 * e + 1], r[2 * e], 0x05040100u);
                        b[e] = __builtin_amdgcn_perm(r[2 * e + 1], r[2 * e], 0x07060302u);
                    }
                    const kv4_b8 va = kv4_operand(a[0], a[1], a[2], a[3]), vb = kv4_operand(b[0], b[1], b[2], b[3]);
#pragma unroll
                    for (int d = DP - 1; d >= 0; d--) {
                        o[2 * k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, __builtin_bit_cast(kv4_b8, P[w][d]), o[2 * k], 0, 0, 0);
                        o[2 * k + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vb, __builtin_bit_cast(kv4_b8, P[w][d]), o[2 * k + 1], 0, 0, 0);
                    }
                }
            }
        }
        l = kv_rows_sum(l);
        __syncthreads();   /* the queries are read */
        /* the waves' outputs meet in LDS: this lane has elements ND (4 g + i) .. of its column */
        if (c16 < ncol) {
#pragma unroll
            for (int i2 = 0; i2 < 4; i2++)
#pragma unroll
                for (int d = 0; d < ND; d += 4)
                    *(kv_f4 *) (lo + (wave * A.cmax + c16) * LO + ND * (4 * g + i2) + d) = kv_f4{o[d][i2], o[d + 1][i2], o[d + 2][i2], o[d + 3][i2]};
            if (g == 0) {
                lm[wave][c16] = m;
                ll[wave][c16] = l;
            }
        }
        __syncthreads();
        const bool whole = WHOLE || seg == n;
        const size_t at = 2 * (size_t) blockIdx.x + (off == 0 ? 1 : 0);
        constexpr int V = 4;
        for (int k = tid; k < ncol * (HD / V); k += NT) {
            const int cc = k / (HD / V), d = V * (k % (HD / V));
            float M = lm[0][cc], L = 0.0f;
#pragma unroll
            for (int w = 1; w < WAVES; w++) M = fmaxf(M, lm[w][cc]);
            kv_f4 v = kv_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < WAVES; w++) {
                const float r = lm[w][cc] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(lm[w][cc] - M);
                L += lm[w][cc] == -INFINITY ? ll[w][cc] : r * ll[w][cc];
                v += r * *(const kv_f4 *) (lo + (w * A.cmax + cc) * LO + d);
            }
            const float y[4] = {v[0], v[1], v[2], v[3]};
            if (whole) {
                const int t = (col0 + cc) / G;
                kv_write<V>(A.q, s.row + t, h * G + (col0 + cc) - t * G, HD, d, y, L);
            } else {
                *(kv_f4 *) (A.po + (at * A.cmax + cc) * HD + d) = v;
                if (d == 0) {
                    A.pml[(at * A.cmax + cc) * 2] = M;
                    A.pml[(at * A.cmax + cc) * 2 + 1] = L;
                }
            }
        }
        __syncthreads();
        u += seg;
    }
}

/* Joins the partial results of one column of a (tile, kv head), in the order of its
 * pages: its first share wrote slot 1, the later ones slot 0. */
template <int HD>
__global__ __launch_bounds__(512) void kv4_flat_join_kernel(const Kv4Flat A) {
    __shared__ float wts[kKv4Most];
    __shared__ __attribute__((aligned(16))) float acc[7 * HD];
    __shared__ int lfind[16];
    const int h = blockIdx.y, c = blockIdx.z, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int kvh = A.c.kv_heads, G = A.q.heads / kvh;
    KvSeq s;
    int place, i;
    if (!kv_find_tile(A.b, A.c, G, kKv4Cols, blockIdx.x, lfind, s, place)) return;
    i = lfind[0];
    int tiles, first;
    const int cost = kv4_cost(s, G, A.q.window, tiles), col0 = place * kKv4Cols, ncol = min(kKv4Cols, s.count * G - col0);
    if (c >= ncol) return;
    const int n = kv_span(s, col0 / G, (col0 + ncol - 1) / G + 1, A.q.window, first), share = A.pre[A.b.nseq + 1];
    const long a = (long) A.pre[i] * kvh + ((long) h * tiles + place) * cost;
    const int w0 = (int) (a / share), w1 = (int) ((a + n - 1) / share);
    if (w0 == w1) return;
    float o[HD / 64];
    const float L = kv_join<HD, 8>(A.po, A.pml, w1 - w0 + 1, [&](int k) { return (2 * (size_t) (w0 + k) + (k == 0)) * A.cmax + c; },
                                   wts, acc, wave, lane, o);
    if (wave) return;
    const int t = (col0 + c) / G;
    kv_write<HD / 64>(A.q, s.row + t, h * G + (col0 + c) - t * G, HD, HD / 64 * lane, o, L);
}

/* -------------------------------------------------------------------- host */

struct Kv4Plan {
    int max_q, cmax;
    bool whole;
    long tiles;
    int groups;
    size_t pre, po, pml, bytes;
};

Kv4Plan kv4_plan(const sparkmv_kv4_cache * c, const sparkmv_kv_batch * b, int heads, int window) {
    Kv4Plan p = {};
    const int G = heads / c->kv_heads;
    p.max_q = b->qstart ? (b->max_q < b->ntok ? b->max_q : b->ntok) : 1;
    const long cols = (long) p.max_q * G, hd = c->head_dim;
    const long len = b->max_len > 0 ? b->max_len : (long) c->max_pages * kKvPage;
    const long pages = (len + kKvPage - 1) / kKvPage;
    size_t off = 0;
    auto take = [&](size_t bytes) { const size_t o = off; off += (bytes + 255) & ~(size_t) 255; return o; };
    p.cmax = (int) (cols < kKv4Cols ? cols : kKv4Cols);
    const long in_window = ((long) window + kKvPage - 2) / kKvPage + 1, seen = window > 0 && in_window < pages ? in_window : pages;
    p.whole = cols <= kKv4Cols && seen <= 16;
    p.tiles = cols <= kKv4Cols ? b->nseq : (long) b->ntok * G / kKv4Cols + b->nseq;
    const long most = 2 * cu_count() < kKv4Most ? 2 * cu_count() : kKv4Most, all = pages * p.tiles * c->kv_heads;
    p.groups = (int) (all < 1 ? 1 : (all < most ? all : most));
    p.pre = take(((size_t) b->nseq + 2) * 4);
    p.po = take((size_t) p.groups * 2 * p.cmax * hd * 4);
    p.pml = take((size_t) p.groups * 2 * p.cmax * 2 * 4);
    p.bytes = off;
    return p;
}

}  // namespace

}  // namespace sparkmv

using namespace sparkmv;

extern "C" {

size_t sparkmv_kv4_attend_work(const sparkmv_kv4_cache * cache, const sparkmv_kv_batch * batch, int heads) {
    if (kv4_check_cache(cache) || kv_check_batch(batch) || heads < 1 || heads % cache->kv_heads) return 0;
    if (batch->nseq == 0 || batch->ntok == 0) return 0;
    return kv4_plan(cache, batch, heads, 0).bytes;
}

int sparkmv_kv4_attend(const sparkmv_kv4_cache * cache, const sparkmv_kv_batch * batch, const sparkmv_kv_query * query,
                       void * stream) {
    if (kv4_check_cache(cache) || kv_check_batch(batch)) return -1;
    if (!query) { set_error("kv query is null"); return -1; }
    const sparkmv_kv_query & q = *query;
    if (kv_check_dtype("queries", q.q_dtype) || kv_check_dtype("attention output", q.out_dtype)) return -1;
    if (q.heads < 1 || q.heads % cache->kv_heads || q.heads / cache->kv_heads > kKvMaxGroup) {
        set_error("%d query heads are not 1..%d times %d kv heads", q.heads, kKvMaxGroup, cache->kv_heads);
        return -1;
    }
    if (q.window < 0) { set_error("window %d is negative", q.window); return -1; }
    if (!(fabsf(q.scale) < INFINITY)) { set_error("the scale of the scores is not finite"); return -1; }
    if (batch->nseq == 0 || batch->ntok == 0) return 0;
    const long qd = (long) q.heads * cache->head_dim;
    if (kv_check_rows("queries", q.q, q.ldq, qd, q.q_dtype, batch->ntok) ||
        kv_check_rows("attention output", q.out, q.ldo, qd, q.out_dtype, batch->ntok))
        return -1;
    if (q.gate && batch->ntok > 1 && q.ldg < q.heads) {
        set_error("gate: a row stride of %d holds no %d heads", q.ldg, q.heads);
        return -1;
    }
    const Kv4Plan p = kv4_plan(cache, batch, q.heads, q.window);
    /* the count of pages, and where the last shares would end */
    if (p.tiles > (0x7fffffffl - 2 * kKv4Most) / (cache->max_pages + kKv4Item) / cache->kv_heads) {
        set_error("%d sequences and %d tokens over up to %d pages and %d kv heads are too many for one call", batch->nseq,
                  batch->ntok, cache->max_pages, cache->kv_heads);
        return -1;
    }
    if (!q.work || !kv_aligned(q.work, 256) || q.work_bytes < p.bytes) {
        set_error("attention needs %zu bytes of 256-byte aligned workspace, not %zu", p.bytes, q.work ? q.work_bytes : 0);
        return -1;
    }
    hipStream_t s = (hipStream_t) stream;
    uint8_t * mem = (uint8_t *) q.work;
    const int hd = cache->head_dim;
    Kv4Flat f;
    f.c = *cache; f.b = *batch; f.q = q;
    f.b.max_q = p.max_q;
    f.cmax = p.cmax;
    f.pre = (int *) (mem + p.pre); f.po = (float *) (mem + p.po); f.pml = (float *) (mem + p.pml);
    const dim3 join((unsigned) p.tiles, (unsigned) cache->kv_heads, (unsigned) p.cmax);
    const uint32_t pre = ((uint32_t) batch->nseq + 1) * 4;
#define KV4_FLAT_N(H, DQ, DP, W, GRID, LDS)                                                                          \
    do {                                                                                                             \
        static LdsAllowed allowed;                                                                                   \
        if (lds_allow(allowed, (const void *) kv4_flat_kernel<H, DQ, DP, W>, (LDS) + 2048, "LDS opt-in for the kv4 attention")) \
            return -1;                                                                                               \
        hipLaunchKernelGGL((kv4_flat_kernel<H, DQ, DP, W>), dim3((unsigned) (GRID)), dim3(64 * W), LDS, s, f);       \
    } while (0)
#define KV4_FLAT(H, DQ, DP)                                                                                          \
    do {                                                                                                             \
        if (p.whole) {                                                                                               \
            KV4_FLAT_N(H, DQ, DP, 8, (long) batch->nseq * cache->kv_heads, (uint32_t) kv4_lds(H, DQ, 8, p.cmax));    \
        } else {                                                                                                     \
            KV4_FLAT_N(H, DQ, DP, 4, p.groups, (uint32_t) kv4_lds(H, DQ, 4, p.cmax) + pre);                          \
            hipLaunchKernelGGL(kv4_flat_join_kernel<H>, join, dim3(512), 0, s, f);                                   \
        }                                                                                                            \
    } while (0)
#define KV4_FLAT_D(H)                                                                                                \
    do {                                                                                                             \
        if (q.q_dtype == SPARKMV_X_F32) {                                                                            \
            if (q.out_dtype == SPARKMV_X_F32) KV4_FLAT(H, 3, 3);                                                     \
            else KV4_FLAT(H, 3, 2);                                                                                  \
        } else {                                                                                                     \
            if (q.out_dtype == SPARKMV_X_F32) KV4_FLAT(H, 1, 3);                                                     \
            else KV4_FLAT(H, 1, 2);                                                                                  \
        }                                                                                                            \
    } while (0)
    if (hd == 64) KV4_FLAT_D(64);
    else if (hd == 128) KV4_FLAT_D(128);
    else KV4_FLAT_D(256);
#undef KV4_FLAT_D
#undef KV4_FLAT
#undef KV4_FLAT_N
    return kv_check_launch("kv4 attention launch");
}

}  // extern "C"
