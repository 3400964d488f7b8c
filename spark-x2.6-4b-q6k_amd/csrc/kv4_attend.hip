/* kv4_attend.hip — attention over the paged 4-bit cache (include/sparkmv.h):
 *   out = sum_p softmax_p(scale * q . k_p) v_p (* sigmoid(gate))
 * over the positions p that a token sees.
 *
 * Codes become bf16 with their scale in one instruction a pair, exactly, and products
 * run on the bf16 matrix instruction, 16 x 16 x 32, which keeps an f32 sum; the scores
 * of many columns on the one that takes 4-bit codes as they are (below). What meets the
 * codes is an f32 query element or weight as a sum of bf16 numbers:
 *
 *   few columns: a query element as three, each the leading 8 bits of what the ones
 *   before left out, which is all of f32 down to bf16's 2^-133; bf16 queries need one;
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

/* one lane's parts in all lanes of its quad, each taking the one that its mask leaves */
template <int CTRL>
__device__ __forceinline__ uint32_t kv4_quad_part(const uint32_t * part, uint32_t m0, uint32_t m1, uint32_t m2) {
    return ((uint32_t) kv_quad<CTRL>((int) part[0]) & m0) | ((uint32_t) kv_quad<CTRL>((int) part[1]) & m1) |
           ((uint32_t) kv_quad<CTRL>((int) part[2]) & m2);
}

constexpr int kKv4Cols = 16;      /* columns (token, query head) of a kv head that the flat kernels take at a time */
/* pages that beginning a kv head of a sequence counts: with 4, 8, 12 and 16, 48 sequences of up to 12000
 * take 70.0, 57.7, 54.3 and 54.3 us, 3 of 6000 with 8 tokens each 19.8, 20.2, 20.1 and 21.1 */
constexpr int kKv4Item = 12;
constexpr int kKv4Most = 1024;    /* workgroups of shares, at most */

struct Kv4Flat {
    sparkmv_kv4_cache c;
    sparkmv_kv_batch b;
    sparkmv_kv_query q;
    int cmax;        /* columns of a sequence and kv head, at most */
    int * pre;       /* [nseq + 2]: what one kv head of the sequences before counts; the share */
    float * po;      /* [workgroups][2][cmax][HD] */
    float * pml;     /* [workgroups][2][cmax][2] */
};

/* what a kv head of a sequence counts: its tiles of 16 columns, each with the pages of all
 * of its tokens (exact where there is one tile) and what beginning it costs */
__device__ __forceinline__ int kv4_cost(const KvSeq & s, int G, int window, int & tiles) {
    int first;
    tiles = (s.count * G + kKv4Cols - 1) / kKv4Cols;
    return s.count > 0 ? kv_span(s, 0, s.count, window, first) + kKv4Item : 0;
}

/* LDS of a flat kernel: the queries' operands, and once they are read the waves' outputs */
constexpr int kv4_lds(int hd, int dq, int waves, int cmax) {
    const int q = (dq ? dq : 1) * (hd / 32) * 1024, o = waves * cmax * (hd + 4) * 4;
    return q > o ? q : o;
}

/* ------------------------------------------------------------- few columns
 *
 * Sixteen columns of a kv head at a time: decode steps and short blocks. Bound by
 * reading the codes, 272 bytes a kv head and position of 256: with four heads, 131072
 * positions (143 MB) take 43.5 us and 48 sequences of up to 12000 (155313, 169 MB) 54.1,
 * the joins' 5 and 6 included; one of 1004 takes 11.6, most of it latency.
 *
 * DQ 0, up to four columns: an instruction's sixteen columns are the four columns
 * times the parts of a query element or weight, so that f32's whole precision costs
 * no further instruction. The four lanes of a quad add their parts' sums up so that
 * each ends with a quarter of the column's scores, takes their weights, and hands the
 * others the parts that they multiply. DQ 1 or 3, DP 2 or 3: sixteen columns, an
 * instruction for each part.
 *
 * WAVES 4: workgroups take equal shares of all (sequence, kv head, page) in that
 * order, so lengths may differ by any amount; a kv head of a sequence counts kKv4Item
 * pages more than it has, for what beginning it costs. A share's pages of one kv head
 * go to the waves in turn, whose results meet in LDS; a kv head's pages that lie in
 * one share are written out at once, others as a partial result that a second launch
 * joins. WAVES 8: a workgroup takes all of a sequence's kv head, and no join follows.
 *
 * A wave requests the next page's codes into the registers that it has just read,
 * and its first page's before it looks at the queries. */
template <int HD, int DQ, int DP, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void kv4_flat_kernel(const Kv4Flat A) {
    constexpr bool QUAD = DQ == 0, WHOLE = WAVES == 8;
    constexpr int NQ = QUAD ? 1 : DQ, NP = QUAD ? 1 : DP, NX = QUAD ? 1 : 4;
    constexpr int NW = HD / 32, ND = HD / 16, NB = HD / 32, NT = 64 * WAVES, LO = HD + 4;
    constexpr int KB = HD / 8;                       /* bytes of keys a lane and 16 positions */
    constexpr int NJ = HD >= 128 ? HD / 128 : 1;     /* scales of keys a lane and 16 positions */
    constexpr int NL = ND / 4;                       /* 16-byte pieces of values a lane and 32 positions */
    extern __shared__ __attribute__((aligned(16))) uint8_t ldyn[];
    float * lo = (float *) ldyn;                     /* [WAVES][cmax][LO]: a wave's output */
    kv4_u4 * lq = (kv4_u4 *) ldyn;                   /* [NQ][NW][64]: the queries as the lanes take them */
    __shared__ int lsum[4];
    __shared__ float lm[WAVES][16], ll[WAVES][16];
    int * lpre = (int *) (ldyn + kv4_lds(HD, DQ, WAVES, A.cmax));   /* [nseq + 1], shares of more than 64 sequences only */
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 4, c16 = lane & 15;
    const int dg = c16 & 3;
    const int kvh = A.c.kv_heads, G = A.q.heads / kvh, nseq = A.b.nseq;
    /* shares: what a kv head of each sequence counts. Up to 64 sequences a lane
     * each, in every wave; more through LDS */
    const bool few = nseq <= 64;
    KvSeq mine = {0, 0, 0, 0};
    int before = 0;
    int ubeg = blockIdx.x, uend = ubeg + 1;
    if constexpr (!WHOLE) {
        int total;
        if (few) {
            if (lane < nseq) mine = kv_seq(A.b, lane, A.c.nslots, A.c.max_pages);
            int tiles;
            const int each = kv4_cost(mine, G, A.q.window, tiles), cost = each * tiles;
            int scan = cost;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int v = __shfl_up(scan, o, 64);
                if (lane >= o) scan += v;
            }
            before = scan - cost;
            total = __builtin_amdgcn_readlane(scan, 63);
        } else {
            const int per = (nseq + NT - 1) / NT, i0 = min(nseq, tid * per), i1 = min(nseq, i0 + per);
            int sum = 0;
            for (int i = i0; i < i1; i++) {
                int tiles;
                lpre[i] = sum;
                const int each = kv4_cost(kv_seq(A.b, i, A.c.nslots, A.c.max_pages), G, A.q.window, tiles);
                sum += each * tiles;
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
            total = __builtin_amdgcn_readfirstlane(lpre[nseq]);
        }
        const int share = max((total * kvh + (int) gridDim.x - 1) / (int) gridDim.x, 1);
        if (blockIdx.x == 0) {
            if (few) {
                if (tid < nseq) A.pre[tid] = before;
            } else {
                for (int i = tid; i < nseq; i += NT) A.pre[i] = lpre[i];
            }
            if (tid == 0) {
                A.pre[nseq] = total;
                A.pre[nseq + 1] = share;
            }
        }
        ubeg = (int) blockIdx.x * share;
        uend = min(total * kvh, ubeg + share);
    }
    for (int u = ubeg; u < uend;) {
        int h, off = 0, n, seg, first, col0 = 0;
        KvSeq s;
        if constexpr (WHOLE) {
            const int i = u / kvh;
            h = u - i * kvh;
            s = kv_seq(A.b, i, A.c.nslots, A.c.max_pages);
            if (s.count <= 0) return;
        } else {
            /* the sequence: the last one that begins at or before u */
            int in;
            if (few) {
                const int i = 63 - __builtin_clzll(__ballot(lane < nseq && before * kvh <= u));
                s.slot = __builtin_amdgcn_readlane(mine.slot, i);
                s.pos = __builtin_amdgcn_readlane(mine.pos, i);
                s.row = __builtin_amdgcn_readlane(mine.row, i);
                s.count = __builtin_amdgcn_readlane(mine.count, i);
                in = u - __builtin_amdgcn_readlane(before, i) * kvh;
            } else {
                int i = 0;
                for (int b = nseq; b - i > 1;) {
                    const int mid = (i + b) >> 1;
                    if (__builtin_amdgcn_readfirstlane(lpre[mid]) * kvh <= u) i = mid;
                    else b = mid;
                }
                s = kv_seq(A.b, i, A.c.nslots, A.c.max_pages);
                s.slot = __builtin_amdgcn_readfirstlane(s.slot);
                s.pos = __builtin_amdgcn_readfirstlane(s.pos);
                s.row = __builtin_amdgcn_readfirstlane(s.row);
                s.count = __builtin_amdgcn_readfirstlane(s.count);
                in = u - __builtin_amdgcn_readfirstlane(lpre[i]) * kvh;
            }
            int tiles;
            const int each = kv4_cost(s, G, A.q.window, tiles), item = in / each;
            off = in - item * each;
            h = QUAD ? item : item / tiles;
            col0 = QUAD ? 0 : (item - h * tiles) * kKv4Cols;
        }
        /* the tile's columns col0 .. and its tokens t0 .. t1 - 1 */
        const int ncol = min(kKv4Cols, s.count * G - col0), t0 = QUAD ? 0 : col0 / G, t1 = QUAD ? s.count : (col0 + ncol - 1) / G + 1;
        n = seg = kv_span(s, t0, t1, A.q.window, first);
        if constexpr (!WHOLE) {
            if (off >= n) {
                int tiles;
                u += kv4_cost(s, G, A.q.window, tiles) - off;
                continue;
            }
            seg = min(n - off, uend - u);
        }
        const int col = min(QUAD ? c16 >> 2 : c16, ncol - 1), tok = (col0 + col) / G, pos_c = s.pos + tok;
        const int beg_c = A.q.window > 0 && pos_c + 1 > A.q.window ? pos_c + 1 - A.q.window : 0;
        /* positions that every column sees */
        const int all_lo = A.q.window > 0 && s.pos + t1 > A.q.window ? s.pos + t1 - A.q.window : 0, all_hi = s.pos + t0;
        const int * table = A.c.pages + (size_t) s.slot * A.c.max_pages + first + off;
        /* 64 pages of this wave at a time: their numbers are held one a lane */
        int id, count;
        uint64_t there;
        uint32_t kr[4][KB / 4], ks[NJ], vs[4];
        kv4_u4 vr[2][NL];
        /* buffer loads: a page's base is uniform, so all of its addresses take one
         * register a lane */
        auto page_at = [&](int j) {
            const uint64_t at = (uint64_t) A.c.data + ((uint64_t) (uint32_t) __builtin_amdgcn_readlane(id, j) * (uint32_t) kvh + (uint32_t) h) * (68 * HD);
            const uint64_t lo32 = (uint32_t) __builtin_amdgcn_readfirstlane((int) (uint32_t) at);
            const uint64_t hi32 = (uint32_t) __builtin_amdgcn_readfirstlane((int) (at >> 32));
            return __builtin_amdgcn_make_buffer_rsrc((void *) (hi32 << 32 | lo32), 0, 68 * HD, 0x00027000);
        };
        const uint32_t kslane = ((HD == 64 ? g >> 1 : g) * 16 + c16) * 4 * NJ, vslane = (g * NB + (c16 * ND) / 32) * 16;
        auto fetch_k = [&](int j) {
            const auto p = page_at(j);
            if constexpr (NJ == 2) {
                const auto v = __builtin_amdgcn_raw_buffer_load_b64(p, kslane, 64 * HD, 0);
                ks[0] = v[0];
                ks[1] = v[1];
            } else {
                ks[0] = __builtin_amdgcn_raw_buffer_load_b32(p, kslane, 64 * HD, 0);
            }
#pragma unroll
            for (int t = 0; t < 4; t++) {
                if constexpr (HD >= 128) {
#pragma unroll
                    for (int jj = 0; jj < NJ; jj++) {
                        const kv4_u4 v = (kv4_u4) __builtin_amdgcn_raw_buffer_load_b128(p, lane * 16, (t * NJ + jj) * 1024, 0);
#pragma unroll
                        for (int e = 0; e < 4; e++) kr[t][4 * jj + e] = v[e];
                    }
                } else {
                    const auto v = __builtin_amdgcn_raw_buffer_load_b64(p, lane * 8, t * 512, 0);
                    kr[t][0] = v[0];
                    kr[t][1] = v[1];
                }
            }
        };
        auto fetch_vs = [&](int j) {
            const kv4_u4 v = (kv4_u4) __builtin_amdgcn_raw_buffer_load_b128(page_at(j), vslane, 66 * HD, 0);
#pragma unroll
            for (int e = 0; e < 4; e++) vs[e] = v[e];
        };
        auto fetch_v = [&](int j, int w) {
            const auto p = page_at(j);
#pragma unroll
            for (int k = 0; k < NL; k++) vr[w][k] = (kv4_u4) __builtin_amdgcn_raw_buffer_load_b128(p, lane * 16, 32 * HD + (w * NL + k) * 1024, 0);
        };
        auto begin = [&](int base) {
            count = min((seg - base + WAVES - 1) / WAVES, 64);
            id = 0;
            bool have = false;
            if (lane < count) {
                id = table[base + WAVES * lane];
                have = id >= 0 && id < A.c.npages;
                id = have ? id : 0;
            }
            there = __ballot(have);
            fetch_k(0);
            fetch_vs(0);
            fetch_v(0, 0);
            fetch_v(0, 1);
            __builtin_amdgcn_sched_barrier(0);
        };
        /* the queries, eight elements of a column a thread, requested before the codes:
         * loads return in order */
        constexpr int QW = (QUAD ? NW * 16 : NW * 64) / NT ? (QUAD ? NW * 16 : NW * 64) / NT : 1;   /* threads' shares */
        float x8[QW][8];
        int q_w[QW], q_c[QW], q_g[QW];
#pragma unroll
        for (int r = 0; r < QW; r++) {
            const int k = tid + r * NT;
            q_w[r] = QUAD ? k >> 4 : k >> 6;
            q_c[r] = QUAD ? k >> 2 & 3 : k & 15;
            q_g[r] = QUAD ? k & 3 : k >> 4 & 3;
            const int d = HD >= 128 ? 32 * (4 * (q_w[r] >> 2) + q_g[r]) + 8 * (q_w[r] & 3) : 16 * q_g[r] + 8 * q_w[r];
#pragma unroll
            for (int e = 0; e < 8; e++) x8[r][e] = 0.0f;
            if (q_w[r] < NW && q_c[r] < ncol) {
                const int t = (col0 + q_c[r]) / G, head = h * G + (col0 + q_c[r]) - t * G;
                const size_t at = (size_t) (s.row + t) * A.q.ldq + (size_t) head * HD + d;
                if (DQ == 3 || (QUAD && A.q.q_dtype == SPARKMV_X_F32)) {
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const kv_f4 v = *(const kv_f4 *) ((const float *) A.q.q + at + 4 * e);
#pragma unroll
                        for (int f = 0; f < 4; f++) x8[r][4 * e + f] = v[f];
                    }
                } else {
                    const kv4_u4 v = *(const kv4_u4 *) ((const uint16_t *) A.q.q + at);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        x8[r][2 * e] = __uint_as_float(v[e] << 16);
                        x8[r][2 * e + 1] = __uint_as_float(v[e] & 0xffff0000u);
                    }
                }
            }
        }
        if (wave < seg) begin(wave);
#pragma unroll
        for (int r = 0; r < QW; r++) {
            if (q_w[r] >= NW) continue;
            if constexpr (QUAD) {
                kv4_u4 o3[3];
                kv4_split8<3>(x8[r], o3);
#pragma unroll
                for (int d2 = 0; d2 < 4; d2++)
                    lq[q_w[r] * 64 + 16 * q_g[r] + 4 * q_c[r] + d2] = d2 < 3 ? o3[d2] : kv4_u4{0, 0, 0, 0};
            } else {
                kv4_u4 o3[NQ];
                kv4_split8<NQ>(x8[r], o3);
#pragma unroll
                for (int d2 = 0; d2 < NQ; d2++) lq[(d2 * NW + q_w[r]) * 64 + 16 * q_g[r] + q_c[r]] = o3[d2];
            }
        }
        __syncthreads();
        const float f = A.q.scale * kKvLog2e;
        float m = -INFINITY, l = 0.0f;
        kv_f4 o[ND];
#pragma unroll
        for (int d = 0; d < ND; d++) o[d] = kv_f4{0.f, 0.f, 0.f, 0.f};
        for (int base = wave; base < seg; base += 64 * WAVES) {
            if (base > wave) begin(base);
            for (int j = 0; j < count; j++) {
                const int nx = min(j + 1, count - 1);
                /* read again for each page: held, they would leave too few registers */
                asm volatile("" ::: "memory");
                /* scores: tile t's positions 4 g + e of a column's part */
                kv_f4 a[4];
#pragma unroll
                for (int w = 0; w < NJ; w++) ks[w] |= (kv4_bad(ks[w]) >> 7) * 0xffu;
#pragma unroll
                for (int t = 0; t < 4; t++) a[t] = kv_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < NW; w++) {
                    kv4_u4 qd[NQ];
#pragma unroll
                    for (int d = 0; d < NQ; d++) qd[d] = lq[(d * NW + w) * 64 + lane];
#pragma unroll
                    for (int t = 0; t < 4; t++) {
                        const int k = t * NJ + w / 4;   /* its scale: byte k of ks */
                        const float sc = k % 4 == 0 ? kv4_scale<0>(ks[k / 4]) : (k % 4 == 1 ? kv4_scale<1>(ks[k / 4]) :
                                         (k % 4 == 2 ? kv4_scale<2>(ks[k / 4]) : kv4_scale<3>(ks[k / 4])));
                        const uint32_t c = kr[t][w];
                        const kv4_b8 kf = kv4_operand(kv4_pair<0>(c, sc), kv4_pair<1>(c, sc), kv4_pair<2>(c, sc), kv4_pair<3>(c, sc));
#pragma unroll
                        for (int d = NQ - 1; d >= 0; d--)
                            a[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, __builtin_bit_cast(kv4_b8, qd[d]), a[t], 0, 0, 0);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
                fetch_k(nx);
                __builtin_amdgcn_sched_barrier(0);
                /* x[t][e]: the score of position 16 t + 4 g + e, with parts in lanes t = dg alone */
                float x[NX][4];
                if constexpr (QUAD) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float k0 = (dg & 2 ? a[2][e] : a[0][e]) + kv_quad<kKvXor2>(dg & 2 ? a[0][e] : a[2][e]);
                        const float k1 = (dg & 2 ? a[3][e] : a[1][e]) + kv_quad<kKvXor2>(dg & 2 ? a[1][e] : a[3][e]);
                        x[0][e] = ((dg & 1 ? k1 : k0) + kv_quad<kKvXor1>(dg & 1 ? k0 : k1)) * f;
                    }
                } else {
#pragma unroll
                    for (int t = 0; t < NX; t++)
#pragma unroll
                        for (int e = 0; e < 4; e++) x[t][e] = a[t][e] * f;
                }
                const int p0 = (first + off + base + WAVES * j) * kKvPage;
                const bool ok = there >> j & 1;
                if (!ok || p0 < all_lo || p0 + kKvPage - 1 > all_hi) {
#pragma unroll
                    for (int t = 0; t < NX; t++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const int p = p0 + 16 * (QUAD ? dg : t) + 4 * g + e;
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
                            if (here && (!QUAD || dg == k) && x[QUAD ? 0 : k][e] != -INFINITY) l = __uint_as_float(0x7fc00000u);
                        }
                        vs[k] &= ~((b >> 7) * 0xffu);
                    }
                }
                float mp = -INFINITY;
#pragma unroll
                for (int t = 0; t < NX; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++) mp = fmaxf(mp, x[t][e]);
                if constexpr (QUAD) {
                    mp = fmaxf(mp, kv_quad<kKvXor1>(mp));
                    mp = fmaxf(mp, kv_quad<kKvXor2>(mp));
                }
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
                for (int t = 0; t < NX; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        x[t][e] = __builtin_amdgcn_exp2f(x[t][e] - mref);
                        l += x[t][e];
                    }
                /* the weights' parts, pairs of positions */
                kv4_u4 P[2][NP];
                if constexpr (QUAD) {
                    uint32_t part[2][3];
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        float y = x[0][2 * k], z = x[0][2 * k + 1];
#pragma unroll
                        for (int d = 0; d < 3; d++) {
                            part[k][d] = kv_bf16x2(y, z);
                            y -= __uint_as_float(part[k][d] << 16);
                            z -= __uint_as_float(part[k][d] & 0xffff0000u);
                        }
                    }
                    /* tile t's weights are lane t's of the quad; this lane takes part dg of them */
                    const uint32_t m0 = dg == 0 ? ~0u : 0u, m1 = dg == 1 ? ~0u : 0u, m2 = dg == 2 ? ~0u : 0u;
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        P[0][0][k] = kv4_quad_part<0x00>(part[k], m0, m1, m2);
                        P[0][0][2 + k] = kv4_quad_part<0x55>(part[k], m0, m1, m2);
                        P[1][0][k] = kv4_quad_part<0xaa>(part[k], m0, m1, m2);
                        P[1][0][2 + k] = kv4_quad_part<0xff>(part[k], m0, m1, m2);
                    }
                } else {
#pragma unroll
                    for (int w = 0; w < 2; w++)
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            float y = x[(2 * w + (k >> 1)) % NX][2 * (k & 1)], z = x[(2 * w + (k >> 1)) % NX][2 * (k & 1) + 1];
#pragma unroll
                            for (int d = 0; d < NP; d++) {
                                P[w][d][k] = kv_bf16x2(y, z);
                                y -= __uint_as_float(P[w][d][k] << 16);
                                z -= __uint_as_float(P[w][d][k] & 0xffff0000u);
                            }
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
                        uint32_t ea[4], eb[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            ea[e] = __builtin_amdgcn_perm(r[2 * e + 1], r[2 * e], 0x05040100u);
                            eb[e] = __builtin_amdgcn_perm(r[2 * e + 1], r[2 * e], 0x07060302u);
                        }
                        const kv4_b8 va = kv4_operand(ea[0], ea[1], ea[2], ea[3]), vb = kv4_operand(eb[0], eb[1], eb[2], eb[3]);
#pragma unroll
                        for (int d = NP - 1; d >= 0; d--) {
                            o[2 * k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, __builtin_bit_cast(kv4_b8, P[w][d]), o[2 * k], 0, 0, 0);
                            o[2 * k + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vb, __builtin_bit_cast(kv4_b8, P[w][d]), o[2 * k + 1], 0, 0, 0);
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    if (w == 1) fetch_vs(nx);
                    fetch_v(nx, w);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        if constexpr (QUAD) {
            l += kv_quad<kKvXor1>(l);
            l += kv_quad<kKvXor2>(l);
        }
        l = kv_rows_sum(l);
        __syncthreads();   /* the queries are read */
        /* the waves' outputs meet in LDS: this lane has elements ND (4 g + i) .. of its column,
         * for i = 0 .. 3, or with parts in lanes the sums of i = dg */
        if constexpr (QUAD) {
#pragma unroll
            for (int d0 = 0; d0 < ND; d0 += 4) {
                kv_f4 v;
#pragma unroll
                for (int d = 0; d < 4; d++) {
                    const kv_f4 y = o[d0 + d];
                    const float k0 = (dg & 2 ? y[2] : y[0]) + kv_quad<kKvXor2>(dg & 2 ? y[0] : y[2]);
                    const float k1 = (dg & 2 ? y[3] : y[1]) + kv_quad<kKvXor2>(dg & 2 ? y[1] : y[3]);
                    v[d] = (dg & 1 ? k1 : k0) + kv_quad<kKvXor1>(dg & 1 ? k0 : k1);
                }
                if (c16 >> 2 < ncol) *(kv_f4 *) (lo + (wave * A.cmax + (c16 >> 2)) * LO + ND * (4 * g + dg) + d0) = v;
            }
        } else if (c16 < ncol) {
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int d = 0; d < ND; d += 4)
                    *(kv_f4 *) (lo + (wave * A.cmax + c16) * LO + ND * (4 * g + i) + d) = kv_f4{o[d][i], o[d + 1][i], o[d + 2][i], o[d + 3][i]};
        }
        if (g == 0 && (!QUAD || dg == 0)) {
            lm[wave][QUAD ? c16 >> 2 : c16] = m;
            ll[wave][QUAD ? c16 >> 2 : c16] = l;
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
            if (whole) {
                const float y[4] = {v[0], v[1], v[2], v[3]};
                kv_write<V>(A.q, s.row + (col0 + cc) / G, h * G + (col0 + cc) % G, HD, d, y, L);
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

/* Joins the partial results of one column of a (sequence, tile, kv head), in the order
 * of its pages: its first share wrote slot 1, the later ones slot 0. */
template <int HD>
__global__ __launch_bounds__(512) void kv4_flat_join_kernel(const Kv4Flat A) {
    __shared__ float wts[kKv4Most];
    __shared__ __attribute__((aligned(16))) float acc[7 * HD];
    const int i = blockIdx.x, h = blockIdx.y, col0 = (int) blockIdx.z / A.cmax * kKv4Cols, c = (int) blockIdx.z % A.cmax;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, kvh = A.c.kv_heads, G = A.q.heads / kvh;
    const KvSeq s = kv_seq(A.b, i, A.c.nslots, A.c.max_pages);
    int tiles, first;
    const int each = kv4_cost(s, G, A.q.window, tiles), ncol = min(kKv4Cols, s.count * G - col0);
    if (c >= ncol) return;
    const int n = kv_span(s, col0 / G, (col0 + ncol - 1) / G + 1, A.q.window, first), share = A.pre[A.b.nseq + 1];
    const int a = A.pre[i] * kvh + (h * tiles + col0 / kKv4Cols) * each, w0 = a / share, w1 = (a + n - 1) / share;
    if (w0 == w1) return;
    float o[HD / 64];
    const float L = kv_join<HD, 8>(A.po, A.pml, w1 - w0 + 1, [&](int k) { return (2 * (size_t) (w0 + k) + (k == 0)) * A.cmax + c; },
                                   wts, acc, wave, lane, o);
    if (wave) return;
    kv_write<HD / 64>(A.q, s.row + (col0 + c) / G, h * G + (col0 + c) % G, HD, HD / 64 * lane, o, L);
}

/* -------------------------------------------------------------- many columns
 *
 * A workgroup of eight waves takes 128 columns (token, query head) of a kv head, 16 a
 * wave, and a share of the pages that they see. A page enters LDS while the one before
 * it is worked on: codes of keys as they lie, by direct loads; values as the bf16
 * operands that they become, converted once for all waves.
 *
 * 512 bf16 tokens of 16 heads of 256 at 16384 take 220 us with the join's 13: 140 GFLOP
 * as the formula counts them, 0.63 PFLOP/s, where a large bf16 product reaches 1.2. With
 * four of the scores' five parts left out it would be 195, without the values' conversion
 * 191, without their products 206, without exponentials no less: the vector and matrix
 * pipes take turns, two waves a SIMD being all that the registers hold.
 *
 * The scores use the instruction that multiplies 4-bit codes as they are, 16 x 16 x 128
 * with a power of two for every 32 elements. A query element enters it as a sum of
 * parts, each the nearest small number to what the ones before left out; 32 neighbours
 * share a power of two. Five parts of 6 bits (E2M3, four times as fast a product as
 * bf16's), at most 4 in magnitude and off by 1 / 8 at most: 2^-24 of the largest of the 32 is
 * what may be lost, and nothing of a bf16 element down to 2^-17 of it. Six parts for
 * head_dim 64, where an instruction takes two.
 * Two parts of 8 bits (E4M3) would do for bf16 (205 us for the call above) but for the
 * sum: within 16 elements of a lane the instruction drops what lies below 2^-13 of the
 * largest product, which left outputs off by 1e-5. Products of a 6-bit part and a code
 * are multiples of 1 / 16 up to 24, so none of them is cut.
 *
 * Weights times values as in the flat kernels. */
constexpr int kKv4Tile = 128;       /* columns of a workgroup */
/* pages that beginning a tile's kv head counts: with 2, 4, 6 and 12, 512 tokens at 16384
 * take 223, 222, 220 and 225 us, at 1000 54.9, 54.2, 54.5 and 55.5 */
constexpr int kKv4TileItem = 6;
constexpr int kKv4Tiles = 2048;     /* tiles that are split among equal shares, at most */
constexpr int kKv4Ids = 256;        /* page numbers held at a time */

struct Kv4Tile {
    sparkmv_kv4_cache c;
    sparkmv_kv_batch b;
    sparkmv_kv_query q;
    int tiles;       /* of the batch, at most */
    int share;       /* 0: a workgroup takes a whole tile and kv head */
    int * pre;       /* [tiles + 2]: what the tiles before count; the share */
    float * po;      /* [workgroups][2][128][HD] */
    float * pml;     /* [workgroups][2][128][2] */
};

/* parts of a query element: an even number where an instruction takes two */
constexpr int kv4_tile_parts(int hd) { return hd == 64 ? 6 : 5; }
/* instructions' parts of the queries that wait in LDS: all of them leave too few registers */
constexpr int kv4_tile_far(int hd) { return hd == 256 ? 2 : 0; }
constexpr int kv4_tile_lds(int hd) { return 2 * (32 + 128) * hd + kv4_tile_far(hd) * (hd / 128) * 8 * 1536; }

/* the sequence and the place within it of tile number j, from the tiles before each sequence */
__device__ __forceinline__ KvSeq kv4_tile_seq(const sparkmv_kv_batch & b, const sparkmv_kv4_cache & c, const int * lseq, int j, int & place) {
    int i = 0;
    for (int e = b.nseq; e - i > 1;) {
        const int mid = (i + e) >> 1;
        if (lseq[mid] <= j) i = mid;
        else e = mid;
    }
    place = j - lseq[i];
    return kv_seq(b, i, c.nslots, c.max_pages);
}

/* exclusive sums over the workgroup's threads; total in all of them */
__device__ __forceinline__ int kv4_scan(int v, int * lsum, int wave, int lane, int nw, int & total) {
    int scan = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int x = __shfl_up(scan, o, 64);
        if (lane >= o) scan += x;
    }
    __syncthreads();
    if (lane == 63) lsum[wave] = scan;
    __syncthreads();
    int before = 0;
    total = 0;
    for (int w = 0; w < nw; w++) {
        if (w < wave) before += lsum[w];
        total += lsum[w];
    }
    return before + scan - v;
}

/* what tile j of the batch counts, and its place in the list, as every workgroup finds
 * them: lseq[i], the tiles before sequence i, and lpre[j], what the tiles before count */
template <int NT>
__device__ __forceinline__ int kv4_tile_shares(const Kv4Tile & A, int G, int * lseq, int * lpre, int * lsum) {
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, nseq = A.b.nseq;
    int tiles = 0, all = 0;
    for (int i0 = 0; i0 < nseq; i0 += NT) {
        int n = 0, sum;
        if (i0 + tid < nseq) n = (int) (((long) kv_seq(A.b, i0 + tid, A.c.nslots, A.c.max_pages).count * G + kKv4Tile - 1) / kKv4Tile);
        const int at = tiles + kv4_scan(n, lsum, wave, lane, NT / 64, sum);
        if (i0 + tid < nseq) lseq[i0 + tid] = at;
        tiles += sum;
    }
    __syncthreads();
    tiles = min(tiles, A.tiles);   /* more only if rows are claimed twice */
    for (int j0 = 0; j0 < tiles; j0 += NT) {
        int n = 0, sum;
        const int j = j0 + tid;
        if (j < tiles) {
            int place, first;
            const KvSeq s = kv4_tile_seq(A.b, A.c, lseq, j, place);
            const int c0 = place * kKv4Tile, c1 = min(c0 + kKv4Tile, s.count * G) - 1;
            n = kv_span(s, c0 / G, c1 / G + 1, A.q.window, first) + kKv4TileItem;
        }
        const int at = all + kv4_scan(n, lsum, wave, lane, NT / 64, sum);
        if (j < tiles) lpre[j] = at;
        all += sum;
    }
    if (tid == 0) lpre[tiles] = all;
    __syncthreads();
    return tiles;
}

typedef float kv4_f16 __attribute__((ext_vector_type(16)));
typedef float kv4_f32 __attribute__((ext_vector_type(32)));
typedef uint32_t kv4_u6 __attribute__((ext_vector_type(6)));
typedef int kv4_i8 __attribute__((ext_vector_type(8)));

template <int HD, int DP>
__global__ __launch_bounds__(512, 2) void kv4_tile_kernel(const Kv4Tile A) {
    constexpr int ND = HD / 16, NB = HD / 32, BUF = (32 + 128) * HD;
    constexpr int NJ = HD >= 128 ? HD / 128 : 1;         /* instructions of 128 elements a head */
    constexpr int DQ = kv4_tile_parts(HD);               /* parts of a query element */
    constexpr int NM = HD == 64 ? DQ / 2 : DQ;           /* instructions a score tile and 128 elements */
    constexpr int PW = 6, NR = NM - kv4_tile_far(HD);    /* words of a part; instructions' parts in registers */
    typedef __attribute__((address_space(3))) void lds_void;
    extern __shared__ __attribute__((aligned(16))) uint8_t lbuf[];   /* [2][keys' codes, values' operands] */
    uint8_t * lfar = lbuf + 2 * BUF;                      /* [wave][part][NJ][64 lanes' 16 bytes, 64 lanes' 8] */
    int * lseq = (int *) (lbuf + kv4_tile_lds(HD)), * lpre = lseq + A.b.nseq;
    __shared__ int lid[kKv4Ids], lsum[10];
    __shared__ uint32_t lnan[2][2];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 4, c16 = lane & 15;
    const int kvh = A.c.kv_heads, G = A.q.heads / kvh;
    long ubeg = blockIdx.x, uend = ubeg + 1;
    int tiles = 0;
    if (A.share) {
        tiles = kv4_tile_shares<512>(A, G, lseq, lpre, lsum);
        const long total = (long) lpre[tiles] * kvh, share = (total + gridDim.x - 1) / gridDim.x;
        if (blockIdx.x == 0) {
            for (int j = tid; j <= tiles; j += 512) A.pre[j] = lpre[j];
            if (tid == 0) A.pre[A.tiles + 1] = (int) share;
        }
        ubeg = min((long) blockIdx.x * share, total);
        uend = min(ubeg + share, total);
    }
    for (long u = ubeg; u < uend;) {
        KvSeq s;
        int place, h, off = 0, seg;
        if (A.share) {
            /* kv heads outside, tiles inside */
            h = (int) (u / lpre[tiles]);
            const int in = (int) (u - (long) h * lpre[tiles]);
            int j = 0;
            for (int e = tiles; e - j > 1;) {
                const int mid = (j + e) >> 1;
                if (lpre[mid] <= in) j = mid;
                else e = mid;
            }
            off = in - lpre[j];
            s = kv4_tile_seq(A.b, A.c, lseq, j, place);
        } else {
            h = blockIdx.x % kvh;
            if (!kv_find_tile(A.b, A.c, G, kKv4Tile, blockIdx.x / kvh, lsum, s, place)) return;
        }
        s.slot = __builtin_amdgcn_readfirstlane(s.slot);
        s.pos = __builtin_amdgcn_readfirstlane(s.pos);
        s.row = __builtin_amdgcn_readfirstlane(s.row);
        s.count = __builtin_amdgcn_readfirstlane(s.count);
        h = __builtin_amdgcn_readfirstlane(h);
        off = __builtin_amdgcn_readfirstlane(off);
        place = __builtin_amdgcn_readfirstlane(place);
        const int ncols = s.count * G, col0 = place * kKv4Tile, last = min(col0 + kKv4Tile, ncols) - 1;
        int first;
        const int n = kv_span(s, col0 / G, last / G + 1, A.q.window, first);
        seg = n - off;
        if (A.share) {
            if (off >= n) {
                u += n + kKv4TileItem - off;
                continue;
            }
            seg = (int) min((long) seg, uend - u);
        }
        first += off;
        const int * table = A.c.pages + (size_t) s.slot * A.c.max_pages + first;
        auto ids = [&](int j0) {   /* pages j0 .. of the share; a barrier on both sides */
            __syncthreads();
            if (tid < kKv4Ids && j0 + tid < seg) {
                const int id = table[j0 + tid];
                lid[tid] = id >= 0 && id < A.c.npages ? id : -1;
            }
            __syncthreads();
        };
        /* this wave's part of a page: eight positions' words of codes and their scales.
         * 256 elements: two bytes of a position's eight; 128: one of four; 64: one of two */
        const int vu = wave & 1, vk = wave >> 1;
        const bool converts = HD > 64 || wave < 4;
        uint32_t vr[8], vsc[2], ks[NJ];
        /* buffer loads: a page's base is uniform, so its addresses are three registers a lane */
        const uint32_t lane16 = 16 * lane, kslane = ((HD == 64 ? g & 1 : g) * 16 + c16) * 4 * NJ, vslane = (g * NB + (c16 * ND) / 32) * 16;
        auto fetch = [&](int j, int b) {
            const uint64_t at = (uint64_t) A.c.data + ((uint64_t) (uint32_t) max(__builtin_amdgcn_readfirstlane(lid[j & (kKv4Ids - 1)]), 0) * (uint32_t) kvh + (uint32_t) h) * (68 * HD);
            const uint64_t lo32 = (uint32_t) __builtin_amdgcn_readfirstlane((int) (uint32_t) at), hi32 = (uint32_t) __builtin_amdgcn_readfirstlane((int) (at >> 32));
            const auto page = __builtin_amdgcn_make_buffer_rsrc((void *) (hi32 << 32 | lo32), 0, 68 * HD, 0x00027000);
            if (wave < HD / 32)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(page, (lds_void *) (lbuf + (size_t) b * BUF + wave * 1024), 16, lane16, wave * 1024, 0, 0);
            if constexpr (NJ == 2) {
                const auto v = __builtin_amdgcn_raw_buffer_load_b64(page, kslane, 64 * HD, 0);
                ks[0] = v[0];
                ks[1] = v[1];
            } else {
                ks[0] = __builtin_amdgcn_raw_buffer_load_b32(page, kslane, 64 * HD, 0);
            }
            if (converts) {
                const int vp = 32 * HD + vu * (ND / 4) * 1024;
                if constexpr (HD == 256) {
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        vr[e] = __builtin_amdgcn_raw_buffer_load_b32(page, lane16 + (e & 1) * 8, vp + (e >> 1) * 1024 + (vk >> 1) * 4, 0);
                } else {
#pragma unroll
                    for (int w = 0; w < HD / 64; w++) {
                        const kv4_u4 v = (kv4_u4) __builtin_amdgcn_raw_buffer_load_b128(page, lane16, vp + w * 1024, 0);
#pragma unroll
                        for (int e = 0; e < 4; e++) vr[4 * w + e] = v[e];
                    }
                }
                const auto v = __builtin_amdgcn_raw_buffer_load_b64(page, vslane + 8 * vu, 66 * HD, 0);
                vsc[0] = v[0];
                vsc[1] = v[1];
            }
        };
        auto convert = [&](int b) {
            if (!converts) return;
            uint8_t * to = lbuf + (size_t) b * BUF + 32 * HD;
            uint32_t bad = kv4_bad(vsc[0]) | kv4_bad(vsc[1]), which = 0;
            if (__any(bad != 0)) {
                /* values that are not numbers count as zero, and are marked */
#pragma unroll
                for (int w = 0; w < 2; w++) {
                    bad = kv4_bad(vsc[w]);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const uint64_t who = __ballot(bad >> (8 * e + 7) & 1);
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            if (who >> (16 * k) & 0xffff) which |= 1u << (16 * w + 4 * k + e);
                    }
                    vsc[w] &= ~((bad >> 7) * 0xffu);
                }
            }
            if (vk == 0 && lane == 0) lnan[b][vu] = which;
            const float sc[8] = {kv4_scale<0>(vsc[0]), kv4_scale<1>(vsc[0]), kv4_scale<2>(vsc[0]), kv4_scale<3>(vsc[0]),
                                 kv4_scale<0>(vsc[1]), kv4_scale<1>(vsc[1]), kv4_scale<2>(vsc[1]), kv4_scale<3>(vsc[1])};
            constexpr int NK = HD == 256 ? 2 : 1;   /* bytes, pairs of elements */
            uint32_t r[NK][8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                if constexpr (HD == 256) {
                    const uint32_t v = vr[e] >> (16 * (vk & 1));
                    r[0][e] = kv4_pair<0>(v, sc[e]);
                    r[NK - 1][e] = kv4_pair<1>(v, sc[e]);
                } else if constexpr (HD == 128) {
                    r[0][e] = kv4_pair<0>(vr[e] >> (8 * vk), sc[e]);
                } else {
                    r[0][e] = kv4_pair<0>(vr[e / 2] >> (16 * (e & 1) + 8 * vk), sc[e]);
                }
            }
#pragma unroll
            for (int k = 0; k < NK; k++) {
                const int dt = 2 * (vk * NK + k);
                kv4_u4 x, y;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    x[e] = __builtin_amdgcn_perm(r[k][2 * e + 1], r[k][2 * e], 0x05040100u);
                    y[e] = __builtin_amdgcn_perm(r[k][2 * e + 1], r[k][2 * e], 0x07060302u);
                }
                *(kv4_u4 *) (to + ((vu * ND + dt) * 64 + lane) * 16) = x;
                *(kv4_u4 *) (to + ((vu * ND + dt + 1) * 64 + lane) * 16) = y;
            }
        };
        ids(0);
        fetch(0, 0);
        /* this wave's columns */
        const int wfirst = col0 + 16 * wave, cc = min(wfirst + c16, last), tok = cc / G, head = h * G + cc - tok * G;
        const bool live = wfirst <= last;   /* uniform in the wave */
        const int pos_c = s.pos + tok, beg_c = A.q.window > 0 && pos_c + 1 > A.q.window ? pos_c + 1 - A.q.window : 0;
        const int wpos_lo = s.pos + min(wfirst, last) / G, wpos_hi = s.pos + min(wfirst + 15, last) / G;   /* the wave's first and last token */
        const int wbeg_lo = A.q.window > 0 && wpos_lo + 1 > A.q.window ? wpos_lo + 1 - A.q.window : 0;
        const int wbeg_hi = A.q.window > 0 && wpos_hi + 1 > A.q.window ? wpos_hi + 1 - A.q.window : 0;
        uint32_t qd[NR][NJ][PW] = {};
        uint8_t * far = lfar + wave * (NM - NR) * NJ * 1536;
        uint32_t qs[NJ][2];   /* the parts' scales, a byte each */
        float f;
        {
            int ex[NJ], most = -1000;
            bool bad = false;
            float x[32];
            const size_t row = (size_t) (s.row + tok) * A.q.ldq + (size_t) head * HD;
            auto load = [&](int at) {   /* 32 elements */
                if (A.q.q_dtype == SPARKMV_X_F32) {
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const kv_f4 v = *(const kv_f4 *) ((const float *) A.q.q + row + at + 4 * e);
#pragma unroll
                        for (int i = 0; i < 4; i++) x[4 * e + i] = v[i];
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const kv4_u4 v = *(const kv4_u4 *) ((const uint16_t *) A.q.q + row + at + 8 * e);
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            x[8 * e + 2 * i] = __uint_as_float(v[i] << 16);
                            x[8 * e + 2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
                        }
                    }
                }
            };
#pragma unroll
            for (int j = 0; j < NJ; j++) {
                load(32 * (HD == 64 ? g & 1 : 4 * j + g));
                uint32_t big = 0;
#pragma unroll
                for (int e = 0; e < 32; e++) big = max(big, __float_as_uint(x[e]) & 0x7fffffffu);
                bad = bad || big >= 0x7f800000u;
                int e2 = 0;
                (void) frexpf(__uint_as_float(big >= 0x7f800000u ? 0u : big), &e2);
                ex[j] = big ? e2 : -1000;
                most = max(most, ex[j]);
                __builtin_amdgcn_sched_barrier(0);
            }
            /* the column's exponent */
            most = max(most, __shfl_xor(most, 16, 64));
            most = max(most, __shfl_xor(most, 32, 64));
            uint32_t any = bad;
            any |= __shfl_xor((int) any, 16, 64);
            any |= __shfl_xor((int) any, 32, 64);
            /* Scores are summed up with the column's elements below 2^-9, so that 256 products with
             * codes of up to 6 * 2^125 stay within f32, and f brings them back. Where f would be no
             * normal number they are larger or smaller than that, and a sum leaves f32 with its score */
            int es;
            (void) frexpf(fabsf(A.q.scale), &es);
            const int up = min(max(most + 9, -120 - es), 120 - es);
            f = any ? __uint_as_float(0x7fc00000u) : ldexpf(fabsf(A.q.scale) * kKvLog2e, up);
            const float sign = A.q.scale < 0.0f ? -1.0f : 1.0f;
#pragma unroll
            for (int j = 0; j < NJ; j++) {
                const int low = min(max(ex[j] - up, -200), 127);
                /* below 4 in magnitude; part d in steps of 2^(-5 d) of that.
                 * Read again: all blocks at once would not fit the registers */
                load(32 * (HD == 64 ? g & 1 : 4 * j + g));
#pragma unroll
                for (int e = 0; e < 32; e++) x[e] = any ? 0.0f : ldexpf(x[e] * sign, 2 - ex[j]);
                qs[j][0] = qs[j][1] = 0;
#pragma unroll
                for (int d = 0; d < DQ; d++) {
                    uint32_t part[PW];
                    kv4_f16 ev, od;
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        ev[e] = x[2 * e];
                        od[e] = x[2 * e + 1];
                    }
                    const kv4_u6 six = __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(ev, od, 1.0f);
                    const kv4_f32 back = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(six, 1.0f);
#pragma unroll
                    for (int e = 0; e < 6; e++) part[e] = six[e];
#pragma unroll
                    for (int e = 0; e < 32; e++) x[e] = (x[e] - back[e]) * 32.0f;
                    /* a part that no scale reaches is below 2^-126, 2^-116 of the column's largest element */
                    const int exp = 127 + low - 2 - 5 * d;
                    const uint32_t sb = (uint32_t) max(exp, 0);
#pragma unroll
                    for (int e = 0; e < PW; e++) part[e] = exp < 0 ? 0u : part[e];
                    if constexpr (HD == 64) {
                        /* two parts an instruction: the second one in the place of blocks 2 and 3 */
                        const bool mine = (g >> 1) == (d & 1);
#pragma unroll
                        for (int e = 0; e < PW; e++) qd[d / 2][j][e] = mine || !(d & 1) ? part[e] : qd[d / 2][j][e];
                        if (mine) qs[j][0] |= sb << (8 * (d / 2));
                    } else {
                        if (d < NR) {
#pragma unroll
                            for (int e = 0; e < PW; e++) qd[d % NR][j][e] = part[e];
                        } else {
                            uint8_t * to = far + ((d - NR) * NJ + j) * 1536;
                            *(kv4_u4 *) (to + 16 * lane) = kv4_u4{part[0], part[1], part[2], part[3]};
                            *(kv4_u2 *) (to + 1024 + 8 * lane) = kv4_u2{part[4], part[5]};
                        }
                        qs[j][d / 4] |= sb << (8 * (d % 4));
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        convert(0);
        float m = -INFINITY, l = 0.0f;
        kv_f4 o[ND];
#pragma unroll
        for (int d = 0; d < ND; d++) o[d] = kv_f4{0.f, 0.f, 0.f, 0.f};
        int idn = lid[0];
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   /* this wave's part of page 0 */
        for (int j = 0; j < seg; j++) {
            __syncthreads();   /* everyone's part of page j, and everyone is done with the other buffer */
            const int b = j & 1, id = idn, p0 = (first + j) * kKvPage;
            uint32_t ksj[NJ];
#pragma unroll
            for (int w = 0; w < NJ; w++) ksj[w] = ks[w];
            if (j + 1 < seg) {
                if (((j + 1) & (kKv4Ids - 1)) == 0) ids(j + 1);
                idn = lid[(j + 1) & (kKv4Ids - 1)];
                fetch(j + 1, b ^ 1);
            }
            const uint8_t * kp = lbuf + (size_t) b * BUF, * vp = kp + 32 * HD + 16 * lane;
            if (live && id >= 0 && p0 <= wpos_hi && p0 + kKvPage - 1 >= wbeg_lo) {   /* uniform in the wave */
                /* scores: tile t's positions 4 g + e of this lane's column. Four tiles at a time,
                 * so that no product waits for the sum before it */
                kv_f4 x[4];
                kv_i4 kf[4];
                auto keys = [&](int jj) {
#pragma unroll
                    for (int t = 0; t < 4; t++) {
                        if constexpr (HD >= 128) {
                            kf[t] = *(const kv_i4 *) (kp + ((t * NJ + jj) * 64 + lane) * 16);
                        } else {
#pragma unroll
                            for (int w = 0; w < 2; w++) {
                                const kv4_u2 v = *(const kv4_u2 *) (kp + ((t * 4 + 2 * (g & 1) + w) * 16 + c16) * 8);
                                kf[t][2 * w] = (int) v[0];
                                kf[t][2 * w + 1] = (int) v[1];
                            }
                        }
                    }
                };
#pragma unroll
                for (int t = 0; t < 4; t++) x[t] = kv_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int jj = 0; jj < NJ; jj++) {
                    keys(jj);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int d = NM - 1; d >= 0; d--) {
                        kv4_i8 qf = {0, 0, 0, 0, 0, 0, 0, 0};
                        if (d < NR) {
#pragma unroll
                            for (int e = 0; e < PW; e++) qf[e] = (int) qd[d % NR][jj][e];
                        } else {
                            const uint8_t * from = far + ((d - NR) * NJ + jj) * 1536;
                            const kv4_u4 v4 = *(const kv4_u4 *) (from + 16 * lane);
                            const kv4_u2 v2 = *(const kv4_u2 *) (from + 1024 + 8 * lane);
#pragma unroll
                            for (int e = 0; e < 4; e++) qf[e] = (int) v4[e];
                            qf[4] = (int) v2[0];
                            qf[5] = (int) v2[1];
                        }
#pragma unroll
                        for (int t = 0; t < 4; t++) {
                            const kv_i4 v = kf[t];
                            const kv4_i8 k8 = {v[0], v[1], v[2], v[3], 0, 0, 0, 0};
                            const int k = t * NJ + jj;   /* its scale: byte k of ksj */
#define KV4_SCORE(KB, QB) x[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(k8, qf, x[t], 4, 2, KB, (int) ksj[k / 4], QB, (int) qs[jj][d / 4])
#define KV4_SCORE_Q(QB)                                                                                              \
    do {                                                                                                             \
        if (k % 4 == 0) KV4_SCORE(0, QB);                                                                            \
        else if (k % 4 == 1) KV4_SCORE(1, QB);                                                                       \
        else if (k % 4 == 2) KV4_SCORE(2, QB);                                                                       \
        else KV4_SCORE(3, QB);                                                                                       \
    } while (0)
                            if (d % 4 == 0) KV4_SCORE_Q(0);
                            else if (d % 4 == 1) KV4_SCORE_Q(1);
                            else if (d % 4 == 2) KV4_SCORE_Q(2);
                            else KV4_SCORE_Q(3);
#undef KV4_SCORE_Q
#undef KV4_SCORE
                        }
                    }
                }
                /* positions that are not numbers: bits 0 .. 63 */
                uint64_t nan = (uint64_t) __builtin_amdgcn_readfirstlane((int) lnan[b][1]) << 32 | (uint32_t) __builtin_amdgcn_readfirstlane((int) lnan[b][0]);
                uint32_t kbad = 0;
#pragma unroll
                for (int w = 0; w < NJ; w++) kbad |= kv4_bad(ksj[w]);
                if (__any(kbad != 0)) {
#pragma unroll
                    for (int t = 0; t < 4; t++)
#pragma unroll
                        for (int jj = 0; jj < NJ; jj++) {
                            const int k = t * NJ + jj;
                            uint64_t who = __ballot(kv4_bad(ksj[k / 4]) >> (8 * (k % 4) + 7) & 1);
                            who |= who >> 32;
                            nan |= ((who | who >> 16) & 0xffff) << (16 * t);
                        }
                }
                float ff = f;
                if (p0 < wbeg_hi || p0 + kKvPage - 1 > wpos_lo || nan) {
                    const uint32_t nan_lo = (uint32_t) nan >> (4 * g), nan_hi = (uint32_t) (nan >> 32) >> (4 * g);
#pragma unroll
                    for (int t = 0; t < 4; t++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const int p = p0 + 16 * t + 4 * g + e;
                            const bool seen = p >= beg_c && p <= pos_c, num = !((t < 2 ? nan_lo : nan_hi) >> (16 * (t & 1) + e) & 1);
                            x[t][e] = seen && num ? x[t][e] * f : -INFINITY;
                            if (seen && !num) l = __uint_as_float(0x7fc00000u);
                        }
                    ff = 1.0f;
                }
                float mp = -INFINITY;
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++) mp = fmaxf(mp, x[t][e]);
                mp = kv_rows_max(mp) * ff;
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
                        x[t][e] = __builtin_amdgcn_exp2f(fmaf(x[t][e], ff, -mref));
                        l += x[t][e];
                    }
                /* the weights' parts, pairs of positions */
                kv4_u4 P[2][DP];
#pragma unroll
                for (int w = 0; w < 2; w++)
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        float y = x[2 * w + (k >> 1)][2 * (k & 1)], z = x[2 * w + (k >> 1)][2 * (k & 1) + 1];
#pragma unroll
                        for (int d = 0; d < DP; d++) {
                            P[w][d][k] = kv_bf16x2(y, z);
                            y -= __uint_as_float(P[w][d][k] << 16);
                            z -= __uint_as_float(P[w][d][k] & 0xffff0000u);
                        }
                    }
                /* the values' operands, VG at a time, one group ahead of the products */
                constexpr int VG = 2;
                kv4_b8 vf[2][VG];
                auto values = [&](int n4) {
#pragma unroll
                    for (int e = 0; e < VG; e++) vf[n4 & 1][e] = *(const kv4_b8 *) (vp + (VG * n4 + e) * 1024);
                };
                values(0);
#pragma unroll
                for (int n4 = 0; n4 < 2 * ND / VG; n4++) {
                    if (n4 + 1 < 2 * ND / VG) values(n4 + 1);
                    __builtin_amdgcn_sched_barrier(0);
                    const int w = n4 / (ND / VG), d0 = VG * (n4 % (ND / VG));
#pragma unroll
                    for (int i = DP - 1; i >= 0; i--)
#pragma unroll
                        for (int e = 0; e < VG; e++)
                            o[d0 + e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[n4 & 1][e], __builtin_bit_cast(kv4_b8, P[w][i]), o[d0 + e], 0, 0, 0);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            if (j + 1 < seg) {
                convert(b ^ 1);
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   /* this wave's part of page j + 1 */
            }
        }
        l = kv_rows_sum(l);
        const bool whole = seg == n && off == 0;
        if (wfirst + c16 <= last) {
            if (whole) {
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int d = 0; d < ND; d += 4) {
                        const float v[4] = {o[d][i], o[d + 1][i], o[d + 2][i], o[d + 3][i]};
                        kv_write<4>(A.q, s.row + tok, head, HD, ND * (4 * g + i) + d, v, l);
                    }
            } else {
                const size_t at = (2 * (size_t) blockIdx.x + (off == 0 ? 1 : 0)) * kKv4Tile + 16 * wave + c16;
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int d = 0; d < ND; d += 4)
                        *(kv_f4 *) (A.po + at * HD + ND * (4 * g + i) + d) = kv_f4{o[d][i], o[d + 1][i], o[d + 2][i], o[d + 3][i]};
                if (g == 0) {
                    A.pml[2 * at] = m;
                    A.pml[2 * at + 1] = l;
                }
            }
        }
        if (!A.share) return;
        u += seg;
    }
}

/* Joins the shares of a (tile, kv head), a wave one column after another: lane k holds
 * share k's m and l, and eight rows of HD elements are in flight. */
template <int HD>
__global__ __launch_bounds__(256) void kv4_tile_join_kernel(const Kv4Tile A, int each) {
    constexpr int E = HD / 64;
    typedef float fe __attribute__((ext_vector_type(E)));
    extern __shared__ int lseq[];
    __shared__ int lsum[8];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int) threadIdx.x >> 6);
    const int kvh = A.c.kv_heads, G = A.q.heads / kvh, h = blockIdx.y, tile = blockIdx.x;
    int tiles = 0;
    for (int i0 = 0; i0 < A.b.nseq; i0 += 256) {
        int n = 0, sum;
        const int i = i0 + (int) threadIdx.x;
        if (i < A.b.nseq) n = (int) (((long) kv_seq(A.b, i, A.c.nslots, A.c.max_pages).count * G + kKv4Tile - 1) / kKv4Tile);
        const int at = tiles + kv4_scan(n, lsum, wave, lane, 4, sum);
        if (i < A.b.nseq) lseq[i] = at;
        tiles += sum;
    }
    __syncthreads();
    tiles = min(tiles, A.tiles);
    if (tile >= tiles) return;
    int place, first;
    const KvSeq s = kv4_tile_seq(A.b, A.c, lseq, tile, place);
    const int col0 = place * kKv4Tile, last = min(col0 + kKv4Tile, s.count * G) - 1;
    const int n = kv_span(s, col0 / G, last / G + 1, A.q.window, first), share = A.pre[A.tiles + 1];
    const long a = (long) h * A.pre[tiles] + A.pre[tile];
    const int w0 = (int) (a / share), w1 = (int) ((a + n - 1) / share), np = w1 - w0 + 1;
    if (np == 1) return;
    for (int r = 0; r < each; r++) {
        const int c = ((int) blockIdx.z * each + r) * 4 + wave;
        if (col0 + c > last) return;
        auto at = [&](int k) { return (2 * (size_t) (w0 + k) + (k == 0)) * kKv4Tile + c; };
        /* the first rows are requested before their weights are known */
        fe v[8];
        auto load = [&](int k0) {
#pragma unroll
            for (int k = 0; k < 8; k++) v[k] = *(const fe *) (A.po + at(min(k0 + k, np - 1)) * HD + E * lane);
        };
        const float2 first64 = *(const float2 *) (A.pml + 2 * at(min(lane, np - 1)));
        load(0);
        float M = first64.x, L = 0.0f;
        for (int k = lane + 64; k < np; k += 64) M = fmaxf(M, A.pml[2 * at(k)]);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
        fe sum = (fe) 0.0f;
        for (int k0 = 0; k0 < np; k0 += 64) {
            float f = 0.0f;
            if (k0 + lane < np) {
                const float2 ml = k0 ? *(const float2 *) (A.pml + 2 * at(k0 + lane)) : first64;
                f = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - M);
                L += ml.x == -INFINITY ? ml.y : f * ml.y;
            }
            const int upto = min(64, np - k0);
            for (int k1 = 0; k1 < upto; k1 += 8) {
                if (k0 + k1 > 0) load(k0 + k1);
#pragma unroll
                for (int k = 0; k < 8; k++)
                    if (k1 + k < upto) sum += __int_as_float(__builtin_amdgcn_readlane(__float_as_int(f), k1 + k)) * v[k];
            }
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) L += __shfl_xor(L, o, 64);
        float o[E];
#pragma unroll
        for (int e = 0; e < E; e++) o[e] = sum[e];
        const int tok = (col0 + c) / G;
        kv_write<E>(A.q, s.row + tok, h * G + (col0 + c) - tok * G, HD, E * lane, o, L);
    }
}

/* -------------------------------------------------------------------- host */

struct Kv4Plan {
    int max_q;
    bool flat, quad, whole;   /* the few-column kernels: with parts in columns, with no join */
    int cmax, seq_tiles;      /* their columns, and tiles of a sequence, at most */
    long tiles;               /* the many-column kernel's, of the batch */
    int groups;               /* workgroups of shares; 0: a workgroup a tile and kv head */
    size_t pre, po, pml, bytes;
};

Kv4Plan kv4_plan(const sparkmv_kv4_cache * c, const sparkmv_kv_batch * b, int heads, int window) {
    Kv4Plan p = {};
    const int G = heads / c->kv_heads;
    p.max_q = b->qstart ? (b->max_q < b->ntok ? b->max_q : b->ntok) : 1;
    const long cols = (long) p.max_q * G, hd = c->head_dim;
    const long len = b->max_len > 0 ? b->max_len : (long) c->max_pages * kKvPage;
    const long pages = (len + kKvPage - 1) / kKvPage;
    const long in_window = ((long) window + kKvPage - 2) / kKvPage + 1, seen = window > 0 && in_window < pages ? in_window : pages;
    size_t off = 0;
    auto take = [&](size_t bytes) { const size_t o = off; off += (bytes + 255) & ~(size_t) 255; return o; };
    /* few columns read a tile's pages again for each 16; blocks of 12 bf16 tokens with 4
     * heads each (48 columns) of 3 sequences of up to 6000 23.8 us, tiles of 128 30.3, of one
     * of 60000 49 and 55; of 16 tokens 29.8 and 33.8, 57.7 and 57.1 */
    p.flat = cols <= 3 * kKv4Cols;
    if (p.flat) {
        p.quad = cols <= 4;
        p.cmax = (int) (cols < kKv4Cols ? cols : kKv4Cols);
        p.seq_tiles = (int) ((cols + kKv4Cols - 1) / kKv4Cols);
        /* whole contexts against shares and a join: 16 pages of one sequence 11.6 and 13.3
         * us, 32 17.4 and 13.4; 9 pages of 24 sequences 10.7 and 19.6 */
        p.whole = cols <= kKv4Cols && seen <= 16;
        /* One workgroup a CU has fewer results to join than two, which keep more loads in
         * flight and even out lengths that differ. The host knows no lengths: `all` is what
         * max_len allows, which sequences of unequal lengths do not reach. One against two
         * with four kv heads, us. head_dim 256, one sequence of 8000 14.4 and 17.3, of 32000
         * 21.0 and 25.3, of 128000 43.4 and 44.0; 16 of 16000 68 and 70, of 24000 93 and 100;
         * of up to 16000 21.8 and 25.5, 48 of up to 12000 54.8 both, 32 of up to 32000 79
         * and 77. 128: one of 64000 15.9 and 17.1, 16 of 8000 22.3 and 21.5, 64 of 16000 103
         * and 111; 48 of up to 12000 27.9 and 25.3. 64: one of 64000 13.4 and 14.1, 16 of
         * 8000 18.5 and 16.9, of 32000 45.6 and 35.9; 48 of up to 12000 23.4 and 20.7 */
        const long all = seen * p.seq_tiles * b->nseq * c->kv_heads;
        const long two = all >= (long) cu_count() * (hd == 256 ? 56 : 24) ? 2 : 1;
        const long most = two * cu_count() < kKv4Most ? two * cu_count() : kKv4Most;
        p.groups = (int) (all < 1 ? 1 : (all < most ? all : most));
        p.pre = take(((size_t) b->nseq + 2) * 4);
        p.po = take((size_t) p.groups * 2 * p.cmax * hd * 4);
        p.pml = take((size_t) p.groups * 2 * p.cmax * 2 * 4);
    } else {
        p.tiles = (long) b->ntok * G / kKv4Tile + b->nseq;
        /* shares while their counts fit, one a CU: 512 tokens at 1000 54.4 us, with half as
         * many 68.0 */
        if (p.tiles <= kKv4Tiles && p.tiles * ((long) c->max_pages + kKv4TileItem) <= 0x7fffffffl / c->kv_heads) {
            const long all = pages * p.tiles * c->kv_heads, most = cu_count();
            p.groups = (int) (all < 1 ? 1 : (all < most ? all : most));
            p.pre = take(((size_t) p.tiles + 2) * 4);
            p.po = take((size_t) p.groups * 2 * kKv4Tile * hd * 4);
            p.pml = take((size_t) p.groups * 2 * kKv4Tile * 2 * 4);
        }
    }
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
    /* the few-column kernels' count of pages, and where the last shares would end */
    if (p.flat && (long) batch->nseq * p.seq_tiles > (0x7fffffffl - 2 * kKv4Most) / ((long) cache->max_pages + kKv4Item) / cache->kv_heads) {
        set_error("%d sequences of up to %d pages and %d kv heads are too many for one call", batch->nseq, cache->max_pages,
                  cache->kv_heads);
        return -1;
    }
    if (!p.flat && p.tiles * cache->kv_heads > kKvThreads / 512) {
        set_error("attention over %ld tiles of tokens is too much for one call", p.tiles * cache->kv_heads);
        return -1;
    }
    if (p.bytes && (!q.work || !kv_aligned(q.work, 256) || q.work_bytes < p.bytes)) {
        set_error("attention needs %zu bytes of 256-byte aligned workspace, not %zu", p.bytes, q.work ? q.work_bytes : 0);
        return -1;
    }
    hipStream_t s = (hipStream_t) stream;
    uint8_t * mem = (uint8_t *) q.work;
    const int hd = cache->head_dim;
    if (!p.flat) {
        Kv4Tile t;
        t.c = *cache; t.b = *batch; t.q = q;
        t.b.max_q = p.max_q;
        t.tiles = (int) p.tiles;
        t.share = p.groups;
        t.pre = (int *) (mem + p.pre); t.po = (float *) (mem + p.po); t.pml = (float *) (mem + p.pml);
        const uint32_t lists = p.groups ? ((uint32_t) batch->nseq + (uint32_t) p.tiles + 1) * 4 : 0;
        const dim3 grid((unsigned) (p.groups ? p.groups : p.tiles * cache->kv_heads));
        /* columns a wave of the join: one or two, with 12 tiles' kv heads 27.5 us for the call
         * and 30.3, with 68 40.8 and 39.1 */
        const int each = p.tiles * cache->kv_heads * (kKv4Tile / 4) > 4 * cu_count() ? 2 : 1;
        const dim3 join((unsigned) p.tiles, (unsigned) cache->kv_heads, (unsigned) (kKv4Tile / 4 / each));
#define KV4_TILE(H, DP)                                                                                              \
    do {                                                                                                             \
        static LdsAllowed allowed;                                                                                   \
        if (lds_allow(allowed, (const void *) kv4_tile_kernel<H, DP>, kv4_tile_lds(H) + lists + 2048,                \
                      "LDS opt-in for the kv4 attention"))                                                           \
            return -1;                                                                                               \
        hipLaunchKernelGGL((kv4_tile_kernel<H, DP>), grid, dim3(512), kv4_tile_lds(H) + lists, s, t);                \
    } while (0)
#define KV4_TILE_D(H)                                                                                                \
    do {                                                                                                             \
        if (q.out_dtype == SPARKMV_X_F32) KV4_TILE(H, 3);                                                            \
        else KV4_TILE(H, 2);                                                                                         \
        if (p.groups)                                                                                                \
            hipLaunchKernelGGL(kv4_tile_join_kernel<H>, join, dim3(256), ((uint32_t) batch->nseq + 1) * 4, s, t, each); \
    } while (0)
        if (hd == 64) KV4_TILE_D(64);
        else if (hd == 128) KV4_TILE_D(128);
        else KV4_TILE_D(256);
#undef KV4_TILE_D
#undef KV4_TILE
        return kv_check_launch("kv4 attention launch");
    }
    Kv4Flat f;
    f.c = *cache; f.b = *batch; f.q = q;
    f.b.max_q = p.max_q;
    f.cmax = p.cmax;
    f.pre = (int *) (mem + p.pre); f.po = (float *) (mem + p.po); f.pml = (float *) (mem + p.pml);
    const dim3 join((unsigned) batch->nseq, (unsigned) cache->kv_heads, (unsigned) (p.cmax * p.seq_tiles));
    const uint32_t pre = batch->nseq > 64 ? ((uint32_t) batch->nseq + 1) * 4 : 0;
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
        if (p.quad) {                                                                                                \
            KV4_FLAT(H, 0, 3);                                                                                       \
        } else if (q.q_dtype == SPARKMV_X_F32) {                                                                     \
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
