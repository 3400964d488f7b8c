/* kv_attend.hip — attention over the paged 8-bit cache (include/sparkmv.h):
 *   out = sum_p softmax_p(scale * q . k_p) v_p (* sigmoid(gate))
 * over the positions p that a token sees.
 *
 * Both products run on the 8-bit integer matrix instructions, 16 x 16 x 64,
 * with the codes as they lie in memory: nothing is converted. What meets them
 * is an f32 query element or weight as an integer, written in D signed digits
 * of base 256 (d0 2^8(D-1) + .. + d(D-1)); a digit's sums are exact in i32
 * (256 * 127 * 128 < 2^23), and D digits' sums make the product.
 *
 *   A query element is an integer at a power of two that the head's largest
 *   element sets: 31 bits with four digits, more than f32 holds; 23 with three,
 *   f32's own 24 bits of the largest element to within one.
 *
 *   A weight e^(s - m) takes as m the largest score of its own page, so its
 *   integer is fine against the page's weights whatever the rest of the sequence
 *   holds: with four digits 31 bits of the page's largest, with three 23 bits of
 *   the page's sum. The page's sum enters the f32 output times value scale *
 *   e^(m - M), where M, a running reference, moves only when a page passes it by
 *   2^kKvLag.
 *
 * Four digits serve f32 outputs; three serve bf16 ones, except where four cost
 * nothing. Two would be enough only for rows without outliers: with one query
 * element 100 times the others 15 bits of it leave their scores off by 1 %, and
 * where the first position has nearly all the weight (and next to no value)
 * those of the others are a few steps of 2^-15 each. Scores, weights' sums and
 * outputs are f32. */
#include "kv.h"
#include "kv_attend.h"

#include <math.h>

namespace sparkmv {

namespace {

/* 16 query elements as f32 */
__device__ __forceinline__ void kv_load16(const sparkmv_kv_query & q, size_t at, float * x) {
    if (q.q_dtype == SPARKMV_X_F32) {
        const float * p = (const float *) q.q + at;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const kv_f4 v = *(const kv_f4 *) (p + 4 * k);
#pragma unroll
            for (int i = 0; i < 4; i++) x[4 * k + i] = v[i];
        }
    } else {
        const uint16_t * p = (const uint16_t *) q.q + at;
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
}

/* the exponent that the largest element sets, over the lanes of a column (which
 * hold its elements between them); bad: one is not finite */
template <int NC>
__device__ __forceinline__ int kv_q_exponent(const float (&x)[NC][16], bool & bad) {
    uint32_t big = 0;
#pragma unroll
    for (int c = 0; c < NC; c++)
#pragma unroll
        for (int e = 0; e < 16; e++) big = max(big, __float_as_uint(x[c][e]) & 0x7fffffffu);
    big = max(big, (uint32_t) __shfl_xor((int) big, 16, 64));
    big = max(big, (uint32_t) __shfl_xor((int) big, 32, 64));
    bad = big >= 0x7f800000u;
    int ex = 0;
    (void) frexpf(__uint_as_float(bad ? 0u : big), &ex);
    return ex;
}

/* ------------------------------------------------------------- few columns
 *
 * Up to four columns (token, query head) of a kv head: a decode step of up to
 * four query heads per kv head. Bound by reading the codes once. The sixteen
 * columns of a tile are the four columns times four digits, so f32's whole
 * precision costs no further instruction. The four lanes of a quad add their
 * digits' sums up so that each ends with a quarter of the column's scores, takes
 * their weights, and hands them back as integers for the others' digits.
 *
 * Workgroups take equal shares of all (sequence, kv head, page) in that order,
 * so lengths may differ by any amount; a kv head of a sequence counts kKvItem
 * pages more than it has, for what beginning it costs. A share's pages of one
 * kv head go to the four waves in turn, whose results meet in LDS; a kv head's
 * pages that lie in one share are written out at once, others as a partial
 * result that a second launch joins.
 *
 * A short call is bound by its chain of reads (positions, page numbers, codes)
 * and by fetching instructions that run once, about 0.5 us a kilobyte: so the
 * codes are requested before the queries are looked at, and what runs once is
 * kept in loops.
 *
 * 16 query and 4 kv heads of 256: one token at position 131071 55.4 us (4.85 TB/s)
 * and 7.2 for the join, 48 at up to 12000 66.6 (4.8 TB/s) and 6.6, one at 1003 (one
 * launch) 12.1, 24 in windows of 512 11.6. */
constexpr int kKvItem = 8;          /* 48 sequences of up to 12000: 83 us, without it 184 */
constexpr int kKvFlatMost = 1024;   /* workgroups, at most */
/* Pages of a sequence that one workgroup takes alone, in turns of its eight waves;
 * above, shares and a join. us alone and in shares, 4 kv heads of 256: one sequence of
 * 8 pages 9.6 and 11.9, 16 12.1 and 12.2, 24 15.0 and 12.3; 8 sequences of 24 pages
 * 16.7 and 17.3, 32 19.8 and 18.2; 24 of 24 17.9 and 26.9, 32 31.0 and 31.3. So 16, or
 * 24 from 32 workgroups on. */
int kv_whole(long items) { return items < 32 ? 16 : 24; }

struct KvFlat {
    sparkmv_kv_cache c;
    sparkmv_kv_batch b;
    sparkmv_kv_query q;
    int * pre;       /* [nseq + 2]: what one kv head of the sequences before counts; the share */
    float * po;      /* [workgroups][2][4][HD] */
    float * pml;     /* [workgroups][2][4][2] */
};

constexpr int kv_flat_lds(int hd, int waves) { return waves * 16 * (hd + 4) * 4 + 16 * hd; }

/* WAVES 4: shares; 8: workgroup i * kv_heads + h takes the whole of a sequence's
 * kv head, and no join follows */
template <int HD, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void kv_flat_kernel(const KvFlat A) {
    constexpr int NC = HD / 64, ND = HD / 16, NT = 64 * WAVES, E = HD / 64, LO = HD + 4;
    constexpr int V = WAVES == 8 ? 2 : 4;   /* elements a thread at the end */
    constexpr bool WHOLE = WAVES == 8;
    extern __shared__ __attribute__((aligned(16))) uint8_t ldyn[];
    float * lo = (float *) ldyn;                      /* [WAVES][16][LO]: a wave's output, digit by digit */
    uint8_t * lq = ldyn + WAVES * 16 * LO * 4;        /* [16 * HD]: query digits as the matrix instruction's lanes take them */
    int * lpre = (int *) (lq + 16 * HD);              /* [nseq + 1], shares of more than 64 sequences only */
    __shared__ int lsum[4];
    __shared__ float lcs[4], lbad[4], lm[WAVES][4], ll[WAVES][4];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 4, c16 = lane & 15;
    const int col = c16 >> 2, dg = c16 & 3;
    const int kvh = A.c.kv_heads, G = A.q.heads / kvh, nseq = A.b.nseq;
    /* shares: what a kv head of each sequence counts. Up to 64 sequences a lane
     * each, in every wave; more through LDS */
    const bool few = nseq <= 64;
    KvSeq mine = {0, 0, 0, 0};
    int cost = 0, before = 0;
    int ubeg = blockIdx.x, uend = ubeg + 1;
    if constexpr (!WHOLE) {
        int total;
        if (few) {
            if (lane < nseq) mine = kv_seq(A.b, lane, A.c.nslots, A.c.max_pages);
            int first;
            if (mine.count > 0) cost = kv_span(mine, 0, mine.count, A.q.window, first) + kKvItem;
            int scan = cost;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int v = __shfl_up(scan, o, 64);
                if (lane >= o) scan += v;
            }
            before = scan - cost;
            total = __builtin_amdgcn_readlane(scan, 63);
        } else {
            const int per = (nseq + 255) / 256, i0 = min(nseq, tid * per), i1 = min(nseq, i0 + per);
            int sum = 0;
            for (int i = i0; i < i1; i++) {
                int first;
                const KvSeq s = kv_seq(A.b, i, A.c.nslots, A.c.max_pages);
                lpre[i] = sum;
                if (s.count > 0) sum += kv_span(s, 0, s.count, A.q.window, first) + kKvItem;
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
            if (tid == 255) lpre[nseq] = base + sum;
            __syncthreads();
            total = __builtin_amdgcn_readfirstlane(lpre[nseq]);
        }
        const int share = max((total * kvh + (int) gridDim.x - 1) / (int) gridDim.x, 1);
        if (blockIdx.x == 0) {
            if (few) {
                if (tid < nseq) A.pre[tid] = before;
            } else {
                for (int i = tid; i < nseq; i += 256) A.pre[i] = lpre[i];
            }
            if (tid == 0) {
                A.pre[nseq] = total;
                A.pre[nseq + 1] = share;
            }
        }
        ubeg = (int) blockIdx.x * share;
        uend = min(total * kvh, ubeg + share);
    }
    const float wdig = (float) (1 << (8 * (3 - dg)));
    const uint32_t sel = (uint32_t) (3 - dg) | (uint32_t) (7 - dg) << 8 | 0x0c0c0000u, flip = dg ? 0x80808080u : 0u;
    /* byte 3 - dg of four integers with 0x808080 added: the digit, its sign bit
     * turned in the lower three */
    auto digits = [&](uint32_t a, uint32_t b, uint32_t c, uint32_t d) -> int {
        const uint32_t lo2 = __builtin_amdgcn_perm(b, a, sel), hi2 = __builtin_amdgcn_perm(d, c, sel);
        return (int) ((lo2 | hi2 << 16) ^ flip);
    };
    for (int u = ubeg; u < uend;) {
        int h, off = 0, n, seg, first;
        KvSeq s;
        if constexpr (WHOLE) {
            const int i = u / kvh;
            h = u - i * kvh;
            s = kv_seq(A.b, i, A.c.nslots, A.c.max_pages);
            if (s.count <= 0) return;
            seg = n = kv_span(s, 0, s.count, A.q.window, first);
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
            n = kv_span(s, 0, s.count, A.q.window, first);
            h = in / (n + kKvItem);
            off = in - h * (n + kKvItem);
            if (off >= n) {
                u += n + kKvItem - off;
                continue;
            }
            seg = min(n - off, uend - u);
        }
        const int ncol = s.count * G, tok = min(col / G, s.count - 1);
        const int pos_c = s.pos + tok, beg_c = A.q.window > 0 && pos_c + 1 > A.q.window ? pos_c + 1 - A.q.window : 0;
        /* positions that every column sees */
        const int all_lo = A.q.window > 0 && s.pos + s.count > A.q.window ? s.pos + s.count - A.q.window : 0, all_hi = s.pos;
        const int * table = A.c.pages + (size_t) s.slot * A.c.max_pages + first + off;
        /* 64 pages of this wave at a time: their numbers and scales are held one a lane */
        int id, count;
        float ks, vs;
        uint64_t there;
        kv_i4 kr[NC][4], vr[ND];
        /* buffer loads: a page's base is uniform, so all of its 32 addresses take
         * one register a lane (64-bit ones took 60, which then spilled) */
        const uint32_t klane = c16 * 64 + 16 * g, vlane = (g * HD + c16) * 16;
        auto page_at = [&](const int8_t * p, int j) {
            const uint64_t at = (uint64_t) p + ((uint64_t) (uint32_t) __builtin_amdgcn_readlane(id, j) * (uint32_t) kvh + (uint32_t) h) * (kKvPage * HD);
            const uint64_t lo = (uint32_t) __builtin_amdgcn_readfirstlane((int) (uint32_t) at);
            const uint64_t hi = (uint32_t) __builtin_amdgcn_readfirstlane((int) (at >> 32));
            return __builtin_amdgcn_make_buffer_rsrc((void *) (hi << 32 | lo), 0, kKvPage * HD, 0x00027000);
        };
        auto fetch_k = [&](int j) {
            const auto p = page_at(A.c.k, j);
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int t = 0; t < 4; t++) kr[c][t] = (kv_i4) __builtin_amdgcn_raw_buffer_load_b128(p, klane, c * 4096 + t * 1024, 0);
        };
        auto begin = [&](int base) {
            count = min((seg - base + WAVES - 1) / WAVES, 64);
            id = 0;
            ks = vs = 0.0f;
            bool have = false;
            if (lane < count) {
                id = table[base + WAVES * lane];
                have = id >= 0 && id < A.c.npages;
                id = have ? id : 0;
                const uint64_t at = (uint64_t) (uint32_t) id * (uint32_t) kvh + (uint32_t) h;
                ks = A.c.k_scale[at];
                vs = A.c.v_scale[at];
            }
            there = __ballot(have);
            fetch_k(0);
            __builtin_amdgcn_sched_barrier(0);
        };
        auto begin_v = [&]() {
            const auto p = page_at(A.c.v, 0);
#pragma unroll
            for (int d = 0; d < ND; d++) vr[d] = (kv_i4) __builtin_amdgcn_raw_buffer_load_b128(p, vlane, d * 256, 0);
            __builtin_amdgcn_sched_barrier(0);
        };
        /* the columns' digits, a wave a column and E elements a lane. The elements
         * are requested before the codes: loads return in order */
        const bool live = wave < ncol;
        float x[E];
        if (wave < 4) {
            const int t = live ? wave / G : 0, head = h * G + (live ? wave % G : 0);
            const size_t at = (size_t) (s.row + t) * A.q.ldq + (size_t) head * HD + E * lane;
#pragma unroll
            for (int e = 0; e < E; e++)
                x[e] = A.q.q_dtype == SPARKMV_X_F32 ? kv_load((const float *) A.q.q + at + e) : kv_load((const uint16_t *) A.q.q + at + e);
        }
        if (wave < seg) begin(wave);
        if (wave < 4) {
            uint32_t big = 0, y[4] = {0, 0, 0, 0};
#pragma unroll
            for (int e = 0; e < E; e++) big = max(big, __float_as_uint(x[e]) & 0x7fffffffu);
            /* non-negative floats, a NaN above the infinities, order as integers do */
            big = kv_wave_max(big);
            const bool bad = big >= 0x7f800000u;
            int ex = 0;
            (void) frexpf(__uint_as_float(bad ? 0u : big), &ex);
#pragma unroll
            for (int e = 0; e < E; e++) y[e] = (live && !bad ? (uint32_t) (int) rintf(ldexpf(x[e], 30 - ex)) : 0u) + 0x808080u;
            /* element d of digit column n at ((d / 64 * 64 + d / 16 % 4 * 16 + n) * 16 + d % 16 */
            const int d0 = E * lane;
            uint8_t * to = lq + (((d0 >> 6) * 64 + (d0 >> 4 & 3) * 16 + 4 * wave) * 16 + (d0 & 15));
#pragma unroll
            for (int d = 0; d < 4; d++) {
                const uint32_t b = 3 - d, pick = b | (b + 4) << 8 | 0x0c0c0000u, turn = d ? 0x80808080u : 0u;
                const uint32_t w = (__builtin_amdgcn_perm(y[1], y[0], pick) | __builtin_amdgcn_perm(y[3], y[2], pick) << 16) ^ turn;
                if constexpr (E == 4) *(uint32_t *) (to + 16 * d) = w;
                else if constexpr (E == 2) *(uint16_t *) (to + 16 * d) = (uint16_t) w;
                else to[16 * d] = (uint8_t) w;
            }
            if (lane == 0) {
                lcs[wave] = ldexpf(A.q.scale * kKvLog2e, ex - 30);
                lbad[wave] = bad ? __uint_as_float(0x7fc00000u) : 0.0f;
            }
        }
        if (wave < seg) begin_v();
        __syncthreads();
        const float cs = lcs[col];
        float m = -INFINITY, l = 0.0f;
        kv_f4 o[ND];
#pragma unroll
        for (int d = 0; d < ND; d++) o[d] = kv_f4{0.f, 0.f, 0.f, 0.f};
        for (int base = wave; base < seg; base += 64 * WAVES) {
            if (base > wave) {
                begin(base);
                begin_v();
            }
            for (int j = 0; j < count; j++) {
                const int nx = min(j + 1, count - 1);
                float a[4][4];
                /* read again for each page: held, they would leave too few registers */
                asm volatile("" ::: "memory");
                kv_i4 qd[NC];
#pragma unroll
                for (int c = 0; c < NC; c++) qd[c] = *(const kv_i4 *) (lq + (c * 64 + lane) * 16);
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    kv_i4 acc = kv_i4{0, 0, 0, 0};
#pragma unroll
                    for (int c = 0; c < NC; c++) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(kr[c][t], qd[c], acc, 0, 0, 0);
#pragma unroll
                    for (int e = 0; e < 4; e++) a[t][e] = (float) acc[e] * wdig;
                }
                __builtin_amdgcn_sched_barrier(0);
                fetch_k(nx);
                __builtin_amdgcn_sched_barrier(0);
                const float kscale = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(ks), j));
                const float vscale = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(vs), j));
                const float f = cs * kscale;
                /* x[e]: the score of position 16 dg + 4 g + e, the digits' sums of the quad added up */
                float x[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float k0 = (dg & 2 ? a[2][e] : a[0][e]) + kv_quad<kKvXor2>(dg & 2 ? a[0][e] : a[2][e]);
                    const float k1 = (dg & 2 ? a[3][e] : a[1][e]) + kv_quad<kKvXor2>(dg & 2 ? a[1][e] : a[3][e]);
                    x[e] = ((dg & 1 ? k1 : k0) + kv_quad<kKvXor1>(dg & 1 ? k0 : k1)) * f;
                }
                const int p0 = (first + off + base + WAVES * j) * kKvPage;
                const bool ok = there >> j & 1;
                if (!ok || p0 < all_lo || p0 + kKvPage - 1 > all_hi || kscale != kscale) {
                    bool any = false;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int p = p0 + 16 * dg + 4 * g + e;
                        const bool seen = ok && p >= beg_c && p <= pos_c;
                        any = any || seen;
                        x[e] = seen && kscale == kscale ? x[e] : -INFINITY;
                    }
                    if (any && kscale != kscale) l = kscale;   /* NaN to the end for a column that sees some of it */
                }
                float mp = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
                mp = fmaxf(mp, kv_quad<kKvXor1>(mp));
                mp = fmaxf(mp, kv_quad<kKvXor2>(mp));
                mp = kv_rows_max(mp);
                if (__any(mp > m + kKvLag)) {
                    const float mn = fmaxf(m, mp);
                    const float r = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
                    l *= r;
#pragma unroll
                    for (int d = 0; d < ND; d++) o[d] *= r;
                    m = mn;
                }
                const float mref = mp == -INFINITY ? 0.0f : mp;
                float sum = 0.0f;
                int y[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float p = __builtin_amdgcn_exp2f(x[e] - mref);
                    sum += p;
                    y[e] = (int) (p * 1073741824.0f) + 0x808080;
                }
                /* tile t's weights are lane t's of the quad */
                kv_i4 P;
                P[0] = digits(kv_quad<0x00>(y[0]), kv_quad<0x00>(y[1]), kv_quad<0x00>(y[2]), kv_quad<0x00>(y[3]));
                P[1] = digits(kv_quad<0x55>(y[0]), kv_quad<0x55>(y[1]), kv_quad<0x55>(y[2]), kv_quad<0x55>(y[3]));
                P[2] = digits(kv_quad<0xaa>(y[0]), kv_quad<0xaa>(y[1]), kv_quad<0xaa>(y[2]), kv_quad<0xaa>(y[3]));
                P[3] = digits(kv_quad<0xff>(y[0]), kv_quad<0xff>(y[1]), kv_quad<0xff>(y[2]), kv_quad<0xff>(y[3]));
                const float step = mp == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mp - m);
                l += sum * step;
                const float w = mp == -INFINITY ? 0.0f : step * vscale;
                /* four at a time: with all of them ahead their sums would not fit the registers */
                const auto vnext = page_at(A.c.v, nx);
#pragma unroll
                for (int d0 = 0; d0 < ND; d0 += 4) {
                    kv_i4 acc[4];
#pragma unroll
                    for (int d = 0; d < 4; d++) acc[d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(vr[d0 + d], P, kv_i4{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
                    for (int d = 0; d < 4; d++) vr[d0 + d] = (kv_i4) __builtin_amdgcn_raw_buffer_load_b128(vnext, vlane, (d0 + d) * 256, 0);
#pragma unroll
                    for (int d = 0; d < 4; d++)
#pragma unroll
                        for (int e = 0; e < 4; e++) o[d0 + d][e] += w * (float) acc[d][e];
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        l += kv_quad<kKvXor1>(l);
        l += kv_quad<kKvXor2>(l);
        l = kv_rows_sum(l);
        /* the waves' outputs meet in LDS */
#pragma unroll
        for (int d = 0; d < ND; d++) *(kv_f4 *) (lo + (wave * 16 + c16) * LO + 16 * d + 4 * g) = o[d];
        if (g == 0 && dg == 0) {
            lm[wave][col] = m;
            ll[wave][col] = l + lbad[col];
        }
        __syncthreads();
        const bool whole = WHOLE || seg == n;
        const size_t at = 2 * (size_t) blockIdx.x + (off == 0 ? 1 : 0);
        for (int k = tid; k < ncol * (HD / V); k += NT) {
            const int cc = k / (HD / V), d = V * (k % (HD / V));
            float M = lm[0][cc], L = 0.0f, v[V];
#pragma unroll
            for (int w = 1; w < WAVES; w++) M = fmaxf(M, lm[w][cc]);
#pragma unroll
            for (int e = 0; e < V; e++) v[e] = 0.0f;
#pragma unroll 4
            for (int w = 0; w < WAVES; w++) {
                typedef float fv __attribute__((ext_vector_type(V)));
                fv p[4];
#pragma unroll
                for (int i = 0; i < 4; i++) p[i] = *(const fv *) (lo + (w * 16 + 4 * cc + i) * LO + d);
                const float r = lm[w][cc] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(lm[w][cc] - M);
                L += lm[w][cc] == -INFINITY ? ll[w][cc] : r * ll[w][cc];
                /* digits 2^24 .. 2^0, over the weight's 2^30 */
#pragma unroll
                for (int e = 0; e < V; e++) v[e] += r * (((p[3][e] * 0x1p-30f + p[2][e] * 0x1p-22f) + p[1][e] * 0x1p-14f) + p[0][e] * 0x1p-6f);
            }
            if (whole) {
                kv_write<V>(A.q, s.row + cc / G, h * G + cc % G, HD, d, v, L);
            } else {
                float * to = A.po + (at * 4 + cc) * HD + d;
#pragma unroll
                for (int e = 0; e < V; e++) to[e] = v[e];
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

/* Joins the partial results of one column of a (sequence, kv head), in the order
 * of its pages: its first share wrote slot 1, the later ones slot 0. */
template <int HD>
__global__ __launch_bounds__(512) void kv_flat_join_kernel(const KvFlat A) {
    __shared__ float wts[kKvFlatMost];
    __shared__ __attribute__((aligned(16))) float acc[7 * HD];
    const int i = blockIdx.x, h = blockIdx.y, c = blockIdx.z, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int kvh = A.c.kv_heads, G = A.q.heads / kvh;
    const int before = A.pre[i], all = A.pre[i + 1] - before, n = all - kKvItem, share = A.pre[A.b.nseq + 1];
    if (all == 0) return;
    const int a = before * kvh + h * all, w0 = a / share, w1 = (a + n - 1) / share;
    if (w0 == w1) return;
    const KvSeq s = kv_seq(A.b, i, A.c.nslots, A.c.max_pages);
    if (c >= s.count * G) return;
    float o[HD / 64];
    const float L = kv_join<HD, 8>(A.po, A.pml, w1 - w0 + 1, [&](int k) { return (2 * (size_t) (w0 + k) + (k == 0)) * 4 + c; },
                                   wts, acc, wave, lane, o);
    if (wave) return;
    kv_write<HD / 64>(A.q, s.row + c / G, h * G + c % G, HD, HD / 64 * lane, o, L);
}

/* -------------------------------------------------------------- many columns
 *
 * A workgroup takes 16 * WQ columns (token, query head) of a kv head and a share
 * of the pages they see. A page's codes go to LDS as they lie (direct loads, the
 * next page's while this one is worked). WQ waves take 16 columns each; with
 * WQ < 4 the other waves work on the same columns and take a part of the
 * elements in the product with the values (and repeat the scores). Each digit is
 * an instruction of its own here, on the same codes. Work that is split over the
 * pages is joined by a second launch.
 *
 * A chunk of 512 tokens at 16384 (16 query, 4 kv heads of 256, bf16 out): the call
 * with its join takes 233 us for 140 GFLOP, 300 with f32 outputs and their four
 * digits; bound by the vector instructions around the products (535 a wave and page,
 * half of them the values' sums from i32; VALU 67 % busy, MFMA 40). Six waves a
 * workgroup, for three a SIMD, took half as long again: they do not fill the SIMDs
 * evenly. Three blocks of 8 at 6001 (f32 out): 19 us and 6.9 for the join. */
struct KvTile {
    sparkmv_kv_cache c;
    sparkmv_kv_batch b;
    sparkmv_kv_query q;
    int nsplit;
    float * po;      /* [tiles][kv_heads][columns][nsplit][HD] */
    float * pml;     /* [tiles][kv_heads][columns][nsplit][2] */
};

constexpr int kKvIds = 256;   /* page numbers held at a time */

template <int HD, int D, int WQ>
__global__ __launch_bounds__(256, 2) void kv_tile_kernel(const KvTile A) {
    constexpr int NC = HD / 64, WD = 4 / WQ, ND = HD / 16 / WD, HALF = kKvPage * HD;
    /* what a weight of 1, or all of a page's weights together, becomes: 2^30; below
     * 0x7f7f7f by what the f32 roundings may add, so that three digits hold it */
    constexpr float PMAX = D == 3 ? 8355584.0f : 1073741824.0f;
    constexpr uint32_t BIAS = D == 3 ? 0x8080u : 0x808080u;
    typedef __attribute__((address_space(3))) void lds_void;
    extern __shared__ __attribute__((aligned(16))) uint8_t lbuf[];   /* [2][keys, values] */
    __shared__ int lfind[8];
    __shared__ int lid[kKvIds];
    __shared__ float lks[kKvIds], lvs[kKvIds];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, g = lane >> 4, c16 = lane & 15;
    const int wq = wave % WQ, wd = wave / WQ, kvh = A.c.kv_heads, G = A.q.heads / kvh;
    /* splits next to each other, then kv heads, then tiles: the tiles that the batch
     * does not fill are no XCD's alone, and an XCD sees few (split, kv head) */
    const int split = (int) blockIdx.x % A.nsplit, th = (int) blockIdx.x / A.nsplit, h = th % kvh, tile = th / kvh;
    KvSeq s;
    int place;
    if (!kv_find_tile(A.b, A.c, G, 16 * WQ, tile, lfind, s, place)) return;
    const int ncol = s.count * G, col0 = place * 16 * WQ, t0 = col0 / G, t1 = min(col0 + 16 * WQ - 1, ncol - 1) / G + 1;
    int first;
    const int npages = kv_span(s, t0, t1, A.q.window, first), per = (npages + A.nsplit - 1) / A.nsplit;
    const int jbeg = split * per, jend = min(npages, jbeg + per);
    if (jbeg >= jend) return;
    first += jbeg;
    const int n = jend - jbeg;
    const int * table = A.c.pages + (size_t) s.slot * A.c.max_pages + first;
    auto ids = [&](int j0) {   /* pages j0 .. of the share; a barrier on both sides */
        __syncthreads();
        if (j0 + tid < n) {
            int id = table[j0 + tid];
            const bool have = id >= 0 && id < A.c.npages;
            lid[tid] = have ? id : -1;
            lks[tid] = have ? A.c.k_scale[(size_t) id * kvh + h] : 0.0f;
            lvs[tid] = have ? A.c.v_scale[(size_t) id * kvh + h] : 0.0f;
        }
        __syncthreads();
    };
    /* a kilobyte of keys, 16 positions x 64 bytes, enters LDS as the matrix
     * instruction's lanes take it (lane 16 g + position: 16 bytes), so that reads
     * are contiguous: as it lies, sixteen lanes would read at a stride of 64 bytes */
    const uint32_t klane = c16 * 64 + 16 * g;
    auto fetch = [&](int j, int b) {
        const size_t at = ((size_t) max(__builtin_amdgcn_readfirstlane(lid[j & (kKvIds - 1)]), 0) * kvh + h) * (size_t) HALF;
        const int8_t * kc = A.c.k + at, * vc = A.c.v + at;
        uint8_t * to = lbuf + (size_t) b * 2 * HALF;
#pragma unroll
        for (int k = 0; k < HALF / 4096; k++) {
            const int o = (4 * k + wave) * 1024;
            __builtin_amdgcn_global_load_lds((const void *) (kc + o + klane), (lds_void *) (to + o), 16, 0, 0);
            __builtin_amdgcn_global_load_lds((const void *) (vc + o + 16 * lane), (lds_void *) (to + HALF + o), 16, 0, 0);
        }
    };
    ids(0);
    fetch(0, 0);
    /* this wave's columns */
    const int wfirst = col0 + 16 * wq, cc = min(wfirst + c16, ncol - 1), tok = cc / G, head = h * G + cc - tok * G;
    const bool live = wfirst < ncol;   /* uniform in the wave */
    const int pos_c = s.pos + tok, beg_c = A.q.window > 0 && pos_c + 1 > A.q.window ? pos_c + 1 - A.q.window : 0;
    const int tlo = min(wfirst, ncol - 1) / G, thi = min(wfirst + 15, ncol - 1) / G;
    const int wpos_lo = s.pos + tlo, wpos_hi = s.pos + thi;   /* the wave's first and last token */
    const int wbeg_lo = A.q.window > 0 && wpos_lo + 1 > A.q.window ? wpos_lo + 1 - A.q.window : 0;
    const int wbeg_hi = A.q.window > 0 && wpos_hi + 1 > A.q.window ? wpos_hi + 1 - A.q.window : 0;
    kv_i4 qd[D][NC];
    float cs;
    bool qbad;
    {
        float x[NC][16];
        const size_t at = (size_t) (s.row + tok) * A.q.ldq + (size_t) head * HD + 16 * g;
#pragma unroll
        for (int c = 0; c < NC; c++) kv_load16(A.q, at + 64 * c, x[c]);
        const int ex = kv_q_exponent<NC>(x, qbad);
        constexpr int B = D == 3 ? 22 : 30;
        /* a negative scale turns the queries, so that scores grow with their sums */
        const float sign = A.q.scale < 0.0f ? -1.0f : 1.0f;
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int w = 0; w < 4; w++) {
                uint32_t y[4];
#pragma unroll
                for (int e = 0; e < 4; e++) y[e] = (uint32_t) (int) rintf(ldexpf(qbad ? 0.0f : x[c][4 * w + e] * sign, B - ex)) + BIAS;
#pragma unroll
                for (int d = 0; d < D; d++) {
                    const uint32_t b = D - 1 - d, sel = b | (b + 4) << 8 | 0x0c0c0000u;
                    const uint32_t lo2 = __builtin_amdgcn_perm(y[1], y[0], sel), hi2 = __builtin_amdgcn_perm(y[3], y[2], sel);
                    qd[d][c][w] = (int) ((lo2 | hi2 << 16) ^ (d ? 0x80808080u : 0u));
                }
            }
        cs = ldexpf(fabsf(A.q.scale) * kKvLog2e, ex - B);
    }
    /* the value of a product's digit sums: of a score; of a page's output, which
     * with three digits is below 127 * 2^23 */
    auto score = [&](const kv_i4 * a, int e) -> float {
        if constexpr (D == 3) return fmaf((float) (a[0][e] * 256 + a[1][e]), 256.0f, (float) a[2][e]);
        else return fmaf((float) (a[0][e] * 256 + a[1][e]), 65536.0f, (float) (a[2][e] * 256 + a[3][e]));
    };
    auto value = [&](const kv_i4 * a, int e) -> float {
        if constexpr (D == 3) {
            int hi = a[0][e] * 256 + a[1][e];
            asm("" : "+v"(hi));   /* two shifted adds: as one sum it takes three instructions */
            return (float) (hi * 256 + a[2][e]);
        } else {
            return score(a, e);
        }
    };
    float m = -INFINITY, l = 0.0f;
    kv_f4 o[ND];
#pragma unroll
    for (int d = 0; d < ND; d++) o[d] = kv_f4{0.f, 0.f, 0.f, 0.f};
    for (int j = 0; j < n; j++) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   /* this wave's part of page j */
        __syncthreads();                                    /* everyone's, and everyone is done with the other buffer */
        const int k = j & (kKvIds - 1);
        const int id = lid[k];
        const float kscale = lks[k], vscale = lvs[k];
        if (j + 1 < n) {
            if (k == kKvIds - 1) ids(j + 1);
            fetch(j + 1, (j + 1) & 1);
        }
        const int p0 = (first + j) * kKvPage;
        if (!live || id < 0 || p0 > wpos_hi || p0 + kKvPage - 1 < wbeg_lo) continue;   /* uniform in the wave */
        const uint8_t * kp = lbuf + (size_t) (j & 1) * 2 * HALF + 16 * lane;
        const uint8_t * vp = lbuf + (size_t) (j & 1) * 2 * HALF + HALF + (g * HD + 16 * ND * wd + c16) * 16;
        float x[4][4];
        float f = cs * kscale;   /* of the sums; a scale is not negative */
#pragma unroll
        for (int t = 0; t < 4; t++) {
            kv_i4 acc[D];
#pragma unroll
            for (int d = 0; d < D; d++) acc[d] = kv_i4{0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < NC; c++) {
                const kv_i4 kf = *(const kv_i4 *) (kp + c * 4096 + t * 1024);
#pragma unroll
                for (int d = 0; d < D; d++) acc[d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf, qd[d][c], acc[d], 0, 0, 0);
            }
#pragma unroll
            for (int e = 0; e < 4; e++) x[t][e] = score(acc, e);
        }
        if (p0 < wbeg_hi || p0 + kKvPage - 1 > wpos_lo || kscale != kscale) {
            bool any = false;
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int p = p0 + 16 * t + 4 * g + e;
                    const bool seen = p >= beg_c && p <= pos_c;
                    any = any || seen;
                    x[t][e] = seen && kscale == kscale ? x[t][e] * f : -INFINITY;
                }
            f = 1.0f;
            if (any && kscale != kscale) l = kscale;   /* NaN to the end for a column that sees some of it */
        }
        float mp = -INFINITY;
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) mp = fmaxf(mp, x[t][e]);
        mp = kv_rows_max(mp) * f;
        /* a large score times f, not rounded, lies above or below the reference by up to
         * 2^-9 at 2^16, by 1 at 2^25, where four digits no longer hold the weight, and by 128
         * at 2^32, where no f32 does */
        if (__any(fabsf(mp) >= 0x1p16f)) {
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) x[t][e] *= f;
            f = 1.0f;
        }
        if (__any(mp > m + kKvLag)) {
            const float mn = fmaxf(m, mp);
            const float a = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
            l *= a;
#pragma unroll
            for (int d = 0; d < ND; d++) o[d] *= a;
            m = mn;
        }
        const float mref = mp == -INFINITY ? 0.0f : mp;
        kv_i4 P[D];
        float sum = 0.0f;
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                x[t][e] = __builtin_amdgcn_exp2f(fmaf(x[t][e], f, -mref));
                sum += x[t][e];
            }
        /* the integer of a weight of 1, and back: with three digits what makes the
         * page's weights PMAX together */
        float up = PMAX, down = 1.0f / PMAX;
        if constexpr (D == 3) {
            const float all = kv_rows_sum(sum);
            up = all > 0.0f ? PMAX * __builtin_amdgcn_rcpf(all) : 0.0f;
            down *= all;
        }
#pragma unroll
        for (int t = 0; t < 4; t++) {
            uint32_t y[4];
            /* with the digits' bias. Three: 2^23 more leaves the nearest integer in the
             * lower bits of the f32; 2^30 + 0x808080 would not be exact */
#pragma unroll
            for (int e = 0; e < 4; e++)
                y[e] = D == 3 ? __float_as_uint(fmaf(x[t][e], up, 8388608.0f + BIAS)) : (uint32_t) (int) (x[t][e] * up) + BIAS;
#pragma unroll
            for (int d = 0; d < D; d++) {
                const uint32_t b = D - 1 - d, sel = b | (b + 4) << 8 | 0x0c0c0000u;
                const uint32_t lo2 = __builtin_amdgcn_perm(y[1], y[0], sel), hi2 = __builtin_amdgcn_perm(y[3], y[2], sel);
                P[d][t] = (int) ((lo2 | hi2 << 16) ^ (d ? 0x80808080u : 0u));
            }
        }
        const float step = mp == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mp - m);
        l += sum * step;
        const float w = mp == -INFINITY ? 0.0f : step * vscale * down;
        if (vscale == vscale) {
#pragma unroll
            for (int d = 0; d < ND; d++) {
                const kv_i4 vf = *(const kv_i4 *) (vp + d * 256);
                kv_i4 acc[D];
#pragma unroll
                for (int k2 = 0; k2 < D; k2++) acc[k2] = __builtin_amdgcn_mfma_i32_16x16x64_i8(vf, P[k2], kv_i4{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
                for (int e = 0; e < 4; e++) o[d][e] += w * value(acc, e);
            }
        } else if (mp != -INFINITY) {
            l = vscale;
        }
    }
    l = kv_rows_sum(l);
    if (qbad) l = __uint_as_float(0x7fc00000u);
    if (wfirst + c16 >= ncol) return;
    if (A.nsplit == 1) {
#pragma unroll
        for (int d = 0; d < ND; d++) {
            const float v[4] = {o[d][0], o[d][1], o[d][2], o[d][3]};
            kv_write<4>(A.q, s.row + tok, head, HD, 16 * (ND * wd + d) + 4 * g, v, l);
        }
        return;
    }
    const size_t at = (((size_t) tile * kvh + h) * (16 * WQ) + 16 * wq + c16) * A.nsplit + split;
#pragma unroll
    for (int d = 0; d < ND; d++) *(kv_f4 *) (A.po + at * HD + 16 * (ND * wd + d) + 4 * g) = o[d];
    if (wd == 0 && g == 0) {
        A.pml[2 * at] = m;
        A.pml[2 * at + 1] = l;
    }
}

/* Joins the splits of a tile, a wave `each` columns one after another: lane k holds
 * split k's m and l, and eight rows of HD elements are in flight. With four waves
 * a column, as above, a chunk of 512 tokens in four splits took 36 us, not 12: most
 * waves had one row. One column a wave where that gives fewer than eight
 * workgroups a CU (three blocks of 8 tokens: 6.9 us, with four 12.7), else four. */
constexpr int kKvSplits = 64;
constexpr int kKvAlone = 8;   /* pages that take about as long as a join and its launch */
template <int HD>
__global__ __launch_bounds__(256) void kv_tile_join_kernel(const KvTile A, int cols, int each) {
    constexpr int E = HD / 64;
    typedef float fe __attribute__((ext_vector_type(E)));
    __shared__ int lfind[8];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int) threadIdx.x >> 6);
    const int kvh = A.c.kv_heads, G = A.q.heads / kvh;
    const int parts = cols / (4 * each), part = (int) blockIdx.x % parts, th = (int) blockIdx.x / parts, h = th % kvh, tile = th / kvh;
    KvSeq s;
    int place;
    if (!kv_find_tile(A.b, A.c, G, cols, tile, lfind, s, place)) return;
    const int ncol = s.count * G, col0 = place * cols, t0 = col0 / G, t1 = min(col0 + cols - 1, ncol - 1) / G + 1;
    int first;
    const int npages = kv_span(s, t0, t1, A.q.window, first), per = (npages + A.nsplit - 1) / A.nsplit, n = (npages + per - 1) / per;
    for (int u = 0; u < each; u++) {
        const int c = 4 * each * part + each * wave + u, cc = col0 + c;
        if (cc >= ncol) return;
        const size_t row = (((size_t) tile * kvh + h) * cols + c) * A.nsplit;
        float m = -INFINITY, l = 0.0f;
        if (lane < n) {
            m = A.pml[2 * (row + lane)];
            l = A.pml[2 * (row + lane) + 1];
        }
        const float * p = A.po + row * HD + E * lane;
        fe v[8], sum = (fe) 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = *(const fe *) (p + (size_t) min(j, n - 1) * HD);
        float M = m;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
        const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - M);
        float L = m == -INFINITY ? l : f * l;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) L += __shfl_xor(L, o, 64);
        for (int k0 = 0; k0 < n; k0 += 8) {
            if (k0) {
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] = *(const fe *) (p + (size_t) min(k0 + j, n - 1) * HD);
            }
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (k0 + j < n) sum += __int_as_float(__builtin_amdgcn_readlane(__float_as_int(f), k0 + j)) * v[j];
        }
        float o[E];
#pragma unroll
        for (int e = 0; e < E; e++) o[e] = sum[e];
        const int tok = cc / G;
        kv_write<E>(A.q, s.row + tok, h * G + cc - tok * G, HD, E * lane, o, L);
    }
}

/* -------------------------------------------------------------------- host */

struct KvPlan {
    int max_q;                /* the batch's, at most its rows */
    int flat;                 /* the few-column kernel: 1 shares, 2 whole kv heads */
    int groups;               /* its workgroups */
    long tiles;
    int wq, nsplit;           /* the many-column kernel's */
    size_t pre, po, pml, bytes;
};

KvPlan kv_plan(const sparkmv_kv_cache * c, const sparkmv_kv_batch * b, int heads, int window) {
    KvPlan p = {};
    const int G = heads / c->kv_heads;
    p.max_q = b->qstart ? (b->max_q < b->ntok ? b->max_q : b->ntok) : 1;
    const long cols = (long) p.max_q * G, hd = c->head_dim;
    long len = b->max_len > 0 ? b->max_len : (long) c->max_pages * kKvPage;
    const long pages = (len + kKvPage - 1) / kKvPage;
    size_t off = 0;
    auto take = [&](size_t bytes) { const size_t o = off; off += (bytes + 255) & ~(size_t) 255; return o; };
    if (cols <= 4) {
        /* up to kv_whole() pages a sequence: a workgroup each, nothing to join */
        const long in_window = ((long) window + kKvPage - 2) / kKvPage + 1, seen = window > 0 && in_window < pages ? in_window : pages;
        p.flat = seen <= kv_whole((long) b->nseq * c->kv_heads) ? 2 : 1;
        const long most = 2 * cu_count() < kKvFlatMost ? 2 * cu_count() : kKvFlatMost, all = pages * b->nseq * c->kv_heads;
        p.groups = (int) (all < 1 ? 1 : (all < most ? all : most));
        p.pre = take(((size_t) b->nseq + 2) * 4);
        p.po = take((size_t) p.groups * 2 * 4 * hd * 4);
        p.pml = take((size_t) p.groups * 2 * 4 * 2 * 4);
    } else {
        /* columns a workgroup: as a sequence's tokens give (16 sequences at 6000 of 4
         * tokens with 1, 2 and 4, bf16 out: 57, 67 and 90 us, of 8: 79, 62 and 74, of 16: 129,
         * 91 and 77; f32 60, 67, 100, 95, 69, 82, 161, 111, 87), fewer where that leaves half
         * of the CUs idle however it is split (one of 32 tokens at 1000: 19.6, 22.1 and 23.6) */
        const long most = pages <= kKvAlone ? 1 : (pages / 3 < kKvSplits ? pages / 3 : kKvSplits);
        auto busy = [&]() { return ((long) b->ntok * G + 16 * p.wq - 1) / (16 * p.wq) * c->kv_heads; };
        p.wq = cols <= 16 ? 1 : (cols <= 32 ? 2 : 4);
        while (p.wq > 1 && 2 * busy() * most <= cu_count()) p.wq /= 2;
        p.tiles = (long) b->ntok * G / (16 * p.wq) + b->nseq;
        /* as many as two workgroups a CU hold, four pages a split about (three blocks of
         * 8 tokens at 6001, the call: 8 pages 35 us, 4 25.5, 3 27.3, 2 29.5); one if that
         * spares no more pages than the join costs */
        long n = 2 * cu_count() / busy();
        n = n < 1 ? 1 : (n < most ? n : most);
        /* one and a half turns of the CUs in halves are three shorter ones. us in halves and
         * whole, bf16 outputs: three blocks of 512 at 2500 161 and 170, 3000 165 and 182,
         * 6000 279 and 325, 12000 516 and 613; one of 1100 at 2500 143 and 152, 12000 501 and
         * 604; f32 3000 202 and 234. Of fewer pages halves gain less and from about 30 on lose:
         * three at 1700 115 and 120, 1200 104 and 98, 700 89 and 77 */
        if (n == 1 && most > 1 && busy() > cu_count() && 2 * busy() <= 3 * cu_count() && pages >= 48) n = 2;
        p.nsplit = pages - pages / n <= kKvAlone ? 1 : (int) n;
        if (p.nsplit > 1) {
            const size_t rows = (size_t) p.tiles * c->kv_heads * 16 * p.wq * p.nsplit;
            p.po = take(rows * hd * 4);
            p.pml = take(rows * 2 * 4);
        }
    }
    p.bytes = off;
    return p;
}

}  // namespace

}  // namespace sparkmv

using namespace sparkmv;

extern "C" {

size_t sparkmv_kv_attend_work(const sparkmv_kv_cache * cache, const sparkmv_kv_batch * batch, int heads) {
    if (kv_check_cache(cache) || kv_check_batch(batch) || heads < 1 || heads % cache->kv_heads) return 0;
    if (batch->nseq == 0 || batch->ntok == 0) return 0;
    return kv_plan(cache, batch, heads, 0).bytes;
}

int sparkmv_kv_attend(const sparkmv_kv_cache * cache, const sparkmv_kv_batch * batch, const sparkmv_kv_query * query,
                      void * stream) {
    if (kv_check_cache(cache) || kv_check_batch(batch)) return -1;
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
    /* the few-column kernel's count of pages, and where its last shares would end */
    if ((long) batch->nseq * (cache->max_pages + kKvItem) * cache->kv_heads > 0x7fffffffl - kKvFlatMost) {
        set_error("%d sequences of up to %d pages and %d kv heads are too many for one call", batch->nseq, cache->max_pages,
                  cache->kv_heads);
        return -1;
    }
    const KvPlan p = kv_plan(cache, batch, q.heads, q.window);
    if (p.bytes && (!q.work || !kv_aligned(q.work, 256) || q.work_bytes < p.bytes)) {
        set_error("attention needs %zu bytes of 256-byte aligned workspace, not %zu", p.bytes, q.work ? q.work_bytes : 0);
        return -1;
    }
    hipStream_t s = (hipStream_t) stream;
    uint8_t * mem = (uint8_t *) q.work;
    const int hd = cache->head_dim;
    if (p.flat) {
        KvFlat f;
        f.c = *cache; f.b = *batch; f.q = q;
        f.b.max_q = p.max_q;
        f.pre = (int *) (mem + p.pre); f.po = (float *) (mem + p.po); f.pml = (float *) (mem + p.pml);
        const dim3 join((unsigned) batch->nseq, (unsigned) cache->kv_heads, (unsigned) (p.max_q * (q.heads / cache->kv_heads)));
        const uint32_t pre = batch->nseq > 64 ? ((uint32_t) batch->nseq + 1) * 4 : 0;
#define KV_FLAT_N(H, W, GRID, LDS)                                                                                   \
    do {                                                                                                             \
        static LdsAllowed allowed;                                                                                   \
        if (lds_allow(allowed, (const void *) kv_flat_kernel<H, W>, LDS + 1024, "LDS opt-in for the kv attention"))  \
            return -1;                                                                                               \
        hipLaunchKernelGGL((kv_flat_kernel<H, W>), dim3((unsigned) (GRID)), dim3(64 * W), LDS, s, f);                \
    } while (0)
#define KV_FLAT(H)                                                                                                   \
    do {                                                                                                             \
        if (p.flat == 2) {                                                                                           \
            KV_FLAT_N(H, 8, batch->nseq * cache->kv_heads, kv_flat_lds(H, 8));                                       \
        } else {                                                                                                     \
            KV_FLAT_N(H, 4, p.groups, kv_flat_lds(H, 4) + pre);                                                      \
            hipLaunchKernelGGL(kv_flat_join_kernel<H>, join, dim3(512), 0, s, f);                                    \
        }                                                                                                            \
    } while (0)
        if (hd == 64) KV_FLAT(64);
        else if (hd == 128) KV_FLAT(128);
        else KV_FLAT(256);
#undef KV_FLAT
#undef KV_FLAT_N
        return kv_check_launch("kv attention launch");
    }
    KvTile t;
    t.c = *cache; t.b = *batch; t.q = q;
    t.b.max_q = p.max_q;
    t.nsplit = p.nsplit;
    t.po = (float *) (mem + p.po); t.pml = (float *) (mem + p.pml);
    const long th = p.tiles * cache->kv_heads;
    if (th > kKvThreads / 256 / p.nsplit) { set_error("attention over %ld tiles of tokens is too much for one call", th); return -1; }
    const dim3 grid((unsigned) (th * p.nsplit));
    const uint32_t lds = 4 * kKvPage * (uint32_t) hd;
    const int each = th * 4 * p.wq < 8 * cu_count() ? 1 : 4;
#define KV_TILE(H, D, W)                                                                                             \
    do {                                                                                                             \
        static LdsAllowed allowed;                                                                                   \
        if (lds_allow(allowed, (const void *) kv_tile_kernel<H, D, W>, lds + 4096, "LDS opt-in for the kv attention")) \
            return -1;                                                                                               \
        hipLaunchKernelGGL((kv_tile_kernel<H, D, W>), grid, dim3(256), lds, s, t);                                   \
    } while (0)
#define KV_TILE_D(H, W)                                                                                              \
    do {                                                                                                             \
        if (q.out_dtype == SPARKMV_X_F32) KV_TILE(H, 4, W);                                                          \
        else KV_TILE(H, 3, W);                                                                                       \
    } while (0)
#define KV_TILE_W(H)                                                                                                 \
    do {                                                                                                             \
        if (p.wq == 1) KV_TILE_D(H, 1);                                                                              \
        else if (p.wq == 2) KV_TILE_D(H, 2);                                                                         \
        else KV_TILE_D(H, 4);                                                                                        \
        if (p.nsplit > 1)                                                                                            \
            hipLaunchKernelGGL(kv_tile_join_kernel<H>, dim3((unsigned) (th * 4 * p.wq / each)), dim3(256), 0, s, t, 16 * p.wq, each); \
    } while (0)
    if (hd == 64) KV_TILE_W(64);
    else if (hd == 128) KV_TILE_W(128);
    else KV_TILE_W(256);
#undef KV_TILE_W
#undef KV_TILE_D
#undef KV_TILE
    return kv_check_launch("kv attention launch");
}

}  // extern "C"
