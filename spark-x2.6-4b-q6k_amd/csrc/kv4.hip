/* kv4.hip — the paged 4-bit cache: the append with the heads' norm and rotation on
 * the way, and reading positions back (include/sparkmv.h has the cache's rules,
 * kv4.h its layout, kv4_attend.hip attention over it). */
#include "kv4.h"

#include <math.h>

#include "heads.h"

namespace sparkmv {

namespace {

/* -------------------------------------------------------------------- append
 * A wave takes 64 / lanes heads at a time, a workgroup up to 4 * U such groups of one
 * token: queries, keys and values. C and S (heads.h) are worked out once a workgroup.
 * Bound by the chain of batch, position, table row, LDS, turn and code: 4.0 us for a
 * token, 9.0 for 512 of 24 bf16 heads of 256, 11 MB.
 * Positions share nothing, so that no page is read and a token's codes do not
 * depend on what was there. Keys are rounded once to f32 after norm and rotation
 * (heads.h, 64 bits), and the rest is exact: the scale is a power of two from the
 * largest element's bits, and the conversion rounds to the nearest of the eight
 * magnitudes, ties to the even code. */
struct Kv4Append {
    sparkmv_kv4_cache c;
    sparkmv_kv_batch b;
    sparkmv_kv4_new n;
    double inv_hd;
    int vec;                       /* halves are whole pieces of a lane */
    int sh;                        /* lanes of a head, as a shift */
    int qgroups, kgroups, groups;  /* groups of a token's queries, of its keys (and of its values), of the token */
    int parts;                     /* workgroups of a token */
};

/* the token in row tok: its slot and position; false if it is of no sequence */
__device__ __forceinline__ bool kv4_find_row(const Kv4Append & A, int tok, int lane, int & slot, int & pos) {
    if (!A.b.qstart) {
        if (tok >= A.b.nseq) return false;
        const KvSeq s = kv_seq(A.b, tok, A.c.nslots, A.c.max_pages);
        slot = s.slot;
        pos = s.pos;
        return s.count > 0;
    }
    for (int i0 = 0; i0 < A.b.nseq; i0 += 64) {
        KvSeq s = {0, 0, 0, 0};
        if (i0 + lane < A.b.nseq) s = kv_seq(A.b, i0 + lane, A.c.nslots, A.c.max_pages);
        const bool mine = s.count > 0 && tok >= s.row && tok < s.row + s.count;
        const uint64_t who = __ballot(mine);
        if (who) {
            const int w = __builtin_ctzll(who);
            slot = __builtin_amdgcn_readlane(s.slot, w);
            pos = __builtin_amdgcn_readlane(s.pos, w) + tok - __builtin_amdgcn_readlane(s.row, w);
            return true;
        }
    }
    return false;
}

template <int CTRL>
__device__ __forceinline__ uint32_t kv4_dpp(uint32_t v) {
    return (uint32_t) __builtin_amdgcn_mov_dpp((int) v, CTRL, 0xf, 0xf, true);
}

/* four elements a lane, eight lanes a block: the codes (16 bits a lane) and the scale */
__device__ __forceinline__ uint32_t kv4_code(const float * x, uint32_t & byte) {
    uint32_t big = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) big = max(big, __float_as_uint(x[i]) & 0x7fffffffu);
    big = max(big, kv4_dpp<0xb1>(big));    /* lane ^ 1 */
    big = max(big, kv4_dpp<0x4e>(big));    /* lane ^ 2 */
    big = max(big, kv4_dpp<0x141>(big));   /* lane 7 - i of eight */
    /* the smallest e with big <= 7 * 2^e: one more where the leading bits exceed 1.75 */
    const bool bad = big >= 0x7f800000u;
    byte = bad ? 255u : (uint32_t) min(max((int) ((big + 0x1fffffu) >> 23) - 2, kKv4Low), kKv4High);
    if (bad) return 0;
    const float s = __uint_as_float(byte << 23);
    uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x[0], x[1], s, 0);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], s, 1) & 0xffffu;
}

template <typename X, int U>
__global__ __launch_bounds__(256) void kv4_append_kernel(const Kv4Append A) {
    typedef typename HeadArith<X>::T T;
    __shared__ T qc[kHeadMax], qs[kHeadMax];
    __shared__ double kc[kHeadMax], ks[kHeadMax];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int tok = (int) blockIdx.x / A.parts, g0 = ((int) blockIdx.x - tok * A.parts) * 4 + wave;
    const int l = lane & ((1 << A.sh) - 1), e0 = 4 * l, per = 64 >> A.sh;
    const int hd = A.c.head_dim, kvh = A.c.kv_heads, inter = A.n.turn.interleaved, half = A.n.turn.rope_dim / 2;
    HeadRaw<X, 4> x[U];
    const X * at[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        int g = g0 + 4 * u * A.parts;
        if (g >= A.groups) continue;
        const int which = g < A.qgroups ? 0 : (g < A.qgroups + A.kgroups ? 1 : 2);   /* queries, keys, values */
        g -= which == 0 ? 0 : (which == 1 ? A.qgroups : A.qgroups + A.kgroups);
        const int h = min(g * per + (lane >> A.sh), (which ? kvh : A.n.heads) - 1);
        at[u] = (const X *) (which == 0 ? A.n.q : (which == 1 ? A.n.k : A.n.v)) +
                (size_t) tok * (which == 0 ? A.n.ldq : (which == 1 ? A.n.ldk : A.n.ldv)) + (size_t) h * hd;
        head_load<4>(at[u] + e0, x[u]);
    }
    int slot, pos;
    if (!kv4_find_row(A, tok, lane, slot, pos)) return;
    const int page = A.c.pages[(size_t) slot * A.c.max_pages + pos / kKvPage], p = pos & (kKvPage - 1);
    if (tid < hd) {
        const HeadFactor k = head_factor(tid, half, inter, A.n.turn.k_norm);
        float c = 1.0f, s = 0.0f;
        if (k.at >= 0) {
            const float * row = A.n.turn.rope + (size_t) pos * A.n.turn.rope_dim + k.at;
            c = row[0];
            s = row[half];
        }
        head_coef(k, c, s, kc[tid], ks[tid]);
        if (A.qgroups) head_coef(head_factor(tid, half, inter, A.n.turn.q_norm), c, s, qc[tid], qs[tid]);
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; u++) {
        int g = g0 + 4 * u * A.parts;
        if (g >= A.groups) return;
        const int which = g < A.qgroups ? 0 : (g < A.qgroups + A.kgroups ? 1 : 2);
        g -= which == 0 ? 0 : (which == 1 ? A.qgroups : A.qgroups + A.kgroups);
        const int h = g * per + (lane >> A.sh);
        const bool on = h < (which ? kvh : A.n.heads);
        float a[4], b[4];
        head_wide<4>(x[u], at[u], e0, hd, which == 2 ? 0 : half, inter, A.vec, a, b);
        if (which == 0) {
            T C[4], S[4], o[4];
#pragma unroll
            for (int i = 0; i < 4; i++) { C[i] = qc[e0 + i]; S[i] = qs[e0 + i]; }
            const double r = head_norm<4, T>(a, A.n.turn.q_norm != nullptr, A.n.turn.eps, A.inv_hd, A.sh);
            head_turn<4>(C, S, a, b, r, o);
            if (on) head_store<4>((X *) A.n.q_out + (size_t) tok * A.n.ldqo + (size_t) h * hd + e0, o);
            continue;
        }
        if (which == 1) {
            double C[4], S[4], o[4];
#pragma unroll
            for (int i = 0; i < 4; i++) { C[i] = kc[e0 + i]; S[i] = ks[e0 + i]; }
            const double r = head_norm<4, double>(a, A.n.turn.k_norm != nullptr, A.n.turn.eps, A.inv_hd, A.sh);
            head_turn<4>(C, S, a, b, r, o);
#pragma unroll
            for (int i = 0; i < 4; i++) a[i] = (float) o[i];
        }
        uint32_t byte;
        const uint32_t code = kv4_code(a, byte);
        if (!on || page < 0 || page >= A.c.npages) continue;
        uint8_t * to = A.c.data + ((size_t) page * kvh + h) * (size_t) kv4_head_bytes(hd);
        *(uint16_t *) (to + (which == 1 ? kv4_key_at(p, e0, hd) : kv4_value_at(p, e0, hd))) = (uint16_t) code;
        if ((l & 7) == 0) to[which == 1 ? kv4_key_scale_at(p, e0, hd) : kv4_value_scale_at(p, e0, hd)] = (uint8_t) byte;
    }
}

/* ---------------------------------------------------------------------- read
 * One workgroup per (sequence, page its positions touch, kv head, keys or values),
 * eight elements a thread at a time. Bound by latency: 64 single pages all over the pool
 * 9.8 us, 512 positions of one sequence in bf16 5.8. */
__device__ __forceinline__ void kv4_store8(uint16_t * to, const uint32_t * v) { *(uint4 *) to = uint4{v[0], v[1], v[2], v[3]}; }
__device__ __forceinline__ void kv4_store8(float * to, const uint32_t * v) {
#pragma unroll
    for (int k = 0; k < 2; k++)
        *(float4 *) (to + 4 * k) = float4{__uint_as_float(v[2 * k] << 16), __uint_as_float(v[2 * k] & 0xffff0000u),
                                          __uint_as_float(v[2 * k + 1] << 16), __uint_as_float(v[2 * k + 1] & 0xffff0000u)};
}

template <typename X>
__global__ __launch_bounds__(256) void kv4_read_kernel(const sparkmv_kv4_cache c, const int * slots, const int * from, int n,
                                                       int nb, X * ko, X * vo) {
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
    const uint8_t * data = c.data + (have ? (size_t) page * kvh + h : 0) * (size_t) kv4_head_bytes(hd);
    out += ((size_t) i * n * kvh + h) * hd;
    const int sh = 31 - __clz(hd / 8), cnt = (int) (hi - lo) << sh, r0 = (int) (lo - p0);
    for (int k0 = 0; k0 < cnt; k0 += 1024) {
        uint32_t code[4], byte[4];
#pragma unroll
        for (int w = 0; w < 4; w++) {
            code[w] = byte[w] = 0;
            const int k = k0 + tid + 256 * w, p = r0 + (k >> sh), d = 8 * (k & ((1 << sh) - 1));
            if (k >= cnt || !have) continue;
            if (which && hd == 64)
                code[w] = *(const uint16_t *) (data + kv4_value_at(p, d, hd)) | (uint32_t) *(const uint16_t *) (data + kv4_value_at(p, d + 4, hd)) << 16;
            else
                code[w] = *(const uint32_t *) (data + (which ? kv4_value_at(p, d, hd) : kv4_key_at(p, d, hd)));
            byte[w] = data[which ? kv4_value_scale_at(p, d, hd) : kv4_key_scale_at(p, d, hd)];
        }
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const int k = k0 + tid + 256 * w, p = r0 + (k >> sh), d = 8 * (k & ((1 << sh) - 1));
            if (k >= cnt) continue;
            const float s = __uint_as_float((byte[w] > kKv4High ? 255u : byte[w]) << 23);
            const uint32_t v[4] = {kv4_pair<0>(code[w], s), kv4_pair<1>(code[w], s), kv4_pair<2>(code[w], s), kv4_pair<3>(code[w], s)};
            kv4_store8(out + (size_t) (p0 + p - f) * kvh * hd + d, v);
        }
    }
}

}  // namespace

int kv4_check_cache(const sparkmv_kv4_cache * c) {
    if (!c) { set_error("kv4 cache is null"); return -1; }
    if (c->kv_heads < 1 || c->kv_heads > 1024) { set_error("kv_heads %d is outside 1..1024", c->kv_heads); return -1; }
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) {
        set_error("head_dim %d is not 64, 128 or 256", c->head_dim);
        return -1;
    }
    if (c->npages < 1 || c->nslots < 1 || c->max_pages < 1) {
        set_error("kv4 cache of %d pages, %d slots of %d pages", c->npages, c->nslots, c->max_pages);
        return -1;
    }
    if (c->max_pages > (1 << 24)) { set_error("max_pages %d is above %d", c->max_pages, 1 << 24); return -1; }
    if (!c->data || !c->pages) { set_error("kv4 cache has a null array"); return -1; }
    if (!kv_aligned(c->data, 16)) { set_error("kv4 cache data is not 16-byte aligned"); return -1; }
    return 0;
}

}  // namespace sparkmv

using namespace sparkmv;

extern "C" {

size_t sparkmv_kv4_bytes(int kv_heads, int head_dim, int npages) {
    if (kv_heads < 1 || head_dim < 1 || npages < 1) return 0;
    return (size_t) npages * kv_heads * kv4_head_bytes(head_dim);
}

int sparkmv_kv4_append(const sparkmv_kv4_cache * cache, const sparkmv_kv_batch * batch, const sparkmv_kv4_new * rows,
                       void * stream) {
    if (kv4_check_cache(cache) || kv_check_batch(batch)) return -1;
    if (!rows) { set_error("kv rows are null"); return -1; }
    const sparkmv_kv4_new & n = *rows;
    const int hd = cache->head_dim;
    if (kv_check_dtype("kv rows", n.x_dtype)) return -1;
    /* an array of no rows may be null */
    const bool any = batch->nseq > 0 && batch->ntok > 0;
    if (n.heads < 0 || (any && ((n.heads > 0) != (n.q != nullptr) || (n.heads > 0) != (n.q_out != nullptr)))) {
        set_error("%d query heads, queries and their output do not agree", n.heads);
        return -1;
    }
    if (n.heads > 65536) { set_error("%d query heads are above 65536", n.heads); return -1; }
    if (check_turn("kv4 append", &n.turn, hd, (long) cache->max_pages * kKvPage)) return -1;
    if (batch->nseq == 0 || batch->ntok == 0) return 0;
    if (n.heads && n.q == n.q_out && n.ldq != n.ldqo && batch->ntok > 1) {
        set_error("queries turned in place with two row strides, %d and %d", n.ldq, n.ldqo);
        return -1;
    }
    const long kvd = (long) cache->kv_heads * hd, qd = (long) n.heads * hd;
    if (kv_check_rows("keys", n.k, n.ldk, kvd, n.x_dtype, batch->ntok) ||
        kv_check_rows("values", n.v, n.ldv, kvd, n.x_dtype, batch->ntok))
        return -1;
    if (n.heads && (kv_check_rows("queries", n.q, n.ldq, qd, n.x_dtype, batch->ntok) ||
                    kv_check_rows("turned queries", n.q_out, n.ldqo, qd, n.x_dtype, batch->ntok)))
        return -1;
    Kv4Append a;
    a.c = *cache; a.b = *batch; a.n = n;
    a.b.max_q = batch->qstart ? batch->max_q : 1;
    a.vec = n.turn.rope_dim / 2 % 4 == 0;
    a.inv_hd = 1.0 / hd;
    a.sh = head_lane_shift(hd, 4);
    const int per = 64 >> a.sh;
    a.qgroups = (n.heads + per - 1) / per;
    a.kgroups = (cache->kv_heads + per - 1) / per;
    a.groups = a.qgroups + 2 * a.kgroups;
    auto parts = [&](int u) { return (a.groups + 4 * u - 1) / (4 * u); };
    /* one group a wave, or up to four: with 24 f32 heads of 256, read back included, 64
     * tokens of 64 sequences 13.8 and 15.0 us, 512 of one 16.5 and 15.3, 4096 76 and 64 */
    const int u = (long) batch->ntok * parts(4) >= 4 * cu_count() ? 4 : 1;
    a.parts = parts(u);
    const long wg = (long) batch->ntok * a.parts;
    if (wg > kKvThreads / 256) { set_error("an append of %ld workgroups is too much for one call", wg); return -1; }
    const dim3 grid((unsigned) wg), block(256);
    hipStream_t s = (hipStream_t) stream;
    if (n.x_dtype == SPARKMV_X_F32) {
        if (u == 4) hipLaunchKernelGGL((kv4_append_kernel<float, 4>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((kv4_append_kernel<float, 1>), grid, block, 0, s, a);
    } else {
        if (u == 4) hipLaunchKernelGGL((kv4_append_kernel<uint16_t, 4>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((kv4_append_kernel<uint16_t, 1>), grid, block, 0, s, a);
    }
    return kv_check_launch("kv4 append launch");
}

int sparkmv_kv4_read(const sparkmv_kv4_cache * cache, int nseq, const int * slot, const int * from, int n, void * k_out,
                     void * v_out, int out_dtype, void * stream) {
    if (kv4_check_cache(cache) || kv_check_dtype("kv4 read", out_dtype)) return -1;
    if (nseq < 0 || nseq > kKvMaxSeq) { set_error("%d sequences are outside 0..%d", nseq, kKvMaxSeq); return -1; }
    if (n < 0) { set_error("%d positions", n); return -1; }
    if (nseq == 0 || n == 0 || (!k_out && !v_out)) return 0;
    if (!from) { set_error("kv4 read has no positions"); return -1; }
    if (!kv_aligned(k_out, 16) || !kv_aligned(v_out, 16)) { set_error("kv4 read: rows do not start 16-byte aligned"); return -1; }
    const long nb = ((long) n + kKvPage - 2) / kKvPage + 1, wgs = (long) nseq * nb;
    if (wgs > kKvThreads / 256) { set_error("a read of %ld pages is too much for one call", wgs); return -1; }
    const dim3 grid((unsigned) wgs, (unsigned) cache->kv_heads, 2), block(256);
    hipStream_t s = (hipStream_t) stream;
    if (out_dtype == SPARKMV_X_F32)
        hipLaunchKernelGGL(kv4_read_kernel<float>, grid, block, 0, s, *cache, slot, from, n, (int) nb, (float *) k_out,
                           (float *) v_out);
    else
        hipLaunchKernelGGL(kv4_read_kernel<uint16_t>, grid, block, 0, s, *cache, slot, from, n, (int) nb,
                           (uint16_t *) k_out, (uint16_t *) v_out);
    return kv_check_launch("kv4 read launch");
}

}  // extern "C"
