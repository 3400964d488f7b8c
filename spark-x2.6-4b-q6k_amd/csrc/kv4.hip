/* kv4.hip — the paged 4-bit cache: the append with the heads' norm and rotation on
 * the way, and reading positions back (include/sparkmv.h has the cache's rules,
 * kv4.h its layout, kv4_attend.hip attention over it). */
#include "kv4.h"

#include <math.h>

#include "heads.h"

namespace sparkmv {

namespace {

/* -------------------------------------------------------------------- append
 * A wave takes up to U * (64 / lanes) heads of one token: queries, keys or values.
 * Positions share nothing, so that no page is read and a token's codes do not
 * depend on what was there. Keys are rounded once to f32 after norm and rotation
 * (heads.h, 64 bits), and the rest is exact: the scale is a power of two from the
 * largest element's bits, and the conversion rounds to the nearest of the eight
 * magnitudes, ties to the even code. */
struct Kv4Append {
    sparkmv_kv4_cache c;
    sparkmv_kv_batch b;
    sparkmv_kv4_new n;
    HeadVec vec;
    double inv_hd;
    int sh;                       /* lanes of a head, as a shift */
    int qparts, kparts, parts;    /* waves of a token's queries, of its keys (and of its values), of the token */
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
    const long w = ((long) blockIdx.x * 256 + threadIdx.x) >> 6;
    const int tok = __builtin_amdgcn_readfirstlane((int) (w / A.parts));
    if (tok >= A.b.ntok) return;
    const int lane = threadIdx.x & 63, l = lane & ((1 << A.sh) - 1), e0 = 4 * l, per = 64 >> A.sh;
    int part = __builtin_amdgcn_readfirstlane((int) (w - (long) tok * A.parts));
    const int which = part < A.qparts ? 0 : (part < A.qparts + A.kparts ? 1 : 2);   /* queries, keys, values */
    part -= which == 0 ? 0 : (which == 1 ? A.qparts : A.qparts + A.kparts);
    const int hd = A.c.head_dim, kvh = A.c.kv_heads, inter = A.n.turn.interleaved;
    const int half = which == 2 ? 0 : A.n.turn.rope_dim / 2, nh = which ? kvh : A.n.heads;
    const X * in = (const X *) (which == 0 ? A.n.q : (which == 1 ? A.n.k : A.n.v)) +
                   (size_t) tok * (which == 0 ? A.n.ldq : (which == 1 ? A.n.ldk : A.n.ldv));
    const float * weight = which == 0 ? A.n.turn.q_norm : (which == 1 ? A.n.turn.k_norm : nullptr);
    const int h0 = part * U * per + (lane >> A.sh);
    float x[U][4], y[U][4];
#pragma unroll
    for (int u = 0; u < U; u++) head_fetch<4>(in + (size_t) min(h0 + u * per, nh - 1) * hd, e0, hd, half, inter, A.vec, x[u], y[u]);
    int slot, pos;
    if (!kv4_find_row(A, tok, lane, slot, pos)) return;
    const float * row = half ? A.n.turn.rope + (size_t) pos * A.n.turn.rope_dim : nullptr;
    if (which == 0) {
        typedef typename HeadArith<X>::T T;
        T C[4], S[4];
        head_coef<4>(C, S, e0, hd, row, half, inter, weight, A.vec);
#pragma unroll
        for (int u = 0; u < U; u++) {
            T o[4];
            const double r = head_norm<4>(x[u], weight != nullptr, A.n.turn.eps, A.inv_hd, A.sh);
            head_turn<4>(C, S, x[u], y[u], r, o);
            if (h0 + u * per < nh) head_store<4>((X *) A.n.q_out + (size_t) tok * A.n.ldqo + (size_t) (h0 + u * per) * hd + e0, o);
        }
        return;
    }
    const int page = A.c.pages[(size_t) slot * A.c.max_pages + pos / kKvPage], p = pos & (kKvPage - 1);
    if (page < 0 || page >= A.c.npages) return;
    const int code_at = which == 1 ? kv4_key_at(p, e0, hd) : kv4_value_at(p, e0, hd);
    const int scale_at = which == 1 ? kv4_key_scale_at(p, e0, hd) : kv4_value_scale_at(p, e0, hd);
    double C[4], S[4];
    if (which == 1) head_coef<4>(C, S, e0, hd, row, half, inter, weight, A.vec);
#pragma unroll
    for (int u = 0; u < U; u++) {
        if (which == 1) {
            double o[4];
            const double r = head_norm<4>(x[u], weight != nullptr, A.n.turn.eps, A.inv_hd, A.sh);
            head_turn<4>(C, S, x[u], y[u], r, o);
#pragma unroll
            for (int i = 0; i < 4; i++) x[u][i] = (float) o[i];
        }
        uint32_t byte;
        const uint32_t code = kv4_code(x[u], byte);
        const int head = h0 + u * per;
        if (head >= nh) continue;
        uint8_t * to = A.c.data + ((size_t) page * kvh + head) * (size_t) kv4_head_bytes(hd);
        *(uint16_t *) (to + code_at) = (uint16_t) code;
        if ((l & 7) == 0) to[scale_at] = (uint8_t) byte;
    }
}

/* ---------------------------------------------------------------------- read
 * One workgroup per (sequence, page its positions touch, kv head, keys or values),
 * eight elements a thread at a time. */
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
    if (n.heads < 0 || (n.heads > 0) != (n.q != nullptr) || (n.heads > 0) != (n.q_out != nullptr)) {
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
    a.vec = head_vec(n.turn, 4);
    a.inv_hd = 1.0 / hd;
    a.sh = head_lane_shift(hd, 4);
    const int per = 64 >> a.sh;
    auto waves = [&](int heads, int u) { return (heads + u * per - 1) / (u * per); };
    const long all = (long) batch->ntok * (waves(n.heads, 1) + 2 * waves(cache->kv_heads, 1));
    const int u = all > 16 * cu_count() ? 4 : 1;
    a.qparts = waves(n.heads, u);
    a.kparts = waves(cache->kv_heads, u);
    a.parts = a.qparts + 2 * a.kparts;
    const long wg = ((long) batch->ntok * a.parts + 3) / 4;
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
