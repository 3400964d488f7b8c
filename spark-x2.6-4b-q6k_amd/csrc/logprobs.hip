/* logprobs.hip — log probabilities of given tokens, a row's entropy and its
 * largest logits (include/sparkmv.h).
 *
 * With M a row's largest logit, z = sum e^(x - M) and e = sum (x - M) e^(x - M):
 *   log p(t) = x_t - M - log z,   entropy = log z - e / z.
 * Both sums add up over parts of a row, each taken against its own largest.
 *
 * The row is read once. The first launch streams it, a workgroup a part: the
 * part's (M, z, e), and the largest logit of every 32 neighbours. The k largest
 * logits lie in the k segments whose largest is largest (equal ones: the
 * earlier segment), so the second launch, a workgroup a row, finds those among
 * n / 32 values, reads them again, 32 k logits, and ranks what can count. */
#include <hip/hip_runtime.h>
#include <math.h>

#include "../../include/sparkmv.h"
#include "common.h"

namespace sparkmv {

namespace {

constexpr int kLpMaxK = 32;
constexpr int kLpSeg = 32;            /* logits of a segment */
constexpr int kLpMaxN = 1 << 19;      /* logits of a row: what the second launch's lists are sized for */
constexpr float kLpLog2e = 1.44269504088896340736f;

typedef float lp_f4 __attribute__((ext_vector_type(4)));
typedef uint32_t lp_u4 __attribute__((ext_vector_type(4)));

struct LpArgs {
    const void * x;
    int n, k, nparts, nseg;
    size_t ld;
    const int * tokens;
    float * logprob, * entropy, * top_lp;
    int * top_id;
    lp_f4 * parts;       /* [rows][nparts]: M, z, e */
    float * seg;         /* [rows][nseg]: largest of 32, NaN for none */
};

__device__ __forceinline__ float lp_one(const float * p) { return *p; }
__device__ __forceinline__ float lp_one(const uint16_t * p) { return __uint_as_float((uint32_t) *p << 16); }

/* V neighbours, 16 bytes aligned where V > 1 */
template <int V>
__device__ __forceinline__ void lp_load(const float * p, float * v) {
    if constexpr (V == 4) {
        const lp_f4 w = *(const lp_f4 *) p;
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = w[i];
    } else {
        v[0] = *p;
    }
}
template <int V>
__device__ __forceinline__ void lp_load(const uint16_t * p, float * v) {
    if constexpr (V == 8) {
        const lp_u4 w = *(const lp_u4 *) p;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    } else {
        v[0] = lp_one(p);
    }
}

template <int CTRL>
__device__ __forceinline__ float lp_dpp(float v) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true));
}
/* the largest of L neighbouring lanes, in each; NaN only if all are */
template <int L>
__device__ __forceinline__ float lp_group_max(float v) {
    v = fmaxf(v, lp_dpp<0xb1>(v));                          /* lane ^ 1 */
    v = fmaxf(v, lp_dpp<0x4e>(v));                          /* lane ^ 2 */
    if constexpr (L >= 8) v = fmaxf(v, lp_dpp<0x141>(v));   /* 7 - lane of eight */
    if constexpr (L >= 16) v = fmaxf(v, lp_dpp<0x140>(v));  /* 15 - lane of sixteen */
    if constexpr (L >= 32) v = fmaxf(v, __shfl_xor(v, 16, 64));
    return v;
}

/* NL loads of 64 * V logits a wave; four waves a part. Bound by the read: 512 rows
 * of 131072 f32 51 us, 5.2 TB/s. */
template <typename X, int V, int NL>
__global__ __launch_bounds__(256) void lp_stream_kernel(const LpArgs A) {
    constexpr int L = kLpSeg / V, PER = 64 * V * NL;
    __shared__ float red[3][4];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, r = blockIdx.y;
    const int base = ((int) blockIdx.x * 4 + wave) * PER;
    const X * row = (const X *) A.x + (size_t) r * A.ld;
    float v[NL][V];
    float m = -INFINITY;
    const bool full = base + PER <= A.n;   /* uniform in the wave */
    if (full) {
#pragma unroll
        for (int j = 0; j < NL; j++) lp_load<V>(row + base + (j * 64 + lane) * V, v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < NL; j++)
#pragma unroll
            for (int i = 0; i < V; i++) {
                const int at = base + (j * 64 + lane) * V + i;
                v[j][i] = at < A.n ? lp_one(row + at) : NAN;
            }
    }
    if (A.k) {
        float * seg = A.seg + (size_t) r * A.nseg;
#pragma unroll
        for (int j = 0; j < NL; j++) {
            float s = v[j][0];
#pragma unroll
            for (int i = 1; i < V; i++) s = fmaxf(s, v[j][i]);
            s = lp_group_max<L>(s);
            m = fmaxf(m, s);
            const int at = (base + j * 64 * V) / kLpSeg + lane / L;
            if (lane % L == 0 && at < A.nseg) seg[at] = s;
        }
    } else {
#pragma unroll
        for (int j = 0; j < NL; j++)
#pragma unroll
            for (int i = 0; i < V; i++) m = fmaxf(m, v[j][i]);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    /* a NaN anywhere, or a +inf, ends up in z; -inf adds nothing. Where nothing
     * is above -inf, z is 0 or, for a NaN, NaN */
    float z = 0.0f, e = 0.0f;
    const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int j = 0; j < NL; j++)
#pragma unroll
        for (int i = 0; i < V; i++) {
            if (!full && base + (j * 64 + lane) * V + i >= A.n) continue;
            const float d = v[j][i] - ref, p = __builtin_amdgcn_exp2f(d * kLpLog2e);
            z += p;
            e = fmaf(p, fmaxf(d, -3.0e38f), e);
        }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        z += __shfl_xor(z, o, 64);
        e += __shfl_xor(e, o, 64);
    }
    if (lane == 0) {
        red[0][wave] = m;
        red[1][wave] = z;
        red[2][wave] = e;
    }
    __syncthreads();
    if (tid == 0) {
        float M = -INFINITY, Z = 0.0f, E = 0.0f;
        for (int w = 0; w < 4; w++) M = fmaxf(M, red[0][w]);
        for (int w = 0; w < 4; w++) {
            const float d = red[0][w] == -INFINITY ? 0.0f : fmaxf(red[0][w] - M, -1.0e30f), f = red[0][w] == -INFINITY ? 1.0f : expf(d);
            Z += f * red[1][w];
            E += f * fmaf(red[1][w], d, red[2][w]);
        }
        lp_f4 out = {M, Z, E, 0.0f};
        A.parts[(size_t) r * A.nparts + blockIdx.x] = out;
    }
}

/* A logit and its place as one number that grows with the logit and, of equal
 * ones, with the lower place; 0 for a NaN. -0 counts as 0. */
__device__ __forceinline__ uint64_t lp_key(float x, int i) {
    if (x != x) return 0;
    const uint32_t u = __float_as_uint(x + 0.0f);
    const uint32_t o = u & 0x80000000u ? ~u : u | 0x80000000u;
    return (uint64_t) o << 32 | (uint32_t) ~i;
}
__device__ __forceinline__ float lp_value(uint64_t key) {
    const uint32_t o = (uint32_t) (key >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ int lp_place(uint64_t key) { return (int) ~(uint32_t) key; }

/* how many of the n keys are larger; zeros follow the list up to a multiple of
 * kLpPad, whose reads are in flight together (the join of one row of 131072:
 * 10.4 us with one read at a time, 8.7 so, 7.6 with waves ranking first) */
constexpr int kLpPad = 16;
__device__ __forceinline__ int lp_rank(const uint64_t * keys, int n, uint64_t mine) {
    typedef uint64_t u2 __attribute__((ext_vector_type(2)));
    int c = 0;
#pragma unroll 1
    for (int i = 0; i < n; i += kLpPad) {
        u2 v[kLpPad / 2];
#pragma unroll
        for (int j = 0; j < kLpPad / 2; j++) v[j] = *(const u2 *) (keys + i + 2 * j);
#pragma unroll
        for (int j = 0; j < kLpPad / 2; j++) c += (v[j][0] > mine) + (v[j][1] > mine);
    }
    return c;
}

constexpr int kLpList = kLpMaxK * (kLpMaxN / kLpSeg / 256);   /* segments of k threads */

/* segments a thread keeps in registers: rows of up to 163840 logits are not read again */
constexpr int kLpHeld = 20;

/* Bound by its chain, two reads and three rankings: one row of 131072 with 8
 * alternatives 7.7 us, 512 rows with 20 13.2. */
template <typename X>
__global__ __launch_bounds__(256) void lp_join_kernel(const LpArgs A) {
    __shared__ __attribute__((aligned(16))) uint64_t lkey[256];
    __shared__ __attribute__((aligned(16))) uint64_t lseg[kLpList + kLpPad];
    __shared__ uint64_t lpick[kLpMaxK], lleast;
    __shared__ float red[3][4];
    __shared__ __attribute__((aligned(16))) uint64_t lcand[4 * kLpMaxK + kLpPad];
    __shared__ int count[3];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = blockIdx.x, k = A.k;
    const X * row = (const X *) A.x + (size_t) r * A.ld;
    if (tid < 3) count[tid] = 0;
    if (tid < 4 * kLpMaxK + kLpPad) lcand[tid] = 0;
    const int tok = A.tokens ? A.tokens[r] : -1;
    const float given = tok >= 0 && tok < A.n ? lp_one(row + tok) : 0.0f;
    /* this thread's segments, requested before anything is waited for */
    const float * seg = A.seg + (size_t) r * A.nseg;
    const int nseg = k ? A.nseg : 0;
    float held[kLpHeld];
#pragma unroll
    for (int j = 0; j < kLpHeld; j++) held[j] = tid + 256 * j < nseg ? seg[tid + 256 * j] : NAN;
    /* the row's M, z and e */
    float M = -INFINITY, z = 0.0f, e = 0.0f;
    const lp_f4 * parts = A.parts + (size_t) r * A.nparts;
#pragma unroll 1
    for (int i = tid; i < A.nparts; i += 256) M = fmaxf(M, parts[i][0]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
    if (lane == 0) red[0][wave] = M;
    uint64_t best = 0;
#pragma unroll
    for (int j = 0; j < kLpHeld; j++) {
        const uint64_t key = lp_key(held[j], tid + 256 * j);
        best = key > best ? key : best;
    }
#pragma unroll 1
    for (int i = tid + 256 * kLpHeld; i < nseg; i += 256) {
        const uint64_t key = lp_key(seg[i], i);
        best = key > best ? key : best;
    }
    if (tid == 0) lleast = 1;
    lkey[tid] = best;
    __syncthreads();
    M = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
#pragma unroll 1
    for (int i = tid; i < A.nparts; i += 256) {
        const lp_f4 p = parts[i];
        const float d = p[0] == -INFINITY ? 0.0f : fmaxf(p[0] - M, -1.0e30f), f = p[0] == -INFINITY ? 1.0f : expf(d);
        z += f * p[1];
        e += f * fmaf(p[1], d, p[2]);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        z += __shfl_xor(z, o, 64);
        e += __shfl_xor(e, o, 64);
    }
    if (lane == 0) {
        red[1][wave] = z;
        red[2][wave] = e;
    }
    /* the k best segments are among those of the k threads whose best is best,
     * and none of them is below the last of these threads' best */
    int place = k;
    if (k) {
        /* first among its wave's, then among the waves' k best: all 256 at once read
         * four times the LDS and took 2.8 us of the launch, this 0.9 */
        if (best) place = lp_rank(lkey + 64 * wave, 64, best);
        if (place < k) lcand[atomicAdd(&count[2], 1)] = best;
        __syncthreads();
        if (place < k) place = lp_rank(lcand, count[2], best);
        if (place == k - 1) lleast = best;
    }
    __syncthreads();
    if (place < k) {
        const uint64_t least = lleast;
#pragma unroll
        for (int j = 0; j < kLpHeld; j++) {
            const uint64_t key = lp_key(held[j], tid + 256 * j);
            if (key >= least) lseg[atomicAdd(&count[0], 1)] = key;
        }
#pragma unroll 1
        for (int i = tid + 256 * kLpHeld; i < nseg; i += 256) {
            const uint64_t key = lp_key(seg[i], i);
            if (key >= least) lseg[atomicAdd(&count[0], 1)] = key;
        }
    }
    __syncthreads();
    z = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
    e = (red[2][0] + red[2][1]) + (red[2][2] + red[2][3]);
    const bool bad = z != z;
    /* log z = exponent * log 2 + log of 1 .. 2, and what follows, in 64 bits: in f32 the
     * three roundings of a result were more than the sums' own */
    int ex = 0;
    const float part = frexpf(z, &ex);
    const double lz = (double) (ex - 1) * 0.693147180559945309417 + (double) logf(2.0f * part);
    auto lp = [&](float v) -> float { return bad ? NAN : (v == -INFINITY ? -INFINITY : (float) ((double) v - (double) M - lz)); };
    if (tid == 0) {
        if (A.entropy) A.entropy[r] = bad ? NAN : (M == -INFINITY ? 0.0f : (float) (lz - (double) e / (double) z));
        if (A.tokens) A.logprob[r] = tok >= 0 && tok < A.n ? lp(given) : NAN;
    }
    if (!k) return;
    const int nc = count[0];
    if (tid < kLpPad) lseg[nc + tid] = 0;
    if (tid < kLpMaxK) lpick[tid] = 0;
    __syncthreads();
#pragma unroll 1
    for (int i = tid; i < nc; i += 256) {
        const int rank = lp_rank(lseg, nc, lseg[i]);
        if (rank < k) lpick[rank] = lseg[i];
    }
    __syncthreads();
    /* their logits that are not below the last one's largest */
    const int nk = min(k, nc);
    const float floor_ = nk == k ? lp_value(lpick[k - 1]) : -INFINITY;
    uint64_t * list = lseg;   /* nk * 32 <= 1024 keys */
    static_assert(kLpList >= kLpMaxK * kLpSeg, "the list holds every logit of the picked segments");
#pragma unroll 1
    for (int i = tid; i < nk * kLpSeg; i += 256) {
        const int at = lp_place(lpick[i / kLpSeg]) * kLpSeg + i % kLpSeg;
        if (at >= A.n) continue;
        const float v = lp_one(row + at);
        if (v >= floor_) list[atomicAdd(&count[1], 1)] = lp_key(v, at);
    }
    __syncthreads();
    const int nl = count[1];
    if (tid < kLpPad) list[nl + tid] = 0;
    __syncthreads();
#pragma unroll 1
    for (int i = tid; i < nl; i += 256) {
        const uint64_t key = list[i];
        const int rank = lp_rank(list, nl, key);
        if (rank < k) {
            A.top_id[(size_t) r * k + rank] = lp_place(key);
            A.top_lp[(size_t) r * k + rank] = lp(lp_value(key));
        }
    }
#pragma unroll 1
    for (int i = nl + tid; i < k; i += 256) {
        A.top_id[(size_t) r * k + i] = -1;
        A.top_lp[(size_t) r * k + i] = bad ? NAN : -INFINITY;
    }
}

struct LpPlan {
    int nseg;
    size_t parts, seg, bytes;
};

/* A row's parts are 512 logits at least (two loads of one), so that the size does
 * not depend on type and alignment */
LpPlan lp_plan(int rows, int n, int k) {
    LpPlan p = {};
    p.nseg = (n + kLpSeg - 1) / kLpSeg;
    size_t off = 0;
    auto take = [&](size_t bytes) { const size_t o = off; off += (bytes + 255) & ~(size_t) 255; return o; };
    p.parts = take((size_t) rows * ((n + 511) / 512) * sizeof(lp_f4));
    p.seg = take(k ? (size_t) rows * p.nseg * 4 : 0);
    p.bytes = off;
    return p;
}

}  // namespace

}  // namespace sparkmv

using namespace sparkmv;

extern "C" {

size_t sparkmv_logprobs_work(int rows, int n, int k) {
    if (rows < 1 || n < 1 || n > kLpMaxN || k < 0 || k > kLpMaxK) return 0;
    return lp_plan(rows, n, k).bytes;
}

int sparkmv_logprobs(const void * logits, int x_dtype, int rows, int n, size_t ld, const int * tokens, int k,
                     float * logprob, float * entropy, int * top_id, float * top_logprob, void * work,
                     size_t work_bytes, void * stream) {
    if (x_dtype != SPARKMV_X_F32 && x_dtype != SPARKMV_X_BF16) { set_error("logits: unknown type %d", x_dtype); return -1; }
    if (rows < 0 || n < 1) { set_error("log probabilities of %d rows of %d logits", rows, n); return -1; }
    if (n > kLpMaxN) { set_error("rows of %d logits are above %d", n, kLpMaxN); return -1; }
    if (rows > 65535) { set_error("%d rows of logits are above 65535", rows); return -1; }
    if (k < 0 || k > kLpMaxK) { set_error("%d alternatives are outside 0..%d", k, kLpMaxK); return -1; }
    if (rows == 0) return 0;
    if (!logits) { set_error("logits are null"); return -1; }
    if (rows > 1 && ld < (size_t) n) { set_error("logits: a row stride of %zu holds no %d values", ld, n); return -1; }
    if ((tokens != nullptr) != (logprob != nullptr)) { set_error("given tokens and their log probabilities do not agree"); return -1; }
    if (k && (!top_id || !top_logprob)) { set_error("alternatives without room for them"); return -1; }
    const LpPlan p = lp_plan(rows, n, k);
    if (!work || ((uintptr_t) work & 255) || work_bytes < p.bytes) {
        set_error("log probabilities need %zu bytes of 256-byte aligned workspace, not %zu", p.bytes, work ? work_bytes : 0);
        return -1;
    }
    const bool f32 = x_dtype == SPARKMV_X_F32;
    const bool wide = ((uintptr_t) logits & 15) == 0 && (rows == 1 || ld * (f32 ? 4 : 2) % 16 == 0);
    const int per = wide ? (f32 ? 4 : 8) : 1;          /* logits of a load */
    /* 2 loads a lane until 8 would still give two workgroups a CU. With 2 and 8, us:
     * one row of 131072 12.5 and 13.7, 16 13.8 and 14.2, 512 rows of 30001 at an odd
     * stride 31.2 and 15.2; 512 of 131072 the same within 3 % */
    const int most = 4 * 64 * per * 8;
    const int loads = (long) rows * ((n + most - 1) / most) >= 2 * cu_count() ? 8 : 2;
    LpArgs a;
    a.x = logits; a.n = n; a.k = k; a.ld = ld; a.tokens = tokens;
    a.logprob = logprob; a.entropy = entropy; a.top_id = top_id; a.top_lp = top_logprob;
    a.nparts = (n + 4 * 64 * per * loads - 1) / (4 * 64 * per * loads);
    a.nseg = p.nseg;
    a.parts = (lp_f4 *) ((uint8_t *) work + p.parts);
    a.seg = (float *) ((uint8_t *) work + p.seg);
    hipStream_t s = (hipStream_t) stream;
    const dim3 grid((unsigned) a.nparts, (unsigned) rows), block(256);
#define LP_STREAM(X, V)                                                                                              \
    do {                                                                                                             \
        if (loads == 8) hipLaunchKernelGGL((lp_stream_kernel<X, V, 8>), grid, block, 0, s, a);                       \
        else hipLaunchKernelGGL((lp_stream_kernel<X, V, 2>), grid, block, 0, s, a);                                  \
    } while (0)
    if (f32 && wide) LP_STREAM(float, 4);
    else if (f32) LP_STREAM(float, 1);
    else if (wide) LP_STREAM(uint16_t, 8);
    else LP_STREAM(uint16_t, 1);
#undef LP_STREAM
    if (f32) hipLaunchKernelGGL(lp_join_kernel<float>, dim3((unsigned) rows), block, 0, s, a);
    else hipLaunchKernelGGL(lp_join_kernel<uint16_t>, dim3((unsigned) rows), block, 0, s, a);
    hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : fail_hip("log probabilities launch", e);
}

}  // extern "C"
