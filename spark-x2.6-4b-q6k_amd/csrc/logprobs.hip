/* logprobs.hip — log probabilities of given tokens, a row's entropy and its
 * largest logits (include/sparkmv.h). */
#include <hip/hip_runtime.h>
#include <math.h>

#include "../../include/sparkmv.h"
#include "common.h"

namespace sparkmv {

namespace {

constexpr int kLpMaxK = 32;

__device__ __forceinline__ float lp_load(const float * p) { return *p; }
__device__ __forceinline__ float lp_load(const uint16_t * p) { return __uint_as_float((uint32_t) *p << 16); }

/* A logit and its place as one 64-bit number that grows with the logit and, of
 * equal ones, with the lower place; 0 for a NaN. -0 counts as 0. */
__device__ __forceinline__ uint64_t lp_key(float x, int i) {
    if (x != x) return 0;
    const uint32_t u = __float_as_uint(x + 0.0f);
    const uint32_t o = u & 0x80000000u ? ~u : u | 0x80000000u;
    return (uint64_t) o << 32 | (uint32_t) ~i;
}
__device__ __forceinline__ float lp_of(uint64_t key) {
    const uint32_t o = (uint32_t) (key >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

/* One workgroup a row. */
template <typename X>
__global__ __launch_bounds__(1024) void lp_kernel(const X * logits, int n, size_t ld, const int * tokens, int k,
                                                  float * logprob, float * entropy, int * top_id, float * top_lp) {
    __shared__ float red[16], red2[16];
    __shared__ uint64_t rk[16];
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const X * x = logits + (size_t) r * ld;
    float m = -INFINITY;
    bool bad = false;
    for (int i = tid; i < n; i += 1024) {
        const float v = lp_load(x + i);
        bad = bad || v != v || v == INFINITY;
        m = fmaxf(m, v);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    if (lane == 0) red[wave] = m;
    bad = __syncthreads_or(bad);
    for (int w = 0; w < 16; w++) m = fmaxf(m, red[w]);
    float z = 0.0f, e = 0.0f;
    if (m > -INFINITY)
        for (int i = tid; i < n; i += 1024) {
            const float d = lp_load(x + i) - m, p = expf(d);
            z += p;
            if (p > 0.0f) e += p * d;
        }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        z += __shfl_xor(z, o, 64);
        e += __shfl_xor(e, o, 64);
    }
    __syncthreads();
    if (lane == 0) {
        red[wave] = z;
        red2[wave] = e;
    }
    __syncthreads();
    z = e = 0.0f;
    for (int w = 0; w < 16; w++) {
        z += red[w];
        e += red2[w];
    }
    const float lz = logf(z);
    auto lp = [&](float v) { return bad ? NAN : (v == -INFINITY ? -INFINITY : v - m - lz); };
    if (tid == 0) {
        if (entropy) entropy[r] = bad ? NAN : (m == -INFINITY ? 0.0f : lz - e / z);
        if (tokens) {
            const int t = tokens[r];
            logprob[r] = t >= 0 && t < n ? lp(lp_load(x + t)) : NAN;
        }
    }
    uint64_t below = ~0ull;
    for (int j = 0; j < k; j++) {
        uint64_t best = 0;
        for (int i = tid; i < n; i += 1024) {
            const uint64_t key = lp_key(lp_load(x + i), i);
            if (key < below && key > best) best = key;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const uint64_t other = __shfl_xor((unsigned long long) best, o, 64);
            best = other > best ? other : best;
        }
        __syncthreads();
        if (lane == 0) rk[wave] = best;
        __syncthreads();
        for (int w = 0; w < 16; w++) best = rk[w] > best ? rk[w] : best;
        if (tid == 0) {
            top_id[(size_t) r * k + j] = best ? (int) ~(uint32_t) best : -1;
            top_lp[(size_t) r * k + j] = bad ? NAN : (best ? lp(lp_of(best)) : -INFINITY);
        }
        below = best ? best : 1;   /* nothing is below 1 but "none" */
    }
}

}  // namespace

}  // namespace sparkmv

using namespace sparkmv;

extern "C" {

size_t sparkmv_logprobs_work(int rows, int n, int k) {
    (void) rows; (void) n; (void) k;
    return 0;
}

int sparkmv_logprobs(const void * logits, int x_dtype, int rows, int n, size_t ld, const int * tokens, int k,
                     float * logprob, float * entropy, int * top_id, float * top_logprob, void * work,
                     size_t work_bytes, void * stream) {
    if (x_dtype != SPARKMV_X_F32 && x_dtype != SPARKMV_X_BF16) { set_error("logits: unknown type %d", x_dtype); return -1; }
    if (rows < 0 || n < 1) { set_error("log probabilities of %d rows of %d logits", rows, n); return -1; }
    if (k < 0 || k > kLpMaxK) { set_error("%d alternatives are outside 0..%d", k, kLpMaxK); return -1; }
    if (rows == 0) return 0;
    if (!logits) { set_error("logits are null"); return -1; }
    if (rows > 1 && ld < (size_t) n) { set_error("logits: a row stride of %zu holds no %d values", ld, n); return -1; }
    if ((tokens != nullptr) != (logprob != nullptr)) { set_error("given tokens and their log probabilities do not agree"); return -1; }
    if (k && (!top_id || !top_logprob)) { set_error("alternatives without room for them"); return -1; }
    const size_t need = sparkmv_logprobs_work(rows, n, k);
    if (need && (!work || ((uintptr_t) work & 255) || work_bytes < need)) {
        set_error("log probabilities need %zu bytes of 256-byte aligned workspace, not %zu", need, work ? work_bytes : 0);
        return -1;
    }
    hipStream_t s = (hipStream_t) stream;
    if (x_dtype == SPARKMV_X_F32)
        hipLaunchKernelGGL(lp_kernel<float>, dim3((unsigned) rows), dim3(1024), 0, s, (const float *) logits, n, ld, tokens,
                           k, logprob, entropy, top_id, top_logprob);
    else
        hipLaunchKernelGGL(lp_kernel<uint16_t>, dim3((unsigned) rows), dim3(1024), 0, s, (const uint16_t *) logits, n, ld,
                           tokens, k, logprob, entropy, top_id, top_logprob);
    hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : fail_hip("log probabilities launch", e);
}

}  // extern "C"
