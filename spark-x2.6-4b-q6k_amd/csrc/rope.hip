/* rope.hip — rotary tables scaled for long contexts, and the norm and rotation of
 * query and key heads in one pass (include/sparkmv.h). */
#include "heads.h"

#include <math.h>

namespace sparkmv {

namespace {

/* ---------------------------------------------------------------- the table
 * A thread owns one frequency and walks `run` positions from its first: the sine and
 * cosine there, and from one to the next a rotation by the frequency's own, each off by
 * some 2^-52, which 32 of them do not bring near f32's 2^-24. Bound by the stores: 131072
 * rows of 256 24.7 us, 5.4 TB/s; with a sine and cosine for each pair 47.6. */
struct RopeTable {
    float * table;
    int rows, half, run;
    double freq[kHeadMax / 2];
    double attention;
};

__global__ __launch_bounds__(256) void rope_table_kernel(const RopeTable A) {
    const size_t n = (size_t) blockIdx.x * 256 + threadIdx.x;
    const int j = (int) (n % A.half);
    const long p0 = (long) (n / A.half) * A.run, p1 = min(p0 + A.run, (long) A.rows);
    if (p0 >= p1) return;
    const double f = A.freq[j];
    double s, c, sf, cf;
    sincos((double) p0 * f, &s, &c);
    sincos(f, &sf, &cf);
    s *= A.attention;
    c *= A.attention;
    float * row = A.table + (size_t) p0 * 2 * A.half + j;
    for (long p = p0; p < p1; p++, row += 2 * A.half) {
        row[0] = (float) c;
        row[A.half] = (float) s;
        const double t = fma(c, cf, -(s * sf));
        s = fma(s, cf, c * sf);
        c = t;
    }
}

/* ------------------------------------------------------- norm and rotation
 * A wave takes 64 / lanes heads at a time, a workgroup up to 4 * U such groups of one
 * token, queries' and then keys'. C and S (heads.h) are worked out once a workgroup, an
 * element a thread, and shared through LDS: loaded by every lane from the table and the
 * weights they are four times the bytes of the heads themselves, and what bounds (8192
 * tokens of 40 bf16 heads of 128 68.5 us). Now the rows in and out do: 37.3 us, 4.5 TB/s,
 * where a copy of them takes 33. */
struct QkRope {
    sparkmv_qk_rows r;
    sparkmv_head_turn t;
    double inv_hd;
    int vec;             /* halves are whole pieces of a lane */
    int sh;              /* lanes of a head, as a shift */
    int qgroups, groups; /* groups of a token's queries, and of the token */
    int parts;           /* workgroups of a token */
};

template <typename X, int EL, int U>
__global__ __launch_bounds__(256) void qk_rope_kernel(const QkRope A) {
    typedef typename HeadArith<X>::T T;
    __shared__ T lc[2][kHeadMax], ls[2][kHeadMax];   /* queries', keys' */
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int tok = (int) blockIdx.x / A.parts, g0 = ((int) blockIdx.x - tok * A.parts) * 4 + wave;
    const int hd = A.r.head_dim, half = A.t.rope_dim / 2, inter = A.t.interleaved;
    const int e0 = EL * (lane & ((1 << A.sh) - 1)), per = 64 >> A.sh;
    const int p = half ? A.r.pos[tok] : 0;
    HeadFactor qf, kf;
    if (tid < hd) {
        qf = head_factor(tid, half, inter, A.t.q_norm);
        kf = head_factor(tid, half, inter, A.t.k_norm);
    }
    HeadRaw<X, EL> x[U];
    const X * at[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int g = g0 + 4 * u * A.parts;
        if (g >= A.groups) continue;
        const bool key = g >= A.qgroups;
        const int h = min((key ? g - A.qgroups : g) * per + (lane >> A.sh), (key ? A.r.kv_heads : A.r.heads) - 1);
        at[u] = (const X *) (key ? A.r.k : A.r.q) + (size_t) tok * (key ? A.r.ldk : A.r.ldq) + (size_t) h * hd;
        if (e0 < hd) head_load<EL>(at[u] + e0, x[u]);
    }
    if (half && (p < 0 || p >= A.t.rope_rows)) return;
    if (tid < hd) {
        float c = 0.0f, s = 0.0f;
        if (qf.at >= 0) {
            const float * row = A.t.rope + (size_t) p * A.t.rope_dim + qf.at;
            c = row[0];
            s = row[half];
        }
        head_coef(qf, c, s, lc[0][tid], ls[0][tid]);
        head_coef(kf, c, s, lc[1][tid], ls[1][tid]);
    }
    __syncthreads();
    T C[EL], S[EL];
    int have = -1;
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int g = g0 + 4 * u * A.parts;
        if (g >= A.groups) return;
        const int key = g >= A.qgroups, h = (key ? g - A.qgroups : g) * per + (lane >> A.sh);
        if (key != have) {
#pragma unroll
            for (int i = 0; i < EL; i++) { C[i] = lc[key][e0 + i]; S[i] = ls[key][e0 + i]; }
            have = key;
        }
        float v[EL], w[EL];
        T o[EL];
        head_wide<EL>(x[u], at[u], e0, hd, half, inter, A.vec, v, w);
        const double r = head_norm<EL, T>(v, (key ? A.t.k_norm : A.t.q_norm) != nullptr, A.t.eps, A.inv_hd, A.sh);
        head_turn<EL>(C, S, v, w, r, o);
        if (e0 < hd && h < (key ? A.r.kv_heads : A.r.heads))
            head_store<EL>((X *) (key ? A.r.k_out : A.r.q_out) + (size_t) tok * (key ? A.r.ldko : A.r.ldqo) + (size_t) h * hd + e0, o);
    }
}

}  // namespace

int check_turn(const char * what, const sparkmv_head_turn * t, int hd, long nrow) {
    if (t->rope_dim < 0 || t->rope_dim % 2 || t->rope_dim > hd) {
        set_error("%s: rope_dim %d is not even within 0..%d", what, t->rope_dim, hd);
        return -1;
    }
    if (t->rope_dim && !t->rope) { set_error("%s: rope table is null", what); return -1; }
    if (t->rope_dim && t->rope_rows < nrow) {
        set_error("%s: a rope table of %d rows does not cover %ld positions", what, t->rope_rows, nrow);
        return -1;
    }
    if ((t->q_norm || t->k_norm) && !(t->eps > 0.0f && t->eps < INFINITY)) {
        set_error("%s: a norm's eps must be positive", what);
        return -1;
    }
    return 0;
}

}  // namespace sparkmv

using namespace sparkmv;

extern "C" {

int sparkmv_rope_table_scaled(float * table, int rows, int rope_dim, double theta, const sparkmv_rope_scaling * scaling,
                              void * stream) {
    if (!table) { set_error("rope table is null"); return -1; }
    if (rows < 1 || rope_dim < 2 || rope_dim % 2 || rope_dim > kHeadMax) {
        set_error("rope table of %d rows and %d values", rows, rope_dim);
        return -1;
    }
    if (!(theta > 0.0 && theta < INFINITY)) { set_error("theta must be positive"); return -1; }
    RopeTable a;
    a.table = table; a.rows = rows; a.half = rope_dim / 2;
    sparkmv_rope_scaling z = {};
    if (scaling) z = *scaling;
    if (z.kind < SPARKMV_ROPE_NONE || z.kind > SPARKMV_ROPE_BANDS) { set_error("unknown rope scaling %d", z.kind); return -1; }
    if (z.kind != SPARKMV_ROPE_NONE && !(z.factor >= 1.0 && z.factor < INFINITY)) {
        set_error("a rope scaling's factor must be 1 or more");
        return -1;
    }
    if ((z.kind == SPARKMV_ROPE_YARN || z.kind == SPARKMV_ROPE_BANDS) && !(z.original > 0.0 && z.original < INFINITY)) {
        set_error("a rope scaling by wavelength needs the original context");
        return -1;
    }
    if (!(z.attention >= 0.0 && z.attention < INFINITY)) { set_error("a rope scaling's attention factor is negative"); return -1; }
    if (z.kind == SPARKMV_ROPE_YARN && !(z.beta_slow > 0.0 && z.beta_fast >= z.beta_slow && z.beta_fast < INFINITY)) {
        set_error("yarn needs 0 < beta_slow <= beta_fast");
        return -1;
    }
    if (z.kind == SPARKMV_ROPE_YARN && theta <= 1.0) { set_error("yarn needs a theta above 1"); return -1; }
    if (z.kind == SPARKMV_ROPE_BANDS && !(z.low > 0.0 && z.high > z.low && z.high < INFINITY)) {
        set_error("bands need 0 < low < high");
        return -1;
    }
    const double pi = 3.14159265358979323846, d = (double) rope_dim;
    double lo = 0.0, hi = 0.0;
    if (z.kind == SPARKMV_ROPE_YARN) {
        auto at = [&](double turns) { return d * log(z.original / (2.0 * pi * turns)) / (2.0 * log(theta)); };
        lo = fmax(floor(at(z.beta_fast)), 0.0);
        hi = fmin(ceil(at(z.beta_slow)), d - 1.0);
    }
    const double base = z.kind == SPARKMV_ROPE_NTK && rope_dim > 2 ? theta * pow(z.factor, d / (d - 2.0)) : theta;
    for (int i = 0; i < a.half; i++) {
        double f = pow(base, -2.0 * i / d);
        if (z.kind == SPARKMV_ROPE_LINEAR) {
            f /= z.factor;
        } else if (z.kind == SPARKMV_ROPE_YARN) {
            const double t = fmin(fmax(((double) i - lo) / fmax(hi - lo, 0.001), 0.0), 1.0);
            f = f * (1.0 - t) + f / z.factor * t;
        } else if (z.kind == SPARKMV_ROPE_BANDS) {
            const double turns = z.original * f / (2.0 * pi), t = (turns - z.low) / (z.high - z.low);
            if (turns < z.low) f /= z.factor;
            else if (turns <= z.high) f *= (1.0 - t) / z.factor + t;
        }
        a.freq[i] = f;
    }
    a.attention = z.attention > 0.0 ? z.attention : (z.kind == SPARKMV_ROPE_YARN ? 0.1 * log(z.factor) + 1.0 : 1.0);
    /* few rows: shorter walks, for eight waves a CU (4096 rows of 64 17.9 -> 4.5 us) */
    const long most = 512l * cu_count();
    a.run = 32;
    auto threads = [&]() { return ((long) rows + a.run - 1) / a.run * a.half; };
    while (a.run > 4 && threads() < most) a.run /= 2;
    const long wg = (threads() + 255) / 256;
    if (wg > kKvThreads / 256) { set_error("rope table of %d rows and %d values is too large", rows, rope_dim); return -1; }
    hipLaunchKernelGGL(rope_table_kernel, dim3((unsigned) wg), dim3(256), 0, (hipStream_t) stream, a);
    return kv_check_launch("rope table launch");
}

int sparkmv_qk_rope(const sparkmv_qk_rows * rows, const sparkmv_head_turn * turn, void * stream) {
    if (!rows || !turn) { set_error("qk rope: rows or turn is null"); return -1; }
    const sparkmv_qk_rows & r = *rows;
    if (kv_check_dtype("qk rope", r.x_dtype)) return -1;
    if (r.head_dim < 4 || r.head_dim > kHeadMax || r.head_dim % 4) {
        set_error("qk rope: head_dim %d is not a multiple of 4 within 4..%d", r.head_dim, kHeadMax);
        return -1;
    }
    if (r.ntok < 0) { set_error("%d tokens", r.ntok); return -1; }
    if (r.heads < 0 || r.kv_heads < 0 || r.heads > 65536 || r.kv_heads > 65536) {
        set_error("qk rope: %d query and %d key heads are outside 0..65536", r.heads, r.kv_heads);
        return -1;
    }
    /* an array of no rows may be null */
    if (r.ntok > 0 && ((r.heads > 0) != (r.q != nullptr) || (r.heads > 0) != (r.q_out != nullptr))) {
        set_error("%d query heads, queries and their output do not agree", r.heads);
        return -1;
    }
    if (r.ntok > 0 && ((r.kv_heads > 0) != (r.k != nullptr) || (r.kv_heads > 0) != (r.k_out != nullptr))) {
        set_error("%d key heads, keys and their output do not agree", r.kv_heads);
        return -1;
    }
    if (check_turn("qk rope", turn, r.head_dim, 1)) return -1;
    if (r.ntok == 0 || (r.heads == 0 && r.kv_heads == 0)) return 0;
    if (turn->rope_dim && !r.pos) { set_error("qk rope has no positions"); return -1; }
    const long qd = (long) r.heads * r.head_dim, kd = (long) r.kv_heads * r.head_dim;
    if (r.heads && (kv_check_rows("queries", r.q, r.ldq, qd, r.x_dtype, r.ntok) ||
                    kv_check_rows("turned queries", r.q_out, r.ldqo, qd, r.x_dtype, r.ntok)))
        return -1;
    if (r.kv_heads && (kv_check_rows("keys", r.k, r.ldk, kd, r.x_dtype, r.ntok) ||
                       kv_check_rows("turned keys", r.k_out, r.ldko, kd, r.x_dtype, r.ntok)))
        return -1;
    if (r.ntok > 1 && ((r.heads && r.q == r.q_out && r.ldq != r.ldqo) || (r.kv_heads && r.k == r.k_out && r.ldk != r.ldko))) {
        set_error("rows turned in place with two row strides");
        return -1;
    }
    QkRope a;
    a.r = r; a.t = *turn;
    /* 16 bytes a lane where heads and halves allow */
    const int half = turn->rope_dim / 2;
    const int el = r.x_dtype == SPARKMV_X_BF16 && r.head_dim % 8 == 0 && (turn->interleaved || half % 8 == 0) ? 8 : 4;
    a.vec = half % el == 0;
    a.inv_hd = 1.0 / r.head_dim;
    a.sh = head_lane_shift(r.head_dim, el);
    const int per = 64 >> a.sh;
    a.qgroups = (r.heads + per - 1) / per;
    a.groups = a.qgroups + (r.kv_heads + per - 1) / per;
    auto parts = [&](int u) { return (a.groups + 4 * u - 1) / (4 * u); };
    /* one group a wave, or up to four: 20 f32 heads of 256, 256 tokens 5.0 and 5.6 us, 512
     * 8.2 and 8.2, 4096 49.3 and 41.8 */
    const int u = (long) r.ntok * parts(4) >= 4 * cu_count() ? 4 : 1;
    a.parts = parts(u);
    const long wg = (long) r.ntok * a.parts;
    if (wg > kKvThreads / 256) { set_error("qk rope of %d tokens is too much for one call", r.ntok); return -1; }
    const dim3 grid((unsigned) wg), block(256);
    hipStream_t s = (hipStream_t) stream;
#define QK_ROPE(X, EL)                                                                                               \
    do {                                                                                                             \
        if (u == 4) hipLaunchKernelGGL((qk_rope_kernel<X, EL, 4>), grid, block, 0, s, a);                            \
        else hipLaunchKernelGGL((qk_rope_kernel<X, EL, 1>), grid, block, 0, s, a);                                   \
    } while (0)
    if (r.x_dtype == SPARKMV_X_F32) QK_ROPE(float, 4);
    else if (el == 8) QK_ROPE(uint16_t, 8);
    else QK_ROPE(uint16_t, 4);
#undef QK_ROPE
    return kv_check_launch("qk rope launch");
}

}  // extern "C"
