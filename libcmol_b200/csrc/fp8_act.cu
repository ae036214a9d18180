// fp8_act.cu — activations in 8 bits: RMS norm with the residual's addition,
// and SwiGLU, each leaving e4m3 values with a scale for every 128 of a row
// (cmolcu_fp8_rmsnorm, cmolcu_fp8_swiglu).
#include "../../include/cmolcu.h"
#include "fp8.cuh"
#include "gemv_launch.cuh"

#include <algorithm>
#include <type_traits>

struct Fp8Out {
    uint8_t  *q;
    long long q_ld;
    float    *s;              // scale of (row c, block b) at s[c * s_ld + b * s_inc]
    long long s_ld, s_inc;
};

// Values a lane holds of a row: 32 bytes of x, so that the work a lane does once
// (addresses, a block's scale) is shared by 16 values of the 16-bit types.
template <typename T>
constexpr int lane_values() { return 32 / (int)sizeof(T); }

struct Fp8None {};

struct Fp8ActArgs {
    const void *x, *r;        // input; residual (norm, quantise) or second input (SwiGLU)
    void       *r_out;
    long long   x_ld, r_ld, r_out_ld;
    const float *g;           // norm gains
    float       eps;
    int         n, k;
    int         vx, vr, vo, vg;   // access widths of x, r, r_out, g (fp8_vec)
    Fp8Out      o;
};

// Writes V values of (row, chunk c) in 8 bits; the lanes of a block call it
// together, those past the row with `in` false.
template <int V>
__device__ __forceinline__ void put(const Fp8Out &o, long long row, int c, float (&v)[V], bool in) {
    const float s = fp8_scale(fp8_block_amax<V>(v, in));
    if (!in) return;
    fp8_store<V>(o.q + row * o.q_ld + (long long)c * V, v, s);
    constexpr int L = FP8_BLOCK / V;
    if (c % L == 0) o.s[row * o.s_ld + (long long)(c / L) * o.s_inc] = s;
}

// ---------------------------------------------------------------------------
// RMS norm
// ---------------------------------------------------------------------------
//   h = x + r,  r' = rn(h),  v = g * (h / sqrt(mean(h^2) + eps)),  (q, s) of v
// h stays in f32 between the addition and the norm: only the residual that is
// stored is rounded.  The sum of squares is in f32.
//
// Bound by memory: x and r are read once and stay in registers between the
// sum of squares and the output.  A row is held by W warps (blockDim.x =
// 32 W), V consecutive values a lane and C such chunks; the 128 values of a
// block are 8 or 16 lanes of one warp, so its amax is three or four shuffles.  A
// CTA goes through its rows with the next row's loads on their way and the gains
// in registers.  Rows that are longer (k > 16384; 12288 with f32
// values) are read twice.
template <typename TX, typename TR, int C>
struct NormRow {
    static constexpr int  V = lane_values<TX>();
    static constexpr bool RES = !std::is_same<TR, Fp8None>::value;
    using TRV = typename std::conditional<RES, TR, TX>::type;
    Fp8Vec<TX, V>  x[C];
    Fp8Vec<TRV, V> r[RES ? C : 1];
    // chunks base + i * T + t of a row
    __device__ __forceinline__ void load(const Fp8ActArgs &a, long long row, int first, int T) {
        const int nchunk = a.k / V;
        const TX *xr = static_cast<const TX *>(a.x) + row * a.x_ld;
        const TRV *rr = static_cast<const TRV *>(a.r) + row * a.r_ld;
#pragma unroll
        for (int i = 0; i < C; i++) {
            const int c = first + i * T;
            x[i].zero();
            if (c < nchunk) x[i].load(xr + (long long)c * V, a.vx);
            if constexpr (RES) {
                r[i].zero();
                if (c < nchunk) r[i].load(rr + (long long)c * V, a.vr);
            }
        }
    }
    __device__ __forceinline__ void sum(float (&v)[C][V]) const {
#pragma unroll
        for (int i = 0; i < C; i++)
#pragma unroll
            for (int e = 0; e < V; e += 2) {
                float2 h = make_float2(fp8_f(x[i].e[e]), fp8_f(x[i].e[e + 1]));
                if constexpr (RES) h = fp8_add2(h, make_float2(fp8_f(r[i].e[e]), fp8_f(r[i].e[e + 1])));
                v[i][e] = h.x;
                v[i][e + 1] = h.y;
            }
    }
    __device__ __forceinline__ static void store_sum(const Fp8ActArgs &a, long long row, int c, const float (&v)[V]) {
        if constexpr (RES) {
            Fp8Vec<TRV, V> h;
#pragma unroll
            for (int e = 0; e < V; e++) h.e[e] = fp8_t<TRV>(v[e]);
            h.store(static_cast<TRV *>(a.r_out) + row * a.r_out_ld + (long long)c * V, a.vo);
        }
    }
};

// ss + the squares of v.
template <int V>
__device__ __forceinline__ float2 squares(float2 ss, const float (&v)[V]) {
#pragma unroll
    for (int e = 0; e < V; e += 2) {
        const float2 h = make_float2(v[e], v[e + 1]);
        ss = fp8_fma2(h, h, ss);
    }
    return ss;
}

// v = g * (v * ir)
template <int V>
__device__ __forceinline__ void normalise(float (&v)[V], const float *g, float ir) {
#pragma unroll
    for (int e = 0; e < V; e += 2) {
        const float2 h = fp8_mul2(make_float2(g[e], g[e + 1]), fp8_mul2(make_float2(v[e], v[e + 1]), make_float2(ir, ir)));
        v[e] = h.x;
        v[e + 1] = h.y;
    }
}

// Sum over the T threads of a row; red: a float a warp, of this row's own.
__device__ __forceinline__ float row_sum(float v, int T, float *red) {
    v = warp_sum(v);
    if (T > 32) {                                          // blockDim.y is 1 when a row has several warps
        const int lane = threadIdx.x & 31;
        if (lane == 0) red[threadIdx.x >> 5] = v;
        __syncthreads();
        v = warp_sum(lane < (T >> 5) ? red[lane] : 0.f);
    }
    return v;
}

// Most warps a row: the chunks a lane holds bound the threads that the registers allow.
// (The 16-bit types without a residual would take 73 registers at 24 warps, which leaves
// 25 warps an SM where 64 leave 30: 8192x2560 f16 19.5 us against 17.6.)
template <typename TX, typename TR>
constexpr int norm_warps(int c) {
    constexpr bool half = sizeof(TX) == 2;
    return c == 1 ? (half && std::is_same<TR, Fp8None>::value ? 32 : 24)
                  : c == 2 && !(half && std::is_same<TR, float>::value) ? 16 : 12;
}

template <typename TX, typename TR, int C>
__global__ void __launch_bounds__(32 * norm_warps<TX, TR>(C)) k_fp8_norm(const Fp8ActArgs a) {
    using Row = NormRow<TX, TR, C>;
    constexpr int V = Row::V;
    const int T = blockDim.x, t = threadIdx.x, nchunk = a.k / V;
    const long long step = (long long)gridDim.x * blockDim.y;
    long long row = (long long)blockIdx.x * blockDim.y + threadIdx.y;
    __shared__ float red[2][norm_warps<TX, TR>(C)];
    int flip = 0;
    pdl_wait();
    pdl_launch_dependents();
    Row x;
    if (row < a.n) x.load(a, row, t, T);
    Fp8Vec<float, V> g[C];
#pragma unroll
    for (int i = 0; i < C; i++) {
        g[i].zero();
        if (i * T + t < nchunk) g[i].load(a.g + (long long)(i * T + t) * V, a.vg);
    }
    for (; row < a.n; row += step) {                        // the rows of a CTA with several warps a row: all or none
        float v[C][V];
        float2 ss2 = make_float2(0.f, 0.f);
        x.sum(v);
        if (row + step < a.n) x.load(a, row + step, t, T);
#pragma unroll
        for (int i = 0; i < C; i++) ss2 = squares(ss2, v[i]);
        const float ss = row_sum(ss2.x + ss2.y, T, red[flip]);
        flip ^= 1;
        const float ir = 1.0f / sqrtf(ss / (float)a.k + a.eps);
#pragma unroll
        for (int i = 0; i < C; i++) {
            const int c = i * T + t;
            const bool in = c < nchunk;
            if (in) Row::store_sum(a, row, c, v[i]);
            normalise(v[i], g[i].e, ir);
            put<V>(a.o, row, c, v[i], in);
        }
    }
}

// Rows longer than a CTA's registers hold: one CTA a row, read twice (2048x20000 with the
// residual: bf16 72 us, f32 112; 4.0 and 4.8 TB/s of the bytes counted once).
template <typename TX, typename TR>
__global__ void __launch_bounds__(512) k_fp8_norm_long(const Fp8ActArgs a) {
    using Row = NormRow<TX, TR, 1>;
    constexpr int V = Row::V;
    const int T = blockDim.x, t = threadIdx.x, nchunk = a.k / V;
    const long long row = blockIdx.x;
    __shared__ float red[16];
    pdl_wait();
    pdl_launch_dependents();
    Row x;
    float v[1][V];
    float2 ss = make_float2(0.f, 0.f);
    for (int c = t; c < nchunk; c += T) {
        x.load(a, row, c, T);
        x.sum(v);
        ss = squares(ss, v[0]);
    }
    const float ir = 1.0f / sqrtf(row_sum(ss.x + ss.y, T, red) / (float)a.k + a.eps);
    for (int c0 = 0; c0 < nchunk; c0 += T) {                // whole warps: the lanes of a block stay together
        const int c = c0 + t;
        const bool in = c < nchunk;
        Fp8Vec<float, V> g;
        g.zero();
        if (in) g.load(a.g + (long long)c * V, a.vg);
        x.load(a, row, c, T);
        x.sum(v);
        if (in) Row::store_sum(a, row, c, v[0]);
        normalise(v[0], g.e, ir);
        put<V>(a.o, row, c, v[0], in);
    }
}

template <typename TX, typename TR>
static cudaError_t norm_launch(const Fp8ActArgs &a, cudaStream_t st) {
    constexpr int V = lane_values<TX>(), CMAX = 32 / V;     // at most 32 values of a row a lane
    const int sms = device_sm_count(), warps = (a.k / V + 31) / 32;
    if (warps > norm_warps<TX, TR>(CMAX) * CMAX)
        return launch_k(k_fp8_norm_long<TX, TR>, dim3((unsigned)a.n), dim3(512), 0, st, true, a);
    // Chunks a lane and resident warps an SM, as measured (us, 1 / 2 chunks): a few rows are latency, spread over
    // all lanes (1x960 f32 1.6 / 1.9); up to a wave, fewer warps that wait for the row's sum (256x2048 f32 3.2 / 2.7,
    // 1000x960 bf16 3.3 / 3.1); many rows of up to 8 warps want warps (8191x2048 bf16 20.5 / 21.2, 8192x960 f32 17.8 /
    // 17.9), longer ones fewer at the barrier (2048x8192 bf16 24.2 / 22.2).
    const long long rw = (long long)a.n * warps;
    int c = rw <= sms * 4LL || (rw > sms * 32LL && warps <= 8) ? 1 : 2;
    const int resident = c == 1 ? 48 : 32;
    while (c < CMAX && (warps + c - 1) / c > norm_warps<TX, TR>(c)) c <<= 1;
    const int w = (warps + c - 1) / c, rows = w == 1 ? 4 : 1;
    const long long ctas = ((long long)a.n - 1) / rows + 1;
    const dim3 grid((unsigned)std::min<long long>(ctas, (long long)sms * std::max(1, resident / (w * rows))));
    const dim3 block(32 * w, rows);
    if (c == 1) return launch_k(k_fp8_norm<TX, TR, 1>, grid, block, 0, st, true, a);
    if (c == 2) return launch_k(k_fp8_norm<TX, TR, 2>, grid, block, 0, st, true, a);
    if constexpr (CMAX >= 4) return launch_k(k_fp8_norm<TX, TR, 4>, grid, block, 0, st, true, a);
    return cudaErrorInvalidValue;
}

// ---------------------------------------------------------------------------
// Value by value: SwiGLU, and the 8-bit form of x (+ r) as it is
// ---------------------------------------------------------------------------
//   SwiGLU: v = x / (1 + exp(-x)) * r;  else h = x + r, r' = rn(h), v = h
// A thread takes one chunk of a row.  Bound by memory: 71 us at 8192x11008 bf16
// (6.4 TB/s), the 8-bit form alone 22.4 at 4099x11008 f16 (6.1).
//
// SwiGLU in f32, within 16 * 2^-24 before the 8 bits: exp(-x) = 2^t (1 - n) is the fast 2^t
// of the rounded t = -x log2(e) with n = x + t ln(2) to first order (t's rounding alone
// would cost |x| 2^-24; n^2 is below 2^-33, and f32's ln(2) is off by 2^-28 of itself),
// and the quotient the fast reciprocal.  Each is within two units of the last place.
__device__ __forceinline__ float ex2(float t) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
    return r;
}
__device__ __forceinline__ float rcp(float d) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
    return r;
}
__device__ __forceinline__ float2 swiglu2(float2 x, float2 r) {
    const float c = -1.44269502f, l = 0.693147182f;
    const float2 t = fp8_mul2(x, make_float2(c, c)), m = make_float2(-1.f, -1.f);
    const float2 n = fp8_fma2(t, make_float2(l, l), x);
    const float2 h = make_float2(ex2(t.x), ex2(t.y));
    const float2 d = fp8_fma2(h, n, fp8_fma2(h, m, m));                          // -(1 + exp(-x))
    return fp8_mul2(fp8_mul2(x, make_float2(rcp(-d.x), rcp(-d.y))), r);
}
// Past |x| = 87, where exp(-x) or the reciprocal leaves f32's normal numbers: x exp(x/2) r exp(x/2),
// which may lie far above the scales' floor (x = -100 with r = 2^120 gives -5e-6).
__device__ __forceinline__ float swiglu_far(float x, float r) {
    if (x > 0.f) return x * r;
    const float p = expf(0.5f * x);
    return x * p * r * p;
}

template <typename TX, typename TR, bool SWIGLU>
__global__ void __launch_bounds__(256) k_fp8_map(const Fp8ActArgs a) {
    using Row = NormRow<TX, TR, 1>;
    constexpr int V = Row::V;
    pdl_wait();
    pdl_launch_dependents();
    const long long row = (long long)blockIdx.x * blockDim.y + threadIdx.y;
    const int c = blockIdx.y * blockDim.x + threadIdx.x;
    const bool in = row < a.n && c < a.k / V;
    float v[1][V];
    Row x;
    if (in) x.load(a, row, c, 0);
    if constexpr (SWIGLU) {
        float most = 0.f;
#pragma unroll
        for (int e = 0; e < V; e += 2) {
            const float2 g = make_float2(fp8_f(x.x[0].e[e]), fp8_f(x.x[0].e[e + 1]));
            most = fp8_amax(most, g.x, g.y);
            const float2 h = swiglu2(g, make_float2(fp8_f(x.r[0].e[e]), fp8_f(x.r[0].e[e + 1])));
            v[0][e] = h.x;
            v[0][e + 1] = h.y;
        }
        if (in && !(most <= 87.f)) {                        // read again: kept, they would cost registers
            const TX *gate = static_cast<const TX *>(a.x) + row * a.x_ld + (long long)c * V;
            const TR *up = static_cast<const TR *>(a.r) + row * a.r_ld + (long long)c * V;
#pragma unroll
            for (int e = 0; e < V; e++) {
                const float g = fp8_f(gate[e]);
                if (fabsf(g) > 87.f) v[0][e] = swiglu_far(g, fp8_f(up[e]));
            }
        }
    } else {
        x.sum(v);
        if (in) Row::store_sum(a, row, c, v[0]);
    }
    put<V>(a.o, row, c, v[0], in);
}

template <typename TX, typename TR, bool SWIGLU>
static cudaError_t map_launch(const Fp8ActArgs &a, cudaStream_t st) {
    constexpr int V = lane_values<TX>(), L = FP8_BLOCK / V;
    const int chunks = a.k / V, span = (chunks + L - 1) / L * L;      // whole blocks
    // a narrow row takes part of a CTA (whole warps in all), a wide one several
    const int bx = span <= 64 ? span : std::min(256, (span + 31) / 32 * 32);
    const int by = bx <= 64 ? 256 / bx / 4 * 4 : std::max(1, 256 / bx);
    const dim3 grid((unsigned)((a.n - 1) / by + 1), (unsigned)((chunks - 1) / bx + 1)), block(bx, by);
    if (grid.y > 65535) return cudaErrorInvalidConfiguration;
    return launch_k(k_fp8_map<TX, TR, SWIGLU>, grid, block, 0, st, true, a);
}

// ---------------------------------------------------------------------------
// C ABI
// ---------------------------------------------------------------------------
// Checks of the 8-bit output; 0 or -1 with the message set.
static int out_check(const char *who, int n, int k, void *q, long long q_ld, const float *s, long long s_ld,
                     long long s_inc) {
    if (n < 0 || k < 16 || k % 16) {
        cmolcu_set_error("%s: bad shape n=%d k=%d (k is a multiple of 16)", who, n, k);
        return -1;
    }
    if (n == 0) return 0;
    if (!q || !s) { cmolcu_set_error("%s: NULL argument", who); return -1; }
    if (fp8_misaligned(who, s, 4)) return -1;
    if ((reinterpret_cast<uintptr_t>(q) & 15) || (n > 1 && (q_ld < k || q_ld % 16))) {
        cmolcu_set_error("%s: q rows must start on 16-byte boundaries (q_ld=%lld)", who, q_ld);
        return -1;
    }
    const int kb = fp8_blocks(k);
    if ((n > 1 && s_ld < 1) || (kb > 1 && s_inc < 1) ||
        (n > 1 && kb > 1 && s_ld < (kb - 1) * s_inc + 1 && s_inc < (n - 1) * s_ld + 1)) {
        cmolcu_set_error("%s: scales overlap (s_ld=%lld s_inc=%lld)", who, s_ld, s_inc);
        return -1;
    }
    return 0;
}

extern "C" int cmolcu_fp8_rmsnorm(int device, const void *x, int x_dtype, long long x_ld, const void *res,
                                  long long res_ld, void *res_out, long long res_out_ld, int res_dtype,
                                  const float *norm_w, float eps, int n, int k, void *q, long long q_ld,
                                  float *scales, long long s_ld, long long s_inc, void *stream) {
    static const char *who = "cmolcu_fp8_rmsnorm";
    if (out_check(who, n, k, q, q_ld, scales, s_ld, s_inc)) return -1;
    const int xb = fp8_elem_bytes(x_dtype), rb = res ? fp8_elem_bytes(res_dtype) : 4;
    if (!xb || !rb) { cmolcu_set_error("%s: unsupported dtype %d", who, xb ? res_dtype : x_dtype); return -1; }
    if (n == 0) return 0;
    if (!x || (res && !res_out) || (!res && res_out)) {
        cmolcu_set_error("%s: NULL argument", who);
        return -1;
    }
    if (fp8_misaligned(who, x, xb) || fp8_misaligned(who, res, rb) || fp8_misaligned(who, res_out, rb) ||
        fp8_misaligned(who, norm_w, 4))
        return -1;
    if (res && n > 1 && res_out_ld < k) {
        cmolcu_set_error("%s: rows of the residual overlap (res_out_ld=%lld)", who, res_out_ld);
        return -1;
    }
    Fp8Device dev(device);
    FP8_TRY(who, dev.err);
    Fp8ActArgs a = {};
    a.x = x; a.x_ld = x_ld;
    a.r = res; a.r_ld = res_ld;
    a.r_out = res_out; a.r_out_ld = res_out_ld;
    a.g = norm_w; a.eps = eps; a.n = n; a.k = k;
    a.vx = fp8_vec(x, n > 1 ? x_ld * xb : 0);
    a.vr = fp8_vec(res, n > 1 ? res_ld * rb : 0);
    a.vo = fp8_vec(res_out, n > 1 ? res_out_ld * rb : 0);
    a.vg = fp8_vec(norm_w, 0);
    a.o = {static_cast<uint8_t *>(q), q_ld, scales, s_ld, s_inc};
    const cudaStream_t st = (cudaStream_t)stream;
    FP8_TRY(who, fp8_with_type(x_dtype, [&](auto tx) {
        using TX = decltype(tx);
        if (!res) return norm_w ? norm_launch<TX, Fp8None>(a, st) : map_launch<TX, Fp8None, false>(a, st);
        return fp8_with_type(res_dtype, [&](auto tr) {
            using TR = decltype(tr);
            return norm_w ? norm_launch<TX, TR>(a, st) : map_launch<TX, TR, false>(a, st);
        });
    }));
    return 0;
}

extern "C" int cmolcu_fp8_swiglu(int device, const void *gate, long long gate_ld, const void *up, long long up_ld,
                                 int dtype, int n, int k, void *q, long long q_ld, float *scales, long long s_ld,
                                 long long s_inc, void *stream) {
    static const char *who = "cmolcu_fp8_swiglu";
    if (out_check(who, n, k, q, q_ld, scales, s_ld, s_inc)) return -1;
    const int eb = fp8_elem_bytes(dtype);
    if (!eb) { cmolcu_set_error("%s: unsupported dtype %d", who, dtype); return -1; }
    if (n == 0) return 0;
    if (!gate || !up) { cmolcu_set_error("%s: NULL argument", who); return -1; }
    if (fp8_misaligned(who, gate, eb) || fp8_misaligned(who, up, eb)) return -1;
    Fp8Device dev(device);
    FP8_TRY(who, dev.err);
    Fp8ActArgs a = {};
    a.x = gate; a.x_ld = gate_ld; a.r = up; a.r_ld = up_ld; a.n = n; a.k = k;
    a.vx = fp8_vec(gate, n > 1 ? gate_ld * eb : 0);
    a.vr = fp8_vec(up, n > 1 ? up_ld * eb : 0);
    a.o = {static_cast<uint8_t *>(q), q_ld, scales, s_ld, s_inc};
    FP8_TRY(who, fp8_with_type(dtype, [&](auto t) {
        return map_launch<decltype(t), decltype(t), true>(a, (cudaStream_t)stream);
    }));
    return 0;
}
