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

// ---------------------------------------------------------------------------
// RMS norm
// ---------------------------------------------------------------------------
//   h = x + r,  r' = rn(h),  v = g * (h / sqrt(mean(h^2) + eps)),  (q, s) of v
// h stays in f32 between the addition and the norm: only the residual that is
// stored is rounded.  The sum of squares is in f32.
//
// Bound by memory: x and r are read once and stay in registers between the
// sum of squares and the output.  A row is held by W warps (blockDim.x =
// 32 W), 8 consecutive values a lane and C such octets; the 128 values of a
// block are 16 lanes of one warp, so its amax is four shuffles.  Rows longer
// than a CTA holds (k > 65536) are read twice.
struct Fp8NormArgs {
    const void  *x, *r;
    void        *r_out;
    long long    x_ld, r_ld, r_out_ld;
    const float *g;           // NULL: no norm
    float        eps;
    int          n, k;
    int          vx, vr, vo, vg;   // 16-byte accesses of x, r, r_out, g
    Fp8Out       o;
};

struct Fp8None {};

// Most warps a row: octets of 8 f32 values in registers bound the threads.
static constexpr int norm_warps(int c) { return c == 1 ? 32 : c == 8 ? 8 : 16; }

template <typename TX, typename TR, int C>
__global__ void __launch_bounds__(32 * norm_warps(C)) k_fp8_norm(const Fp8NormArgs a) {
    constexpr bool RES = !std::is_same<TR, Fp8None>::value;
    pdl_wait();
    pdl_launch_dependents();
    const int T = blockDim.x, t = threadIdx.x, lane = t & 31;
    const long long row = (long long)blockIdx.x * blockDim.y + threadIdx.y;
    const bool live = row < a.n;
    const int nchunk = a.k >> 3;
    const int iters = (nchunk - 1) / (T * C) + 1;
    float v[C][8];

    auto load = [&](int it) {
        Fp8Oct<TX> x[C];
        const TX *xr = static_cast<const TX *>(a.x) + row * a.x_ld;
#pragma unroll
        for (int i = 0; i < C; i++) {
            const int c = (it * C + i) * T + t;
            if (live && c < nchunk) x[i].load(xr + (long long)c * 8, a.vx);
        }
        if constexpr (RES) {
            Fp8Oct<TR> r[C];
            const TR *rr = static_cast<const TR *>(a.r) + row * a.r_ld;
#pragma unroll
            for (int i = 0; i < C; i++) {
                const int c = (it * C + i) * T + t;
                if (live && c < nchunk) r[i].load(rr + (long long)c * 8, a.vr);
            }
#pragma unroll
            for (int i = 0; i < C; i++)
#pragma unroll
                for (int e = 0; e < 8; e++)
                    v[i][e] = live && (it * C + i) * T + t < nchunk ? fp8_f(x[i].e[e]) + fp8_f(r[i].e[e]) : 0.f;
        } else {
#pragma unroll
            for (int i = 0; i < C; i++)
#pragma unroll
                for (int e = 0; e < 8; e++)
                    v[i][e] = live && (it * C + i) * T + t < nchunk ? fp8_f(x[i].e[e]) : 0.f;
        }
    };

    float ir = 1.f;
    if (a.g) {
        float ss = 0.f;
        for (int it = 0; it < iters; it++) {
            load(it);
#pragma unroll
            for (int i = 0; i < C; i++)
#pragma unroll
                for (int e = 0; e < 8; e++) ss = __fmaf_rn(v[i][e], v[i][e], ss);
        }
        ss = warp_sum(ss);
        if (T > 32) {
            __shared__ float red[32];                  // blockDim.y is 1 when a row has several warps
            if (lane == 0) red[t >> 5] = ss;
            __syncthreads();
            ss = warp_sum(lane < (T >> 5) ? red[lane] : 0.f);
        }
        ir = 1.0f / sqrtf(ss / (float)a.k + a.eps);
    }
    for (int it = 0; it < iters; it++) {
        if (!a.g || iters > 1) load(it);
#pragma unroll
        for (int i = 0; i < C; i++) {
            const int c = (it * C + i) * T + t;
            const bool in = live && c < nchunk;
            if constexpr (RES) {
                if (in) {
                    Fp8Oct<TR> h;
#pragma unroll
                    for (int e = 0; e < 8; e++) h.e[e] = fp8_t<TR>(v[i][e]);
                    h.store(static_cast<TR *>(a.r_out) + row * a.r_out_ld + (long long)c * 8, a.vo);
                }
            }
            if (a.g) {
                Fp8Oct<float> g;
                if (in) g.load(a.g + (long long)c * 8, a.vg);
#pragma unroll
                for (int e = 0; e < 8; e++) v[i][e] = in ? g.e[e] * (v[i][e] * ir) : 0.f;
            }
            const float s = fp8_scale(fp8_amax16(v[i]));
            if (in) {
                *reinterpret_cast<uint2 *>(a.o.q + row * a.o.q_ld + (long long)c * 8) =
                    fp8_pack8(v[i], __frcp_rn(s));
                if ((lane & 15) == 0) a.o.s[row * a.o.s_ld + (long long)(c >> 4) * a.o.s_inc] = s;
            }
        }
    }
}

template <typename TX, typename TR>
static cudaError_t norm_launch(const Fp8NormArgs &a, cudaStream_t st) {
    const int chunks = (a.k + 255) / 256;              // warps a row at one octet a lane
    int c = 8;
    while (c > 1 && (long long)a.n * ((chunks + c - 1) / c) < 148 * 16) c >>= 1;
    while (c < 8 && (chunks + c - 1) / c > norm_warps(c)) c <<= 1;
    const int w = std::min(norm_warps(c), (chunks + c - 1) / c);
    const int rows = w == 1 ? 4 : 1;
    const dim3 grid((unsigned)((a.n - 1) / rows + 1)), block(32 * w, rows);
    switch (c) {
    case 1: return launch_k(k_fp8_norm<TX, TR, 1>, grid, block, 0, st, true, a);
    case 2: return launch_k(k_fp8_norm<TX, TR, 2>, grid, block, 0, st, true, a);
    case 4: return launch_k(k_fp8_norm<TX, TR, 4>, grid, block, 0, st, true, a);
    default: return launch_k(k_fp8_norm<TX, TR, 8>, grid, block, 0, st, true, a);
    }
}

// ---------------------------------------------------------------------------
// SwiGLU
// ---------------------------------------------------------------------------
//   v = gate / (1 + exp(-gate)) * up,  (q, s) of v
struct Fp8SwigluArgs {
    const void *g, *u;
    long long   g_ld, u_ld;
    int         n, k;
    int         vg, vu;
    Fp8Out      o;
};

template <typename T>
__global__ void __launch_bounds__(256) k_fp8_swiglu(const Fp8SwigluArgs a) {
    pdl_wait();
    pdl_launch_dependents();
    const long long row = blockIdx.x;
    const int c = blockIdx.y * 256 + threadIdx.x;
    const bool in = c < (a.k >> 3);
    Fp8Oct<T> g, u;
    if (in) {
        g.load(static_cast<const T *>(a.g) + row * a.g_ld + (long long)c * 8, a.vg);
        u.load(static_cast<const T *>(a.u) + row * a.u_ld + (long long)c * 8, a.vu);
    }
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float x = fp8_f(g.e[e]);
        v[e] = in ? x / (1.0f + expf(-x)) * fp8_f(u.e[e]) : 0.f;
    }
    const float s = fp8_scale(fp8_amax16(v));
    if (in) {
        *reinterpret_cast<uint2 *>(a.o.q + row * a.o.q_ld + (long long)c * 8) = fp8_pack8(v, __frcp_rn(s));
        if ((threadIdx.x & 15) == 0) a.o.s[row * a.o.s_ld + (long long)(c >> 4) * a.o.s_inc] = s;
    }
}

// ---------------------------------------------------------------------------
// C ABI
// ---------------------------------------------------------------------------
static bool aligned16(const void *p, long long ld, int elem) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld * elem) % 16 == 0;
}

// Checks of the 8-bit output; 0 or -1 with the message set.
static int out_check(const char *who, int n, int k, void *q, long long q_ld, const float *s, long long s_ld,
                     long long s_inc) {
    if (n < 0 || k < 16 || k % 16) {
        cmolcu_set_error("%s: bad shape n=%d k=%d (k is a multiple of 16)", who, n, k);
        return -1;
    }
    if (n == 0) return 0;
    if (!q || !s) { cmolcu_set_error("%s: NULL argument", who); return -1; }
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
    if (res && n > 1 && res_out_ld < k) {
        cmolcu_set_error("%s: rows of the residual overlap (res_out_ld=%lld)", who, res_out_ld);
        return -1;
    }
    Fp8Device dev(device);
    CUDA_TRY(dev.err);
    Fp8NormArgs a = {};
    a.x = x; a.x_ld = x_ld;
    a.r = res; a.r_ld = res_ld;
    a.r_out = res_out; a.r_out_ld = res_out_ld;
    a.g = norm_w; a.eps = eps; a.n = n; a.k = k;
    a.vx = aligned16(x, n > 1 ? x_ld : 0, xb);
    a.vr = aligned16(res, n > 1 ? res_ld : 0, rb);
    a.vo = aligned16(res_out, n > 1 ? res_out_ld : 0, rb);
    a.vg = aligned16(norm_w, 0, 4);
    a.o = {static_cast<uint8_t *>(q), q_ld, scales, s_ld, s_inc};
    CUDA_TRY(fp8_with_type(x_dtype, [&](auto tx) {
        using TX = decltype(tx);
        if (!res) return norm_launch<TX, Fp8None>(a, (cudaStream_t)stream);
        return fp8_with_type(res_dtype, [&](auto tr) { return norm_launch<TX, decltype(tr)>(a, (cudaStream_t)stream); });
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
    Fp8Device dev(device);
    CUDA_TRY(dev.err);
    Fp8SwigluArgs a = {};
    a.g = gate; a.g_ld = gate_ld; a.u = up; a.u_ld = up_ld; a.n = n; a.k = k;
    a.vg = aligned16(gate, n > 1 ? gate_ld : 0, eb);
    a.vu = aligned16(up, n > 1 ? up_ld : 0, eb);
    a.o = {static_cast<uint8_t *>(q), q_ld, scales, s_ld, s_inc};
    const dim3 grid((unsigned)n, (unsigned)((k - 1) / 2048 + 1));
    if (grid.y > 65535) { cmolcu_set_error("%s: k=%d is too long", who, k); return -1; }
    CUDA_TRY(fp8_with_type(dtype, [&](auto t) {
        return launch_k(k_fp8_swiglu<decltype(t)>, grid, dim3(256), 0, (cudaStream_t)stream, true, a);
    }));
    return 0;
}
