// fp8_matmul.cu — matrix product of e4m3 activations (a scale for each 128 of
// a row) with e4m3 weights (a scale for each block of 128 x 128).
//
//   y(c, r) = sum_b sx(c, b) * sw(r / 128, b) * sum_{k in block b} qx(c, k) * qw(r, k)
//
// The scale of a block is applied to its finished sum, so the inner sums are
// products of e4m3 values alone.
#include "../../include/cmolcu.h"
#include "fp8_weight.cuh"
#include "gemv_launch.cuh"

#include <cuda_fp8.h>

struct Fp8MmArgs {
    Fp8W           w;
    const uint8_t *q;
    long long      q_ld;
    const float   *s;
    long long      s_ld, s_inc;
    int            n;
    void          *y;
    long long      y_ld;
};

__device__ __forceinline__ float e4m3_f(uint8_t b) {
    __nv_fp8_e4m3 v;
    v.__x = b;
    return (float)v;
}

// One thread a value of y, 16 columns x 16 rows a CTA: every product formed
// in f32.
template <typename TY>
__global__ void __launch_bounds__(256) k_fp8_mm_simple(const Fp8MmArgs a) {
    pdl_wait();
    pdl_launch_dependents();
    const int r = blockIdx.x * 16 + (threadIdx.x & 15);
    const long long c = (long long)blockIdx.y * 16 + (threadIdx.x >> 4);
    if (r >= a.w.rows || c >= a.n) return;
    float acc = 0.f;
    for (int b = 0; b < a.w.kblocks; b++) {
        const uint8_t *t = a.w.tiles + ((size_t)(r >> 7) * a.w.kblocks + b) * FP8_TILE_BYTES;
        const uint8_t *x = a.q + c * a.q_ld + (long long)b * FP8_BLOCK;
        const int len = min(FP8_BLOCK, a.w.k - b * FP8_BLOCK);
        float d = 0.f;
        for (int k = 0; k < len; k++) d = __fmaf_rn(e4m3_f(x[k]), e4m3_f(t[fp8_tile_byte(r & 127, k)]), d);
        acc = __fmaf_rn(d, a.s[c * a.s_ld + b * a.s_inc] * a.w.scales[(size_t)(r >> 7) * a.w.kblocks + b], acc);
    }
    static_cast<TY *>(a.y)[c * a.y_ld + r] = fp8_t<TY>(acc);
}

extern "C" int cmolcu_fp8_matmul(const cmolcu_fp8_weight_t *w, const void *q, long long q_ld, const float *scales,
                                 long long s_ld, long long s_inc, int n, void *y, int y_dtype, long long y_ld,
                                 void *stream) {
    static const char *who = "cmolcu_fp8_matmul";
    if (!w) { cmolcu_set_error("%s: NULL argument", who); return -1; }
    if (n < 0) { cmolcu_set_error("%s: n=%d", who, n); return -1; }
    if (!fp8_elem_bytes(y_dtype)) { cmolcu_set_error("%s: unsupported dtype %d", who, y_dtype); return -1; }
    if (n == 0) return 0;
    if (!q || !scales || !y) { cmolcu_set_error("%s: NULL argument", who); return -1; }
    if (n == 1) q_ld = (w->w.k + 15) / 16 * 16;        // a single row has no stride
    if ((reinterpret_cast<uintptr_t>(q) & 15) || q_ld < w->w.k || q_ld % 16) {
        cmolcu_set_error("%s: q rows must start on 16-byte boundaries (q_ld=%lld)", who, q_ld);
        return -1;
    }
    if (n > 1 && y_ld < w->w.rows) { cmolcu_set_error("%s: rows of y overlap (y_ld=%lld)", who, y_ld); return -1; }
    Fp8Device dev(w->device);
    CUDA_TRY(dev.err);
    Fp8MmArgs a = {};
    a.w = w->w;
    a.q = static_cast<const uint8_t *>(q); a.q_ld = q_ld;
    a.s = scales; a.s_ld = s_ld; a.s_inc = s_inc;
    a.n = n; a.y = y; a.y_ld = y_ld;
    const dim3 grid((a.w.rows + 15) / 16, (n + 15) / 16);
    CUDA_TRY(fp8_with_type(y_dtype, [&](auto t) {
        return launch_k(k_fp8_mm_simple<decltype(t)>, grid, dim3(256), 0, (cudaStream_t)stream, true, a);
    }));
    return 0;
}
