// fp8_weight.cu — e4m3 weights: upload of given blocks, quantisation of a
// matrix, and reading them back (cmolcu_fp8_weight_*).
#include "../../include/cmolcu.h"
#include "fp8_weight.cuh"
#include "gemv_launch.cuh"

#include <new>

// One CTA per block: 16-byte chunks of its rows to their place in the tile.
// k is a multiple of 16, so a chunk lies inside the matrix or past it.
__global__ void __launch_bounds__(256) k_fp8_tile(const uint8_t *q, long long q_ld, Fp8W w, uint8_t *tiles) {
    const int kb = blockIdx.x, rb = blockIdx.y;
    uint8_t *t = tiles + ((size_t)rb * w.kblocks + kb) * FP8_TILE_BYTES;
    for (int i = threadIdx.x; i < FP8_BLOCK * 8; i += 256) {
        const int r = i >> 3, c = (i & 7) * 16;
        const long long row = (long long)rb * FP8_BLOCK + r;
        const int col = kb * FP8_BLOCK + c;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (row < w.rows && col < w.k) v = *reinterpret_cast<const uint4 *>(q + row * q_ld + col);
        *reinterpret_cast<uint4 *>(t + fp8_tile_byte(r, c)) = v;
    }
}

// The way back: tiles to rows.
__global__ void __launch_bounds__(256) k_fp8_untile(Fp8W w, uint8_t *q, long long q_ld) {
    const int kb = blockIdx.x, rb = blockIdx.y;
    const uint8_t *t = w.tiles + ((size_t)rb * w.kblocks + kb) * FP8_TILE_BYTES;
    for (int i = threadIdx.x; i < FP8_BLOCK * 8; i += 256) {
        const int r = i >> 3, c = (i & 7) * 16;
        const long long row = (long long)rb * FP8_BLOCK + r;
        const int col = kb * FP8_BLOCK + c;
        if (row < w.rows && col < w.k)
            *reinterpret_cast<uint4 *>(q + row * q_ld + col) = *reinterpret_cast<const uint4 *>(t + fp8_tile_byte(r, c));
    }
}

// One CTA per block of a matrix of f32, f16 or bf16: its values stay in
// registers (8 rows of 8 a thread) between the block's amax and the output.
template <typename T>
__global__ void __launch_bounds__(256) k_fp8_weight_quant(const T *src, long long ld, int vec, Fp8W w, uint8_t *tiles,
                                                          float *scales) {
    __shared__ float red[8];
    const int kb = blockIdx.x, rb = blockIdx.y, tid = threadIdx.x;
    const int c = (tid & 15) * 8, col = kb * FP8_BLOCK + c;
    float v[8][8], amax = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const long long row = (long long)rb * FP8_BLOCK + i * 16 + (tid >> 4);
        Fp8Vec<T, 8> o;
        const bool in = row < w.rows && col < w.k;
        if (in) o.load(src + row * ld + col, vec);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            v[i][e] = in ? fp8_f(o.e[e]) : 0.f;
            amax = fp8_amax(amax, v[i][e]);
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fp8_amax(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if ((tid & 31) == 0) red[tid >> 5] = amax;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; i++) amax = fp8_amax(amax, red[i]);
    const float s = fp8_scale(amax);
    uint8_t *t = tiles + ((size_t)rb * w.kblocks + kb) * FP8_TILE_BYTES;
#pragma unroll
    for (int i = 0; i < 8; i++) fp8_store<8>(t + fp8_tile_byte(i * 16 + (tid >> 4), c), v[i], s);
    if (tid == 0) scales[(size_t)rb * w.kblocks + kb] = s;
}

// Allocates the handle of a [rows x k] matrix on the current device.
static int weight_new(const char *who, int device, int rows, int k, cmolcu_fp8_weight_t **out) {
    cmolcu_fp8_weight *h = new (std::nothrow) cmolcu_fp8_weight();
    if (!h) { cmolcu_set_error("%s: out of host memory", who); return -1; }
    Fp8W &w = h->w;
    w.rows = rows; w.k = k;
    w.rblocks = fp8_blocks(rows); w.kblocks = fp8_blocks(k);
    const size_t nb = (size_t)w.rblocks * w.kblocks;
    cudaError_t e = cudaMalloc(&h->base, nb * (FP8_TILE_BYTES + sizeof(float)));
    if (e != cudaSuccess) {
        cudaGetLastError();
        cmolcu_set_error("%s: %s", who, cudaGetErrorString(e));
        delete h;
        return -1;
    }
    h->device = device;
    w.tiles = static_cast<uint8_t *>(h->base);
    w.scales = reinterpret_cast<float *>(static_cast<uint8_t *>(h->base) + nb * FP8_TILE_BYTES);
    *out = h;
    return 0;
}

static int shape_check(const char *who, const void *src, int rows, int k, long long ld, cmolcu_fp8_weight_t **out) {
    if (!out) { cmolcu_set_error("%s: NULL argument", who); return -1; }
    *out = nullptr;
    if (!src) { cmolcu_set_error("%s: NULL argument", who); return -1; }
    if (rows < 1 || k < 16 || k % 16 || ld < k) {
        cmolcu_set_error("%s: bad shape rows=%d k=%d ld=%lld (k is a multiple of 16)", who, rows, k, ld);
        return -1;
    }
    if (fp8_blocks(rows) > 65535) { cmolcu_set_error("%s: rows=%d is too many", who, rows); return -1; }
    return 0;
}

// Waits for the layout's launch; frees the handle when something failed.
static int weight_done(const char *who, cudaError_t e, cudaStream_t st, cmolcu_fp8_weight_t *h,
                       cmolcu_fp8_weight_t **out) {
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    if (e == cudaSuccess && !cmolcu_fault_word(h->device)) e = cudaErrorMemoryAllocation;   // the product's, made here
    if (e != cudaSuccess) {
        cudaGetLastError();
        cmolcu_set_error("%s: %s", who, cudaGetErrorString(e));
        cmolcu_fp8_weight_free(h);
        return -1;
    }
    *out = h;
    return 0;
}

static cudaError_t tile_launch(const void *q, long long q_ld, const float *scales, cudaMemcpyKind kind,
                               cmolcu_fp8_weight_t *h, cudaStream_t st) {
    const Fp8W &w = h->w;
    cudaError_t e = cudaMemcpyAsync(const_cast<float *>(w.scales), scales,
                                    (size_t)w.rblocks * w.kblocks * sizeof(float), kind, st);
    if (e != cudaSuccess) return e;
    return launch_k(k_fp8_tile, dim3(w.kblocks, w.rblocks), dim3(256), 0, st, false, static_cast<const uint8_t *>(q),
                    q_ld, w, const_cast<uint8_t *>(w.tiles));
}

extern "C" int cmolcu_fp8_weight_upload(int device, const void *q, const float *scales, int rows, int k,
                                        cmolcu_fp8_weight_t **out) {
    static const char *who = "cmolcu_fp8_weight_upload";
    if (shape_check(who, q, rows, k, k, out)) return -1;
    if (!scales) { cmolcu_set_error("%s: NULL argument", who); return -1; }
    Fp8Device dev(device);
    FP8_TRY(who, dev.err);
    cmolcu_fp8_weight_t *h = nullptr;
    if (weight_new(who, device, rows, k, &h)) return -1;
    void *tmp = nullptr;
    cudaError_t e = cudaMalloc(&tmp, (size_t)rows * k);
    if (e == cudaSuccess) e = cudaMemcpy(tmp, q, (size_t)rows * k, cudaMemcpyHostToDevice);
    if (e == cudaSuccess) e = tile_launch(tmp, k, scales, cudaMemcpyHostToDevice, h, 0);
    if (e == cudaSuccess) e = cudaStreamSynchronize(0);
    cudaFree(tmp);
    return weight_done(who, e, 0, h, out);
}

extern "C" int cmolcu_fp8_weight_upload_dev(int device, const void *q, long long q_ld, const float *scales, int rows,
                                            int k, void *stream, cmolcu_fp8_weight_t **out) {
    static const char *who = "cmolcu_fp8_weight_upload_dev";
    if (shape_check(who, q, rows, k, q_ld, out)) return -1;
    if (!scales) { cmolcu_set_error("%s: NULL argument", who); return -1; }
    if (fp8_misaligned(who, scales, 4)) return -1;
    if ((reinterpret_cast<uintptr_t>(q) & 15) || q_ld % 16) {
        cmolcu_set_error("%s: rows must start on 16-byte boundaries (q_ld=%lld)", who, q_ld);
        return -1;
    }
    Fp8Device dev(device);
    FP8_TRY(who, dev.err);
    cmolcu_fp8_weight_t *h = nullptr;
    if (weight_new(who, device, rows, k, &h)) return -1;
    const cudaError_t e = tile_launch(q, q_ld, scales, cudaMemcpyDeviceToDevice, h, (cudaStream_t)stream);
    return weight_done(who, e, (cudaStream_t)stream, h, out);
}

extern "C" int cmolcu_fp8_weight_quantize_dev(int device, const void *w, int dtype, long long ld, int rows, int k,
                                              void *stream, cmolcu_fp8_weight_t **out) {
    static const char *who = "cmolcu_fp8_weight_quantize_dev";
    if (shape_check(who, w, rows, k, ld, out)) return -1;
    const int eb = fp8_elem_bytes(dtype);
    if (!eb) { cmolcu_set_error("%s: unsupported dtype %d", who, dtype); return -1; }
    if (fp8_misaligned(who, w, eb)) return -1;
    Fp8Device dev(device);
    FP8_TRY(who, dev.err);
    cmolcu_fp8_weight_t *h = nullptr;
    if (weight_new(who, device, rows, k, &h)) return -1;
    const int vec = fp8_vec(w, ld * eb);
    const cudaError_t e = fp8_with_type(dtype, [&](auto t) {
        using T = decltype(t);
        return launch_k(k_fp8_weight_quant<T>, dim3(h->w.kblocks, h->w.rblocks), dim3(256), 0, (cudaStream_t)stream,
                        false, static_cast<const T *>(w), ld, vec, h->w, const_cast<uint8_t *>(h->w.tiles),
                        const_cast<float *>(h->w.scales));
    });
    return weight_done(who, e, (cudaStream_t)stream, h, out);
}

extern "C" int cmolcu_fp8_weight_read_dev(const cmolcu_fp8_weight_t *h, void *q, long long q_ld, float *scales,
                                          void *stream) {
    static const char *who = "cmolcu_fp8_weight_read_dev";
    if (!h || !q || !scales) { cmolcu_set_error("%s: NULL argument", who); return -1; }
    if (fp8_misaligned(who, scales, 4)) return -1;
    const Fp8W &w = h->w;
    if ((reinterpret_cast<uintptr_t>(q) & 15) || (w.rows > 1 && (q_ld < w.k || q_ld % 16))) {
        cmolcu_set_error("%s: rows must start on 16-byte boundaries (q_ld=%lld)", who, q_ld);
        return -1;
    }
    Fp8Device dev(h->device);
    FP8_TRY(who, dev.err);
    FP8_TRY(who, cudaMemcpyAsync(scales, w.scales, (size_t)w.rblocks * w.kblocks * sizeof(float),
                             cudaMemcpyDeviceToDevice, (cudaStream_t)stream));
    FP8_TRY(who, launch_k(k_fp8_untile, dim3(w.kblocks, w.rblocks), dim3(256), 0, (cudaStream_t)stream, false, w,
                      static_cast<uint8_t *>(q), q_ld));
    return 0;
}

extern "C" void cmolcu_fp8_weight_free(cmolcu_fp8_weight_t *h) {
    if (!h) return;
    Fp8Device dev(h->device);
    // A handle may go, collected in some language's runtime, while a stream is captured, by this thread or another:
    // only in the relaxed mode does freeing memory leave that capture alone.
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    const cudaError_t e = cudaThreadExchangeStreamCaptureMode(&mode);
    if (cudaFree(h->base) != cudaSuccess) cudaGetLastError();
    if (e == cudaSuccess) cudaThreadExchangeStreamCaptureMode(&mode);
    delete h;
}

extern "C" size_t cmolcu_fp8_weight_bytes(const cmolcu_fp8_weight_t *h) {
    return h ? (size_t)h->w.rows * h->w.k + (size_t)h->w.rblocks * h->w.kblocks * sizeof(float) : 0;
}
