// fp8.cuh — shared pieces of the 8-bit floating point path (cmolcu_fp8_*):
// element types, e4m3 conversion, block scales, argument checks.
//
// A value v of a block is stored as q = rn_e4m3(v / s), s = max(amax / 448,
// 2^-126), where amax is the block's largest magnitude: 448 is e4m3's largest
// value, and the floor keeps 1 / s finite for blocks of zeros or of
// subnormals.  In f32: s is amax times the rounded 1 / 448, and the quotient is
// rounded to nearest before its rounding to 8 bits.  A NaN in a block
// makes its scale and its q NaN; an infinity makes the scale infinite, its own q
// NaN and the finite values' q zero: every product with such a block is NaN, as it
// is NaN or infinite without the rounding to 8 bits.
#pragma once
#include "common.cuh"

#include <cuda_bf16.h>

#define FP8_BLOCK 128

enum : int { DT_BF16 = 30 };          // GGUF numbering

__host__ __device__ inline int fp8_blocks(int k) { return (k - 1) / FP8_BLOCK + 1; }

// Bytes of an activation element, 0 for a type that the path does not take.
inline int fp8_elem_bytes(int dt) { return dt == DT_F32 ? 4 : dt == DT_F16 || dt == DT_BF16 ? 2 : 0; }

// Whether an address is no multiple of its elements' size (accesses there would fault);
// sets the message.
inline bool fp8_misaligned(const char *who, const void *p, int elem_bytes) {
    if (reinterpret_cast<uintptr_t>(p) % elem_bytes == 0) return false;
    cmolcu_set_error("%s: an address is no multiple of its element's size", who);
    return true;
}

// Calls f with a value of the element type of tag `dt` (checked by the caller).
template <typename F>
auto fp8_with_type(int dt, F f) {
    switch (dt) {
    case DT_F16: return f(__half());
    case DT_BF16: return f(__nv_bfloat16());
    default: return f(float());
    }
}

// The current device for the life of a call; the caller's is put back.
struct Fp8Device {
    int prev = -1;
    cudaError_t err;
    explicit Fp8Device(int dev) {
        err = cudaGetDevice(&prev);
        if (err == cudaSuccess && dev != prev) err = cudaSetDevice(dev);
        else prev = -1;
    }
    ~Fp8Device() {
        if (prev >= 0) cudaSetDevice(prev);
    }
};

// Returns -1 from the calling entry point with the message set when `expr` fails,
// and leaves no error behind for the program's next look at the runtime's last one.
#define FP8_TRY(who, expr)                                                      \
    do {                                                                        \
        const cudaError_t e_ = (expr);                                          \
        if (e_ != cudaSuccess) {                                                \
            cudaGetLastError();                                                 \
            cmolcu_set_error("%s: %s", who, cudaGetErrorString(e_));            \
            return -1;                                                          \
        }                                                                       \
    } while (0)

// Device fault word of the kernels behind cmolcu.h (seam.cu), null where there is none.
unsigned int *cmolcu_fault_word(int device);

// ---------------------------------------------------------------------------
// Device: 8 values at a time
// ---------------------------------------------------------------------------
__device__ __forceinline__ float fp8_f(float v) { return v; }
__device__ __forceinline__ float fp8_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float fp8_f(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T fp8_t(float v);
template <>
__device__ __forceinline__ float fp8_t<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half fp8_t<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 fp8_t<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// V consecutive elements as they lie in memory, in accesses of 32 or 16 bytes
// (`vec` 2 or 1: the address is a multiple of that) or one by one (0).
template <typename T, int V>
struct Fp8Vec {
    static constexpr int B = V * (int)sizeof(T);
    static_assert(B % 16 == 0, "whole 16-byte accesses");
    alignas(32) T e[V];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < B / 16; i++) reinterpret_cast<uint4 *>(e)[i] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void load(const T *p, int vec) {
        if (B % 32 == 0 && vec == 2) {
            uint32_t *r = reinterpret_cast<uint32_t *>(e);
#pragma unroll
            for (int i = 0; i < B / 32; i++)
                asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                             : "=r"(r[8 * i]), "=r"(r[8 * i + 1]), "=r"(r[8 * i + 2]), "=r"(r[8 * i + 3]),
                               "=r"(r[8 * i + 4]), "=r"(r[8 * i + 5]), "=r"(r[8 * i + 6]), "=r"(r[8 * i + 7])
                             : "l"(reinterpret_cast<const uint8_t *>(p) + 32 * i));
        } else if (vec) {
#pragma unroll
            for (int i = 0; i < B / 16; i++)
                reinterpret_cast<uint4 *>(e)[i] = *(reinterpret_cast<const uint4 *>(p) + i);
        } else {
#pragma unroll
            for (int i = 0; i < V; i++) e[i] = p[i];
        }
    }
    __device__ __forceinline__ void store(T *p, int vec) const {
        if (vec) {
#pragma unroll
            for (int i = 0; i < B / 16; i++)
                *(reinterpret_cast<uint4 *>(p) + i) = reinterpret_cast<const uint4 *>(e)[i];
        } else {
#pragma unroll
            for (int i = 0; i < V; i++) p[i] = e[i];
        }
    }
};

// The widest access that every row of a buffer starts on.
inline int fp8_vec(const void *p, long long ld_bytes) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p) | (uintptr_t)ld_bytes;
    return a % 32 == 0 ? 2 : a % 16 == 0 ? 1 : 0;
}

// Two f32 operations in one instruction: the activation kernels stream memory
// under the power limit, where instructions cost clock.
__device__ __forceinline__ float2 fp8_mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 d, a, b;\n\t"
        "mov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 fp8_add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\t"
        "mov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 fp8_fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}

// max(a, |b|) and max(a, |b|, |c|) that keep a NaN of any side (a >= 0).
__device__ __forceinline__ float fp8_amax(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(b)));
    return r;
}
__device__ __forceinline__ float fp8_amax(float a, float b, float c) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// 1 / s of a scale as hi + lo, within 2^-45 of itself: hi is the approximate reciprocal
// less two units, so below 1 / s, and lo = hi (e + e^2) with the exact e = 1 - s hi.  Then
// v hi + v lo, with one rounding after the second product, is v / s rounded to nearest
// (a quotient of f32 values is not that close to a midpoint but once in 2^20 values, and
// beside e4m3's midpoints, where it would show, far less often); lo >= 0 keeps a zero's
// sign.  lo is normal up to s = 2^90.
struct Fp8Inv {
    float hi, lo;
};
#define FP8_MOST_SCALE 1.2379401e27f           // 2^90
__device__ __forceinline__ Fp8Inv fp8_inv(float s) {
    float r;
    asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(s));
    r *= 0.99999976f;                              // 1 - 2^-22
    const float e = fmaf(-s, r, 1.f);
    return {r, r * fmaf(e, e, e)};
}
__device__ __forceinline__ float2 fp8_div2(float2 v, Fp8Inv i) {
    return fp8_fma2(v, make_float2(i.hi, i.hi), fp8_mul2(v, make_float2(i.lo, i.lo)));
}

// Scale of a block from its largest magnitude: by the rounded 1 / 448, as torch divides a
// tensor on a GPU by a number, within 2^-23 of amax / 448.
__device__ __forceinline__ float fp8_scale(float amax) {
    const float s = amax * (1.f / 448.f), lo = 1.17549435e-38f;
    return s < lo ? lo : s;           // infinite and NaN pass
}

// Two e4m3 values, the first in the low byte (round to nearest even; a NaN
// gives e4m3's NaN).
__device__ __forceinline__ uint32_t fp8_pack2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ uint2 fp8_pack8(const float *v, Fp8Inv inv) {
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 p = fp8_div2(make_float2(v[2 * i], v[2 * i + 1]), inv);
        h[i] = fp8_pack2(p.x, p.y);
    }
    return make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
}

// v / s of V values in 8 bits, to consecutive bytes (V-byte aligned).
template <int V>
__device__ __forceinline__ void fp8_store(uint8_t *q, float (&v)[V], float s) {
    Fp8Inv inv = fp8_inv(s);
    if (s > FP8_MOST_SCALE) {
        if (s <= 3.40282347e38f) {                 // both 2^-64 times as large: what that loses vanishes in e4m3
            inv = fp8_inv(s * 5.4210109e-20f);
#pragma unroll
            for (int i = 0; i < V; i++) v[i] *= 5.4210109e-20f;
        } else {
            inv = {0.f, 0.f};                      // infinite: v times zero
        }
    }
    if constexpr (V == 8) {
        *reinterpret_cast<uint2 *>(q) = fp8_pack8(v, inv);
    } else {
        const uint2 a = fp8_pack8(v, inv), b = fp8_pack8(v + 8, inv);
        *reinterpret_cast<uint4 *>(q) = make_uint4(a.x, a.y, b.x, b.y);
    }
}

// Largest magnitude of the 128 values that 128 / V consecutive lanes hold, V each;
// lanes that are not `in` count as zeros.
template <int V>
__device__ __forceinline__ float fp8_block_amax(const float v[V], bool in) {
    float a = 0.f;
#pragma unroll
    for (int i = 0; i < V; i += 2) a = fp8_amax(a, v[i], v[i + 1]);
    a = in ? a : 0.f;
#pragma unroll
    for (int o = FP8_BLOCK / V / 2; o > 0; o >>= 1) a = fp8_amax(a, __shfl_xor_sync(0xffffffffu, a, o));
    return a;
}
