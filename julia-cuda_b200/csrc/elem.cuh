// Element access for kernels that take f16, bf16 or f32 tensors: every value is worked on in f32
// and rounded once, to nearest even, when it is stored.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace jc {

// V consecutive elements of T as f32. V * sizeof(T) is 16 bytes (p 16-byte aligned) or V is 1.
template <class T, int V>
struct Elem;

template <class T>
struct Elem<T, 1> {
    static __device__ __forceinline__ void load(const T *p, float *v) { v[0] = static_cast<float>(*p); }
    static __device__ __forceinline__ void store(T *p, const float *v) { *p = static_cast<T>(v[0]); }
};

template <>
struct Elem<__half, 8> {
    static __device__ __forceinline__ void unpack(uint4 q, float *v) {
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
    static __device__ __forceinline__ void load(const __half *p, float *v) {
        unpack(*reinterpret_cast<const uint4 *>(p), v);
    }
    static __device__ __forceinline__ void store(__half *p, const float *v) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
        *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
};

template <>
struct Elem<__nv_bfloat16, 8> {
    static __device__ __forceinline__ void unpack(uint4 q, float *v) {
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
    static __device__ __forceinline__ void load(const __nv_bfloat16 *p, float *v) {
        unpack(*reinterpret_cast<const uint4 *>(p), v);
    }
    static __device__ __forceinline__ void store(__nv_bfloat16 *p, const float *v) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
        *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
};

template <>
struct Elem<float, 4> {
    static __device__ __forceinline__ void load(const float *p, float *v) {
        const float4 q = *reinterpret_cast<const float4 *>(p);
        v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
    }
    static __device__ __forceinline__ void store(float *p, const float *v) {
        *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
    }
};

// Two f32 operations in one instruction (each rounded as its scalar form): a pair is two neighbours of
// an array of even length.
__device__ __forceinline__ void add2(float *d, const float *a, const float *b) {
    asm("{.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
        "add.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;}"
        : "=f"(d[0]), "=f"(d[1])
        : "f"(a[0]), "f"(a[1]), "f"(b[0]), "f"(b[1]));
}
__device__ __forceinline__ void mul2(float *d, const float *a, const float *b) {
    asm("{.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
        "mul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;}"
        : "=f"(d[0]), "=f"(d[1])
        : "f"(a[0]), "f"(a[1]), "f"(b[0]), "f"(b[1]));
}
__device__ __forceinline__ void fma2(float *d, const float *a, const float *b, const float *c) {
    asm("{.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
        "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;}"
        : "=f"(d[0]), "=f"(d[1])
        : "f"(a[0]), "f"(a[1]), "f"(b[0]), "f"(b[1]), "f"(c[0]), "f"(c[1]));
}

// Elements of a 16-byte access.
template <class T>
constexpr int VEC = 16 / (int)sizeof(T);

}  // namespace jc
