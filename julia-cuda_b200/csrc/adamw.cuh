// One AdamW step over many tensors in one launch.
//
//   g' = g grad_scale
//   m = beta1 m + (1 - beta1) g'        v = beta2 v + (1 - beta2) g'^2
//   p = p (1 - lr decay) - lr (m / (1 - beta1^t)) / (sqrt(v / (1 - beta2^t)) + eps)
//
// p, and m and v with 32-bit states, are f32. With 8-bit states m and v are e4m3 codes with one f32
// scale for each 256 consecutive elements (the largest magnitude / 448), taken up and written back
// each step around the same f32 arithmetic; a v above 0 never takes the code 0, so no step divides by
// eps alone while f32 holds the block's v at all. v itself is held, not its root: nearest rounding then follows the 32-bit average with
// no bias (its root within 0.85..1.25 of it for 90% of elements at beta2 0.999, 256 elements of
// log-normal scale sharing a block; a root in e4m3: 0.78..1.34).
#pragma once
#include <cuda_fp8.h>

#include "common.cuh"
#include "elem.cuh"
#include "train.h"

namespace jc {

struct AdamwParams {
    const AdamwTensor *tensors;
    const uint2 *chunks;  // (tensor, chunk of it)
    uint32_t n_chunks;
    const float *grad_scale;
    float beta1, beta2, one_minus_beta1, one_minus_beta2, lr, eps;
    float inv_bias1, inv_bias2;  // 1 / (1 - beta^t)
    float minus_zero;
};

// The largest of a warp's values, none below 0: their bits order as they do.
__device__ __forceinline__ float warp_max_positive(float v) {
    return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v)));
}

// Eight consecutive values at p[0..n) (n up to 8; `vec`: 16-byte aligned and all eight there).
template <class T>
__device__ __forceinline__ void load8(const T *p, uint32_t n, bool vec, float *v) {
    if (vec) {
#pragma unroll
        for (int i = 0; i < 8; i += VEC<T>) Elem<T, VEC<T>>::load(p + i, v + i);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = i < (int)n ? static_cast<float>(p[i]) : 0.0f;
    }
}

template <class T>
__device__ __forceinline__ void store8(T *p, uint32_t n, bool vec, const float *v) {
    if (vec) {
#pragma unroll
        for (int i = 0; i < 8; i += VEC<T>) Elem<T, VEC<T>>::store(p + i, v + i);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < (int)n) p[i] = static_cast<T>(v[i]);
    }
}

// Eight e4m3 codes as f32 times `scale`, and back.
__device__ __forceinline__ void unpack_codes(uint2 q, float scale, float *v) {
    const float s[2] = {scale, scale};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t w = (i < 2 ? q.x : q.y) >> (16 * (i & 1));
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xFFFF), __NV_E4M3);
        const float2 f = __half22float2(__half2(h));
        const float c[2] = {f.x, f.y};
        mul2(v + 2 * i, c, s);
    }
}

__device__ __forceinline__ void load_codes(const uint8_t *p, uint32_t n, float scale, float *v) {
    uint2 q = make_uint2(0, 0);
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (i < (int)n) (i < 4 ? q.x : q.y) |= (uint32_t)p[i] << (8 * (i & 3));
    unpack_codes(q, scale, v);
}

__device__ __forceinline__ void store_codes(uint8_t *p, uint32_t n, bool vec, const float *v) {
    uint32_t q[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t c = __nv_cvt_float2_to_fp8x2(make_float2(v[2 * i], v[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
        q[i >> 1] |= c << (16 * (i & 1));
    }
    if (vec) {
        *reinterpret_cast<uint2 *>(p) = make_uint2(q[0], q[1]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < (int)n) p[i] = (uint8_t)(q[i >> 2] >> (8 * (i & 3)));
    }
}

constexpr float FP8_MAX = 448.0f, FP8_MIN = 0.001953125f;  // e4m3: largest, smallest above 0

// sqrt(x) and a / b on the special-function unit, subnormals taken as 0 (their handling is four more
// instructions each, a sixth of the kernel).
__device__ __forceinline__ float sqrt_fast(float x) {
    float y;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float div_fast(float a, float b) {
    float y;
    asm("div.approx.ftz.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
constexpr float ROOT_MIN = 1.0842022e-19f;  // the root of the smallest normal f32

// Brings a block's scale s below 2^-64, and the values x that it will divide, up by 2^64, which rounds
// nothing and leaves the quotients as they are. A scale fades with its block's gradients (the first
// moment's to below 2^-128 in some 700 steps without any), and the reciprocal of such a one is infinite.
__device__ __forceinline__ void lift8(float *x, float &s) {
    if (s >= 0x1p-64f) return;  // alike in the whole warp
    s *= 0x1p64f;
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] *= 0x1p64f;
}

// x / s for a pair, s at least 2^-85 (lift8), given -s and inv = 1 / s rounded to nearest: the product's
// remainder, exact in one fused multiply-add, corrects it (Markstein, "Computation of elementary functions
// on the IBM RISC System/6000 processor", 1990). The correctly rounded quotient wherever that remainder
// does not underflow, at a fifth of a division's instructions. It underflows only for an x below 2^-95,
// a thousandth of the scale, whose code is 0 either way.
__device__ __forceinline__ void div2(float *x, const float *minus_s, const float *inv) {
    float q[2], r[2];
    mul2(q, x, inv);
    fma2(r, q, minus_s, x);
    fma2(x, r, inv, q);
}

// One thread's eight elements as they lie in memory, with 8-bit states.
struct AdamwRaw {
    uint4 g[2], p[2];
    uint2 m, v;
    float ms, vs;
};

// Blocks stay and walk the chunks, eight consecutive elements a thread (a warp holds the 256 elements
// that share an 8-bit state's scale). The tensors of the two next chunks are looked up, into shared
// memory, while the current one's data is on its way: looked up when needed, the two dependent reads in
// front of every chunk left the memory idle for a third of the time. With 8-bit states, whose elements
// are half the bytes for more arithmetic, the next chunk's data is requested before the current one is
// worked on too (485 -> 470 us for 160 million elements; with 32-bit states the bus is full without).
// Bound by memory: 160 million elements with bf16 gradients and copies, 32-bit states 686 us, 6.5 TB/s, as
// fast as a copy; 8-bit states 492 to 497 us from three models in turn, 5.2 TB/s: half of the issue slots
// are taken, the rest waits for loads that 24 warps a SM (80 registers, 28 bytes spilled) keep too few of
// in flight.
constexpr uint32_t ADAMW_WORDS = sizeof(AdamwTensor) / 4;

template <int BITS>
__global__ void __launch_bounds__(ADAMW_THREADS, BITS == 8 ? 3 : 4) adamw_kernel(const AdamwParams p) {
    constexpr bool AHEAD = BITS == 8;
    __shared__ alignas(16) uint32_t desc[3][ADAMW_WORDS];
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t tid = threadIdx.x;
    auto entry = [&](uint64_t i) { return i < p.n_chunks ? __ldg(p.chunks + i) : make_uint2(0, 0); };
    // Chunk i's tensor into desc[slot]; visible after the next barrier.
    auto look_up = [&](uint64_t i, uint2 ch, int slot) {
        if (i < p.n_chunks && tid < ADAMW_WORDS)
            desc[slot][tid] = __ldg(reinterpret_cast<const uint32_t *>(p.tensors + ch.x) + tid);
    };
    const uint64_t g1 = gridDim.x;
    uint2 ch = entry(blockIdx.x), next = entry(blockIdx.x + g1), after = entry(blockIdx.x + 2 * g1);
    look_up(blockIdx.x, ch, 0);
    look_up(blockIdx.x + g1, next, 1);
    const float gs = p.grad_scale ? *p.grad_scale : 1.0f;
    __syncthreads();
    AdamwRaw raw, coming;
    auto request = [&](const AdamwTensor &t, uint32_t chunk, AdamwRaw &r) {
        const uint64_t at = (uint64_t)chunk * ADAMW_CHUNK + tid * 8;
        if (!t.aligned || at + 8 > t.n) return;
        const uint4 *g = reinterpret_cast<const uint4 *>(static_cast<const uint8_t *>(t.g) + at * (t.grad_type == JC_F32 ? 4 : 2));
        r.g[0] = g[0];
        if (t.grad_type == JC_F32) r.g[1] = g[1];
        r.p[0] = reinterpret_cast<const uint4 *>(t.p + at)[0];
        r.p[1] = reinterpret_cast<const uint4 *>(t.p + at)[1];
        r.m = *reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(t.m) + at);
        r.v = *reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(t.v) + at);
        r.ms = t.m_scale[at / ADAMW_BLOCK];
        r.vs = t.v_scale[at / ADAMW_BLOCK];
    };
    if (AHEAD) request(*reinterpret_cast<const AdamwTensor *>(desc[0]), ch.y, raw);
    int slot = 0;
    for (uint64_t i = blockIdx.x; i < p.n_chunks; i += g1) {
        const int slot1 = slot == 2 ? 0 : slot + 1, slot2 = slot1 == 2 ? 0 : slot1 + 1;
        const AdamwTensor &t = *reinterpret_cast<const AdamwTensor *>(desc[slot]);
        const uint64_t at = (uint64_t)ch.y * ADAMW_CHUNK + tid * 8;
        const bool some = (at & ~uint64_t(255)) < t.n;  // of this warp
        const uint32_t n = at >= t.n ? 0 : (uint32_t)min((uint64_t)8, t.n - at);
        const bool vec = t.aligned && n == 8;
        if (AHEAD && i + g1 < p.n_chunks) request(*reinterpret_cast<const AdamwTensor *>(desc[slot1]), next.y, coming);
        float g[8], m[8], v[8], w[8];
        if (AHEAD && vec) {
            if (t.grad_type == JC_F32) {
                Elem<float, 4>::load(reinterpret_cast<const float *>(&raw.g[0]), g);
                Elem<float, 4>::load(reinterpret_cast<const float *>(&raw.g[1]), g + 4);
            } else if (t.grad_type == JC_F16) {
                Elem<__half, 8>::unpack(raw.g[0], g);
            } else {
                Elem<__nv_bfloat16, 8>::unpack(raw.g[0], g);
            }
            Elem<float, 4>::load(reinterpret_cast<const float *>(&raw.p[0]), w);
            Elem<float, 4>::load(reinterpret_cast<const float *>(&raw.p[1]), w + 4);
            unpack_codes(raw.m, raw.ms, m);
            unpack_codes(raw.v, raw.vs, v);
        } else if (some) {
            if (t.grad_type == JC_F32)
                load8(static_cast<const float *>(t.g) + at, n, vec, g);
            else if (t.grad_type == JC_F16)
                load8(static_cast<const __half *>(t.g) + at, n, vec, g);
            else
                load8(static_cast<const __nv_bfloat16 *>(t.g) + at, n, vec, g);
            load8(t.p + at, n, vec, w);
            if constexpr (BITS == 8) {
                load_codes(static_cast<const uint8_t *>(t.m) + at, n, t.m_scale[at / ADAMW_BLOCK], m);
                load_codes(static_cast<const uint8_t *>(t.v) + at, n, t.v_scale[at / ADAMW_BLOCK], v);
            } else {
                load8(static_cast<const float *>(t.m) + at, n, vec, m);
                load8(static_cast<const float *>(t.v) + at, n, vec, v);
            }
        }
        look_up(i + 2 * g1, after, slot2);
        if (some) {
            const float k = 1.0f - p.lr * t.decay, up = -p.lr * p.inv_bias1;
            const float keep[2] = {k, k}, rate[2] = {up, up}, gs2[2] = {gs, gs}, b1[2] = {p.beta1, p.beta1},
                        b2[2] = {p.beta2, p.beta2}, c1[2] = {p.one_minus_beta1, p.one_minus_beta1},
                        c2[2] = {p.one_minus_beta2, p.one_minus_beta2}, ib2[2] = {p.inv_bias2, p.inv_bias2},
                        eps[2] = {p.eps, p.eps}, none[2] = {p.minus_zero, p.minus_zero};
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                // Each operation of the states is rounded by itself, so that an 8-bit code is that of the
                // formula's own operations. A pair's multiplication and addition the assembler fuses
                // even when both say .rn; a product written as a fused multiply-add of a -0 that it
                // does not know stays apart.
                float a[2], b[2];
                mul2(g + j, g + j, gs2);
                fma2(m + j, m + j, b1, none);
                fma2(a, g + j, c1, none);
                add2(m + j, m + j, a);
                fma2(v + j, v + j, b2, none);
                mul2(a, g + j, c2);
                fma2(a, a, g + j, none);
                add2(v + j, v + j, a);
                // The quotient and root to a few ulp: their error is far below the parameter's own. A
                // subnormal v divides by ROOT_MIN + eps: finite with eps 0 too.
                mul2(a, v + j, ib2);
                a[0] = fmaxf(sqrt_fast(a[0]), ROOT_MIN);
                a[1] = fmaxf(sqrt_fast(a[1]), ROOT_MIN);
                add2(a, a, eps);
                mul2(b, m + j, rate);
                b[0] = div_fast(b[0], a[0]);
                b[1] = div_fast(b[1], a[1]);
                fma2(w + j, w + j, keep, b);
            }
            store8(t.p + at, n, vec, w);
            if (t.copy_type == JC_F16)
                store8(static_cast<__half *>(t.copy) + at, n, vec, w);
            else if (t.copy_type == JC_BF16)
                store8(static_cast<__nv_bfloat16 *>(t.copy) + at, n, vec, w);
            if constexpr (BITS == 8) {
                float mm = 0.0f, vm = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    mm = fmaxf(mm, fabsf(m[j]));
                    vm = fmaxf(vm, v[j]);
                }
                mm = __fmul_rn(warp_max_positive(mm), 1.0f / FP8_MAX);
                vm = __fmul_rn(warp_max_positive(vm), 1.0f / FP8_MAX);
                float sm = mm > 0.0f ? mm : 1.0f, sv = vm > 0.0f ? vm : 1.0f;
                lift8(m, sm);
                lift8(v, sv);
                const float im = __frcp_rn(sm), iv = __frcp_rn(sv);
                const float nsm[2] = {-sm, -sm}, nsv[2] = {-sv, -sv}, im2[2] = {im, im}, iv2[2] = {iv, iv};
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const bool a = v[j] > 0.0f, b = v[j + 1] > 0.0f;
                    div2(m + j, nsm, im2);
                    div2(v + j, nsv, iv2);
                    v[j] = a ? fmaxf(v[j], FP8_MIN) : v[j];
                    v[j + 1] = b ? fmaxf(v[j + 1], FP8_MIN) : v[j + 1];
                }
                store_codes(static_cast<uint8_t *>(t.m) + at, n, vec, m);
                store_codes(static_cast<uint8_t *>(t.v) + at, n, vec, v);
                if ((tid & 31) == 0) {
                    t.m_scale[at / ADAMW_BLOCK] = mm;
                    t.v_scale[at / ADAMW_BLOCK] = vm;
                }
            } else {
                store8(static_cast<float *>(t.m) + at, n, vec, m);
                store8(static_cast<float *>(t.v) + at, n, vec, v);
            }
        }
        __syncthreads();  // the tensor after the next is there, and nobody reads this one any more
        ch = next;
        next = after;
        after = entry(i + 3 * g1);
        slot = slot1;
        if (AHEAD) raw = coming;
    }
}

}  // namespace jc
