// The linear layer for training and its gradients.
//
//   forward   z = x w^T + bias, y = act(z) + res
//   backward  dz = dy act'(z), dx = dz w, dw = dz^T x, dbias = sum over rows of dz
//
// x [m][k], w [n][k], y, z, res, dy [m][n], all of one 16-bit type; bias and dbias f32. Products are
// summed in f32. dz is rounded to the 16-bit type before the two products that read it, since the
// tensor cores take 16-bit operands; dbias sums it before that rounding.
#pragma once
#include "common.cuh"
#include "elem.cuh"

namespace jc {

// act(z) and act'(z); act: 0, JC_EPI_RELU or JC_EPI_GELU (the GELU of the forward GEMMs).
template <uint32_t ACT>
__device__ __forceinline__ float act_fwd(float z) {
    if constexpr (ACT == JC_EPI_RELU) return z < 0.0f ? 0.0f : z;  // a NaN stays one
    if constexpr (ACT == JC_EPI_GELU) return gelu_as(z);
    return z;
}

// GELU'(z) = Phi(z) + z phi(z), with gelu_as's approximation of Phi (1e-7 absolute).
template <uint32_t ACT>
__device__ __forceinline__ float act_bwd(float z) {
    if constexpr (ACT == JC_EPI_RELU) return z > 0.0f ? 1.0f : 0.0f;
    if constexpr (ACT == JC_EPI_GELU) {
        const float t = __fdividef(1.0f, 1.0f + 0.2316419f * fabsf(z));
        float p = 0.5f * 1.061405429f;
        p = p * t + 0.5f * -1.453152027f;
        p = p * t + 0.5f * 1.421413741f;
        p = p * t + 0.5f * -0.284496736f;
        p = p * t + 0.5f * 0.254829592f;
        const float e = __expf(-0.5f * z * z), q = p * t * e;
        return (z >= 0.0f ? 1.0f - q : q) + z * e * 0.3989422804f;
    }
    return 1.0f;
}

// A matrix operand: element (i, k) at p[i si + k sk].
struct LinearOperand {
    const void *p;
    size_t si, sk;
};

// c [m][n] = the sum of `splits` partial products in ws, in their order.
template <class T>
__global__ void __launch_bounds__(256) linear_join_kernel(const float *ws, uint32_t splits, uint32_t m,
                                                          uint32_t n, T *c, size_t ldc) {
    pdl_wait();
    pdl_launch_dependents();
    const size_t all = (size_t)m * n;
    for (size_t i = blockIdx.x * (size_t)256 + threadIdx.x; i < all; i += (size_t)gridDim.x * 256) {
        float v = 0.0f;
        for (uint32_t s = 0; s < splits; s++) v += ws[s * all + i];
        c[i / n * ldc + i % n] = static_cast<T>(v);
    }
}

struct DzParams {
    const void *dy;
    size_t lddy;
    const void *z;
    size_t ldz;
    uint32_t m, n;
    void *dz;  // [m][n], or nullptr
    size_t lddz;
    float *part;  // [gridDim.y][n] column sums, or nullptr
};

constexpr int DZ_ROWS = 64;  // rows a block covers

// dz = dy act'(z) and its sums over each block's rows: a thread walks V columns down every eighth
// row, the block's eight warps meet in shared memory in order.
template <class T, uint32_t ACT, int V>
__global__ void __launch_bounds__(256) linear_dz_kernel(const DzParams p) {
    __shared__ float s[8][32 * V];
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t c = (blockIdx.x * 32 + lane) * V;
    float sum[V];
#pragma unroll
    for (int i = 0; i < V; i++) sum[i] = 0.0f;
    if (c < p.n)
#pragma unroll 2
        for (uint32_t r = blockIdx.y * DZ_ROWS + warp; r < min(p.m, (blockIdx.y + 1) * DZ_ROWS); r += 8) {
            float d[V];
            Elem<T, V>::load(static_cast<const T *>(p.dy) + r * p.lddy + c, d);
            if constexpr (ACT != 0) {
                float z[V];
                Elem<T, V>::load(static_cast<const T *>(p.z) + r * p.ldz + c, z);
                // Rounded by itself: the sums must not depend on whether dz is stored too.
#pragma unroll
                for (int i = 0; i < V; i++) d[i] = __fmul_rn(d[i], act_bwd<ACT>(z[i]));
            }
            if (p.dz) Elem<T, V>::store(static_cast<T *>(p.dz) + r * p.lddz + c, d);
#pragma unroll
            for (int i = 0; i < V; i++) sum[i] += d[i];
        }
    if (!p.part) return;
#pragma unroll
    for (int i = 0; i < V; i++) s[warp][lane * V + i] = sum[i];
    __syncthreads();
    for (uint32_t j = threadIdx.x; j < 32 * V; j += 256) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < 8; w++) v += s[w][j];
        const uint32_t cc = blockIdx.x * 32 * V + j;
        if (cc < p.n) p.part[(size_t)blockIdx.y * p.n + cc] = v;
    }
}

}  // namespace jc
