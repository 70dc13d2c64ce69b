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

struct LinearParams {
    LinearOperand a, b;
    uint32_t m, n, k;  // c [m][n] = a [m][k] b [n][k]^T
    uint32_t act;
    const float *bias;
    const void *res;
    size_t ldres;
    void *c;
    size_t ldc;
    void *z;
    size_t ldz;
    float *ws;  // split over k: [gridDim.z][m][n] partial sums instead of c
};

constexpr int LIN_T = 64, LIN_K = 16;  // the tile and its depth

template <class T>
__device__ __forceinline__ void lin_load(const LinearOperand &o, uint32_t i0, uint32_t rows, uint32_t k0,
                                         uint32_t k1, float (*s)[LIN_T + 4]) {
#pragma unroll
    for (int l = 0; l < LIN_T * LIN_K / 256; l++) {
        const uint32_t e = threadIdx.x + 256 * l;
        // Consecutive threads read along the operand's contiguous axis.
        const uint32_t i = o.sk == 1 ? e / LIN_K : e % LIN_T, k = o.sk == 1 ? e % LIN_K : e / LIN_T;
        float v = 0.0f;
        if (i0 + i < rows && k0 + k < k1)
            v = static_cast<float>(static_cast<const T *>(o.p)[(size_t)(i0 + i) * o.si + (size_t)(k0 + k) * o.sk]);
        s[k][i] = v;
    }
}

template <class T, uint32_t ACT>
__global__ void __launch_bounds__(256) linear_kernel(const LinearParams p) {
    __shared__ float sa[LIN_K][LIN_T + 4], sb[LIN_K][LIN_T + 4];
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t m0 = blockIdx.y * LIN_T, n0 = blockIdx.x * LIN_T;
    const uint32_t tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const uint32_t blocks = (p.k + LIN_K - 1) / LIN_K;
    const uint32_t kb = (uint32_t)((uint64_t)blocks * blockIdx.z / gridDim.z) * LIN_K;
    const uint32_t ke = min(p.k, (uint32_t)((uint64_t)blocks * (blockIdx.z + 1) / gridDim.z) * LIN_K);
    float acc[4][4] = {};
    for (uint32_t k0 = kb; k0 < ke; k0 += LIN_K) {
        __syncthreads();
        lin_load<T>(p.a, m0, p.m, k0, ke, sa);
        lin_load<T>(p.b, n0, p.n, k0, ke, sb);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < LIN_K; k++) {
            float a[4], b[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                a[i] = sa[k][ty * 4 + i];
                b[i] = sb[k][tx * 4 + i];
            }
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = fmaf(a[i], b[j], acc[i][j]);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t r = m0 + ty * 4 + i;
        if (r >= p.m) continue;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t c = n0 + tx * 4 + j;
            if (c >= p.n) continue;
            float v = acc[i][j];
            if (p.ws) {
                p.ws[((size_t)blockIdx.z * p.m + r) * p.n + c] = v;
                continue;
            }
            if (p.bias) v += p.bias[c];
            if (p.z) static_cast<T *>(p.z)[r * p.ldz + c] = static_cast<T>(v);
            v = act_fwd<ACT>(v);
            if (p.res) v += static_cast<float>(static_cast<const T *>(p.res)[r * p.ldres + c]);
            static_cast<T *>(p.c)[r * p.ldc + c] = static_cast<T>(v);
        }
    }
}

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
    void *dz;  // [m][n] dense, or nullptr
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
#pragma unroll
                for (int i = 0; i < V; i++) d[i] *= act_bwd<ACT>(z[i]);
                Elem<T, V>::store(static_cast<T *>(p.dz) + r * p.lddz + c, d);
            }
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
