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

// z Phi(z) = z / (1 + 2^(-z q(z^2))): q is a polynomial of degree 6 fitted (iteratively reweighted
// least squares) to log2(Phi(z) / Phi(-z)) / z on |z| <= 5.5, weighted by its effect on the result:
// within 6.7e-8 everywhere, and Phi's tails keep their relative size. Past 5.5 q stays and the
// exponent grows with z. Half the instructions of gelu_as, which set the pace of the GELU epilogue.
__device__ __forceinline__ float gelu_fit(float z) {
    const float u = fminf(z * z, 30.25f);
    float q = 5.20991383e-9f;
    q = fmaf(q, u, -3.85045240e-7f);
    q = fmaf(q, u, 1.14524337e-5f);
    q = fmaf(q, u, -1.59389441e-4f);
    q = fmaf(q, u, -9.55928408e-5f);
    q = fmaf(q, u, 0.10483858f);
    q = fmaf(q, u, 2.30220723f);
    return __fdividef(z, 1.0f + ex2_approx(-z * q));
}

// act(z) and act'(z); act: 0, JC_EPI_RELU or JC_EPI_GELU.
template <uint32_t ACT>
__device__ __forceinline__ float act_fwd(float z) {
    if constexpr (ACT == JC_EPI_RELU) return z < 0.0f ? 0.0f : z;  // a NaN stays one
    if constexpr (ACT == JC_EPI_GELU) return gelu_fit(z);
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

// Copies of up to two matrices (rows x cols, any row distance) whose rows start on 16-byte boundaries,
// for TMA: eight elements a thread, blocks [0, first) the one, the others the other. Costs one pass over
// the operand; loaded element by element into the tensor tiles instead, a product of 12288 x 2048 x 767
// took 1037 us.
struct PadParams {
    const uint16_t *src[2];
    size_t ld[2];
    uint32_t rows[2], cols[2];
    uint16_t *dst[2];
    size_t ldd[2];  // a multiple of 8
    uint32_t first;
};

__global__ void __launch_bounds__(256) linear_pad_kernel(const PadParams p) {
    pdl_wait();
    pdl_launch_dependents();
    const int w = blockIdx.x < p.first ? 0 : 1;
    const uint32_t per = (uint32_t)(p.ldd[w] / 8), blocks = w == 0 ? p.first : gridDim.x - p.first;
    const size_t all = (size_t)p.rows[w] * per;
    for (size_t i = (size_t)(blockIdx.x - (w ? p.first : 0)) * 256 + threadIdx.x; i < all; i += (size_t)blocks * 256) {
        const uint32_t r = (uint32_t)(i / per), c = (uint32_t)(i % per) * 8;
        const uint16_t *s = p.src[w] + r * p.ld[w] + c;
        uint32_t v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = c + j < p.cols[w] ? s[j] : 0;
        *reinterpret_cast<uint4 *>(p.dst[w] + r * p.ldd[w] + c) =
            make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
    }
}

// The backward pass's last kernel: the first `join_blocks` blocks write c [m][n] = the sum of `splits`
// partial products in ws, in their order, V columns a thread; the others dbias = the sums of `parts`
// rows of column sums, 32 columns a block, eight threads a column. The partial sums come from L2 (three of
// 2048 x 768: 6.8 us, 8.4 from cold caches).
struct LinearFinishParams {
    const float *ws;
    uint32_t splits, m, n, join_blocks;
    void *c;
    size_t ldc;
    const float *part;
    uint32_t parts, bias_n;
    float *dbias;
};

template <class T, int V>
__global__ void __launch_bounds__(256) linear_finish_kernel(const LinearFinishParams p) {
    __shared__ float sh[8][32];
    pdl_wait();
    pdl_launch_dependents();
    if (blockIdx.x >= p.join_blocks) {
        const uint32_t c = threadIdx.x & 31, k = threadIdx.x >> 5, j = (blockIdx.x - p.join_blocks) * 32 + c;
        float v = 0.0f;
        if (j < p.bias_n)
            for (uint32_t i = k; i < p.parts; i += 8) v += p.part[(size_t)i * p.bias_n + j];
        sh[k][c] = v;
        __syncthreads();
        if (k == 0 && j < p.bias_n) {
#pragma unroll
            for (int i = 1; i < 8; i++) v += sh[i][c];
            p.dbias[j] = v;
        }
        return;
    }
    const size_t all = (size_t)p.m * p.n;
    const uint32_t width = p.n / V;
    for (size_t i = blockIdx.x * (size_t)256 + threadIdx.x; i < all / V; i += (size_t)p.join_blocks * 256) {
        const uint32_t r = (uint32_t)(i / width), c = (uint32_t)(i % width) * V;
        float v[V];
#pragma unroll
        for (int j = 0; j < V; j++) v[j] = 0.0f;
#pragma unroll 4
        for (uint32_t s = 0; s < p.splits; s++) {
            const float *src = p.ws + s * all + i * V;
#pragma unroll
            for (int j = 0; j < V; j += V == 1 ? 1 : 4) {
                float t[4];
                Elem<float, V == 1 ? 1 : 4>::load(src + j, t);
#pragma unroll
                for (int q = 0; q < (V == 1 ? 1 : 4); q++) v[j + q] += t[q];
            }
        }
        Elem<T, V>::store(static_cast<T *>(p.c) + (size_t)r * p.ldc + c, v);
    }
}

struct DzParams {
    const void *dy;
    size_t lddy;
    const void *z;
    size_t ldz;
    uint32_t m, n, rows;  // rows: of a block
    void *dz;  // [m][n], or nullptr
    size_t lddz;
    float *part;  // [gridDim.y][n] column sums, or nullptr
};

constexpr uint32_t DZ_ROWS = 64;  // rows a block covers (few rows: twice that; past 65535 blocks: more)

// dz = dy act'(z) and its sums over each block's rows: a thread walks V columns down every eighth
// row, the block's eight warps meet in shared memory in order. Bound by memory: 12288 x 2048 f16, two
// reads and a write, 25 us.
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
        for (uint32_t r = blockIdx.y * p.rows + warp; r < min(p.m, (blockIdx.y + 1) * p.rows); r += 8) {
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
