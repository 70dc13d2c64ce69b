// Layer norm of rows and its gradients.
//
//   forward   mean = sum(x) / d, rstd = 1 / sqrt(sum((x - mean)^2) / d + eps)
//             y = (x - mean) rstd gamma + beta
//   backward  xh = (x - mean) rstd, u = dy gamma
//             dx = rstd (u - sum(u) / d - xh sum(u xh) / d) [+ add]
//             dgamma = sum over rows of dy xh, dbeta = sum over rows of dy
//
// A row is held by G threads, E of its elements in each thread's registers as f32 (G x E >= d), so
// it is read once: the mean is known before the squared deviations are summed, from the same
// registers. Thread t of the row's group holds chunks t, t + G, ... of V elements (16 bytes, or one
// element where the rows are not 16-byte aligned).
#pragma once
#include "common.cuh"
#include "elem.cuh"

namespace jc {

constexpr int NORM_MAX_D = 16384;

// Sum over the G threads of a row's group (G 32: a warp; else the whole block), in a fixed order.
// `part`: one float a warp in shared memory; every thread of the block calls it.
template <int G>
__device__ __forceinline__ float norm_sum(float v, float *part) {
    v = warp_sum(v);
    if constexpr (G > 32) {
        const uint32_t warp = threadIdx.x >> 5;
        __syncthreads();
        if ((threadIdx.x & 31) == 0) part[warp] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int w = 0; w < G / 32; w++) v += part[w];
    }
    return v;
}

// This thread's elements of a row; places past d are 0.
template <class T, int V, int G, int E>
__device__ __forceinline__ void norm_load(const T *row, uint32_t t, uint32_t d, float *v) {
#pragma unroll
    for (int c = 0; c < E / V; c++) {
        const uint32_t j = (c * G + t) * V;
        if (j < d) {
            Elem<T, V>::load(row + j, v + c * V);
        } else {
#pragma unroll
            for (int i = 0; i < V; i++) v[c * V + i] = 0.0f;
        }
    }
}

struct NormParams {
    const void *x;
    size_t ldx;
    const float *gamma, *beta;
    float eps;
    uint32_t rows, d;
    void *y;
    size_t ldy;
    float *stats;
};

template <class T, int V, int G, int E>
__global__ void __launch_bounds__(G < 128 ? 128 : G) norm_kernel(const NormParams p) {
    constexpr int THREADS = G < 128 ? 128 : G;
    __shared__ float part[THREADS / 32];
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t t = threadIdx.x % G;
    const uint32_t r = blockIdx.x * (THREADS / G) + threadIdx.x / G;
    if (G == 32 && r >= p.rows) return;  // a whole warp
    float v[E];
    norm_load<T, V, G, E>(static_cast<const T *>(p.x) + (size_t)r * p.ldx, t, p.d, v);
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < E; i++) s += v[i];
    const float mean = norm_sum<G>(s, part) / (float)p.d;
    s = 0.0f;
#pragma unroll
    for (int c = 0; c < E / V; c++)
        if ((c * G + t) * V < p.d)
#pragma unroll
            for (int i = 0; i < V; i++) {
                const float u = v[c * V + i] - mean;
                s = fmaf(u, u, s);
            }
    const float rstd = rsqrtf(norm_sum<G>(s, part) / (float)p.d + p.eps);
    T *out = static_cast<T *>(p.y) + (size_t)r * p.ldy;
#pragma unroll
    for (int c = 0; c < E / V; c++) {
        const uint32_t j = (c * G + t) * V;
        if (j >= p.d) continue;
        float o[V];
#pragma unroll
        for (int i = 0; i < V; i++) {
            o[i] = (v[c * V + i] - mean) * rstd * __ldg(p.gamma + j + i);
            if (p.beta) o[i] += __ldg(p.beta + j + i);
        }
        Elem<T, V>::store(out + j, o);
    }
    if (p.stats && t == 0) *reinterpret_cast<float2 *>(p.stats + 2 * (size_t)r) = make_float2(mean, rstd);
}

struct NormBwdParams {
    const void *dy;
    size_t lddy;
    const void *x;
    size_t ldx;
    const float *gamma, *stats;
    const void *add;
    size_t ldadd;
    uint32_t rows, d;
    void *dx;
    size_t lddx;
    float *ws;  // [gridDim.x][2][d]: each block's sums for dgamma and dbeta (nullptr: neither is wanted)
};

template <class T, int V, int G, int E>
__global__ void __launch_bounds__(G < 128 ? 128 : G) norm_bwd_kernel(const NormBwdParams p) {
    constexpr int THREADS = G < 128 ? 128 : G, ROWS = THREADS / G;
    __shared__ float part[THREADS / 32];
    extern __shared__ float sums[];  // [2][d], for blocks that hold several rows
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t t = threadIdx.x % G, g = threadIdx.x / G;
    float dg[E], db[E];
#pragma unroll
    for (int i = 0; i < E; i++) dg[i] = db[i] = 0.0f;
    const float inv_d = 1.0f / (float)p.d;
    for (uint32_t r = blockIdx.x * ROWS + g; r < p.rows; r += gridDim.x * ROWS) {
        float x[E], dy[E];
        norm_load<T, V, G, E>(static_cast<const T *>(p.x) + (size_t)r * p.ldx, t, p.d, x);
        norm_load<T, V, G, E>(static_cast<const T *>(p.dy) + (size_t)r * p.lddy, t, p.d, dy);
        const float2 st = *reinterpret_cast<const float2 *>(p.stats + 2 * (size_t)r);
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int c = 0; c < E / V; c++) {
            const uint32_t j = (c * G + t) * V;
            if (j >= p.d) continue;
#pragma unroll
            for (int i = 0; i < V; i++) {
                const int e = c * V + i;
                const float xh = (x[e] - st.x) * st.y, u = dy[e] * __ldg(p.gamma + j + i);
                s1 += u;
                s2 = fmaf(u, xh, s2);
                dg[e] = fmaf(dy[e], xh, dg[e]);
                db[e] += dy[e];
                x[e] = xh;
                dy[e] = u;
            }
        }
        s1 = norm_sum<G>(s1, part) * inv_d;
        s2 = norm_sum<G>(s2, part) * inv_d;
#pragma unroll
        for (int c = 0; c < E / V; c++) {
            const uint32_t j = (c * G + t) * V;
            if (j >= p.d) continue;
            float o[V];
#pragma unroll
            for (int i = 0; i < V; i++) o[i] = st.y * (dy[c * V + i] - s1 - x[c * V + i] * s2);
            if (p.add) {
                float a[V];
                Elem<T, V>::load(static_cast<const T *>(p.add) + (size_t)r * p.ldadd + j, a);
#pragma unroll
                for (int i = 0; i < V; i++) o[i] += a[i];
            }
            Elem<T, V>::store(static_cast<T *>(p.dx) + (size_t)r * p.lddx + j, o);
        }
    }
    if (!p.ws) return;
    // The block's rows meet in shared memory, group after group, so the order of the sums is fixed.
    float *out = p.ws + (size_t)blockIdx.x * 2 * p.d;
#pragma unroll 1
    for (uint32_t k = 0; k < (uint32_t)ROWS; k++) {
        if (g == k) {
#pragma unroll
            for (int c = 0; c < E / V; c++) {
                const uint32_t j = (c * G + t) * V;
                if (j >= p.d) continue;
#pragma unroll
                for (int i = 0; i < V; i++) {
                    float a = dg[c * V + i], b = db[c * V + i];
                    if (k > 0) {
                        a += sums[j + i];
                        b += sums[p.d + j + i];
                    }
                    if (k + 1 < (uint32_t)ROWS) {
                        sums[j + i] = a;
                        sums[p.d + j + i] = b;
                    } else {
                        out[j + i] = a;
                        out[p.d + j + i] = b;
                    }
                }
            }
        }
        if (ROWS > 1) __syncthreads();
    }
}

// out_a[j] = sum over parts of ws[part][j], j < n, and out_b[j] the same of ws[part][n + j] (either
// may be nullptr): 32 columns a block, eight threads a column each summing every eighth part.
__global__ void __launch_bounds__(256) column_sum_kernel(const float *ws, uint32_t parts, uint32_t n,
                                                         uint32_t columns, float *out_a, float *out_b) {
    __shared__ float s[8][32];
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t c = threadIdx.x & 31, k = threadIdx.x >> 5, j = blockIdx.x * 32 + c;
    float v = 0.0f;
    if (j < columns)
        for (uint32_t i = k; i < parts; i += 8) v += ws[(size_t)i * columns + j];
    s[k][c] = v;
    __syncthreads();
    if (k == 0 && j < columns) {
#pragma unroll
        for (int i = 1; i < 8; i++) v += s[i][c];
        if (j < n) {
            if (out_a) out_a[j] = v;
        } else if (out_b) {
            out_b[j - n] = v;
        }
    }
}

}  // namespace jc
