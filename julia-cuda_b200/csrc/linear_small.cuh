// The linear layer where one dimension is tiny: nothing fills a 128-row tensor tile, and the time is
// that of one trip to memory.
//
//   linear_rows_kernel      few rows (a request's markers): the weights are read once for each 16 of
//                           them, straight into mma.sync fragments
//   linear_thin_kernel,     up to 8 output columns (a scorer's last layer): x is read once; forward a
//   linear_thin_bwd_kernel  dot product a row, backward one pass for dx, dw and dbias
#pragma once
#include "common.cuh"
#include "elem.cuh"
#include "linear.cuh"

namespace jc {

// ---------------------------------------------------------------------------------------------
// few rows

struct LinearRowsParams {
    const void *x;
    size_t ldx;
    const void *w;
    size_t ldw;
    const float *bias;
    const void *res;
    size_t ldres;
    void *y;
    size_t ldy;
    void *z;
    size_t ldz;
    uint32_t m, n, k;
};

// d += a b, m16n8k16, f32 sums.
template <class T>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Eight elements, of which `left` exist (VEC: all, on a 16-byte boundary).
template <bool VEC, class T>
__device__ __forceinline__ uint4 eight(const T *p, uint32_t left) {
    if constexpr (VEC) return *reinterpret_cast<const uint4 *>(p);
    const uint16_t *s = reinterpret_cast<const uint16_t *>(p);
    uint32_t v[8];
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = j < (int)min(left, 8u) ? s[j] : 0;
    return make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
}

constexpr int LR_WARPS = 8, LR_AHEAD = 4;

// A block computes 16 rows x 8 columns; its warps take every eighth group of 32 contracted elements and
// their sums meet in shared memory, in order. The contraction's order is free, so a lane loads the 16
// bytes (8 elements) that make its fragments of two MMAs: lane 4 g + q holds elements 8 q .. 8 q + 7 of
// column g of w, and of rows g and g + 8 of x, and takes them in pairs as the MMA's k places 2 q, 2 q + 8.
// Bound by latency: 12 x 768 x 384 takes 1.9 us, 4.9 from cold caches, where a tensor tile takes 5.6.
template <class T, uint32_t ACT, bool VEC>
__global__ void __launch_bounds__(32 * LR_WARPS) linear_rows_kernel(const LinearRowsParams p) {
    __shared__ float sums[LR_WARPS][128];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    const uint32_t c0 = blockIdx.x * 8, r0 = blockIdx.y * 16;
    const T *w = static_cast<const T *>(p.w) + (size_t)(c0 + g) * p.ldw;
    const T *xa = static_cast<const T *>(p.x) + (size_t)(r0 + g) * p.ldx, *xb = xa + 8 * p.ldx;
    const bool col = c0 + g < p.n, ra = r0 + g < p.m, rb = r0 + g + 8 < p.m;
    const uint4 none = make_uint4(0, 0, 0, 0);
    pdl_wait();
    pdl_launch_dependents();
    float d[4] = {};
    for (uint32_t k0 = warp * 32; k0 < p.k; k0 += LR_WARPS * 32 * LR_AHEAD) {
        uint4 b[LR_AHEAD], a0[LR_AHEAD], a1[LR_AHEAD];
#pragma unroll
        for (int i = 0; i < LR_AHEAD; i++) {
            const uint32_t k = k0 + i * LR_WARPS * 32 + 8 * q;
            const bool in = k < p.k;
            b[i] = in && col ? eight<VEC>(w + k, p.k - k) : none;
            a0[i] = in && ra ? eight<VEC>(xa + k, p.k - k) : none;
            a1[i] = in && rb ? eight<VEC>(xb + k, p.k - k) : none;
        }
#pragma unroll
        for (int i = 0; i < LR_AHEAD; i++) {
            const uint32_t lo[4] = {a0[i].x, a1[i].x, a0[i].y, a1[i].y}, hi[4] = {a0[i].z, a1[i].z, a0[i].w, a1[i].w};
            mma_16816<T>(d, lo, b[i].x, b[i].y);
            mma_16816<T>(d, hi, b[i].z, b[i].w);
        }
    }
    // d: rows g and g + 8, columns 2 q and 2 q + 1.
    sums[warp][g * 8 + 2 * q] = d[0];
    sums[warp][g * 8 + 2 * q + 1] = d[1];
    sums[warp][(g + 8) * 8 + 2 * q] = d[2];
    sums[warp][(g + 8) * 8 + 2 * q + 1] = d[3];
    __syncthreads();
    if (threadIdx.x >= 128) return;
    const uint32_t r = r0 + threadIdx.x / 8, c = c0 + threadIdx.x % 8;
    if (r >= p.m || c >= p.n) return;
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < LR_WARPS; i++) v += sums[i][threadIdx.x];
    if (p.bias) v += p.bias[c];
    if (p.z) static_cast<T *>(p.z)[r * p.ldz + c] = static_cast<T>(v);
    v = act_fwd<ACT>(v);
    if (p.res) v += static_cast<float>(static_cast<const T *>(p.res)[r * p.ldres + c]);
    static_cast<T *>(p.y)[r * p.ldy + c] = static_cast<T>(v);
}

// ---------------------------------------------------------------------------------------------
// few columns

constexpr int LTHIN_MAX = 8;
constexpr uint32_t LTHIN_MAX_K = 65535 * 256;  // the backward kernel's grid has 256 of k along y

// Eight of a row's elements for a lane, starting at c0 + 8 lane where rows are on 16-byte boundaries,
// else c0 + lane, c0 + lane + 32, ...; places past the row are 0.
template <class T, bool VEC>
__device__ __forceinline__ void thin_load(const T *row, uint32_t c0, uint32_t k, float *v) {
    const uint32_t lane = threadIdx.x & 31;
    if constexpr (VEC) {
        const uint32_t c = c0 + 8 * lane;
        if (c < k) {
            Elem<T, 8>::load(row + c, v);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = 0.0f;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = c0 + lane + 32 * i < k ? static_cast<float>(row[c0 + lane + 32 * i]) : 0.0f;
    }
}

// A warp a row (LTHIN_ROWS rows at once, so that their loads overlap): y[r][j] for j < n <= N.
constexpr int LTHIN_ROWS = 2;

template <class T, int N, bool VEC, uint32_t ACT>
__global__ void __launch_bounds__(256) linear_thin_kernel(const LinearRowsParams p) {
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t r0 = (blockIdx.x * 8 + (threadIdx.x >> 5)) * LTHIN_ROWS;
    if (r0 >= p.m) return;
    float acc[LTHIN_ROWS][N] = {};
    for (uint32_t c0 = 0; c0 < p.k; c0 += 256) {
        float x[LTHIN_ROWS][8];
#pragma unroll
        for (int i = 0; i < LTHIN_ROWS; i++)
            thin_load<T, VEC>(static_cast<const T *>(p.x) + (size_t)min(r0 + i, p.m - 1) * p.ldx, c0, p.k, x[i]);
#pragma unroll
        for (int j = 0; j < N; j++) {
            if (j >= (int)p.n) break;
            float w[8];
            thin_load<T, VEC>(static_cast<const T *>(p.w) + (size_t)j * p.ldw, c0, p.k, w);
#pragma unroll
            for (int i = 0; i < LTHIN_ROWS; i++)
#pragma unroll
                for (int e = 0; e < 8; e++) acc[i][j] = fmaf(x[i][e], w[e], acc[i][j]);
        }
    }
#pragma unroll
    for (int i = 0; i < LTHIN_ROWS; i++)
#pragma unroll
        for (int j = 0; j < N; j++) {
            float v = warp_sum(acc[i][j]);
            const uint32_t r = r0 + i;
            if (lane != 0 || r >= p.m || j >= (int)p.n) continue;
            if (p.bias) v += p.bias[j];
            if (p.z) static_cast<T *>(p.z)[r * p.ldz + j] = static_cast<T>(v);
            v = act_fwd<ACT>(v);
            if (p.res) v += static_cast<float>(static_cast<const T *>(p.res)[r * p.ldres + j]);
            static_cast<T *>(p.y)[r * p.ldy + j] = static_cast<T>(v);
        }
}

struct LinearThinBwdParams {
    const void *dy;
    size_t lddy;
    const void *x;
    size_t ldx;
    const void *w;
    size_t ldw;
    const void *z;
    size_t ldz;
    uint32_t m, n, k;
    void *dx;  // or nullptr
    size_t lddx;
    float *part;  // [gridDim.x][n k + n]: sums for dw, then dbias (nullptr: neither is wanted)
    bool dw;
};

// blockIdx.y: 256 of the k columns, eight a lane; blockIdx.x: rows, a warp every gridDim.x * 8th. The
// sums for dw stay in registers, the block's warps add theirs up in shared memory in order. dz stays
// f32 here: nothing multiplies it on the tensor cores. 1531 x 384 x 1 with the kernel after it: 6.6 us a
// call, two launches; by tensor tiles, whose launches were four, 10 us more.
template <class T, int N, bool VEC, uint32_t ACT>
__global__ void __launch_bounds__(256) linear_thin_bwd_kernel(const LinearThinBwdParams p) {
    __shared__ float s[8][257];
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c0 = blockIdx.y * 256;
    float w[N][8], dw[N][8], db[N];
#pragma unroll
    for (int j = 0; j < N; j++) {
        db[j] = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) dw[j][e] = w[j][e] = 0.0f;
        if (p.dx && j < (int)p.n) thin_load<T, VEC>(static_cast<const T *>(p.w) + (size_t)j * p.ldw, c0, p.k, w[j]);
    }
    for (uint32_t r = blockIdx.x * 8 + warp; r < p.m; r += gridDim.x * 8) {
        float x[8], o[8];
        if (p.dw) thin_load<T, VEC>(static_cast<const T *>(p.x) + (size_t)r * p.ldx, c0, p.k, x);
#pragma unroll
        for (int e = 0; e < 8; e++) o[e] = 0.0f;
#pragma unroll
        for (int j = 0; j < N; j++) {
            if (j >= (int)p.n) break;
            float dz = static_cast<float>(static_cast<const T *>(p.dy)[r * p.lddy + j]);
            if constexpr (ACT != 0) dz = __fmul_rn(dz, act_bwd<ACT>(static_cast<float>(static_cast<const T *>(p.z)[r * p.ldz + j])));
            db[j] += dz;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                if (p.dw) dw[j][e] = fmaf(dz, x[e], dw[j][e]);
                o[e] = fmaf(dz, w[j][e], o[e]);
            }
        }
        if (!p.dx) continue;
        T *out = static_cast<T *>(p.dx) + (size_t)r * p.lddx;
        if constexpr (VEC) {
            if (c0 + 8 * lane < p.k) Elem<T, 8>::store(out + c0 + 8 * lane, o);
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (c0 + lane + 32 * e < p.k) out[c0 + lane + 32 * e] = static_cast<T>(o[e]);
        }
    }
    if (!p.part) return;
    float *out = p.part + (size_t)blockIdx.x * (p.n * p.k + p.n);
#pragma unroll
    for (int j = 0; j < N; j++) {
        if (j >= (int)p.n) break;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 8; e++) s[warp][VEC ? 8 * lane + e : lane + 32 * e] = dw[j][e];
        if (lane == 0) s[warp][256] = db[j];
        __syncthreads();
        float v = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) v += s[i][threadIdx.x];
        if (p.dw && c0 + threadIdx.x < p.k) out[j * p.k + c0 + threadIdx.x] = v;
        if (threadIdx.x == 0 && blockIdx.y == 0) {
            v = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) v += s[i][256];
            out[p.n * p.k + j] = v;
        }
    }
}

// dw [n][k] and dbias [n] from the blocks' sums: 32 columns a block, 32 threads a column.
template <class T>
__global__ void __launch_bounds__(1024) linear_thin_finish_kernel(const float *part, uint32_t parts, uint32_t n,
                                                                 uint32_t k, T *dw, size_t lddw, float *dbias) {
    __shared__ float s[32][32];
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t c = threadIdx.x & 31, g = threadIdx.x >> 5, j = blockIdx.x * 32 + c, all = n * k + n;
    const bool want = j < all && (j < n * k ? dw != nullptr : dbias != nullptr);
    float v = 0.0f;
    if (want)
#pragma unroll 4
        for (uint32_t i = g; i < parts; i += 32) v += part[(size_t)i * all + j];
    s[g][c] = v;
    __syncthreads();
    if (g != 0 || !want) return;
#pragma unroll
    for (int i = 1; i < 32; i++) v += s[i][c];
    if (j < n * k)
        dw[(size_t)(j / k) * lddw + j % k] = static_cast<T>(v);
    else
        dbias[j - n * k] = v;
}

}  // namespace jc
