// Layer norm of rows and its gradients.
//
//   forward   mean = sum(x) / d, rstd = 1 / sqrt(sum((x - mean)^2) / d + eps)
//             y = (x - mean) rstd gamma + beta
//   backward  xh = (x - mean) rstd, u = dy gamma
//             dx = rstd (u - sum(u) / d - xh sum(u xh) / d) [+ add]
//             dgamma = sum over rows of dy xh, dbeta = sum over rows of dy
//
// Both are bound by memory: each row is read from it once, by bulk copies into shared memory a row or
// two ahead, and worked on by G threads with E elements each. The mean is known before the squared
// deviations are summed. Blocks stay and walk rows, with gamma and beta in shared memory. Measured
// (f16 / bf16): forward 196608 x 768 98 us, 6.2 TB/s; 65537 x 1001, whose rows are off every boundary,
// 57 us, 4.6 TB/s, where the masks and edge stores set the pace; backward with residual 196608 x 768 184
// us, 6.6 TB/s, and 12288 x 768 21.5 us, 3.5 TB/s, of which 10 us are its two kernels' starts and ends.
// f32: 65536 x 768 forward 71 us, 5.7 TB/s, backward with residual 124 us, 6.5 TB/s; the backward of rows
// above 32 KB, which reads them from memory twice, 4096 x 12000 424 us, 1.9 TB/s.
//
// Rows are read in 16-byte chunks whatever their width: a row that starts `shift` elements into a
// 16-byte chunk is worked on as the chunks that cover it, the first and last element by element.
// Rows P apart start alike (P: elements in 16 bytes; 1 when every row starts on a boundary), so
// block b takes rows that are b modulo P and one shifted copy of gamma and beta serves it. Tensors
// whose rows start differently from each other are read element by element (V = 1).
#pragma once
#include "common.cuh"
#include "elem.cuh"

namespace jc {

constexpr int NORM_MAX_D = 16384;

// Sums over the G threads of a row's group, in a fixed order: K values at once. `part`: K floats a warp
// in shared memory; G > 32: every thread of the block calls it.
template <int G, int K>
__device__ __forceinline__ void norm_sum(float (&v)[K], float *part) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int k = 0; k < K; k++) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
    if constexpr (G > 32) {
        const uint32_t warp = threadIdx.x >> 5, first = warp / (G / 32) * (G / 32);
        __syncthreads();
        if ((threadIdx.x & 31) == 0)
#pragma unroll
            for (int k = 0; k < K; k++) part[warp * K + k] = v[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; k++) {
            v[k] = 0.0f;
#pragma unroll
            for (int w = 0; w < G / 32; w++) v[k] += part[(first + w) * K + k];
        }
    }
}

// Thread t's share of a row of d elements that starts `shift` elements into its first chunk: chunk c
// holds elements first(c) .. first(c) + V. What lies outside the row is masked in the chunks that need
// it (`edges`, the same for a whole warp and for every row).
template <class T, int V, int G, int E>
struct NormRow {
    static constexpr int N = E / V;
    uint32_t t, shift, d, edges;
    __device__ __forceinline__ NormRow(uint32_t t_, uint32_t shift_, uint32_t d_) : t(t_), shift(shift_), d(d_), edges(0) {
#pragma unroll
        for (int c = 0; c < N; c++)
            if (__any_sync(0xffffffffu, !whole(c))) edges |= 1u << c;
    }
    __device__ __forceinline__ uint32_t place(int c) const { return (c * G + t) * V; }
    __device__ __forceinline__ int first(int c) const { return (int)place(c) - (int)shift; }
    __device__ __forceinline__ bool whole(int c) const {
        return V == 1 ? place(c) < d : first(c) >= 0 && first(c) + V <= (int)d;
    }
    __device__ __forceinline__ bool some(int c) const {
        return V == 1 ? place(c) < d : first(c) + V > 0 && first(c) < (int)d;
    }
    __device__ __forceinline__ bool has(int c, int i) const {
        return (uint32_t)(first(c) + i) < d;  // below 0 wraps past d
    }
    __device__ __forceinline__ bool edge(int c) const { return edges >> c & 1; }
    // Whether row r's outer chunks may reach past the tensor's first or last element.
    __device__ __forceinline__ bool ends(uint64_t r, uint32_t rows) const {
        return V > 1 && (r * d < V || (rows - 1 - r) * d < V);
    }
    // Chunk c of a row in global memory as f32, 0 outside the row.
    __device__ __forceinline__ void chunk(const T *row, int c, bool ends, float *v) const {
        if (!edge(c) || (ends ? whole(c) : some(c))) {
            Elem<T, V>::load(row + first(c), v);
            mask(c, v);
        } else {
#pragma unroll
            for (int i = 0; i < V; i++) v[i] = has(c, i) ? static_cast<float>(row[first(c) + i]) : 0.0f;
        }
    }
    // 0 outside the row.
    __device__ __forceinline__ void mask(int c, float *v) const {
        if (edge(c))
#pragma unroll
            for (int i = 0; i < V; i++) v[i] = has(c, i) ? v[i] : 0.0f;
    }
    __device__ __forceinline__ void store(T *row, int c, const float *v) const {
        if (!edge(c) || whole(c)) {
            Elem<T, V>::store(row + first(c), v);
        } else if (V > 1 && some(c)) {
#pragma unroll
            for (int i = 0; i < V; i++)
                if (has(c, i)) row[first(c) + i] = static_cast<T>(v[i]);
        }
    }
};

// The sum of v[0..E), two running sums side by side.
template <int E>
__device__ __forceinline__ float norm_add_up(const float *v) {
    float s[2] = {v[0], v[1]};
#pragma unroll
    for (int i = 2; i < E; i += 2) add2(s, s, v + i);
    return s[0] + s[1];
}

// gamma or beta in shared memory at the places the rows' elements have, 0 outside the row. Eight a
// chunk are kept as two arrays of four, so that a warp's 16-byte reads are free of bank conflicts.
template <int V, int G, int E>
__device__ __forceinline__ uint32_t norm_param_at(uint32_t place) {
    if constexpr (V == 8) return (place & 4) / 4 * (G * E / 2) + place / 8 * 4 + (place & 3);
    return place;
}

template <int V, int G, int E>
__device__ __forceinline__ void norm_stage_param(float *s, const float *g, uint32_t shift, uint32_t d,
                                                 uint32_t threads) {
    for (uint32_t k = threadIdx.x; k < (uint32_t)(G * E); k += threads)
        s[norm_param_at<V, G, E>(k)] = g && k - shift < d ? g[k - shift] : 0.0f;
}

template <int V, int G, int E>
__device__ __forceinline__ void norm_param(const float *s, uint32_t place, float *v) {
    if constexpr (V == 1) {
        v[0] = s[place];
    } else {
        Elem<float, 4>::load(s + norm_param_at<V, G, E>(place), v);
        if constexpr (V == 8) Elem<float, 4>::load(s + norm_param_at<V, G, E>(place + 4), v + 4);
    }
}

// `bytes` (a multiple of 16, both addresses on 16-byte boundaries) of global into shared memory,
// completing on `bar`.
__device__ __forceinline__ void bulk_load(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                     smem_u32(dst)),
                 "l"(src), "r"(bytes), "r"(smem_u32(bar))
                 : "memory");
}

struct NormParams {
    const void *x;
    size_t ldx;
    const float *gamma, *beta;
    float eps;
    uint32_t rows, d, period;  // period: P above; gridDim.x is a multiple of it
    void *y;
    size_t ldy;
    float *stats;
    unsigned int *err;
};

// How a block of the forward kernel is made up: rows of x come into shared memory by bulk copies, STAGES
// times ROWS rows ahead, each group its own, and ROWS rows are worked on side by side. A warp's two rows
// have one stage: with two stages 14 MB were in flight and 196608 x 768 took 113 us instead of 98 (6.15
// TB/s); one row at a time took 109. STAGES 0 (V = 1): read where they are used.
template <class T, int V, int G, int E>
struct NormShape {
    static constexpr int ROW = G * E * (int)sizeof(T);  // bytes
    static constexpr int ROWS = V > 1 && G == 32 ? 2 : 1;
    static constexpr int STAGES = V == 1 ? 0 : G == 32 || ROW > 32768 ? 1 : 2;
    static constexpr int THREADS = G > 256 ? G : 256, GROUPS = THREADS / G;
    static constexpr int SMEM = 2 * G * E * 4 + GROUPS * STAGES * ROWS * ROW;  // gamma, beta, the rings
    // Blocks an SM should hold: what the registers of a row allow.
    static constexpr int RESIDENT = G > 256 ? 1 : E == 8 ? (ROWS == 2 ? 5 : 6) : E == 16 ? (ROWS == 2 ? 3 : 4)
                                    : E == 24 ? (ROWS == 2 ? 2 : 4) : ROWS == 2 ? 2 : G < 256 ? 3 : sizeof(T) == 4 ? 1 : 2;
    static_assert(SMEM <= 227 * 1024 - 1024, "shared memory");
};

template <class T, int V, int G, int E>
__global__ void __launch_bounds__(NormShape<T, V, G, E>::THREADS, NormShape<T, V, G, E>::RESIDENT)
    norm_kernel(const NormParams p) {
    using S = NormShape<T, V, G, E>;
    using Row = NormRow<T, V, G, E>;
    constexpr int THREADS = S::THREADS, GROUPS = S::GROUPS, STAGES = S::STAGES, R = S::ROWS;
    __shared__ float part[R * THREADS / 32];
    __shared__ uint64_t bars[GROUPS * (STAGES ? STAGES : 1)];
    extern __shared__ __align__(16) float smem[];
    dev_err_bind(p.err);
    const uint32_t g = threadIdx.x / G, cls = blockIdx.x % p.period, step = gridDim.x / p.period * GROUPS * R;
    const T *x = static_cast<const T *>(p.x);
    const Row row(threadIdx.x % G,
                  V == 1 ? 0 : (uint32_t)(reinterpret_cast<uintptr_t>(x + (size_t)cls * p.ldx) % 16 / sizeof(T)), p.d);
    // Rows i .. i + R of this group are rows cls + i period ..; a group that is out of rows keeps its
    // block's company.
    uint32_t i = blockIdx.x / p.period * GROUPS * R + g * R;
    auto at = [&](uint32_t k) { return (uint64_t)cls + (uint64_t)k * p.period; };
    float *gs = smem, *bs = smem + G * E;
    T *ring = reinterpret_cast<T *>(smem + 2 * G * E) + g * (STAGES * R * G * E);
    uint64_t *bar = bars + g * STAGES;
    if (STAGES && row.t == 0) {
        for (int k = 0; k < STAGES; k++) mbar_init(&bar[k], 1);
        fence_barrier_init();
    }
    pdl_wait();
    pdl_launch_dependents();
    // One thread of a group requests its rows' chunks. Rows whose outer chunks may reach past the tensor
    // are copied by the group itself, element by element, when their turn comes.
    auto copied = [&](uint64_t r) { return r < p.rows && (p.period == 1 || !row.ends(r, p.rows)); };
    auto request = [&](uint32_t k, uint32_t st) {
        if (STAGES == 0 || row.t != 0 || at(k) >= p.rows) return;
        const uint32_t bytes = (row.shift + p.d + V - 1) / V * 16;
        uint32_t all = 0;
#pragma unroll
        for (int q = 0; q < R; q++) all += copied(at(k + q)) ? bytes : 0;
        mbar_arrive_expect_tx(&bar[st], all);
#pragma unroll
        for (int q = 0; q < R; q++)
            if (copied(at(k + q))) bulk_load(ring + (st * R + q) * (G * E), x + at(k + q) * p.ldx - row.shift, bytes, &bar[st]);
    };
#pragma unroll
    for (int k = 0; k < STAGES; k++) request(i + k * step, k);
    norm_stage_param<V, G, E>(gs, p.gamma, row.shift, p.d, THREADS);
    norm_stage_param<V, G, E>(bs, p.beta, row.shift, p.d, THREADS);
    __syncthreads();
    const float inv_d = 1.0f / (float)p.d;
    uint32_t st = 0, phases = 0;  // the stage, and a bit a stage: its barrier's parity
    for (uint32_t k = blockIdx.x / p.period * GROUPS * R; at(k) < p.rows; k += step, i += step) {
        const bool mine = at(i) < p.rows;
        if (G == 32 && !mine) break;  // a warp by itself
        float v[R][E];
        if constexpr (STAGES > 0) {
            T *stage = ring + st * (R * G * E);
            if (mine) {
                mbar_wait(&bar[st], phases >> st & 1, JC_DEV_TIMEOUT_FULL);
                phases ^= 1u << st;
#pragma unroll
                for (int q = 0; q < R; q++) {
                    const uint64_t r = at(i + q);
                    if (r >= p.rows || copied(r)) continue;
                    for (uint32_t j = row.t; j < p.d; j += G) stage[q * G * E + row.shift + j] = x[r * p.ldx + j];
                    fence_proxy_async();  // these stores come before the bulk copy that takes the stage next
                }
            }
            if (G == 32)
                __syncwarp();
            else if (p.period > 1)
                __syncthreads();
#pragma unroll
            for (int q = 0; q < R; q++)
#pragma unroll
                for (int c = 0; c < Row::N; c++) {
                    Elem<T, V>::load(stage + q * G * E + row.place(c), v[q] + c * V);
                    row.mask(c, v[q] + c * V);
                }
        } else {
#pragma unroll
            for (int c = 0; c < E; c++)
                v[0][c] = mine && row.place(c) < p.d ? static_cast<float>(x[at(i) * p.ldx + row.place(c)]) : 0.0f;
        }
        float s[R], mean[R], rstd[R];
#pragma unroll
        for (int q = 0; q < R; q++) s[q] = norm_add_up<E>(v[q]);
        norm_sum<G>(s, part);
        if constexpr (STAGES > 0) {
            // The group has read the stage (every lane has added into the sums): the rows STAGES times R
            // further on may take it.
            if (G == 32) __syncwarp();
            request(i + STAGES * step, st);
            st = st + 1 == STAGES ? 0 : st + 1;
        }
#pragma unroll
        for (int q = 0; q < R; q++) {
            mean[q] = s[q] * inv_d;
            const float off[2] = {-mean[q], -mean[q]};
            float sq[2] = {0.0f, 0.0f};
            if constexpr (V == 1) {
#pragma unroll
                for (int c = 0; c < E; c++) {
                    v[q][c] = row.place(c) < p.d ? v[q][c] - mean[q] : 0.0f;
                    sq[c & 1] = fmaf(v[q][c], v[q][c], sq[c & 1]);
                }
            } else {
#pragma unroll
                for (int c = 0; c < Row::N; c++) {
                    float *w = v[q] + c * V;
#pragma unroll
                    for (int e = 0; e < V; e += 2) add2(w + e, w + e, off);
                    row.mask(c, w);
#pragma unroll
                    for (int e = 0; e < V; e += 2) fma2(sq, w + e, w + e, sq);
                }
            }
            s[q] = sq[0] + sq[1];
        }
        norm_sum<G>(s, part);
#pragma unroll
        for (int q = 0; q < R; q++) rstd[q] = rsqrtf(s[q] * inv_d + p.eps);
        if (!mine) continue;
        T *out = static_cast<T *>(p.y) + at(i) * p.ldy;
        const bool two = R == 2 && at(i + 1) < p.rows;
#pragma unroll
        for (int c = 0; c < Row::N; c++) {
            float ga[V], be[V];
            norm_param<V, G, E>(gs, row.place(c), ga);
            norm_param<V, G, E>(bs, row.place(c), be);
#pragma unroll
            for (int q = 0; q < R; q++) {
                float *w = v[q] + c * V;
                T *to = out + (size_t)q * p.period * p.ldy;
                if constexpr (V == 1) {
                    w[0] = fmaf(w[0] * rstd[q], ga[0], be[0]);
                    if (row.place(c) < p.d) to[row.place(c)] = static_cast<T>(w[0]);
                } else {
                    const float by[2] = {rstd[q], rstd[q]};
#pragma unroll
                    for (int e = 0; e < V; e += 2) {
                        mul2(w + e, w + e, by);
                        fma2(w + e, w + e, ga + e, be + e);
                    }
                    if (q == 0 || two) row.store(to, c, w);
                }
            }
        }
        if (p.stats && row.t == 0) {
            *reinterpret_cast<float2 *>(p.stats + 2 * at(i)) = make_float2(mean[0], rstd[0]);
            if (R == 2 && two) *reinterpret_cast<float2 *>(p.stats + 2 * at(i + 1)) = make_float2(mean[R - 1], rstd[R - 1]);
        }
    }
}

struct NormBwdParams {
    const void *dy;
    size_t lddy;
    const void *x;
    size_t ldx;
    const float *gamma, *stats;
    const void *add;
    size_t ldadd;
    uint32_t rows, d, period;
    void *dx;
    size_t lddx;
    float *ws;  // [gridDim.x][2][d]: each block's sums for dgamma and dbeta
    float *dgamma, *dbeta;  // either may be nullptr
    unsigned int *err;
};

// How a block of the backward kernel is made up. Rows of x, dy and add come into shared memory by bulk
// copies, STAGES rows ahead, each group its own; a row is then read twice from there, which leaves the
// registers to the two running sums. Held in registers instead, with the next row's raw elements, a
// row cost 170 registers a thread, and twelve warps a SM moved 4.1 TB/s at 1000 elements a row.
// STAGES 0 (V = 1, and f32 rows too wide for the ring): each pass reads global memory.
template <class T, int V, int G, int E>
struct NormBwdShape {
    static constexpr int ROW = G * E * (int)sizeof(T);  // bytes
    static constexpr int STAGES = V == 1 || ROW > 32768 ? 0 : ROW * 2 > 32768 ? 1 : 2;
    static constexpr int THREADS = G > 512 ? G : STAGES && ROW * (512 / G) * STAGES * 3 > 200000 ? (G > 256 ? G : 256) : 512;
    static constexpr int GROUPS = THREADS / G;
    static constexpr int RING = GROUPS * STAGES * 3 * ROW, SUMS = GROUPS * 2 * G * E * 4;
    static constexpr int SMEM = G * E * 4 + (RING > SUMS ? RING : SUMS);  // gamma, then the ring, later the sums
    static_assert(SMEM <= 227 * 1024 - 1024, "shared memory");
};

// A block's groups keep their sums for dgamma and dbeta in registers over all their rows and add them
// up in shared memory once, group after group; one row of sums a block goes to ws, or, from a block
// alone, to dgamma and dbeta themselves.
template <class T, int V, int G, int E>
__global__ void __launch_bounds__(NormBwdShape<T, V, G, E>::THREADS, 1) norm_bwd_kernel(const NormBwdParams p) {
    using S = NormBwdShape<T, V, G, E>;
    using Row = NormRow<T, V, G, E>;
    constexpr int THREADS = S::THREADS, GROUPS = S::GROUPS, STAGES = S::STAGES;
    __shared__ float part[2 * THREADS / 32];
    __shared__ uint64_t bars[GROUPS * (STAGES ? STAGES : 1)];
    extern __shared__ __align__(16) float smem[];
    dev_err_bind(p.err);
    const uint32_t g = threadIdx.x / G, cls = blockIdx.x % p.period, step = gridDim.x / p.period * GROUPS;
    const T *x = static_cast<const T *>(p.x), *dy = static_cast<const T *>(p.dy), *add = static_cast<const T *>(p.add);
    const Row row(threadIdx.x % G,
                  V == 1 ? 0 : (uint32_t)(reinterpret_cast<uintptr_t>(x + (size_t)cls * p.ldx) % 16 / sizeof(T)), p.d);
    uint32_t i = blockIdx.x / p.period * GROUPS + g;
    auto at = [&](uint32_t k) { return (uint64_t)cls + (uint64_t)k * p.period; };
    uint8_t *ring = reinterpret_cast<uint8_t *>(smem + G * E) + g * (STAGES * 3 * S::ROW);
    uint64_t *bar = bars + g * STAGES;
    if (STAGES && row.t == 0) {
        for (int k = 0; k < STAGES; k++) mbar_init(&bar[k], 1);
        fence_barrier_init();
    }
    pdl_wait();
    pdl_launch_dependents();
    // One thread of a group requests a row's chunks of every tensor. Rows whose outer chunks may reach
    // past the tensor are copied by the group itself, element by element, when their turn comes.
    auto whole_chunks = [&](uint64_t r) { return p.period == 1 || !row.ends(r, p.rows); };
    auto request = [&](uint64_t r, uint32_t st) {
        if (STAGES == 0 || row.t != 0 || r >= p.rows || !whole_chunks(r)) return;
        const uint32_t bytes = (row.shift + p.d + V - 1) / V * 16;
        uint8_t *to = ring + st * (3 * S::ROW);
        mbar_arrive_expect_tx(&bar[st], (p.add ? 3 : 2) * bytes);
        bulk_load(to, x + r * p.ldx - row.shift, bytes, &bar[st]);
        bulk_load(to + S::ROW, dy + r * p.lddy - row.shift, bytes, &bar[st]);
        if (p.add) bulk_load(to + 2 * S::ROW, add + r * p.ldadd - row.shift, bytes, &bar[st]);
    };
#pragma unroll
    for (int k = 0; k < STAGES; k++) request(at(i + k * step), k);
    norm_stage_param<V, G, E>(smem, p.gamma, row.shift, p.d, THREADS);
    float2 next_st = at(i) < p.rows ? *reinterpret_cast<const float2 *>(p.stats + 2 * at(i)) : make_float2(0.0f, 0.0f);
    __syncthreads();  // gamma, and the barriers
    float dg[E], db[E];
#pragma unroll
    for (int e = 0; e < E; e++) dg[e] = db[e] = 0.0f;
    const float inv_d = 1.0f / (float)p.d;
    uint32_t st = 0, phases = 0;  // the stage, and a bit a stage: its barrier's parity
    for (uint32_t k = blockIdx.x / p.period * GROUPS; at(k) < p.rows; k += step, i += step) {
        const uint64_t r = at(i);
        const bool mine = r < p.rows;
        if (G == 32 && !mine) break;  // a warp by itself
        T *stage = reinterpret_cast<T *>(ring + st * (3 * S::ROW));
        constexpr int ELEMS = S::ROW / (int)sizeof(T);
        if constexpr (STAGES > 0) {
            const bool copied = mine && whole_chunks(r);
            if (copied) {
                mbar_wait(&bar[st], phases >> st & 1, JC_DEV_TIMEOUT_FULL);
                phases ^= 1u << st;
            } else if (mine) {
                for (uint32_t j = row.t; j < p.d; j += G) {
                    stage[row.shift + j] = x[r * p.ldx + j];
                    stage[ELEMS + row.shift + j] = dy[r * p.lddy + j];
                    if (p.add) stage[2 * ELEMS + row.shift + j] = add[r * p.ldadd + j];
                }
                fence_proxy_async();  // these stores come before the bulk copies that take the stage next
            }
            if (G == 32)
                __syncwarp();
            else if (p.period > 1)
                __syncthreads();
        }
        // Chunk c of a tensor as f32, 0 outside the row.
        auto get = [&](int which, const T *global, int c, float *v) {
            if constexpr (STAGES > 0) {
                Elem<T, V>::load(stage + which * ELEMS + row.place(c), v);
                row.mask(c, v);
            } else if constexpr (V == 1) {
                v[0] = row.place(c) < p.d ? static_cast<float>(global[row.place(c)]) : 0.0f;
            } else {
                const bool ends = p.period > 1 && row.ends(r, p.rows);
                row.chunk(global, c, ends, v);
            }
        };
        const T *xr = x + r * p.ldx, *dyr = dy + r * p.lddy, *ar = add + r * p.ldadd;
        const float rstd = next_st.y, by[2] = {rstd, rstd}, off[2] = {-next_st.x * rstd, -next_st.x * rstd};
        if (at(i + step) < p.rows) next_st = *reinterpret_cast<const float2 *>(p.stats + 2 * at(i + step));
        constexpr int PER = V == 1 ? 2 : 1, W = V == 1 ? 2 : V;  // chunks, elements worked on together
        float s[2] = {0.0f, 0.0f}, s2[2] = {0.0f, 0.0f};
        if (mine) {
#pragma unroll
            for (int c = 0; c < Row::N; c += PER) {
                float xh[W], u[W], ga[W];
#pragma unroll
                for (int q = 0; q < PER; q++) {
                    get(0, xr, c + q, xh + q);
                    get(1, dyr, c + q, u + q);
                    norm_param<V, G, E>(smem, row.place(c + q), ga + q);
                }
#pragma unroll
                for (int e = 0; e < W; e += 2) {
                    // Outside the row dy and gamma are 0: nothing is added there.
                    const int j = c * V + e;
                    fma2(xh + e, xh + e, by, off);
                    fma2(dg + j, u + e, xh + e, dg + j);
                    add2(db + j, db + j, u + e);
                    mul2(u + e, u + e, ga + e);
                    add2(s, s, u + e);
                    fma2(s2, u + e, xh + e, s2);
                }
            }
        }
        float both[2] = {s[0] + s[1], s2[0] + s2[1]};
        norm_sum<G>(both, part);
        if (G == 32) __syncwarp();  // or the compiler keeps the first pass's f32 values, and spills
        if (mine) {
            // dx = rstd u - rstd (s1 + xh s2) [+ add]
            const float m1 = -both[0] * inv_d * rstd, m2 = -both[1] * inv_d * rstd, a1[2] = {m1, m1}, a2[2] = {m2, m2};
            T *out = static_cast<T *>(p.dx) + r * p.lddx;
#pragma unroll
            for (int c = 0; c < Row::N; c += PER) {
                float o[W], xh[W], u[W], ga[W];
#pragma unroll
                for (int q = 0; q < PER; q++) {
                    get(0, xr, c + q, xh + q);
                    get(1, dyr, c + q, u + q);
                    norm_param<V, G, E>(smem, row.place(c + q), ga + q);
                    if (p.add) get(2, ar, c + q, o + q);
                }
#pragma unroll
                for (int e = 0; e < W; e += 2) {
                    float h[2];
                    fma2(xh + e, xh + e, by, off);
                    mul2(u + e, u + e, ga + e);
                    fma2(h, xh + e, a2, a1);
                    fma2(h, u + e, by, h);
                    if (p.add)
                        add2(o + e, o + e, h);
                    else
                        o[e] = h[0], o[e + 1] = h[1];
                }
                if constexpr (V == 1) {
                    if (row.place(c) < p.d) out[row.place(c)] = static_cast<T>(o[0]);
                    if (row.place(c + 1) < p.d) out[row.place(c + 1)] = static_cast<T>(o[1]);
                } else {
                    row.store(out, c, o);
                }
            }
        }
        if constexpr (STAGES > 0) {
            // The group has read the stage; the row STAGES further on may take it.
            if (G == 32)
                __syncwarp();
            else
                __syncthreads();
            request(at(i + STAGES * step), st);
            st = st + 1 == STAGES ? 0 : st + 1;
        }
    }
    if (!p.dgamma && !p.dbeta) return;
    // Every group's sums into shared memory (chunk order, conflict-free; the rings are empty), then one
    // thread a column.
    __syncthreads();
    float *sums = smem + G * E;
#pragma unroll
    for (int c = 0; c < Row::N; c++) {
        float *a = sums + (size_t)g * 2 * G * E, *b = a + G * E;
        if constexpr (V == 1) {
            a[row.place(c)] = dg[c];
            b[row.place(c)] = db[c];
        } else {
#pragma unroll
            for (int e = 0; e < V; e += 4) {
                const uint32_t at4 = norm_param_at<V, G, E>(row.place(c) + e);
                Elem<float, 4>::store(a + at4, dg + c * V + e);
                Elem<float, 4>::store(b + at4, db + c * V + e);
            }
        }
    }
    __syncthreads();
    const bool alone = gridDim.x == 1;
    float *og = alone ? p.dgamma : p.ws + (size_t)blockIdx.x * 2 * p.d, *ob = alone ? p.dbeta : og + p.d;
    for (uint32_t j = threadIdx.x; j < p.d; j += THREADS) {
        const uint32_t k = norm_param_at<V, G, E>(j + row.shift);
        float a = 0.0f, b = 0.0f;
#pragma unroll 4
        for (int q = 0; q < GROUPS; q++) {
            a += sums[(size_t)(2 * q) * G * E + k];
            b += sums[(size_t)(2 * q + 1) * G * E + k];
        }
        if (og) og[j] = a;
        if (ob) ob[j] = b;
    }
}

// out_a[j] = sum over parts of ws[part][j], j < n, and out_b[j] the same of ws[part][n + j] (either
// may be nullptr): 32 columns a block, 32 threads a column each summing every 32nd part, so that all of
// a column's reads are in flight at once (148 parts of 1536 columns: 3.8 us, 6.7 from cold caches, all latency).
__global__ void __launch_bounds__(1024) column_sum_kernel(const float *ws, uint32_t parts, uint32_t n,
                                                         uint32_t columns, float *out_a, float *out_b) {
    __shared__ float s[32][32];
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t c = threadIdx.x & 31, k = threadIdx.x >> 5, j = blockIdx.x * 32 + c;
    float v = 0.0f;
    if (j < columns)
#pragma unroll 5
        for (uint32_t i = k; i < parts; i += 32) v += ws[(size_t)i * columns + j];
    s[k][c] = v;
    __syncthreads();
    if (k == 0 && j < columns) {
#pragma unroll
        for (int i = 1; i < 32; i++) v += s[i][c];
        if (j < n) {
            if (out_a) out_a[j] = v;
        } else if (out_b) {
            out_b[j - n] = v;
        }
    }
}

}  // namespace jc
