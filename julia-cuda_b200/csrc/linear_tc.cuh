// The linear layer's products on the tensor cores: c [m][n] = a b^T, a [m][k], b [n][k] of one 16-bit
// type, f32 accumulators in tensor memory (tcgen05.mma, kind::f16).
//
// The three products of a training step differ in which axis of their operands is contiguous:
//   forward   y  = x w^T    contracts over k, contiguous in both
//   dx        dx = dz w     contracts over n: contiguous in dz, the row axis of w
//   dw        dw = dz^T x   contracts over m: the row axis of both
// An operand whose contiguous axis is not the contracted one needs no transposed copy: it is loaded
// as it lies, in blocks of 64 (contiguous) x 64 (contracted), and its shared-memory descriptor says
// so ("MN-major").
//
// Operands come by TMA, whose rows start on 16-byte boundaries; others are laid out so first
// (linear_pad_kernel). One CTA per SM walks the tiles: a warp loads, one issues the MMAs, eight run the
// epilogue of one tile under the main loop of the next (two accumulators). CTAS 2: pairs of CTAs on 256 x
// BN tiles (cta_group::2), each with 128 rows of a and half of the rows of b, for a third fewer operand
// bytes per SM than a 128 x 256 tile: alone, such a tile asks an SM for 48 KB per 512 tensor cycles, more
// than the 64 bytes a cycle it can take in. The two products of the backward pass, whose second operands
// lie alike, are one launch (GRADS): dw's few long items first, dx's many short ones after them, so no SM
// waits for the other product's last tiles and dw's partial sums go out under dx's main loop.
//
// Bound by the matrix rate: 12288 x 2048 x 768 bf16, inputs in L2, takes 27.7 us (1.40 PFLOP/s, 85% of the
// measured burst rate; a library product of that shape 28.4), 30.2 with bias and residual; from memory
// 38. Its 144 tiles are two rounds of 72 pairs; what is left is the clock under load, the first tiles'
// loads and the last epilogue. Short contractions are bound by the epilogue: 12288 x 768 x 2048 with
// GELU and z 52 us in short bursts, where its operations would take 24.
#pragma once
#include <type_traits>

#include "common.cuh"
#include "elem.cuh"
#include "linear.cuh"

namespace jc {

constexpr int LT_BM = 128, LT_BK = 64;
constexpr int LT_EPI_WARPS = 8;
constexpr int LT_STAGE_BUF = 4096;  // a warp's staging tile: 32 rows x 128 bytes

// The instruction descriptor: umma_idesc_f16 with the operands' type and major axes.
template <class T>
__host__ __device__ constexpr uint32_t lt_idesc(int m, int n, bool a_mn, bool b_mn) {
    const uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    return umma_idesc_f16(m, n) | (fmt << 7) | (fmt << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16);
}

// Shared-memory descriptor of an operand tile at saddr (1024-byte aligned), 128-byte swizzle.
//   K-major:  rows of 64 contracted elements (128 bytes), 8-row groups 1024 bytes apart.
//   MN-major: blocks of 64 rows of the contracted axis x 64 elements of the other (8 KB); the next
//             8 contracted rows 1024 bytes on, the next 64 of the other axis a block on.
__device__ __forceinline__ uint64_t lt_desc(uint32_t saddr, bool MN) {
    uint64_t d = umma_desc_sw128(saddr);
    if (MN) d = (d & ~((uint64_t)0x3FFF << 16)) | ((uint64_t)(8192 >> 4) << 16);
    return d;
}

// Descriptor step (16-byte units) for the next 16 contracted elements: 32 bytes inside a row, or 16
// rows on.
__device__ __forceinline__ uint32_t lt_step(bool MN) { return MN ? (16 * 128) >> 4 : 32 >> 4; }

struct LinearTcParams {
    uint32_t m, n, k;
    const float *bias;
    const void *res;
    size_t ldres;
    void *c;
    size_t ldc;
    void *z;
    size_t ldz;
    float *ws;        // split over k: [splits][m][n] partial sums instead of c
    uint32_t splits;
    uint32_t tiles_m, tiles_n;
};

// One product, or (GRADS) dw's and dx's, dw's a MN-major. Items of the second follow the first's.
struct LinearTcKernelParams {
    CUtensorMap map_a[2], map_b[2];
    LinearTcParams p[2];
    uint32_t items[2];
    unsigned int *err;
};

template <int BN>
struct LtShape {
    static constexpr int CW = BN / 2 < 64 ? BN / 2 : 64;  // columns of an epilogue chunk
    static constexpr int CHUNKS = BN / 2 / CW;            // chunks of a warp: half of the columns
};

// ---------------------------------------------------------------------------------------------
// epilogue

// Moves a warp's 32 x CW tile between global memory and its staging buffer (rows of 128 bytes, 16-byte
// chunk c of row r at chunk c ^ (r % 8), so that both a lane's own row and eight lanes to a row are
// free of bank conflicts). VEC: global rows are on 16-byte boundaries; r0, c0: the tile's place; W:
// bytes of an element.
template <int CW, int W, bool VEC>
__device__ __forceinline__ void lt_copy_out(const uint8_t *buf, uint8_t *g, size_t ld, uint32_t r0,
                                            uint32_t c0, uint32_t rows, uint32_t cols) {
    const uint32_t lane = threadIdx.x & 31;
    if constexpr (VEC) {
        constexpr int PER = CW * W / 16, STEP = 32 / PER;  // 16-byte chunks a row, rows a pass
        const uint32_t c = lane % PER;
        const uint32_t left = c0 + c * (16 / W) < cols && r0 < rows ? rows - r0 : 0;  // rows this lane writes
        uint8_t *d = g + ((size_t)(r0 + lane / PER) * ld + c0) * W + c * 16;
#pragma unroll
        for (int i = 0; i < 32 / STEP; i++, d += (size_t)STEP * ld * W) {
            const uint32_t r = i * STEP + lane / PER;
            const uint4 v = *reinterpret_cast<const uint4 *>(buf + r * 128 + ((c ^ (r & 7)) << 4));
            if (r < left) *reinterpret_cast<uint4 *>(d) = v;
        }
    } else {
        for (uint32_t e = lane; e < 32u * CW; e += 32) {
            const uint32_t r = e / CW, c = e % CW, at = c * W;
            const uint8_t *s = buf + r * 128 + (((at >> 4) ^ (r & 7)) << 4) + (at & 15);
            uint8_t *d = g + ((size_t)(r0 + r) * ld + c0 + c) * W;
            if (r0 + r < rows && c0 + c < cols) {
                if constexpr (W == 2)
                    *reinterpret_cast<uint16_t *>(d) = *reinterpret_cast<const uint16_t *>(s);
                else
                    *reinterpret_cast<uint32_t *>(d) = *reinterpret_cast<const uint32_t *>(s);
            }
        }
    }
}

// The 16-byte chunks lt_copy_out would write, brought into the buffer instead, asynchronously: the
// residual waits there rather than in registers, which it made spill (lt_res_wait, then __syncwarp).
template <int CW>
__device__ __forceinline__ void lt_res_request(uint8_t *buf, const uint8_t *g, size_t ld, uint32_t r0, uint32_t c0,
                                               uint32_t rows, uint32_t cols) {
    constexpr int PER = CW * 2 / 16, STEP = 32 / PER;
    const uint32_t lane = threadIdx.x & 31, c = lane % PER;
    const uint32_t left = c0 + c * 8 < cols && r0 < rows ? rows - r0 : 0;
    const uint8_t *s = g + ((size_t)(r0 + lane / PER) * ld + c0) * 2 + c * 16;
#pragma unroll
    for (int i = 0; i < 32 / STEP; i++, s += (size_t)STEP * ld * 2) {
        const uint32_t r = i * STEP + lane / PER;
        if (r < left)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(buf + r * 128 + ((c ^ (r & 7)) << 4))),
                         "l"(s)
                         : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
}
__device__ __forceinline__ void lt_res_wait() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }

// Any alignment: element by element into the buffer.
template <int CW>
__device__ __forceinline__ void lt_copy_in(uint8_t *buf, const uint8_t *g, size_t ld, uint32_t r0, uint32_t c0,
                                           uint32_t rows, uint32_t cols) {
    for (uint32_t e = threadIdx.x & 31; e < 32u * CW; e += 32) {
        const uint32_t r = e / CW, c = e % CW, at = c * 2;
        uint16_t v = 0;
        if (r0 + r < rows && c0 + c < cols)
            v = *reinterpret_cast<const uint16_t *>(g + ((size_t)(r0 + r) * ld + c0 + c) * 2);
        *reinterpret_cast<uint16_t *>(buf + r * 128 + (((at >> 4) ^ (r & 7)) << 4) + (at & 15)) = v;
    }
}

// A chunk's bias: requested early, a lane or two columns each, and passed round the warp. Read from global
// memory where it is used, each of those reads would wait for the one before it: 3.4 us a tile.
template <int CW>
struct LtBias {
    float v[CW / 32];
    __device__ __forceinline__ void load(const float *bias, uint32_t c0, uint32_t n) {
#pragma unroll
        for (int i = 0; i < CW / 32; i++) {
            const uint32_t c = c0 + 32 * i + (threadIdx.x & 31);
            v[i] = bias && c < n ? __ldg(bias + c) : 0.0f;
        }
    }
    __device__ __forceinline__ void add(float *acc) const {
#pragma unroll
        for (int j = 0; j < CW; j++) acc[j] += __shfl_sync(0xffffffffu, v[j / 32], j & 31);
    }
};

// A lane's own row of the buffer, written or read eight elements at a time.
template <class T, int CW>
__device__ __forceinline__ void lt_put_row(uint8_t *buf, const float *v) {
    const uint32_t r = threadIdx.x & 31;
#pragma unroll
    for (int c = 0; c < CW / 8; c++)
        Elem<T, 8>::store(reinterpret_cast<T *>(buf + r * 128 + ((c ^ (r & 7)) << 4)), v + 8 * c);
}

template <class T, int CW>
__device__ __forceinline__ void lt_add_row(const uint8_t *buf, float *v) {
    const uint32_t r = threadIdx.x & 31;
#pragma unroll
    for (int c = 0; c < CW / 8; c++) {
        float t[8];
        Elem<T, 8>::load(reinterpret_cast<const T *>(buf + r * 128 + ((c ^ (r & 7)) << 4)), t);
#pragma unroll
        for (int i = 0; i < 8; i++) v[8 * c + i] += t[i];
    }
}

// CW columns of this lane's accumulator row.
template <int CW>
__device__ __forceinline__ void lt_acc(uint32_t taddr, float *v) {
#pragma unroll
    for (int i = 0; i < CW; i += 32) tmem_ld32(taddr + i, *reinterpret_cast<float(*)[32]>(v + i));
    tc_wait_ld();
}

// One warp's share of a finished tile: rows 32 (warp % 4).. and half warp / 4 of the columns. `acc`:
// the tile's accumulator; `bias`: the first chunk's. Its residual, too, was requested before the
// accumulator was ready, into the buffer (VEC; where z does not go through the buffer first).
// GRADS: partial sums or plain values, nothing added.
template <class T, int BN, bool GRADS, uint32_t ACT, bool VEC>
__device__ __forceinline__ void lt_epilogue(const LinearTcParams &p, uint32_t acc, uint8_t *buf, uint32_t warp,
                                            uint32_t m0, uint32_t n0, uint32_t split,
                                            LtBias<LtShape<BN>::CW> &bias) {
    using S = LtShape<BN>;
    constexpr int CW = S::CW;
    const uint32_t r0 = m0 + 32 * (warp & 3);
    const uint32_t lane_acc = acc + ((32 * (warp & 3)) << 16);
#pragma unroll 1
    for (int ch = 0; ch < S::CHUNKS; ch++) {
        const uint32_t cc = (warp >> 2) * (BN / 2) + ch * CW, c0 = n0 + cc;
        float v[CW];
        lt_acc<CW>(lane_acc + cc, v);
        if (GRADS && p.ws) {
            // Partial sums, f32, 32 columns (128 bytes) at a time.
            uint8_t *ws = reinterpret_cast<uint8_t *>(p.ws + (size_t)split * p.m * p.n);
            constexpr int PW = 32;
#pragma unroll
            for (int h = 0; h < CW / PW; h++) {
                const uint32_t r = threadIdx.x & 31;
                __syncwarp();
#pragma unroll
                for (int c = 0; c < PW / 4; c++)
                    *reinterpret_cast<float4 *>(buf + r * 128 + ((c ^ (r & 7)) << 4)) =
                        make_float4(v[h * PW + 4 * c], v[h * PW + 4 * c + 1], v[h * PW + 4 * c + 2], v[h * PW + 4 * c + 3]);
                __syncwarp();
                lt_copy_out<PW, 4, VEC>(buf, ws, p.n, r0, c0 + h * PW, p.m, p.n);
            }
            continue;
        }
        if (!GRADS && p.bias) {
            bias.add(v);
            if (ch + 1 < S::CHUNKS) bias.load(p.bias, c0 + CW, p.n);
        }
        if (!GRADS && p.z) {
            __syncwarp();
            lt_put_row<T, CW>(buf, v);
            __syncwarp();
            lt_copy_out<CW, 2, VEC>(buf, static_cast<uint8_t *>(p.z), p.ldz, r0, c0, p.m, p.n);
            __syncwarp();
            if (VEC && p.res) lt_res_request<CW>(buf, static_cast<const uint8_t *>(p.res), p.ldres, r0, c0, p.m, p.n);
        }
        if constexpr (ACT != 0) {
#pragma unroll
            for (int j = 0; j < CW; j++) v[j] = act_fwd<ACT>(v[j]);
        }
        if (!GRADS && p.res) {
            if constexpr (VEC)
                lt_res_wait();
            else
                lt_copy_in<CW>(buf, static_cast<const uint8_t *>(p.res), p.ldres, r0, c0, p.m, p.n);
            __syncwarp();
            lt_add_row<T, CW>(buf, v);
        }
        lt_put_row<T, CW>(buf, v);  // a lane's own row: read above, if anything, by the lane itself
        __syncwarp();
        lt_copy_out<CW, 2, VEC>(buf, static_cast<uint8_t *>(p.c), p.ldc, r0, c0, p.m, p.n);
        __syncwarp();
        if (!GRADS && VEC && p.res && !p.z && ch + 1 < S::CHUNKS)
            lt_res_request<CW>(buf, static_cast<const uint8_t *>(p.res), p.ldres, r0, c0 + CW, p.m, p.n);
    }
}

// ---------------------------------------------------------------------------------------------
// TMA kernel

// An operand's tile of one stage: rows [row0, row0 + ROWS) x the 64 contracted from k0. CTAS 2: `bar`
// is the leader's barrier.
template <int CTAS, int ROWS, bool MN>
__device__ __forceinline__ void lt_tma(uint8_t *dst, const CUtensorMap *map, uint64_t *bar, uint32_t leader_bar,
                                       uint32_t row0, uint32_t k0) {
#pragma unroll
    for (int j = 0; j < (MN ? ROWS / 64 : 1); j++) {
        const int32_t x = (int32_t)(MN ? row0 + 64 * j : k0), y = (int32_t)(MN ? k0 : row0);
        if constexpr (CTAS == 2)
            tma_load_2d_pair(dst + j * 8192, map, leader_bar, x, y);
        else
            tma_load_2d(dst + j * 8192, map, bar, x, y);
    }
}

template <int BN, int CTAS>
struct LtTcSmem {
    static constexpr int A_BYTES = LT_BM * 128, B_BYTES = BN / CTAS * 128, STAGE = A_BYTES + B_BYTES;
    static constexpr int STAGES = 196608 / STAGE < 8 ? 196608 / STAGE : 8;
    static constexpr int BYTES = STAGES * STAGE + LT_EPI_WARPS * LT_STAGE_BUF + 256 + 1024;
};

constexpr int LT_TC_THREADS = 32 * (LT_EPI_WARPS + 2);

template <class T, int BN, int CTAS, bool GRADS, uint32_t ACT, bool VEC>
__global__ void __launch_bounds__(LT_TC_THREADS, 1)
    linear_tc_kernel(const __grid_constant__ LinearTcKernelParams kp) {
    using S = LtShape<BN>;
    using M = LtTcSmem<BN, CTAS>;
    constexpr int STAGES = M::STAGES;
    constexpr bool B_MN = GRADS;
    dev_err_bind(kp.err);
    extern __shared__ uint8_t smem_raw[];
    uint8_t *base = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *bufs = base + STAGES * M::STAGE;
    uint64_t *full = reinterpret_cast<uint64_t *>(bufs + LT_EPI_WARPS * LT_STAGE_BUF);
    uint64_t *empty = full + STAGES, *acc_full = empty + STAGES, *acc_empty = acc_full + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(acc_empty + 2);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = CTAS == 2 ? cluster_rank() : 0, unit = blockIdx.x / CTAS, units = gridDim.x / CTAS;
    constexpr uint32_t COLS = 2 * BN;
    if (threadIdx.x == 0) {
        // Pairs: the leader's producer arms a stage for both CTAs' bytes, and its commits release it,
        // and hand over an accumulator, in both.
        for (int s = 0; s < STAGES; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&acc_full[i], 1);
            mbar_init(&acc_empty[i], CTAS * LT_EPI_WARPS);
        }
        fence_barrier_init();
    }
    if (warp == LT_EPI_WARPS + 1) {
        if constexpr (CTAS == 2)
            tmem_alloc_pair(tmem_slot, COLS);
        else
            tmem_alloc(tmem_slot, COLS);
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (CTAS == 2) {
        cluster_arrive();  // both CTAs' barriers are ready before either signals the other
        cluster_wait();
    }
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_wait();
    pdl_launch_dependents();

    // Item i: which product (w), its tile's first column and row, its split and its k-blocks.
    struct Item {
        uint32_t w, n0, m0, z, k0, k1;
    };
    const uint32_t items = kp.items[0] + (GRADS ? kp.items[1] : 0);
    auto item = [&](uint32_t i) {
        Item e;
        e.w = GRADS && i >= kp.items[0];
        const LinearTcParams &p = kp.p[e.w];
        const uint32_t j = e.w ? i - kp.items[0] : i, tiles = p.tiles_m * p.tiles_n, t = j % tiles;
        const uint32_t blocks = (p.k + LT_BK - 1) / LT_BK;
        e.z = j / tiles;
        e.n0 = t % p.tiles_n * BN;
        e.m0 = (t / p.tiles_n * CTAS + rank) * LT_BM;
        e.k0 = (uint32_t)((uint64_t)blocks * e.z / p.splits);
        e.k1 = (uint32_t)((uint64_t)blocks * (e.z + 1) / p.splits);
        return e;
    };
    if (warp == LT_EPI_WARPS) {
        if (lane == 0) {
            const uint32_t leader = CTAS == 2 ? map_to_rank(smem_u32(full), 0) : 0;
            uint32_t it = 0;
            bool ok = true;
            for (uint32_t i = unit; ok && i < items; i += units) {
                const Item e = item(i);
                const CUtensorMap *map_a = &kp.map_a[e.w], *map_b = &kp.map_b[e.w];
                for (uint32_t kb = e.k0; kb < e.k1; kb++, it++) {
                    const uint32_t s = it % STAGES, round = it / STAGES;
                    if (round > 0 && !mbar_wait(&empty[s], (round & 1) ^ 1, JC_DEV_TIMEOUT_EMPTY)) {
                        ok = false;
                        break;
                    }
                    uint8_t *st = base + s * M::STAGE;
                    if (rank == 0) mbar_arrive_expect_tx(&full[s], CTAS * M::STAGE);
                    if (GRADS && e.w == 0)
                        lt_tma<CTAS, LT_BM, true>(st, map_a, &full[s], leader + s * 8, e.m0, kb * LT_BK);
                    else
                        lt_tma<CTAS, LT_BM, false>(st, map_a, &full[s], leader + s * 8, e.m0, kb * LT_BK);
                    lt_tma<CTAS, BN / CTAS, B_MN>(st + M::A_BYTES, map_b, &full[s], leader + s * 8,
                                                  e.n0 + rank * (BN / CTAS), kb * LT_BK);
                }
            }
            // Every stage in use is released before the CTA may leave: all its copies have landed and
            // (pairs) the leader's last commits have arrived.
            for (uint32_t j = it > STAGES ? it - STAGES : 0; j < it; j++)
                if (!mbar_wait(&empty[j % STAGES], (j / STAGES) & 1, JC_DEV_TIMEOUT_EMPTY)) break;
        }
    } else if (warp == LT_EPI_WARPS + 1) {
        if (lane == 0 && rank == 0) {
            uint32_t it = 0, done = 0;
            bool ok = true;
            for (uint32_t i = unit; ok && i < items; i += units, done++) {
                const Item e = item(i);
                const bool a_mn = GRADS && e.w == 0;
                const uint32_t idesc = lt_idesc<T>(CTAS * LT_BM, BN, a_mn, B_MN), a_step = lt_step(a_mn), b_step = lt_step(B_MN);
                const uint32_t buf = done & 1, use = done >> 1;
                if (use > 0 && !mbar_wait(&acc_empty[buf], (use & 1) ^ 1, JC_DEV_TIMEOUT_MMA)) break;
                tc_fence_after();
                const uint32_t acc = tmem + buf * BN;
                for (uint32_t kb = e.k0; kb < e.k1; kb++, it++) {
                    const uint32_t s = it % STAGES;
                    if (!mbar_wait(&full[s], (it / STAGES) & 1, JC_DEV_TIMEOUT_FULL)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint64_t ad = lt_desc(smem_u32(base + s * M::STAGE), a_mn);
                    const uint64_t bd = lt_desc(smem_u32(base + s * M::STAGE + M::A_BYTES), B_MN);
#pragma unroll
                    for (int kk = 0; kk < LT_BK / 16; kk++) {
                        if constexpr (CTAS == 2)
                            tc_mma_f16_pair(acc, ad + kk * a_step, bd + kk * b_step, idesc, kb > e.k0 || kk > 0);
                        else
                            tc_mma_f16(acc, ad + kk * a_step, bd + kk * b_step, idesc, kb > e.k0 || kk > 0);
                    }
                    if constexpr (CTAS == 2)
                        tc_commit_pair(&empty[s]);
                    else
                        tc_commit(&empty[s]);
                }
                if constexpr (CTAS == 2)
                    tc_commit_pair(&acc_full[buf]);
                else
                    tc_commit(&acc_full[buf]);
            }
        }
    } else {
        uint8_t *buf = bufs + warp * LT_STAGE_BUF;
        const uint32_t leader = CTAS == 2 ? map_to_rank(smem_u32(acc_empty), 0) : 0;
        LtBias<S::CW> bias;
        uint32_t done = 0;
        for (uint32_t i = unit; i < items; i += units, done++) {
            const Item e = item(i);
            const LinearTcParams &p = kp.p[e.w];
            // The first chunk's bias and residual are on their way while the accumulator is being summed.
            if (!GRADS) bias.load(p.bias, e.n0 + (warp >> 2) * (BN / 2), p.n);
            if (!GRADS && VEC && p.res && !p.z)
                lt_res_request<S::CW>(buf, static_cast<const uint8_t *>(p.res), p.ldres, e.m0 + 32 * (warp & 3),
                                      e.n0 + (warp >> 2) * (BN / 2), p.m, p.n);
            if (!mbar_wait_sleep(&acc_full[done & 1], (done >> 1) & 1, JC_DEV_TIMEOUT_MMA)) break;
            tc_fence_after();
            lt_epilogue<T, BN, GRADS, ACT, VEC>(p, tmem + (done & 1) * BN, buf, warp, e.m0, e.n0, e.z, bias);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (rank == 0)
                    mbar_arrive(&acc_empty[done & 1]);
                else
                    mbar_arrive_remote(leader + (done & 1) * 8);
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if constexpr (CTAS == 2) {
        cluster_arrive();  // every MMA into either CTA's accumulators is done and read
        cluster_wait();
    }
    if (warp == LT_EPI_WARPS + 1) {
        tc_fence_after();
        if constexpr (CTAS == 2)
            tmem_dealloc_pair(tmem, COLS);
        else
            tmem_dealloc(tmem, COLS);
    }
}

}  // namespace jc
