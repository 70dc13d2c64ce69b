// The translation unit of the fine-tuning operators: their kernel templates are instantiated here,
// next to their host launchers (variant choice, launch shape, PDL attribute).
#include "train.h"

#include <algorithm>
#include <cmath>
#include <string>

#include "adamw.cuh"
#include "launch.h"
#include "linear.cuh"
#include "loss.cuh"
#include "norm.cuh"

namespace jc {

static int sm_count() {
    int dev = 0, sms = 148;
    if (cudaGetDevice(&dev) == cudaSuccess)
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    return sms;
}

static bool aligned16(const void *p, size_t ld, size_t size) {
    return (reinterpret_cast<uintptr_t>(p) | (ld * size)) % 16 == 0;
}

// ---------------------------------------------------------------------------------------------
// layer norm

// Calls f<T>() for an element type.
template <class F>
static bool with_type(uint32_t type, F &&f) {
    if (type == JC_F16) return f(__half());
    if (type == JC_BF16) return f(__nv_bfloat16());
    return f(float());
}

template <int N>
using Int = std::integral_constant<int, N>;

// The group that holds a row of d elements: the smallest G x E that does (a warp up to 1024, so
// that no reduction crosses warps, then four warps, then sixteen).
template <class F>
static bool with_group(uint32_t d, F &&f) {
    if (d <= 256) return f(Int<32>(), Int<8>());
    if (d <= 512) return f(Int<32>(), Int<16>());
    if (d <= 768) return f(Int<32>(), Int<24>());
    if (d <= 1024) return f(Int<32>(), Int<32>());
    if (d <= 2048) return f(Int<128>(), Int<16>());
    if (d <= 4096) return f(Int<128>(), Int<32>());
    return f(Int<512>(), Int<32>());
}

bool launch_norm(const NormArgs &a, cudaStream_t s) {
    if (a.rows == 0) return true;
    return with_type(a.type, [&](auto t) {
        using T = decltype(t);
        const bool vec = a.d % VEC<T> == 0 && aligned16(a.x, a.ldx, sizeof(T)) && aligned16(a.y, a.ldy, sizeof(T));
        return with_group(a.d, [&](auto g, auto e) {
            constexpr int G = g, E = e, ROWS = G < 128 ? 128 / G : 1;
            const NormParams p{a.x, a.ldx, a.gamma, a.beta, a.eps, a.rows, a.d, a.y, a.ldy, a.stats};
            const dim3 grid((a.rows + ROWS - 1) / ROWS), block(G < 128 ? 128 : G);
            return vec ? launch_ex(norm_kernel<T, VEC<T>, G, E>, grid, block, 0, s, true, "layer_norm", p)
                       : launch_ex(norm_kernel<T, 1, G, E>, grid, block, 0, s, true, "layer_norm", p);
        });
    });
}

// Blocks of the backward kernel: each leaves a row of partial sums.
static uint32_t norm_bwd_blocks(uint32_t rows, uint32_t d) {
    const uint32_t per = d <= 1024 ? 4 : 1;
    return std::min((rows + per - 1) / per, 148u * 4);
}

size_t norm_bwd_ws_floats(uint32_t rows, uint32_t d) { return (size_t)norm_bwd_blocks(rows, d) * 2 * d; }

static bool launch_column_sum(const float *ws, uint32_t parts, uint32_t n, uint32_t columns, float *a,
                              float *b, cudaStream_t s) {
    return launch_ex(column_sum_kernel, dim3((columns + 31) / 32), dim3(256), 0, s, true, "column sums", ws,
                     parts, n, columns, a, b);
}

bool launch_norm_bwd(const NormBwdArgs &a, cudaStream_t s) {
    const bool sums = a.dgamma || a.dbeta;
    const uint32_t blocks = norm_bwd_blocks(a.rows, a.d);
    if (a.rows > 0) {
        const bool ok = with_type(a.type, [&](auto t) {
            using T = decltype(t);
            const bool vec = a.d % VEC<T> == 0 && aligned16(a.x, a.ldx, sizeof(T)) &&
                             aligned16(a.dy, a.lddy, sizeof(T)) && aligned16(a.dx, a.lddx, sizeof(T)) &&
                             (!a.add || aligned16(a.add, a.ldadd, sizeof(T)));
            return with_group(a.d, [&](auto g, auto e) {
                constexpr int G = g, E = e;
                const NormBwdParams p{a.dy, a.lddy, a.x, a.ldx, a.gamma, a.stats, a.add, a.ldadd, a.rows,
                                      a.d, a.dx, a.lddx, sums ? a.ws : nullptr};
                const dim3 block(G < 128 ? 128 : G);
                const size_t smem = G == 32 ? 2 * (size_t)a.d * sizeof(float) : 0;
                return vec ? launch_ex(norm_bwd_kernel<T, VEC<T>, G, E>, dim3(blocks), block, smem, s, true,
                                       "layer_norm_backward", p)
                           : launch_ex(norm_bwd_kernel<T, 1, G, E>, dim3(blocks), block, smem, s, true,
                                       "layer_norm_backward", p);
            });
        });
        if (!ok) return false;
    }
    return !sums || launch_column_sum(a.ws, blocks, a.d, 2 * a.d, a.dgamma, a.dbeta, s);
}

// ---------------------------------------------------------------------------------------------
// linear

template <class F>
static bool with_half(uint32_t type, F &&f) {
    return type == JC_F16 ? f(__half()) : f(__nv_bfloat16());
}

template <class F>
static bool with_act(uint32_t act, F &&f) {
    if (act == JC_EPI_RELU) return f(std::integral_constant<uint32_t, JC_EPI_RELU>());
    if (act == JC_EPI_GELU) return f(std::integral_constant<uint32_t, JC_EPI_GELU>());
    return f(std::integral_constant<uint32_t, 0>());
}

template <class T>
static bool launch_product(uint32_t act, const LinearParams &p, uint32_t splits, cudaStream_t s) {
    const dim3 grid((p.n + LIN_T - 1) / LIN_T, (p.m + LIN_T - 1) / LIN_T, splits);
    if (grid.y > 65535) {
        set_error("linear: too many rows");
        return false;
    }
    return with_act(act, [&](auto a) {
        return launch_ex(linear_kernel<T, decltype(a)::value>, grid, dim3(256), 0, s, true, "linear", p);
    });
}

bool launch_linear(const LinearArgs &a, cudaStream_t s) {
    if (a.m == 0) return true;
    LinearParams p{};
    p.a = LinearOperand{a.x, a.ldx, 1};
    p.b = LinearOperand{a.w, a.ldw, 1};
    p.m = a.m;
    p.n = a.n;
    p.k = a.k;
    p.bias = a.bias;
    p.res = a.res;
    p.ldres = a.ldres;
    p.c = a.y;
    p.ldc = a.ldy;
    p.z = a.z;
    p.ldz = a.ldz;
    return with_half(a.type, [&](auto t) { return launch_product<decltype(t)>(a.act, p, 1, s); });
}

// The backward pass's workspace: dz (16 bits), the column sums' parts, dw's partial products, each
// from a 256-byte boundary.
struct LinearBwdPlan {
    uint32_t dz_parts, splits;
    size_t lddz, dz_at, part_at, ws_at, bytes;
};

static LinearBwdPlan plan_linear_bwd(uint32_t act, uint32_t m, uint32_t n, uint32_t k) {
    LinearBwdPlan p{};
    auto up = [](size_t v) { return (v + 255) / 256 * 256; };
    p.dz_parts = (m + DZ_ROWS - 1) / DZ_ROWS;
    p.lddz = n;
    p.part_at = act ? up((size_t)m * p.lddz * 2) : 0;
    p.ws_at = p.part_at + up((size_t)p.dz_parts * n * 4);
    const uint64_t tiles = (uint64_t)((n + LIN_T - 1) / LIN_T) * ((k + LIN_T - 1) / LIN_T);
    p.splits = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(std::min<uint64_t>(64, 296 / tiles), m / 64));
    p.bytes = p.ws_at + (p.splits > 1 ? up((size_t)p.splits * n * k * 4) : 0);
    return p;
}

size_t linear_bwd_ws_bytes(uint32_t act, uint32_t m, uint32_t n, uint32_t k) {
    return plan_linear_bwd(act, m, n, k).bytes;
}

bool launch_linear_bwd(const LinearBwdArgs &a, cudaStream_t s) {
    const LinearBwdPlan plan = plan_linear_bwd(a.act, a.m, a.n, a.k);
    uint8_t *ws = static_cast<uint8_t *>(a.ws);
    float *part = reinterpret_cast<float *>(ws + plan.part_at);
    return with_half(a.type, [&](auto t) {
        using T = decltype(t);
        const T *dz = static_cast<const T *>(a.dy);
        size_t lddz = a.lddy;
        const bool need_dz = a.act && (a.dx || a.dw);
        if (a.m > 0 && (need_dz || a.dbias)) {
            T *out = reinterpret_cast<T *>(ws + plan.dz_at);
            const DzParams p{a.dy, a.lddy, a.z, a.ldz, a.m, a.n, out, plan.lddz, a.dbias ? part : nullptr};
            if (a.act) {
                dz = out;
                lddz = plan.lddz;
            }
            const bool vec = a.n % 8 == 0 && aligned16(a.dy, a.lddy, 2) && (!a.act || aligned16(a.z, a.ldz, 2));
            const uint32_t cols = vec ? 256 : 32;
            const dim3 grid((a.n + cols - 1) / cols, plan.dz_parts);
            if (!with_act(a.act, [&](auto act) {
                    constexpr uint32_t ACT = decltype(act)::value;
                    return vec ? launch_ex(linear_dz_kernel<T, ACT, 8>, grid, dim3(256), 0, s, true, "dz", p)
                               : launch_ex(linear_dz_kernel<T, ACT, 1>, grid, dim3(256), 0, s, true, "dz", p);
                }))
                return false;
        }
        if (a.dbias && !launch_column_sum(part, a.m ? plan.dz_parts : 0, a.n, a.n, a.dbias, nullptr, s)) return false;
        if (a.dx && a.m > 0) {
            LinearParams p{};
            p.a = LinearOperand{dz, lddz, 1};
            p.b = LinearOperand{a.w, 1, a.ldw};
            p.m = a.m;
            p.n = a.k;
            p.k = a.n;
            p.c = a.dx;
            p.ldc = a.lddx;
            if (!launch_product<T>(0, p, 1, s)) return false;
        }
        if (a.dw) {
            LinearParams p{};
            p.a = LinearOperand{dz, 1, lddz};
            p.b = LinearOperand{a.x, 1, a.ldx};
            p.m = a.n;
            p.n = a.k;
            p.k = a.m;
            p.c = a.dw;
            p.ldc = a.lddw;
            p.ws = plan.splits > 1 ? reinterpret_cast<float *>(ws + plan.ws_at) : nullptr;
            if (!launch_product<T>(0, p, plan.splits, s)) return false;
            if (p.ws) {
                const size_t all = (size_t)a.n * a.k;
                const uint32_t blocks = (uint32_t)std::min<size_t>((all + 255) / 256, 148 * 8);
                if (!launch_ex(linear_join_kernel<T>, dim3(blocks), dim3(256), 0, s, true, "linear join",
                               (const float *)p.ws, plan.splits, a.n, a.k, static_cast<T *>(a.dw), a.lddw))
                    return false;
            }
        }
        return true;
    });
}

// ---------------------------------------------------------------------------------------------
// loss and optimizer

bool launch_choice_loss(const LossArgs &a, cudaStream_t s) {
    if (a.requests == 0) return true;
    unsigned int *err = module_error_word();
    if (!err) return false;
    const LossParams p{a.logits, a.n_logits, a.offsets, a.gold, a.weight, a.requests, a.loss, a.dlogits, err};
    return launch_ex(choice_loss_kernel, dim3((a.requests + 3) / 4), dim3(128), 0, s, true, "choice_loss", p);
}

bool launch_adamw(const AdamwStep &a, cudaStream_t s) {
    if (a.n_chunks == 0) return true;
    AdamwParams p{};
    p.tensors = a.tensors;
    p.chunks = a.chunks;
    p.grad_scale = a.grad_scale;
    p.beta1 = (float)a.beta1;
    p.beta2 = (float)a.beta2;
    p.one_minus_beta1 = (float)(1.0 - a.beta1);
    p.one_minus_beta2 = (float)(1.0 - a.beta2);
    p.lr = a.lr;
    p.eps = a.eps;
    p.inv_bias1 = (float)(1.0 / (1.0 - std::pow(a.beta1, (double)a.step)));
    p.inv_bias2 = (float)(1.0 / (1.0 - std::pow(a.beta2, (double)a.step)));
    return a.bits == 8 ? launch_ex(adamw_kernel<8>, dim3(a.n_chunks), dim3(ADAMW_THREADS), 0, s, true, "adamw", p)
                       : launch_ex(adamw_kernel<32>, dim3(a.n_chunks), dim3(ADAMW_THREADS), 0, s, true, "adamw", p);
}

}  // namespace jc
