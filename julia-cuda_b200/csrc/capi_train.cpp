// The C ABI of the fine-tuning operators (include/julia_cuda.h): argument checks and the optimizer's
// handle over the launchers of train.cu.
#include <cuda_runtime.h>

#include <cmath>
#include <memory>
#include <string>
#include <vector>

#include "../../include/julia_cuda.h"
#include "capi_guard.h"
#include "train.h"

using jc::guarded;

namespace {

int fail(const std::string &msg) {
    jc::set_error(msg);
    return -1;
}

size_t type_size(uint32_t type) { return type == JC_F32 ? 4 : 2; }

bool misaligned(const void *p, size_t size) { return reinterpret_cast<uintptr_t>(p) % size != 0; }

// A matrix argument: there, on whole elements, rows no closer than their width.
bool check_matrix(const char *op, const char *name, const void *p, size_t ld, uint32_t width, size_t size,
                  bool needed) {
    std::string why;
    if (!p && needed) why = " is null";
    if (p && misaligned(p, size)) why = " is not aligned to its elements";
    if (p && ld < width) why = "'s rows overlap";
    if (why.empty()) return true;
    jc::set_error(std::string(op) + ": " + name + why);
    return false;
}

bool check_vector(const char *op, const char *name, const void *p, size_t align, bool needed) {
    if ((p || !needed) && !misaligned(p, align)) return true;
    jc::set_error(std::string(op) + ": " + name + (p ? " is misaligned" : " is null"));
    return false;
}

bool check_act(const char *op, uint32_t type, uint32_t act) {
    if (type != JC_F16 && type != JC_BF16)
        jc::set_error(std::string(op) + ": type must be JC_F16 or JC_BF16");
    else if (act != 0 && act != JC_EPI_RELU && act != JC_EPI_GELU)
        jc::set_error(std::string(op) + ": act must be 0, JC_EPI_RELU or JC_EPI_GELU");
    else
        return true;
    return false;
}

// Kernels count rows in 32 bits and step past the last one, and TMA's coordinates are signed.
constexpr uint32_t MAX_SIZE = 0x7FFFFFFFu;

bool check_norm(const char *op, uint32_t type, uint32_t rows, uint32_t d) {
    if (type > JC_F32)
        jc::set_error(std::string(op) + ": unknown element type");
    else if (rows > MAX_SIZE)
        jc::set_error(std::string(op) + ": at most 2^31 - 1 rows");
    else if (d == 0 || d > 16384)
        jc::set_error(std::string(op) + ": rows of 1 to 16384 elements");
    else
        return true;
    return false;
}

bool check_sizes(const char *op, uint32_t m, uint32_t n, uint32_t k) {
    if (n == 0 || k == 0)
        jc::set_error(std::string(op) + ": n and k must not be 0");
    else if (m > MAX_SIZE || n > MAX_SIZE || k > MAX_SIZE)
        jc::set_error(std::string(op) + ": m, n and k are at most 2^31 - 1");
    else
        return true;
    return false;
}

}  // namespace

struct JcAdamW {
    jc::AdamwTensor *tensors = nullptr;
    uint2 *chunks = nullptr;
    uint32_t n_chunks = 0, bits = 32;
    int device = 0;
    ~JcAdamW() {
        cudaFree(tensors);
        cudaFree(chunks);
    }
};

extern "C" {

int jc_layer_norm(uint32_t type, const void *x, size_t ldx, const float *gamma, const float *beta,
                  float eps, uint32_t rows, uint32_t d, void *y, size_t ldy, float *stats, void *stream) {
    return guarded(nullptr, 0, [&]() -> int {
        const char *op = "layer_norm";
        const bool any = rows > 0;
        if (!check_norm(op, type, rows, d)) return -1;
        if (!(eps >= 0.0f) || std::isinf(eps)) return fail("layer_norm: eps must be finite and not negative");
        const size_t size = type_size(type);
        if (!check_matrix(op, "x", x, ldx, d, size, any) || !check_matrix(op, "y", y, ldy, d, size, any) ||
            !check_vector(op, "gamma", gamma, 4, true) || !check_vector(op, "beta", beta, 4, false) ||
            !check_vector(op, "stats", stats, 8, false))
            return -1;
        jc::NormArgs a;
        a.type = type;
        a.x = x;
        a.ldx = ldx;
        a.gamma = gamma;
        a.beta = beta;
        a.eps = eps;
        a.rows = rows;
        a.d = d;
        a.y = y;
        a.ldy = ldy;
        a.stats = stats;
        return jc::launch_norm(a, (cudaStream_t)stream) ? 0 : -1;
    });
}

size_t jc_layer_norm_ws_floats(uint32_t rows, uint32_t d) { return jc::norm_bwd_ws_floats(rows, d); }

int jc_layer_norm_backward(uint32_t type, const void *dy, size_t lddy, const void *x, size_t ldx,
                           const float *gamma, const float *stats, const void *add, size_t ldadd,
                           uint32_t rows, uint32_t d, void *dx, size_t lddx, float *dgamma, float *dbeta,
                           float *ws, void *stream) {
    return guarded(nullptr, 0, [&]() -> int {
        const char *op = "layer_norm_backward";
        const bool any = rows > 0;
        if (!check_norm(op, type, rows, d)) return -1;
        const size_t size = type_size(type);
        if (!check_matrix(op, "dy", dy, lddy, d, size, any) || !check_matrix(op, "x", x, ldx, d, size, any) ||
            !check_matrix(op, "add", add, ldadd, d, size, false) ||
            !check_matrix(op, "dx", dx, lddx, d, size, any) || !check_vector(op, "gamma", gamma, 4, true) ||
            !check_vector(op, "stats", stats, 8, any) || !check_vector(op, "dgamma", dgamma, 4, false) ||
            !check_vector(op, "dbeta", dbeta, 4, false) ||
            !check_vector(op, "ws", ws, 16, (dgamma || dbeta) && jc::norm_bwd_ws_floats(rows, d) > 0))
            return -1;
        jc::NormBwdArgs a;
        a.type = type;
        a.dy = dy;
        a.lddy = lddy;
        a.x = x;
        a.ldx = ldx;
        a.gamma = gamma;
        a.stats = stats;
        a.add = add;
        a.ldadd = ldadd;
        a.rows = rows;
        a.d = d;
        a.dx = dx;
        a.lddx = lddx;
        a.dgamma = dgamma;
        a.dbeta = dbeta;
        a.ws = ws;
        return jc::launch_norm_bwd(a, (cudaStream_t)stream) ? 0 : -1;
    });
}

int jc_linear(uint32_t type, uint32_t act, const void *x, size_t ldx, const void *w, size_t ldw,
              const float *bias, const void *res, size_t ldres, void *y, size_t ldy, void *z, size_t ldz,
              uint32_t m, uint32_t n, uint32_t k, void *ws, void *stream) {
    return guarded(nullptr, 0, [&]() -> int {
        const char *op = "linear";
        const bool any = m > 0;
        if (!check_act(op, type, act)) return -1;
        if (!check_sizes(op, m, n, k)) return -1;
        if (!check_matrix(op, "x", x, ldx, k, 2, any) || !check_matrix(op, "w", w, ldw, k, 2, true) ||
            !check_vector(op, "bias", bias, 4, false) || !check_matrix(op, "res", res, ldres, n, 2, false) ||
            !check_matrix(op, "y", y, ldy, n, 2, any) || !check_matrix(op, "z", z, ldz, n, 2, false) ||
            !check_vector(op, "ws", ws, 256, any && !ws && jc::linear_ws_bytes(x, ldx, w, ldw, m, n, k) > 0))
            return -1;
        jc::LinearArgs a;
        a.ws = ws;
        a.type = type;
        a.act = act;
        a.x = x;
        a.ldx = ldx;
        a.w = w;
        a.ldw = ldw;
        a.bias = bias;
        a.res = res;
        a.ldres = ldres;
        a.y = y;
        a.ldy = ldy;
        a.z = z;
        a.ldz = ldz;
        a.m = m;
        a.n = n;
        a.k = k;
        return jc::launch_linear(a, (cudaStream_t)stream) ? 0 : -1;
    });
}

size_t jc_linear_ws_bytes(const void *x, size_t ldx, const void *w, size_t ldw, uint32_t m, uint32_t n, uint32_t k) {
    return n && k ? jc::linear_ws_bytes(x, ldx, w, ldw, m, n, k) : 0;
}

size_t jc_linear_backward_ws_bytes(const void *x, size_t ldx, const void *w, size_t ldw, uint32_t m, uint32_t n,
                                   uint32_t k) {
    return n && k ? jc::linear_bwd_ws_bytes(x, ldx, w, ldw, m, n, k) : 0;
}

int jc_linear_backward(uint32_t type, uint32_t act, const void *dy, size_t lddy, const void *x, size_t ldx,
                       const void *w, size_t ldw, const void *z, size_t ldz, uint32_t m, uint32_t n,
                       uint32_t k, void *dx, size_t lddx, void *dw, size_t lddw, float *dbias, void *ws,
                       void *stream) {
    return guarded(nullptr, 0, [&]() -> int {
        const char *op = "linear_backward";
        const bool any = m > 0;
        if (!check_act(op, type, act)) return -1;
        if (!check_sizes(op, m, n, k)) return -1;
        if (!check_matrix(op, "dy", dy, lddy, n, 2, any) || !check_matrix(op, "x", x, ldx, k, 2, any && dw) ||
            !check_matrix(op, "w", w, ldw, k, 2, any && dx) ||
            !check_matrix(op, "z", z, ldz, n, 2, any && act) ||
            !check_matrix(op, "dx", dx, lddx, k, 2, false) || !check_matrix(op, "dw", dw, lddw, k, 2, false) ||
            !check_vector(op, "dbias", dbias, 4, false) ||
            !check_vector(op, "ws", ws, 256, any && !ws && jc::linear_bwd_ws_bytes(dw ? x : nullptr, ldx, dx ? w : nullptr, ldw, m, n, k) > 0))
            return -1;
        jc::LinearBwdArgs a;
        a.type = type;
        a.act = act;
        a.dy = dy;
        a.lddy = lddy;
        a.x = x;
        a.ldx = ldx;
        a.w = w;
        a.ldw = ldw;
        a.z = z;
        a.ldz = ldz;
        a.m = m;
        a.n = n;
        a.k = k;
        a.dx = dx;
        a.lddx = lddx;
        a.dw = dw;
        a.lddw = lddw;
        a.dbias = dbias;
        a.ws = ws;
        return jc::launch_linear_bwd(a, (cudaStream_t)stream) ? 0 : -1;
    });
}

int jc_choice_loss(const float *logits, uint32_t n_logits, const int32_t *offsets, const int32_t *gold,
                   const float *weight, uint32_t requests, float *loss, float *dlogits, void *stream) {
    return guarded(nullptr, 0, [&]() -> int {
        const char *op = "choice_loss";
        const bool any = requests > 0;
        if (!check_vector(op, "logits", logits, 4, any && n_logits > 0) ||
            !check_vector(op, "offsets", offsets, 4, any) || !check_vector(op, "gold", gold, 4, any) ||
            !check_vector(op, "weight", weight, 4, false) || !check_vector(op, "loss", loss, 4, any) ||
            !check_vector(op, "dlogits", dlogits, 4, false))
            return -1;
        if (n_logits > MAX_SIZE || requests > MAX_SIZE)
            return fail("choice_loss: at most 2^31 - 1 logits and requests");
        jc::LossArgs a;
        a.logits = logits;
        a.n_logits = n_logits;
        a.offsets = offsets;
        a.gold = gold;
        a.weight = weight;
        a.requests = requests;
        a.loss = loss;
        a.dlogits = dlogits;
        return jc::launch_choice_loss(a, (cudaStream_t)stream) ? 0 : -1;
    });
}

JcAdamW *jc_adamw_create(const jc_adamw_tensor *tensors, size_t count, uint32_t bits) {
    return guarded(nullptr, 0, [&]() -> JcAdamW * {
        auto refuse = [](const std::string &why) -> JcAdamW * {
            jc::set_error("adamw: " + why);
            return nullptr;
        };
        if (bits != 8 && bits != 32) return refuse("states of 32 or 8 bits");
        if (!tensors && count) return refuse("tensors is null");
        std::vector<jc::AdamwTensor> table;
        std::vector<uint2> chunks;
        for (size_t i = 0; i < count; i++) {
            const jc_adamw_tensor &t = tensors[i];
            const std::string at = "tensor " + std::to_string(i) + ": ";
            if (t.n == 0) continue;
            if (!t.p || !t.g || !t.m || !t.v) return refuse(at + "null parameters, gradients or moments");
            if (bits == 8 && (!t.m_scale || !t.v_scale)) return refuse(at + "8-bit states need scales");
            if (t.grad_type > JC_F32) return refuse(at + "unknown gradient type");
            if (t.copy && t.copy_type != JC_F16 && t.copy_type != JC_BF16)
                return refuse(at + "copy_type must be JC_F16 or JC_BF16");
            if (!std::isfinite(t.weight_decay)) return refuse(at + "weight_decay is not finite");
            const size_t state = bits == 8 ? 1 : 4;
            if (misaligned(t.p, 4) || misaligned(t.g, type_size(t.grad_type)) || misaligned(t.m, state) ||
                misaligned(t.v, state) || misaligned(t.m_scale, 4) || misaligned(t.v_scale, 4) ||
                misaligned(t.copy, 2))
                return refuse(at + "a pointer is not aligned to its elements");
            jc::AdamwTensor d{};
            d.p = t.p;
            d.g = t.g;
            d.m = t.m;
            d.v = t.v;
            d.m_scale = t.m_scale;
            d.v_scale = t.v_scale;
            d.copy = t.copy;
            d.n = t.n;
            d.decay = t.weight_decay;
            d.grad_type = t.grad_type;
            d.copy_type = t.copy ? t.copy_type : JC_F32;
            d.aligned = !misaligned(t.p, 16) && !misaligned(t.g, 16) && !misaligned(t.m, 16) &&
                        !misaligned(t.v, 16) && !misaligned(t.copy, 16);
            const uint64_t n = (t.n + jc::ADAMW_CHUNK - 1) / jc::ADAMW_CHUNK;
            if (chunks.size() + n > 0x7FFFFFFFull) return refuse("too many elements");
            for (uint64_t c = 0; c < n; c++) chunks.push_back(make_uint2((unsigned)table.size(), (unsigned)c));
            table.push_back(d);
        }
        std::unique_ptr<JcAdamW> opt(new JcAdamW);
        opt->bits = bits;
        opt->n_chunks = (uint32_t)chunks.size();
        if (!jc::cuda_ok(cudaGetDevice(&opt->device), "cudaGetDevice")) return nullptr;
        if (!chunks.empty()) {
            const size_t tb = table.size() * sizeof(table[0]), cb = chunks.size() * sizeof(chunks[0]);
            if (!jc::cuda_ok(cudaMalloc(&opt->tensors, tb), "adamw: cudaMalloc") ||
                !jc::cuda_ok(cudaMalloc(&opt->chunks, cb), "adamw: cudaMalloc") ||
                !jc::cuda_ok(cudaMemcpy(opt->tensors, table.data(), tb, cudaMemcpyHostToDevice), "adamw: table") ||
                !jc::cuda_ok(cudaMemcpy(opt->chunks, chunks.data(), cb, cudaMemcpyHostToDevice), "adamw: table") ||
                // A copy from pageable memory may return before its data has arrived, and a step's stream
                // need not be ordered behind it.
                !jc::cuda_ok(cudaStreamSynchronize(nullptr), "adamw: table"))
                return nullptr;
        }
        return opt.release();
    });
}

int jc_adamw_step(JcAdamW *opt, uint64_t t, float lr, double beta1, double beta2, float eps,
                  const float *grad_scale, void *stream) {
    return guarded(nullptr, 0, [&]() -> int {
        if (!opt) return fail("adamw: no optimizer");
        if (t == 0) return fail("adamw: steps count from 1");
        if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0))
            return fail("adamw: betas must be at least 0 and below 1");
        if (!std::isfinite(lr) || !(eps >= 0.0f) || std::isinf(eps))
            return fail("adamw: lr and eps must be finite, eps not negative");
        if (!check_vector("adamw", "grad_scale", grad_scale, 4, false)) return -1;
        int dev = 0;
        if (!jc::cuda_ok(cudaGetDevice(&dev), "cudaGetDevice")) return -1;
        if (dev != opt->device) return fail("adamw: the optimizer belongs to another device");
        jc::AdamwStep a;
        a.tensors = opt->tensors;
        a.chunks = opt->chunks;
        a.n_chunks = opt->n_chunks;
        a.bits = opt->bits;
        a.lr = lr;
        a.beta1 = beta1;
        a.beta2 = beta2;
        a.eps = eps;
        a.step = t;
        a.grad_scale = grad_scale;
        return jc::launch_adamw(a, (cudaStream_t)stream) ? 0 : -1;
    });
}

void jc_adamw_free(JcAdamW *opt) { delete opt; }

}  // extern "C"
