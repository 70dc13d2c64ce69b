// The fine-tuning operators' host side: argument structs and launchers (train.cu). Every launcher
// takes checked arguments, queues its kernels on `s` and returns false with the error set if a
// launch failed.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "jc_internal.h"

namespace jc {

struct NormArgs {
    uint32_t type = 0;
    const void *x = nullptr;
    size_t ldx = 0;
    const float *gamma = nullptr, *beta = nullptr;
    float eps = 0.f;
    uint32_t rows = 0, d = 0;
    void *y = nullptr;
    size_t ldy = 0;
    float *stats = nullptr;
};
bool launch_norm(const NormArgs &a, cudaStream_t s);

struct NormBwdArgs {
    uint32_t type = 0;
    const void *dy = nullptr;
    size_t lddy = 0;
    const void *x = nullptr;
    size_t ldx = 0;
    const float *gamma = nullptr, *stats = nullptr;
    const void *add = nullptr;
    size_t ldadd = 0;
    uint32_t rows = 0, d = 0;
    void *dx = nullptr;
    size_t lddx = 0;
    float *dgamma = nullptr, *dbeta = nullptr;
    float *ws = nullptr;
};
size_t norm_bwd_ws_floats(uint32_t rows, uint32_t d);
bool launch_norm_bwd(const NormBwdArgs &a, cudaStream_t s);

struct LinearArgs {
    uint32_t type = 0, act = 0;
    const void *x = nullptr;
    size_t ldx = 0;
    const void *w = nullptr;
    size_t ldw = 0;
    const float *bias = nullptr;
    const void *res = nullptr;
    size_t ldres = 0;
    void *y = nullptr;
    size_t ldy = 0;
    void *z = nullptr;
    size_t ldz = 0;
    uint32_t m = 0, n = 0, k = 0;
    void *ws = nullptr;
};
size_t linear_ws_bytes(const void *x, size_t ldx, const void *w, size_t ldw, uint32_t m, uint32_t n, uint32_t k);
bool launch_linear(const LinearArgs &a, cudaStream_t s);

struct LinearBwdArgs {
    uint32_t type = 0, act = 0;
    const void *dy = nullptr;
    size_t lddy = 0;
    const void *x = nullptr;
    size_t ldx = 0;
    const void *w = nullptr;
    size_t ldw = 0;
    const void *z = nullptr;
    size_t ldz = 0;
    uint32_t m = 0, n = 0, k = 0;
    void *dx = nullptr;
    size_t lddx = 0;
    void *dw = nullptr;
    size_t lddw = 0;
    float *dbias = nullptr;
    void *ws = nullptr;
};
size_t linear_bwd_ws_bytes(const void *x, size_t ldx, const void *w, size_t ldw, uint32_t m, uint32_t n, uint32_t k);
bool launch_linear_bwd(const LinearBwdArgs &a, cudaStream_t s);

struct LossArgs {
    const float *logits = nullptr;
    uint32_t n_logits = 0;
    const int32_t *offsets = nullptr, *gold = nullptr;
    const float *weight = nullptr;
    uint32_t requests = 0;
    float *loss = nullptr, *dlogits = nullptr;
};
bool launch_choice_loss(const LossArgs &a, cudaStream_t s);

// AdamW: a chunk is what one block updates, ADAMW_BLOCK elements share an 8-bit state's scale.
constexpr uint32_t ADAMW_THREADS = 256, ADAMW_CHUNK = 8 * ADAMW_THREADS, ADAMW_BLOCK = 256;
struct AdamwTensor {
    float *p;
    const void *g;
    void *m, *v;
    float *m_scale, *v_scale;
    void *copy;
    uint64_t n;
    float decay;
    uint32_t grad_type, copy_type;  // JC_F32 / JC_F16 / JC_BF16; copy_type JC_F32: no copy
    uint32_t aligned;               // every pointer 16-byte aligned
};
struct AdamwStep {
    const AdamwTensor *tensors = nullptr;
    const uint2 *chunks = nullptr;
    uint32_t n_chunks = 0, bits = 32;
    float lr = 0.f;
    double beta1 = 0, beta2 = 0;
    float eps = 0.f;
    uint64_t step = 0;
    const float *grad_scale = nullptr;
};
bool launch_adamw(const AdamwStep &a, cudaStream_t s);

}  // namespace jc
