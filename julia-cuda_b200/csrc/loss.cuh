// The loss of requests that each choose one of their own markers, and its gradient.
//
//   request r: logits l[a..b), a = offsets[r], b = offsets[r + 1], the right one gold[r] (< 0: none)
//   loss[r] = w[r] (log(sum(exp(l))) - l[a + gold[r]])
//   dlogits[i] = w[r] (exp(l[i]) / sum(exp(l)) - (i == a + gold[r]))
//
// A request without an answer, with weight 0, without logits, or with only logits of -infinity
// counts for nothing: its loss and gradients are 0.
#pragma once
#include "common.cuh"

namespace jc {

struct LossParams {
    const float *logits;
    uint32_t n_logits;
    const int32_t *offsets, *gold;
    const float *weight;
    uint32_t requests;
    float *loss, *dlogits;
    unsigned int *err;
};

// One warp a request.
__global__ void __launch_bounds__(128) choice_loss_kernel(const LossParams p) {
    dev_err_bind(p.err);
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t r = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (r >= p.requests) return;
    const int64_t a = p.offsets[r], b = p.offsets[r + 1];
    int32_t gold = p.gold[r];
    float w = p.weight ? p.weight[r] : 1.0f;
    if (a < 0 || b < a || b > (int64_t)p.n_logits || gold >= b - a) {
        // Nothing of the request is read or written but its loss.
        if (lane == 0) {
            p.loss[r] = 0.0f;
            dev_fail(JC_DEV_BAD_INDEX);
        }
        return;
    }
    float top = -INFINITY;
    for (int64_t i = a + lane; i < b; i += 32) top = fmaxf(top, p.logits[i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (top == -INFINITY) top = 0.0f;
    float sum = 0.0f;
    for (int64_t i = a + lane; i < b; i += 32) sum += expf(p.logits[i] - top);
    sum = warp_sum(sum);
    if (gold < 0 || w == 0.0f || sum == 0.0f) {
        gold = -1;
        w = 0.0f;
    }
    if (lane == 0) p.loss[r] = w == 0.0f ? 0.0f : w * (top + logf(sum) - p.logits[a + gold]);
    if (!p.dlogits) return;
    const float inv = w == 0.0f ? 0.0f : 1.0f / sum;
    for (int64_t i = a + lane; i < b; i += 32)
        p.dlogits[i] = w == 0.0f ? 0.0f
                                 : w * (expf(p.logits[i] - top) * inv - (i == a + gold ? 1.0f : 0.0f));
}

}  // namespace jc
