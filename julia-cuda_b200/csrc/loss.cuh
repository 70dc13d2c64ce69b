// The loss of requests that each choose one of their own markers, and its gradient.
//
//   request r: logits l[a..b), a = offsets[r], b = offsets[r + 1], the right one gold[r] (< 0: none)
//   loss[r] = w[r] (log(sum(exp(l - top))) + (top - l[a + gold[r]])), top = max(l): from differences
//             alone, or logits far from 0 would round away a confident request's small loss
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

// exp(x), x at most 0: what would be subnormal is 0 (its handling is half of the function).
__device__ __forceinline__ float exp_below(float x) { return ex2_approx(x * 1.44269504f); }

// Request r's span and right marker, checked: false (recorded) if they are out of range.
__device__ __forceinline__ bool loss_request(const LossParams &p, uint32_t r, uint32_t &a, uint32_t &b, int32_t &gold,
                                             float &w) {
    const int32_t lo = p.offsets[r], hi = p.offsets[r + 1];
    gold = p.gold[r];
    w = p.weight ? p.weight[r] : 1.0f;
    a = (uint32_t)lo;
    b = (uint32_t)hi;
    return lo >= 0 && hi >= lo && b <= p.n_logits && gold < hi - lo;
}

// Sums and maxima over a group of G threads: a warp or the block.
template <int G>
__device__ __forceinline__ float loss_sum(float v, float *part) {
    v = warp_sum(v);
    if constexpr (G > 32) {
        __syncthreads();
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int i = 0; i < G / 32; i++) v += part[i];
    }
    return v;
}
template <int G>
__device__ __forceinline__ float loss_max(float v, float *part) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    if constexpr (G > 32) {
        __syncthreads();
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < G / 32; i++) v = fmaxf(v, part[i]);
    }
    return v;
}

// One request by a group of G threads; its first LOSS_KEEP G logits stay in registers between the
// three passes (maximum, sum, gradient), the others are read again. exp is taken twice rather than
// kept: the second is free beside the memory.
constexpr int LOSS_KEEP = 4;

template <int G>
__device__ __forceinline__ void loss_group(const LossParams &p, uint32_t r, uint32_t t, float *part) {
    uint32_t a, b;
    int32_t gold;
    float w;
    if (!loss_request(p, r, a, b, gold, w)) {
        // Nothing of the request is read or written but its loss.
        if (t == 0) {
            p.loss[r] = 0.0f;
            dev_fail(JC_DEV_BAD_INDEX);
        }
        return;
    }
    float v[LOSS_KEEP], top = -INFINITY;
#pragma unroll
    for (int k = 0; k < LOSS_KEEP; k++) v[k] = b - a > k * G + t ? p.logits[a + k * G + t] : -INFINITY;
    const float right = gold >= 0 ? p.logits[a + gold] : 0.0f;
#pragma unroll
    for (int k = 0; k < LOSS_KEEP; k++) top = fmaxf(top, v[k]);
    for (uint32_t i = LOSS_KEEP * G + t; i < b - a; i += G) top = fmaxf(top, p.logits[a + i]);
    top = loss_max<G>(top, part);
    if (top == -INFINITY) top = 0.0f;
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < LOSS_KEEP; k++) sum += exp_below(v[k] - top);
    for (uint32_t i = LOSS_KEEP * G + t; i < b - a; i += G) sum += exp_below(p.logits[a + i] - top);
    sum = loss_sum<G>(sum, part);
    const bool counts = gold >= 0 && w != 0.0f && sum != 0.0f;
    if (t == 0) p.loss[r] = counts ? w * (logf(sum) + (top - right)) : 0.0f;
    if (!p.dlogits) return;
    const float inv = 1.0f / sum;
    auto grad = [&](uint32_t i, float l) {
        p.dlogits[a + i] = counts ? w * (exp_below(l - top) * inv - (i == (uint32_t)gold ? 1.0f : 0.0f)) : 0.0f;
    };
#pragma unroll
    for (int k = 0; k < LOSS_KEEP; k++)
        if (b - a > k * G + t) grad(k * G + t, v[k]);
    for (uint32_t i = LOSS_KEEP * G + t; i < b - a; i += G) grad(i, p.logits[a + i]);
}

// G 32: four requests a block; G 256: one.
template <int G>
__global__ void __launch_bounds__(G < 128 ? 128 : G) loss_group_kernel(const LossParams p) {
    constexpr int PER = G < 128 ? 128 / G : 1;
    __shared__ float part[G / 32];
    dev_err_bind(p.err);
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t r = blockIdx.x * PER + threadIdx.x / G;
    if (r < p.requests) loss_group<G>(p, r, threadIdx.x % G, part);
}

// Requests of a few markers: a lane takes a request, a warp 32 consecutive ones. A lane reads its logits
// where they are (neighbours share the lines, so the first reads bring the others into L1) and keeps up
// to LOSS_REGS of them in registers; the gradients go out through the warp's part of shared memory in
// whole lines. Warps stay and walk the requests, the next ones' spans requested ahead. A warp whose
// gradients do not fit (a long request among short ones), or whose requests lie out of order, takes them
// one by one instead. A million requests of 6.5 logits: 22.2 us, 3.1 TB/s; bound by the latency of the
// reads one behind the other (spans, logits), of which 32 warps a SM hide half.
constexpr int LOSS_WARPS = 4, LOSS_SMEM = 768, LOSS_REGS = 16;

__global__ void __launch_bounds__(32 * LOSS_WARPS, 8) loss_short_kernel(const LossParams p) {
    __shared__ float smem[LOSS_WARPS][LOSS_SMEM];
    dev_err_bind(p.err);
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t t = threadIdx.x & 31, step = gridDim.x * LOSS_WARPS * 32;
    float *s = smem[threadIdx.x / 32];
    // A request's span, right marker and weight; none past the last request.
    struct Request {
        uint32_t a, b;
        int32_t gold;
        float w;
        bool ok;
    };
    auto look_up = [&](uint64_t r) {
        Request q{0, 0, -1, 0.0f, true};
        if (r < p.requests) q.ok = loss_request(p, (uint32_t)r, q.a, q.b, q.gold, q.w);
        return q;
    };
    uint64_t r0 = ((uint64_t)blockIdx.x * LOSS_WARPS + threadIdx.x / 32) * 32;
    Request next = look_up(r0 + t);
    for (; r0 < p.requests; r0 += step) {
        const Request q = next;
        next = look_up(r0 + step + t);
        const uint32_t n = (uint32_t)min((uint64_t)32, p.requests - r0), len = q.b - q.a;
        const uint32_t lo = __shfl_sync(0xffffffffu, q.a, 0), hi = __shfl_sync(0xffffffffu, q.b, n - 1);
        const bool fits = q.ok && (t >= n || (q.a >= lo && q.b <= hi)) && hi >= lo && hi - lo <= LOSS_SMEM;
        if (!__all_sync(0xffffffffu, fits)) {
            for (uint32_t k = 0; k < n; k++) loss_group<32>(p, (uint32_t)(r0 + k), t, nullptr);
            continue;
        }
        const float *l = p.logits + q.a;
        float *out = s + (t < n ? q.a - lo : 0);
        const uint32_t longest = __reduce_max_sync(0xffffffffu, len);
        const bool regs = longest <= LOSS_REGS;
        float top = -INFINITY, sum = 0.0f, v[LOSS_REGS];
        const float right = q.gold >= 0 ? l[q.gold] : 0.0f;
        if (regs) {
#pragma unroll
            for (int i = 0; i < LOSS_REGS; i += 4)
                if (i < longest)
#pragma unroll
                    for (int j = i; j < i + 4; j++) v[j] = j < len ? l[j] : -INFINITY;
#pragma unroll
            for (int i = 0; i < LOSS_REGS; i += 4)
                if (i < longest) top = fmaxf(top, fmaxf(fmaxf(v[i], v[i + 1]), fmaxf(v[i + 2], v[i + 3])));
        } else {
            for (uint32_t i = 0; i < len; i++) top = fmaxf(top, l[i]);
        }
        if (top == -INFINITY) top = 0.0f;
        if (regs) {
#pragma unroll
            for (int i = 0; i < LOSS_REGS; i += 4)
                if (i < longest)
#pragma unroll
                    for (int j = i; j < i + 4; j++) {
                        v[j] = exp_below(v[j] - top);
                        sum += v[j];
                    }
        } else {
            for (uint32_t i = 0; i < len; i++) sum += exp_below(l[i] - top);
        }
        const bool counts = q.gold >= 0 && q.w != 0.0f && sum != 0.0f;
        if (t < n) p.loss[r0 + t] = counts ? q.w * (logf(sum) + (top - right)) : 0.0f;
        if (!p.dlogits) continue;
        const float f = q.w / sum;
        if (regs) {
#pragma unroll
            for (int i = 0; i < LOSS_REGS; i += 4)
                if (i < longest)
#pragma unroll
                    for (int j = i; j < i + 4; j++)
                        if (j < len) out[j] = counts ? v[j] * f : 0.0f;
        } else {
            for (uint32_t i = 0; i < len; i++) out[i] = counts ? exp_below(l[i] - top) * f : 0.0f;
        }
        if (counts) out[q.gold] -= q.w;
        __syncwarp();
#pragma unroll 8
        for (uint32_t i = t; i < hi - lo; i += 32) p.dlogits[lo + i] = s[i];
        __syncwarp();
    }
}

}  // namespace jc
