// Scores and weights of the router's selection, shared by the kernels that make it.
#pragma once
#include <float.h>
#include <limits.h>
#include <math.h>

#include "common.hpp"

namespace mfq {

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}

__device__ __forceinline__ float topk_weight(float raw, int mode, float smax, float ssum) {
    if (mode == MFQ_TOPK_SIGMOID) return 1.f / (1.f + expf(-raw));
    if (mode == MFQ_TOPK_SQRT_SOFTPLUS) return sqrtf(raw > 20.f ? raw : log1pf(expf(raw)));
    if (mode == MFQ_TOPK_SOFTMAX) return expf(raw - smax) / ssum;
    return raw;
}
// order-preserving map of the float to a signed int (-0 and +0 compare equal, as they do as floats)
__device__ __forceinline__ int topk_key(float score) {
    const int b = __float_as_int(score + 0.f), key = b ^ ((b >> 31) & 0x7fffffff);
    return key == INT_MIN ? INT_MIN + 1 : key;  // unreachable from a float; keeps key - 1 from wrapping
}
// the weights of the selection, lane = rank
__device__ __forceinline__ float topk_finish(float v, int k, int lane, int mode, int normalize, float norm_floor) {
    if (mode == MFQ_TOPK_DELAYED_SOFTMAX) {
        const float mx = wave_max(lane < k ? v : -INFINITY);
        v = lane < k ? expf(v - mx) : 0.f;
        return v / wave_sum(v);
    }
    return normalize ? v / fmaxf(wave_sum(v), norm_floor) : v;
}

}  // namespace mfq
