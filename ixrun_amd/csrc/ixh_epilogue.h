// What is done to a product's sum, in fp32, before its one rounding to bf16.
#pragma once
#include "ixh_dev.h"

namespace ixh {

// e^v, within 2 |v| + 2 steps of fp32, and a quotient within 2: they stand in a factor between 0 and 1 of what is rounded to 8 bits.
// (expf and the division of IEEE 754 take 40 instructions an activation against 6: half of the time that k_experts_prompt spent behind its
// products.)
__device__ __forceinline__ float ep_exp(float v) { return __builtin_amdgcn_exp2f(v * 1.44269504088896341f); }
__device__ __forceinline__ float ep_ratio(float a, float b) { return a * __builtin_amdgcn_rcpf(b); }

// The sum's activation.  Where exp overflows the quotient is the limit, 0 (of -infinity itself NaN, as infinity times 0 is).
// 0.5 (1 + tanh(t)) is 1 / (1 + e^(-2 t)).
__device__ __forceinline__ float ep_activation(int act, float v) {
    switch (act) {
        case IXH_ACT_SILU: return ep_ratio(v, 1.0f + ep_exp(-v));
        case IXH_ACT_GELU: return 0.5f * v * (1.0f + erff(v * 0.70710678118654752f));
        case IXH_ACT_GELU_TANH: return ep_ratio(v, 1.0f + ep_exp(-1.5957691216057308f * (v + 0.044715f * v * v * v)));
        case IXH_ACT_RELU: return v < 0.0f ? 0.0f : v;
        case IXH_ACT_RELU2: v = v < 0.0f ? 0.0f : v; return v * v;
        default: return v;
    }
}
// four sums', one way for all
template <class V> __device__ __forceinline__ void ep_activations(int act, V &v) {
    switch (act) {
#define EP_EACH(A)                                            \
    case A:                                                   \
        for (int k = 0; k < 4; ++k) v[k] = ep_activation(A, v[k]); \
        break;
        EP_EACH(IXH_ACT_SILU)
        EP_EACH(IXH_ACT_GELU)
        EP_EACH(IXH_ACT_GELU_TANH)
        EP_EACH(IXH_ACT_RELU)
        EP_EACH(IXH_ACT_RELU2)
#undef EP_EACH
    }
}
inline bool ep_known(int act) { return act >= IXH_ACT_NONE && act <= IXH_ACT_RELU2; }

// round-to-nearest-even, NaN stays NaN whatever its bits
__device__ __forceinline__ uint16_t ep_bf16(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }

// bf16(act(sum + bias) * multiplier + residual); multiplier and residual bf16 [rows, ld], or NULL.
struct Epilogue {
    const uint16_t *multiplier, *residual;
    int64_t ld_multiplier, ld_residual;
    int activation;
    __device__ __forceinline__ uint16_t output(float sum, uint32_t r, uint32_t at) const {
        float v = ep_activation(activation, sum);
        if (multiplier) v *= bf16_bits_to_f32(multiplier[(int64_t)r * ld_multiplier + at]);
        if (residual) v += bf16_bits_to_f32(residual[(int64_t)r * ld_residual + at]);
        return ep_bf16(v);
    }
};

int launch_epilogue(const uint16_t *v, int64_t ldv, uint32_t m, uint32_t out_f, uint16_t *y, int64_t ldy, Epilogue ep, hipStream_t s);

}  // namespace ixh

// The kernels of ixh_lanes*.hip exist twice: by themselves, and with an epilogue in place of their own output, from the same text, which
// ixh_lanes*_ep.hip include with IXH_EP.  (As functions that both kernels call, the plain kernels came out with other schedules and, in
// k_lanes_rows, up to 48 instructions more.)
#ifdef IXH_EP
#define EP(name) name##_ep
#define EP_PARAM , Epilogue ep
#define EP_ARG , ep
#else
#define EP(name) name
#define EP_PARAM
#define EP_ARG
#endif
