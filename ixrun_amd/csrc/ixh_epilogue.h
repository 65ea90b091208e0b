// What is done to a product's sum, in fp32, before its one rounding to bf16.
#pragma once
#include "ixh_dev.h"

namespace ixh {

// e^v, within 2 |v| + 2 steps of fp32, and a quotient within 2 (0 where b is above 2^126, whose reciprocal is no normal number): they stand in a factor
// between 0 and 1 of what is rounded to 8 bits, off by some 2^-20 of it, or by 2^-126 where it is smaller than that.
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
typedef uint32_t EpPairs __attribute__((ext_vector_type(2)));  // four columns
struct EpFour { EpPairs bias, multiplier, residual; };
struct Epilogue {
    const uint16_t *multiplier, *residual;
    int64_t ld_multiplier, ld_residual;
    int activation;
    bool wide;  // bias, multiplier, residual and y allow accesses of four columns
    __device__ __forceinline__ uint16_t output(float sum, uint32_t r, uint32_t at) const {
        float v = ep_activation(activation, sum);
        if (multiplier) v *= bf16_bits_to_f32(multiplier[(int64_t)r * ld_multiplier + at]);
        if (residual) v += bf16_bits_to_f32(residual[(int64_t)r * ld_residual + at]);
        return ep_bf16(v);
    }
    // The same for four columns: what is read can be asked for while the sums are on their way.  (With accesses of two bytes and a way of its own for
    // each element: k_lanes_prompt_reduce, 10240 x 5120 at 333 rows, 17.0 us, 10.4 so; k_lanes_gemm, 17408 x 1024 at 17 / 100 rows, calls of 14.2 / 27.1 and
    // 11.7 / 18.5.)
    __device__ __forceinline__ EpFour fetch(const uint16_t *bias, uint32_t r, uint32_t at) const {
        EpFour f{};
        if (bias) f.bias = *reinterpret_cast<const EpPairs *>(bias + at);
        if (multiplier) f.multiplier = *reinterpret_cast<const EpPairs *>(multiplier + (int64_t)r * ld_multiplier + at);
        if (residual) f.residual = *reinterpret_cast<const EpPairs *>(residual + (int64_t)r * ld_residual + at);
        return f;
    }
    template <class V> __device__ __forceinline__ void put(V v, const EpFour &f, bool biased, uint16_t *to) const {
        const auto of = [](const EpPairs &p, int k) { return bf16_bits_to_f32(k & 1 ? p[k >> 1] >> 16 : p[k >> 1] & 0xFFFFu); };
        if (biased)
            for (int k = 0; k < 4; ++k) v[k] += of(f.bias, k);
        ep_activations(activation, v);
        if (multiplier)
            for (int k = 0; k < 4; ++k) v[k] *= of(f.multiplier, k);
        if (residual)
            for (int k = 0; k < 4; ++k) v[k] += of(f.residual, k);
        *reinterpret_cast<EpPairs *>(to) = EpPairs{ep_bf16(v[0]) | (uint32_t)ep_bf16(v[1]) << 16, ep_bf16(v[2]) | (uint32_t)ep_bf16(v[3]) << 16};
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
#define EP_OUT  // (the outputs may be the multiplier or the residual)
#else
#define EP(name) name
#define EP_PARAM
#define EP_ARG
#define EP_OUT __restrict__
#endif
