// What is done to a product's sum, in fp32, before its one rounding to bf16.
#pragma once
#include "ixh_dev.h"

namespace ixh {

// The sum's activation.  Where exp overflows the quotient is the limit, 0 (of -infinity itself NaN, as infinity times 0 is).
__device__ __forceinline__ float ep_activation(int act, float v) {
    switch (act) {
        case IXH_ACT_SILU: return v / (1.0f + expf(-v));
        case IXH_ACT_GELU: return 0.5f * v * (1.0f + erff(v * 0.70710678118654752f));
        case IXH_ACT_GELU_TANH: return 0.5f * v * (1.0f + tanhf(0.79788456080286536f * (v + 0.044715f * v * v * v)));
        case IXH_ACT_RELU: return v < 0.0f ? 0.0f : v;
        case IXH_ACT_RELU2: v = v < 0.0f ? 0.0f : v; return v * v;
        default: return v;
    }
}
inline bool ep_known(int act) { return act >= IXH_ACT_NONE && act <= IXH_ACT_RELU2; }

// round-to-nearest-even, NaN stays NaN whatever its bits
__device__ __forceinline__ uint16_t ep_bf16(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }

}  // namespace ixh
