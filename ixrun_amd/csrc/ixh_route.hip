// Routing of tokens to experts: the choice among their logits, and the weights.
#include <type_traits>

#include "ixh_experts.h"

namespace ixh {

constexpr uint32_t kRtWaves = 4;

// ---- all lanes of a token's group get the same: exchanges with the lane 1, 2, (3 and 12 in the mirrored halves), 16 and 32 away ----
template <int CTRL> __device__ __forceinline__ uint32_t rt_dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
template <int CTRL> __device__ __forceinline__ float rt_dpp(float v) { return __uint_as_float(rt_dpp<CTRL>(__float_as_uint(v))); }
template <int CTRL> __device__ __forceinline__ uint64_t rt_dpp(uint64_t v) {
    return (uint64_t)rt_dpp<CTRL>((uint32_t)(v >> 32)) << 32 | rt_dpp<CTRL>((uint32_t)v);
}
template <int CTRL> __device__ __forceinline__ double rt_dpp(double v) {
    return __builtin_bit_cast(double, rt_dpp<CTRL>(__builtin_bit_cast(uint64_t, v)));
}
// a value of the lane and of the one 16 or 32 further, in either order
template <class V> struct RtTwo { V a, b; };
template <int BY> __device__ __forceinline__ RtTwo<uint32_t> rt_swapped(uint32_t v) {
    if constexpr (BY == 16) {
        const auto h = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return {h[0], h[1]};
    } else {
        const auto h = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return {h[0], h[1]};
    }
}
template <int BY> __device__ __forceinline__ RtTwo<uint64_t> rt_swapped(uint64_t v) {
    const auto lo = rt_swapped<BY>((uint32_t)v), hi = rt_swapped<BY>((uint32_t)(v >> 32));
    return {(uint64_t)hi.a << 32 | lo.a, (uint64_t)hi.b << 32 | lo.b};
}
template <int BY> __device__ __forceinline__ RtTwo<float> rt_swapped(float v) {
    const auto h = rt_swapped<BY>(__float_as_uint(v));
    return {__uint_as_float(h.a), __uint_as_float(h.b)};
}
template <int BY> __device__ __forceinline__ RtTwo<double> rt_swapped(double v) {
    const auto h = rt_swapped<BY>(__builtin_bit_cast(uint64_t, v));
    return {__builtin_bit_cast(double, h.a), __builtin_bit_cast(double, h.b)};
}
template <int LT, class V, class F> __device__ __forceinline__ V rt_all(V v, F f) {
    v = f(v, rt_dpp<0xB1>(v));   // quad_perm 1, 0, 3, 2
    v = f(v, rt_dpp<0x4E>(v));   // quad_perm 2, 3, 0, 1
    v = f(v, rt_dpp<0x141>(v));  // row_half_mirror
    v = f(v, rt_dpp<0x140>(v));  // row_mirror
    if constexpr (LT == 64) {
        const auto rows = rt_swapped<16>(v);
        v = f(rows.a, rows.b);
        const auto halves = rt_swapped<32>(v);
        v = f(halves.a, halves.b);
    }
    return v;
}
template <int LT, class V> __device__ __forceinline__ V rt_most(V v) { return rt_all<LT>(v, [](V a, V b) { return a > b ? a : b; }); }
template <int LT, class V> __device__ __forceinline__ V rt_least(V v) { return rt_all<LT>(v, [](V a, V b) { return a < b ? a : b; }); }
template <int LT, class V> __device__ __forceinline__ V rt_sum(V v) { return rt_all<LT>(v, [](V a, V b) { return a + b; }); }

// ---- a choice as a whole number of the same order: 0 is closed, NaN as infinity ----
__device__ __forceinline__ uint32_t rt_key(float v) {
    if (v == -__builtin_huge_valf()) return 0u;
    if (v != v) v = __builtin_huge_valf();
    const uint32_t b = __float_as_uint(v + 0.0f);  // (-0 is 0)
    return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t rt_key(double v) {
    if (v == -__builtin_huge_val()) return 0u;
    if (v != v) v = __builtin_huge_val();
    const uint64_t b = __builtin_bit_cast(uint64_t, v + 0.0);
    return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ double rt_of_key(uint64_t k) { return k ? __builtin_bit_cast(double, k >> 63 ? k & ~(1ull << 63) : ~k) : -__builtin_huge_val(); }
// 16-bit logits: their own bits in the high half
template <class T> __device__ __forceinline__ uint32_t rt_key_16(T t) {
    const float v = (float)t;
    if (v == -__builtin_huge_valf()) return 0u;
    const uint32_t b = v != v ? (uint32_t)__builtin_bit_cast(uint16_t, (T)__builtin_huge_valf()) : v == 0.0f ? 0u : (uint32_t)__builtin_bit_cast(uint16_t, t);
    return (b >> 15 ? ~b & 0xFFFFu : b | 0x8000u) << 16;
}

// ---------------------------------------------------------------------------------------------------------------
// k_route<T, LT, NV, BIAS>: LT lanes a token, expert LT v + l in register v of lane l.
//
// Scores p = softmax(l) or sigmoid(l) over the experts that are open (l above -infinity).  The choice is by l itself without a bias, which
// has the order of the scores, and by p + bias with one, in 64 bits: which experts are chosen must not hang on how exp is rounded.  A NaN
// counts as the largest, so that it reaches the output.  Equal values go to the lowest index.
//
// Bound: vector instructions.  Choices are whole numbers of their order, of 16-bit logits with the index below them in one word, so that a
// round of the choice is a largest number over the registers, four exchanges within the sixteen lanes of a row and a comparison to strike
// it out, for four tokens at once: 30 instructions at 128 experts.  (A wave a token, 64-bit pairs of choice and index by permutes through
// LDS: 16384 tokens by 128 experts, 8 chosen, 35 us; so 6.2, the vector unit busy for 71 % of it.  96 tokens by 160 experts with a bias, in groups, 7.3 us:
// 28 %, the rest are the exponentials' and exchanges' chains.)  Without a bias only the chosen experts' scores are worked out, the sum over
// all only where the weights are not divided by their own.
// ---------------------------------------------------------------------------------------------------------------
template <class T, int LT, int NV, bool BIAS>
__global__ void __launch_bounds__(kRtWaves *kWave)
k_route(const T *__restrict__ logits, int64_t ld, uint32_t tokens, RouteDev R, const float *__restrict__ bias, int32_t *__restrict__ ids,
        float *__restrict__ weights) {
    extern __shared__ __attribute__((aligned(16))) uint8_t rt_smem[];
    constexpr bool JOINT = !BIAS && sizeof(T) == 2;  // choice and index in one word
    using Key = std::conditional_t<BIAS, uint64_t, uint32_t>;
    const uint32_t l = threadIdx.x & (LT - 1u), in_block = threadIdx.x / LT, t = blockIdx.x * (kRtWaves * kWave / LT) + in_block;
    const T *const row = logits + (int64_t)min(t, tokens - 1u) * ld;
    const double inf = __builtin_huge_val();
    T raw[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) raw[v] = row[min(v * LT + l, R.experts - 1u)];
    auto logit = [&](int v) { return v * LT + l < R.experts ? (float)raw[v] : -__builtin_huge_valf(); };

    // ---- softmax: the largest logit and the sum, where they are needed ----
    float most = 0.0f;
    double sum = 1.0, of_most[BIAS ? NV : 1];  // of_most: exp(l - most)
    if (!R.sigmoid && (BIAS || !R.renormalize)) {
        most = -__builtin_huge_valf();
#pragma unroll
        for (int v = 0; v < NV; ++v) most = fmaxf(most, logit(v));
        most = rt_all<LT>(most, [](float a, float b) { return fmaxf(a, b); });
        if (most == -__builtin_huge_valf()) most = 0.0f;  // no open expert, or NaN alone
        sum = 0.0;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const double p = exp((double)logit(v) - (double)most);
            if constexpr (BIAS) of_most[v] = p;
            sum += p;
        }
        sum = rt_sum<LT>(sum);
        if (sum == 0.0) sum = 1.0;
    }
    auto score = [&](float v) {
        if (v == -__builtin_huge_valf()) return 0.0;
        return R.sigmoid ? 1.0 / (1.0 + exp(-(double)v)) : exp((double)v - (double)most) / sum;
    };

    // ---- the choices ----
    Key key[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const uint32_t e = v * LT + l;
        if constexpr (BIAS) {
            const float of = logit(v);
            key[v] = of == -__builtin_huge_valf() ? 0u : rt_key((R.sigmoid ? score(of) : of_most[v] / sum) + (double)bias[e]);
        } else if constexpr (JOINT) {
            const uint32_t k = e < R.experts ? rt_key_16(raw[v]) : 0u;
            key[v] = k ? k | (0xFFFFu - e) : 0u;
        } else {
            key[v] = rt_key(logit(v));
        }
    }
    if (R.groups > 1u) {
        // 2^k lanes work out a group (of more groups than lanes each lane several): its best, or the sum of its two best where a bias takes part
        // (2 tokens by 508 experts in 4 groups: 19.4 us with a lane a group and the powers worked out twice, 11.0)
        Key *const mine = reinterpret_cast<Key *>(rt_smem) + in_block * (R.experts + 64u), *const of_group = mine + R.experts;
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if (v * LT + l < R.experts) mine[v * LT + l] = JOINT ? key[v] & 0xFFFF0000u : key[v];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        uint32_t k = 0;
        while ((R.groups << (k + 1u)) <= (uint32_t)LT) ++k;
        for (uint32_t g = l >> k; g < R.groups; g += LT >> k) {
            Key best = 0, second = 0;
#pragma unroll 4
            for (uint32_t i = l & ((1u << k) - 1u); i < R.group_size; i += 1u << k) {
                const Key c = mine[g * R.group_size + i];
                second = c > best ? best : c > second ? c : second;
                best = c > best ? c : best;
            }
            for (uint32_t by = 1; by < 1u << k; by <<= 1) {
                const Key a = __shfl_xor(best, (int)by), b = __shfl_xor(second, (int)by), less = a < best ? a : best;
                best = a > best ? a : best;
                second = b > second ? b : second;
                second = less > second ? less : second;
            }
            if constexpr (BIAS)
                if (best && second) best = rt_key(rt_of_key(best) + rt_of_key(second));
            of_group[g] = best;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        uint64_t kept = 0;
        for (uint32_t g = l; g < R.groups; g += LT) {
            const Key own = of_group[g];
            uint32_t before = 0;
            for (uint32_t h = 0; h < R.groups; ++h) before += of_group[h] > own || (of_group[h] == own && h < g);
            kept |= (uint64_t)(before < R.top_groups) << g;
        }
        kept = rt_all<LT>(kept, [](uint64_t a, uint64_t b) { return a | b; });
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if (!((kept >> min((v * LT + l) / R.group_size, 63u)) & 1u)) key[v] = 0;
    }

    // ---- the chosen ones: lane r has the r-th ----
    uint32_t id = ~0u;
    for (uint32_t r = 0; r < R.top_k; ++r) {
        Key best = key[0];
#pragma unroll
        for (int v = 1; v < NV; ++v) best = key[v] > best ? key[v] : best;
        best = rt_most<LT>(best);
        uint32_t at;
        if constexpr (JOINT) {
            at = best ? 0xFFFFu - (best & 0xFFFFu) : ~0u;
#pragma unroll
            for (int v = 0; v < NV; ++v) key[v] = key[v] == best ? 0u : key[v];
        } else {
            at = ~0u;
#pragma unroll
            for (int v = NV - 1; v >= 0; --v) at = key[v] == best ? v * LT + l : at;
            at = rt_least<LT>(best ? at : ~0u);
#pragma unroll
            for (int v = 0; v < NV; ++v) key[v] = v * LT + l == at ? 0u : key[v];
        }
        if (l == r) id = at;
    }
    const float chosen = id != ~0u ? (float)row[id] : -__builtin_huge_valf();
    if (!R.sigmoid && !BIAS && R.renormalize) {  // (their ratios hang on no more than the largest of them)
        most = __shfl(chosen, (int)(threadIdx.x & 63u & ~(LT - 1u)));
        if (most == -__builtin_huge_valf()) most = 0.0f;
    }
    double weight = score(chosen);
    if (R.renormalize) {
        const double all = rt_sum<LT>(weight);
        weight = all == 0.0 ? 0.0 : weight / all;
    }
    if (l < R.top_k && t < tokens) {
        ids[(size_t)t * R.top_k + l] = (int32_t)id;
        weights[(size_t)t * R.top_k + l] = id == ~0u ? 0.0f : (float)(weight * R.scale);
    }
}

template <class T, int LT, int NV>
static void route_launch(const T *logits, int64_t ld, uint32_t tokens, const RouteDev &R, const float *bias, int32_t *ids, float *weights, hipStream_t s) {
    constexpr uint32_t per = kRtWaves * kWave / LT;
    const dim3 grid((tokens + per - 1u) / per), block(kRtWaves * kWave);
    const size_t lds = R.groups > 1u ? per * (R.experts + 64u) * (bias ? 8u : 4u) : 0;
    if (bias) IXH_LAUNCH((k_route<T, LT, NV, true>), grid, block, lds, s, logits, ld, tokens, R, bias, ids, weights);
    else IXH_LAUNCH((k_route<T, LT, NV, false>), grid, block, lds, s, logits, ld, tokens, R, bias, ids, weights);
}

template <class T>
static int route_type(const void *logits, int64_t ld, uint32_t tokens, const RouteDev &R, const float *bias, int32_t *ids, float *weights, hipStream_t s) {
    const T *const l = static_cast<const T *>(logits);
    if (R.experts <= 64u && R.top_k <= 16u) route_launch<T, 16, 4>(l, ld, tokens, R, bias, ids, weights, s);
    else if (R.experts <= 128u && R.top_k <= 16u) route_launch<T, 16, 8>(l, ld, tokens, R, bias, ids, weights, s);
    else if (R.experts <= 128u) route_launch<T, 64, 2>(l, ld, tokens, R, bias, ids, weights, s);
    else if (R.experts <= 256u) route_launch<T, 64, 4>(l, ld, tokens, R, bias, ids, weights, s);
    else if (R.experts <= 512u) route_launch<T, 64, 8>(l, ld, tokens, R, bias, ids, weights, s);
    else route_launch<T, 64, 16>(l, ld, tokens, R, bias, ids, weights, s);
    return hipGetLastError() == hipSuccess ? IXH_OK : IXH_ELAUNCH;
}

int launch_route(const void *logits, int dtype, int64_t ld, uint32_t tokens, const RouteDev &R, const float *bias, int32_t *ids, float *weights,
                 hipStream_t s) {
    switch (dtype) {
        case IXH_F32: return route_type<float>(logits, ld, tokens, R, bias, ids, weights, s);
        case IXH_F16: return route_type<_Float16>(logits, ld, tokens, R, bias, ids, weights, s);
        default: return route_type<__bf16>(logits, ld, tokens, R, bias, ids, weights, s);
    }
}

}  // namespace ixh
