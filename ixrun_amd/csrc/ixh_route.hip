// Routing of tokens to experts: the choice among their logits, and the weights.
#include "ixh_experts.h"

namespace ixh {

constexpr uint32_t kRtWaves = 4;  // tokens of a workgroup

template <class T> __device__ __forceinline__ float rt_logit(T v) { return (float)v; }

__device__ __forceinline__ double rt_shfl_xor(double v, int by) { return __shfl_xor(v, by); }

// ---------------------------------------------------------------------------------------------------------------
// k_route<T, NV>: one wave a token, expert 64 v + lane in register v of the lane.
//
// Scores p = softmax(l) or sigmoid(l) over the experts that are open (l above -infinity).  The choice is by l itself without a bias, which
// has the order of the scores, and by p + bias with one, in 64 bits: which experts are chosen must not hang on how exp is rounded.  A NaN
// counts as the largest, so that it reaches the output.  Equal values go to the lowest index.
// ---------------------------------------------------------------------------------------------------------------
template <class T, int NV>
__global__ void __launch_bounds__(kRtWaves *kWave)
k_route(const T *__restrict__ logits, int64_t ld, uint32_t tokens, RouteDev R, const float *__restrict__ bias, int32_t *__restrict__ ids,
        float *__restrict__ weights) {
    extern __shared__ __attribute__((aligned(16))) uint8_t rt_smem[];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, t = blockIdx.x * kRtWaves + wave;
    if (t >= tokens) return;
    const double inf = __builtin_huge_val();
    const T *const row = logits + (int64_t)t * ld;
    float l[NV];
    double p[NV], choice[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const uint32_t e = 64u * v + lane;
        l[v] = e < R.experts ? rt_logit(row[e]) : -__builtin_huge_valf();
    }
    if (R.sigmoid) {
#pragma unroll
        for (int v = 0; v < NV; ++v) p[v] = 1.0 / (1.0 + exp(-(double)l[v]));
    } else {
        float most = -__builtin_huge_valf();
#pragma unroll
        for (int v = 0; v < NV; ++v) most = fmaxf(most, l[v]);
        for (int by = 32; by; by >>= 1) most = fmaxf(most, __shfl_xor(most, by));
        if (most == -__builtin_huge_valf()) most = 0.0f;  // no open expert
        double sum = 0.0;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            p[v] = exp((double)l[v] - (double)most);
            sum += p[v];
        }
        for (int by = 32; by; by >>= 1) sum += rt_shfl_xor(sum, by);
        if (sum != 0.0)
#pragma unroll
            for (int v = 0; v < NV; ++v) p[v] /= sum;
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const uint32_t e = 64u * v + lane;
        const bool open = !(l[v] == -__builtin_huge_valf());
        choice[v] = l[v];
        if (bias && open) choice[v] = p[v] + (double)bias[e];
        if (choice[v] != choice[v]) choice[v] = inf;
        if (!open) choice[v] = -inf, p[v] = 0.0;
    }
    if (R.groups > 1u) {
        // lane g works out group g: its best, or the sum of its two best where a bias takes part
        double *const mine = reinterpret_cast<double *>(rt_smem) + wave * (R.experts + 64u), *const score = mine + R.experts;
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if (64u * v + lane < R.experts) mine[64u * v + lane] = choice[v];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        double best = -inf, second = -inf;
        if (lane < R.groups)
            for (uint32_t i = 0; i < R.group_size; ++i) {
                const double c = mine[lane * R.group_size + i];
                second = c > best ? best : c > second ? c : second;
                best = c > best ? c : best;
            }
        if (bias && best != -inf && second != -inf) best += second;
        score[lane] = best;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        uint32_t before = 0;
        for (uint32_t g = 0; g < R.groups; ++g) before += score[g] > best || (score[g] == best && g < lane);
        const uint64_t kept = __ballot(lane < R.groups && before < R.top_groups);
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if (!((kept >> min((64u * v + lane) / R.group_size, 63u)) & 1u)) choice[v] = -inf;
    }
    int32_t id = -1;
    double weight = 0.0;
    for (uint32_t r = 0; r < R.top_k; ++r) {
        double best = -inf;
        uint32_t at = ~0u;
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if (choice[v] > best) best = choice[v], at = 64u * v + lane;
        for (int by = 32; by; by >>= 1) {
            const double other = rt_shfl_xor(best, by);
            const uint32_t other_at = __shfl_xor(at, by);
            if (other > best || (other == best && other_at < at)) best = other, at = other_at;
        }
        if (best == -inf) break;
        double of = 0.0;
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if (64u * v + lane == at) of = p[v], choice[v] = -inf;
        of = __shfl(of, (int)(at & 63u));
        if (lane == r) id = (int32_t)at, weight = of;
    }
    if (R.renormalize) {
        double sum = weight;
        for (int by = 32; by; by >>= 1) sum += rt_shfl_xor(sum, by);
        weight = sum == 0.0 ? 0.0 : weight / sum;
    }
    if (lane < R.top_k) {
        ids[(size_t)t * R.top_k + lane] = id;
        weights[(size_t)t * R.top_k + lane] = id < 0 ? 0.0f : (float)(weight * R.scale);
    }
}

template <class T>
static int route_launch(const void *logits, int64_t ld, uint32_t tokens, const RouteDev &R, const float *bias, int32_t *ids, float *weights,
                        hipStream_t s) {
    const dim3 grid((tokens + kRtWaves - 1u) / kRtWaves), block(kRtWaves * kWave);
    const size_t lds = R.groups > 1u ? kRtWaves * (R.experts + 64u) * sizeof(double) : 0;
    const T *const l = static_cast<const T *>(logits);
    if (R.experts <= 64u) IXH_LAUNCH((k_route<T, 1>), grid, block, lds, s, l, ld, tokens, R, bias, ids, weights);
    else if (R.experts <= 128u) IXH_LAUNCH((k_route<T, 2>), grid, block, lds, s, l, ld, tokens, R, bias, ids, weights);
    else if (R.experts <= 256u) IXH_LAUNCH((k_route<T, 4>), grid, block, lds, s, l, ld, tokens, R, bias, ids, weights);
    else if (R.experts <= 512u) IXH_LAUNCH((k_route<T, 8>), grid, block, lds, s, l, ld, tokens, R, bias, ids, weights);
    else IXH_LAUNCH((k_route<T, 16>), grid, block, lds, s, l, ld, tokens, R, bias, ids, weights);
    return hipGetLastError() == hipSuccess ? IXH_OK : IXH_ELAUNCH;
}

int launch_route(const void *logits, int dtype, int64_t ld, uint32_t tokens, const RouteDev &R, const float *bias, int32_t *ids, float *weights,
                 hipStream_t s) {
    switch (dtype) {
        case IXH_F32: return route_launch<float>(logits, ld, tokens, R, bias, ids, weights, s);
        case IXH_F16: return route_launch<_Float16>(logits, ld, tokens, R, bias, ids, weights, s);
        default: return route_launch<__bf16>(logits, ld, tokens, R, bias, ids, weights, s);
    }
}

}  // namespace ixh
