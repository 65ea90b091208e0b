// Experts with many tokens: the rows gathered in operand order, and the launches of both matrices.
#include <type_traits>

#include "ixh_experts_prompt.h"

namespace ixh {

// ---------------------------------------------------------------------------------------------------------------
// k_experts_xtile: the tokens' rows, gathered by expert, in operand order: block b of 16 rows and 32 columns kb is 1 KB at (b n_kb + kb)
// KB, lane l's 16 bytes are row l % 16, columns 8 (l / 16) .. + 7; zeros past the last column and in rows without a slot.
//
// Bound: memory.  24576 rows of 2048 columns, 117 MB: 32 us (34 us with a piece at a time).  (The products could gather for themselves, but
// take each row once per 64 weight rows, and half a line of the L2 at a time.)
// ---------------------------------------------------------------------------------------------------------------
constexpr uint32_t kExGather = 4;  // pieces of 32 columns a wave asks for at once
template <bool WHOLE>
__global__ void __launch_bounds__(256)
k_experts_xtile(const uint16_t *__restrict__ x, int64_t ldx, uint32_t top_k, uint32_t in_f, uint32_t n_kb, const uint32_t *__restrict__ n_blocks,
                const uint32_t *__restrict__ order, ln_u32x4 *__restrict__ xt) {
    const uint32_t block = blockIdx.x, lane = threadIdx.x & 63u, kb0 = (blockIdx.y * 4u + (threadIdx.x >> 6)) * kExGather;
    if (block >= *n_blocks || kb0 >= n_kb) return;
    const uint32_t slot = order[block * 16u + (lane & 15u)];
    const uint16_t *const row = x + (int64_t)(slot == kEpNone ? 0u : slot / top_k) * ldx;
    ln_u32x4 v[kExGather];
#pragma unroll
    for (uint32_t k = 0; k < kExGather; ++k) {
        const uint32_t col = (kb0 + k) * 32u + (lane >> 4) * 8u;
        if constexpr (WHOLE) {
            v[k] = *reinterpret_cast<const ln_u32x4 *>(row + min(col, in_f - 8u));
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) v[k][i] = row[min(col + 2u * i, in_f - 1u)] | (uint32_t)row[min(col + 2u * i + 1u, in_f - 1u)] << 16;
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) v[k][i] &= (col + 2u * i < in_f ? 0xFFFFu : 0u) | (col + 2u * i + 1u < in_f ? 0xFFFF0000u : 0u);
        }
        if (slot == kEpNone || col >= in_f) v[k] = ln_u32x4{0u, 0u, 0u, 0u};
    }
    ln_u32x4 *const to = xt + ((size_t)block * n_kb + kb0) * 64u + lane;  // (n_kb is a multiple of sixteen)
#pragma unroll
    for (uint32_t k = 0; k < kExGather; ++k) to[k * 64u] = v[k];
}

int launch_experts_prompt(const ExDev &X, const ExCall &call, const ExPlan &plan, uint32_t row_tiles, uint32_t blocks, void *xt, void *inner,
                          float *per_slot, hipStream_t s) {
    EpCall R{};
    R.xt = static_cast<const ln_u32x4 *>(xt), R.n_tiles = plan.n_tiles, R.tiles = plan.tiles, R.order = plan.order;
    R.inner = static_cast<uint8_t *>(inner), R.n_kb_inner = X.second.n_cells * 16u;
    R.activation = X.activation, R.gated = X.gated;
    const uint32_t n_kb = X.first.n_cells * 16u;
    const bool whole = ((uintptr_t)call.x & 15u) == 0 && call.ldx % 8 == 0 && X.hidden % 8u == 0;
    const auto gather = [&](auto is_whole) {
        IXH_LAUNCH(k_experts_xtile<is_whole()>, dim3(blocks, n_kb / (4u * kExGather)), dim3(256), 0, s, call.x, call.ldx, call.top_k, X.hidden, n_kb,
                   plan.n_blocks, plan.order, static_cast<ln_u32x4 *>(xt));
    };
    if (whole) gather(std::true_type{});
    else gather(std::false_type{});
    int rc = ep_first(X.first, R, row_tiles, s);
    if (rc != IXH_OK) return rc;
    R.xt = static_cast<const ln_u32x4 *>(inner), R.out = per_slot;
    return ep_second(X.second, R, row_tiles, s);
}

}  // namespace ixh
