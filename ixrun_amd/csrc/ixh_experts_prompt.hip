// Experts with many tokens: the rows gathered in operand order, and the launches of both matrices.
#include <algorithm>

#include "ixh_experts_prompt.h"

namespace ixh {

// ---------------------------------------------------------------------------------------------------------------
// k_experts_xtile: the tokens' rows, gathered by expert, in operand order: block b of 16 rows and 32 columns kb is 1 KB at (b n_kb + kb)
// KB, lane l's 16 bytes are row l % 16, columns 8 (l / 16) .. + 7; zeros past the last column and in rows without a slot.
// ---------------------------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(256)
k_experts_xtile(const uint16_t *__restrict__ x, int64_t ldx, uint32_t top_k, uint32_t in_f, uint32_t n_kb, bool whole,
                const uint32_t *__restrict__ n_blocks, const uint32_t *__restrict__ order, ln_u32x4 *__restrict__ xt) {
    const uint32_t block = blockIdx.x, lane = threadIdx.x & 63u;
    if (block >= *n_blocks) return;
    const uint32_t slot = order[block * 16u + (lane & 15u)];
    const uint16_t *const row = x + (int64_t)(slot == kEpNone ? 0u : slot / top_k) * ldx;
    for (uint32_t kb = blockIdx.y * 4u + (threadIdx.x >> 6); kb < n_kb; kb += gridDim.y * 4u) {
        const uint32_t col = kb * 32u + (lane >> 4) * 8u;
        ln_u32x4 v = {0u, 0u, 0u, 0u};
        if (slot != kEpNone && col < in_f) {
            if (whole) {
                v = *reinterpret_cast<const ln_u32x4 *>(row + col);
            } else {
#pragma unroll
                for (uint32_t k = 0; k < 8; ++k)
                    if (col + k < in_f) v[k >> 1] |= (uint32_t)row[col + k] << (16u * (k & 1u));
            }
        }
        xt[((size_t)block * n_kb + kb) * 64u + lane] = v;
    }
}

int launch_experts_prompt(const ExDev &X, const ExCall &call, const ExPlan &plan, uint32_t row_tiles, uint32_t blocks, void *xt, void *inner,
                          float *per_slot, hipStream_t s) {
    EpCall R{};
    R.xt = static_cast<const ln_u32x4 *>(xt), R.n_tiles = plan.n_tiles, R.tiles = plan.tiles, R.order = plan.order;
    R.inner = static_cast<uint8_t *>(inner), R.n_kb_inner = X.second.n_cells * 16u;
    R.activation = X.activation, R.gated = X.gated;
    const uint32_t n_kb = X.first.n_cells * 16u;
    const bool whole = ((uintptr_t)call.x & 15u) == 0 && call.ldx % 8 == 0 && X.hidden % 8u == 0;
    IXH_LAUNCH(k_experts_xtile, dim3(blocks, std::min((n_kb + 15u) / 16u, 16u)), dim3(256), 0, s, call.x, call.ldx, call.top_k, X.hidden, n_kb, whole,
               plan.n_blocks, plan.order, static_cast<ln_u32x4 *>(xt));
    int rc = ep_first(X.first, R, row_tiles, s);
    if (rc != IXH_OK) return rc;
    R.xt = static_cast<const ln_u32x4 *>(inner), R.out = per_slot;
    return ep_second(X.second, R, row_tiles, s);
}

}  // namespace ixh
