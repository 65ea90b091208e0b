// The experts' products of single tokens: each slot (token, j) by itself.
#include <algorithm>

#include "ixh_epilogue.h"
#include "ixh_experts.h"
#include "ixh_lanes_dev.h"

namespace ixh {

// ---------------------------------------------------------------------------------------------------------------
// k_experts_one<BITS, FIRST, JOIN, CELLS>: one slot by a run of blocks of 16 weight rows, a wave for each cell (16 rows x 512 columns), or for two of them.
//
// Bound: a launch, one chain of requests (the expert's id, then its codes, the extents of their lists, scale and activations at once, then the
// lists) and the instructions of a cell.  Products and listed elements as in k_experts_rows, of whose kernel for one row some 350 of 1100
// instructions a wave only find its share: one token by 6 experts of 2048 x 1024 at 5 bits, first / second matrix 13.2 / 9.6 us there, 9.2 / 6.4 us here
// (20.6 and 10.7 MB read; vector unit busy for 43 and 50 % of the CUs' time, LDS for 34 and 37 %, the second one joined as below).
//
// JOIN, the second matrix for a few tokens: a workgroup has a block of rows of all of a token's slots, with a pair table and activations for
// each, and ends with the sum over them, in their order, so that no launch follows: second matrix and sum 6.4 + 2.8 -> 7.8 us for that token.
// ---------------------------------------------------------------------------------------------------------------
struct EoJoin {  // what a token's outputs are made with
    const float *weights;
    const uint16_t *residual;
    int64_t ld_residual;
};
template <int BITS, bool FIRST, bool JOIN, int CELLS>
__global__ void __launch_bounds__(1024)
k_experts_one(const int32_t *__restrict__ ids, const uint32_t *__restrict__ plane, const uint16_t *__restrict__ x, const uint32_t *__restrict__ exc_off,
              const uint16_t *__restrict__ scale_at, uint32_t shape, uint32_t n_tiles, uint32_t plane_words, uint32_t experts, uint32_t in_f, int64_t ldx,
              const uint16_t *__restrict__ exc_pos, const int8_t *__restrict__ exc_val, const uint16_t *__restrict__ bias, void *out,
              int64_t ld_out, uint32_t outputs, int activation, EoJoin join) {
    extern __shared__ __attribute__((aligned(16))) uint8_t eo_smem[];
    using P = LnPairs<BITS, false>;
    const uint32_t smem = (uint32_t)(uintptr_t)(LN_LDS(uint8_t) *)eo_smem;
    // items: the workgroup's blocks of a slot, or (JOIN) a block of each of a token's slots; an item's cells to a wave each, or (CELLS = 2)
    // the first and the second half of them to the same waves
    const uint32_t C = shape & 31u, CW = CELLS == 2 ? (C + 1u) >> 1 : C, items = (shape >> 5) & 31u, inv_cells = shape >> 12;
    const bool gated = (shape >> 10) & 1u, whole = (shape >> 11) & 1u;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), item = (wave * inv_cells) >> 16, c = wave - item * CW;
    const uint32_t slot = JOIN ? blockIdx.z * items + item : blockIdx.z * gridDim.y + blockIdx.y, id = (uint32_t)ids[slot];
    if (!JOIN && id >= experts) return;
    const uint32_t e = min(id, experts - 1u);  // (what a place without an expert adds is not used)
    // the threads that share a pair table and a row of activations
    const uint32_t tid = JOIN ? threadIdx.x - item * CW * kWave : threadIdx.x, n_threads = (JOIN ? CW : items * CW) * kWave, own = JOIN ? item : 0u;
    const uint32_t lane = threadIdx.x & 63u, n = lane & 15u, kg = lane >> 4, b0 = blockIdx.x * (JOIN ? 1u : items), b = JOIN ? 0u : item;

    // ---- all requests ----
    const uint32_t scale_raw = scale_at[e];
    constexpr uint32_t kCell = 256u * BITS, kLane = BITS == 3 ? 12u : 16u;
    const __amdgpu_buffer_rsrc_t codes_rs = __builtin_amdgcn_make_buffer_rsrc((void *)(plane + (size_t)e * plane_words), 0, (int)(plane_words * 4u), 0x00020000);
    const uint32_t quad = 4u * (b0 + b), in_cell = 4u * kg + (n & 3u), codes = min(quad + (n >> 2), n_tiles - 1u) * (C * kCell) + in_cell * kLane;
    uint32_t w[CELLS][4][BITS], l0[CELLS], l1[CELLS];  // (a wave without a second cell: the last one, of which nothing is taken)
#pragma unroll
    for (uint32_t k = 0; k < CELLS; ++k) {
        const uint32_t cell = k ? min(c + CW, C - 1u) : c;
#pragma unroll
        for (uint32_t q = 0; q < 4; ++q) {
            uint32_t(&d)[BITS] = w[k][q];
            if constexpr (BITS == 3) {
                const ln_u32x3 v = __builtin_bit_cast(ln_u32x3, __builtin_amdgcn_raw_buffer_load_b96(codes_rs, (int)(codes + q * 192u), (int)(cell * kCell), 0));
                d[0] = v[0]; d[1] = v[1]; d[2] = v[2];
            } else {
                const ln_u32x4 v = __builtin_bit_cast(ln_u32x4, __builtin_amdgcn_raw_buffer_load_b128(codes_rs, (int)(codes + q * 256u), (int)(cell * kCell), 0));
                d[0] = v[0]; d[1] = v[1]; d[2] = v[2]; d[3] = v[3];
                if constexpr (BITS == 5)
                    d[4] = __builtin_amdgcn_raw_buffer_load_b32(codes_rs, (int)(codes - 12u * in_cell + (1024u + q * 64u)), (int)(cell * kCell), 0);
                if constexpr (BITS == 8) {
                    const ln_u32x4 u = __builtin_bit_cast(ln_u32x4, __builtin_amdgcn_raw_buffer_load_b128(codes_rs, (int)(codes + (1024u + q * 256u)), (int)(cell * kCell), 0));
                    d[4] = u[0]; d[5] = u[1]; d[6] = u[2]; d[7] = u[3];
                }
            }
        }
        const uint32_t *const off = exc_off + (size_t)e * (n_tiles * C + 1u) + (min(quad + kg, n_tiles - 1u) * C + cell);
        l0[k] = off[0], l1[k] = quad + kg < n_tiles && c + k * CW < C ? off[1] : l0[k];
    }
    // a piece of eight columns a thread: there are as many threads as pieces, or more
    const uint16_t *const row = x + (int64_t)(FIRST ? blockIdx.z : slot) * ldx;
    const uint32_t col = tid * 8u;
    ln_u32x4 piece = {0u, 0u, 0u, 0u};
    if (whole) {
        piece = *reinterpret_cast<const ln_u32x4 *>(row + min(col, in_f - 8u));
    } else {
        uint32_t h[8];
#pragma unroll
        for (uint32_t k = 0; k < 8; ++k) h[k] = row[min(col + k, in_f - 1u)];
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) piece[k] = (col + 2u * k < in_f ? h[2 * k] : 0u) | (col + 2u * k + 1u < in_f ? h[2 * k + 1] << 16 : 0u);
    }
    float plus = 0.0f, residual = 0.0f;
    if constexpr (JOIN) {
        if (bias && c == 0u && n < 4u) plus = bf16_bits_to_f32(bias[(size_t)e * outputs + min(b0 * 16u + 4u * kg + n, outputs - 1u)]);
        if (join.residual && threadIdx.x < 16u)
            residual = bf16_bits_to_f32(join.residual[(int64_t)blockIdx.z * join.ld_residual + min(b0 * 16u + threadIdx.x, outputs - 1u)]);
    }
    const float weight = JOIN ? join.weights[slot] : 0.0f;
    struct Group { ln_u32x2 pos; uint32_t val; };
    auto quad_of = [&](uint32_t k, uint32_t i) { return (l0[k] & ~3u) + 16u * i + (n & ~3u); };
    auto g_load = [&](uint32_t k, uint32_t i) {
        const uint32_t q = quad_of(k, i), at = q < l1[k] ? lane_listed(q, n & 3u) : 0u;
        return Group{*reinterpret_cast<const ln_u32x2 *>(exc_pos + at), *reinterpret_cast<const uint32_t *>(exc_val + at)};
    };
    Group list[CELLS][2];
#pragma unroll
    for (uint32_t k = 0; k < CELLS; ++k)
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) list[k][i] = g_load(k, i);
    __builtin_amdgcn_sched_barrier(0);

    // ---- pair table and activations to LDS ----
    const float scale = bf16_bits_to_f32(scale_raw);
    const uint32_t tables = JOIN ? items : 1u, x_none = C * 1024u, lut = smem + own * P::kLutBytes;
    ln_build_lut<BITS, false>(lut, scale, tid, n_threads);
    const uint32_t x_at = smem + tables * P::kLutBytes + own * (x_none + 64u);
    float *const parts = reinterpret_cast<float *>(eo_smem + tables * (P::kLutBytes + x_none + 64u));  // [wave][16]
    float *const pluses = parts + items * CW * 16u, *const item_weights = pluses + items * 16u;         // JOIN: [item][16], [item]{weight, whether it has an expert}
    if (tid < C * 64u) {
        if (whole && col >= in_f) piece = ln_u32x4{0u, 0u, 0u, 0u};
        *reinterpret_cast<LN_LDS(ln_u32x4) *>((uintptr_t)(x_at + lane_offset(col))) = piece;
    }
    if (tid < 4u) *reinterpret_cast<LN_LDS(ln_u32x4) *>((uintptr_t)(x_at + x_none + tid * 16u)) = ln_u32x4{0u, 0u, 0u, 0u};
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");

    // ---- a cell's products: the row's activations in all sixteen columns (columns 128 q + 32 i of a cell lie at 128 q + 32 (i ^ q)) ----
    const uint32_t lut_lane = lut + ((lane & ((1u << P::kCopies) - 1u)) << 2), x_cell = x_at + c * 1024u + kg * 16u;
    ln_f32x4 acc = {0, 0, 0, 0};
    float ex = 0.0f;
    const uint32_t scale_bits = __float_as_uint(scale) & 0x7FFFFFFFu;
    auto listed = [&](const Group &g, uint32_t k, uint32_t i) {
        const uint32_t q = quad_of(k, i) - l0[k];
        const uint32_t w01 = ln_pack((float)(int)(int8_t)g.val * scale, (float)(int)(int8_t)(g.val >> 8) * scale);
        const uint32_t w23 = ln_pack((float)(int)(int8_t)(g.val >> 16) * scale, (float)((int)g.val >> 24) * scale);
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            const uint32_t p = j & 1 ? g.pos[j >> 1] >> 16 : g.pos[j >> 1] & 0xFFFFu;  // (rows of up to 16 cells: places without an element have one of their own)
            const uint32_t h = *reinterpret_cast<const LN_LDS(uint16_t) *>((uintptr_t)(x_at + (q + j < l1[k] - l0[k] ? p : x_none)));
            const uint32_t wj = j & 2 ? w23 : w01, wbits = j & 1 ? wj & 0xFFFF0000u : wj << 16;
            ex = __fmaf_rn(__uint_as_float(wbits) - __uint_as_float((wbits & 0x80000000u) | scale_bits), __uint_as_float(h << 16), ex);
        }
    };
#pragma unroll
    for (uint32_t k = 0; k < CELLS; ++k) {
        if (k && c + CW >= C) break;
#pragma unroll
        for (uint32_t q = 0; q < 4; ++q) {
            uint32_t o[16];
            ln_decode<BITS, false>(w[k][q], lut_lane, scale, o);
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const ln_u32x4 a = *reinterpret_cast<const LN_LDS(ln_u32x4) *>((uintptr_t)(x_cell + k * CW * 1024u + q * 256u + ((q ^ i) << 6)));
                acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(ln_bf16x8, ln_u32x4{o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]}),
                                                              __builtin_bit_cast(ln_bf16x8, a), acc, 0, 0, 0);
            }
        }
        // its listed elements
        const uint32_t groups = l1[k] > l0[k] ? (l1[k] - (l0[k] & ~3u) + 15u) / 16u : 0u;
        if (__any(groups > 0u)) listed(list[k][0], k, 0);
        if (__any(groups > 1u)) listed(list[k][1], k, 1);
#pragma unroll 1
        for (uint32_t i = 2; __any(groups > i); ++i) listed(g_load(k, i), k, i);
    }
    ex += ln_dpp<0x124>(ex);
    ex += ln_dpp<0x128>(ex);
    // row 4 kg + k: the plane's sum is acc[k] of any lane of kg, the list's is with lane n = k
    const float plane_sum = n == 0u ? acc[0] : n == 1u ? acc[1] : n == 2u ? acc[2] : acc[3];
    if (n < 4u) parts[wave * 16u + 4u * kg + n] = plane_sum + ex;
    if constexpr (JOIN) {
        if (c == 0u) {
            if (n < 4u) pluses[item * 16u + 4u * kg + n] = plus;
            if (lane == 0u) item_weights[2u * item] = weight, item_weights[2u * item + 1u] = id < experts ? 1.0f : 0.0f;
        }
        __syncthreads();
        // y = residual + the sum over the slots, in their order
        const uint32_t row_out = b0 * 16u + threadIdx.x;
        if (threadIdx.x >= 16u || row_out >= outputs) return;
        float v = 0.0f;
        for (uint32_t j = 0; j < items; ++j) {
            float p = 0.0f;
            for (uint32_t k = 0; k < CW; ++k) p += parts[(j * CW + k) * 16u + threadIdx.x];
            if (bias) p += pluses[j * 16u + threadIdx.x];
            if (item_weights[2u * j + 1u] != 0.0f) v = __fmaf_rn(item_weights[2u * j], p, v);
        }
        static_cast<uint16_t *>(out)[(int64_t)blockIdx.z * ld_out + row_out] = ep_bf16(join.residual ? v + residual : v);
        return;
    }
    __syncthreads();

    // ---- outputs: a row's sums over the columns ----
    const uint32_t per = FIRST && gated ? 2u : 1u, at = tid & 15u, of = tid >> 4, out_row = (b0 / per + of) * 16u + at;
    if (of * per >= items || out_row >= outputs) return;
    auto sum_of = [&](uint32_t block) {
        float v = 0.0f;
        for (uint32_t k = 0; k < CW; ++k) v += parts[(block * CW + k) * 16u + at];
        return v;
    };
    const uint16_t *const biases = bias ? bias + (size_t)e * (per * outputs) : nullptr;
    float v = sum_of(of * per);
    if (biases) v += bf16_bits_to_f32(biases[out_row]);
    if constexpr (FIRST) {
        v = ep_activation(activation, v);
        if (gated) {
            float u = sum_of(of * 2u + 1u);
            if (biases) u += bf16_bits_to_f32(biases[outputs + out_row]);
            v *= u;
        }
        static_cast<uint16_t *>(out)[(int64_t)slot * ld_out + out_row] = ep_bf16(v);
    } else {
        static_cast<float *>(out)[(int64_t)slot * ld_out + out_row] = v;
    }
}

// Cells of a wave: two where sixteen waves are too few for the cells of a gated pair of blocks (an item of one block has threads for its activations
// with a cell each only).  One token by 2 of 16 experts of 5120 x 1536: 20.8 us a call, of k_experts_rows 27.
static uint32_t eo_cells(const ExMatrix &W, uint32_t per) { return per == 2u && W.n_cells > 8u ? 2u : 1u; }
static uint32_t eo_waves(const ExMatrix &W, uint32_t per) { return eo_cells(W, per) == 2u ? (W.n_cells + 1u) / 2u : W.n_cells; }  // of a block
bool experts_one_takes(const ExMatrix &W, bool gated) { return W.n_cells <= 16u && eo_waves(W, gated ? 2u : 1u) * (gated ? 2u : 1u) <= 16u; }

// blocks of a workgroup: as many as sixteen waves have cells for, and few enough for a workgroup to each CU
static uint32_t eo_blocks(const ExMatrix &W, uint32_t per, uint32_t slots) {
    const uint32_t all = (W.n_tiles + 3u) / 4u;
    return std::max(std::min(std::min(16u / eo_waves(W, per), all * slots / ln_cus()), all) / per * per, per);
}

template <int BITS, bool JOIN> static size_t eo_lds(uint32_t C, uint32_t items, uint32_t CW) {
    return (JOIN ? items : 1u) * (LnPairs<BITS, false>::kLutBytes + C * 1024u + 64u) + items * CW * 64u + (JOIN ? items * 72u : 0u);
}

template <int BITS, bool FIRST, bool JOIN, int CELLS> static int eo_launch(const ExMatrix &W, const ExOne &R, hipStream_t s) {
    const uint32_t per = FIRST && R.gated ? 2u : 1u, C = W.n_cells, CW = CELLS == 2 ? (C + 1u) / 2u : C, all = (W.n_tiles + 3u) / 4u;
    const uint32_t blocks = JOIN ? 1u : eo_blocks(W, per, R.tokens * R.top_k), items = JOIN ? R.top_k : blocks;
    if (C > 16u || items * CW > 16u || (CELLS == 2 && (JOIN || items < 2u))) return IXH_EUNSUPPORTED;
    const bool whole = ((uintptr_t)R.x & 15u) == 0 && W.in_f % 8u == 0 && (R.ldx % 8 == 0 || R.rows == 1u);
    const size_t lds = eo_lds<BITS, JOIN>(C, items, CW);
    if constexpr (JOIN) {
        static const bool raised = hipFuncSetAttribute(reinterpret_cast<const void *>(k_experts_one<BITS, FIRST, JOIN, CELLS>),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, (int)kLnLds) == hipSuccess;
        if (!raised || lds > kLnLds) return IXH_ELAUNCH;
    }
    // (a wave / CW as a product with 2^16 / CW, rounded up: exact for sixteen waves)
    const uint32_t shape = C | items << 5 | (uint32_t)R.gated << 10 | (uint32_t)whole << 11 | (65536u / CW + 1u) << 12;
    IXH_LAUNCH((k_experts_one<BITS, FIRST, JOIN, CELLS>), dim3((all + blocks - 1u) / blocks, JOIN ? 1u : R.top_k, R.tokens), dim3(items * CW * kWave), lds, s,
               R.ids, W.plane, R.x, W.exc_off, W.scale, shape, W.n_tiles, (uint32_t)W.plane_words, R.experts, W.in_f, R.ldx, W.exc_pos, W.exc_val, W.bias,
               R.out, R.ld_out, W.outputs, R.activation, EoJoin{R.weights, R.residual, R.ld_residual});
    return hipGetLastError() == hipSuccess ? IXH_OK : IXH_ELAUNCH;
}
template <bool FIRST, bool JOIN, int CELLS> static int eo_matrix(const ExMatrix &W, const ExOne &R, hipStream_t s) {
    switch (W.bits) {
        case 3: return eo_launch<3, FIRST, JOIN, CELLS>(W, R, s);
        case 4: return eo_launch<4, FIRST, JOIN, CELLS>(W, R, s);
        case 5: return eo_launch<5, FIRST, JOIN, CELLS>(W, R, s);
        default: return eo_launch<8, FIRST, JOIN, CELLS>(W, R, s);
    }
}
int launch_experts_one(const ExMatrix &W, const ExOne &R, bool first, hipStream_t s) {
    if (!first) return eo_matrix<false, false, 1>(W, R, s);
    return eo_cells(W, R.gated ? 2u : 1u) == 2u ? eo_matrix<true, false, 2>(W, R, s) : eo_matrix<true, false, 1>(W, R, s);
}

static size_t eo_joined_lds(const ExMatrix &W, uint32_t top_k) {
    switch (W.bits) {
        case 3: return eo_lds<3, true>(W.n_cells, top_k, W.n_cells);
        case 4: return eo_lds<4, true>(W.n_cells, top_k, W.n_cells);
        case 5: return eo_lds<5, true>(W.n_cells, top_k, W.n_cells);
        default: return eo_lds<8, true>(W.n_cells, top_k, W.n_cells);
    }
}
// Fewer than one and a half times as many workgroups (one to a block of rows and token, each with the tables and waves of all of the token's slots) as
// the CUs hold at once.  us of a call apart / joined, ids and weights others from call to call, 1 / 2 / 3 / 4 / 6 / 8 tokens by 6 of 64 experts of 2048 x
// 1024 at 5 bits (two workgroups a CU: up to five tokens) 18.3 / 24.8 / 31.2 / 32.9 / 42.9 / 48.0 and 16.5 / 21.0 / 28.1 / 30.1 / 41.0 / 48.1; by 8 (one:
// two tokens) 18.0 / 25.3 / 33.2 / 37.2 / 48.4 / 65.0 and 18.1 / 23.8 / 36.0 / 40.1 / 55.9 / -; by 8 of 128 of 2048 x 512 (two) 14.6 / 18.4 / 25.4 / 25.7 /
// 33.3 / 37.8 and 13.6 / 16.8 / 22.8 / 24.4 / 33.3 / 39.3; by 2 of 16 of 4096 x 1536 (five: seven tokens) 16.8 / 22.9 / 30.4 / 32.1 / 42.0 / 49.3 and 14.1 /
// 20.1 / 25.7 / 28.1 / 38.7 / 45.7; by 12 of 128 of 2048 x 512 at 3 bits (one) 15.5 / 19.3 / 23.7 / 24.9 / 32.2 / 35.9 and 13.9 / 16.8 / 25.7 / 27.4 / 38.0 /
// 46.9.  Over 924 calls (13 layers, planes of 3 to 8 bits, 1 to 16 slots and 1 to 12 tokens) this takes 0.5 % longer than the better one each time, never
// joined 13.7 %, always 1.5 %.
bool experts_joined_takes(const ExMatrix &W, uint32_t tokens, uint32_t top_k) {
    const uint64_t waves = (uint64_t)top_k * W.n_cells;
    if (waves > 16u) return false;
    const uint64_t a_cu = std::min<uint64_t>(kLnLds / eo_joined_lds(W, top_k), 32u / waves), all = (W.n_tiles + 3u) / 4u;
    return 2u * all * tokens < 3u * a_cu * ln_cus();
}
int launch_experts_joined(const ExMatrix &W, const ExOne &R, hipStream_t s) { return eo_matrix<false, true, 1>(W, R, s); }

}  // namespace ixh
