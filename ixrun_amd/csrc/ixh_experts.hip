// The experts' products over packed weights: y[t] = residual[t] + sum_j weights[t, j] * second_e(act(first_e(x[t]))), e = ids[t, j].
#include "ixh_experts.h"

#include <algorithm>

#include "ixh_epilogue.h"
#include "ixh_lanes_dev.h"

namespace ixh {

// ---------------------------------------------------------------------------------------------------------------
// k_experts_plan: the slots (token, j) that have an expert, by expert and in their order within one, cut into tiles of `rows` slots.
//
// A workgroup an expert, no two of which wait for each other: each counts the slots of all experts (in LDS; sums of whole numbers do not
// hang on their order), so it knows where its own begin, and then writes these.  Reads the ids twice, from the L2.
// ---------------------------------------------------------------------------------------------------------------
constexpr uint32_t kExPlanThreads = 1024, kExPlanWaves = kExPlanThreads / kWave;

// Tiles of an expert with n slots: of up to `rows` of them; with rows = 0 of up to 32 blocks of 16, as even as whole eights of blocks
// allow (what is left of an eighth is as long as the whole).
__device__ __forceinline__ uint32_t ex_eights(uint32_t n) { return (n + 127u) / 128u; }
__device__ __forceinline__ uint32_t ex_tiles(uint32_t n, uint32_t rows) { return rows ? (n + rows - 1u) / rows : (ex_eights(n) + 3u) / 4u; }
// How many of these are of 4, 3, 2 and 1 eights of blocks: the order of the tiles, so that the last ones to be taken are short.  (Tiles of
// `rows` slots are in the order of the experts.)
constexpr uint32_t kExSizes = 4;
struct ExSizes { uint32_t n[kExSizes]; };
__device__ __forceinline__ ExSizes ex_sizes(uint32_t n, uint32_t rows) {
    ExSizes of{};
    if (rows) {
        of.n[0] = ex_tiles(n, rows);
    } else if (n) {
        const uint32_t tiles = ex_tiles(n, 0), each = ex_eights(n) / tiles, longer = ex_eights(n) - each * tiles;
#pragma unroll
        for (uint32_t k = 0; k < kExSizes; ++k) of.n[k] = each == 4u - k ? tiles - longer : each + 1u == 4u - k ? longer : 0u;
    }
    return of;
}
__device__ __forceinline__ uint32_t ex_places(uint32_t n, uint32_t rows) { return rows ? n : (n + 15u) & ~15u; }

__global__ void __launch_bounds__(kExPlanThreads)
k_experts_plan(const int32_t *__restrict__ ids, uint32_t slots, uint32_t experts, uint32_t rows, ExPlan plan) {
    __shared__ uint32_t hist[kExMostExperts], of_wave[kExPlanWaves], sums[1u + kExSizes][kExPlanWaves];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, e = blockIdx.x;
    for (uint32_t i = tid; i < experts; i += kExPlanThreads) hist[i] = 0;
    __syncthreads();
    // a wave has whole 64 slots one after another
    const uint32_t share = ((slots + kExPlanThreads - 1u) / kExPlanThreads) * kWave, from = min(wave * share, slots), to = min(from + share, slots);
    constexpr uint32_t N = 8;  // ids of a lane in flight
    uint32_t mine = 0;
    for (uint32_t i0 = from; i0 < to; i0 += N * kWave) {
        uint32_t id[N];
#pragma unroll
        for (uint32_t k = 0; k < N; ++k) id[k] = (uint32_t)ids[min(i0 + k * kWave + lane, to - 1u)];
#pragma unroll
        for (uint32_t k = 0; k < N; ++k) {
            if (i0 + k * kWave + lane >= to) id[k] = ~0u;
            if (id[k] < experts) atomicAdd(hist + id[k], 1u);
            mine += id[k] == e;
        }
    }
    for (int by = 32; by; by >>= 1) mine += __shfl_xor(mine, by);
    if (lane == 0) of_wave[wave] = mine;
    __syncthreads();
    // in front of this expert: places, and, of each size, tiles; with them all tiles of larger sizes
    uint32_t sum[1u + kExSizes] = {};
    for (uint32_t i = tid; i < experts; i += kExPlanThreads) {
        const ExSizes of = ex_sizes(hist[i], rows);
        if (i < e) sum[0] += ex_places(hist[i], rows);
#pragma unroll
        for (uint32_t k = 0; k < kExSizes; ++k) {
            uint32_t larger = 0;
#pragma unroll
            for (uint32_t l = 0; l < k; ++l) larger += of.n[l];
            sum[1u + k] += larger + (i < e ? of.n[k] : 0u);
        }
    }
#pragma unroll
    for (uint32_t k = 0; k <= kExSizes; ++k) {
        for (int by = 32; by; by >>= 1) sum[k] += __shfl_xor(sum[k], by);
        if (lane == 0) sums[k][wave] = sum[k];
    }
    __syncthreads();
#pragma unroll
    for (uint32_t k = 0; k <= kExSizes; ++k) {
        sum[k] = 0;
        for (uint32_t w = 0; w < kExPlanWaves; ++w) sum[k] += sums[k][w];
    }
    const uint32_t before = sum[0], n = hist[e], n_tiles = ex_tiles(n, rows), places = ex_places(n, rows);
    const ExSizes own_sizes = ex_sizes(n, rows);
    for (uint32_t i = tid; i < n_tiles; i += kExPlanThreads) {
        if (rows) {
            uint32_t *const t = plan.tiles + 3u * (sum[1] + i);
            t[0] = e, t[1] = before + i * rows, t[2] = min(rows, n - i * rows);
        } else {  // the longer ones of an expert's tiles come first
            const uint32_t eights = ex_eights(n), each = eights / n_tiles, longer = eights - each * n_tiles;
            const uint32_t b0 = (i * each + min(i, longer)) * 8u, size = each + (i < longer);
            uint32_t at = i < longer ? i : i - longer;
#pragma unroll
            for (uint32_t k = 0; k < kExSizes; ++k) at += size == 4u - k ? sum[1u + k] : 0u;
            uint32_t *const t = plan.tiles + 3u * at;
            t[0] = e, t[1] = before / 16u + b0, t[2] = min(size * 8u, places / 16u - b0);
        }
    }
    for (uint32_t i = n + tid; i < places; i += kExPlanThreads) plan.order[before + i] = ~0u;
    if (e + 1u == experts && tid == 0) {
        *plan.n_tiles = rows ? sum[1] + n_tiles : sum[kExSizes] + own_sizes.n[kExSizes - 1u];  // (in front of this one: all larger ones, and all others')
        *plan.n_blocks = (before + places) / 16u;
    }
    uint32_t at = before;
    for (uint32_t w = 0; w < wave; ++w) at += of_wave[w];
    for (uint32_t i0 = from; i0 < to; i0 += N * kWave) {
        uint32_t id[N];
#pragma unroll
        for (uint32_t k = 0; k < N; ++k) id[k] = (uint32_t)ids[min(i0 + k * kWave + lane, to - 1u)];
#pragma unroll
        for (uint32_t k = 0; k < N; ++k) {
            const uint32_t i = i0 + k * kWave + lane;
            const bool own = i < to && id[k] == e;
            const uint64_t all = __ballot(own);
            if (own) plan.order[at + lanes_below(all)] = i;
            at += (uint32_t)__popcll(all);
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------
// k_experts_rows<BITS, MT, FIRST>: a tile of up to MT slots of one expert by a run of blocks of 16 weight rows.
//
// As in k_lanes_rows a lane's decoded weights are its operand of v_mfma_f32_16x16x32_bf16 as they are, the activations of the tile lie in
// LDS a column's rows together (transposing reads make them the other operand), and listed elements are multiplied in fp32 by the lane of
// their row.  A wave has whole cells of 512 columns of a block, and with a cell its list.  Rows longer than LDS holds are taken in
// chunks of cells; the sums stay in LDS over them.  FIRST: the rows are gathered from the tokens, and the epilogue is the bias, the
// activation and, gated, the product of the two halves; else they are those of the intermediate and the sums go out in fp32.
// ---------------------------------------------------------------------------------------------------------------
constexpr uint32_t kExWaves = 8, kExThreads = kExWaves * kWave;

struct ExRows {
    const uint16_t *x;
    int64_t ldx;
    const int32_t *ids;
    const uint32_t *n_tiles, *tiles, *order;  // n_tiles NULL: a tile is a slot
    void *out;
    int64_t ld_out;
    uint32_t experts, top_k, n_blocks, all_blocks, waves_along, chunk_cells;  // waves along the columns
    int activation;
    bool gated, pairs;
};

template <int BITS> constexpr uint32_t kExXAt = (LnPairs<BITS, BITS == 4>::kLutBytes + 4095u) & ~4095u;

template <int BITS, int MT, bool FIRST>
__global__ void __launch_bounds__(kExThreads) __attribute__((amdgpu_waves_per_eu(4)))
k_experts_rows(ExMatrix W, ExRows R) {
    extern __shared__ __attribute__((aligned(16))) uint8_t ex_smem[];
    using P = LnPairs<BITS, BITS == 4>;
    constexpr bool WIDE = BITS == 4;
    constexpr uint32_t ROW = 2u * MT;
    const uint32_t smem = (uint32_t)(uintptr_t)(LN_LDS(uint8_t) *)ex_smem;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, n = lane & 15u, kg = lane >> 4;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6));

    // ---- the tile ----
    uint32_t e, first = blockIdx.x, count = 1;
    if (R.n_tiles) {
        const uint32_t *const t = R.tiles + 3u * blockIdx.x;
        e = t[0], first = t[1], count = t[2];
        if (blockIdx.x >= *R.n_tiles) return;
    } else {
        e = (uint32_t)R.ids[blockIdx.x];
        if (e >= R.experts) return;
    }
    const uint32_t slot = R.n_tiles ? R.order[first + min(lane, count - 1u)] : first;  // of the tile's row `lane`
    const int64_t x_row = (int64_t)(FIRST ? slot / R.top_k : first + min(lane, count - 1u)) * R.ldx;
    const uint32_t b0 = blockIdx.y * R.n_blocks, n_blocks = min(R.n_blocks, R.all_blocks - b0);

    const uint32_t C = W.n_cells;
    const uint8_t *const plane = reinterpret_cast<const uint8_t *>(W.plane + (size_t)e * W.plane_words);
    const uint32_t *const exc_off = W.exc_off + (size_t)e * (W.n_tiles * C + 1u);
    const float scale = bf16_bits_to_f32(W.scale[e]);
    const uint32_t x_at = smem + kExXAt<BITS>, x_none = R.chunk_cells * kLnCols * ROW;
    float *const parts = reinterpret_cast<float *>(ex_smem + kExXAt<BITS> + x_none + 16u * ROW);  // [wave along][block][16][MT]
    constexpr uint32_t PART = 16u * MT;

    ln_build_lut<BITS, WIDE>(smem, scale, tid, kExThreads);
    for (uint32_t i = tid; i < R.waves_along * R.n_blocks * PART; i += kExThreads) parts[i] = 0.0f;
    if (tid < 16u) *reinterpret_cast<LN_LDS(ln_u32x4) *>((uintptr_t)(x_at + x_none + tid * 16u)) = ln_u32x4{0, 0, 0, 0};

    const uint32_t lut_lane = smem + ((lane & ((1u << P::kCopies) - 1u)) << 2);
    const uint32_t piece = MT == 16 ? n & 3u : n & 1u;
    const uint32_t x_mine = (x_at + lr_place<MT>((8u * kg + (n >> 2)) * ROW)) ^ (piece * 8u);
    const uint32_t scale_bits = __float_as_uint(scale) & 0x7FFFFFFFu;
    const uint32_t wc = wave % R.waves_along, wb = wave / R.waves_along, waves_across = kExWaves / R.waves_along;
    const uint32_t my_blocks = n_blocks > wb ? (n_blocks - wb + waves_across - 1u) / waves_across : 0u;

    for (uint32_t c0 = 0; c0 < C; c0 += R.chunk_cells) {
        const uint32_t cells = min(R.chunk_cells, C - c0);
        if (c0) __syncthreads();  // the last chunk's activations are in use until here
        // ---- activations: a pair of columns a lane, all rows ----
        for (uint32_t task = wave; task < 4u * cells; task += kExWaves) {
            const uint32_t col = c0 * kLnCols + task * 128u + 2u * lane;
            uint32_t v[MT];
#pragma unroll
            for (uint32_t k = 0; k < MT; ++k) {
                v[k] = 0;
                if (k < count) {
                    const uint16_t *const row = R.x + (((int64_t)__builtin_amdgcn_readlane((int)(x_row >> 32), (int)k) << 32) |
                                                       (uint32_t)__builtin_amdgcn_readlane((int)x_row, (int)k));
                    if (R.pairs) {
                        if (col < W.in_f) v[k] = *reinterpret_cast<const uint32_t *>(row + col);
                    } else {
                        if (col < W.in_f) v[k] = row[col];
                        if (col + 1u < W.in_f) v[k] |= (uint32_t)row[col + 1u] << 16;
                    }
                }
            }
            const uint32_t to = lane_offset(task * 128u + 2u * lane) * MT;
#pragma unroll
            for (uint32_t j = 0; j < 2; ++j)
#pragma unroll
                for (uint32_t h = 0; h < MT / 8u; ++h) {
                    ln_u32x4 o;
#pragma unroll
                    for (uint32_t k = 0; k < 4; ++k)
                        o[k] = __builtin_amdgcn_perm(v[8 * h + 2 * k + 1], v[8 * h + 2 * k], j ? 0x07060302u : 0x05040100u);
                    *reinterpret_cast<LN_LDS(ln_u32x4) *>((uintptr_t)(x_at + (lr_place<MT>(to + j * ROW) ^ (h * 16u)))) = o;
                }
        }
        __syncthreads();

        // ---- this wave's cells: those of its share of the chunk, block after block ----
        const uint32_t c_lo = cells * wc / R.waves_along, c_n = cells * (wc + 1u) / R.waves_along - c_lo;
        const uint32_t units = my_blocks * c_n;
        if (units == 0) continue;
        struct Cursor { uint32_t j, c; };  // its j-th block, cell c of its share
        auto after = [&](const Cursor &k) { return k.c + 1u < c_n ? Cursor{k.j, k.c + 1u} : k.j + 1u < my_blocks ? Cursor{k.j + 1u, 0u} : k; };
        auto quad = [&](const Cursor &k, uint32_t q) { return 4u * (b0 + wb + k.j * waves_across) + q; };
        uint32_t w[2][BITS];
        auto load = [&](const Cursor &k, uint32_t half) {
            const uint32_t t = min(quad(k, n >> 2), W.n_tiles - 1u);
            const uint8_t *const cell = plane + (size_t)(t * C + c0 + c_lo + k.c) * (256u * BITS);
#pragma unroll
            for (uint32_t j = 0; j < 2; ++j)
                ln_load_lane<BITS>(reinterpret_cast<const uint32_t *>(cell), 32u * half + 16u * j + 4u * kg + (n & 3u), w[j]);
        };
        struct Extent { uint32_t first, end; };
        auto extent = [&](const Cursor &k) {
            const uint32_t t = quad(k, kg), cell = min(t, W.n_tiles - 1u) * C + c0 + c_lo + k.c;
            const uint32_t a = exc_off[cell], b = exc_off[cell + 1u];
            return Extent{a, t < W.n_tiles ? b : a};
        };
        struct Group { ln_u32x2 pos; uint32_t val; };
        auto quad_of = [&](const Extent &x, uint32_t i) { return (x.first & ~3u) + 16u * i + (n & ~3u); };
        auto g_load = [&](const Extent &x, uint32_t i) {
            const uint32_t q = quad_of(x, i), at = q < x.end ? lane_listed(q, n & 3u) : 0u;
            return Group{*reinterpret_cast<const ln_u32x2 *>(W.exc_pos + at), *reinterpret_cast<const uint32_t *>(W.exc_val + at)};
        };
        auto groups_of = [&](const Extent &x) {  // of the row quad that has most
            const int g = (int)(x.end > x.first ? (x.end - (x.first & ~3u) + 15u) / 16u : 0u);
            return (uint32_t)max(max(__builtin_amdgcn_readlane(g, 0), __builtin_amdgcn_readlane(g, 16)),
                                 max(__builtin_amdgcn_readlane(g, 32), __builtin_amdgcn_readlane(g, 48)));
        };
        Cursor now{0u, 0u}, next = after(now);
        load(now, 0);
        Extent e_now = extent(now), e_next = extent(next);
        Group list[2];
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) list[i] = g_load(e_now, i);
        ln_f32x4 acc = {0, 0, 0, 0};
        float ex[MT];
#pragma unroll
        for (int r = 0; r < MT; ++r) ex[r] = 0.0f;
        const uint32_t c_seg = c0 * 1024u;
        auto listed = [&](const Group &g, const Extent &x, uint32_t i) {
            const uint32_t q = quad_of(x, i);
            uint32_t at[4];
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) {
                const uint32_t p = ((g.pos[k >> 1] >> (16 * (k & 1))) - c_seg) & 0xFFFFu;
                const bool is = q + k >= x.first && q + k < x.end && ((g.val >> (8 * k)) & 255u);
                at[k] = is ? min(p * MT, x_none) : x_none;
            }
            const uint32_t w01 = ln_pack((float)(int)(int8_t)g.val * scale, (float)(int)(int8_t)(g.val >> 8) * scale);
            const uint32_t w23 = ln_pack((float)(int)(int8_t)(g.val >> 16) * scale, (float)((int)g.val >> 24) * scale);
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) {
                const uint32_t wk = k & 2 ? w23 : w01, wbits = k & 1 ? wk & 0xFFFF0000u : wk << 16;
                const float wv = __uint_as_float(wbits) - __uint_as_float((wbits & 0x80000000u) | scale_bits);  // (no element: times 0)
#pragma unroll
                for (uint32_t h = 0; h < MT / 8u; ++h) {
                    const ln_u32x4 v = *reinterpret_cast<const LN_LDS(ln_u32x4) *>((uintptr_t)(x_at + (lr_place<MT>(at[k]) ^ (h * 16u))));
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j) {
                        ex[8 * h + 2 * j] = __fmaf_rn(wv, __uint_as_float(v[j] << 16), ex[8 * h + 2 * j]);
                        ex[8 * h + 2 * j + 1] = __fmaf_rn(wv, __uint_as_float(v[j] & 0xFFFF0000u), ex[8 * h + 2 * j + 1]);
                    }
                }
            }
        };
#pragma unroll 1
        for (uint32_t u = 0; u < units; ++u) {
            const uint32_t x_cell = x_mine + (c_lo + now.c) * (512u * ROW);
#pragma unroll
            for (uint32_t half = 0; half < 2; ++half) {
                uint32_t o[2][16];
                ln_decode<BITS, WIDE>(w[0], lut_lane, scale, o[0]);
                ln_decode<BITS, WIDE>(w[1], lut_lane, scale, o[1]);
                load(half ? next : now, half ^ 1u);
                // (columns 128 q + 32 i of a cell lie at 128 q + 32 (i ^ q))
#pragma unroll
                for (uint32_t j = 0; j < 2; ++j)
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i) {
                        const uint32_t q = 2u * half + j, a = (x_cell + q * (128u * ROW)) ^ ((q ^ i) * (32u * ROW));
                        const lr_bf16x4 lo = lr_turned(a), hi = lr_turned(MT == 16 ? a ^ (4u * ROW) : a + 4u * ROW);
                        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                            __builtin_bit_cast(ln_bf16x8, ln_u32x4{o[j][4 * i], o[j][4 * i + 1], o[j][4 * i + 2], o[j][4 * i + 3]}),
                            __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7), acc, 0, 0, 0);
                    }
            }
            const uint32_t groups = groups_of(e_now);
            if (groups) listed(list[0], e_now, 0);
            if (groups > 1u) listed(list[1], e_now, 1);
#pragma unroll 1
            for (uint32_t i = 2; i < groups; ++i) listed(g_load(e_now, i), e_now, i);
            if (next.j != now.j || u + 1u == units) {
                // the block's sums: of listed elements over the four lanes of a row, of the plane as they are
                float *const part = parts + (wc * R.n_blocks + wb + now.j * waves_across) * PART;
#pragma unroll
                for (int r = 0; r < MT; ++r) {
                    ex[r] += ln_dpp<0x124>(ex[r]);
                    ex[r] += ln_dpp<0x128>(ex[r]);
                }
                if (n < 4u)
#pragma unroll
                    for (uint32_t r = 0; r < MT; ++r) part[(4u * kg + n) * MT + r] += ex[r];
                ln_wave_order();
                if (n < MT)
#pragma unroll
                    for (uint32_t k = 0; k < 4; ++k) part[(4u * kg + k) * MT + n] += acc[k];
                ln_wave_order();
                acc = ln_f32x4{0, 0, 0, 0};
#pragma unroll
                for (int r = 0; r < MT; ++r) ex[r] = 0.0f;
            }
            now = next;
            next = after(now);
            e_now = e_next;
#pragma unroll
            for (uint32_t i = 0; i < 2; ++i) list[i] = g_load(e_now, i);
            e_next = extent(next);
        }
    }
    __syncthreads();

    // ---- outputs: the waves' parts, in column order ----
    auto sum_of = [&](uint32_t block, uint32_t row, uint32_t r) {
        float v = 0.0f;
        for (uint32_t k = 0; k < R.waves_along; ++k) v += parts[(k * R.n_blocks + block) * PART + row * MT + r];
        return v;
    };
    const uint32_t per = FIRST && R.gated ? 2u : 1u, n_out = n_blocks / per * 16u, at0 = b0 / per * 16u;
    const uint16_t *const bias = W.bias ? W.bias + (size_t)e * (per * W.outputs) : nullptr;
    for (uint32_t i = tid; i < n_out * count; i += kExThreads) {
        const uint32_t r = i / n_out, at = i - r * n_out, block = (at >> 4) * per, row = at & 15u, out = at0 + at;
        if (out >= W.outputs) continue;
        float v = sum_of(block, row, r);
        if (bias) v += bf16_bits_to_f32(bias[out]);
        if constexpr (FIRST) {
            v = ep_activation(R.activation, v);
            if (R.gated) {
                float u = sum_of(block + 1u, row, r);
                if (bias) u += bf16_bits_to_f32(bias[W.outputs + out]);
                v *= u;
            }
            static_cast<uint16_t *>(R.out)[(int64_t)(first + r) * R.ld_out + out] = ep_bf16(v);
        } else {
            const uint32_t to = R.n_tiles ? R.order[first + r] : first;
            static_cast<float *>(R.out)[(int64_t)to * R.ld_out + out] = v;
        }
    }
}

// y[t] = residual[t] + sum_j weights[t, j] * (what its expert made of it), in the order of j.  Bound: memory.  N columns a thread.
template <int N>
__global__ void __launch_bounds__(256)
k_experts_join(const float *__restrict__ per_slot, ExCall call, uint32_t experts, uint32_t hidden) {
    const uint32_t t = blockIdx.x, at = (blockIdx.y * 256u + threadIdx.x) * N;
    if (at >= hidden) return;
    typedef float Sums __attribute__((ext_vector_type(4)));
    float v[N] = {};
    const int32_t *const ids = call.ids + (size_t)t * call.top_k;
    const float *const weights = call.weights + (size_t)t * call.top_k;
    const float *const from = per_slot + (size_t)t * call.top_k * hidden + at;
#pragma unroll 4
    for (uint32_t j = 0; j < call.top_k; ++j) {
        if ((uint32_t)ids[j] >= experts) continue;
        const float w = weights[j];
        if constexpr (N == 4) {
            const Sums p = *reinterpret_cast<const Sums *>(from + (size_t)j * hidden);
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = __fmaf_rn(w, p[k], v[k]);
        } else {
            v[0] = __fmaf_rn(w, from[(size_t)j * hidden], v[0]);
        }
    }
    uint16_t *const y = call.y + (int64_t)t * call.ldy + at;
    const uint16_t *const residual = call.residual + (int64_t)t * call.ld_residual + at;
#pragma unroll
    for (int k = 0; k < N; ++k) y[k] = ep_bf16(call.residual ? v[k] + bf16_bits_to_f32(residual[k]) : v[k]);
}

// ---- host ----
struct ExShape { uint32_t rows, n_blocks, waves_along, chunk_cells; size_t lds; };

template <int BITS>
static size_t ex_lds(uint32_t rows, uint32_t cells, uint32_t waves_along, uint32_t n_blocks) {
    return kExXAt<BITS> + (size_t)(cells * kLnCols + 16u) * 2u * rows + (size_t)waves_along * n_blocks * 16u * rows * sizeof(float);
}

// How a matrix is cut: blocks of a workgroup, waves along the columns, cells of a chunk.
template <int BITS>
static ExShape ex_shape(const ExMatrix &W, uint32_t rows, uint32_t n_tiles, uint32_t step) {
    const uint32_t all = (W.n_tiles + 3u) / 4u;
    ExShape p{};
    p.rows = rows;
    // as many blocks to a workgroup as leave two workgroups to a CU
    const uint32_t wanted = std::max(2u * ln_cus() / std::max(n_tiles, 1u), 1u);
    p.n_blocks = std::min(std::max((all + wanted - 1u) / wanted, step), 16u);
    p.n_blocks = (p.n_blocks + step - 1u) / step * step;
    p.waves_along = 1;
    while (p.waves_along < kExWaves && p.n_blocks * p.waves_along < kExWaves && 2u * p.waves_along <= W.n_cells) p.waves_along *= 2u;
    for (uint32_t chunks = 1;; ++chunks) {
        p.chunk_cells = (W.n_cells + chunks - 1u) / chunks;
        if (p.chunk_cells == 1u) break;
        if (p.chunk_cells <= kLnSegCells && ex_lds<BITS>(rows, p.chunk_cells, p.waves_along, p.n_blocks) <= kLnLds / 2u) break;
    }
    p.lds = ex_lds<BITS>(rows, p.chunk_cells, p.waves_along, p.n_blocks);
    return p;
}

template <int BITS, int MT, bool FIRST>
static int ex_rows(const ExMatrix &W, ExRows R, uint32_t n_tiles, hipStream_t s) {
    const uint32_t step = FIRST && R.gated ? 2u : 1u;
    const ExShape p = ex_shape<BITS>(W, MT, n_tiles, step);
    if (p.lds > kLnLds) return IXH_EUNSUPPORTED;
    static const bool raised = hipFuncSetAttribute(reinterpret_cast<const void *>(k_experts_rows<BITS, MT, FIRST>),
                                                   hipFuncAttributeMaxDynamicSharedMemorySize, (int)kLnLds) == hipSuccess;
    if (!raised) return IXH_ELAUNCH;
    R.n_blocks = p.n_blocks, R.all_blocks = (W.n_tiles + 3u) / 4u, R.waves_along = p.waves_along, R.chunk_cells = p.chunk_cells;
    R.pairs = ((uintptr_t)R.x & 3u) == 0 && W.in_f % 2u == 0 && R.ldx % 2 == 0;
    IXH_LAUNCH((k_experts_rows<BITS, MT, FIRST>), dim3(n_tiles, (R.all_blocks + p.n_blocks - 1u) / p.n_blocks), dim3(kExThreads), p.lds, s, W, R);
    return hipGetLastError() == hipSuccess ? IXH_OK : IXH_ELAUNCH;
}

template <bool FIRST> static int ex_matrix(const ExMatrix &W, const ExRows &R, uint32_t rows, uint32_t n_tiles, hipStream_t s) {
#define EX_ROWS(B) (rows <= 8 ? ex_rows<B, 8, FIRST>(W, R, n_tiles, s) : ex_rows<B, 16, FIRST>(W, R, n_tiles, s))
    switch (W.bits) {
        case 3: return EX_ROWS(3);
        case 4: return EX_ROWS(4);
        case 5: return EX_ROWS(5);
        default: return EX_ROWS(8);
    }
#undef EX_ROWS
}

// Many tokens to an expert: 16 and more in the mean.
// (Rows of up to 2^20 columns: offsets within a tile's rows are 32 bits.)
static bool ex_many(const ExDev &X, uint32_t slots) {
    return slots >= 16u * X.experts && std::max(X.first.n_cells, X.second.n_cells) <= 2048u;
}

// A call's scratch: the plan, the intermediate, what each slot's expert makes of it, and in k_experts_prompt the gathered rows.
struct ExScratch {
    bool many;
    uint32_t rows, n_tiles, blocks;  // slots of a tile (0: see ExPlan); tiles and blocks at most
    size_t tiles, order, x, inner, per_slot, bytes;
    int64_t ld_inner;
};
static ExScratch ex_scratch(const ExDev &X, uint32_t tokens, uint32_t top_k) {
    ExScratch w{};
    const uint32_t slots = tokens * top_k;
    w.many = ex_many(X, slots);
    size_t at = 256;
    auto take = [&](size_t n) { const size_t from = at; at += (n + 255u) & ~(size_t)255u; return from; };
    if (w.many) {
        w.n_tiles = std::min(slots, X.experts) + slots / 512u;
        w.blocks = std::min(slots, X.experts) + slots / 16u;
        w.tiles = take((size_t)w.n_tiles * 12u);
        w.order = take((size_t)w.blocks * 64u);
        w.x = take((size_t)w.blocks * X.first.n_cells * 16384u);
        w.inner = take((size_t)w.blocks * X.second.n_cells * 16384u);
    } else {
        w.rows = slots <= 4u * X.experts ? 8u : 16u;
        w.n_tiles = std::min(slots, X.experts + slots / 8u);
        w.tiles = take((size_t)w.n_tiles * 12u);
        w.order = take((size_t)slots * 4u);
        w.ld_inner = (int64_t)((X.inner + 7u) & ~7u);  // rows of whole 16 bytes
        w.inner = take((size_t)slots * (size_t)w.ld_inner * 2u);
    }
    w.per_slot = take((size_t)slots * X.hidden * 4u);
    w.bytes = at + 255u;  // to the next whole 256 bytes of whatever address is given
    return w;
}

// Callers may hold a scratch of a larger call: enough for any count of tokens up to this one.
size_t experts_workspace_bytes(const ExDev &X, uint32_t tokens, uint32_t top_k) {
    if (!tokens) return 0;
    const uint32_t few = std::min(tokens, (16u * X.experts - 1u) / top_k);  // the most that are not many
    return std::max(ex_scratch(X, tokens, top_k).bytes, few ? ex_scratch(X, few, top_k).bytes : 0u);
}

int launch_experts(const ExDev &X, const ExCall &call, void *workspace, hipStream_t s) {
    const uint32_t slots = call.tokens * call.top_k;
    const ExScratch w = ex_scratch(X, call.tokens, call.top_k);
    uint8_t *const ws = reinterpret_cast<uint8_t *>(((uintptr_t)workspace + 255u) & ~(uintptr_t)255u);
    const bool planned = w.many || (slots > X.experts / 4u && call.tokens > 1u);
    const uint32_t n_tiles = planned ? w.n_tiles : slots;
    uint32_t *const counts = reinterpret_cast<uint32_t *>(ws);
    const ExPlan plan{counts, counts + 1, reinterpret_cast<uint32_t *>(ws + w.tiles), reinterpret_cast<uint32_t *>(ws + w.order)};
    float *const per_slot = reinterpret_cast<float *>(ws + w.per_slot);
    if (planned) IXH_LAUNCH(k_experts_plan, dim3(X.experts), dim3(kExPlanThreads), 0, s, call.ids, slots, X.experts, w.rows, plan);
    int rc;
    if (w.many) {
        rc = launch_experts_prompt(X, call, plan, n_tiles, w.blocks, ws + w.x, ws + w.inner, per_slot, s);
    } else {
        ExRows R{};
        R.x = call.x, R.ldx = call.ldx, R.ids = call.ids, R.experts = X.experts, R.top_k = call.top_k;
        if (planned) R.n_tiles = plan.n_tiles, R.tiles = plan.tiles, R.order = plan.order;
        R.out = ws + w.inner, R.ld_out = w.ld_inner, R.activation = X.activation, R.gated = X.gated;
        rc = ex_matrix<true>(X.first, R, planned ? w.rows : 1u, n_tiles, s);
        if (rc != IXH_OK) return rc;
        R.x = reinterpret_cast<const uint16_t *>(ws + w.inner), R.ldx = w.ld_inner;
        R.out = per_slot, R.ld_out = X.hidden;
        rc = ex_matrix<false>(X.second, R, planned ? w.rows : 1u, n_tiles, s);
    }
    if (rc != IXH_OK) return rc;
    if (X.hidden % 4u == 0)
        IXH_LAUNCH(k_experts_join<4>, dim3(call.tokens, (X.hidden / 4u + 255u) / 256u), dim3(256), 0, s, per_slot, call, X.experts, X.hidden);
    else
        IXH_LAUNCH(k_experts_join<1>, dim3(call.tokens, (X.hidden + 255u) / 256u), dim3(256), 0, s, per_slot, call, X.experts, X.hidden);
    return hipGetLastError() == hipSuccess ? IXH_OK : IXH_ELAUNCH;
}

}  // namespace ixh
