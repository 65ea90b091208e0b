// The experts' products over packed weights: y[t] = residual[t] + sum_j weights[t, j] * second_e(act(first_e(x[t]))), e = ids[t, j].
#include "ixh_experts.h"

#include <algorithm>
#include <type_traits>

#include "ixh_epilogue.h"
#include "ixh_lanes_dev.h"

namespace ixh {

// ---------------------------------------------------------------------------------------------------------------
// k_experts_plan: the slots (token, j) that have an expert, by expert and in their order within one, cut into tiles of `rows` slots.
//
// A workgroup an expert, no two of which wait for each other: each counts the slots of all experts (in LDS; sums of whole numbers do not
// hang on their order), so it knows where its own begin, and then writes these.
//
// Bound: a launch and two waits for memory with few slots (384 and 615 slots of 64 and 20 experts 5.2 us), the counting in LDS with many
// (24576 slots of 64 experts 12 us; ids that all are kept from the first look to the second make no difference there).
// ---------------------------------------------------------------------------------------------------------------
constexpr uint32_t kExPlanThreads = 1024, kExPlanWaves = kExPlanThreads / kWave;

// How an expert's slots are cut into tiles: of up to `rows` of them; with rows = 0 of up to `most` layers, a layer being 64 slots, a block of 16
// to each wave of k_experts_prompt, as even as whole layers allow (what is left of a layer takes as long as the whole).
constexpr uint32_t kExLayer = 64;
struct ExCut {
    uint32_t rows, most;  // most: layers of a tile
    __device__ __forceinline__ uint32_t layers(uint32_t n) const { return (n + kExLayer - 1u) / kExLayer; }
    __device__ __forceinline__ uint32_t tiles(uint32_t n) const { return rows ? (n + rows - 1u) / rows : (layers(n) + most - 1u) / most; }
    __device__ __forceinline__ uint32_t places(uint32_t n) const { return rows ? n : (n + 15u) & ~15u; }
};
// How many of these are of 4, 3, 2 and 1 layers: the order of the tiles, so that the last ones to be taken are short.  (Tiles of `rows` slots
// are in the order of the experts.)
constexpr uint32_t kExSizes = 4;
struct ExSizes { uint32_t n[kExSizes]; };
__device__ __forceinline__ ExSizes ex_sizes(uint32_t n, const ExCut &cut) {
    ExSizes of{};
    if (cut.rows) {
        of.n[0] = cut.tiles(n);
    } else if (n) {
        const uint32_t tiles = cut.tiles(n), each = cut.layers(n) / tiles, longer = cut.layers(n) - each * tiles;
#pragma unroll
        for (uint32_t k = 0; k < kExSizes; ++k) of.n[k] = each == 4u - k ? tiles - longer : each + 1u == 4u - k ? longer : 0u;
    }
    return of;
}

// (N ids a lane at a time, kept from the first look at them to the second where that is all of them: 615 slots 6.2 -> 5.2 us)
template <uint32_t N>
__global__ void __launch_bounds__(kExPlanThreads)
k_experts_plan(const int32_t *__restrict__ ids, uint32_t slots, uint32_t experts, ExCut cut, ExPlan plan) {
    __shared__ uint32_t hist[kExMostExperts], of_wave[kExPlanWaves], sums[1u + kExSizes][kExPlanWaves];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, e = blockIdx.x;
    // a wave has whole 64 slots one after another
    const uint32_t share = ((slots + kExPlanThreads - 1u) / kExPlanThreads) * kWave, from = min(wave * share, slots), to = min(from + share, slots);
    uint32_t id[N];
    auto load = [&](uint32_t i0) {
#pragma unroll
        for (uint32_t k = 0; k < N; ++k) id[k] = (uint32_t)ids[min(i0 + k * kWave + lane, slots - 1u)];
#pragma unroll
        for (uint32_t k = 0; k < N; ++k)
            if (i0 + k * kWave + lane >= to) id[k] = ~0u;
    };
    load(from);
    for (uint32_t i = tid; i < experts; i += kExPlanThreads) hist[i] = 0;
    __syncthreads();
    uint32_t mine = 0;
    for (uint32_t i0 = from; i0 < to; i0 += N * kWave) {
        if (i0 != from) load(i0);
#pragma unroll
        for (uint32_t k = 0; k < N; ++k) {
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
        const ExSizes of = ex_sizes(hist[i], cut);
        if (i < e) sum[0] += cut.places(hist[i]);
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
    const uint32_t before = sum[0], n = hist[e], n_tiles = cut.tiles(n), places = cut.places(n);
    const ExSizes own_sizes = ex_sizes(n, cut);
    for (uint32_t i = tid; i < n_tiles; i += kExPlanThreads) {
        if (cut.rows) {
            uint32_t *const t = plan.tiles + 3u * (sum[1] + i);
            t[0] = e, t[1] = before + i * cut.rows, t[2] = min(cut.rows, n - i * cut.rows);
        } else {  // the longer ones of an expert's tiles come first
            const uint32_t layers = cut.layers(n), each = layers / n_tiles, longer = layers - each * n_tiles;
            const uint32_t b0 = (i * each + min(i, longer)) * (kExLayer / 16u), size = each + (i < longer);
            uint32_t at = i < longer ? i : i - longer;
#pragma unroll
            for (uint32_t k = 0; k < kExSizes; ++k) at += size == 4u - k ? sum[1u + k] : 0u;
            uint32_t *const t = plan.tiles + 3u * at;
            t[0] = e, t[1] = before / 16u + b0, t[2] = min(size * (kExLayer / 16u), places / 16u - b0);
        }
    }
    for (uint32_t i = n + tid; i < places; i += kExPlanThreads) plan.order[before + i] = ~0u;
    if (e + 1u == experts && tid == 0) {
        *plan.n_tiles = cut.rows ? sum[1] + n_tiles : sum[kExSizes] + own_sizes.n[kExSizes - 1u];  // (in front of this one: all larger ones, and all others')
        *plan.n_blocks = (before + places) / 16u;
    }
    uint32_t at = before;
    for (uint32_t w = 0; w < wave; ++w) at += of_wave[w];
    const bool again = share > N * kWave;
    for (uint32_t i0 = from; i0 < to; i0 += N * kWave) {
        if (again) load(i0);
#pragma unroll
        for (uint32_t k = 0; k < N; ++k) {
            const bool own = id[k] == e;
            const uint64_t all = __ballot(own);
            if (own) plan.order[at + lanes_below(all)] = i0 + k * kWave + lane;
            at += (uint32_t)__popcll(all);
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------
// k_experts_rows<BITS, MT, WIDE, FIRST>: tiles of up to MT slots of one expert, MT = 1 or 8.
//
// As in k_lanes_rows a lane's decoded weights are its operand of v_mfma_f32_16x16x32_bf16 as they are, the activations of the tile lie in
// LDS a column's rows together (transposing reads make them the other operand), and listed elements are multiplied in fp32 by the lane of
// their row.  FIRST: the rows are gathered from the tokens, and the epilogue is the bias, the activation and, gated, the product of the two
// halves; else they are those of the intermediate and the sums go out in fp32.
//
// How many tiles there are is known on the device only.  All of them are one list of items (16 weight rows of a tile, or a pair of blocks),
// of which each workgroup, one a CU, has an equal run: its parts of one tile after another.  Of such a part the cells (16 rows x 512
// columns) are dealt to the waves in equal runs as well; what a wave has of a block goes to LDS, and the epilogue adds the waves' parts in
// the columns' order.  Rows longer than LDS holds are taken in chunks of cells, whose sums are added there.
//
// The intermediate is rounded to bf16, which the matrix unit's operands have to be: half a step, 2^-9 to 2^-8 of each element, which a row of the second
// matrix averages (relative error of a call 0.0017 from the output's own rounding, 0.0023 with it).
//
// Bound: memory, then vector instructions.  64 tokens by 6 of 64 experts of 2048 x 1024, 5 bits: 54 us for the first matrix, which reads 204 MB
// (3.8 TB/s; 168 MB of codes, some experts' twice), the vector unit busy for 69 % of it, LDS for 59 %; 35 us for the second, 87 MB, 65 % and 49 %.
// ---------------------------------------------------------------------------------------------------------------
// (Tiles of 16, which halve the decoding of an expert with more than eight, take longer: their listed elements cost twice as much, and 24 registers
// go to memory.  us of a call, 8 / 16, 64 experts of 2048 x 1024 with 2, 8 and 16 tokens each: 68 / 91, 101 / 124, 149 / 156.)
constexpr uint32_t kExTileRows = 8;
constexpr uint32_t kExWaves = 16, kExThreads = kExWaves * kWave;

struct ExRows {
    const uint16_t *x;
    int64_t ldx;
    const int32_t *ids;
    const uint32_t *n_tiles, *tiles, *order;  // n_tiles NULL: a tile is a slot
    void *out;
    int64_t ld_out;
    uint32_t experts, top_k, slots;
    uint32_t per_tile, most_blocks, chunk_cells;  // items of a tile; blocks that LDS has room for; cells of a chunk
    uint32_t of_tile;                             // workgroups of each tile, or 0: of all of them
    int activation;
    bool gated, pairs;
};

template <int BITS, bool WIDE> constexpr uint32_t kExXAt = (LnPairs<BITS, WIDE>::kLutBytes + 4095u) & ~4095u;

template <int BITS, int MT, bool WIDE, bool FIRST>
__global__ void __launch_bounds__(kExThreads)
k_experts_rows(ExMatrix W, ExRows R) {
    extern __shared__ __attribute__((aligned(16))) uint8_t ex_smem[];
    using P = LnPairs<BITS, WIDE>;
    static_assert(MT == 1 || MT == 8, "rows of a tile");
    constexpr uint32_t ROW = 2u * MT, PART = 16u * MT;
    constexpr uint32_t kZeros = MT == 1 ? 64u : 256u;  // bytes behind the activations
    const uint32_t smem = (uint32_t)(uintptr_t)(LN_LDS(uint8_t) *)ex_smem;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, n = lane & 15u, kg = lane >> 4;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6));
    const uint32_t C = W.n_cells, per = FIRST && R.gated ? 2u : 1u;  // blocks of an item
    const uint32_t x_at = smem + kExXAt<BITS, WIDE>, x_none = R.chunk_cells * kLnCols * ROW;
    float *const parts = reinterpret_cast<float *>(ex_smem + kExXAt<BITS, WIDE> + x_none + kZeros);  // [wave + block][16][MT]
    float *const totals = parts + (kExWaves + R.most_blocks) * PART;  // [block][16][MT], with several chunks
    const uint32_t lut_lane = smem + ((lane & ((1u << P::kCopies) - 1u)) << 2);
    // Where the lane's operands begin in the activations: of sixteen lanes pieces of four columns (of all rows), of one row the lane's eight
    // columns.  What comes on top is the same for all lanes.
    const uint32_t x_mine = x_at + (MT == 1 ? kg * 16u : (8u * kg + (n >> 2)) * ROW + (n & 1u) * 8u);

    // (below 2^31 items)
    const uint32_t all_items = (R.n_tiles ? *R.n_tiles : R.slots) * R.per_tile;
    uint32_t item, item_end;
    if (R.of_tile) {
        const uint32_t tile = blockIdx.x / R.of_tile, part = blockIdx.x - tile * R.of_tile;
        item = tile * R.per_tile + part * R.per_tile / R.of_tile, item_end = min(tile * R.per_tile + (part + 1u) * R.per_tile / R.of_tile, all_items);
    } else {
        // (workgroups go round the eight XCDs: those of one have runs in a row, so that the tiles of an expert share its weights in an L2)
        const uint32_t share = all_items / gridDim.x, more = all_items - share * gridDim.x;
        const uint32_t run = gridDim.x & 7u ? blockIdx.x : (blockIdx.x & 7u) * (gridDim.x >> 3) + (blockIdx.x >> 3);
        item = run * share + min(run, more), item_end = item + share + (run < more);
    }
    uint32_t staged = ~0u, e_table = ~0u;  // the tile whose activations are in LDS, the expert whose pairs are
    for (uint32_t blocks; item < item_end; item += blocks / per) {
        const uint32_t tile = item / R.per_tile, b0 = (item - tile * R.per_tile) * per;
        blocks = min(min(R.per_tile * per - b0, R.most_blocks), (item_end - item) * per);
        // ---- the tile ----
        uint32_t e, first = tile, count = 1;
        if (R.n_tiles) {
            const uint32_t *const t = R.tiles + 3u * tile;
            e = t[0], first = t[1], count = t[2];
        } else {
            e = (uint32_t)R.ids[tile];
            if (e >= R.experts) continue;
        }
        const uint32_t slot = R.n_tiles ? R.order[first + min(lane, count - 1u)] : first;  // of the tile's row `lane`
        const int64_t x_row = (int64_t)(FIRST ? slot / R.top_k : first + min(lane, count - 1u)) * R.ldx;
        const __amdgpu_buffer_rsrc_t codes_rs = __builtin_amdgcn_make_buffer_rsrc((void *)(W.plane + (size_t)e * W.plane_words), 0, -1, 0x00020000);
        const uint32_t *const exc_off = W.exc_off + (size_t)e * (W.n_tiles * C + 1u);
        const uint32_t scale_raw = W.scale[e];

        for (uint32_t c0 = 0; c0 < C; c0 += R.chunk_cells) {
            const uint32_t cells = min(R.chunk_cells, C - c0), units = blocks * cells;
            const uint32_t u0 = wave * units / kExWaves, u1 = (wave + 1u) * units / kExWaves;
            // ---- what depends on nothing that LDS holds is asked for ----
            // (requests past the last cell of the share are for that one again)
            struct Cursor { uint32_t b, c; };  // a block of the part, a cell of the chunk
            const uint32_t last_unit = u1 ? u1 - 1u : 0u, b_last = last_unit / cells, c_last = last_unit - b_last * cells;
            auto after = [&](const Cursor &k) {
                if (k.b == b_last && k.c == c_last) return k;
                return k.c + 1u < cells ? Cursor{k.b, k.c + 1u} : Cursor{k.b + 1u, 0u};
            };
            // bytes of the lane's codes, and places of its quad's cell, of a block in front of its cells (below 2^31)
            constexpr uint32_t kCell = 256u * BITS, kLane = BITS == 3 ? 12u : 16u;
            const uint32_t in_cell = 4u * kg + (n & 3u);
            auto codes_of = [&](uint32_t block) { return (min(4u * (b0 + block) + (n >> 2), W.n_tiles - 1u) * C + c0) * kCell + in_cell * kLane; };
            auto cells_of = [&](uint32_t block) { return min(4u * (b0 + block) + kg, W.n_tiles - 1u) * C + c0; };
            uint32_t w[2][2][BITS];  // the halves of a cell: each is asked for again, for the next cell, as soon as it is decoded
            auto load = [&](uint32_t codes, uint32_t c, uint32_t half) {
#pragma unroll
                for (uint32_t j = 0; j < 2; ++j) {
                    const uint32_t q = 2u * half + j, at = c * kCell;
                    uint32_t(&d)[BITS] = w[half][j];
                    if constexpr (BITS == 3) {
                        const ln_u32x3 v = __builtin_bit_cast(ln_u32x3, __builtin_amdgcn_raw_buffer_load_b96(codes_rs, (int)(codes + q * 192u), (int)at, 0));
                        d[0] = v[0]; d[1] = v[1]; d[2] = v[2];
                    } else {
                        const ln_u32x4 v = __builtin_bit_cast(ln_u32x4, __builtin_amdgcn_raw_buffer_load_b128(codes_rs, (int)(codes + q * 256u), (int)at, 0));
                        d[0] = v[0]; d[1] = v[1]; d[2] = v[2]; d[3] = v[3];
                        if constexpr (BITS == 5)
                            d[4] = __builtin_amdgcn_raw_buffer_load_b32(codes_rs, (int)(codes - 12u * in_cell + (1024u + q * 64u)), (int)at, 0);
                        if constexpr (BITS == 8) {
                            const ln_u32x4 u = __builtin_bit_cast(ln_u32x4, __builtin_amdgcn_raw_buffer_load_b128(codes_rs, (int)(codes + (1024u + q * 256u)), (int)at, 0));
                            d[4] = u[0]; d[5] = u[1]; d[6] = u[2]; d[7] = u[3];
                        }
                    }
                }
            };
            struct Extent { uint32_t first, end; };
            auto extent = [&](uint32_t from, const Cursor &k) {  // (behind the last row quad: the last one's, of which nothing is taken)
                const uint32_t a = exc_off[from + k.c], b = exc_off[from + k.c + 1u];
                return Extent{a, 4u * (b0 + k.b) + kg < W.n_tiles ? b : a};
            };
            struct Group { ln_u32x2 pos; uint32_t val; };
            auto quad_of = [&](const Extent &x, uint32_t i) { return (x.first & ~3u) + 16u * i + (n & ~3u); };
            auto g_load = [&](const Extent &x, uint32_t i) {
                const uint32_t q = quad_of(x, i), at = q < x.end ? lane_listed(q, n & 3u) : 0u;
                return Group{*reinterpret_cast<const ln_u32x2 *>(W.exc_pos + at), *reinterpret_cast<const uint32_t *>(W.exc_val + at)};
            };
            const uint32_t b_first = min(u0 / cells, blocks - 1u);  // (an empty share at the end)
            Cursor now{b_first, min(u0 - b_first * cells, cells - 1u)}, next = after(now);
            uint32_t codes = codes_of(now.b), places = cells_of(now.b);
            load(codes, now.c, 0);
            load(codes, now.c, 1);
            Extent e_now = extent(places, now);
            if (next.b != now.b) codes = codes_of(next.b), places = cells_of(next.b);  // of the cell that is asked for next
            Extent e_next = extent(places, next);
            const float scale = bf16_bits_to_f32(scale_raw);
            const uint32_t scale_bits = __float_as_uint(scale) & 0x7FFFFFFFu;

            if (staged != tile || cells != C) {
                // activations: a pair of columns a lane, all rows (rows past the last are the last one's, columns past the last the last ones)
                for (uint32_t task = wave; task < 4u * cells; task += kExWaves) {
                    const uint32_t col = c0 * kLnCols + task * 128u + 2u * lane;
                    const uint32_t keep = (col < W.in_f ? 0xFFFFu : 0u) | (col + 1u < W.in_f ? 0xFFFF0000u : 0u);
                    uint32_t v[MT];
#pragma unroll
                    for (uint32_t k = 0; k < MT; ++k) {
                        const uint32_t r = min(k, count - 1u);
                        const uint16_t *const row = R.x + (((int64_t)__builtin_amdgcn_readlane((int)(x_row >> 32), (int)r) << 32) |
                                                           (uint32_t)__builtin_amdgcn_readlane((int)x_row, (int)r));
                        if (R.pairs) v[k] = *reinterpret_cast<const uint32_t *>(row + min(col, W.in_f - 2u));
                        else v[k] = row[min(col, W.in_f - 1u)] | (uint32_t)row[min(col + 1u, W.in_f - 1u)] << 16;
                    }
#pragma unroll
                    for (uint32_t k = 0; k < MT; ++k) v[k] = k < count ? v[k] & keep : 0u;
                    const uint32_t to = lane_offset(task * 128u + 2u * lane) * MT;
                    if constexpr (MT == 1) {
                        *reinterpret_cast<LN_LDS(uint32_t) *>((uintptr_t)(x_at + to)) = v[0];
                    } else {
#pragma unroll
                        for (uint32_t j = 0; j < 2; ++j) {
                            ln_u32x4 o;
#pragma unroll
                            for (uint32_t k = 0; k < 4; ++k) o[k] = __builtin_amdgcn_perm(v[2 * k + 1], v[2 * k], j ? 0x07060302u : 0x05040100u);
                            *reinterpret_cast<LN_LDS(ln_u32x4) *>((uintptr_t)(x_at + to + j * ROW)) = o;
                        }
                    }
                }
                if (tid < kZeros / 16u) *reinterpret_cast<LN_LDS(ln_u32x4) *>((uintptr_t)(x_at + x_none + tid * 16u)) = ln_u32x4{0, 0, 0, 0};
                staged = tile;
            }
            if (e_table != e) {
                ln_build_lut<BITS, WIDE>(smem, scale, tid, kExThreads);
                e_table = e;
            }
            Group list[2];
#pragma unroll
            for (uint32_t i = 0; i < 2; ++i) list[i] = g_load(e_now, i);
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");

            // ---- this wave's cells ----
            ln_f32x4 acc = {0, 0, 0, 0};
            float ex[MT];
#pragma unroll
            for (int r = 0; r < MT; ++r) ex[r] = 0.0f;
            const uint32_t c_seg = c0 * 1024u;
            auto listed = [&](const Group &g, const Extent &x, uint32_t i) {
                const uint32_t q = quad_of(x, i);
                const uint32_t w01 = ln_pack((float)(int)(int8_t)g.val * scale, (float)(int)(int8_t)(g.val >> 8) * scale);
                const uint32_t w23 = ln_pack((float)(int)(int8_t)(g.val >> 16) * scale, (float)((int)g.val >> 24) * scale);
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k) {
                    const uint32_t p = ((g.pos[k >> 1] >> (16 * (k & 1))) - c_seg) & 0xFFFFu;
                    const bool is = q + k >= x.first && q + k < x.end && ((g.val >> (8 * k)) & 255u);
                    if (!__any(is)) continue;  // (a cell of few listed elements has them in the first quads of the first lanes)
                    const uint32_t at = is ? min(p * MT, x_none) : x_none;
                    const uint32_t wk = k & 2 ? w23 : w01, wbits = k & 1 ? wk & 0xFFFF0000u : wk << 16;
                    const float wv = __uint_as_float(wbits) - __uint_as_float((wbits & 0x80000000u) | scale_bits);  // (no element: times 0)
                    if constexpr (MT == 1) {
                        const uint32_t h = *reinterpret_cast<const LN_LDS(uint16_t) *>((uintptr_t)(x_at + at));
                        ex[0] = __fmaf_rn(wv, __uint_as_float(h << 16), ex[0]);
                    }
                    if constexpr (MT == 8) {
                        const ln_u32x4 v = *reinterpret_cast<const LN_LDS(ln_u32x4) *>((uintptr_t)(x_at + at));
#pragma unroll
                        for (uint32_t j = 0; j < 4; ++j) {
                            ex[2 * j] = __fmaf_rn(wv, __uint_as_float(v[j] << 16), ex[2 * j]);
                            ex[2 * j + 1] = __fmaf_rn(wv, __uint_as_float(v[j] & 0xFFFF0000u), ex[2 * j + 1]);
                        }
                    }
                }
            };
#pragma unroll 1
            for (uint32_t u = u0; u < u1; ++u) {
                const uint32_t x_cell = x_mine + now.c * (512u * ROW);
#pragma unroll
                for (uint32_t half = 0; half < 2; ++half) {
                    uint32_t o[2][16];
                    ln_decode<BITS, WIDE>(w[half][0], lut_lane, scale, o[0]);
                    ln_decode<BITS, WIDE>(w[half][1], lut_lane, scale, o[1]);
                    load(codes, next.c, half);
                    // (columns 128 q + 32 i of a cell lie at 128 q + 32 (i ^ q))
#pragma unroll
                    for (uint32_t j = 0; j < 2; ++j)
#pragma unroll
                        for (uint32_t i = 0; i < 4; ++i) {
                            const uint32_t q = 2u * half + j, at = (q * 128u + (q ^ i) * 32u) * ROW;
                            ln_bf16x8 x;
                            if constexpr (MT == 1) {  // (one row in all sixteen columns of the product)
                                x = __builtin_bit_cast(ln_bf16x8, *reinterpret_cast<const LN_LDS(ln_u32x4) *>((uintptr_t)(x_cell + at)));
                            } else {
                                const lr_bf16x4 lo = lr_turned(x_cell + at), hi = lr_turned(x_cell + at + 4u * ROW);
                                x = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                            }
                            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                                __builtin_bit_cast(ln_bf16x8, ln_u32x4{o[j][4 * i], o[j][4 * i + 1], o[j][4 * i + 2], o[j][4 * i + 3]}), x, acc, 0, 0, 0);
                        }
                }
                const uint32_t g = e_now.end > e_now.first ? (e_now.end - (e_now.first & ~3u) + 15u) / 16u : 0u;
                if (__any(g > 0u)) listed(list[0], e_now, 0);
                if (__any(g > 1u)) listed(list[1], e_now, 1);
#pragma unroll 1
                for (uint32_t i = 2; __any(g > i); ++i) listed(g_load(e_now, i), e_now, i);
                if (next.b != now.b || u + 1u == u1) {
                    // the block's sums: of listed elements over the four lanes of a row, of the plane as they are
                    float *const part = parts + (wave + now.b) * PART;
#pragma unroll
                    for (int r = 0; r < MT; ++r) {
                        ex[r] += ln_dpp<0x124>(ex[r]);
                        ex[r] += ln_dpp<0x128>(ex[r]);
                    }
                    if constexpr (MT == 1) {
                        if (n < 4u) part[4u * kg + n] = ex[0];
                    } else if (n < 4u)
#pragma unroll
                        for (uint32_t r = 0; r < MT; r += 4)
                            *reinterpret_cast<ln_f32x4 *>(part + (4u * kg + n) * MT + r) = ln_f32x4{ex[r], ex[r + 1], ex[r + 2], ex[r + 3]};
                    ln_wave_order();
                    if (n < MT)
#pragma unroll
                        for (uint32_t k = 0; k < 4; ++k) part[(4u * kg + k) * MT + n] += acc[k];
                    acc = ln_f32x4{0, 0, 0, 0};
#pragma unroll
                    for (int r = 0; r < MT; ++r) ex[r] = 0.0f;
                }
                now = next;
                next = after(now);
                e_now = e_next;
#pragma unroll
                for (uint32_t i = 0; i < 2; ++i) list[i] = g_load(e_now, i);
                if (next.b != now.b) codes = codes_of(next.b), places = cells_of(next.b);
                e_next = extent(places, next);
            }
            __syncthreads();

            // ---- the waves' parts of a block, in column order ----
            auto sum_of = [&](uint32_t block, uint32_t at) {
                const uint32_t wa = ((block * cells + 1u) * kExWaves - 1u) / units, wb = ((block + 1u) * cells * kExWaves - 1u) / units;
                float v = 0.0f;
                for (uint32_t k = wa; k <= wb; ++k)  // (waves without a cell left no part)
                    if (k * units / kExWaves != (k + 1u) * units / kExWaves) v += parts[(k + block) * PART + at];
                return v;
            };
            const bool last = c0 + cells == C;
            if (cells != C) {  // chunks: their sums are added up
                for (uint32_t i = tid; i < blocks * PART; i += kExThreads) {
                    const float v = sum_of(i / PART, i % PART);
                    totals[i] = c0 ? totals[i] + v : v;
                }
                __syncthreads();
                if (!last) continue;
            }
            auto value = [&](uint32_t block, uint32_t at) { return cells != C ? totals[block * PART + at] : sum_of(block, at); };
            // ---- outputs ----
            const uint32_t n_out = blocks / per * 16u, at0 = b0 / per * 16u;
            const uint16_t *const bias = W.bias ? W.bias + (size_t)e * (per * W.outputs) : nullptr;
            for (uint32_t i = tid; i < n_out * count; i += kExThreads) {
                const uint32_t r = i / n_out, at = i - r * n_out, block = (at >> 4) * per, in_part = (at & 15u) * MT + r, out = at0 + at;
                if (out >= W.outputs) continue;
                float v = value(block, in_part);
                if (bias) v += bf16_bits_to_f32(bias[out]);
                if constexpr (FIRST) {
                    v = ep_activation(R.activation, v);
                    if (R.gated) {
                        float u = value(block + 1u, in_part);
                        if (bias) u += bf16_bits_to_f32(bias[W.outputs + out]);
                        v *= u;
                    }
                    static_cast<uint16_t *>(R.out)[(int64_t)(first + r) * R.ld_out + out] = ep_bf16(v);
                } else {
                    const uint32_t to = R.n_tiles ? R.order[first + r] : first;
                    static_cast<float *>(R.out)[(int64_t)to * R.ld_out + out] = v;
                }
            }
            __syncthreads();
        }
    }
}

// y[t] = residual[t] + sum_j weights[t, j] * (what its expert made of it), in the order of j.  Bound: memory (4096 tokens of 6 experts, 2048 columns:
// 218 MB in 39 us, some of it from the last-level cache) or a launch (64 tokens 4.1 us).  N columns a thread.
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
    constexpr uint32_t AHEAD = 8;  // experts asked for at a time (behind the last that one again; what no expert wrote is not used)
    for (uint32_t j0 = 0; j0 < call.top_k; j0 += AHEAD) {
        Sums p[AHEAD];
        bool is[AHEAD];
        float w[AHEAD];
#pragma unroll
        for (uint32_t i = 0; i < AHEAD; ++i) {
            const uint32_t j = min(j0 + i, call.top_k - 1u);
            is[i] = j0 + i < call.top_k && (uint32_t)ids[j] < experts;
            w[i] = weights[j];
            if constexpr (N == 4) p[i] = *reinterpret_cast<const Sums *>(from + (size_t)j * hidden);
            else p[i][0] = from[(size_t)j * hidden];
        }
#pragma unroll
        for (uint32_t i = 0; i < AHEAD; ++i)
#pragma unroll
            for (int k = 0; k < N; ++k) v[k] = is[i] ? __fmaf_rn(w[i], p[i][k], v[k]) : v[k];
    }
    uint16_t *const y = call.y + (int64_t)t * call.ldy + at;
    const uint16_t *const residual = call.residual + (int64_t)t * call.ld_residual + at;
#pragma unroll
    for (int k = 0; k < N; ++k) y[k] = ep_bf16(call.residual ? v[k] + bf16_bits_to_f32(residual[k]) : v[k]);
}

// ---- host ----
template <int BITS, int MT, bool WIDE> static size_t ex_lds(uint32_t cells, uint32_t blocks, bool chunks) {
    return kExXAt<BITS, WIDE> + (size_t)cells * kLnCols * 2u * MT + 256u + (size_t)(kExWaves + blocks * (chunks ? 2u : 1u)) * 16u * MT * sizeof(float);
}

template <int BITS, int MT, bool WIDE, bool FIRST>
static int ex_launch(const ExMatrix &W, ExRows R, uint32_t n_tiles, hipStream_t s) {
    const uint32_t per = FIRST && R.gated ? 2u : 1u, all = (W.n_tiles + 3u) / 4u;
    R.per_tile = all / per;
    // as few chunks as leave room for the sums of eight blocks, and as many blocks of a part as then fit, up to those that a workgroup has at all
    // Few tiles: as many workgroups to each, so that none begins a second one (which takes as long as some ten cells).
    const uint64_t items = (uint64_t)n_tiles * R.per_tile;
    if (items >= 1ull << 31) return IXH_EUNSUPPORTED;  // (their numbers are 32 bits)
    R.of_tile = R.n_tiles || n_tiles > ln_cus() ? 0u : std::min(ln_cus() / n_tiles, R.per_tile);
    const uint32_t groups = R.of_tile ? n_tiles * R.of_tile : (uint32_t)std::min<uint64_t>(items, ln_cus());
    const uint32_t share = (uint32_t)std::min<uint64_t>((items + groups - 1u) / groups, R.per_tile) * per;
    for (uint32_t chunks = 1;; ++chunks) {
        R.chunk_cells = (W.n_cells + chunks - 1u) / chunks;
        if (R.chunk_cells <= kLnSegCells && ex_lds<BITS, MT, WIDE>(R.chunk_cells, 8u, chunks > 1u) <= kLnLds) break;
        if (R.chunk_cells == 1u) return IXH_EUNSUPPORTED;
    }
    const bool chunks = R.chunk_cells < W.n_cells;
    R.most_blocks = std::max(share, per);
    while (R.most_blocks > 8u && ex_lds<BITS, MT, WIDE>(R.chunk_cells, R.most_blocks, chunks) > kLnLds) R.most_blocks -= per;
    const size_t lds = ex_lds<BITS, MT, WIDE>(R.chunk_cells, R.most_blocks, chunks);
    static const bool raised = hipFuncSetAttribute(reinterpret_cast<const void *>(k_experts_rows<BITS, MT, WIDE, FIRST>),
                                                   hipFuncAttributeMaxDynamicSharedMemorySize, (int)kLnLds) == hipSuccess;
    if (!raised) return IXH_ELAUNCH;
    R.pairs = ((uintptr_t)R.x & 3u) == 0 && W.in_f % 2u == 0 && R.ldx % 2 == 0;
    IXH_LAUNCH((k_experts_rows<BITS, MT, WIDE, FIRST>), dim3(groups), dim3(kExThreads), lds, s, W, R);
    return hipGetLastError() == hipSuccess ? IXH_OK : IXH_ELAUNCH;
}

template <int BITS, bool FIRST> static int ex_rows(const ExMatrix &W, const ExRows &R, uint32_t rows, uint32_t n_tiles, hipStream_t s) {
    // The larger pair table where a CU has cells enough to repay its writing, and LDS room for it beside the activations and the sums of all
    // that a workgroup has of a tile (us, smaller / larger: 64 tokens by 6 of 64 experts, 17 blocks of two cells a workgroup 39 / 34.4; 35 of
    // four, which the larger one takes in three parts, 55.6 / 59).
    if constexpr (BITS == 5) {
        const uint32_t per = FIRST && R.gated ? 2u : 1u, blocks = (W.n_tiles + 3u) / 4u;
        const uint32_t share = std::min((uint32_t)(((uint64_t)n_tiles * blocks / per + ln_cus() - 1u) / ln_cus()) * per, blocks);
        if (rows > 1u && (uint64_t)n_tiles * W.n_tiles * W.n_cells > 128ull * ln_cus() && W.n_cells <= kLnSegCells &&
            ex_lds<5, 8, true>(W.n_cells, share, false) <= kLnLds)
            return ex_launch<5, 8, true, FIRST>(W, R, n_tiles, s);
    }
    constexpr bool WIDE = BITS == 4;
    return rows == 1u ? ex_launch<BITS, 1, WIDE, FIRST>(W, R, n_tiles, s) : ex_launch<BITS, 8, WIDE, FIRST>(W, R, n_tiles, s);
}
template <bool FIRST> static int ex_matrix(const ExMatrix &W, const ExRows &R, uint32_t rows, uint32_t n_tiles, hipStream_t s) {
    switch (W.bits) {
        case 3: return ex_rows<3, FIRST>(W, R, rows, n_tiles, s);
        case 4: return ex_rows<4, FIRST>(W, R, rows, n_tiles, s);
        case 5: return ex_rows<5, FIRST>(W, R, rows, n_tiles, s);
        default: return ex_rows<8, FIRST>(W, R, rows, n_tiles, s);
    }
}

// Many tokens to an expert: 9 and more in the mean (us of a call with 6 / 8 / 9 / 12 / 16 tokens each, by k_experts_rows and by k_experts_prompt:
// 64 experts of 2048 x 1024 at 5 % listed 118 / 131 / 146 / 168 / 198 and 130 / 135 / 136 / 140 / 151; next to none listed 88 / 97 / 106 / 122 /
// 142 and 99 / 107 / 107 / 114 / 124; 16 of 4096 x 1536 82 / 92 / 103 / 107 / 130 and 91 / 93 / 93 / 93 / 96; 20 of 1400 x 744
// 56 / 59 / 59 / 65 / 71 and 49 / 50 / 50 / 55 / 56).
constexpr uint32_t kExMany = 9;
// (Rows of up to 2^20 columns: offsets within a tile's rows are 32 bits.)
static bool ex_many(const ExDev &X, uint32_t slots) {
    return slots >= kExMany * X.experts && std::max(X.first.n_cells, X.second.n_cells) <= 2048u;
}

// Layers of a tile of k_experts_prompt, two instead of four where the workgroups then still are all there at once, three a CU.  us with four / two at 5
// bits: 2279 tokens by 3 of 7 experts of 512 x 192, which are 480 of 768 workgroups at most, 49 / 44; 500 and 1000 by 2 of 8 of 2048 x 512, 480 and 736,
// 53 / 50 and 65 / 58; beyond, 4000 by 3 of 7 of 512 x 192, 800, 58.7 / 59.5; 600, 800 and 1500 by 2 of 8 of 4096 x 1536, 1088, 1280 and 1984, 99 / 109,
// 115 / 124 and 170 / 198; 1600 by 2 of 8 of 2048 x 512, 1056, 70 / 72; 1333 by 3 of 20 of 1400 x 744, 1224, 83 / 87 (800, 912, 64.9 / 63.7); 512 and 1600 by
// 2 of 16 of 4096 x 1536, 1536 and 2624, 106 / 106 and 199 / 232; with 3 bits and with 10 % listed the same sides.
static uint32_t ex_layers(const ExDev &X, uint32_t slots) {
    const uint64_t w_tiles = (std::max(X.first.n_tiles, X.second.n_tiles) + 15u) / 16u;
    return (slots / (2u * kExLayer) + X.experts) * w_tiles <= 3ull * ln_cus() ? 2u : 4u;
}

// Slots one by one, of k_experts_one, up to 160 cells a CU (us one by one / planned: 64 experts of 2048 x 1024, 24 / 48 / 72 slots, which are 72 / 144 /
// 216 cells a CU, 34 / 50 / 67, 53 / 54 / 61; 16 of 4096 x 1536, 8 / 16 / 24 slots 31 / 47 / 60, 46 / 52 / 59; 128 of 2048 x 768, 48 / 96 slots 46 / 72,
// 58 / 69; one token by 8 of 7168 x 2048, 168 cells a CU, 58, by k_experts_rows 55; by 2 of 5120 x 1536 20.8, 27).
static bool ex_one_by_one(const ExDev &X, uint32_t slots) {
    const auto cells = [](const ExMatrix &W) { return (uint64_t)((W.n_tiles + 3u) / 4u) * W.n_cells; };
    return experts_one_takes(X.first, X.gated) && experts_one_takes(X.second, false) && slots * (cells(X.first) + cells(X.second)) <= 160ull * ln_cus();
}

// A call's scratch: the plan, the intermediate, what each slot's expert makes of it, and in k_experts_prompt the gathered rows.
struct ExScratch {
    bool many;
    uint32_t rows, most, n_tiles, blocks;  // as ExCut; tiles and blocks at most
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
        w.most = ex_layers(X, slots);
        w.n_tiles = std::min(slots, X.experts) + slots / (w.most * kExLayer);
        w.blocks = std::min(slots, X.experts) + slots / 16u;
        w.tiles = take((std::min(slots, X.experts) + slots / (2u * kExLayer)) * (size_t)12u);  // (of either height)
        w.order = take((size_t)w.blocks * 64u);
        w.x = take((size_t)w.blocks * X.first.n_cells * 16384u);
        w.inner = take((size_t)w.blocks * X.second.n_cells * 16384u);
    } else {
        w.rows = kExTileRows;
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
    const uint32_t few = std::min(tokens, (kExMany * X.experts - 1u) / top_k);  // the most that are not many
    return std::max(ex_scratch(X, tokens, top_k).bytes, few ? ex_scratch(X, few, top_k).bytes : 0u);
}

int launch_experts(const ExDev &X, const ExCall &call, void *workspace, hipStream_t s) {
    const uint32_t slots = call.tokens * call.top_k;
    const ExScratch w = ex_scratch(X, call.tokens, call.top_k);
    uint8_t *const ws = reinterpret_cast<uint8_t *>(((uintptr_t)workspace + 255u) & ~(uintptr_t)255u);
    // (else k_experts_rows: by expert where tiles of several slots are likely)
    const bool apart = !w.many && ex_one_by_one(X, slots), planned = w.many || (!apart && call.tokens > 1u && slots > X.experts / 4u);
    const uint32_t n_tiles = planned ? w.n_tiles : slots;
    uint32_t *const counts = reinterpret_cast<uint32_t *>(ws);
    const ExPlan plan{counts, counts + 1, reinterpret_cast<uint32_t *>(ws + w.tiles), reinterpret_cast<uint32_t *>(ws + w.order)};
    float *const per_slot = reinterpret_cast<float *>(ws + w.per_slot);
    if (planned) {
        const auto run = [&](auto n) {
            IXH_LAUNCH(k_experts_plan<n()>, dim3(X.experts), dim3(kExPlanThreads), 0, s, call.ids, slots, X.experts, ExCut{w.rows, w.most}, plan);
        };
        if (slots <= kExPlanThreads) run(std::integral_constant<uint32_t, 1>{});
        else run(std::integral_constant<uint32_t, 8>{});
    }
    int rc;
    if (w.many) {
        rc = launch_experts_prompt(X, call, plan, n_tiles, w.blocks, ws + w.x, ws + w.inner, per_slot, s);
    } else {
        ExRows R{};
        R.x = call.x, R.ldx = call.ldx, R.ids = call.ids, R.experts = X.experts, R.top_k = call.top_k, R.slots = slots;
        if (planned) R.n_tiles = plan.n_tiles, R.tiles = plan.tiles, R.order = plan.order;
        R.out = ws + w.inner, R.ld_out = w.ld_inner, R.activation = X.activation, R.gated = X.gated;
        ExOne one{call.x, call.ldx, call.tokens, call.ids, R.out, R.ld_out, X.experts, call.tokens, call.top_k, X.activation, X.gated,
                  call.weights, call.residual, call.ld_residual};
        if (apart) rc = launch_experts_one(X.first, one, true, s);
        else rc = ex_matrix<true>(X.first, R, planned ? w.rows : 1u, n_tiles, s);
        if (rc != IXH_OK) return rc;
        R.x = reinterpret_cast<const uint16_t *>(ws + w.inner), R.ldx = w.ld_inner;
        R.out = per_slot, R.ld_out = X.hidden;
        one.x = R.x, one.ldx = R.ldx, one.rows = slots;
        if (apart && experts_joined_takes(X.second, call.tokens, call.top_k)) {
            one.out = call.y, one.ld_out = call.ldy;
            return launch_experts_joined(X.second, one, s);
        }
        one.out = R.out, one.ld_out = R.ld_out;
        if (apart) rc = launch_experts_one(X.second, one, false, s);
        else rc = ex_matrix<false>(X.second, R, planned ? w.rows : 1u, n_tiles, s);
    }
    if (rc != IXH_OK) return rc;
    if (X.hidden % 4u == 0)
        IXH_LAUNCH(k_experts_join<4>, dim3(call.tokens, (X.hidden / 4u + 255u) / 256u), dim3(256), 0, s, per_slot, call, X.experts, X.hidden);
    else
        IXH_LAUNCH(k_experts_join<1>, dim3(call.tokens, (X.hidden + 255u) / 256u), dim3(256), 0, s, per_slot, call, X.experts, X.hidden);
    return hipGetLastError() == hipSuccess ? IXH_OK : IXH_ELAUNCH;
}

}  // namespace ixh
