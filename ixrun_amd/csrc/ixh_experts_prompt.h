// k_experts_prompt: the experts' products where an expert has many tokens, decode and matrix products side by side, as in ixh_lanes_prompt.hip.
#pragma once
#include "ixh_epilogue.h"
#include "ixh_experts.h"
#include "ixh_lanes_dev.h"

namespace ixh {

constexpr uint32_t kEpWaves = 4, kEpThreads = kEpWaves * kWave;
constexpr uint32_t kEpRows = 16u * kEpWaves;       // weight rows of a workgroup
constexpr uint32_t kEpTile = kEpRows * 128u * 2u;  // bytes of a stage's weights: 64 rows x 128 columns
constexpr uint32_t kEpRounds = 3;                  // groups of 16 quads of a cell's list that a wave holds
constexpr uint32_t kEpNone = ~0u;

struct EpCall {
    const ln_u32x4 *xt;       // the rows in operand order
    const uint32_t *n_tiles;  // row tiles
    const uint32_t *tiles;    // {expert, first block, blocks} each, up to four blocks of 16 rows to each wave
    const uint32_t *order;    // slots of the blocks' rows, or kEpNone
    uint8_t *inner;           // FIRST: the other matrix's rows in operand order
    float *out;               // else: what each slot's expert makes of it
    uint32_t n_kb_inner, w_tiles;
    int activation;
    bool gated;
};

// ---------------------------------------------------------------------------------------------------------------
// k_experts_prompt<BITS, FIRST>: a tile of up to 256 rows of one expert by 64 weight rows.
//
// Four waves decode 64 weight rows x 128 columns a stage to LDS in operand order, 16 rows each, while they multiply the stage before; the
// activations come from the L2 straight to registers as operands.  A wave has MI blocks of 16 rows, MI = 1 .. 4 by the tile's, and all 64
// weight rows.  The tiles of one expert's rows run on one XCD, whose L2 holds them.
//
// NARROW, one block of rows: each wave multiplies the 16 weight rows that it decodes, and no wave waits for another before the end (us of a call
// with 12 tokens to each expert, of the others' kind / this: 64 experts of 2048 x 1024 at 5 % listed 161 / 140, next to none 126 / 114, 16 of
// 4096 x 1536 97 / 93).  With two and four blocks the rows, which each wave then takes from the L2, cost more than that saves (32 / 64 tokens
// each, 64 experts, next to none listed: 135 / 162 become 156 / 192).
//
// Bound: nothing alone.  With 384 rows an expert the vector unit is busy for 45 % of the time, matrix unit 37 %, LDS 46 % and L1 50 %, and the L2
// gives 12 TB/s; a call of 558 us without its products' waits for the L2 took 470, without lists 494, without any decode 425.  With 64 rows LDS:
// each wave reads all 64 weight rows for a block of its own.
// Three workgroups to a CU, by registers (168) and LDS (53 KB with the smaller pair table), fill in for one another.  us of a call here / with
// eight waves, 128 weight rows, up to 512 rows and the larger table as in k_lanes_prompt, which waits alone: 64 experts of 2048 x 1024 at 5 % listed
// with 64, 128, 200, 400, 600 tokens each 191 / 252, 249 / 308, 324 / 386, 550 / 566, 778 / 760, 16 of 4096 x 1536 with next to none 120 / 197,
// 189 / 220, 239 / 284, 390 / 404, 506 / 505.  Tiles of up to 384 rows and two workgroups, which decode half as often: 200, 384, 600 tokens 329 /
// 344, 523 / 549, 787 / 779.  Operands of weights asked for two and three blocks ahead, and issue priority for the products: the same.  Two or
// four weight tiles one after another by a workgroup, with one pair table: 3 to 30 % longer.
// ---------------------------------------------------------------------------------------------------------------
template <int BITS, int MI, bool NARROW, bool FIRST>
__device__ __forceinline__ void ep_tile(const ExMatrix &W, const EpCall &R, uint32_t e, uint32_t block0, uint32_t n_blocks, uint32_t tile,
                                        uint8_t *ep_smem) {
    using P = LnPairs<BITS, false>;
    constexpr uint32_t NI = NARROW ? 1 : kEpWaves;  // a wave's blocks of weight rows
    constexpr uint32_t AHEAD = MI == 1 ? 8 : MI == 2 ? 4 : 2;  // steps of 32 columns that the activations' operands are asked for ahead
    constexpr uint32_t CODES = 2;  // stages that the codes are asked for ahead of their decode
    const uint32_t smem = (uint32_t)(uintptr_t)(LN_LDS(uint8_t) *)ep_smem;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, n = lane & 15u, kg = lane >> 4;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6));
    const uint32_t n_cells = W.n_cells, n_tiles = W.n_tiles, n_kb = n_cells * 16u;
    const uint32_t mb0 = NARROW ? 0u : wave * MI;  // the wave's first block of rows, in the tile
    const float scale = bf16_bits_to_f32(W.scale[e]);

    // ---- the wave's part of the decode: block `wave` of the workgroup's four, lane (n, kg) the codes of row n ----
    const uint32_t *const exc_off = W.exc_off + (size_t)e * (n_tiles * n_cells + 1u);
    const uint16_t *const exc_pos = W.exc_pos;
    const int8_t *const exc_val = W.exc_val;
    const uint32_t quad0 = (tile * kEpWaves + wave) * 4u;  // the block's first row quad
    const uint32_t first = min(quad0, n_tiles - 1u), per_quad = n_cells * (256u * BITS);
    const __amdgpu_buffer_rsrc_t codes_rs = __builtin_amdgcn_make_buffer_rsrc(
        (void *)(reinterpret_cast<const uint8_t *>(W.plane + (size_t)e * W.plane_words) + (size_t)first * per_quad), 0,
        (int)(min(n_tiles - first, 4u) * per_quad), 0x00020000);
    const uint32_t in_cell = 4u * kg + (n & 3u), codes_at = (min(quad0 + (n >> 2), n_tiles - 1u) - first) * per_quad + in_cell * (BITS == 3 ? 12u : 16u);
    uint32_t w[CODES][BITS];
    auto codes = [&](uint32_t c, uint32_t q) {
        const uint32_t at = c * (256u * BITS) + q * (BITS == 3 ? 192u : 256u);
        uint32_t(&d)[BITS] = w[q % CODES];
        if constexpr (BITS == 3) {
            const ln_u32x3 v = __builtin_bit_cast(ln_u32x3, __builtin_amdgcn_raw_buffer_load_b96(codes_rs, (int)codes_at, (int)at, 0));
            d[0] = v[0]; d[1] = v[1]; d[2] = v[2];
        } else {
            const ln_u32x4 v = __builtin_bit_cast(ln_u32x4, __builtin_amdgcn_raw_buffer_load_b128(codes_rs, (int)codes_at, (int)at, 0));
            d[0] = v[0]; d[1] = v[1]; d[2] = v[2]; d[3] = v[3];
            if constexpr (BITS == 5)
                d[4] = __builtin_amdgcn_raw_buffer_load_b32(codes_rs, (int)(codes_at - 12u * in_cell), (int)(at + 1024u - q * 192u), 0);
            if constexpr (BITS == 8) {
                const ln_u32x4 u = __builtin_bit_cast(ln_u32x4, __builtin_amdgcn_raw_buffer_load_b128(codes_rs, (int)codes_at, (int)(at + 1024u), 0));
                d[4] = u[0]; d[5] = u[1]; d[6] = u[2]; d[7] = u[3];
            }
        }
    };
    struct Extent { uint32_t first, end; };
    // the lane's place in a list, worked out where it is used: held over the loop it would cost registers that the sums need
    struct Place { uint32_t row, quad, kg; };
    auto place = [&] {
        uint32_t l = lane;
        asm volatile("" : "+v"(l));
        return Place{l & 3u, l & 12u, l >> 4};
    };
    auto extent = [&](uint32_t c) {
        const uint32_t t = quad0 + place().kg, cell = min(t, n_tiles - 1u) * n_cells + min(c, n_cells - 1u);
        const uint32_t a = exc_off[cell], b = exc_off[cell + 1u];
        return Extent{a, t < n_tiles ? b : a};
    };
    struct Quads { ln_u32x2 pos[kEpRounds]; uint32_t val[kEpRounds]; };
    auto quads = [&](const Extent &x) {
        Quads l;
        const Place me = place();
#pragma unroll
        for (uint32_t r = 0; r < kEpRounds; ++r) {
            const uint32_t quad = (x.first & ~3u) + me.quad + 16u * r, at = quad < x.end ? lane_listed(quad, me.row) : 0u;
            l.pos[r] = *reinterpret_cast<const ln_u32x2 *>(exc_pos + at);
            l.val[r] = *reinterpret_cast<const uint32_t *>(exc_val + at);
        }
        return l;
    };
    codes(0u, 0);
    if (CODES == 2) codes(0u, 1);
    Extent e_now = extent(0u);
    Quads list = quads(e_now);

    const __amdgpu_buffer_rsrc_t x_rs = __builtin_amdgcn_make_buffer_rsrc((void *)(R.xt + (size_t)block0 * n_kb * 64u), 0,
                                                                          (int)(n_blocks * n_kb * 1024u), 0x00020000);
    ln_u32x4 a[AHEAD][MI];
    uint32_t x_block[MI];  // (past the tile's blocks the last one again)
#pragma unroll
    for (uint32_t i = 0; i < MI; ++i) x_block[i] = min(mb0 + i, n_blocks - 1u) * n_kb * 1024u;
    auto x_load = [&](uint32_t c, uint32_t t) {  // step t of the cell's sixteen: place t % 4 of stage q holds columns 32 (t % 4 ^ q)
        const uint32_t at = (16u * c + (t ^ (t >> 2))) * 1024u;
#pragma unroll
        for (uint32_t i = 0; i < MI; ++i)
            a[t % AHEAD][i] = __builtin_bit_cast(ln_u32x4, __builtin_amdgcn_raw_buffer_load_b128(x_rs, (int)(lane * 16u), (int)(at + x_block[i]), 0));
    };
#pragma unroll
    for (uint32_t t = 0; t < AHEAD; ++t) x_load(0u, t);
    ln_build_lut<BITS, false>(smem, scale, tid, kEpThreads);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");

    const uint32_t lut_lane = smem + ((lane & ((1u << P::kCopies) - 1u)) << 2);
    const uint32_t store_at = smem + P::kLutBytes + wave * 4096u;
    const LN_LDS(ln_u32x4) *const w_at = reinterpret_cast<const LN_LDS(ln_u32x4) *>((uintptr_t)(smem + P::kLutBytes + lane * 16u));
    LN_LDS(ln_u32x4) *const put_at = reinterpret_cast<LN_LDS(ln_u32x4) *>((uintptr_t)(smem + P::kLutBytes + 2u * kEpTile + tid * (16u * kEpRounds)));
    uint32_t in_stage[kEpRounds];  // bit q: the block has elements of the cell's stage q in the round
    bool any[kEpRounds], more;     // (8 bits list next to nothing: whether it has any, which takes fewer registers)
    uint32_t c_put;
    // listed elements of a cell: value (high half), where it goes in the wave's part of a stage's tile (bits 0 .. 11), the stage of
    // the cell (bits 12 .. 14; none of the four where there is no element)
    auto take_list = [&](uint32_t c) {
        c_put = c;
        const Place me = place();
#pragma unroll
        for (uint32_t r = 0; r < kEpRounds; ++r) {
            if constexpr (BITS != 8) {
                in_stage[r] = 0;
                if (!__any((e_now.first & ~3u) + 16u * r < e_now.end)) continue;
            }
            const uint32_t quad = (e_now.first & ~3u) + me.quad + 16u * r;
            ln_u32x4 put;
            uint32_t stages = 0;
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) {
                const uint32_t p = (k & 1) ? list.pos[r][k >> 1] >> 16 : list.pos[r][k >> 1];
                const int v = quad + k - e_now.first < e_now.end - e_now.first ? (int)(list.val[r] << (24 - 8 * k)) >> 24 : 0;
                put[k] = (ln_pack(0.0f, (float)v * scale) & 0xFFFF0000u) | (v != 0 ? (p & 0x300u) << 4 : 0x4000u) |
                         (((p & 0xF0u) << 4) + (p & 14u) + (me.kg << 6) + me.row * 16u);
                if constexpr (BITS != 8) stages |= 1u << ((put[k] >> 12) & 7u);
            }
            put_at[r] = put;
            if constexpr (BITS == 8) any[r] = __any((e_now.first & ~3u) + 16u * r < e_now.end);
            else
#pragma unroll
                for (uint32_t q = 0; q < 4; ++q) in_stage[r] |= (uint32_t)(__any(stages & (1u << q)) != 0) << q;
        }
        more = __any((e_now.first & ~3u) + 16u * kEpRounds < e_now.end);
        e_now = extent(c + 1u);
    };
    auto store = [&](uint32_t q) {  // stage q of the cell, to its half of the tile
        const uint32_t base = store_at + (q & 1u) * kEpTile;
        uint32_t o[16];
        ln_decode<BITS, false>(w[q % CODES], lut_lane, scale, o);
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k)
            *reinterpret_cast<LN_LDS(ln_u32x4) *>((uintptr_t)(base + ((k ^ q) << 10) + lane * 16u)) =
                ln_u32x4{o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]};
    };
    auto patch = [&](uint32_t q) {  // the listed elements of that stage over it
        const uint32_t base = store_at + (q & 1u) * kEpTile;
        ln_wave_order();
#pragma unroll
        for (uint32_t r = 0; r < kEpRounds; ++r)
            if (BITS == 8 ? any[r] : (in_stage[r] & (1u << q)) != 0) {
                const ln_u32x4 put = put_at[r];
                // (elements of other stages go aside, a dword a lane)
                const Place me = place();
                const uint32_t aside = smem + P::kLutBytes + 2u * kEpTile + kEpThreads * (16u * kEpRounds) + (me.kg * 16u + me.quad + me.row) * 4u;
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k) {
                    const uint32_t to = (put[k] ^ (q << 12)) & 0x7FFFu;
                    *reinterpret_cast<LN_LDS(uint16_t) *>((uintptr_t)(to < 4096u ? base + to : aside)) = (uint16_t)(put[k] >> 16);
                }
            }
        if (more) {  // rows with yet more listed elements in the cell
            const Extent x = extent(c_put);
            const Place me = place();
            for (uint32_t f = (x.first & ~3u) + 16u * kEpRounds + (me.quad >> 2); f < x.end; f += 4u) {
                const uint32_t p = exc_pos[lane_listed(f, me.row)];
                const int v = exc_val[lane_listed(f, me.row)];
                if (v != 0 && (p & 0x300u) == (q << 8))
                    *reinterpret_cast<LN_LDS(uint16_t) *>((uintptr_t)(base + (me.kg << 6) + me.row * 16u + ((p & 0xF0u) << 4) + (p & 14u))) =
                        (uint16_t)(ln_pack((float)v * scale, 0.0f) & 0xFFFFu);
            }
        }
    };

    take_list(0u);
    store(0);
    patch(0);
    codes(0u, CODES);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");

    ln_f32x4 acc[MI][NI];
#pragma unroll
    for (uint32_t i = 0; i < MI; ++i)
#pragma unroll
        for (uint32_t j = 0; j < NI; ++j) acc[i][j] = ln_f32x4{0, 0, 0, 0};
    if constexpr (NARROW) {
        // A wave's weights are its own: nothing waits for another wave.
        const LN_LDS(ln_u32x4) *const own = w_at + wave * 256u;
#pragma unroll 1
        for (uint32_t c = 0; c < n_cells; ++c) {
            const uint32_t c_next = min(c + 1u, n_cells - 1u);
#pragma unroll
            for (uint32_t q = 0; q < 4; ++q) {
                const uint32_t p = (q + 1u) & 3u;
                if (q == 1) list = quads(e_now);
                if (q == 3) take_list(c + 1u);
                ln_wave_order();
                ln_u32x4 v[4];
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) v[j] = own[(q & 1u) * (kEpTile / 16u) + j * 64u];
                store(p);
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) {
                    const uint32_t t = 4u * q + j;
#pragma unroll
                    for (uint32_t i = 0; i < MI; ++i)
                        acc[i][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(ln_bf16x8, v[j]), __builtin_bit_cast(ln_bf16x8, a[t % AHEAD][i]),
                                                                            acc[i][0], 0, 0, 0);
                    x_load(t + AHEAD < 16u ? c : c_next, (t + AHEAD) & 15u);
                }
                patch(p);
                codes(q + 1u + CODES < 4u ? c : c_next, (q + 1u + CODES) & 3u);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
    if constexpr (!NARROW) {
        // A stage of products, and the next stage's decode (past the end: the last cell's first stage again, which nobody reads).  Requests are
        // never inside a branch: the compiler counts what is in flight.
        if (mb0 >= n_blocks) {  // no rows: the decode only
#pragma unroll 1
            for (uint32_t c = 0; c < n_cells; ++c) {
                const uint32_t c_next = min(c + 1u, n_cells - 1u);
#pragma unroll
                for (uint32_t q = 0; q < 4; ++q) {
                    if (q == 1) list = quads(e_now);
                    if (q == 3) take_list(c + 1u);
                    store((q + 1u) & 3u);
                    patch((q + 1u) & 3u);
                    codes(q + 1u + CODES < 4u ? c : c_next, (q + 1u + CODES) & 3u);
                    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
                }
            }
            return;
        }
#pragma unroll 1
        for (uint32_t c = 0; c < n_cells; ++c) {
            const uint32_t c_next = min(c + 1u, n_cells - 1u);
#pragma unroll
            for (uint32_t q = 0; q < 4; ++q) {
                constexpr uint32_t PER = 16 / NI;  // pairs of weights decoded with each block's products
                const uint32_t p = (q + 1u) & 3u, base = store_at + (p & 1u) * kEpTile + lane * 16u;
                uint32_t o[16];
                auto piece = [&](uint32_t k) {
                    *reinterpret_cast<LN_LDS(ln_u32x4) *>((uintptr_t)(base + ((k ^ p) << 10))) = ln_u32x4{o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]};
                };
                auto products = [&](uint32_t j) {
                    const uint32_t t = 4u * q + j;
                    ln_u32x4 v[2];
                    auto weights = [&](uint32_t b) { v[b & 1u] = w_at[(q & 1u) * (kEpTile / 16u) + b * 256u + j * 64u]; };
                    weights(0);
#pragma unroll
                    for (uint32_t b = 0; b < NI; ++b) {
                        if (b + 1 < NI) weights(b + 1);
                        if (j == 0) {
                            if (b && b * PER % 4 == 0) piece(b * PER / 4 - 1);
                            uint32_t d[16];
                            ln_decode<BITS, false>(w[p % CODES], lut_lane, scale, d);
#pragma unroll
                            for (uint32_t k = b * PER; k < b * PER + PER; ++k) o[k] = d[k];
                            __builtin_amdgcn_sched_barrier(0);
                        }
#pragma unroll
                        for (uint32_t i = 0; i < MI; ++i)
                            acc[i][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(ln_bf16x8, v[b & 1u]),
                                                                                __builtin_bit_cast(ln_bf16x8, a[t % AHEAD][i]), acc[i][b], 0, 0, 0);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    if (j == 0) piece(3);
                    x_load(t + AHEAD < 16u ? c : c_next, (t + AHEAD) & 15u);
                    __builtin_amdgcn_sched_barrier(0);
                };
                if (q == 1) list = quads(e_now);
                if (q == 3) {
                    take_list(c + 1u);
                    __builtin_amdgcn_sched_barrier(0);
                }
                products(0);
                products(1);
                patch(p);
                __builtin_amdgcn_sched_barrier(0);
                codes(q + 1u + CODES < 4u ? c : c_next, (q + 1u + CODES) & 3u);
                products(2);
                products(3);
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            }
        }

    }
    // ---- the sums: lane (n, kg) of block (i, b) has weight rows 4 kg .. + 3 of row n ----
    if constexpr (FIRST) {
        // The sums of a block of rows go through LDS, which takes an index, so that a short loop works out four columns at a time: a copy of
        // the activations for each register of sums is 60 KB of instructions, of which every tile fetches what it passes through (512 rows
        // 14.7 us).
        const uint16_t *const bias = W.bias ? W.bias + (size_t)e * (R.gated ? 2u * W.outputs : W.outputs) : nullptr;
        LN_LDS(ln_f32x4) *const sums = reinterpret_cast<LN_LDS(ln_f32x4) *>((uintptr_t)(smem + P::kLutBytes + wave * 4096u + lane * 16u));
        const uint32_t per = R.gated ? 2u : 1u;
        // (of narrow tiles a wave has a block of rows, of which the four waves have the weight rows)
        constexpr uint32_t BLOCKS = NARROW ? 1 : MI;
        const uint32_t m0 = NARROW ? wave : mb0;
        if constexpr (NARROW) {
            __syncthreads();
#pragma unroll
            for (uint32_t i = 0; i < MI; ++i) sums[((int)i - (int)wave) * 256 + (int)wave * 64] = acc[i][0];
            __syncthreads();
        }
#pragma unroll
        for (uint32_t i = 0; i < BLOCKS; ++i) {
            if (m0 + i >= n_blocks) break;
            if constexpr (!NARROW) {
#pragma unroll
                for (uint32_t b = 0; b < NI; ++b) sums[b * 64u] = acc[i][b];
                ln_wave_order();
            }
            uint8_t *const block = R.inner + (size_t)(block0 + m0 + i) * R.n_kb_inner * 1024u;
#pragma unroll 1
            for (uint32_t b = 0; b < kEpWaves; b += per) {
                const uint32_t col = (tile * kEpWaves + b) / per * 16u + 4u * kg;
                if (col >= R.n_kb_inner * 32u) continue;
                ln_f32x4 v = sums[b * 64u];
                if (bias)
#pragma unroll
                    for (uint32_t k = 0; k < 4; ++k) v[k] += bf16_bits_to_f32(bias[min(col + k, W.outputs - 1u)]);
                ep_activations(R.activation, v);
                if (R.gated) {
                    ln_f32x4 u = sums[(b + 1u) * 64u];
                    if (bias)
#pragma unroll
                        for (uint32_t k = 0; k < 4; ++k) u[k] += bf16_bits_to_f32(bias[W.outputs + min(col + k, W.outputs - 1u)]);
#pragma unroll
                    for (uint32_t k = 0; k < 4; ++k) v[k] *= u[k];
                }
                uint32_t h[4];
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k) h[k] = col + k < W.outputs ? ep_bf16(v[k]) : 0u;
                *reinterpret_cast<ln_u32x2 *>(block + (col >> 5) * 1024u + (((col >> 3) & 3u) * 16u + n) * 16u + (col & 4u) * 2u) =
                    ln_u32x2{h[0] | h[1] << 16, h[2] | h[3] << 16};
            }
            ln_wave_order();
        }
        // columns of the intermediate's last cell that no weight row makes: zeros
        if (tile + 1u == R.w_tiles) {
            const uint32_t from = R.w_tiles * (kEpRows / per) / 32u;
            for (uint32_t i = 0; i < BLOCKS && m0 + i < n_blocks; ++i)
                for (uint32_t kb = from; kb < R.n_kb_inner; ++kb)
                    reinterpret_cast<ln_u32x4 *>(R.inner)[((size_t)(block0 + m0 + i) * R.n_kb_inner + kb) * 64u + lane] = ln_u32x4{0u, 0u, 0u, 0u};
        }
    } else {
        const uint16_t *const bias = W.bias ? W.bias + (size_t)e * W.outputs : nullptr;
#pragma unroll
        for (uint32_t i = 0; i < MI; ++i) {
            if (mb0 + i >= n_blocks) break;
            const uint32_t slot = R.order[(block0 + mb0 + i) * 16u + n];
            if (slot == kEpNone) continue;
            float *const to = R.out + (size_t)slot * W.outputs;
#pragma unroll
            for (uint32_t b = 0; b < NI; ++b) {
                const uint32_t col = (tile * kEpWaves + (NARROW ? wave : b)) * 16u + 4u * kg;
                ln_f32x4 v = acc[i][b];
                if (bias)
#pragma unroll
                    for (uint32_t k = 0; k < 4; ++k) v[k] += bf16_bits_to_f32(bias[min(col + k, W.outputs - 1u)]);
                if (W.outputs % 4u == 0) {  // (rows of whole 16 bytes)
                    if (col < W.outputs) *reinterpret_cast<ln_f32x4 *>(to + col) = v;
                } else {
#pragma unroll
                    for (uint32_t k = 0; k < 4; ++k)
                        if (col + k < W.outputs) to[col + k] = v[k];
                }
            }
        }
    }
}

template <int BITS, bool FIRST>
__global__ void __launch_bounds__(kEpThreads) __attribute__((amdgpu_waves_per_eu(3)))
k_experts_prompt(ExMatrix W, EpCall R) {
    extern __shared__ __attribute__((aligned(16))) uint8_t ep_smem[];
    // workgroups go round the eight XCDs: all weight tiles of a row tile to one of them
    const uint32_t id = blockIdx.x, turn = id >> 3, row_tile = (turn / R.w_tiles) * 8u + (id & 7u), tile = turn % R.w_tiles;
    if (row_tile >= *R.n_tiles) return;
    const uint32_t e = R.tiles[3u * row_tile], block0 = R.tiles[3u * row_tile + 1u], n_blocks = R.tiles[3u * row_tile + 2u];
    if (n_blocks == 1u) ep_tile<BITS, 1, true, FIRST>(W, R, e, block0, n_blocks, tile, ep_smem);
    else if (n_blocks <= kEpWaves) ep_tile<BITS, 1, false, FIRST>(W, R, e, block0, n_blocks, tile, ep_smem);
    else if (n_blocks <= 2u * kEpWaves) ep_tile<BITS, 2, false, FIRST>(W, R, e, block0, n_blocks, tile, ep_smem);
    else if (n_blocks <= 3u * kEpWaves) ep_tile<BITS, 3, false, FIRST>(W, R, e, block0, n_blocks, tile, ep_smem);
    else ep_tile<BITS, 4, false, FIRST>(W, R, e, block0, n_blocks, tile, ep_smem);
}

template <int BITS, bool FIRST> int ep_launch(const ExMatrix &W, EpCall R, uint32_t row_tiles, hipStream_t s) {
    constexpr size_t lds = LnPairs<BITS, false>::kLutBytes + 2u * kEpTile + 16u * kEpRounds * kEpThreads + kWave * 4u;
    static_assert(3u * lds <= kLnLds, "LDS of a CU");
    static const bool raised = hipFuncSetAttribute(reinterpret_cast<const void *>(k_experts_prompt<BITS, FIRST>),
                                                   hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) == hipSuccess;
    if (!raised) return IXH_ELAUNCH;
    R.w_tiles = (W.n_tiles * 4u + kEpRows - 1u) / kEpRows;
    IXH_LAUNCH((k_experts_prompt<BITS, FIRST>), dim3((row_tiles + 7u) / 8u * 8u * R.w_tiles), dim3(kEpThreads), lds, s, W, R);
    return hipGetLastError() == hipSuccess ? IXH_OK : IXH_ELAUNCH;
}
template <bool FIRST> int ep_matrix(const ExMatrix &W, const EpCall &R, uint32_t row_tiles, hipStream_t s) {
    switch (W.bits) {
        case 3: return ep_launch<3, FIRST>(W, R, row_tiles, s);
        case 4: return ep_launch<4, FIRST>(W, R, row_tiles, s);
        case 5: return ep_launch<5, FIRST>(W, R, row_tiles, s);
        default: return ep_launch<8, FIRST>(W, R, row_tiles, s);
    }
}
// (a source file each: they take the compiler a while)
int ep_first(const ExMatrix &W, const EpCall &R, uint32_t row_tiles, hipStream_t s);
int ep_second(const ExMatrix &W, const EpCall &R, uint32_t row_tiles, hipStream_t s);

}  // namespace ixh
