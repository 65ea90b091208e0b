// Routing to experts and the experts' products: what the launchers of ixh_route.hip and ixh_experts*.hip take.
#pragma once
#include "ixh_dev.h"
#include "ixh_lanes.h"

namespace ixh {

struct RouteDev {
    uint32_t experts, top_k, groups, group_size, top_groups;
    bool sigmoid, renormalize;
    double scale;
};
constexpr uint32_t kRtMostExperts = 1024, kRtMostGroups = 64, kRtMostChosen = 64;
int launch_route(const void *logits, int dtype, int64_t ld, uint32_t tokens, const RouteDev &R, const float *bias, int32_t *ids, float *weights,
                 hipStream_t s);

// One matrix of every expert in the lane layout (ixh_lanes.h): the experts' planes and cell tables one after another, one list.
struct ExMatrix {
    const uint32_t *plane;    // plane_words each
    const uint32_t *exc_off;  // n_tiles * n_cells + 1 each, counted through all experts
    const uint16_t *exc_pos;
    const int8_t *exc_val;
    const uint16_t *scale;    // one each
    const uint16_t *bias;     // or NULL: `outputs` each, of a gated first matrix `outputs` of the gate and as many of the other half
    uint64_t plane_words;
    uint32_t n_tiles, n_cells, in_f, outputs;
    int bits;
};

// Of a gated first matrix the blocks of 16 rows take turns: 16 of the gate, then the same 16 of the other half.
struct ExDev {
    ExMatrix first, second;
    uint32_t experts, hidden, inner;
    int activation;
    bool gated;
};

constexpr uint32_t kExMostExperts = 1024;
constexpr uint32_t kExMostSlots = 1u << 20;  // of a call: tokens times experts of each

struct ExCall {
    const uint16_t *x;
    int64_t ldx;
    uint32_t tokens, top_k;
    const int32_t *ids;
    const float *weights;
    const uint16_t *residual;
    int64_t ld_residual;
    uint16_t *y;
    int64_t ldy;
};

// The slots by expert.  For k_experts_rows tiles of a few slots each, {expert, first place in `order`, how many}; for k_experts_prompt
// an expert's places are filled up to whole blocks of 16 (with ~0), and the tiles are {expert, first block, blocks}, up to 16 of them.
struct ExPlan {
    uint32_t *n_tiles, *n_blocks, *tiles, *order;
};
// many tokens to an expert (ixh_experts_prompt.hip); row_tiles and blocks: how many there may be
int launch_experts_prompt(const ExDev &X, const ExCall &call, const ExPlan &plan, uint32_t row_tiles, uint32_t blocks, void *xt, void *inner,
                          float *per_slot, hipStream_t s);

// a slot by itself (ixh_experts_one.hip): rows of up to sixteen cells
struct ExOne {
    const uint16_t *x;
    int64_t ldx;
    uint32_t rows;  // of x
    const int32_t *ids;
    void *out;  // the intermediate in bf16, fp32, or (joined) y
    int64_t ld_out;
    uint32_t experts, tokens, top_k;
    int activation;
    bool gated;
    const float *weights;  // joined: what a token's slots are added with
    const uint16_t *residual;
    int64_t ld_residual;
};
bool experts_one_takes(const ExMatrix &W, bool gated);
int launch_experts_one(const ExMatrix &W, const ExOne &R, bool first, hipStream_t s);
// the second matrix with the sum over a token's slots
bool experts_joined_takes(const ExMatrix &W, uint32_t tokens, uint32_t top_k);
int launch_experts_joined(const ExMatrix &W, const ExOne &R, hipStream_t s);

size_t experts_workspace_bytes(const ExDev &X, uint32_t tokens, uint32_t top_k);
int launch_experts(const ExDev &X, const ExCall &call, void *workspace, hipStream_t s);

}  // namespace ixh
