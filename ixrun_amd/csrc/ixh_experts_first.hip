// The first matrix of experts with many tokens.
#include "ixh_experts_prompt.h"

namespace ixh {

int ep_first(const ExMatrix &W, const EpCall &R, uint32_t row_tiles, hipStream_t s) { return ep_matrix<true>(W, R, row_tiles, s); }

}  // namespace ixh
