// The second matrix of experts with many tokens.
#include "ixh_experts_prompt.h"

namespace ixh {

int ep_second(const ExMatrix &W, const EpCall &R, uint32_t row_tiles, hipStream_t s) { return ep_matrix<false>(W, R, row_tiles, s); }

}  // namespace ixh
