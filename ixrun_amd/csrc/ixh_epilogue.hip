// An epilogue by itself, for products whose kernel has none.
#include "ixh_epilogue.h"

namespace ixh {

// Bound: its requests, of two bytes a lane, and one row after another a workgroup, so that its accesses are consecutive in each operand.  silu, multiplier
// and residual at 512 x 5120 6.5 us (3.2 TB/s, from caches), 4096 x 4096 47 us (2.9), 4096 x 17408 290 us (2.0, where a copy reaches 4.9); next to a product that
// a layer without an epilogue of its own takes 100 us and more for.
__global__ void __launch_bounds__(256)
k_epilogue(const uint16_t *v, int64_t ldv, uint32_t m, uint32_t out_f, uint16_t *y, int64_t ldy, Epilogue ep) {
    const uint32_t at = blockIdx.y * 256u + threadIdx.x;
    if (at >= out_f) return;
    for (uint32_t r = blockIdx.x; r < m; r += gridDim.x)
        y[(int64_t)r * ldy + at] = ep.output(bf16_bits_to_f32(v[(int64_t)r * ldv + at]), r, at);
}

int launch_epilogue(const uint16_t *v, int64_t ldv, uint32_t m, uint32_t out_f, uint16_t *y, int64_t ldy, Epilogue ep, hipStream_t s) {
    const uint32_t columns = (out_f + 255u) / 256u;
    if (columns > 65535u) return IXH_EUNSUPPORTED;
    IXH_LAUNCH(k_epilogue, dim3(m < 65536u ? m : 65536u, columns), dim3(256), 0, s, v, ldv, m, out_f, y, ldy, ep);
    return hipGetLastError() == hipSuccess ? IXH_OK : IXH_ELAUNCH;
}

}  // namespace ixh
