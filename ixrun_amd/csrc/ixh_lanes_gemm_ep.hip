// The kernels of ixh_lanes_gemm.hip with an epilogue in place of their own output (see ixh_epilogue.h).
#define IXH_EP
#include "ixh_lanes_gemm.hip"
