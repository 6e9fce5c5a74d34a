// The second gfx950 code object: the microscaled types and the scored routing.
#include "qmm_mx_common.h"
#include "qmm_mx_quant_kernels.h"
#include "qmm_mx_gemm_kernels.h"
#include "qmm_route_kernels.h"
