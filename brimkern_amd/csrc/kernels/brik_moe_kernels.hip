// Translation unit of the third gfx950 code object in libbrik.so: what a mixture-of-experts layer runs around its products, and
// products of 8-bit integers.
#include "moe_route.hip"
#include "moe_rows.hip"
#include "quant_i8.hip"
#include "gemm_i8.hip"
