// Translation unit of the second gfx950 code object in libbrik.so: the attention side of a decoder layer. Apart from the
// matmul kernels, so that neither moves the other's code and the two compile side by side.
#include "kv_rows.hip"
#include "attn_few.hip"
#include "attn_tile.hip"
#include "attn_join.hip"
