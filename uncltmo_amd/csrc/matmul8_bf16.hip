// The tiled 8-bit products with bf16 results (matmul8.h).
#include "matmul8.h"

int mm_tiles_bf16(const MmArgs& p, int a_fmt, bool b_tile, hipStream_t s) { return launch_by_format<bf16_t, false>(p, a_fmt, b_tile, s); }
