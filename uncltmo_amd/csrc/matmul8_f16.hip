// The tiled 8-bit products with fp16 results (matmul8.h).
#include "matmul8.h"

int mm_tiles_f16(const MmArgs& p, int a_fmt, bool b_tile, hipStream_t s) { return launch_by_format<f16_t, true>(p, a_fmt, b_tile, s); }
