// The third gfx950 code object of the host library: 8-bit floating point with a
// scale for each 128 (rows quantized by their producers, products with block-scaled
// weights). Compiled and embedded like kernels.hip, beside it.
#include "common.hpp"
#include "tiles.hpp"
#include "f8_rows.hpp"
#include "f8_gemm.hpp"
#include "f8_tile.hpp"
#include "f8_few.hpp"
