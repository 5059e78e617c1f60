// The second gfx950 code object of the host library: products with half-typed
// weight stacks on grouped rows (rfxq_group_rows, rfxq_grouped_gemm,
// rfxq_lora_add). Compiled and embedded like kernels.hip, apart from it so that
// the two compile side by side.
#include "common.hpp"
#include "rows.hpp"
#include "grouped.hpp"
#include "lora.hpp"
