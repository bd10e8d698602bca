// Menu of the compiled 8-bit GEMM variants.
#pragma once
#include "gemm_a8w8_kernel.cuh"

namespace b200 {

struct Variant8 {
  Kernel8Fn fn;
  int tile_q, cta_group, stages, smem_bytes;
};

// packed: both operands' scales are exponent tiles. Otherwise v_vector: the operand on the MMA N axis has a scale per row (otherwise per 128 rows). False: no such variant.
bool variant8(int tile_q, int cta_group, int v_vector, int packed, Variant8* out);

}  // namespace b200
