// Instantiations of the 8-bit block-scaled GEMM kernel. Ring depths are the deepest that fit 227 KB of shared memory next to
// the receive area of cluster split-K (single CTAs) or the store images (pairs); shallower rings were never faster.
#include "gemm_a8w8_variants.h"

namespace b200 {

namespace {
template <int TILE_Q, int STAGES, int CG, bool VVEC, bool PACKED>
Variant8 make_one() {
  using L = Smem8<TILE_Q, STAGES, CG, VVEC, PACKED>;
  static_assert(L::kDynBytes <= 227 * 1024, "shared memory of a variant");
  Variant8 v;
  v.tile_q = TILE_Q, v.cta_group = CG, v.stages = STAGES;
  v.fn = gemm_a8w8_sm100_kernel<TILE_Q, STAGES, CG, VVEC, PACKED>;
  v.smem_bytes = L::kDynBytes;
  return v;
}
template <int TILE_Q, int STAGES, int CG>
Variant8 make(int v_vector) {
  return v_vector ? make_one<TILE_Q, STAGES, CG, true, false>() : make_one<TILE_Q, STAGES, CG, false, false>();
}
}  // namespace

bool variant8(int tile_q, int cta_group, int v_vector, int packed, Variant8* out) {
  if (packed) {
    if (cta_group == 1 && tile_q == 128) return *out = make_one<128, 5, 1, false, true>(), true;
    if (cta_group == 2 && tile_q == 256) return *out = make_one<256, 5, 2, false, true>(), true;
    return false;
  }
  if (cta_group == 1 && tile_q == 16) return *out = make<16, 10, 1>(v_vector), true;
  if (cta_group == 1 && tile_q == 32) return *out = make<32, 9, 1>(v_vector), true;
  if (cta_group == 1 && tile_q == 64) return *out = make<64, 7, 1>(v_vector), true;
  if (cta_group == 1 && tile_q == 128) return *out = make<128, 4, 1>(v_vector), true;
  if (cta_group == 2 && tile_q == 128) return *out = make<128, 7, 2>(v_vector), true;
  if (cta_group == 2 && tile_q == 256) return *out = make<256, 4, 2>(v_vector), true;
  return false;
}

}  // namespace b200
