// The kernels of gqa_scored.hip over caches in the NZ layout.
#include "gqa_attention.h"

int aia::launch_gqa_scored_nz(const AttnArgs& a, const PrefillArgs& pa, const Layout& L,
                              const Geometry& g, int32_t head_dim, int32_t waves, bool one_block,
                              hipStream_t s) {
  return launch_gqa<kKvNz, true>(a, pa, L, g, head_dim, waves, one_block, s);
}
