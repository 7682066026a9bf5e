// GQA attention with modified scores (a tanh cap, a distance bias, a prefix
// that all rows see) over bf16 caches in the standard layout.
#include "gqa_attention.h"

int aia::launch_gqa_scored_nd(const AttnArgs& a, const PrefillArgs& pa, const Layout& L,
                              const Geometry& g, int32_t head_dim, int32_t waves, bool one_block,
                              hipStream_t s) {
  return launch_gqa<kKvNd, true>(a, pa, L, g, head_dim, waves, one_block, s);
}
