// GQA attention with modified scores over 8-bit caches.
#include "gqa_attention.h"

int aia::launch_gqa_fp8_scored(const AttnArgs& a, const PrefillArgs& pa, const Layout& L,
                               const Geometry& g, int32_t head_dim, int32_t waves, bool one_block,
                               hipStream_t s) {
  return launch_gqa<kKvFp8, true>(a, pa, L, g, head_dim, waves, one_block, s);
}
