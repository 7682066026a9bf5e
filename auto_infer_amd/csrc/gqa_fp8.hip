// GQA attention over 8-bit caches (e4m3 values, an e8m0 scale per block and KV
// head).
#include "gqa_attention.h"

int aia::launch_gqa_fp8(const AttnArgs& a, const PrefillArgs& pa, const Layout& L, const Geometry& g,
                        int32_t head_dim, int32_t waves, bool one_block, hipStream_t s) {
  return launch_gqa<kKvFp8, false>(a, pa, L, g, head_dim, waves, one_block, s);
}
