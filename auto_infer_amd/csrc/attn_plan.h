// What the planner and the attention kernels share: tile and item sizes, a
// step's geometry and the layout of its workspace.
#pragma once

#include "common.h"

namespace aia {

// A segment is (request, query block, kv-head group, head block): the
// work-group that owns one of its key ranges runs one wave per kv head of
// the group over the same keys, so every tile reads whole contiguous
// (block_size x Hkv x D) cache slots.
struct Geometry {
  int32_t hkv, group, hb, nhb, qb, nw, nkvg, rb, qs, pf;
  int32_t ncu;   // compute units of the current device (MLA range count and dealing)
};

// Workspace layout (all offsets 256-byte aligned).
struct Layout {
  int64_t hdr, seg, wave, part_ml, part_o, req, mrg, pf, pfm, pfw, pf_o, pf_ml, total;
  int64_t seg_cap, part_cap, mrg_cap, pf_cap, pf_unit_cap, pf_mrg_cap, pf_slots;
};

// What a call does beyond scale * q.k over bf16 caches.  Scores in log2 units:
// with a cap, cap_out * tanh(q.k * scale / cap), as cap_out - 2 cap_out /
// (exp2(q.k * cap_in) + 1); then minus slope_log2 * |query - key position|.
struct ScoreArgs {
  const uint8_t* ks;         // e8m0 scales of 8-bit caches, (num_blocks, Hkv)
  const uint8_t* vs;
  const float* slopes;       // distance bias per query head, or null
  const int32_t* prefix;     // keys of each request that all its rows see, or null
  const int32_t* kvlen;
  float cap_in, cap_out;     // cap_out 0: no cap
  float cap_unit;            // scale / cap
  float cap_small;           // |q.k| up to which cap_poly serves
  float cap_poly[5];         // in (q.k cap_unit)^2, times q.k
  float cap_raw[5];          // the same in (q.k)^2; all 0 where that leaves float32's range
};

struct AttnArgs {
  const uint16_t* q;
  int64_t q_ts, q_hs;
  uint16_t* kc;
  uint16_t* vc;
  // this step's new K/V rows (T, Hkv, D); when set, keys at the new
  // positions are read from them and written into the cache by the kernel
  const uint16_t* kn;
  const uint16_t* vn;
  int64_t kn_ts, vn_ts;
  const int32_t* bt;
  int64_t bt_stride;
  int32_t hkv, group, hb, bs, nb, nw;
  float scale_log2;
  const int32_t* seg;
  const int32_t* wave_rec;
  uint16_t* part_o;          // split partials (fp16, scaled per row)
  float2* part_ml;
  uint16_t* out;
  int64_t o_ts, o_hs;
  int32_t waves;
  const int32_t* hdr;
  int32_t batch, tokens;
  ScoreArgs sc;
};

struct PrefillArgs {
  const uint16_t* q;
  int64_t q_ts, q_hs;
  uint16_t* kc;
  uint16_t* vc;
  const uint16_t* kn;
  const uint16_t* vn;
  int64_t kn_ts, vn_ts;
  const int32_t* bt;
  int64_t bt_stride;
  const int32_t* cu_q;
  const int32_t* kvlen;
  int32_t hkv, group, bs, nb, batch, tokens;
  float scale_log2;
  uint16_t* out;
  int64_t o_ts, o_hs;
  const int4* dealt;         // work-group b: {request, first row, first tile, end tile},
                             // {first query token, query tokens, keys, first tile's block id},
                             // {unit, kv head}
  const int32_t* hdr;
  uint16_t* part_o;          // partials of chunked items, two fp16 row blocks per (unit, kv head)
  float2* part_ml;
  int32_t part_units;        // units the partial buffer holds
  ScoreArgs sc;
};

// Cache formats a GQA kernel is built for.
constexpr int kKvNd = 0, kKvNz = 1, kKvFp8 = 2;

// The attention launches of one call (without the merge) that sources of their
// own build: modified scores over bf16 caches, and 8-bit caches.
using LaunchGqa = int(const AttnArgs& a, const PrefillArgs& pa, const Layout& L, const Geometry& g,
                      int32_t head_dim, int32_t waves, bool one_block, hipStream_t s);
LaunchGqa launch_gqa_scored_nd, launch_gqa_scored_nz, launch_gqa_fp8, launch_gqa_fp8_scored;

}  // namespace aia

namespace {

using aia::AttnArgs;
using aia::Geometry;
using aia::Layout;
using aia::PrefillArgs;
using aia::ScoreArgs;
using aia::float4_t;
using aia::short4_t;

constexpr int kHeadDim = 128;
constexpr int kTile = 16;         // keys per MFMA tile
constexpr int kRows = 16;         // query rows per segment (MFMA N)
// LDS row stride (elements) of a staged V tile: 288 bytes puts the 16 rows
// of a transposing read in distinct banks
constexpr int kVStride = 144;
constexpr int kMaxBatch = 8192;   // planner keeps the request offsets in LDS
constexpr int kDefaultWaves = 2048;
constexpr int kMaxWaves = 16384;
constexpr int kPlanThreads = 512;
// Per-range work record: {segment, first tile, end tile, tiles per range,
// the segment's 8-int record, first logical block, last segment of the
// range, 2 pad, the first 16 block ids of the range} -- everything a
// work-group needs to issue its first K/V loads after one load.
constexpr int kRecInts = 32;
constexpr int kRecBlocks = 16;

constexpr int kMaxGroupWaves = 8;  // kv heads (waves) per work-group

// Prefill routing: a GQA request whose query rows (query tokens x group
// heads) fill at least one prefill work item is planned for the prefill
// kernel (all its rows' keys staged once per 128 rows in LDS) instead of
// split-K segments.  AIA_PREFILL=0 builds the split-K-only planner.
#ifndef AIA_PREFILL
#define AIA_PREFILL 1
#endif
// AIA_MLA_PREFILL=0 keeps absorbed-MLA prefill steps on the split-K kernel.
#ifndef AIA_MLA_PREFILL
#define AIA_MLA_PREFILL 1
#endif
#ifndef AIA_PF_WAVES
#define AIA_PF_WAVES 4
#endif
#ifndef AIA_PF_KEYS
#define AIA_PF_KEYS 64
#endif
#ifndef AIA_PF_RT
#define AIA_PF_RT 2
#endif
constexpr int kPfWaves = AIA_PF_WAVES;       // waves per prefill work-group
constexpr int kPfRt = AIA_PF_RT;             // 16-row MFMA tiles per wave
constexpr int kPfRows = 16 * kPfRt * kPfWaves;   // rows per prefill work item
constexpr int kPfKeys = AIA_PF_KEYS;         // keys per staged K/V tile (32 or 64)
// Items alone fill the chip when items x kv heads reach kPfTargetWgs (a
// little under two resident work-groups per CU); below that, each item's key
// tiles are cut into chunks of at least kPfMinChunk tiles, sized so all units
// still fit in one round (fp16 partials scaled per row, merged with the
// split-K partials' rule).  448 rather than 512: fewer, longer chunks write
// fewer partials, and the CUs left with one work-group take the largest
// units (configs[1] prefill chunks, us per call: 43.1 at 448 or 416, 44.6 at
// 512, 44.1-44.5 at 384, 49.6-49.9 at 256-320; 416 is slower at 32K keys).
#ifndef AIA_PF_TARGET
#define AIA_PF_TARGET 448
#endif
constexpr int kPfTargetWgs = AIA_PF_TARGET;
constexpr int kPfCutSlots = 512;     // most work-groups (units x kv heads) of a step with cut items
static_assert(kPfTargetWgs <= kPlanThreads && kPfCutSlots <= kPlanThreads, "a thread per cut item and unit");
constexpr int kPfRecBytes = 48;      // a dealt work-group's record: three int4
static_assert(2 * kPfTargetWgs >= kPfCutSlots && (2 * kPfTargetWgs - kPfCutSlots) * kPfRows * 8 >=
              kPfCutSlots * kPfRecBytes, "partials and records of a step with cut items");
#ifndef AIA_MLA_LPT
#define AIA_MLA_LPT 1
#endif

constexpr int kPfMinChunk = 8;

#ifndef AIA_MIXED
#define AIA_MIXED 1
#endif
// Prefill units and split-K ranges of a step run in one grid (gqa_mixed_kernel).
__host__ __device__ inline bool mixed_grid(const Geometry& g, int32_t dv) {
  return AIA_MIXED && g.pf && g.nw == kPfWaves && g.rb == 1 && dv == kHeadDim;
}

constexpr int kMergeDims = 16;   // output dims per merge element
constexpr int kMrgInts = 8;      // merge record

}  // namespace
