// Attention for a batch whose requests share prefixes: the keys that a group of
// requests has in common are read once for all of the group's query rows, and each
// request's own keys once for its rows; the parts of a row are joined by their running
// maxima and sums.
//
// With n requests of lk keys of which S are shared, a step reads S + n (lk - S) rows of
// K and V instead of n lk.  The group's query rows (tokens x heads of a KV head) fill
// MFMA tiles against the shared keys: 128 rows against a tile of 64 keys take about as
// long as the tile's 32 KB need from memory, so up to that many rows the shared part
// is bound by memory, beyond by the matrix cores.
//
// The planner finds what is shared by comparing block tables, so a wrong group only
// costs speed.  A request joins those with which it saves most: see shared_level_kernel.
// It cuts the work into units of up to 128 rows of one KV head and a run of
// keys; a work-group takes one, with 64-key tiles of K and V staged in LDS.
#include <algorithm>

#include "row_parts.h"

namespace {

constexpr int kShWaves = 4, kShThreads = 64 * kShWaves;
constexpr int kUnitRows = 128;
constexpr int kRt = kUnitRows / (16 * kShWaves);          // 16-row tiles per wave
constexpr int kLightRows = 64;                            // up to here a unit waits for memory
constexpr int kKeys = 64;                                 // keys of a tile
constexpr int kMaxShared = 4096;                          // requests: the planner's LDS arrays
constexpr int kShPlanT = 1024;
constexpr int kTargetGroups = 512;                        // units to aim at: two per compute unit
// Tiles of a cut: fewer make a unit's queries and its join cost more, more leave small
// steps few units.  16 requests on a prefix of 4K: 21.6 us with eight, 20.4 with four; 40
// requests of three tokens on five prefixes, 8-bit: 21.8 and 23.2.
constexpr int kMinCut = 8;
// Units of a kind in a row.  128 requests on a prefix of 32K, before later steps: 262 us
// with 256 (a unit per compute unit), 272 with all heavy ones first, 281 with 512.
constexpr int kTurn = 256;
constexpr int kMinShare = 128;                            // keys worth a part of their own
constexpr int kLevels = 24;                               // of agreement: kMinShare << level keys
constexpr int kRecord = 12, kHdr = 64;

// What the attention kernels need of a layer's caches.
struct CacheArgs {
  const uint16_t* kc;        // (num_blocks, bs, hkv, D) bf16, or e4m3 bytes
  const uint16_t* vc;
  const uint8_t* ks;         // e8m0 scales (num_blocks, hkv) of 8-bit caches
  const uint8_t* vs;
  int32_t group, bs, nb;
  float scale_log2;          // score factor times log2(e)
};

// A row set against a run of keys: the rows of a group against what it shares, or of
// a request against its own keys.  Rows [0, rows) of one KV head, token-major, in
// tiles of 128; the keys in `cuts` runs.
struct Entity {
  int32_t part_base, rows, k0, k1;                        // part_base -1: straight to the output
  int32_t token_base, cuts, pad0, pad1;
};

struct ShLayout {
  int64_t hdr, lead, common, place, tokreq, order, ent, level, rec, part_head, part_o, total;
  int32_t wg_cap;
  int64_t part_cap;
};
ShLayout sh_layout(int32_t batch, int32_t tokens, int32_t hq, int32_t hkv, int32_t d) {
  auto up = [](int64_t x) { return (x + 255) & ~255ll; };
  ShLayout L;
  // every entity's cuts: its share of kTargetGroups, and one more for each tile
  const int64_t tiles = 2 * ((int64_t)tokens * (hq / hkv) / kUnitRows) + 2ll * batch;
  L.wg_cap = (int32_t)std::min<int64_t>(INT32_MAX / 2, kTargetGroups + tiles * hkv);
  L.part_cap = 2ll * tokens * hq + (int64_t)kTargetGroups * kUnitRows;
  L.hdr = 0;
  L.lead = up(kHdr * 4);
  L.common = L.lead + up(4ll * batch);
  L.place = L.common + up(4ll * batch);
  L.tokreq = L.place + up(4ll * batch);
  L.order = L.tokreq + up(16ll * tokens);
  L.ent = L.order + up(4ll * tokens);
  L.level = L.ent + up((int64_t)sizeof(Entity) * 2 * batch);
  L.rec = L.level + up(4ll * batch);
  L.part_head = L.rec + up(4ll * kRecord * L.wg_cap);
  L.part_o = L.part_head + up((int64_t)sizeof(PartHead) * L.part_cap);
  L.total = L.part_o + up(2 * L.part_cap * d);
  return L;
}

struct ShPlanArgs {
  const int32_t* cu;
  const int32_t* lk;
  const int32_t* bt;
  const int32_t* gid;        // group of each request (negative: alone), or null
  int64_t bt_stride;
  int32_t batch, tokens, bs, width, group, hq, hkv, wg_cap;
  int64_t part_cap;
  int32_t* hdr;              // {work-groups, status}
  int32_t* lead;             // first request of each request's group
  int32_t* common;           // keys that it has in common with that one, in front of its new tokens
  int32_t* place;            // tokens of the group's requests before it
  int4* tokreq;              // {request, token of it, group's first request (-1: alone), place}
  int32_t* order;            // tokens of the sharing groups, group by group
  Entity* ent;               // [0, batch) groups by first request, [batch, 2 batch) requests
  int32_t* level;            // of agreement on which each request's group rests (-1: alone)
  int32_t* rec;
};

// Requests with fewer query rows than a unit share; longer ones use each tile of
// keys 128 times as it is.
__device__ __forceinline__ bool shares(const ShPlanArgs& a, int b) {
  const int lq = a.cu[b + 1] - a.cu[b];
  return lq > 0 && lq * a.group < kUnitRows && a.lk[b] > lq;
}

// ------------------------------------------------------------------ plan

// Keys of a request that others may have in common with it: those in front of its new
// tokens (0: it shares none).
__device__ __forceinline__ int cached_keys(const ShPlanArgs& a, int b) {
  return shares(a, b) && (!a.gid || a.gid[b] >= 0) ? min(a.lk[b] - (a.cu[b + 1] - a.cu[b]), a.width * a.bs) : 0;
}
__device__ __forceinline__ int levels_of(int cached) {        // those whose keys are all cached
  return cached < kMinShare ? 0 : 32 - __builtin_clz(cached / kMinShare);
}
// The requests that a group is made of: of one group_ids entry, or of one first block.
__device__ __forceinline__ int group_key(const ShPlanArgs& a, int b) {
  return a.gid ? a.gid[b] : a.bt[(int64_t)b * a.bt_stride];
}
// The block of the last of a request's first kMinShare << level keys.  Tables that agree in
// it are taken to agree up to it, as those of a prefix cache do.
__device__ __forceinline__ int block_at(const ShPlanArgs& a, int b, int level) {
  return a.bt[(int64_t)b * a.bt_stride + ((kMinShare << level) - 1) / a.bs];
}

// One work-group per request: how far the others agree with it, in powers of two of
// kMinShare keys, and the level at which the keys times the requests that agree so far are
// most.  Requests of one level and block form a group.  So one that has little in common
// with the rest, or is short, does not cut down what they share, and two families behind
// one beginning share by family where that saves more.  It adds 4 to 5 us to a step's plan;
// 128 requests on a prefix of 32K and one more that has 128 keys of it take 240 us, and
// 1,315 where the least common length of all counts.
__global__ __launch_bounds__(256) void shared_level_kernel(ShPlanArgs a) {
  __shared__ int agree[kLevels];             // requests that agree up to a level and not the next
  __shared__ int own[kLevels];
  const int b = blockIdx.x, tid = threadIdx.x;
  const int levels = levels_of(cached_keys(a, b));
  if (tid < kLevels) agree[tid] = 0;
  if (tid < levels) own[tid] = block_at(a, b, tid);
  __syncthreads();
  if (levels > 0) {
    const int key = group_key(a, b);
    for (int o = tid; o < a.batch; o += 256) {
      if (o == b || group_key(a, o) != key) continue;
      const int n = min(levels, levels_of(cached_keys(a, o)));
      int far = 0;                           // levels that agree; eight are loaded at a time
      for (int l0 = 0; l0 < n && far == l0; l0 += 8) {
        bool same[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) same[u] = l0 + u < n && block_at(a, o, min(l0 + u, n - 1)) == own[min(l0 + u, n - 1)];
#pragma unroll
        for (int u = 0; u < 8; ++u) far += far == l0 + u && same[u];
      }
      if (far > 0) atomicAdd(&agree[far - 1], 1);
    }
  }
  __syncthreads();
  if (tid == 0) {
    int best = -1, requests = 0;
    int64_t most = 0;
    for (int l = levels - 1; l >= 0; --l) {
      requests += agree[l];
      const int64_t saved = (int64_t)(kMinShare << l) * requests;
      if (saved > most) { best = l; most = saved; }
    }
    a.level[b] = best;
  }
}

// One work-group per request: its group's first request, its place in the group and
// the keys that it has in common with the first.
__global__ __launch_bounds__(256) void shared_find_kernel(ShPlanArgs a) {
  __shared__ int first, before, differ;
  const int b = blockIdx.x, tid = threadIdx.x;
  const int q0 = a.cu[b], lq = a.cu[b + 1] - q0, level = a.level[b];
  if (tid == 0) { first = b; before = 0; }
  const int32_t* row = a.bt + (int64_t)b * a.bt_stride;
  const bool mine = level >= 0;
  const int cached = mine ? cached_keys(a, b) : 0;
  const int blocks = (cached + a.bs - 1) / a.bs;
  if (tid == 0) differ = blocks;
  __syncthreads();
  if (mine) {
    const int key = group_key(a, b), block = block_at(a, b, level);
    for (int o = tid; o < b; o += 256) {
      if (a.level[o] != level || group_key(a, o) != key || block_at(a, o, level) != block) continue;
      atomicMin(&first, o);
      atomicAdd(&before, a.cu[o + 1] - a.cu[o]);
    }
  }
  __syncthreads();
  const int32_t* lrow = a.bt + (int64_t)first * a.bt_stride;
  for (int i = tid; i < blocks; i += 256)
    if (row[i] != lrow[i]) { atomicMin(&differ, i); break; }
  __syncthreads();
  if (tid == 0) {
    a.lead[b] = mine ? first : -1;
    a.place[b] = before;
    a.common[b] = (int)min((int64_t)cached, (int64_t)differ * a.bs);
  }
  for (int i = tid; i < lq; i += 256)
    if (q0 + i >= 0 && q0 + i < a.tokens) a.tokreq[q0 + i] = make_int4(b, i, mine ? first : -1, before);
}

__device__ __forceinline__ int tiles_of(int keys) { return (keys + kKeys - 1) / kKeys; }

__device__ __forceinline__ int64_t block_sum(int64_t x, int64_t* lds) {
  const int tid = threadIdx.x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) x += __shfl_xor(x, d);
  __syncthreads();
  if ((tid & 63) == 0) lds[tid >> 6] = x;
  __syncthreads();
  x = 0;
  for (int w = 0; w < kShPlanT / 64; ++w) x += lds[w];
  return x;
}

// Exclusive sum over the threads, and the total.
__device__ __forceinline__ int64_t block_scan(int64_t x, int64_t& total, int64_t* lds) {
  const int tid = threadIdx.x, lane = tid & 63;
  int64_t s = x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t y = __shfl_up(s, d);
    if (lane >= d) s += y;
  }
  __syncthreads();
  if (lane == 63) lds[tid >> 6] = s;
  __syncthreads();
  int64_t before = 0;
  total = 0;
  for (int w = 0; w < kShPlanT / 64; ++w) {
    before += w < tid >> 6 ? lds[w] : 0;
    total += lds[w];
  }
  return before + s - x;
}

__global__ __launch_bounds__(kShPlanT) void shared_plan_kernel(ShPlanArgs a) {
  extern __shared__ int lds[];
  int* tok = lds;                            // per group (first request): tokens,
  int* keys = tok + a.batch;                 // shared keys,
  int* members = keys + a.batch;             // requests
  int* first_heavy = members + a.batch;      // per entity (2 batch): its first heavy unit
  int* first_light = first_heavy + 2 * a.batch;       // and light one (kLightRows) among those
  __shared__ int64_t scratch[kShPlanT / 64];
  __shared__ int bad;
  const int tid = threadIdx.x, B = a.batch;
  if (tid == 0) bad = a.cu[0] != 0 || a.cu[B] != a.tokens;
  for (int b = tid; b < B; b += kShPlanT) { tok[b] = 0; keys[b] = INT32_MAX; members[b] = 0; }
  __syncthreads();
  for (int b = tid; b < B; b += kShPlanT) {
    if (a.cu[b + 1] < a.cu[b]) bad = 1;
    const int l = a.lead[b];
    if (l < 0) continue;
    atomicAdd(&tok[l], a.cu[b + 1] - a.cu[b]);
    atomicMin(&keys[l], a.common[b]);
    atomicAdd(&members[l], 1);
  }
  __syncthreads();
  if (bad) {                                 // (uniform: read after the barrier)
    if (tid == 0) { a.hdr[0] = 0; a.hdr[1] = -1; }
    return;
  }
  for (int b = tid; b < B; b += kShPlanT) {
    // whole tiles, so that shared and own keys both begin at a tile
    const int s = members[b] > 1 ? keys[b] / kKeys * kKeys : 0;
    keys[b] = s >= kMinShare ? s : 0;
    if (keys[b] == 0) tok[b] = 0;
  }
  __syncthreads();
  // the work: tiles of keys per KV head, over all row tiles
  auto extent = [&](int e, int& rows, int& k0, int& k1) {
    if (e < B) {
      rows = tok[e] * a.group; k0 = 0; k1 = keys[e];
    } else {
      const int b = e - B, l = a.lead[b];
      rows = (a.cu[b + 1] - a.cu[b]) * a.group;
      k0 = l >= 0 ? keys[l] : 0;
      k1 = (int)min((int64_t)max(a.lk[b], 0), (int64_t)a.width * a.bs);
      k0 = min(k0, k1);
    }
  };
  int64_t work = 0;
  for (int e = tid; e < 2 * B; e += kShPlanT) {
    int rows, k0, k1;
    extent(e, rows, k0, k1);
    work += (int64_t)((rows + kUnitRows - 1) / kUnitRows) * tiles_of(k1 - k0);
  }
  work = block_sum(work, scratch) * a.hkv;
  const int per_cut = (int)max((int64_t)kMinCut, (work + kTargetGroups - 1) / kTargetGroups);
  // entities: units, partial rows and (groups) places in the token order
  int64_t heavy_at = 0, light_at = 0, part_at = 0, order_at = 0;
  for (int e0 = 0; e0 < 2 * B; e0 += kShPlanT) {
    const int e = e0 + tid;
    Entity x = {};
    int64_t heavies = 0, lights = 0, parts = 0;
    if (e < 2 * B) {
      extent(e, x.rows, x.k0, x.k1);
      // (rows without keys still have one cut, which gives zeros)
      x.cuts = max(1, (tiles_of(x.k1 - x.k0) + per_cut - 1) / per_cut);
      const int rest = x.rows % kUnitRows;
      heavies = (int64_t)(x.rows / kUnitRows + (rest > kLightRows)) * x.cuts * a.hkv;
      lights = rest > 0 && rest <= kLightRows ? (int64_t)x.cuts * a.hkv : 0;
      parts = (int64_t)x.rows * x.cuts * a.hkv;
      if (e >= B) {
        const int l = a.lead[e - B];
        if ((l < 0 || keys[l] == 0) && x.cuts == 1) { parts = 0; x.part_base = -1; }
        x.token_base = a.cu[e - B];
      }
    }
    int64_t total;
    const int64_t heavy = heavy_at + block_scan(heavies, total, scratch);
    heavy_at += total;
    const int64_t light = light_at + block_scan(lights, total, scratch);
    light_at += total;
    const int64_t part = part_at + block_scan(parts, total, scratch);
    part_at += total;
    const int64_t at = order_at + block_scan(e < B ? tok[e] : 0, total, scratch);
    order_at += total;
    if (e < 2 * B) {
      if (e < B) x.token_base = (int)at;
      if (x.part_base >= 0) x.part_base = (int)min(part, (int64_t)INT32_MAX);
      a.ent[e] = x;
      first_heavy[e] = (int)min(heavy, (int64_t)a.wg_cap);
      first_light[e] = (int)min(light, (int64_t)a.wg_cap);
    }
  }
  // (the workspace is sized for any step of these sizes; a plan that would not fit is
  // not used)
  if (heavy_at + light_at > a.wg_cap || part_at > a.part_cap) {
    if (tid == 0) { a.hdr[0] = 0; a.hdr[1] = -1; }
    return;
  }
  const int heavies = (int)heavy_at, count = heavies + (int)light_at;
  if (tid == 0) { a.hdr[0] = count; a.hdr[1] = 0; }
  __syncthreads();
  __threadfence_block();
  for (int b = tid; b < B; b += kShPlanT) {
    const int l = a.lead[b];
    if (l < 0 || keys[l] == 0) continue;
    const int at = a.ent[l].token_base + a.place[b], n = a.cu[b + 1] - a.cu[b];
    for (int i = 0; i < n; ++i)
      if (at + i < a.tokens) a.order[at + i] = a.cu[b] + i;
  }
  // the units' records, heavy and light ones in turns of kTurn, so that a compute unit
  // has one that waits for the matrix cores beside one that waits for memory
  for (int w = tid; w < count; w += kShPlanT) {
    const bool heavy = w < heavies;
    const int* first = heavy ? first_heavy : first_light;
    const int j = heavy ? w : w - heavies;   // its number among its kind
    int lo = 0, hi = 2 * B;                  // the last entity with first[lo] <= j
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (first[mid] <= j) lo = mid; else hi = mid;
    }
    const int e = lo;
    const Entity x = a.ent[e];
    const int slot = heavy ? j + min(count - heavies, j / kTurn * kTurn) : j + min(heavies, (j / kTurn + 1) * kTurn);
    const int rest = x.rows % kUnitRows, full = x.rows / kUnitRows;
    const int row_tiles = heavy ? full + (rest > kLightRows) : 1;
    // Units of one run of keys and KV head (they differ in the row tile) are eight
    // apart, so that they fall on one XCD and share its L2.
    const int i = j - first[e], pairs = x.cuts * a.hkv;
    const int block = i / (8 * row_tiles), in = i - block * 8 * row_tiles, here = min(8, pairs - 8 * block);
    const int tile = heavy ? in / here : full;
    const int pair = 8 * block + in % here;
    const int h = pair % a.hkv, c = pair / a.hkv;
    const int rows = min(kUnitRows, x.rows - tile * kUnitRows);
    const int tiles = tiles_of(x.k1 - x.k0);
    const int t0 = (int)((int64_t)tiles * c / x.cuts), t1 = (int)((int64_t)tiles * (c + 1) / x.cuts);
    const int b = e < B ? e : e - B;
    int32_t* r = a.rec + (int64_t)slot * kRecord;
    r[0] = e < B ? 1 : 0;
    r[1] = b;
    r[2] = tile * kUnitRows;
    r[3] = rows;
    r[4] = x.token_base;
    r[5] = x.k0 + t0 * kKeys;
    r[6] = min(x.k1, x.k0 + t1 * kKeys);
    r[7] = h;
    r[8] = e < B ? INT32_MAX / 2 : a.lk[b] - (a.cu[b + 1] - a.cu[b]);
    // a tile's partial rows follow those of the tiles before it: (cut, KV head, row)
    r[9] = x.part_base < 0 ? -1 : x.part_base + (tile * kUnitRows * x.cuts + c * rows) * a.hkv;
    r[10] = r[11] = 0;
  }
}

// ------------------------------------------------------------------ attention

struct ShArgs {
  CacheArgs c;
  const uint16_t* q;
  int64_t q_ts, q_hs;
  const int32_t* bt;
  int64_t bt_stride;
  int32_t batch, tokens, width;
  const int32_t* hdr;
  const int32_t* rec;
  const int32_t* order;
  uint16_t* out;
  int64_t o_ts, o_hs;
  uint16_t* part_o;
  PartHead* part_head;
  int64_t part_cap;
  // for the join
  const Entity* ent;
  const int4* tokreq;
  int32_t hq, hkv;
};

struct Unit {
  bool shared;               // rows of a group, by the token order; all see all keys
  int b, row0, rows, token_base, k0, k1, h, ctx0, part;
};

__device__ __forceinline__ bool load_unit(const ShArgs& a, int w, Unit& u) {
  if (w >= a.hdr[0]) return false;
  const int32_t* r = a.rec + (int64_t)w * kRecord;
  u.shared = r[0] & 1;
  u.b = r[1]; u.row0 = r[2]; u.rows = r[3]; u.token_base = r[4];
  u.k0 = r[5]; u.k1 = r[6]; u.h = r[7]; u.ctx0 = r[8]; u.part = r[9];
  return u.b >= 0 && u.b < a.batch && u.rows > 0 && u.rows <= kUnitRows;
}

// Row r of a unit: its token and its token's index among the unit's.
__device__ __forceinline__ int token_of(const ShArgs& a, const Unit& u, int row, int& index) {
  index = row / a.c.group;
  const int t = u.token_base + index;
  const int tok = u.shared ? a.order[min(t, a.tokens - 1)] : t;
  return min(max(tok, 0), a.tokens - 1);
}

// Q operands of a 16-row MFMA tile: row n from qp (null: zeros).
template <int D>
__device__ __forceinline__ void load_q(const uint16_t* qp, int g, uint4 (&qf)[D / 32]) {
#pragma unroll
  for (int j = 0; j < D / 32; ++j) {
    qf[j] = make_uint4(0, 0, 0, 0);
    if (qp) qf[j] = reinterpret_cast<const uint4*>(qp)[4 * j + g];
  }
}

// Row `row` of the unit, with its token and head found again rather than held through
// the loop, which needs every register.
template <int D>
__device__ __forceinline__ void finish_row(const ShArgs& a, const Unit& u, int kvh, int row, float4_t (&o)[D / 16],
                                           float m, float l, int g) {
  int index;
  const int tok = token_of(a, u, u.row0 + min(row, u.rows - 1), index);
  const int head = kvh * a.c.group + (u.row0 + row) % a.c.group;
  const bool live = row < u.rows;
  if (u.part < 0) {              // the unit has all of the rows' keys
    if (live) write_out<D>(a.out + (int64_t)tok * a.o_ts + (int64_t)head * a.o_hs, o, l, g);
    return;
  }
  const int64_t prow = u.part + (int64_t)kvh * u.rows + row;
  write_part<D>(a.part_o, a.part_head, prow, o, m, l, live && prow < a.part_cap, g);
}

// A unit: K and V in tiles of 64 keys, staged once for the four waves in one of two
// LDS buffers:
//   S^T = K Q^T    K fragments from LDS, Q^T in registers for the whole unit;
//   O^T += V^T P^T V^T by transposing LDS reads, P from where the S^T accumulators
//                  leave it.
// WK waves share 32 rows (two 16-row MFMA tiles) and take a share of each tile's keys:
// 1 where the rows fill the waves, 4 where there are up to 32, whose shares are joined
// in LDS at the end.  One barrier a tile; the next tile's direct loads are issued behind
// QK^T and land during the softmax and PV.  K chunk c of key r sits at c ^ (r % RC), V
// chunk c at c ^ 2 (r % (RC / 2)) (RC = D / 8 chunks a row), which spreads the fragment
// reads over the banks.  8-bit caches: a thread's chunks wait in registers and become
// bf16 on their way to the same places, once per work-group.
//   128 requests on a prefix of 32K with 100 to 2048 keys of their own (64/8 heads, D 128):
// 228 us with the join.  The prefix's 1024 rows a KV head alone take 149 us, 0.92 PFLOP/s,
// bound by the softmax between the matrix products; the requests' own keys alone 137 us,
// 4.2 TB/s, bound by the two tiles in flight per work-group.  16 requests on a prefix of
// 4K: 21.6 us, of which a launch each for units and join and their first loads are most.
template <int D, bool F8, bool ONE_BLOCK, int WK>
__device__ __forceinline__ void unit_rows(const ShArgs& a, const Unit& u, uint16_t* k0b, uint16_t* k1b,
                                          uint16_t* v0b, uint16_t* v1b, int* odd_tile, float2 (*share)[16 * kRt]) {
  constexpr int KJ = D / 32, DT = D / 16, RC = D / 8;
  constexpr int ST = kKeys / 16 / WK;        // 16-key sub-tiles of this wave, from s0 on
  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int kvh = u.h, G = a.c.group;
  const int rw = wid / WK, ws = wid % WK, s0 = ws * ST;
  const int row_elems = a.hkv * D;
  const int32_t* btrow = a.bt + (int64_t)u.b * a.bt_stride;
  const int kend = u.k1;
  const int t0 = u.k0 / kKeys, t1 = (u.k1 + kKeys - 1) / kKeys;

  int lim[kRt];
  uint4 qf[kRt][KJ];
  int wlo = 0x7fffffff, whi = -1;
#pragma unroll
  for (int rt = 0; rt < kRt; ++rt) {
    const int row = (rw * kRt + rt) * 16 + n;
    const bool live = row < u.rows;
    int index;
    const int tok = token_of(a, u, u.row0 + min(row, u.rows - 1), index);
    const int head = kvh * G + (u.row0 + row) % G;
    lim[rt] = live ? min(u.ctx0 + index, kend - 1) : -1;
    if (live) { wlo = min(wlo, lim[rt]); whi = max(whi, lim[rt]); }
    load_q<D>(live ? a.q + (int64_t)tok * a.q_ts + (int64_t)head * a.q_hs : nullptr, g, qf[rt]);
  }
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) {
    wlo = min(wlo, __shfl_xor(wlo, d));
    whi = max(whi, __shfl_xor(whi, d));
  }
  // (All lanes hold the same limits; told so, the compiler joins the masked and the
  // unmasked run of the loop below and spills up to 380 bytes a lane.)

  // loader: thread tid moves 16-byte chunk tid % RCL of keys kLdKeys i + tid / RCL
  constexpr int RCL = F8 ? D / 16 : RC;
  constexpr int kWaveKeys = 64 / RCL, kLdKeys = kShWaves * kWaveKeys, kLdRounds = kKeys / kLdKeys;
  static_assert(kLdKeys % 16 == 0 && kKeys % kLdKeys == 0, "loader rounds of whole 16-key swizzle groups");
  const int lkey = tid / RCL, lc = tid % RCL;
  const int64_t kvoff = (int64_t)kvh * D;
  int bid[kLdRounds];
  int tb = -64, vbid = 0;
  auto fetch_ids = [&](int t) {
    if (ONE_BLOCK) return;
#pragma unroll
    for (int i = 0; i < kLdRounds; ++i) bid[i] = btrow[min(t * kKeys + kLdKeys * i + lkey, kend - 1) / a.c.bs];
  };
  auto tile_bid = [&](int t) {               // lane l holds the block of tile tb + l
    if (t - tb >= 64) {
      tb = t;
      vbid = btrow[min((t + lane) * kKeys, kend - 1) / a.c.bs];
    }
    return __builtin_amdgcn_readlane(vbid, t - tb);
  };
  uint4 kr[F8 ? kLdRounds : 1], vr[F8 ? kLdRounds : 1];
  uint32_t ke[F8 ? kLdRounds : 1], ve[F8 ? kLdRounds : 1];
  auto load_key = [&](int i, int blk, int boff, uint16_t* kdst, uint16_t* vdst) {
    // (the slot in 32 bits: pools of 2^31 slots and more are refused)
    const int64_t e = (int64_t)(blk * a.c.bs + boff) * row_elems + kvoff;
    if constexpr (F8) {
      const int64_t se = (int64_t)blk * a.hkv + kvh;
      kr[i] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(a.c.kc) + e + 16 * lc);
      vr[i] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(a.c.vc) + e + 16 * lc);
      ke[i] = a.c.ks[se];
      ve[i] = a.c.vs[se];
    } else {
      const int rb = (kLdKeys * i + kWaveKeys * wid) * D;       // the wave's first row
      aia::lds_load16(a.c.kc + e + 8 * (lc ^ (lkey & (RC - 1))), kdst + rb);
      aia::lds_load16(a.c.vc + e + 8 * (lc ^ (2 * (lkey & (RC / 2 - 1)))), vdst + rb);
    }
  };
  auto load = [&](int t, auto tag) {
    constexpr int Bf = decltype(tag)::value;
    uint16_t* kdst = Bf ? k1b : k0b;
    uint16_t* vdst = Bf ? v1b : v0b;
    const int kb = t * kKeys;
    if (ONE_BLOCK) {
      const int blk = min(max(tile_bid(t), 0), a.c.nb - 1), boff = kb % a.c.bs, last = kend - 1 - kb;
#pragma unroll
      for (int i = 0; i < kLdRounds; ++i) load_key(i, blk, boff + min(kLdKeys * i + lkey, last), kdst, vdst);
    } else {
#pragma unroll
      for (int i = 0; i < kLdRounds; ++i) {
        const int p = min(kb + kLdKeys * i + lkey, kend - 1);
        load_key(i, min(max(bid[i], 0), a.c.nb - 1), p % a.c.bs, kdst, vdst);
      }
    }
  };
  auto store_fp8 = [&](auto tag) {
    constexpr int Bf = decltype(tag)::value;
    uint16_t* kdst = Bf ? k1b : k0b;
    uint16_t* vdst = Bf ? v1b : v0b;
#pragma unroll
    for (int i = 0; i < (F8 ? kLdRounds : 0); ++i) {
      const int r = (kLdKeys * i + lkey) * D;
      uint4 x[2];
      fp8_to_bf16(kr[i], ke[i], x);
#pragma unroll
      for (int e = 0; e < 2; ++e)
        *reinterpret_cast<u32x4_t*>(kdst + r + 8 * ((2 * lc + e) ^ (lkey & (RC - 1)))) = as_u4(x[e]);
      fp8_to_bf16(vr[i], ve[i], x);
#pragma unroll
      for (int e = 0; e < 2; ++e)
        *reinterpret_cast<u32x4_t*>(vdst + r + 8 * ((2 * lc + e) ^ (2 * (lkey & (RC / 2 - 1))))) = as_u4(x[e]);
    }
  };

  float4_t o[kRt][DT];
  float m[kRt], l[kRt];
#pragma unroll
  for (int rt = 0; rt < kRt; ++rt) {
    clear_row(o[rt]);
    m[rt] = -INFINITY;
    l[rt] = 0.f;
  }
  auto compute = [&](int t, auto tag, auto mask_tag, auto issue_next) {
    constexpr bool MASK = decltype(mask_tag)::value;
    constexpr int Bf = decltype(tag)::value;
    const int kbase = t * kKeys;
    if (MASK && kbase > whi) {               // no row of this wave sees these keys
      issue_next();
      return;
    }
    const uint16_t* kt = Bf ? k1b : k0b;
    const uint16_t* vt = Bf ? v1b : v0b;
    float4_t acc[kRt][ST];
    if (F8) __builtin_amdgcn_s_setprio(1);
    __builtin_amdgcn_sched_barrier(0);       // the block below is scheduled on its own
#pragma unroll
    for (int st = 0; st < ST; ++st) {
      uint4 kf[KJ];
#pragma unroll
      for (int j = 0; j < KJ; ++j)
        kf[j] = *reinterpret_cast<const uint4*>(kt + (16 * (s0 + st) + n) * D + 8 * ((4 * j + g) ^ (n & (RC - 1))));
#pragma unroll
      for (int rt = 0; rt < kRt; ++rt) {
        acc[rt][st] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < KJ; ++j) acc[rt][st] = qk_step(kf[j], qf[rt][j], acc[rt][st]);
      }
    }
    __builtin_amdgcn_sched_group_barrier(kSgDsRead, KJ * (ST < kPfQkAhead ? ST : kPfQkAhead), 0);
#pragma unroll
    for (int st = 0; st < ST; ++st) {
      __builtin_amdgcn_sched_group_barrier(kSgMfma, KJ * kRt, 0);
      if (st + kPfQkAhead < ST) __builtin_amdgcn_sched_group_barrier(kSgDsRead, KJ, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (F8) __builtin_amdgcn_s_setprio(0);
    issue_next();
    uint4 pb[kRt][(ST + 1) / 2];
#pragma unroll
    for (int rt = 0; rt < kRt; ++rt) {
      float x[ST][4];
      const int rel = lim[rt] - kbase - 16 * s0 - 4 * g;
      float top = -INFINITY;
#pragma unroll
      for (int st = 0; st < ST; ++st)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          x[st][v] = !MASK || 16 * st + v <= rel ? acc[rt][st][v] : -INFINITY;
          top = fmaxf(top, x[st][v]);
        }
      top = aia::group4_max(top) * a.c.scale_log2;
      // the maximum moves only when some row's grows by more than kLazyLog2 (weights
      // stay below 2^kLazyLog2), so most tiles rescale nothing
      const bool grow = __any(top > m[rt] + kLazyLog2);
      const float mnew = grow ? fmaxf(m[rt], top) : m[rt];
      const float sub = mnew == -INFINITY ? 0.f : mnew;
      float sum = 0.f;
#pragma unroll
      for (int st = 0; st < ST; ++st)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          x[st][v] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[st][v], a.c.scale_log2, -sub));
          sum += x[st][v];
        }
      if (grow) {
        const float alpha = __builtin_amdgcn_exp2f(m[rt] - sub);
        l[rt] = l[rt] * alpha + sum;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[rt][dt] *= alpha;
      } else {
        l[rt] += sum;
      }
      m[rt] = mnew;
#pragma unroll
      for (int p = 0; p < (ST + 1) / 2; ++p)
        if (ST == 1) pb[rt][p] = make_uint4(aia::pack_bf16x2(x[0][0], x[0][1]), aia::pack_bf16x2(x[0][2], x[0][3]), 0, 0);
        else pb[rt][p] = make_uint4(aia::pack_bf16x2(x[2 * p][0], x[2 * p][1]), aia::pack_bf16x2(x[2 * p][2], x[2 * p][3]),
                               aia::pack_bf16x2(x[(2 * p + 1) % ST][0], x[(2 * p + 1) % ST][1]),
                               aia::pack_bf16x2(x[(2 * p + 1) % ST][2], x[(2 * p + 1) % ST][3]));
    }
    __builtin_amdgcn_sched_barrier(0);
    if (MASK && *reinterpret_cast<volatile int*>(odd_tile + Bf) == t) {
      // a masked tile with a value that is not finite, which a weight of zero would not
      // take out: key by key, each row those that it sees
      for (int kk = 0; kk < 16 * ST; ++kk) {
        const int k = 16 * s0 + kk;
        const uint16_t* vs = vt + k * D + 4 * (g & 1);
        const int sw = 2 * (k & (RC / 2 - 1));
#pragma unroll
        for (int rt = 0; rt < kRt; ++rt) {
          uint32_t word = 0;
#pragma unroll
          for (int w = 0; w < ST * 2; ++w) {      // word w: keys 16 (w / 2) + 4 g + 2 (w % 2), + 1
            const uint4 q = pb[rt][w >> 2];
            const uint32_t y = (w & 3) == 0 ? q.x : (w & 3) == 1 ? q.y : (w & 3) == 2 ? q.z : q.w;
            word = w == 2 * (kk >> 4) + ((kk >> 1) & 1) ? y : word;
          }
          const float p = weight_of(word, n, k);
          if (kbase + k <= lim[rt])
            add_key(o[rt], p, [&](int dt) { return vs + 8 * ((2 * dt + (g >> 1)) ^ sw); });
        }
      }
      return;
    }
    if (F8) __builtin_amdgcn_s_setprio(1);
    const int vrow = 4 * g + (n >> 2);
    if constexpr (ST == 1) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const short4_t x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_short4_t*)(vt + (16 * s0 + vrow) * D + 16 * (dt ^ (vrow & (RC / 2 - 1))) + 4 * (n & 3)));
#pragma unroll
        for (int rt = 0; rt < kRt; ++rt)
          o[rt][dt] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(x0, as_s4(pb[rt][0].x, pb[rt][0].y), o[rt][dt], 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int f = 0; f < ST / 2 * DT; ++f) {
        const int pp = f / DT, dt = f % DT;
        const int vsw = 16 * (dt ^ (vrow & (RC / 2 - 1)));
        const short4_t x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_short4_t*)(vt + (16 * s0 + 32 * pp + vrow) * D + vsw + 4 * (n & 3)));
        const short4_t x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_short4_t*)(vt + (16 * s0 + 32 * pp + 16 + vrow) * D + vsw + 4 * (n & 3)));
        const bf16x8_t va = __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
        for (int rt = 0; rt < kRt; ++rt)
          o[rt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, as_b8(pb[rt][pp]), o[rt][dt], 0, 0, 0);
      }
      __builtin_amdgcn_sched_group_barrier(kSgDsRead, 2 * kPfPvAhead, 0);
#pragma unroll
      for (int f = 0; f < ST / 2 * DT; ++f) {
        __builtin_amdgcn_sched_group_barrier(kSgMfma, kRt, 0);
        if (f + kPfPvAhead < ST / 2 * DT) __builtin_amdgcn_sched_group_barrier(kSgDsRead, 2, 0);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    if (F8) __builtin_amdgcn_s_setprio(0);
  };

  // Tiles from t_care on are masked for some of the unit's rows: as such a tile's
  // bytes arrive, each thread looks through the V values that it loaded and names the
  // tile in odd_tile[its buffer] where one is not finite.  (The unit's first row has
  // its smallest limit.)
  const int t_care = max(t0, min(t1, (min(u.ctx0 + u.row0 / G, kend - 1) + 1) / kKeys));
  auto look = [&](int t, auto tag) {
    constexpr int Bf = decltype(tag)::value;
    if (t < t_care || t >= t1) return;
    bool odd;
    if constexpr (F8) {
      uint32_t x = 0;
#pragma unroll
      for (int i = 0; i < kLdRounds; ++i) x = nan_fp8(vr[i], x);
      odd = x & 0x80808080u;
    } else {
      asm volatile("" ::: "memory");         // after the wait for this wave's direct loads
      uint32_t x = 0;
      const uint16_t* vt = (Bf ? v1b : v0b) + (kWaveKeys * wid) * D + 8 * lane;
#pragma unroll
      for (int i = 0; i < kLdRounds; ++i)
        x = not_finite_bf16(*reinterpret_cast<const uint4*>(vt + kLdKeys * i * D), x);
      odd = x & 0x80008000u;
    }
    if (odd) odd_tile[Bf] = t;
  };

  if (t1 > t0) {
    using buf0 = std::integral_constant<int, 0>;
    using buf1 = std::integral_constant<int, 1>;
    fetch_ids(t0);
    load(t0, buf0{});
    fetch_ids(t0 + 1);
    if (tid < 2) odd_tile[tid] = -1;
    __syncthreads();
    if constexpr (F8) store_fp8(buf0{});
    else __builtin_amdgcn_s_waitcnt(kWaitVmcnt0);
    look(t0, buf0{});
    __syncthreads();
    // Tiles up to the wave's smallest limit need no mask; both runs together take every
    // tile, so all waves pass the same barriers.  A step's buffer is a compile-time
    // choice, so that the compiler sees that its reads and the next tile's loads touch
    // different memory.
    // (A wave without rows, or whose rows see none of the keys, skips them all.)
    const int t_um = whi < 0 ? t0 : max(t0, min(t1, (wlo + 1) / kKeys));
    auto step = [&](int t, auto tag, auto mask_tag) {
      constexpr int Bf = decltype(tag)::value;
      using other = std::integral_constant<int, Bf ^ 1>;
      compute(t, tag, mask_tag, [&]() {
        if (t + 1 < t1) {
          load(t + 1, other{});
          fetch_ids(t + 2);
        }
      });
      if constexpr (F8) {
        if (t + 1 < t1) store_fp8(other{});
      } else {
        __builtin_amdgcn_s_waitcnt(kWaitVmcnt0);
      }
      look(t + 1, other{});
      __syncthreads();
    };
    auto run = [&](int t, int end, auto mask_tag) {
      bool odd = ((t - t0) & 1) != 0;
#pragma clang loop unroll(disable)
      while (t < end) {
        if (!odd) {
          step(t, buf0{}, mask_tag);
          if (++t >= end) break;
        }
        step(t, buf1{}, mask_tag);
        ++t;
        odd = false;
      }
    };
    run(t0, t_um, std::false_type{});
    run(t_um, t1, std::true_type{});
  }
  if constexpr (WK > 1) {
    // The waves' shares of the keys, joined: wave ws takes row tile ws.  (The last tile's
    // barrier is behind every wave; a wave's O fills one of the four buffers.)
    static_assert(kRt * DT * 64 * 16 <= kKeys * D * 2 && kRt <= WK, "a buffer per wave, a wave per row tile");
    auto buffer = [&](int w) { return reinterpret_cast<float4_t*>(w == 0 ? k0b : w == 1 ? k1b : w == 2 ? v0b : v1b); };
#pragma unroll
    for (int rt = 0; rt < kRt; ++rt) {
      l[rt] = aia::group4_sum(l[rt]);
      if (g == 0) share[wid][16 * rt + n] = make_float2(m[rt], l[rt]);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) buffer(wid)[(rt * DT + dt) * 64 + lane] = o[rt][dt];
    }
    __syncthreads();
    if (ws >= kRt) return;
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < WK; ++w) top = fmaxf(top, share[rw * WK + w][16 * ws + n].x);
    float4_t y[DT];
    clear_row(y);
#pragma unroll
    for (int w = 0; w < WK; ++w) {
      const float2 ml = share[rw * WK + w][16 * ws + n];
      // (a share without keys has -inf and 0; one that saw NaN alone -inf and NaN)
      const float f = ml.x == -INFINITY && ml.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(ml.x - top);
      sum += f * ml.y;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) y[dt] += buffer(rw * WK + w)[(ws * DT + dt) * 64 + lane] * f;
    }
    finish_row<D>(a, u, kvh, (rw * kRt + ws) * 16 + n, y, top, sum, g);
    return;
  }
#pragma unroll
  for (int rt = 0; rt < kRt; ++rt)
    finish_row<D>(a, u, kvh, (rw * kRt + rt) * 16 + n, o[rt], m[rt], aia::group4_sum(l[rt]), g);
}

template <int D, bool F8, bool ONE_BLOCK>
__global__ __launch_bounds__(kShThreads) __attribute__((amdgpu_waves_per_eu(2, 2)))
void shared_attn_kernel(ShArgs a) {
  __shared__ __attribute__((aligned(16))) uint16_t k0[kKeys * D];
  __shared__ __attribute__((aligned(16))) uint16_t k1[kKeys * D];
  __shared__ __attribute__((aligned(16))) uint16_t v0[kKeys * D];
  __shared__ __attribute__((aligned(16))) uint16_t v1[kKeys * D];
  __shared__ float2 share[kShWaves][16 * kRt];
  __shared__ int odd_tile[2];
  Unit u;
  if (!load_unit(a, blockIdx.x, u)) return;
  if (u.rows <= 32) unit_rows<D, F8, ONE_BLOCK, 4>(a, u, k0, k1, v0, v1, odd_tile, share);
  else if (u.rows <= 64) unit_rows<D, F8, ONE_BLOCK, 2>(a, u, k0, k1, v0, v1, odd_tile, share);
  else unit_rows<D, F8, ONE_BLOCK, 1>(a, u, k0, k1, v0, v1, odd_tile, share);
}

// ------------------------------------------------------------------ join

// Row r's parts of an entity: the first one's index, their distance and number.
__device__ __forceinline__ void parts_of(const Entity& x, int r, int kvh, int hkv, int64_t& at,
                                         int64_t& step, int& count) {
  const int tile = r / kUnitRows;
  const int rows = min(kUnitRows, x.rows - tile * kUnitRows);
  count = x.cuts;
  step = (int64_t)hkv * rows;
  at = x.part_base + (int64_t)tile * kUnitRows * x.cuts * hkv + (int64_t)kvh * rows + (r - tile * kUnitRows);
}

// W waves per row (token and query head).
template <int D, int W>
__global__ __launch_bounds__(256) void shared_join_kernel(ShArgs a) {
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t = blockIdx.x, head = W > 1 ? blockIdx.y : blockIdx.y * 4 + wid;
  if (head >= a.hq) return;
  uint16_t* op = a.out + (int64_t)t * a.o_ts + (int64_t)head * a.o_hs;
  const int4 tk = a.tokreq[t];
  if (a.hdr[1] != 0) {                       // the lengths do not describe the step
    const int i = 8 * (threadIdx.x & 63);
    if (i < D) {
      *reinterpret_cast<uint2*>(op + i) = make_uint2(0x7fc07fc0u, 0x7fc07fc0u);
      *reinterpret_cast<uint2*>(op + i + 4) = make_uint2(0x7fc07fc0u, 0x7fc07fc0u);
    }
    return;
  }
  const int b = tk.x;
  if (b < 0 || b >= a.batch) return;
  const int kvh = head / a.c.group, hh = head - kvh * a.c.group;
  const Entity own = a.ent[a.batch + b];
  Entity sh = {};
  if (tk.z >= 0) sh = a.ent[tk.z];
  if (own.part_base < 0) return;
  int64_t at0, at1 = 0, step0, step1 = 0;
  int n0, n1 = 0;
  parts_of(own, tk.y * a.c.group + hh, kvh, a.hkv, at0, step0, n0);
  if (sh.rows > 0) parts_of(sh, (tk.w + tk.y) * a.c.group + hh, kvh, a.hkv, at1, step1, n1);
  join_row<D, W>(a.part_o, a.part_head, n0 + n1, [&](int i) { return i < n0 ? at0 + i * step0 : at1 + (i - n0) * step1; }, op);
}

int sh_check(const char* what, int32_t batch, int32_t tokens, int32_t hq, int32_t hkv, int32_t d, int32_t bs,
             int32_t width) {
  using namespace aia;
  if (batch < 0 || tokens < 0 || hq <= 0 || hkv <= 0 || bs <= 0 || width <= 0 || hq % hkv)
    return fail(AIA_ERR_INVALID, "%s: bad sizes (batch %d, tokens %d, heads %d / %d, block %d, table width %d)",
                what, batch, tokens, hq, hkv, bs, width);
  if (d != 128 && d != 64) return fail(AIA_ERR_UNSUPPORTED, "%s: head_dim %d (128 or 64)", what, d);
  if (batch > kMaxShared) return fail(AIA_ERR_UNSUPPORTED, "%s: %d requests (at most %d)", what, batch, kMaxShared);
  if ((int64_t)bs * width > INT32_MAX - 128 * kKeys)
    return fail(AIA_ERR_UNSUPPORTED, "%s: contexts of 2^31 tokens and more", what);
  // partial rows (part_cap of them at most) are numbered in 32 bits
  if (2ll * tokens * hq + (int64_t)kTargetGroups * kUnitRows > INT32_MAX)
    return fail(AIA_ERR_UNSUPPORTED, "%s: %d tokens of %d heads in one step", what, tokens, hq);
  return AIA_OK;
}

int sh_step(const char* what, int32_t batch, int32_t tokens, int32_t hq, int32_t hkv, int32_t d, int32_t bs,
            int32_t width, const void* ws, int64_t ws_bytes, ShLayout& L) {
  using namespace aia;
  if (int rc = sh_check(what, batch, tokens, hq, hkv, d, bs, width)) return rc;
  if (!ws || ((uintptr_t)ws & 255u)) return fail(AIA_ERR_INVALID, "%s: workspace must be 256-byte aligned", what);
  L = sh_layout(batch, tokens, hq, hkv, d);
  if (ws_bytes < L.total)
    return fail(AIA_ERR_CAPACITY, "%s: workspace of %lld bytes, %lld needed", what, (long long)ws_bytes, (long long)L.total);
  return AIA_OK;
}

}  // namespace

extern "C" int aia_shared_workspace_bytes(int32_t batch, int32_t num_tokens, int32_t num_q_heads,
                                          int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                                          int32_t table_width, int64_t* bytes) {
  using namespace aia;
  if (!bytes) return fail(AIA_ERR_INVALID, "aia_shared_workspace_bytes: null pointer argument");
  if (int rc = sh_check("aia_shared_workspace_bytes", batch, num_tokens, num_q_heads, num_kv_heads, head_dim,
                        block_size, table_width))
    return rc;
  *bytes = sh_layout(batch, num_tokens, num_q_heads, num_kv_heads, head_dim).total;
  return AIA_OK;
}

extern "C" int aia_shared_plan(const int32_t* cu_seqlens_q, const int32_t* seqlens_kv, const int32_t* group_ids,
                               const int32_t* block_table, int32_t block_table_stride, int32_t table_width,
                               int32_t block_size, int32_t batch, int32_t num_tokens, int32_t num_q_heads,
                               int32_t num_kv_heads, int32_t head_dim, void* workspace, int64_t workspace_bytes,
                               void* stream) {
  using namespace aia;
  ShLayout L;
  if (int rc = sh_step("aia_shared_plan", batch, num_tokens, num_q_heads, num_kv_heads, head_dim, block_size,
                       table_width, workspace, workspace_bytes, L))
    return rc;
  if (!cu_seqlens_q || (batch > 0 && (!seqlens_kv || !block_table)))
    return fail(AIA_ERR_INVALID, "aia_shared_plan: null pointer argument");
  if (batch > 1 && block_table_stride < table_width)
    return fail(AIA_ERR_INVALID, "aia_shared_plan: table rows overlap");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  ShPlanArgs a;
  a.cu = cu_seqlens_q; a.lk = seqlens_kv; a.bt = block_table; a.gid = group_ids; a.bt_stride = block_table_stride;
  a.batch = batch; a.tokens = num_tokens; a.bs = block_size; a.width = table_width;
  a.group = num_q_heads / num_kv_heads; a.hq = num_q_heads; a.hkv = num_kv_heads;
  a.wg_cap = L.wg_cap; a.part_cap = L.part_cap;
  auto ints = [&](int64_t at) { return reinterpret_cast<int32_t*>(ws + at); };
  a.hdr = ints(L.hdr); a.lead = ints(L.lead); a.common = ints(L.common); a.place = ints(L.place);
  a.tokreq = reinterpret_cast<int4*>(ws + L.tokreq); a.order = ints(L.order); a.rec = ints(L.rec);
  a.ent = reinterpret_cast<Entity*>(ws + L.ent); a.level = ints(L.level);
  hipStream_t s = (hipStream_t)stream;
  if (batch > 0) {
    shared_level_kernel<<<(unsigned)batch, 256, 0, s>>>(a);
    if (int rc = check_hip(hipGetLastError(), "aia_shared_plan launch")) return rc;
    shared_find_kernel<<<(unsigned)batch, 256, 0, s>>>(a);
    if (int rc = check_hip(hipGetLastError(), "aia_shared_plan launch")) return rc;
  }
  const size_t lds = (size_t)(7 * batch) * sizeof(int);
  if (lds > 48 * 1024) {
    if (int rc = check_hip(hipFuncSetAttribute(reinterpret_cast<const void*>(shared_plan_kernel),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds),
                           "aia_shared_plan"))
      return rc;
  }
  shared_plan_kernel<<<1, kShPlanT, lds, s>>>(a);
  return check_hip(hipGetLastError(), "aia_shared_plan launch");
}

extern "C" int aia_paged_attention_shared(const void* query, int64_t q_token_stride, int64_t q_head_stride,
                                          const void* key_cache, const void* value_cache, const void* key_scale,
                                          const void* value_scale, int32_t num_blocks,
                                          const int32_t* cu_seqlens_q, const int32_t* block_table,
                                          int32_t block_table_stride, int32_t table_width, int32_t block_size,
                                          int32_t batch, int32_t num_tokens, int32_t num_q_heads,
                                          int32_t num_kv_heads, int32_t head_dim, float scale, void* out,
                                          int64_t out_token_stride, int64_t out_head_stride, void* workspace,
                                          int64_t workspace_bytes, void* stream) {
  using namespace aia;
  ShLayout L;
  if (int rc = sh_step("aia_paged_attention_shared", batch, num_tokens, num_q_heads, num_kv_heads, head_dim,
                       block_size, table_width, workspace, workspace_bytes, L))
    return rc;
  if (!(scale > 0.f) || !(scale < 1e30f))
    return fail(AIA_ERR_INVALID, "aia_paged_attention_shared: scale must be positive");
  if (num_tokens == 0) return AIA_OK;
  if (!query || !key_cache || !value_cache || !cu_seqlens_q || !block_table || !out || num_blocks <= 0)
    return fail(AIA_ERR_INVALID, "aia_paged_attention_shared: null pointer argument or no blocks");
  if ((key_scale == nullptr) != (value_scale == nullptr))
    return fail(AIA_ERR_INVALID, "aia_paged_attention_shared: key_scale and value_scale go together");
  if ((int64_t)num_blocks * block_size > INT32_MAX)
    return fail(AIA_ERR_INVALID, "aia_paged_attention_shared: caches of 2^31 slots and more");
  auto aligned = [](const void* p) { return ((uintptr_t)p & 15u) == 0; };
  if (!aligned(query) || !aligned(key_cache) || !aligned(value_cache) || q_token_stride % 8 || q_head_stride % 8 ||
      ((uintptr_t)out & 7u) || out_token_stride % 4 || out_head_stride % 4)
    return fail(AIA_ERR_INVALID, "aia_paged_attention_shared: query and caches must be 16-byte aligned with strides a "
                "multiple of 8, out 8-byte aligned with strides a multiple of 4");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  auto ints = [&](int64_t at) { return reinterpret_cast<int32_t*>(ws + at); };
  ShArgs a;
  a.c.kc = static_cast<const uint16_t*>(key_cache); a.c.vc = static_cast<const uint16_t*>(value_cache);
  a.c.ks = static_cast<const uint8_t*>(key_scale); a.c.vs = static_cast<const uint8_t*>(value_scale);
  a.c.group = num_q_heads / num_kv_heads; a.c.bs = block_size; a.c.nb = num_blocks;
  a.c.scale_log2 = scale * kLog2e;
  a.q = static_cast<const uint16_t*>(query); a.q_ts = q_token_stride; a.q_hs = q_head_stride;
  a.bt = block_table; a.bt_stride = block_table_stride; a.batch = batch; a.tokens = num_tokens; a.width = table_width;
  a.hdr = ints(L.hdr); a.rec = ints(L.rec); a.order = ints(L.order);
  a.out = static_cast<uint16_t*>(out); a.o_ts = out_token_stride; a.o_hs = out_head_stride;
  a.part_o = reinterpret_cast<uint16_t*>(ws + L.part_o); a.part_head = reinterpret_cast<PartHead*>(ws + L.part_head);
  a.part_cap = L.part_cap;
  a.ent = reinterpret_cast<const Entity*>(ws + L.ent);
  a.tokreq = reinterpret_cast<const int4*>(ws + L.tokreq); a.hq = num_q_heads; a.hkv = num_kv_heads;
  const bool one = block_size % kKeys == 0;
  auto pick = [&](auto d) {
    constexpr int D = decltype(d)::value;
    return key_scale ? (one ? shared_attn_kernel<D, true, true> : shared_attn_kernel<D, true, false>)
                     : (one ? shared_attn_kernel<D, false, true> : shared_attn_kernel<D, false, false>);
  };
  auto* kernel = head_dim == 128 ? pick(std::integral_constant<int, 128>{}) : pick(std::integral_constant<int, 64>{});
  hipStream_t s = (hipStream_t)stream;
  kernel<<<(unsigned)L.wg_cap, kShThreads, 0, s>>>(a);
  if (int rc = check_hip(hipGetLastError(), "aia_paged_attention_shared launch")) return rc;
  const bool few = (int64_t)num_tokens * num_q_heads < kFewRows;
  auto* join = head_dim == 128 ? (few ? shared_join_kernel<128, 4> : shared_join_kernel<128, 1>)
                               : (few ? shared_join_kernel<64, 4> : shared_join_kernel<64, 1>);
  join<<<dim3((unsigned)num_tokens, (unsigned)(few ? num_q_heads : (num_q_heads + 3) / 4)), 256, 0, s>>>(a);
  return check_hip(hipGetLastError(), "aia_paged_attention_shared: join launch");
}
