// Sparse attention over cache blocks that a cheap score selects for each query
// token and KV head: the step's plan, 8-bit bounds of each block's keys, the
// selection, and the attention over what was selected.
//
// Bounds.  For a block and KV head, hi[d] and lo[d] are the largest and the smallest
// k[d] of the keys that it holds, so q.k <= sum_d max(q[d] hi[d], q[d] lo[d])
// = sum_d q+[d] hi[d] + q-[d] nlo[d] with q+ = max(q, 0), q- = max(-q, 0), nlo = -lo.
// Both are kept as whole numbers times a power of two 2^e of their block and head,
// rounded up, e the least >= -100 with |k| <= 127 * 2^e: half the bytes of one bf16
// key per block.  The query is rounded to whole numbers -127 .. 127 times a power of
// two of its token and KV head, so a score, summed over the group's heads, is a
// whole number times two powers of two: the same bits in any order of summation, and
// a selection that does not depend on how the work is cut.
#include <algorithm>

#include "wave_attention.h"

namespace {

constexpr int kMinExp = -100;
constexpr int kSparseThreads = 256;
constexpr int kMaxSelected = 1024;
constexpr int kHdrInts = 64;
constexpr int64_t kScoreFloats = 1ll << 26;   // scores held at once
constexpr int64_t kPartRows = 1ll << 20;      // and partial rows

// How the attention of a step is cut.  Few tokens: `parts` work-groups share a (token,
// KV head)'s selected keys, about four per compute unit in all, each of 256 keys or
// more.  Many tokens of a request: their selections overlap in a context that no L2
// holds, so the context (as long as the longest that a token sees, which the plan
// knows) is cut into `parts` equal ranges, a multiple of the eight XCDs, so many that a
// range's K and V fit an XCD's L2 in a context as long as the table, and all tokens and
// KV heads take a range there together.  (All KV heads: the rows of one of four lie in a
// quarter of the L2's channels.)  512 tokens behind 32K, 28/4 heads of 128, 32 of 513
// blocks of 64 each, chosen by chance: 180 us in 16 ranges, 186 in 8, 199 in 24, 226 in
// 32, 345 without: a wave's start, four dependent round trips, costs as much as the
// ranges' L2 hits save.  (Later steps took the 16 to 154.)
//   Ranges against parts, same heads and blocks, us: 32 tokens at 32K 28 and 29, 64 tokens
// 39 and 37, 128 tokens 55 and 54, 256 tokens 86 and 117; at 16K two requests of 64 tokens
// 53 and 48, eight of 16 80 and 72.
//   There are 64 ranges at most: those of 131K tokens of 8 heads of 128 are 8.4 MB.  And the
// table's width is what the host knows: in one much wider than the contexts ranges are
// short and launches many.  512 tokens of 2K, 32/8 heads, 32 blocks of 16: 99 us in a table
// of 128 columns, 370 in one of 8,192.
struct SparseCut {
  int32_t parts, tokens;     // tokens per launch
  bool ranges;
};
constexpr int64_t kRangeBytes = 9ll << 19;    // 4.5 MB: a little over an XCD's L2
constexpr int kRangeBlocks = 256, kMaxRanges = 64;           // blocks of a range at most
SparseCut sparse_cut(int32_t batch, int32_t tokens, int32_t hkv, int32_t hblocks, int32_t d, int32_t bs,
                     int32_t width, int32_t selected) {
  SparseCut c{1, tokens, false};
  const int64_t items = std::max<int64_t>(1, (int64_t)tokens * hkv * hblocks);
  if (tokens >= 64 && tokens >= 16 * (int64_t)batch) {
    // (sized for bf16; 8-bit caches' ranges take half the bytes)
    const int64_t bytes = 4ll * d * bs * hkv * width;
    const int64_t ranges = std::min<int64_t>(kMaxRanges, (bytes + 8 * kRangeBytes - 1) / (8 * kRangeBytes) * 8);
    if (bytes > kRangeBytes && (width + ranges - 1) / ranges <= kRangeBlocks) {
      c.ranges = true;
      c.parts = (int32_t)ranges;
      c.tokens = (int32_t)std::min<int64_t>(tokens, std::max<int64_t>(64, kPartRows / ((int64_t)hkv * hblocks * ranges * kRows)));
      return c;
    }
  }
  const int64_t keys = (int64_t)std::min(selected, width) * bs;
  c.parts = (int32_t)std::max<int64_t>(1, std::min<int64_t>(1024 / items, keys / 256));
  return c;
}

struct SparseLayout {
  int64_t hdr, tok, touched, scores, part_o, part_head, total;
  int32_t touched_cap, score_tokens, hblocks;
  SparseCut cut;
};
SparseLayout sparse_layout(int32_t batch, int32_t tokens, int32_t hq, int32_t hkv, int32_t d, int32_t bs,
                           int32_t width, int32_t selected) {
  SparseLayout L;
  auto up = [](int64_t x) { return (x + 255) & ~255ll; };
  const int32_t group = hq / hkv;
  L.hblocks = (group + kRows - 1) / kRows;
  L.touched_cap = (int32_t)std::min<int64_t>(tokens, tokens / bs + 2ll * batch);
  L.score_tokens = (int32_t)std::max<int64_t>(1, std::min<int64_t>(tokens, kScoreFloats / ((int64_t)hkv * std::max(1, width))));
  L.cut = sparse_cut(batch, tokens, hkv, L.hblocks, d, bs, width, selected);
  L.hdr = 0;
  L.tok = up(kHdrInts * 4);
  L.touched = L.tok + up(16ll * tokens);
  L.scores = L.touched + up(16ll * L.touched_cap);
  L.part_o = L.scores + up(4ll * L.score_tokens * hkv * width);
  const int64_t rows = L.cut.parts > 1 ? (int64_t)L.cut.parts * L.cut.tokens * hkv * L.hblocks * kRows : 0;
  L.part_head = L.part_o + up(2 * rows * d);
  L.total = L.part_head + up((int64_t)sizeof(PartHead) * rows);
  return L;
}

// ------------------------------------------------------------------ plan

struct PlanArgs {
  const int32_t* cu;
  const int32_t* lk;
  const int32_t* bt;
  int64_t bt_stride;
  int32_t batch, tokens, bs, width;
  int32_t* hdr;              // {blocks written to by the step, most blocks that a token sees, status}
  int4* tok;                 // {request, -1 or kBadStep, position, visible blocks, 0}
  int4* touched;             // {block id, keys that it holds, 0, 0}
  int32_t touched_cap;
};

constexpr int kPlanT = 1024;
constexpr int kBadStep = -2;               // request of all tokens where the lengths describe more than the step

// Every work-group counts the blocks that each request's new tokens fall into (and
// those of the requests before it), then places its own kPlanT tokens.  Every block that is
// counted is written by the first of its tokens, so lengths whose tokens are not all the
// step's give no blocks at all and a status.
__global__ __launch_bounds__(kPlanT) void sparse_plan_kernel(PlanArgs a) {
  extern __shared__ int lds[];               // cu (batch + 1), first touched entry (batch)
  int* cu = lds;
  int* first = lds + a.batch + 1;
  __shared__ int wave_sum[kPlanT / 64], carry, most;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  if (tid == 0) { carry = 0; most = 0; }
  for (int b = tid; b <= a.batch; b += kPlanT) cu[b] = a.cu[b];
  __syncthreads();
  bool wrong = cu[0] != 0 || cu[a.batch] > a.tokens;
  for (int b = tid; b < a.batch; b += kPlanT) wrong |= cu[b + 1] < cu[b];
  const int t = blockIdx.x * kPlanT + tid;
  if (__syncthreads_or(wrong)) {
    if (blockIdx.x == 0 && tid == 0) { a.hdr[0] = 0; a.hdr[1] = 0; a.hdr[2] = -1; }
    if (t < a.tokens) a.tok[t] = make_int4(kBadStep, -1, 0, 0);
    return;
  }
  for (int b0 = 0; b0 < a.batch; b0 += kPlanT) {
    const int b = b0 + tid;
    int n = 0;
    if (b < a.batch) {
      const int lq = cu[b + 1] - cu[b], lk = a.lk[b];
      const int from = max(0, lk - lq);
      if (lq > 0 && lk > 0) {
        n = (lk - 1) / a.bs - from / a.bs + 1;
        atomicMax(&most, min((lk - 1) / a.bs + 1, a.width));
      }
    }
    int sum = n;                             // inclusive scan of the wave
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int x = __shfl_up(sum, d);
      if (lane >= d) sum += x;
    }
    if (lane == 63) wave_sum[wid] = sum;
    __syncthreads();
    int before = carry;
    for (int w = 0; w < wid; ++w) before += wave_sum[w];
    if (b < a.batch) first[b] = before + sum - n;
    __syncthreads();
    if (tid == kPlanT - 1) carry = before + sum;
    __syncthreads();
  }
  if (blockIdx.x == 0 && tid == 0) { a.hdr[0] = min(carry, a.touched_cap); a.hdr[1] = most; a.hdr[2] = 0; }
  if (t >= a.tokens) return;
  int lo = 0, hi = a.batch;                  // the last request that begins at or before t
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= t) lo = mid; else hi = mid;
  }
  const int b = lo;
  int4 r = make_int4(-1, -1, 0, 0);
  if (a.batch > 0 && t >= cu[b] && t < cu[b + 1]) {
    const int lk = a.lk[b], from = lk - (cu[b + 1] - cu[b]), pos = from + t - cu[b];
    r.x = b;
    r.y = pos;
    if (pos >= 0) {
      const int blk = pos / a.bs;
      r.z = min(blk + 1, a.width);
      const int at = first[b] + blk - max(0, from) / a.bs;
      if ((pos == max(0, from) || pos % a.bs == 0) && blk < a.width && at >= 0 && at < a.touched_cap)
        a.touched[at] = make_int4(a.bt[(int64_t)b * a.bt_stride + blk], min(a.bs, lk - blk * a.bs), 0, 0);
      else if ((pos == max(0, from) || pos % a.bs == 0) && at >= 0 && at < a.touched_cap)
        a.touched[at] = make_int4(-1, 0, 0, 0);     // (behind the table)
    }
  }
  a.tok[t] = r;
}

// ------------------------------------------------------------------ bounds

typedef int16_t short2_t __attribute__((ext_vector_type(2)));

struct SummaryArgs {
  const uint16_t* kc;
  const uint8_t* ks;
  int32_t hkv, bs, nb;
  const int32_t* hdr;
  const int4* touched;
  int8_t* bounds;            // (num_blocks, hkv, 2, D): hi, nlo
  uint8_t* scale;            // (num_blocks, hkv)
};

__device__ __forceinline__ int bound_of(float x, float f) {      // rounded up; a positive one is not lost
  const float y = __builtin_ceilf(x * f);
  return (int)(x > 0.f ? fmaxf(y, 1.f) : y);
}

// The least e >= -100 with amax <= 127 * 2^e, for a bf16 value's bits: 127 = 1.984375
// * 2^6, and bf16 has one significand above it.
__device__ __forceinline__ int bound_exp(uint32_t amax) {
  const int e = (int)(amax >> 7) - 127 - 6 + ((amax & 0x7fu) > 0x7eu ? 1 : 0);
  return max(amax < 0x80u ? kMinExp : e, kMinExp);
}

// WPB waves take a (block, KV head): 64 / (D / 8) rows a pass, a lane 8 dims of one.
// Blocks of 64 keys and more are cut over the work-group's four waves: a decode step
// has few blocks, and the rows of one are loaded at once.  Waiting bounds it (plan,
// touched block, keys), and instructions where there are many blocks, so values are
// compared two at a time as whole numbers; only a wave that meets one that is not finite
// goes over its rows again, one by one.  A decode step's 64 blocks of 64 keys, 8 heads:
// 4.4 us; a prompt step's 1,000 blocks of 16: 10.4 (5.8 and 13.9 one by one).
template <int D, bool F8, int WPB>
__global__ __launch_bounds__(kSparseThreads) void summarize_kernel(SummaryArgs a) {
  constexpr int CH = D / 8, RPW = 64 / CH, DEEP = 8;
  __shared__ float part[WPB > 1 ? 4 : 1][2][D];
  __shared__ uint32_t part_bad[WPB > 1 ? 4 : 1][CH];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int c = lane % CH, r = lane / CH;
  constexpr int HPW = 4 / WPB;               // heads of a work-group
  const int h = blockIdx.y * HPW + wid / WPB, sub = wid % WPB;
  if ((int)blockIdx.x >= a.hdr[0]) return;
  const int4 t = a.touched[blockIdx.x];
  if (t.x < 0 || t.x >= a.nb) return;
  const int held = min(max(t.y, 0), a.bs);
  const bool live = h < a.hkv;
  if (WPB == 1 && !live) return;
  const int64_t row = (int64_t)a.hkv * D;
  const int64_t at = (int64_t)t.x * a.bs * row + (int64_t)h * D + 8 * c;
  const float f8 = F8 && live ? __uint_as_float((uint32_t)a.ks[(int64_t)t.x * a.hkv + h] << 23) : 0.f;
  const int rows = __builtin_amdgcn_readfirstlane(live ? held : 0);
  // f of each row's 8 dims, some rows (the last one) more than once
  auto each = [&](auto f) {
    for (int j0 = __builtin_amdgcn_readfirstlane(sub) * RPW; j0 < rows; j0 += DEEP * WPB * RPW) {
      uint4 w[DEEP];
#pragma unroll
      for (int u = 0; u < DEEP; ++u) {
        if (j0 + u * WPB * RPW >= rows) continue;
        const int j = min(j0 + r + u * WPB * RPW, rows - 1);
        if constexpr (F8) {
          const uint2 x = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(a.kc) + at + j * row);
          const uint2 lo = fp8x4_to_bf16(x.x, f8), up = fp8x4_to_bf16(x.y, f8);
          w[u] = make_uint4(lo.x, lo.y, up.x, up.y);
        } else {
          w[u] = *reinterpret_cast<const uint4*>(a.kc + at + j * row);
        }
      }
#pragma unroll
      for (int u = 0; u < DEEP; ++u)
        if (j0 + u * WPB * RPW < rows) f(w[u]);
    }
  };
  // Two dims at a time, as whole numbers in the values' order: bits of negative values
  // turned but for the sign (which turns them back, too).
  auto turned = [](short2_t x) { return x ^ ((x >> 15) & (short2_t)(int16_t)0x7fff); };
  short2_t top[4], low[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) { top[i] = (short2_t)INT16_MIN; low[i] = (short2_t)INT16_MAX; }
  each([&](const uint4& w) {
    const uint32_t p[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const short2_t x = turned(__builtin_bit_cast(short2_t, p[i]));
      top[i] = __builtin_elementwise_max(top[i], x);
      low[i] = __builtin_elementwise_min(low[i], x);
    }
  });
  float hi[8], nlo[8];
  uint32_t bad = 0;                          // dims with a value that is not finite
  constexpr int16_t kMost = 0x7f7f;          // the largest finite value; the least is ~kMost
  bool odd = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) odd |= top[i][0] > kMost || top[i][1] > kMost || low[i][0] < ~kMost || low[i][1] < ~kMost;
  if (!__any(odd && rows > 0)) {
#pragma unroll
    for (int d = CH; d < 64; d <<= 1) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        top[i] = __builtin_elementwise_max(top[i], __builtin_bit_cast(short2_t, __shfl_xor(__builtin_bit_cast(int, top[i]), d)));
        low[i] = __builtin_elementwise_min(low[i], __builtin_bit_cast(short2_t, __shfl_xor(__builtin_bit_cast(int, low[i]), d)));
      }
    }
    const bool some = sub * RPW < rows;      // (a wave without rows knows nothing)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t x = __builtin_bit_cast(uint32_t, turned(top[i >> 1])), y = __builtin_bit_cast(uint32_t, turned(low[i >> 1]));
      hi[i] = some ? (i & 1 ? aia::bf16_hi(x) : aia::bf16_lo(x)) : -INFINITY;
      nlo[i] = some ? -(i & 1 ? aia::bf16_hi(y) : aia::bf16_lo(y)) : -INFINITY;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) hi[i] = nlo[i] = -INFINITY;
    each([&](const uint4& w) {
      const uint32_t p[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = i & 1 ? aia::bf16_hi(p[i >> 1]) : aia::bf16_lo(p[i >> 1]);
        const bool ok = __builtin_fabsf(x) < INFINITY;
        if (!ok) bad |= 1u << i;
        hi[i] = fmaxf(hi[i], ok ? x : -INFINITY);
        nlo[i] = fmaxf(nlo[i], ok ? -x : -INFINITY);
      }
    });
#pragma unroll
    for (int d = CH; d < 64; d <<= 1) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        hi[i] = fmaxf(hi[i], __shfl_xor(hi[i], d));
        nlo[i] = fmaxf(nlo[i], __shfl_xor(nlo[i], d));
      }
      bad |= (uint32_t)__shfl_xor((int)bad, d);
    }
  }
  if constexpr (WPB > 1) {
    if (r == 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) { part[wid][0][8 * c + i] = hi[i]; part[wid][1][8 * c + i] = nlo[i]; }
      part_bad[wid][c] = bad;
    }
    __syncthreads();
    if (sub != 0 || !live) return;
#pragma unroll
    for (int w = 1; w < WPB; ++w) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        hi[i] = fmaxf(hi[i], part[wid + w][0][8 * c + i]);
        nlo[i] = fmaxf(nlo[i], part[wid + w][1][8 * c + i]);
      }
      bad |= part_bad[wid + w][c];
    }
  }
  float most = 0.f;                          // (a dim without a finite value has -inf in both)
#pragma unroll
  for (int i = 0; i < 8; ++i) most = fmaxf(most, fmaxf(hi[i], nlo[i]));
#pragma unroll
  for (int d = 1; d < CH; d <<= 1) most = fmaxf(most, __shfl_xor(most, d));
  const int e = bound_exp(__float_as_uint(most) >> 16);
  const float f = __builtin_ldexpf(1.f, -e);
  if (r < 2) {
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int x = bad >> i & 1 ? 127 : bound_of(r ? nlo[i] : hi[i], f);
      w[i >> 2] |= (uint32_t)(x & 0xff) << (8 * (i & 3));
    }
    *reinterpret_cast<uint2*>(a.bounds + (((int64_t)t.x * a.hkv + h) * 2 + r) * D + 8 * c) = make_uint2(w[0], w[1]);
    if (lane == 0) a.scale[(int64_t)t.x * a.hkv + h] = (uint8_t)(e + 127);
  }
}

// ------------------------------------------------------------------ scores

typedef int int4v_t __attribute__((ext_vector_type(4)));

struct ScoreKernelArgs {
  const uint16_t* q;
  int64_t q_ts, q_hs;
  const int8_t* bounds;
  const uint8_t* scale;
  const int32_t* bt;
  int64_t bt_stride;
  const int4* tok;
  float* scores;             // (tokens of this launch, hkv, width)
  int32_t t0, t1, hkv, group, nb, width, chunk;        // tokens [t0, t1)
};

// A token's query heads of a KV head are added up before the products: with q+ and q- the
// positive and negative parts of the whole numbers, the sum over the heads of
// q+ . hi + q- . nlo is (sum q+) . hi + (sum q-) . nlo, in whole numbers without a
// difference.  The sums, up to 127 * 256, go as two bytes: s = 256 up + low with low in
// [-128, 127] and up <= 127.

// Numbers 2 i and 2 i + 1 of eight words in order, low or upper bytes, four a word.
__device__ __forceinline__ uint4 low_bytes(const uint32_t s[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_perm(s[2 * i + 1], s[2 * i], 0x06040200u);
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 up_bytes(const uint32_t s[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = __builtin_amdgcn_perm(s[2 * i + 1] + 0x00800080u, s[2 * i] + 0x00800080u, 0x07050301u);
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint32_t finite_max(const uint4& w, uint32_t most) {
  const uint32_t p[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = p[i] & 0x7fffu, up = (p[i] >> 16) & 0x7fffu;
    most = max(most, max(lo < 0x7f80u ? lo : 0u, up < 0x7f80u ? up : 0u));
  }
  return most;
}
// Largest |x| of 8 bf16, as their bits, packed in two halves; infinities and NaN count.
typedef uint16_t ushort2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ ushort2_t any_max(const uint4& w, ushort2_t most) {
  const uint32_t p[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    most = __builtin_elementwise_max(most, __builtin_bit_cast(ushort2_t, p[i] & 0x7fff7fffu));
  return most;
}
// Adds kWhole + the whole numbers of one sign (f: the factor with it) of 8 bf16: |x f| <=
// 127, and adding 1.5 * 2^23 rounds it to a whole number, to even, in the sum's low bits.
// ODD: values that are not finite count as zero.  (With a check, a rounding and a
// conversion for every value, 512 tokens take 23.1 us instead of 20.5.)
constexpr uint32_t kWhole = 0x4b400000u;
template <bool ODD>
__device__ __forceinline__ void add_whole(const uint4& w, float f, uint32_t s[8]) {
  const uint32_t p[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float x = i & 1 ? aia::bf16_hi(p[i >> 1]) : aia::bf16_lo(p[i >> 1]);
    if (ODD && !(__builtin_fabsf(x) < INFINITY)) x = 0.f;
    s[i] += (uint32_t)max((int)__float_as_uint(__builtin_fmaf(x, f, 12582912.f)), (int)kWhole);
  }
}
// The sums of 16 numbers, n of them each, in pairs.
__device__ __forceinline__ void pair_up(const uint32_t s[16], int n, uint32_t (&w)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = (s[2 * i] - n * kWhole) | (s[2 * i + 1] - n * kWhole) << 16;
}

// Sums over rows of CH lanes: lane c of a row gets the row's sum of x[c].  Each step
// exchanges half of the values with the lane across a bit of c.
template <int CTRL>
__device__ __forceinline__ int from_lane(int x) {
  return __builtin_amdgcn_update_dpp(0, x, CTRL, 0xf, 0xf, true);
}
template <int CTRL, int H>
__device__ __forceinline__ void fold(int* x, bool upper) {
#pragma unroll
  for (int i = 0; i < H; ++i) x[i] = (upper ? x[i + H] : x[i]) + from_lane<CTRL>(upper ? x[i] : x[i + H]);
}
template <int CH>
__device__ __forceinline__ int sum_of_own(int* x, int c) {
  if constexpr (CH == 16) fold<0x128, 8>(x, c & 8);        // rotate by 8 lanes
  fold<0x141, 4>(x, c & 4);                                // mirror eight
  fold<0x4e, 2>(x, c & 2);                                 // swap pairs
  fold<0xb1, 1>(x, c & 1);                                 // swap neighbours
  return x[0];
}

// Few tokens of a request: a work-group is a token, a KV head and `chunk` blocks.  A
// wave takes 64 blocks at a time, each load 1 KB of whole rows of bounds, lane (row, c)
// with bytes 16 c .. of [hi, nlo] against the same bytes of [sum q+, sum q-] on
// v_dot4_i32_i8.  8 tokens, 32/8 heads, 1875 to 4096 blocks: 45 MB of bounds in 13.2 us,
// 3.4 TB/s, the chain plan, table, bounds being a third of it.  (The matrix kernel below with
// one token a tile: 18; its loads take 64 bytes of a row at a time.)
template <int D>
__global__ __launch_bounds__(kSparseThreads) void score_token_kernel(ScoreKernelArgs a) {
  constexpr int CH = 2 * D / 16, RP = 64 / CH;             // lanes of a row, rows of a load
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & (CH - 1), r = lane / CH;
  const int t = a.t0 + blockIdx.x, kvh = blockIdx.y;
  const int4 tok = a.tok[t];
  const int c0 = blockIdx.z * a.chunk + 64 * wid, c1 = min(tok.z, (int)(blockIdx.z + 1) * a.chunk);
  if (tok.x < 0 || c0 >= c1) return;
  const int32_t* btrow = a.bt + (int64_t)tok.x * a.bt_stride;
  uint4 w[CH];
  int ebyte;
  const int own = RP * c + r;                // this lane's block of 64
  auto load = [&](int b0) {
    const int blk = b0 + own < c1 ? min(max(btrow[b0 + own], 0), a.nb - 1) : 0;
    ebyte = a.scale[(int64_t)blk * a.hkv + kvh];
#pragma unroll
    for (int i = 0; i < CH; ++i) {           // rows RP i .. RP i + RP - 1
      const int at = __shfl(blk, (lane & ~(CH - 1)) + i);
      w[i] = reinterpret_cast<const uint4*>(a.bounds + ((int64_t)at * a.hkv + kvh) * 2 * D)[c];
    }
  };
  load(c0);
  // the queries, while the bounds arrive: heads r, r + RP, .. of the group
  const uint16_t* qt = a.q + (int64_t)t * a.q_ts + (int64_t)kvh * a.group * a.q_hs + 16 * (c & (CH / 2 - 1));
  uint32_t amax = 0;
  for (int h = r; h < a.group; h += RP) {
    const uint4* qp = reinterpret_cast<const uint4*>(qt + (int64_t)h * a.q_hs);
    amax = finite_max(qp[1], finite_max(qp[0], amax));
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) amax = max(amax, (uint32_t)__shfl_xor((int)amax, d));
  const float f = __builtin_ldexpf(c < CH / 2 ? 1.f : -1.f, -bound_exp(amax));
  uint32_t sum[16] = {}, s[8];
  int heads = 0;
  for (int h = r; h < a.group; h += RP, ++heads) {
    const uint4* qp = reinterpret_cast<const uint4*>(qt + (int64_t)h * a.q_hs);
    add_whole<true>(qp[0], f, sum);
    add_whole<true>(qp[1], f, sum + 8);
  }
  pair_up(sum, heads, s);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
#pragma unroll
    for (int d = CH; d < 64; d <<= 1) s[i] += (uint32_t)__shfl_xor((int)s[i], d);
  }
  const uint4 low = low_bytes(s), up = up_bytes(s);
  float* out = a.scores + ((int64_t)(t - a.t0) * a.hkv + kvh) * a.width;
  for (int b0 = c0;;) {
    int x[CH];
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const uint32_t k[4] = {w[i].x, w[i].y, w[i].z, w[i].w}, l[4] = {low.x, low.y, low.z, low.w},
                     u[4] = {up.x, up.y, up.z, up.w};
      int ls = 0, us = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        ls = __builtin_amdgcn_sdot4((int)l[j], (int)k[j], ls, false);
        us = __builtin_amdgcn_sdot4((int)u[j], (int)k[j], us, false);
      }
      x[i] = ls + (us << 8);
    }
    const int sum = sum_of_own<CH>(x, c), e = ebyte - 127, blk = b0 + own;
    b0 += kSparseThreads;
    if (b0 < c1) load(b0);
    if (blk < c1) out[blk] = __builtin_ldexpf((float)sum, e);
    if (b0 >= c1) break;
  }
}

constexpr int kScoreTiles = 4, kTileTokens = 8 * kScoreTiles;

// Many tokens of a request: a work-group is `tiles` tiles of 8 tokens of a KV head, two
// rows each, low and upper bytes, against `chunk` blocks.
//   A wave holds 64 blocks' bounds in registers; while the first of them arrive, the
// queries become whole numbers in LDS, in MFMA order.  Then it goes over the tiles: S =
// Q B^T on v_mfma_i32_16x16x64_i8, lane (row or block n, group g) with bytes 64 j + 16 g ..
// of [sum q+ (D), sum q- (D)] and of [hi, nlo]; the four accumulators are tokens 2 g and
// 2 g + 1 against block n.  Tokens of several requests are taken one request at a time.
//   512 tokens, 28/4 heads, 513 blocks: 12 us, with the selection 19.4.  (Before the
// selection's last step 20.5, and 25.1 with one tile a work-group, 20.6 with two, 26.2 with
// eight.)  Waiting bounds it, and the instructions that turn the queries to whole numbers;
// a row per head instead of two per token took 28.0.
template <int D>
__global__ __launch_bounds__(kSparseThreads) void score_kernel(ScoreKernelArgs a) {
  constexpr int KS = 2 * D / 64;             // MFMA steps
  __shared__ uint4 qfrag[kScoreTiles * KS * 64];           // [tile][step][lane]
  __shared__ int2 info[kTileTokens];         // the tokens' requests and visible blocks
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int tb = a.t0 + blockIdx.x * kTileTokens;
  const int tokens = min(kTileTokens, a.t1 - tb);
  const int c0 = blockIdx.z * a.chunk;
  // (nothing to do where no token sees the chunk's blocks)
  int see = 0;
  if (lane < tokens) {
    const int4 x = a.tok[tb + lane];
    see = x.z;
    if (wid == 0) info[lane] = make_int2(x.x, x.z);
  }
  if (__ballot(see > c0) == 0) return;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) see = max(see, __shfl_xor(see, d));
  see = __builtin_amdgcn_readfirstlane(see);
  const int kvh = blockIdx.y, own = 64 * wid;
  // the bounds of 64 blocks from b0 on of a request's table row, up to c1
  int4v_t bf[4][KS];
  int eb[4];
  auto load_bounds = [&](int req, int b0, int c1) {
    const int32_t* btrow = a.bt + (int64_t)req * a.bt_stride;
    const int id = b0 + lane < c1 ? min(max(btrow[b0 + lane], 0), a.nb - 1) : 0;
    const int ebyte = a.scale[(int64_t)id * a.hkv + kvh];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int blk = __shfl(id, 16 * s + n);
      eb[s] = __shfl(ebyte, 16 * s + n) - 127;
      const uint4* bp = reinterpret_cast<const uint4*>(a.bounds + ((int64_t)blk * a.hkv + kvh) * 2 * D) + g;
#pragma unroll
      for (int j = 0; j < KS; ++j) bf[s][j] = __builtin_bit_cast(int4v_t, as_u4(bp[4 * j]));
    }
  };
  // The first ones arrive while the queries are prepared.
  const int first_req = __builtin_amdgcn_readfirstlane(a.tok[tb].x);
  const bool ahead = first_req >= 0 && c0 + own < see;
  if (ahead) load_bounds(first_req, c0 + own, min(see, c0 + a.chunk));
  // lane (token n / 2 of the tile, sign n % 2, g) adds up dims 64 j + 16 g .. + 15
  const int tn = n >> 1, sign = n & 1;
  for (int u = wid; 8 * u < tokens; u += kSparseThreads / 64) {
    const int ti = 8 * u + tn;
    const int heads = ti < tokens ? a.group : 0;
    const uint16_t* qt = a.q + (int64_t)(tb + ti) * a.q_ts + (int64_t)kvh * a.group * a.q_hs + 16 * g;
    // largest |q| of the token's heads (four heads' loads at a time; each sign takes half)
    auto largest = [&](auto most, auto of) {
      for (int h0 = 0; h0 < heads; h0 += 4) {
        uint4 w[4][D / 64];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
          for (int j = 0; j < D / 64; ++j)
            w[i][j] = reinterpret_cast<const uint4*>(qt + (int64_t)min(h0 + i, heads - 1) * a.q_hs + 64 * j)[sign];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
          for (int j = 0; j < D / 64; ++j) most = of(w[i][j], most);
        }
      }
      return most;
    };
    const ushort2_t both = largest(ushort2_t{0, 0}, [](const uint4& w, ushort2_t m) { return any_max(w, m); });
    uint32_t amax = max((uint32_t)both[0], (uint32_t)both[1]);
    const bool odd = __any(amax >= 0x7f80u);
    if (odd) amax = largest(0u, [](const uint4& w, uint32_t m) { return finite_max(w, m); });
    amax = max(amax, (uint32_t)__shfl_xor((int)amax, 1));
    amax = max(amax, (uint32_t)__shfl_xor((int)amax, 16));
    amax = max(amax, (uint32_t)__shfl_xor((int)amax, 32));
    const float f = __builtin_ldexpf(sign ? -1.f : 1.f, -bound_exp(amax));
    uint32_t sum[D / 64][16] = {};
    auto add_up = [&](auto tag) {
      for (int h0 = 0; h0 < heads; h0 += 2) {
        uint4 w[2][D / 64][2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int j = 0; j < D / 64; ++j) {
            const uint4* qp = reinterpret_cast<const uint4*>(qt + (int64_t)min(h0 + i, heads - 1) * a.q_hs + 64 * j);
            w[i][j][0] = qp[0];
            w[i][j][1] = qp[1];
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float fi = h0 + i < heads ? f : 0.f;
#pragma unroll
          for (int j = 0; j < D / 64; ++j) {
            add_whole<decltype(tag)::value>(w[i][j][0], fi, sum[j]);
            add_whole<decltype(tag)::value>(w[i][j][1], fi, sum[j] + 8);
          }
        }
      }
    };
    if (odd) add_up(std::true_type{});
    else add_up(std::false_type{});
    uint32_t s[D / 64][8];
#pragma unroll
    for (int j = 0; j < D / 64; ++j) pair_up(sum[j], (heads + 1) / 2 * 2, s[j]);
#pragma unroll
    for (int j = 0; j < D / 64; ++j) {
      uint4* to = qfrag + (u * KS + sign * (D / 64) + j) * 64 + 16 * g + 2 * tn;
      to[0] = low_bytes(s[j]);
      to[1] = up_bytes(s[j]);
    }
  }
  __syncthreads();
  for (int done = 0; done < tokens;) {
    const int from = done, req = __builtin_amdgcn_readfirstlane(info[from].x);
    // tokens [from, done) of one request (a work-group has at most 64)
    const int2 x = from + lane < tokens ? info[from + lane] : make_int2(-2, 0);
    const uint64_t other = __ballot(x.x != req);
    const int here = other ? __builtin_ctzll(other) : 64;
    int vis = lane < here ? x.y : 0;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) vis = max(vis, __shfl_xor(vis, d));
    done += here;
    const int c1 = min(__builtin_amdgcn_readfirstlane(vis), c0 + a.chunk);
    if (req < 0) continue;
    for (int b0 = c0 + own; b0 < c1; b0 += kSparseThreads) {
      if (from > 0 || b0 > c0 + own || !ahead) load_bounds(req, b0, c1);
      for (int m = from / 8; m * 8 < done; ++m) {
        int4v_t acc[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) acc[s] = int4v_t{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < KS; ++j) {
          const int4v_t qf = __builtin_bit_cast(int4v_t, as_u4(qfrag[(m * KS + j) * 64 + lane]));
#pragma unroll
          for (int s = 0; s < 4; ++s) acc[s] = __builtin_amdgcn_mfma_i32_16x16x64_i8(qf, bf[s][j], acc[s], 0, 0, 0);
        }
        const int t = 8 * m + 2 * g;
        float* out = a.scores + ((int64_t)(tb + t - a.t0) * a.hkv + kvh) * a.width + b0 + n;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          if (b0 + 16 * s + n >= c1) continue;
          if (t >= from && t < done) out[16 * s] = __builtin_ldexpf((float)(acc[s][0] + (acc[s][1] << 8)), eb[s]);
          if (t + 1 >= from && t + 1 < done)
            out[(int64_t)a.hkv * a.width + 16 * s] = __builtin_ldexpf((float)(acc[s][2] + (acc[s][3] << 8)), eb[s]);
        }
      }
    }
  }
}

// ------------------------------------------------------------------ selection

struct SelectArgs {
  const float* scores;
  const int4* tok;
  int32_t* out;
  int64_t out_ts, out_hs;
  int32_t t0, rows, hkv, width, selected, sink, local;         // rows (token, KV head) from t0 on
};

// A score's order as an unsigned key; 0xffffffff: blocks that are always kept.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x);
  return min(u & 0x80000000u ? ~u : u | 0x80000000u, 0xfffffffeu);
}
__device__ __forceinline__ uint32_t key_of(const SelectArgs& a, float score, int i, int n) {
  const uint32_t k = i < a.sink || i >= n - a.local ? 0xffffffffu : order_key(score);
  return i < n ? k : 0;
}

// A wave per row, for tables of up to 64 NK blocks: the key of the `selected`-th largest
// score bit by bit, from the highest bit in which the scores differ, counting by ballots,
// until a bound has exactly so many above it; then the blocks above it and the first of those at it, in order.  No
// barriers, no LDS.  2048 rows of 513 blocks: 7.9 us; a work-group per row that counts
// digits in LDS: 17.0.
template <int NK>
__global__ __launch_bounds__(256) void select_wave_kernel(SelectArgs a) {
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = blockIdx.x * 4 + wid;
  if (row >= a.rows) return;
  const int t = row / a.hkv, kvh = row - t * a.hkv;
  const int n = __builtin_amdgcn_readfirstlane(a.tok[a.t0 + t].z);
  int32_t* out = a.out + (int64_t)(a.t0 + t) * a.out_ts + (int64_t)kvh * a.out_hs;
  if (n <= a.selected) {
    for (int i = lane; i < a.selected; i += 64) out[i] = i < n ? i : -1;
    return;
  }
  const float* sc = a.scores + (int64_t)row * a.width;
  float x[NK];                               // (all loads in flight: none under a condition)
#pragma unroll
  for (int j = 0; j < NK; ++j) x[j] = sc[min(64 * j + lane, n - 1)];
  uint32_t k[NK];
#pragma unroll
  for (int j = 0; j < NK; ++j) k[j] = key_of(a, x[j], 64 * j + lane, n);
  // (keys behind the row's end are 0, below every bound that is tried)
  uint32_t p = 0xfffffffeu;                  // (all that is taken are blocks that always are)
  int top = -1;
  if (a.selected > a.sink + a.local) {
    uint32_t most = 0, least = 0xfffffffeu;
#pragma unroll
    for (int j = 0; j < NK; ++j) {
      if (k[j] < 0xffffffffu) most = max(most, k[j]);
      if (64 * j + lane < n) least = min(least, k[j]);
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      most = max(most, (uint32_t)__shfl_xor((int)most, d));
      least = min(least, (uint32_t)__shfl_xor((int)least, d));
    }
    most = (uint32_t)__builtin_amdgcn_readfirstlane((int)most);
    least = (uint32_t)__builtin_amdgcn_readfirstlane((int)least);
    top = most > least ? 31 - __builtin_clz(most ^ least) : -1;
    p = top < 0 ? most : most >> top >> 1 << top << 1;     // the bits in common
  }
#pragma unroll 1
  for (int bit = top; bit >= 0; --bit) {
    const uint32_t bound = p | 1u << bit;
    int count = 0;
#pragma unroll
    for (int j = 0; j < NK; ++j) count += __popcll(__ballot(k[j] >= bound));
    if (count >= a.selected) p = bound;
    if (count == a.selected) break;
  }
  int above = 0;
#pragma unroll
  for (int j = 0; j < NK; ++j) above += __popcll(__ballot(k[j] > p));
  const int need = a.selected - above;       // of the blocks at the bound
  const uint64_t below = (1ull << lane) - 1;
  int at = 0, tied = 0;
#pragma unroll
  for (int j = 0; j < NK; ++j) {
    const bool up = k[j] > p, eq = k[j] == p && 64 * j + lane < n;
    const uint64_t mu = __ballot(up), me = __ballot(eq);
    const int ub = at + __popcll(mu & below), eb = tied + __popcll(me & below);
    if (up || (eq && eb < need)) out[ub + min(eb, need)] = 64 * j + lane;
    at += __popcll(mu);
    tied += __popcll(me);
  }
}

constexpr int kSelThreads = 512, kSelWaves = kSelThreads / 64;
constexpr int kDigits = 2048;

// A work-group per row, for longer tables: the same key by up to 11 bits at a time of what
// it is above the row's least one, counted in LDS.  (Without the least taken off, the
// first digit is mostly the exponent: one pass more and counters that many lanes hit at
// once, 10.5 us for 64 rows of 1875 to 4096 blocks; 7.5 so, of which waiting for the scores
// and the launch are most.)  A wave has a run of the row's blocks,
// up to 64 NK of them in registers (NK 0: any number, read again in every pass).
template <int NK>
__global__ __launch_bounds__(kSelThreads) void select_kernel(SelectArgs a) {
  __shared__ int hist[kDigits];
  __shared__ int wave_a[kSelWaves], wave_b[kSelWaves], found[3];
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int t = blockIdx.x / a.hkv, kvh = blockIdx.x - t * a.hkv;
  const int n = __builtin_amdgcn_readfirstlane(a.tok[a.t0 + t].z);
  int32_t* out = a.out + (int64_t)(a.t0 + t) * a.out_ts + (int64_t)kvh * a.out_hs;
  if (n <= a.selected) {
    for (int i = tid; i < a.selected; i += kSelThreads) out[i] = i < n ? i : -1;
    return;
  }
  const float* sc = a.scores + (int64_t)blockIdx.x * a.width;
  const int rounds = (n + kSelThreads - 1) / kSelThreads, first = wid * 64 * rounds + lane;
  uint32_t held[NK > 0 ? NK : 1];
  if constexpr (NK > 0) {                    // (all loads in flight: none under a condition)
    float x[NK];
#pragma unroll
    for (int j = 0; j < NK; ++j) x[j] = sc[min(first + 64 * min(j, rounds - 1), n - 1)];
#pragma unroll
    for (int j = 0; j < NK; ++j) held[j] = key_of(a, x[j], first + 64 * j, n);
  }
  auto each = [&](auto f) {
    if constexpr (NK > 0) {
#pragma unroll
      for (int j = 0; j < NK; ++j)
        if (j < rounds) f(first + 64 * j, held[j]);
    } else {
      for (int j = 0; j < rounds; ++j) f(first + 64 * j, key_of(a, sc[min(first + 64 * j, n - 1)], first + 64 * j, n));
    }
  };
  for (int i = tid; i < kDigits; i += kSelThreads) hist[i] = 0;
  uint32_t most = 0, least = 0xfffffffeu;
  each([&](int i, uint32_t k) {
    if (k < 0xffffffffu) most = max(most, k);
    if (i < n) least = min(least, k);
  });
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    most = max(most, (uint32_t)__shfl_xor((int)most, d));
    least = min(least, (uint32_t)__shfl_xor((int)least, d));
  }
  if (lane == 0) { wave_a[wid] = (int)most; wave_b[wid] = (int)least; }
  __syncthreads();
  for (int w = 0; w < kSelWaves; ++w) {
    most = max(most, (uint32_t)wave_a[w]);
    least = min(least, (uint32_t)wave_b[w]);
  }
  __syncthreads();
  // The always kept blocks are counted apart: `need` of the others are left to take.
  int need = a.selected - a.sink - a.local;
  uint32_t prefix = need > 0 ? 0u : 0xffffffffu;           // the digits found so far
  int shift = 0;
  int left = need > 0 && most > least ? 32 - __builtin_clz(most - least) : 0;
#pragma unroll 1
  for (bool all = true; left > 0; all = false) {
    const int bits = min(left, 11);
    shift = left - bits;
    each([&](int i, uint32_t k) {
      if (i < n && k < 0xffffffffu && (all || (k - least) >> left == prefix))
        atomicAdd(&hist[(k - least) >> shift & ((1 << bits) - 1)], 1);
    });
    __syncthreads();
    // digits from the largest down: thread tid has kDigits / kSelThreads of them
    constexpr int PER = kDigits / kSelThreads;
    const int top = kDigits - 1 - PER * tid;
    int c[PER], sum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      c[i] = hist[top - i];
      hist[top - i] = 0;
      sum += c[i];
    }
    int upto = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int x = __shfl_up(upto, d);
      if (lane >= d) upto += x;
    }
    if (lane == 63) wave_a[wid] = upto;
    __syncthreads();
    for (int w = 0; w < wid; ++w) upto += wave_a[w];
    int above = upto - sum;
    if (above < need && upto >= need) {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        if (above < need && above + c[i] >= need) { found[0] = top - i; found[1] = need - above; found[2] = c[i]; }
        above += c[i];
      }
    }
    __syncthreads();
    prefix = prefix << bits | (uint32_t)found[0];
    need = found[1];
    left = found[2] == need ? 0 : shift;     // (all of the digit's blocks are taken)
  }
  // the always kept ones, the blocks above the prefix, and the first `need` of those of it
  auto upper = [&](int i, uint32_t k) { return i < n && (k == 0xffffffffu || (k - least) >> shift > prefix); };
  auto equal = [&](int i, uint32_t k) { return i < n && k != 0xffffffffu && (k - least) >> shift == prefix; };
  int more = 0, ties = 0;
  each([&](int i, uint32_t k) {
    more += __popcll(__ballot(upper(i, k)));
    ties += __popcll(__ballot(equal(i, k)));
  });
  __syncthreads();
  if (lane == 0) { wave_a[wid] = more; wave_b[wid] = ties; }
  __syncthreads();
  int at = 0, tied = 0;                      // taken above and equals before this wave's run
  for (int w = 0; w < wid; ++w) { at += wave_a[w]; tied += wave_b[w]; }
  const uint64_t below = (1ull << lane) - 1;
  each([&](int i, uint32_t k) {
    const bool up = upper(i, k), eq = equal(i, k);
    const uint64_t mu = __ballot(up), me = __ballot(eq);
    const int ub = at + __popcll(mu & below), eb = tied + __popcll(me & below);
    if (up || (eq && eb < need)) out[ub + min(eb, need)] = i;
    at += __popcll(mu);
    tied += __popcll(me);
  });
}

// ------------------------------------------------------------------ attention

struct SparseArgs {
  CacheArgs c;
  const uint16_t* q;
  int64_t q_ts, q_hs;
  const int32_t* bt;
  int64_t bt_stride;
  const int4* tok;
  const int32_t* sel;
  int64_t sel_ts, sel_hs;
  int32_t selected, parts, t0, t1;                    // tokens [t0, t1) of this launch
  const int32_t* hdr;
  uint16_t* out;
  int64_t o_ts, o_hs;
  uint16_t* part_o;          // (token, KV head, head block, part): 16 rows of D
  PartHead* part_head;
};

constexpr int kSpWaves = 4;

// A wave's row of 16 query heads: token t, KV head kvh, head block hb.
struct SparseRow {
  int t, kvh, hb;
  int4 tk;                   // {request, position, visible blocks}
  const int32_t* sel;
  const int32_t* btrow;
  __device__ __forceinline__ SparseRow(const SparseArgs& a, int t, int kvh, int hb)
      : t(t), kvh(kvh), hb(hb), tk(a.tok[t]), sel(a.sel + (int64_t)t * a.sel_ts + (int64_t)kvh * a.sel_hs),
        btrow(a.bt + (int64_t)max(tk.x, 0) * a.bt_stride) {}
  // The block ids of the selected blocks in [b0, b1) that the token sees, in order, into
  // list; returns their number and the keys that they hold for it.  Entries that do not
  // exceed all before them drop out, so only the last block, the token's own, can be
  // cut short.
  __device__ __forceinline__ int blocks(const SparseArgs& a, int b0, int b1, int* list, int lane, int& keys) const {
    int count = 0, most = -1;
    bool own = false;
    for (int i = 0; i < a.selected; i += 64) {
      const int e = i + lane < a.selected ? sel[i + lane] : -1;
      int upto = e;                          // the largest entry up to this lane's
      int prev = __shfl_up(upto, 1);
      int last = __popcll(__ballot(e >= 0)) - 1;       // in order: the largest entry's lane
      if (__any(lane && e >= 0 && (prev < 0 || prev >= e))) {
        last = 63;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
          const int x = __shfl_up(upto, d);
          if (lane >= d) upto = max(upto, x);
        }
        prev = __shfl_up(upto, 1);
      }
      const int before = lane ? max(most, prev) : most;
      const bool ok = e >= b0 && e < min(b1, tk.z) && e > before;
      const uint64_t m = __ballot(ok);
      if (ok) list[count + __popcll(m & ((1ull << lane) - 1))] = btrow[e];
      count += __popcll(m);
      own |= __any(ok && e == tk.y / a.c.bs) != 0;
      if (last >= 0) most = max(most, __shfl(upto, last));
      if (most >= b1) break;                 // (the rest is behind the range)
    }
    keys = count * a.c.bs - (own ? a.c.bs - 1 - tk.y % a.c.bs : 0);
    return count;
  }
  // row n's query head within the KV head's group
  __device__ __forceinline__ int head(int n) const { return hb * kRows + n; }
  // what a row without keys has for a sum: NaN where the plan has none
  __device__ __forceinline__ float no_keys() const { return tk.x == kBadStep ? __builtin_nanf("") : 0.f; }
  __device__ __forceinline__ const uint16_t* query(const SparseArgs& a, int n) const {
    return head(n) < a.c.group ? a.q + (int64_t)t * a.q_ts + (int64_t)(kvh * a.c.group + head(n)) * a.q_hs : nullptr;
  }
  __device__ __forceinline__ uint16_t* output(const SparseArgs& a, int n) const {
    return a.out + (int64_t)t * a.o_ts + (int64_t)(kvh * a.c.group + head(n)) * a.o_hs;
  }
};
__device__ __forceinline__ int head_blocks(const SparseArgs& a) { return (a.c.group + kRows - 1) / kRows; }
__device__ __forceinline__ int64_t part_row(const SparseArgs& a, int t, int kvh, int hb, int part) {
  return ((((int64_t)(t - a.t0) * a.c.hkv + kvh) * head_blocks(a) + hb) * a.parts + part) * kRows;
}

// One work-group: 16 query heads of a token and KV head and one of the parts of its
// selected keys, four waves with a run of tiles each, joined in LDS.  8 tokens of 64 blocks
// of 32 keys, 8 heads of 128: 67 MB in 17 us, 3.9 TB/s, with the join 20.9; the first 5 us
// go by before a key arrives.
template <int D, bool F8, bool WHOLE>
__global__ __launch_bounds__(64 * kSpWaves) __attribute__((amdgpu_waves_per_eu(3, 3))) void sparse_attn_kernel(SparseArgs a) {
  constexpr int DT = D / 16;
  constexpr int kJoinBytes = kSpWaves * DT * 64 * 16, kStageBytes = kSpWaves * kStep * 2;
  __shared__ __attribute__((aligned(16))) uint8_t lds[kJoinBytes > kStageBytes ? kJoinBytes : kStageBytes];
  __shared__ int list[kMaxSelected];
  __shared__ float wave_m[kSpWaves][kRows], wave_l[kSpWaves][kRows];
  auto* join = reinterpret_cast<float4_t(*)[DT][64]>(lds);     // the waves' results, after their last V tile
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int item = blockIdx.x / a.parts, part = blockIdx.x - item * a.parts, hblocks = head_blocks(a);
  const SparseRow r(a, a.t0 + item / hblocks / a.c.hkv, item / hblocks % a.c.hkv, item % hblocks);
  uint4 qf[D / 32];
  load_q<D>(r.query(a, n), g, qf);
  int keys;
  const int count = r.blocks(a, 0, INT32_MAX, list, lane, keys);   // (every wave builds the same list)
  __syncthreads();
  const int tiles = (keys + kTile - 1) / kTile, cuts = a.parts * kSpWaves, p = part * kSpWaves + wid;
  const int t0 = (int)((int64_t)tiles * p / cuts), t1 = (int)((int64_t)tiles * (p + 1) / cuts);
  RowState<D> s;
  s.clear();
  attend<D, F8, WHOLE>(a.c, r.kvh, qf, t0 * kTile, min(keys, t1 * kTile), count, [&](int i) { return list[i]; },
                reinterpret_cast<uint16_t*>(lds) + wid * kStep, lane, s);
  s.finish();
  if (keys == 0) s.l = r.no_keys();
  __syncthreads();
  if (g == 0) { wave_m[wid][n] = s.m; wave_l[wid][n] = s.l; }
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) join[wid][dt][lane] = s.o[dt];
  __syncthreads();
  if (wid != 0) return;
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < kSpWaves; ++i) m = fmaxf(m, wave_m[i][n]);
  float4_t o[DT];
  clear_row(o);
#pragma unroll
  for (int i = 0; i < kSpWaves; ++i) {
    // (a wave that saw no key; one that saw NaN alone has -inf and NaN)
    const float w = wave_m[i][n] == -INFINITY && wave_l[i][n] == 0.f ? 0.f : __builtin_amdgcn_exp2f(wave_m[i][n] - m);
    l += w * wave_l[i][n];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] += join[i][dt][lane] * w;
  }
  const bool live = r.head(n) < a.c.group;
  if (a.parts > 1) write_part<D>(a.part_o, a.part_head, part_row(a, r.t, r.kvh, r.hb, part) + n, o, m, l, live, g);
  else if (live) write_out<D>(r.output(a, n), o, l, g);
}

// One wave: 16 query heads of a token and KV head and the selected blocks in one range
// of the context.  A range is taken on one XCD (block ids are dealt to the eight in
// turn).  Four of five lines come from L2, 14 TB/s in all; L1, LDS and VALU are busy a
// third of the time each.
template <int D, bool F8, bool WHOLE>
__global__ __launch_bounds__(64 * kSpWaves) __attribute__((amdgpu_waves_per_eu(3, 3))) void sparse_range_kernel(SparseArgs a) {
  __shared__ __attribute__((aligned(16))) uint16_t vt[kSpWaves][kStep];
  __shared__ int list[kSpWaves][kRangeBlocks];
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4, hblocks = head_blocks(a);
  const int per = ((a.t1 - a.t0) * a.c.hkv * hblocks + kSpWaves - 1) / kSpWaves;      // work-groups of a range
  const int k = blockIdx.x / 8, part = k / per * 8 + blockIdx.x % 8, i = k % per * kSpWaves + wid;
  const int t = a.t0 + i / hblocks / a.c.hkv, kvh = i / hblocks % a.c.hkv;
  if (t >= a.t1) return;
  const SparseRow r(a, t, kvh, i % hblocks);
  uint4 qf[D / 32];                          // (arrives while the list is made)
  load_q<D>(r.query(a, n), g, qf);
  int keys;
  const int blocks = min(kRangeBlocks, (a.hdr[1] + a.parts - 1) / a.parts), b0 = part * blocks;
  const int count = r.blocks(a, b0, b0 + blocks, list[wid], lane, keys);
  const int64_t row = part_row(a, t, kvh, r.hb, part) + n;
  const bool live = r.head(n) < a.c.group;
  if (count == 0) {
    if (live && g == 0) a.part_head[row] = no_part(r.no_keys());
    return;
  }
  RowState<D> s;
  s.clear();
  __builtin_amdgcn_wave_barrier();           // the list is the wave's own
  attend<D, F8, WHOLE>(a.c, kvh, qf, 0, keys, count, [&](int j) { return list[wid][j]; }, vt[wid], lane, s);
  s.finish();
  write_part<D>(a.part_o, a.part_head, row, s.o, s.m, s.l, live, g);
}

// The parts of each row, joined.
template <int D, int W>
__global__ __launch_bounds__(256) void sparse_join_kernel(SparseArgs a) {
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hq = a.c.group * a.c.hkv, t = a.t0 + blockIdx.x, head = W > 1 ? blockIdx.y : blockIdx.y * 4 + wid;
  if (head >= hq) return;
  const int kvh = head / a.c.group, hh = head - kvh * a.c.group;
  const int64_t first = part_row(a, t, kvh, hh / kRows, 0) + hh % kRows;
  join_row<D, W>(a.part_o, a.part_head, a.parts, [&](int i) { return first + i * kRows; },
                 a.out + (int64_t)t * a.o_ts + (int64_t)head * a.o_hs);
}

// ------------------------------------------------------------------ checks

int check_step(const char* what, int32_t batch, int32_t tokens, int32_t hq, int32_t hkv, int32_t d, int32_t bs,
               int32_t width, int32_t selected) {
  using namespace aia;
  if (batch < 0 || tokens < 0 || hq <= 0 || hkv <= 0 || bs <= 0 || width <= 0 || hq % hkv)
    return fail(AIA_ERR_INVALID, "%s: bad sizes (batch %d, tokens %d, heads %d / %d, block %d, table width %d)",
                what, batch, tokens, hq, hkv, bs, width);
  if (d != 128 && d != 64) return fail(AIA_ERR_UNSUPPORTED, "%s: head_dim %d (128 or 64)", what, d);
  if (batch > kMaxBatch) return fail(AIA_ERR_UNSUPPORTED, "%s: %d requests (at most %d)", what, batch, kMaxBatch);
  if (hkv > 65535) return fail(AIA_ERR_UNSUPPORTED, "%s: %d KV heads (at most 65535)", what, hkv);
  if (hq / hkv > 256) return fail(AIA_ERR_UNSUPPORTED, "%s: %d query heads per KV head (at most 256)", what, hq / hkv);
  if ((int64_t)bs * width > INT32_MAX)
    return fail(AIA_ERR_UNSUPPORTED, "%s: contexts of 2^31 tokens and more", what);
  if (selected <= 0 || selected > kMaxSelected)
    return fail(AIA_ERR_UNSUPPORTED, "%s: %d selected blocks (1 to %d)", what, selected, kMaxSelected);
  return AIA_OK;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

}  // namespace

extern "C" int aia_sparse_workspace_bytes(int32_t batch, int32_t num_tokens, int32_t num_q_heads,
                                          int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                                          int32_t table_width, int32_t num_selected, int64_t* bytes) {
  using namespace aia;
  if (!bytes) return fail(AIA_ERR_INVALID, "aia_sparse_workspace_bytes: null pointer argument");
  if (int rc = check_step("aia_sparse_workspace_bytes", batch, num_tokens, num_q_heads, num_kv_heads, head_dim,
                          block_size, table_width, num_selected))
    return rc;
  *bytes = sparse_layout(batch, num_tokens, num_q_heads, num_kv_heads, head_dim, block_size, table_width, num_selected).total;
  return AIA_OK;
}

// What the entry points check of a step and its workspace; fills L.
static int sparse_step(const char* what, int32_t batch, int32_t tokens, int32_t hq, int32_t hkv, int32_t d,
                       int32_t bs, int32_t width, int32_t selected, const void* ws, int64_t ws_bytes,
                       SparseLayout& L) {
  using namespace aia;
  if (int rc = check_step(what, batch, tokens, hq, hkv, d, bs, width, selected)) return rc;
  if (!ws || ((uintptr_t)ws & 255u)) return fail(AIA_ERR_INVALID, "%s: workspace must be 256-byte aligned", what);
  L = sparse_layout(batch, tokens, hq, hkv, d, bs, width, selected);
  if (ws_bytes < L.total)
    return fail(AIA_ERR_CAPACITY, "%s: workspace of %lld bytes, %lld needed", what, (long long)ws_bytes, (long long)L.total);
  return AIA_OK;
}

extern "C" int aia_sparse_plan(const int32_t* cu_seqlens_q, const int32_t* seqlens_kv, const int32_t* block_table,
                               int32_t block_table_stride, int32_t table_width, int32_t block_size, int32_t batch,
                               int32_t num_tokens, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                               int32_t num_selected, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace aia;
  SparseLayout L;
  if (int rc = sparse_step("aia_sparse_plan", batch, num_tokens, num_q_heads, num_kv_heads, head_dim, block_size,
                           table_width, num_selected, workspace, workspace_bytes, L))
    return rc;
  if (!cu_seqlens_q || (batch > 0 && (!seqlens_kv || !block_table)))
    return fail(AIA_ERR_INVALID, "aia_sparse_plan: null pointer argument");
  if (batch > 1 && block_table_stride < table_width)
    return fail(AIA_ERR_INVALID, "aia_sparse_plan: table rows overlap");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  PlanArgs a;
  a.cu = cu_seqlens_q; a.lk = seqlens_kv; a.bt = block_table; a.bt_stride = block_table_stride;
  a.batch = batch; a.tokens = num_tokens; a.bs = block_size; a.width = table_width;
  a.hdr = reinterpret_cast<int32_t*>(ws + L.hdr);
  a.tok = reinterpret_cast<int4*>(ws + L.tok);
  a.touched = reinterpret_cast<int4*>(ws + L.touched);
  a.touched_cap = L.touched_cap;
  const unsigned grid = std::max(1, (num_tokens + kPlanT - 1) / kPlanT);
  const size_t lds = (size_t)(2 * batch + 1) * sizeof(int);
  if (lds > 48 * 1024) {
    if (int rc = check_hip(hipFuncSetAttribute(reinterpret_cast<const void*>(sparse_plan_kernel),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds),
                           "aia_sparse_plan"))
      return rc;
  }
  sparse_plan_kernel<<<grid, kPlanT, lds, (hipStream_t)stream>>>(a);
  return check_hip(hipGetLastError(), "aia_sparse_plan launch");
}

extern "C" int aia_summarize_blocks(const void* key_cache, const void* key_scale, int32_t num_blocks,
                                    void* bounds, void* bounds_scale, int32_t block_size, int32_t table_width,
                                    int32_t batch, int32_t num_tokens, int32_t num_q_heads, int32_t num_kv_heads,
                                    int32_t head_dim, int32_t num_selected, const void* workspace,
                                    int64_t workspace_bytes, void* stream) {
  using namespace aia;
  SparseLayout L;
  if (int rc = sparse_step("aia_summarize_blocks", batch, num_tokens, num_q_heads, num_kv_heads, head_dim,
                           block_size, table_width, num_selected, workspace, workspace_bytes, L))
    return rc;
  if (num_tokens == 0) return AIA_OK;
  if (!key_cache || !bounds || !bounds_scale || num_blocks <= 0)
    return fail(AIA_ERR_INVALID, "aia_summarize_blocks: null pointer argument or no blocks");
  if (!aligned16(key_cache) || !aligned16(bounds))
    return fail(AIA_ERR_INVALID, "aia_summarize_blocks: tensors must be 16-byte aligned");
  const uint8_t* ws = static_cast<const uint8_t*>(workspace);
  SummaryArgs a;
  a.kc = static_cast<const uint16_t*>(key_cache); a.ks = static_cast<const uint8_t*>(key_scale);
  a.hkv = num_kv_heads; a.bs = block_size; a.nb = num_blocks;
  a.hdr = reinterpret_cast<const int32_t*>(ws + L.hdr);
  a.touched = reinterpret_cast<const int4*>(ws + L.touched);
  a.bounds = static_cast<int8_t*>(bounds); a.scale = static_cast<uint8_t*>(bounds_scale);
  const bool cut = block_size >= 64;
  const dim3 grid((unsigned)L.touched_cap, (unsigned)(cut ? num_kv_heads : (num_kv_heads + 3) / 4));
  auto pick = [&](auto d) {
    constexpr int D = decltype(d)::value;
    return key_scale ? (cut ? summarize_kernel<D, true, 4> : summarize_kernel<D, true, 1>)
                     : (cut ? summarize_kernel<D, false, 4> : summarize_kernel<D, false, 1>);
  };
  auto* kernel = head_dim == 128 ? pick(std::integral_constant<int, 128>{}) : pick(std::integral_constant<int, 64>{});
  kernel<<<grid, kSparseThreads, 0, (hipStream_t)stream>>>(a);
  return check_hip(hipGetLastError(), "aia_summarize_blocks launch");
}

extern "C" int aia_select_blocks(const void* query, int64_t q_token_stride, int64_t q_head_stride,
                                 const void* bounds, const void* bounds_scale, int32_t num_blocks,
                                 const int32_t* block_table, int32_t block_table_stride, int32_t table_width,
                                 int32_t block_size, int32_t batch, int32_t num_tokens, int32_t num_q_heads,
                                 int32_t num_kv_heads, int32_t head_dim, int32_t num_selected, int32_t sink,
                                 int32_t local, int32_t* selected, int64_t sel_token_stride,
                                 int64_t sel_head_stride, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace aia;
  SparseLayout L;
  if (int rc = sparse_step("aia_select_blocks", batch, num_tokens, num_q_heads, num_kv_heads, head_dim, block_size,
                           table_width, num_selected, workspace, workspace_bytes, L))
    return rc;
  if (sink < 0 || local < 1 || (int64_t)sink + local > num_selected)
    return fail(AIA_ERR_INVALID, "aia_select_blocks: sink %d and local %d do not fit %d selected blocks (local at least 1)",
                sink, local, num_selected);
  if (num_tokens == 0) return AIA_OK;
  if (!query || !bounds || !bounds_scale || !block_table || !selected || num_blocks <= 0)
    return fail(AIA_ERR_INVALID, "aia_select_blocks: null pointer argument or no blocks");
  if (!aligned16(query) || !aligned16(bounds) || q_token_stride % 8 || q_head_stride % 8)
    return fail(AIA_ERR_INVALID, "aia_select_blocks: tensors must be 16-byte aligned with strides a multiple of 8");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  ScoreKernelArgs a;
  a.q = static_cast<const uint16_t*>(query); a.q_ts = q_token_stride; a.q_hs = q_head_stride;
  a.bounds = static_cast<const int8_t*>(bounds); a.scale = static_cast<const uint8_t*>(bounds_scale);
  a.bt = block_table; a.bt_stride = block_table_stride;
  a.tok = reinterpret_cast<const int4*>(ws + L.tok);
  a.scores = reinterpret_cast<float*>(ws + L.scores);
  a.hkv = num_kv_heads; a.group = num_q_heads / num_kv_heads; a.nb = num_blocks; a.width = table_width;
  // Tokens of a tile share their request's bounds: worth it where requests have several.
  const bool many = num_tokens >= 4 * batch;
  const int per = many ? kTileTokens : 1;
  SelectArgs s;
  s.scores = a.scores; s.tok = a.tok; s.out = selected; s.out_ts = sel_token_stride; s.out_hs = sel_head_stride;
  s.hkv = num_kv_heads; s.width = table_width; s.selected = num_selected; s.sink = sink; s.local = local;
  hipStream_t st = (hipStream_t)stream;
  for (int t0 = 0; t0 < num_tokens; t0 += L.score_tokens) {
    const int t1 = std::min(num_tokens, t0 + L.score_tokens);
    a.t0 = t0; a.t1 = t1; s.t0 = t0; s.rows = (t1 - t0) * num_kv_heads;
    const unsigned gx = (unsigned)((t1 - t0 + per - 1) / per);
    // work-groups: about eight per compute unit, each of 256 blocks (64 a wave) or more
    const int64_t batches = (table_width + kSparseThreads - 1) / kSparseThreads;
    const int64_t cuts = std::max<int64_t>(1, std::min<int64_t>(2048 / std::max<int64_t>(1, (int64_t)gx * num_kv_heads), batches));
    a.chunk = (int)((batches + cuts - 1) / cuts * kSparseThreads);
    const dim3 grid(gx, (unsigned)num_kv_heads, (unsigned)((table_width + a.chunk - 1) / a.chunk));
    auto* score = many ? (head_dim == 128 ? score_kernel<128> : score_kernel<64>)
                       : (head_dim == 128 ? score_token_kernel<128> : score_token_kernel<64>);
    score<<<grid, kSparseThreads, 0, st>>>(a);
    if (int rc = check_hip(hipGetLastError(), "aia_select_blocks: score launch")) return rc;
    // (keys held for the table's width and little more: places behind it cost what keys
    // do, 22.2 us instead of 20.3 for 4,096 blocks with twice as many)
    if (table_width <= 1024) {
      auto* kernel = table_width <= 256   ? select_wave_kernel<4>
                     : table_width <= 384 ? select_wave_kernel<6>
                     : table_width <= 512 ? select_wave_kernel<8>
                     : table_width <= 640 ? select_wave_kernel<10>
                     : table_width <= 768 ? select_wave_kernel<12>
                                          : select_wave_kernel<16>;
      kernel<<<(unsigned)((s.rows + 3) / 4), 256, 0, st>>>(s);
    } else {
      auto* kernel = table_width <= 4 * kSelThreads    ? select_kernel<4>
                     : table_width <= 8 * kSelThreads  ? select_kernel<8>
                     : table_width <= 16 * kSelThreads ? select_kernel<16>
                                                       : select_kernel<0>;
      kernel<<<(unsigned)s.rows, kSelThreads, 0, st>>>(s);
    }
    if (int rc = check_hip(hipGetLastError(), "aia_select_blocks: select launch")) return rc;
  }
  return AIA_OK;
}

extern "C" int aia_paged_attention_sparse(const void* query, int64_t q_token_stride, int64_t q_head_stride,
                                          const void* key_cache, const void* value_cache, const void* key_scale,
                                          const void* value_scale, int32_t num_blocks, const int32_t* block_table,
                                          int32_t block_table_stride, int32_t table_width, int32_t block_size,
                                          int32_t batch, int32_t num_tokens, int32_t num_q_heads,
                                          int32_t num_kv_heads, int32_t head_dim, float scale,
                                          const int32_t* selected, int64_t sel_token_stride, int64_t sel_head_stride,
                                          int32_t num_selected, void* out, int64_t out_token_stride,
                                          int64_t out_head_stride, void* workspace, int64_t workspace_bytes,
                                          void* stream) {
  using namespace aia;
  SparseLayout L;
  if (int rc = sparse_step("aia_paged_attention_sparse", batch, num_tokens, num_q_heads, num_kv_heads, head_dim,
                           block_size, table_width, num_selected, workspace, workspace_bytes, L))
    return rc;
  if (!(scale > 0.f) || !(scale < 1e30f))
    return fail(AIA_ERR_INVALID, "aia_paged_attention_sparse: scale must be positive");
  if (num_tokens == 0) return AIA_OK;
  if (!query || !key_cache || !value_cache || !block_table || !selected || !out || num_blocks <= 0)
    return fail(AIA_ERR_INVALID, "aia_paged_attention_sparse: null pointer argument or no blocks");
  if ((key_scale == nullptr) != (value_scale == nullptr))
    return fail(AIA_ERR_INVALID, "aia_paged_attention_sparse: key_scale and value_scale go together");
  if (!aligned16(query) || !aligned16(key_cache) || !aligned16(value_cache) || q_token_stride % 8 ||
      q_head_stride % 8 || ((uintptr_t)out & 7u) || out_token_stride % 4 || out_head_stride % 4)
    return fail(AIA_ERR_INVALID, "aia_paged_attention_sparse: query and caches must be 16-byte aligned with strides "
                "a multiple of 8, out 8-byte aligned with strides a multiple of 4");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  SparseArgs a;
  a.c.kc = static_cast<const uint16_t*>(key_cache); a.c.vc = static_cast<const uint16_t*>(value_cache);
  a.c.ks = static_cast<const uint8_t*>(key_scale); a.c.vs = static_cast<const uint8_t*>(value_scale);
  a.c.hkv = num_kv_heads; a.c.group = num_q_heads / num_kv_heads; a.c.bs = block_size; a.c.nb = num_blocks;
  a.c.scale_log2 = scale * kLog2e;
  a.q = static_cast<const uint16_t*>(query); a.q_ts = q_token_stride; a.q_hs = q_head_stride;
  a.bt = block_table; a.bt_stride = block_table_stride;
  a.tok = reinterpret_cast<const int4*>(ws + L.tok);
  a.sel = selected; a.sel_ts = sel_token_stride; a.sel_hs = sel_head_stride; a.selected = num_selected;
  a.parts = L.cut.parts; a.hdr = reinterpret_cast<const int32_t*>(ws + L.hdr);
  a.out = static_cast<uint16_t*>(out); a.o_ts = out_token_stride; a.o_hs = out_head_stride;
  a.part_o = reinterpret_cast<uint16_t*>(ws + L.part_o); a.part_head = reinterpret_cast<PartHead*>(ws + L.part_head);
  hipStream_t s = (hipStream_t)stream;
  for (int t0 = 0; t0 < num_tokens; t0 += L.cut.tokens) {
    a.t0 = t0;
    a.t1 = std::min(num_tokens, t0 + L.cut.tokens);
    const int64_t items = (int64_t)(a.t1 - a.t0) * num_kv_heads * L.hblocks;
    const int64_t groups = a.parts * (L.cut.ranges ? (items + kSpWaves - 1) / kSpWaves : items);
    if (groups > INT32_MAX) return fail(AIA_ERR_UNSUPPORTED, "aia_paged_attention_sparse: too many rows in one call");
    auto pick = [&](auto d, auto f8) {
      constexpr int D = decltype(d)::value;
      constexpr bool F8 = decltype(f8)::value, T = true, F = false;
      const bool whole = block_size % kTile == 0;
      return L.cut.ranges ? (whole ? sparse_range_kernel<D, F8, T> : sparse_range_kernel<D, F8, F>)
                            : (whole ? sparse_attn_kernel<D, F8, T> : sparse_attn_kernel<D, F8, F>);
    };
    using d128 = std::integral_constant<int, 128>;
    using d64 = std::integral_constant<int, 64>;
    auto* kernel = head_dim == 128 ? (key_scale ? pick(d128{}, std::true_type{}) : pick(d128{}, std::false_type{}))
                                   : (key_scale ? pick(d64{}, std::true_type{}) : pick(d64{}, std::false_type{}));
    kernel<<<(unsigned)groups, 64 * kSpWaves, 0, s>>>(a);
    if (int rc = check_hip(hipGetLastError(), "aia_paged_attention_sparse launch")) return rc;
    if (a.parts == 1) continue;
    const bool few = (int64_t)(a.t1 - t0) * num_q_heads < kFewRows;
    auto* join = head_dim == 128 ? (few ? sparse_join_kernel<128, 4> : sparse_join_kernel<128, 1>)
                                 : (few ? sparse_join_kernel<64, 4> : sparse_join_kernel<64, 1>);
    join<<<dim3((unsigned)(a.t1 - t0), (unsigned)(few ? num_q_heads : (num_q_heads + 3) / 4)), 256, 0, s>>>(a);
    if (int rc = check_hip(hipGetLastError(), "aia_paged_attention_sparse: join launch")) return rc;
  }
  return AIA_OK;
}
