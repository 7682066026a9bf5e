// KV slot write into 8-bit caches: e4m3 values with one e8m0 (power of two)
// scale per cache block and KV head, for K and V each.
//
// For a block and head that the call's rows touch, amax = the largest finite
// |x| of those rows and need = the least e >= -100 with amax <= 448 * 2^e.  The
// block's exponent becomes need when the call writes its first slot (it starts
// anew), else max(old, need).  A row is stored as x * 2^-e rounded to nearest
// even (not finite: NaN); the other rows of a block whose exponent grew are
// rescaled by 2^(old - e).  Powers of two make that rescaling exact but for
// values that fall below e4m3's normal range, so a block appended to token by
// token holds what one write of all its rows would have stored, up to those.
//
// All of a block's rows in the call have to be known before any is stored.
// The slots may come in any order, so each (block, head) has one work-group:
// that of the call's first token in the block, its leader.
#include <algorithm>
#include <type_traits>

#include "common.h"

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kWavePasses = 4;        // row passes of a run that a wave takes
constexpr int kTableBits = 10, kTable = 1 << kTableBits;
constexpr int kScan = 16;             // slots a thread reads at once in search of a block's tokens
// Work-groups of a long step: more leave fewer runs to each, but more of them
// find none and all scan.  us at 768 (small blocks: 1536), as below, and at twice
// that: 16,384 prompt tokens, 8 heads of 128, blocks of 128 39.0, 31.8, 32.2,
// blocks of 32 43.4, 37.6, 48.1, blocks of 16 35.0, 36.0, 37.7; 1,024 decode rows,
// blocks of 128 20.1, 16.3, 17.7.
constexpr int kTargetGroups = 1024, kTargetGroupsSmall = 2048;
constexpr int kMaxBlock = 8192;       // slots of a block: its tokens are listed in LDS
constexpr int kMinExp = -100;

struct Args {
  const uint16_t* src[2];             // K, V rows
  int64_t ts[2];
  uint8_t* cache[2];
  uint8_t* scale[2];
  const int32_t* slots;
  int32_t tokens, hkv, bs, sub;
  uint32_t div_mul, div_shift;         // slot / bs (bs > 1)
  int64_t num_slots;

  __device__ __forceinline__ int block_of(int slot) const {       // slot >= 0 (see the host side)
    return bs == 1 ? slot : (int)(__umulhi((uint32_t)slot, div_mul) >> div_shift);
  }
};

// A value that all lanes hold, in scalar registers.
__device__ __forceinline__ uint64_t uniform64(uint64_t x) {
  return (uint32_t)__builtin_amdgcn_readfirstlane((int)x) |
         (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32;
}

// Eight consecutive bf16 values.
template <bool VEC>
__device__ __forceinline__ uint4 load8(const uint16_t* p) {
  if (VEC) return *reinterpret_cast<const uint4*>(p);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = p[2 * i] | (uint32_t)p[2 * i + 1] << 16;
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Largest finite |x| of eight bf16 values, as bf16 bits.
__device__ __forceinline__ uint32_t amax8(uint4 v, uint32_t m) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = w[i] & 0x7fffu, hi = (w[i] >> 16) & 0x7fffu;
    m = max(m, lo < 0x7f80u ? lo : 0u);
    m = max(m, hi < 0x7f80u ? hi : 0u);
  }
  return m;
}

// The e8m0 byte for amax (bf16 bits): 448 = 1.75 * 2^8.
__device__ __forceinline__ int needed_byte(uint32_t amax) {
  const int e = (int)(amax >> 7) - 127 - 8 + ((amax & 0x7fu) > 0x60u ? 1 : 0);
  return max(amax < 0x80u ? kMinExp : e, kMinExp) + 127;
}

__device__ __forceinline__ float scaled(float x, float f) {
  return __builtin_fabsf(x) < INFINITY ? x * f : __builtin_nanf("");
}

// Eight bf16 values times f as e4m3.
__device__ __forceinline__ uint2 quantise8(uint4 v, float f) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t o[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int r = 0;
    r = __builtin_amdgcn_cvt_pk_fp8_f32(scaled(aia::bf16_lo(w[2 * i]), f), scaled(aia::bf16_hi(w[2 * i]), f), r, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(scaled(aia::bf16_lo(w[2 * i + 1]), f),
                                        scaled(aia::bf16_hi(w[2 * i + 1]), f), r, true);
    o[i] = (uint32_t)r;
  }
  return make_uint2(o[0], o[1]);
}

// Four e4m3 values times 2^-down.
__device__ __forceinline__ uint32_t rescale4(uint32_t w, int down) {
  const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
  int r = 0;
  r = __builtin_amdgcn_cvt_pk_fp8_f32(__builtin_ldexpf(a[0], -down), __builtin_ldexpf(a[1], -down), r, false);
  r = __builtin_amdgcn_cvt_pk_fp8_f32(__builtin_ldexpf(b[0], -down), __builtin_ldexpf(b[1], -down), r, true);
  return (uint32_t)r;
}

// The tokens of a window of kThreads tokens that start a run (tokens at
// consecutive slots of one block) and, of the window and the next, that
// continue one; returns the thread's token's slot (-1: none).
__device__ __forceinline__ int find_runs(const Args& a, int t0, uint64_t* starts, uint64_t* joins, bool& start) {
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  auto slot_at = [&](int t) { return t >= 0 && t < a.tokens ? a.slots[t] : -1; };
  const int own = slot_at(t0 + tid), before = slot_at(t0 + tid - 1);
  const int next = slot_at(t0 + kThreads + tid), before_next = slot_at(t0 + kThreads + tid - 1);
  // (a slot that follows its predecessor's is in the same block unless it is a
  // block's first; a predecessor that is skipped is followed by none)
  auto follows = [&](int s, int b) {
    return s == b + 1 && b >= 0 && s < a.num_slots && s != a.block_of(s) * a.bs;
  };
  const bool join = follows(own, before), join_next = follows(next, before_next);
  start = own >= 0 && own < a.num_slots && !join;
  const uint64_t s = __ballot(start), j = __ballot(join), k = __ballot(join_next);
  if (lane == 0) { starts[wid] = s; joins[wid] = j; joins[kWaves + wid] = k; }
  __syncthreads();
  return own;
}

// Lists the window's runs sub, sub + a.sub, ...: first slot, first token and
// length as far as the two windows show; returns their number.  (Read the
// lists after a barrier.)
__device__ __forceinline__ int take_runs(const Args& a, int t0, int sub, int own, bool start,
                                         const uint64_t* starts, const uint64_t* joins, int* run_slot,
                                         int* run_tok, int* run_len, int* run_count) {
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  int total = 0, rank = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const uint64_t s = uniform64(starts[w]);
    total += __popcll(s);
    rank += w < wid ? __popcll(s) : w == wid ? __popcll(s & ((1ull << lane) - 1)) : 0;
  }
  if (sub >= total) return 0;
  if (start && rank % a.sub == sub) {
    int len = 1;
    for (int v = wid, from = lane + 1; v < 2 * kWaves; ++v, from = 0) {
      if (from == 64) continue;
      const uint64_t stop = ~joins[v] >> from;
      if (stop) { len += __builtin_ctzll(stop); break; }
      len += 64 - from;
    }
    const int i = rank / a.sub;
    run_slot[i] = own; run_tok[i] = t0 + tid; run_len[i] = len; run_count[i] = 0;
  }
  return (total - sub - 1) / a.sub + 1;
}

// see(slot) for all of the call's slots, kScan independent loads per thread at
// once (-1 past the end).
template <class See>
__device__ __forceinline__ void scan(const Args& a, See see) {
  for (int first = 0; first < a.tokens; first += kThreads * kScan) {
    int s[kScan];
#pragma unroll
    for (int i = 0; i < kScan; ++i) {
      const int at = first + kThreads * i + threadIdx.x;
      s[i] = at < a.tokens ? a.slots[at] : -1;
    }
#pragma unroll
    for (int i = 0; i < kScan; ++i) see(s[i]);
  }
}

__device__ __forceinline__ uint32_t wave_amax(uint32_t v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v = max(v, (uint32_t)__shfl_xor((int)v, d));
  return v;
}

__device__ __forceinline__ void store8(uint8_t* p, uint4 v, float f) {
  *reinterpret_cast<uint2*>(p) = quantise8(v, f);
}

// A block's new exponent byte from its old one and the rows' amax; anew: its
// first slot is written.
__device__ __forceinline__ int new_exp(bool anew, int old, uint32_t amax) {
  const int need = needed_byte(amax);
  return anew ? need : max(old, need);
}

// The rows of a block that are not written, down by 2^down: rows first, first +
// step, ..., 16-byte piece `piece` of each; done(off): row off is written.
template <class Done>
__device__ __forceinline__ void rescale_rest(uint8_t* cache, int64_t row, int bs, int down, int first,
                                             int step, int piece, Done done) {
  for (int off = first; off < bs; off += step) {
    if (done(off)) continue;
    uint4* p = reinterpret_cast<uint4*>(cache + off * row) + piece;
    const uint4 v = *p;
    *p = make_uint4(rescale4(v.x, down), rescale4(v.y, down), rescale4(v.z, down), rescale4(v.w, down));
  }
}

// Grid: (sub x windows of kThreads tokens, KV heads); work-group s of a window
// takes its runs s, s + sub, ...  Almost always a run is all that its block gets
// in the call.  That is checked by counting the block's tokens among all slots,
// one scan for all of the work-group's runs (a small table in LDS finds the run
// of a slot's block); a run of a full count is stored as it stands, short ones by
// a wave each.  The rest go through the general path, which lists the block's
// tokens.  A work-group with one run compares slots with its block directly and
// loads the run's rows and scales meanwhile.
// Measured, us, for 16 decode rows (8 heads of 128, blocks of 16), 16,384 prompt
// tokens (8 heads of 128) in blocks of 128 and of 16, 7,399 ragged tokens (2
// heads of 64, blocks of 16) and 1,024 decode rows (8 heads, blocks of 128):
//   every token listed in LDS, all loads dependent      8.7  32.1     -  21.7     -
//   speculating, K and V in work-groups of their own    4.0  34.4     -  15.9     -
//   K and V together, a scan for each run               4.2  33.9  55.5  11.3  60.5
//   a scan for a work-group's runs (blocks of 16: for
//   four heads, the kernel below)                       4.7  31.8  36.0   8.6  16.3
// The prompt's bytes move at 3.2 TB/s in blocks of 128 (a large copy: 5.1): every
// block's loads are over before its stores begin, and the blocks run side by
// side; without the scan it takes 28.4.
template <int D, bool VEC, int kHold, int N>
__global__ __launch_bounds__(kThreads, 4) void kv_write_fp8_kernel(Args a) {
  constexpr int kLanes = D / 8, kLanes8 = D / 16;   // threads per new row, per cached row (16 bytes each)
  constexpr int kRows = kThreads / kLanes;          // rows per pass of the work-group,
  constexpr int kWaveRows = 64 / kLanes;            // of a wave
  constexpr int kShort = kWavePasses * kWaveRows;   // rows of a run that a wave takes
  extern __shared__ int last[];          // general path: a slot's last token, -1 = none
  __shared__ uint64_t starts[kWaves];    // tokens of the window that start a run
  __shared__ uint64_t joins[2 * kWaves]; // tokens of the window and the next that continue one
  __shared__ int run_slot[kThreads], run_tok[kThreads], run_len[kThreads], run_count[kThreads];
  __shared__ int table[kTable];          // run of a hashed block, -1 = none
  __shared__ int wave_lo[kWaves], wave_hi[kWaves];
  __shared__ uint32_t wave_max[N][kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = blockIdx.y;
  const int64_t row = (int64_t)a.hkv * D;
  // (work-groups of one sub index are neighbours, so those that find no run do
  // not fall on the same XCDs)
  const int windows = gridDim.x / a.sub, sub = blockIdx.x / windows, window = blockIdx.x - sub * windows;
  const int t0 = window * kThreads;
  auto block_of = [&](int s) { return a.block_of(s); };
  auto place_of = [&](int blk) { return (uint32_t)blk * 2654435761u >> (32 - kTableBits); };
  bool start;
  const int own = find_runs(a, t0, starts, joins, start);
  const int runs = take_runs(a, t0, sub, own, start, starts, joins, run_slot, run_tok, run_len, run_count);
  if (runs <= 0) return;
  auto src = [&](int x, int64_t t, int c) { return a.src[x] + t * a.ts[x] + h * D + 8 * c; };
  if (runs > 1) {
    for (int i = tid; i < kTable; i += kThreads) table[i] = -1;
    __syncthreads();
    if (tid < runs) {
      // a place taken by another run (of another block or, with tokens between
      // them, of the same) leaves this one without a count: the general path
      const int at = place_of(block_of(run_slot[tid]));
      if (atomicCAS(&table[at], -1, tid) != -1) run_count[tid] = kThreads * 8 * kMaxBlock;
    }
    __syncthreads();
    auto see = [&](int s) {
      if (s < 0 || s >= a.num_slots) return;
      const int blk = block_of(s), i = table[place_of(blk)];
      if (i >= 0 && block_of(run_slot[i]) == blk) atomicAdd(&run_count[i], 1);
    };
    if (a.tokens <= kThreads) see(own);
    else scan(a, see);
    __syncthreads();
    // short whole runs, a wave each
    const int r = lane / kLanes, c = lane % kLanes;
    for (int i = wid; i < runs; i += kWaves) {
      const int len = __builtin_amdgcn_readfirstlane(run_len[i]);
      if (len > kShort || __builtin_amdgcn_readfirstlane(run_count[i]) != len) continue;
      const int slot = __builtin_amdgcn_readfirstlane(run_slot[i]), t = __builtin_amdgcn_readfirstlane(run_tok[i]);
      const int blk = block_of(slot), lo = slot - blk * a.bs;
      const int64_t scale_at = (int64_t)blk * a.hkv + h;
      uint4 held[N][kWavePasses];
      int old[N];
#pragma unroll
      for (int x = 0; x < N; ++x) {
#pragma unroll
        for (int p = 0; p < kWavePasses; ++p) {
          held[x][p] = make_uint4(0, 0, 0, 0);
          const int k = p * kWaveRows + r;
          if (k < len) held[x][p] = load8<VEC>(src(x, t + k, c));
        }
        old[x] = a.scale[x][scale_at];
      }
#pragma unroll
      for (int x = 0; x < N; ++x) {
        uint32_t m = 0;
#pragma unroll
        for (int p = 0; p < kWavePasses; ++p) m = amax8(held[x][p], m);
        m = wave_amax(m);
        const int e = new_exp(lo == 0, old[x], m);
        const float f = __builtin_ldexpf(1.f, 127 - e);
        uint8_t* cache = a.cache[x] + (int64_t)blk * a.bs * row + h * D;
#pragma unroll
        for (int p = 0; p < kWavePasses; ++p) {
          const int k = p * kWaveRows + r;
          if (k < len) store8(cache + (int64_t)(lo + k) * row + 8 * c, held[x][p], f);
        }
        if (e == old[x]) continue;
        if (lane == 0) a.scale[x][scale_at] = (uint8_t)e;
        if (lo != 0)
          rescale_rest(cache, row, a.bs, e - old[x], lane / kLanes8, 64 / kLanes8, lane % kLanes8,
                       [&](int off) { return off >= lo && off < lo + len; });
      }
    }
  } else {
    __syncthreads();                     // the run's record
  }

  // the other runs, by the work-group
  const int r = tid / kLanes, c = tid % kLanes;
  for (int i = 0; i < runs; ++i) {
    const int len = __builtin_amdgcn_readfirstlane(run_len[i]);
    if (runs > 1 && len <= kShort && __builtin_amdgcn_readfirstlane(run_count[i]) == len) continue;
    const int slot = __builtin_amdgcn_readfirstlane(run_slot[i]), t = __builtin_amdgcn_readfirstlane(run_tok[i]);
    const int blk = block_of(slot), base = blk * a.bs;
    const int64_t scale_at = (int64_t)blk * a.hkv + h;
    uint4 held[N][kHold];
    int old[N];
#pragma unroll
    for (int x = 0; x < N; ++x) {
#pragma unroll
      for (int p = 0; p < kHold; ++p) {
        held[x][p] = make_uint4(0, 0, 0, 0);
        if (p * kRows + r < len) held[x][p] = load8<VEC>(src(x, t + p * kRows + r, c));
      }
      old[x] = a.scale[x][scale_at];
    }
    auto mine = [&](int s) { return (uint32_t)s - (uint32_t)base < (uint32_t)a.bs; };
    if (runs == 1) {
      int count = 0;                     // the block's tokens that this wave sees
      if (a.tokens <= kThreads) count = __popcll(__ballot(mine(own)));
      else scan(a, [&](int s) { count += __popcll(__ballot(mine(s))); });
      if (lane == 0) atomicAdd(&run_count[0], count);
    }
    uint32_t m[N];
    // (the previous run's maxima and list are read no more)
    if (runs > 1) __syncthreads();
#pragma unroll
    for (int x = 0; x < N; ++x) {
      m[x] = 0;
#pragma unroll
      for (int p = 0; p < kHold; ++p) m[x] = amax8(held[x][p], m[x]);
      for (int k = kHold * kRows + r; k < len; k += kRows) m[x] = amax8(load8<VEC>(src(x, t + k, c)), m[x]);
      m[x] = wave_amax(m[x]);
      if (lane == 0) wave_max[x][wid] = m[x];
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
#pragma unroll
      for (int x = 0; x < N; ++x) m[x] = max(m[x], wave_max[x][w]);
    const bool whole = __builtin_amdgcn_readfirstlane(run_count[i]) == len;   // the run is all the block gets
    int lo = slot - base, hi = lo + len - 1;
    if (!whole) {
      for (int k = tid; k < a.bs; k += kThreads) last[k] = -1;
      __syncthreads();
      int earlier = 0;
      lo = a.bs;
      hi = -1;
      for (int k = tid; k < a.tokens; k += kThreads) {
        const int s = a.slots[k];
        if (!mine(s)) continue;
        earlier |= k < t;
        atomicMax(&last[s - base], k);
        lo = min(lo, s - base);
        hi = max(hi, s - base);
      }
      if (__syncthreads_or(earlier)) continue;     // another token leads the block
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        lo = min(lo, __shfl_xor(lo, d));
        hi = max(hi, __shfl_xor(hi, d));
      }
      if (lane == 0) { wave_lo[wid] = lo; wave_hi[wid] = hi; }
#pragma unroll
      for (int x = 0; x < N; ++x) m[x] = 0;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kWaves; ++w) { lo = min(lo, wave_lo[w]); hi = max(hi, wave_hi[w]); }
      for (int off = lo + r; off <= hi; off += kRows) {
        if (last[off] < 0) continue;
#pragma unroll
        for (int x = 0; x < N; ++x) m[x] = amax8(load8<VEC>(src(x, last[off], c)), m[x]);
      }
#pragma unroll
      for (int x = 0; x < N; ++x) {
        m[x] = wave_amax(m[x]);
        if (lane == 0) wave_max[x][wid] = m[x];
      }
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kWaves; ++w)
#pragma unroll
        for (int x = 0; x < N; ++x) m[x] = max(m[x], wave_max[x][w]);
    }
#pragma unroll
    for (int x = 0; x < N; ++x) {
      const int e = new_exp(lo == 0, old[x], m[x]);
      const float f = __builtin_ldexpf(1.f, 127 - e);
      uint8_t* cache = a.cache[x] + (int64_t)base * row + h * D;
      if (whole) {
#pragma unroll
        for (int p = 0; p < kHold; ++p)
          if (p * kRows + r < len) store8(cache + (int64_t)(lo + p * kRows + r) * row + 8 * c, held[x][p], f);
        for (int k = kHold * kRows + r; k < len; k += kRows)
          store8(cache + (int64_t)(lo + k) * row + 8 * c, load8<VEC>(src(x, t + k, c)), f);
      } else {
        for (int off = lo + r; off <= hi; off += kRows)
          if (last[off] >= 0) store8(cache + (int64_t)off * row + 8 * c, load8<VEC>(src(x, last[off], c)), f);
      }
      if (e == old[x]) continue;
      if (tid == 0) a.scale[x][scale_at] = (uint8_t)e;
      if (lo != 0)                       // (the block's first slot is written: it starts anew)
        rescale_rest(cache, row, a.bs, e - old[x], tid / kLanes8, kThreads / kLanes8, tid % kLanes8,
                     [&](int off) { return whole ? off >= lo && off <= hi : last[off] >= 0; });
    }
  }
}

// Blocks of at most kShort slots (16 at head_dim 128, 32 at 64), whose runs fit
// the registers of a wave: a work-group takes a run for kWaves heads, a wave
// each, so that one scan serves them all.
template <int D, bool VEC, int N>
__global__ __launch_bounds__(kThreads) void kv_write_fp8_small_kernel(Args a) {
  constexpr int kLanes = D / 8, kLanes8 = D / 16, kWaveRows = 64 / kLanes;
  __shared__ int last[kWavePasses * kWaveRows];      // general path: a slot's last token, -1 = none
  __shared__ uint64_t starts[kWaves], joins[2 * kWaves];
  __shared__ int run_slot[kThreads], run_tok[kThreads], run_len[kThreads], run_count[kThreads];
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = blockIdx.y * kWaves + wid;
  const bool live = h < a.hkv;           // (waves of no head help to scan)
  const int64_t row = (int64_t)a.hkv * D;
  const int windows = gridDim.x / a.sub, sub = blockIdx.x / windows, window = blockIdx.x - sub * windows;
  const int t0 = window * kThreads;
  bool start;
  const int own = find_runs(a, t0, starts, joins, start);
  const int runs = take_runs(a, t0, sub, own, start, starts, joins, run_slot, run_tok, run_len, run_count);
  if (runs <= 0) return;
  __syncthreads();
  const int r = lane / kLanes, c = lane % kLanes;
  auto src = [&](int x, int64_t t) { return a.src[x] + t * a.ts[x] + h * D + 8 * c; };
  for (int i = 0; i < runs; ++i) {
    const int len = __builtin_amdgcn_readfirstlane(run_len[i]);
    const int slot = __builtin_amdgcn_readfirstlane(run_slot[i]), t = __builtin_amdgcn_readfirstlane(run_tok[i]);
    const int blk = a.block_of(slot), base = blk * a.bs, lo = slot - base;
    const int64_t scale_at = (int64_t)blk * a.hkv + h;
    uint4 held[N][kWavePasses];
    int old[N];
#pragma unroll
    for (int x = 0; x < N; ++x) {
#pragma unroll
      for (int p = 0; p < kWavePasses; ++p) {
        const int k = p * kWaveRows + r;
        held[x][p] = make_uint4(0, 0, 0, 0);
        if (p * kWaveRows < len && live && k < len) held[x][p] = load8<VEC>(src(x, t + k));
      }
      old[x] = live ? a.scale[x][scale_at] : 0;
    }
    auto mine = [&](int s) { return (uint32_t)s - (uint32_t)base < (uint32_t)a.bs; };
    int count = 0;                       // the block's tokens that this wave sees
    if (a.tokens <= kThreads) count = __popcll(__ballot(mine(own)));
    else scan(a, [&](int s) { count += __popcll(__ballot(mine(s))); });
    if (lane == 0) atomicAdd(&run_count[i], count);
    __syncthreads();
    const bool whole = __builtin_amdgcn_readfirstlane(run_count[i]) == len;
    if (!whole) {                        // list the block's tokens
      if (tid < a.bs) last[tid] = -1;
      __syncthreads();
      int earlier = 0;
      for (int k = tid; k < a.tokens; k += kThreads) {
        const int s = a.slots[k];
        if (!mine(s)) continue;
        earlier |= k < t;
        atomicMax(&last[s - base], k);
      }
      if (__syncthreads_or(earlier)) continue;     // another token leads the block
#pragma unroll
      for (int p = 0; p < kWavePasses; ++p) {
        const int off = p * kWaveRows + r, tok = off < a.bs ? last[off] : -1;
#pragma unroll
        for (int x = 0; x < N; ++x) {
          held[x][p] = make_uint4(0, 0, 0, 0);
          if (live && tok >= 0) held[x][p] = load8<VEC>(src(x, tok));
        }
      }
    }
    // (pass p holds row lo + p kWaveRows + r of a whole run, else the block's
    // row p kWaveRows + r)
    const int first = whole ? lo : 0;
    auto written = [&](int off) { return whole ? off >= lo && off < lo + len : last[off] >= 0; };
    const bool anew = written(0);
#pragma unroll
    for (int x = 0; x < N; ++x) {
      if (!live) break;
      uint32_t m = 0;
#pragma unroll
      for (int p = 0; p < kWavePasses; ++p)
        if (!whole || p * kWaveRows < len) m = amax8(held[x][p], m);
      const int e = new_exp(anew, old[x], wave_amax(m));
      const float f = __builtin_ldexpf(1.f, 127 - e);
      uint8_t* cache = a.cache[x] + (int64_t)base * row + h * D;
#pragma unroll
      for (int p = 0; p < kWavePasses; ++p) {
        const int off = first + p * kWaveRows + r;
        if ((!whole || p * kWaveRows < len) && off < a.bs && written(off)) store8(cache + off * row + 8 * c, held[x][p], f);
      }
      if (e == old[x]) continue;
      if (lane == 0) a.scale[x][scale_at] = (uint8_t)e;
      if (!anew) rescale_rest(cache, row, a.bs, e - old[x], lane / kLanes8, 64 / kLanes8, lane % kLanes8, written);
    }
    if (!whole) __syncthreads();         // the list is read no more
  }
}

}  // namespace

extern "C" int aia_kv_write_fp8(const void* key, int64_t key_token_stride, const void* value,
                                int64_t value_token_stride, void* key_cache, void* value_cache,
                                void* key_scale, void* value_scale, const int32_t* slot_mapping,
                                int32_t num_tokens, int32_t num_kv_heads, int32_t head_dim,
                                int32_t block_size, int64_t num_slots, void* stream) {
  using namespace aia;
  if (num_tokens < 0 || num_kv_heads <= 0 || block_size <= 0 || num_slots < 0 ||
      num_slots % block_size || num_slots > INT32_MAX)
    return fail(AIA_ERR_INVALID, "aia_kv_write_fp8: bad sizes (tokens %d, heads %d, block %d, slots %lld)",
                num_tokens, num_kv_heads, block_size, (long long)num_slots);
  if (head_dim != 128 && head_dim != 64)
    return fail(AIA_ERR_UNSUPPORTED, "aia_kv_write_fp8: head_dim %d (128 or 64)", head_dim);
  if (block_size > kMaxBlock)
    return fail(AIA_ERR_UNSUPPORTED, "aia_kv_write_fp8: block_size %d (at most %d)", block_size, kMaxBlock);
  if (num_kv_heads > 65535)
    return fail(AIA_ERR_UNSUPPORTED, "aia_kv_write_fp8: %d KV heads (at most 65535)", num_kv_heads);
  if (num_tokens == 0) return AIA_OK;
  const bool has_v = value != nullptr;
  if (!key || !key_cache || !key_scale || !slot_mapping)
    return fail(AIA_ERR_INVALID, "aia_kv_write_fp8: null key/key_cache/key_scale/slot_mapping");
  if (has_v != (value_cache != nullptr) || has_v != (value_scale != nullptr))
    return fail(AIA_ERR_INVALID, "aia_kv_write_fp8: value, value_cache and value_scale must all be set or all NULL");
  const int64_t row = (int64_t)num_kv_heads * head_dim;
  if (key_token_stride < row || (has_v && value_token_stride < row))
    return fail(AIA_ERR_INVALID, "aia_kv_write_fp8: token stride smaller than the row");
  auto aligned = [](const void* p) { return ((uintptr_t)p & 15u) == 0; };
  if (!aligned(key_cache) || !aligned(value_cache))
    return fail(AIA_ERR_INVALID, "aia_kv_write_fp8: caches must be 16-byte aligned");
  Args a;
  a.src[0] = static_cast<const uint16_t*>(key); a.src[1] = static_cast<const uint16_t*>(value);
  a.ts[0] = key_token_stride; a.ts[1] = value_token_stride;
  a.cache[0] = static_cast<uint8_t*>(key_cache); a.cache[1] = static_cast<uint8_t*>(value_cache);
  a.scale[0] = static_cast<uint8_t*>(key_scale); a.scale[1] = static_cast<uint8_t*>(value_scale);
  a.slots = slot_mapping;
  a.tokens = num_tokens; a.hkv = num_kv_heads; a.bs = block_size; a.num_slots = num_slots;
  // slot / block_size of slots below 2^31 as a multiplication: with l = ceil(log2
  // bs) and p = 31 + l, ceil(2^p / bs) exceeds 2^p / bs by less than bs / bs <=
  // 2^l / bs, which times a slot stays below 2^p / bs.
  uint32_t l = 0;
  while ((1u << l) < (uint32_t)block_size) ++l;
  a.div_mul = (uint32_t)(((1ull << (31 + l)) + block_size - 1) / block_size);
  a.div_shift = l > 0 ? l - 1 : 0;
  const bool small = block_size <= kWavePasses * 64 / (head_dim / 8);
  // Work-groups per window and head (or kWaves heads): one round of them on the
  // chip, so that a decode step's tokens, a run each, spread over many.
  const int groups = small ? (num_kv_heads + kWaves - 1) / kWaves : num_kv_heads;
  const int windows = (num_tokens + kThreads - 1) / kThreads;
  a.sub = std::max(1, std::min({kThreads, num_tokens, (small ? kTargetGroupsSmall : kTargetGroups) / std::max(1, windows * groups)}));
  const dim3 grid((unsigned)windows * (unsigned)a.sub, (unsigned)groups);
  const bool vec = aligned(key) && key_token_stride % 8 == 0 &&
                   (!has_v || (aligned(value) && value_token_stride % 8 == 0));
  const size_t lds = small ? 0 : (size_t)block_size * sizeof(int);
  // row passes kept in registers: all of a block of up to 128 slots (head_dim
  // 128); small blocks' few registers let twice as many work-groups run
  auto pick = [&](auto hold) {
    constexpr int H = decltype(hold)::value;
    if (!has_v)
      return head_dim == 128 ? (vec ? kv_write_fp8_kernel<128, true, H, 1> : kv_write_fp8_kernel<128, false, H, 1>)
                             : (vec ? kv_write_fp8_kernel<64, true, H, 1> : kv_write_fp8_kernel<64, false, H, 1>);
    return head_dim == 128 ? (vec ? kv_write_fp8_kernel<128, true, H, 2> : kv_write_fp8_kernel<128, false, H, 2>)
                           : (vec ? kv_write_fp8_kernel<64, true, H, 2> : kv_write_fp8_kernel<64, false, H, 2>);
  };
  const int passes = (block_size * (head_dim / 8) + kThreads - 1) / kThreads;
  auto pick_small = [&](auto n) {
    constexpr int C = decltype(n)::value;
    return head_dim == 128 ? (vec ? kv_write_fp8_small_kernel<128, true, C> : kv_write_fp8_small_kernel<128, false, C>)
                           : (vec ? kv_write_fp8_small_kernel<64, true, C> : kv_write_fp8_small_kernel<64, false, C>);
  };
  auto* kernel = small         ? (has_v ? pick_small(std::integral_constant<int, 2>{})
                                        : pick_small(std::integral_constant<int, 1>{}))
                 : passes <= 4 ? pick(std::integral_constant<int, 4>{})
                               : pick(std::integral_constant<int, 8>{});
  kernel<<<grid, kThreads, lds, (hipStream_t)stream>>>(a);
  return check_hip(hipGetLastError(), "aia_kv_write_fp8 launch");
}
