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
constexpr int kScan = 16;             // slots a thread reads at once in search of a block's tokens
// Work-groups of a long step.  More leave fewer runs to each but more of them
// find none (7,399 ragged tokens, 2 heads of 64, blocks of 16, us: 13.3 at 1024,
// 11.3 at 2048, 11.9 at 3072; 16,384 prompt tokens, 8 heads of 128, blocks of
// 128: 34.1, 34.3, 36.5).
constexpr int kTargetGroups = 2048;
constexpr int kMaxBlock = 8192;       // slots of a block: its tokens are listed in LDS
constexpr int kMinExp = -100;

struct Args {
  const uint16_t* src[2];             // K, V rows
  int64_t ts[2];
  uint8_t* cache[2];
  uint8_t* scale[2];
  const int32_t* slots;
  int32_t tokens, hkv, bs, sub;
  int64_t num_slots;
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

// Grid: (sub x windows of kThreads tokens, heads of K and V).  A window's runs
// (tokens at consecutive slots of one block) are found by two loads per
// thread, this window's and the next one's slots; work-group s of a window
// takes its runs s, s + sub, ...  A run's rows and its block's scale are loaded
// at once, speculating that the run is all the block gets in this call, while
// all slots are scanned to count the block's tokens: a count equal to the run's
// length confirms it, and the block is done after one barrier.  Otherwise the
// general path lists the block's tokens in LDS.
// K and V of a head share the scan.  Measured, us, for 16 decode rows (8 heads of
// 128, blocks of 16), 16,384 prompt tokens (8 heads of 128, blocks of 128) and
// 7,399 ragged tokens (2 heads of 64, blocks of 16): every token listed in LDS
// and all loads dependent 8.7 / 32.1 / 21.7; speculating, K and V apart 4.0 /
// 34.4 / 15.9; together 4.2 / 33.3 / 11.3, of which the scan is - / 4.9 / 1.9.  The
// prompt's bytes move at 3.0 TB/s (a large copy: 5.1): every block's loads are
// over before its stores begin, and the blocks run side by side.  Four heads per
// work-group (one scan for all): 8.0 / 32.9 / 11.9.
template <int D, bool VEC, int kHold, int N>
__global__ __launch_bounds__(kThreads, 4) void kv_write_fp8_kernel(Args a) {
  constexpr int kLanes = D / 8, kRows = kThreads / kLanes;       // threads per new row, rows per pass
  constexpr int kLanes8 = D / 16, kRows8 = kThreads / kLanes8;   // of 16-byte cached pieces
  extern __shared__ int last[];          // general path: a slot's last token, -1 = none
  __shared__ uint64_t starts[kWaves];    // tokens of the window that start a run
  __shared__ uint64_t joins[2 * kWaves]; // tokens of the window and the next that continue one
  __shared__ int slots[kThreads];
  __shared__ int wave_count[kWaves], wave_lo[kWaves], wave_hi[kWaves];
  __shared__ uint32_t wave_max[N][kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int h = blockIdx.y;
  const int64_t row = (int64_t)a.hkv * D;
  auto src = [&](int x, int64_t t) { return a.src[x] + t * a.ts[x] + h * D + 8 * (tid % kLanes); };
  // (work-groups of one sub index are neighbours, so those that find no run do
  // not fall on the same XCDs)
  const int windows = gridDim.x / a.sub, sub = blockIdx.x / windows, window = blockIdx.x - sub * windows;
  const int t0 = window * kThreads;
  auto slot_at = [&](int t) { return t >= 0 && t < a.tokens ? a.slots[t] : -1; };
  const int own = slot_at(t0 + tid);                        // this thread's token's slot
  {
    const int before = slot_at(t0 + tid - 1);
    const int next = slot_at(t0 + kThreads + tid), before_next = slot_at(t0 + kThreads + tid - 1);
    // (a slot that follows its predecessor's is in the same block unless it
    // is a block's first; a predecessor that is skipped is followed by none)
    auto follows = [&](int s, int b) { return s == b + 1 && b >= 0 && s < a.num_slots && s % a.bs != 0; };
    const bool join = follows(own, before), join_next = follows(next, before_next);
    const uint64_t s = __ballot(own >= 0 && own < a.num_slots && !join);
    const uint64_t j = __ballot(join), k = __ballot(join_next);
    if (lane == 0) { starts[wid] = s; joins[wid] = j; joins[kWaves + wid] = k; }
    slots[tid] = own;
  }
  __syncthreads();
  const int r = tid / kLanes;
  bool again = false;
  int skip = sub;                        // runs of others before this work-group's next one
  int w = 0;
  uint64_t left = uniform64(starts[0]);
  while (true) {
    const int here = __popcll(left);
    if (skip >= here) {
      if (++w == kWaves) return;
      skip -= here;
      left = uniform64(starts[w]);
      continue;
    }
    for (; skip > 0; --skip) left &= left - 1;
    const int bit = __builtin_ctzll(left);
    left &= left - 1;
    skip = a.sub - 1;
    if (again) __syncthreads();          // the previous block's LDS is read no more
    again = true;
    const int t = t0 + 64 * w + bit;
    const int slot = __builtin_amdgcn_readfirstlane(slots[64 * w + bit]);
    const int blk = slot / a.bs, base = blk * a.bs;
    int run = 1;                         // tokens of the run, as far as the two windows show
    for (int v = w, from = bit + 1; v < 2 * kWaves; ++v, from = 0) {
      if (from == 64) continue;
      const uint64_t stop = ~uniform64(joins[v]) >> from;
      if (stop) { run += __builtin_ctzll(stop); break; }
      run += 64 - from;
    }
    uint4 held[N][kHold];
    int old[N];
#pragma unroll
    for (int x = 0; x < N; ++x) {
#pragma unroll
      for (int p = 0; p < kHold; ++p) {
        held[x][p] = make_uint4(0, 0, 0, 0);
        if (p * kRows + r < run) held[x][p] = load8<VEC>(src(x, t + p * kRows + r));
      }
    }
    const int64_t scale_at = (int64_t)blk * a.hkv + h;
#pragma unroll
    for (int x = 0; x < N; ++x) old[x] = a.scale[x][scale_at];
    auto mine = [&](int s) { return (uint32_t)s - (uint32_t)base < (uint32_t)a.bs; };
    int count = 0;                       // the block's tokens that this wave sees
    if (a.tokens <= kThreads) {
      count = __popcll(__ballot(mine(own)));
    } else {
      int first = 0;
      for (; first + kThreads * kScan <= a.tokens; first += kThreads * kScan) {
        int s[kScan];
#pragma unroll
        for (int i = 0; i < kScan; ++i) s[i] = a.slots[first + kThreads * i + tid];
#pragma unroll
        for (int i = 0; i < kScan; ++i) count += __popcll(__ballot(mine(s[i])));
      }
      int s[kScan];
#pragma unroll
      for (int i = 0; i < kScan; ++i) {
        const int at = first + kThreads * i + tid;
        s[i] = at < a.tokens ? a.slots[at] : -1;
      }
#pragma unroll
      for (int i = 0; i < kScan; ++i) count += __popcll(__ballot(mine(s[i])));
    }
    uint32_t m[N];
    auto wave_amax = [&](uint32_t v) {
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) v = max(v, (uint32_t)__shfl_xor((int)v, d));
      return v;
    };
#pragma unroll
    for (int x = 0; x < N; ++x) {
      m[x] = 0;
#pragma unroll
      for (int p = 0; p < kHold; ++p) m[x] = amax8(held[x][p], m[x]);
      for (int k = kHold * kRows + r; k < run; k += kRows) m[x] = amax8(load8<VEC>(src(x, t + k)), m[x]);
      m[x] = wave_amax(m[x]);
      if (lane == 0) wave_max[x][wid] = m[x];
    }
    if (lane == 0) wave_count[wid] = count;
    __syncthreads();
    count = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      count += wave_count[i];
#pragma unroll
      for (int x = 0; x < N; ++x) m[x] = max(m[x], wave_max[x][i]);
    }
    const bool whole = count == run;     // the run is all the block gets
    int lo = slot - base, hi = lo + run - 1;
    if (!whole) {
      for (int i = tid; i < a.bs; i += kThreads) last[i] = -1;
      __syncthreads();
      int earlier = 0;
      lo = a.bs;
      hi = -1;
      for (int i = tid; i < a.tokens; i += kThreads) {
        const int s = a.slots[i];
        if (!mine(s)) continue;
        earlier |= i < t;
        atomicMax(&last[s - base], i);
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
      for (int i = 0; i < kWaves; ++i) { lo = min(lo, wave_lo[i]); hi = max(hi, wave_hi[i]); }
      for (int off = lo + r; off <= hi; off += kRows) {
        if (last[off] < 0) continue;
#pragma unroll
        for (int x = 0; x < N; ++x) m[x] = amax8(load8<VEC>(src(x, last[off])), m[x]);
      }
#pragma unroll
      for (int x = 0; x < N; ++x) {
        m[x] = wave_amax(m[x]);
        if (lane == 0) wave_max[x][wid] = m[x];
      }
      __syncthreads();
#pragma unroll
      for (int x = 0; x < N; ++x)
#pragma unroll
        for (int i = 0; i < kWaves; ++i) m[x] = max(m[x], wave_max[x][i]);
    }
    const bool anew = lo == 0;           // the block's first slot is written
#pragma unroll
    for (int x = 0; x < N; ++x) {
      const int need = needed_byte(m[x]);
      const int e = anew ? need : max(old[x], need);
      const float f = __builtin_ldexpf(1.f, 127 - e);
      uint8_t* cache = a.cache[x] + (int64_t)base * row + h * D;
      auto store = [&](int off, uint4 v) {
        *reinterpret_cast<uint2*>(cache + off * row + 8 * (tid % kLanes)) = quantise8(v, f);
      };
      if (whole) {
#pragma unroll
        for (int p = 0; p < kHold; ++p)
          if (p * kRows + r < run) store(lo + p * kRows + r, held[x][p]);
        for (int k = kHold * kRows + r; k < run; k += kRows) store(lo + k, load8<VEC>(src(x, t + k)));
      } else {
        for (int off = lo + r; off <= hi; off += kRows)
          if (last[off] >= 0) store(off, load8<VEC>(src(x, last[off])));
      }
      if (e == old[x]) continue;
      if (tid == 0) a.scale[x][scale_at] = (uint8_t)e;
      if (anew) continue;
      for (int off = tid / kLanes8; off < a.bs; off += kRows8) {
        if (whole ? off >= lo && off <= hi : last[off] >= 0) continue;
        uint4* p = reinterpret_cast<uint4*>(cache + off * row) + tid % kLanes8;
        const uint4 v = *p;
        *p = make_uint4(rescale4(v.x, e - old[x]), rescale4(v.y, e - old[x]), rescale4(v.z, e - old[x]),
                        rescale4(v.w, e - old[x]));
      }
    }
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
  // Work-groups per window and head: one round of them on the chip, so that a
  // decode step's tokens, a run each, spread over many.
  const int windows = (num_tokens + kThreads - 1) / kThreads;
  a.sub = std::max(1, std::min({kThreads, num_tokens, kTargetGroups / std::max(1, windows * num_kv_heads)}));
  const dim3 grid((unsigned)windows * (unsigned)a.sub, (unsigned)num_kv_heads);
  const bool vec = aligned(key) && key_token_stride % 8 == 0 &&
                   (!has_v || (aligned(value) && value_token_stride % 8 == 0));
  const size_t lds = (size_t)block_size * sizeof(int);
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
  auto* kernel = passes <= 1 ? pick(std::integral_constant<int, 1>{})
                 : passes <= 4 ? pick(std::integral_constant<int, 4>{})
                               : pick(std::integral_constant<int, 8>{});
  kernel<<<grid, kThreads, lds, (hipStream_t)stream>>>(a);
  return check_hip(hipGetLastError(), "aia_kv_write_fp8 launch");
}
