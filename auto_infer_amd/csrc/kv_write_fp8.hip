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
// that of the call's first token in the block (its leader, found by scanning
// the slots), which collects the block's tokens in LDS (the highest token of a
// slot stays), loads their rows once, reduces amax and stores.
#include "common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kHold = 8;              // row passes kept in registers
constexpr int kMaxBlock = 8192;       // slots of a block: its tokens are listed in LDS
constexpr int kMinExp = -100;

struct Args {
  const uint16_t* src[2];             // K, V rows
  int64_t ts[2];
  uint8_t* cache[2];
  uint8_t* scale[2];
  const int32_t* slots;
  int32_t tokens, hkv, bs, window;
  int64_t num_slots;
};

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

template <int D, bool VEC>
__global__ __launch_bounds__(kThreads) void kv_write_fp8_kernel(Args a) {
  constexpr int kLanes = D / 8, kRows = kThreads / kLanes;       // threads per new row, rows per pass
  constexpr int kLanes8 = D / 16, kRows8 = kThreads / kLanes8;   // of 16-byte cached pieces
  extern __shared__ int last[];          // per slot of the block: its last token, -1 = none
  __shared__ int span[2];                // first and last slot written
  __shared__ uint32_t wave_max[kThreads / 64];
  const int tid = threadIdx.x;
  const int which = blockIdx.y / a.hkv, h = blockIdx.y - which * a.hkv;
  const uint16_t* src = a.src[which] + (int64_t)h * D;
  uint8_t* cache = a.cache[which] + (int64_t)h * D;
  const int64_t ts = a.ts[which];
  const int64_t row = (int64_t)a.hkv * D;
  const int t0 = blockIdx.x * a.window, t1 = min(a.tokens, t0 + a.window);
  for (int t = t0; t < t1; ++t) {
    const int slot = a.slots[t];
    if (slot < 0 || slot >= a.num_slots) continue;
    const int blk = slot / a.bs, base = blk * a.bs;
    // a token behind one of its own block is no leader: no scan for it
    if (t > 0 && (uint32_t)a.slots[t - 1] - (uint32_t)base < (uint32_t)a.bs) continue;
    __syncthreads();                     // the previous block's LDS is read no more
    for (int i = tid; i < a.bs; i += kThreads) last[i] = -1;
    if (tid == 0) { span[0] = a.bs; span[1] = -1; }
    __syncthreads();
    int earlier = 0;
    for (int i = tid; i < a.tokens; i += kThreads) {
      const uint32_t off = (uint32_t)a.slots[i] - (uint32_t)base;
      if (off < (uint32_t)a.bs) {
        earlier |= i < t;
        atomicMax(&last[off], i);
        atomicMin(&span[0], (int)off);
        atomicMax(&span[1], (int)off);
      }
    }
    if (__syncthreads_or(earlier)) continue;
    const int lo = span[0], hi = span[1];
    const int passes = (hi - lo) / kRows + 1;
    const int r = tid / kLanes, c = tid % kLanes;
    auto token = [&](int p) {
      const int off = lo + p * kRows + r;
      return off <= hi ? last[off] : -1;
    };
    uint4 held[kHold];
    uint32_t m = 0;
#pragma unroll
    for (int p = 0; p < kHold; ++p) {
      held[p] = make_uint4(0, 0, 0, 0);
      if (p < passes) {
        const int tok = token(p);
        if (tok >= 0) held[p] = load8<VEC>(src + tok * ts + 8 * c);
        m = amax8(held[p], m);
      }
    }
    for (int p = kHold; p < passes; ++p) {
      const int tok = token(p);
      if (tok >= 0) m = amax8(load8<VEC>(src + tok * ts + 8 * c), m);
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d));
    if ((tid & 63) == 0) wave_max[tid >> 6] = m;
    uint8_t* scale = a.scale[which] + (int64_t)blk * a.hkv + h;
    const int old = *scale;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kThreads / 64; ++i) m = max(m, wave_max[i]);
    const bool anew = lo == 0;           // the block's first slot is written
    const int need = needed_byte(m);
    const int e = anew ? need : max(old, need);
    const float f = __builtin_ldexpf(1.f, 127 - e);
    auto store = [&](int p, uint4 v) {
      const int64_t at = (int64_t)(base + lo + p * kRows + r) * row + 8 * c;
      *reinterpret_cast<uint2*>(cache + at) = quantise8(v, f);
    };
#pragma unroll
    for (int p = 0; p < kHold; ++p)
      if (p < passes && token(p) >= 0) store(p, held[p]);
    for (int p = kHold; p < passes; ++p) {
      const int tok = token(p);
      if (tok >= 0) store(p, load8<VEC>(src + tok * ts + 8 * c));
    }
    if (e == old && !anew) continue;
    if (tid == 0) *scale = (uint8_t)e;
    if (anew) continue;
    for (int off = tid / kLanes8; off < a.bs; off += kRows8) {
      if (last[off] >= 0) continue;
      uint4* p = reinterpret_cast<uint4*>(cache + (int64_t)(base + off) * row) + tid % kLanes8;
      const uint4 v = *p;
      *p = make_uint4(rescale4(v.x, e - old), rescale4(v.y, e - old), rescale4(v.z, e - old),
                      rescale4(v.w, e - old));
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
  if (num_kv_heads > 32767)
    return fail(AIA_ERR_UNSUPPORTED, "aia_kv_write_fp8: %d KV heads (at most 32767)", num_kv_heads);
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
  // tokens a work-group looks over for leaders: one in short steps (every
  // decode row leads its block), more where most tokens lead nothing
  const int heads = num_kv_heads * (has_v ? 2 : 1);
  a.window = 1;
  while (a.window < 16 && (int64_t)num_tokens * heads > 8192LL * a.window) a.window *= 2;
  const dim3 grid((unsigned)((num_tokens + a.window - 1) / a.window), (unsigned)heads);
  const bool vec = aligned(key) && key_token_stride % 8 == 0 &&
                   (!has_v || (aligned(value) && value_token_stride % 8 == 0));
  const size_t lds = (size_t)block_size * sizeof(int);
  auto* kernel = head_dim == 128 ? (vec ? kv_write_fp8_kernel<128, true> : kv_write_fp8_kernel<128, false>)
                                 : (vec ? kv_write_fp8_kernel<64, true> : kv_write_fp8_kernel<64, false>);
  kernel<<<grid, kThreads, lds, (hipStream_t)stream>>>(a);
  return check_hip(hipGetLastError(), "aia_kv_write_fp8 launch");
}
