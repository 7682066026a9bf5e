// KV slot write into 8-bit caches: rows as they are in memory.
#include "kv_write_fp8.h"

namespace {

template <int D, bool VEC, int kHold, int N>
__global__ __launch_bounds__(kThreads, 4) void kv_write_fp8_kernel(WriteArgs a) {
  kv_write_fp8_body<D, VEC, kHold, N>(a, PlainRows{}, gridDim.x, blockIdx.x, blockIdx.y);
}

template <int D, bool VEC, int N>
__global__ __launch_bounds__(kThreads) void kv_write_fp8_small_kernel(WriteArgs a) {
  kv_write_fp8_small_body<D, VEC, N>(a, PlainRows{}, gridDim.x, blockIdx.x, blockIdx.y);
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
  WriteArgs a;
  a.src[0] = static_cast<const uint16_t*>(key); a.src[1] = static_cast<const uint16_t*>(value);
  a.ts[0] = key_token_stride; a.ts[1] = value_token_stride;
  a.cache[0] = static_cast<uint8_t*>(key_cache); a.cache[1] = static_cast<uint8_t*>(value_cache);
  a.scale[0] = static_cast<uint8_t*>(key_scale); a.scale[1] = static_cast<uint8_t*>(value_scale);
  a.slots = slot_mapping;
  a.tokens = num_tokens; a.hkv = num_kv_heads; a.bs = block_size; a.num_slots = num_slots;
  set_division(a, block_size);
  const WriteGrid g = cut_write(a, head_dim);
  const bool vec = aligned(key) && key_token_stride % 8 == 0 &&
                   (!has_v || (aligned(value) && value_token_stride % 8 == 0));
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
  auto pick_small = [&](auto n) {
    constexpr int C = decltype(n)::value;
    return head_dim == 128 ? (vec ? kv_write_fp8_small_kernel<128, true, C> : kv_write_fp8_small_kernel<128, false, C>)
                           : (vec ? kv_write_fp8_small_kernel<64, true, C> : kv_write_fp8_small_kernel<64, false, C>);
  };
  auto* kernel = g.small         ? (has_v ? pick_small(std::integral_constant<int, 2>{})
                                        : pick_small(std::integral_constant<int, 1>{}))
                 : g.passes <= 4 ? pick(std::integral_constant<int, 4>{})
                               : pick(std::integral_constant<int, 8>{});
  kernel<<<dim3((unsigned)g.x, (unsigned)g.y), kThreads, g.lds, (hipStream_t)stream>>>(a);
  return check_hip(hipGetLastError(), "aia_kv_write_fp8 launch");
}
