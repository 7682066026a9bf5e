// Appending a step's K and V to the paged caches with the position rotation on the
// way: of a packed qkv projection, Q and K heads are normed (optionally) and turned by
// their positions as aia_rope_qk does it, the same bits; turned Q goes to q_out, turned
// K and V to their slots.  One launch reads each row once and writes it once, where
// rotating in place and then scattering moves K and V twice.
//
// bf16 caches: a work-group takes a token and up to 256 / (D / 16) of its rows (Q, K
// and V heads), so that a decode step's rows are all in flight at once; its first lanes
// compute the token's cos / sin into LDS, D / 16 lanes own a row.
// 8-bit caches: all of a block's rows have to be known before any is stored, so the
// work-groups are those of aia_kv_write_fp8 with K rows turned in registers between
// the loads and the scale; further work-groups of the launch turn Q.
//
// A prompt step moves bytes: 8,300 tokens of 28/4 heads in 37 us, 4.7 TB/s.  A decode step
// waits: 16 tokens of 16/8 heads 3.2 us; 128 tokens of 64/8 heads into 8-bit caches 10.9,
// whose scale, old rows and new scale follow from each other.
#include <algorithm>

#include "kv_write_fp8.h"

namespace {

struct AppendArgs {
  const uint16_t* qkv;
  int64_t ts;
  int32_t hq, hkv, rot, bs, nz;
  const int64_t* pos;
  const int64_t* turns;
  float factor, eps;
  const uint16_t* wq;
  const uint16_t* wk;
  uint16_t* q_out;
  int64_t q_ts;
  uint16_t* kc;
  uint16_t* vc;
  const int32_t* slots;
  int64_t num_slots;
};

__device__ __forceinline__ void unpack8(uint4 w, float* v) {
  const uint32_t p[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { v[2 * i] = aia::bf16_lo(p[i]); v[2 * i + 1] = aia::bf16_hi(p[i]); }
}

__device__ __forceinline__ uint4 pack8(const float* v) {
  return make_uint4(aia::pack_bf16x2(v[0], v[1]), aia::pack_bf16x2(v[2], v[3]),
                    aia::pack_bf16x2(v[4], v[5]), aia::pack_bf16x2(v[6], v[7]));
}

// cos and sin of a position times a frequency (a 64-bit fraction of a turn).
__device__ __forceinline__ float2 cos_sin(int64_t pos, int64_t turns, float factor) {
  const uint64_t turn = (uint64_t)pos * (uint64_t)turns;
  const float x = (float)(int32_t)(turn >> 32) * 0x1p-32f;
  return make_float2(__builtin_amdgcn_cosf(x) * factor, __builtin_amdgcn_sinf(x) * factor);
}

// The rows first, first + kRows of token t: Q rows from 0, K rows from hq and, with
// KV, V rows from hq + hkv, to the caches.
template <int D, bool INTER, bool KV>
__device__ __forceinline__ void turn_token(const AppendArgs& a, int t, int part, float2* cs) {
  constexpr int kLanes = D / 16, kRows = kThreads / kLanes;
  const int tid = threadIdx.x;
  const int j = tid % kLanes, h = part * kRows + tid / kLanes;
  const int half = a.rot / 2;
  const int rows = KV ? a.hq + 2 * a.hkv : a.hq;
  const bool live = h < rows;
  const bool turned = j < a.rot / 16;
  const int c0 = INTER ? 2 * j : turned ? j : a.rot / 8 + 2 * (j - a.rot / 16);
  const int c1 = !INTER && turned ? j + a.rot / 16 : c0 + 1;
  const uint16_t* row = a.qkv + (int64_t)t * a.ts + (int64_t)h * D;
  uint4 w0 = make_uint4(0, 0, 0, 0), w1 = w0;
  if (live) {
    w0 = *reinterpret_cast<const uint4*>(row + 8 * c0);
    w1 = *reinterpret_cast<const uint4*>(row + 8 * c1);
  }
  const int slot = KV ? a.slots[t] : 0;
  if (tid < half) cs[tid] = cos_sin(a.pos[t], a.turns[tid], a.factor);
  const bool isq = h < a.hq;
  const uint16_t* wn = isq ? a.wq : a.wk;
  float wt[16];
  if (wn) {
    unpack8(*reinterpret_cast<const uint4*>(wn + 8 * c0), wt);
    unpack8(*reinterpret_cast<const uint4*>(wn + 8 * c1), wt + 8);
  }
  __syncthreads();
  const bool plain = KV && h >= a.hq + a.hkv;        // a V row
  if (!plain) {
    float x[16];
    unpack8(w0, x);
    unpack8(w1, x + 8);
    if (wn) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) ss += x[i] * x[i];
#pragma unroll
      for (int d = kLanes / 2; d >= 1; d >>= 1) ss += __shfl_xor(ss, d, kLanes);
      const float n = 1.0f / __builtin_sqrtf(ss * (1.0f / D) + a.eps);
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = x[i] * n * wt[i];
    }
    if (turned) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 r = cs[8 * j + i];
        const int u = INTER ? 2 * i : i, v = INTER ? 2 * i + 1 : i + 8;
        const float p = x[u], q = x[v];
        x[u] = p * r.x - q * r.y;
        x[v] = q * r.x + p * r.y;
      }
    }
    w0 = pack8(x);
    w1 = pack8(x + 8);
  }
  if (!live) return;
  if (isq) {
    uint16_t* o = a.q_out + (int64_t)t * a.q_ts + (int64_t)h * D;
    *reinterpret_cast<uint4*>(o + 8 * c0) = w0;
    *reinterpret_cast<uint4*>(o + 8 * c1) = w1;
    return;
  }
  if (!KV || slot < 0 || slot >= a.num_slots) return;
  uint4* cache = reinterpret_cast<uint4*>(plain ? a.vc : a.kc);
  const int kh = plain ? h - a.hq - a.hkv : h - a.hq;
  const int64_t row16 = (int64_t)a.hkv * D / 8;          // 16-byte pieces of a token's heads
  const int p0 = kh * (D / 8) + c0, p1 = kh * (D / 8) + c1;
  if (a.nz) {
    // each block (row / 16, block_size, 16): see aia_kv_write_nz
    const int64_t blk = slot / a.bs, off = slot - blk * a.bs;
    uint4* to = cache + blk * a.bs * row16;
    to[((int64_t)(p0 >> 1) * a.bs + off) * 2 + (p0 & 1)] = w0;
    to[((int64_t)(p1 >> 1) * a.bs + off) * 2 + (p1 & 1)] = w1;
  } else {
    cache[slot * row16 + p0] = w0;
    cache[slot * row16 + p1] = w1;
  }
}

template <int D, bool INTER>
__global__ __launch_bounds__(kThreads) void rope_append_kernel(AppendArgs a) {
  __shared__ float2 cs[D / 2];
  turn_token<D, INTER, true>(a, blockIdx.x, blockIdx.y, cs);
}

// K rows normed and turned between the loads of an 8-bit write and its scale.  Lane
// piece c of a row is one of a pair of pieces (c, `other`) that aia_rope_qk gives to
// one lane, the j-th; the row's sum of squares is taken in that order too.
template <int D, bool INTER>
struct TurnedRows {
  const int64_t* pos;
  const int64_t* turns;
  const uint16_t* wk;
  int32_t rot;
  float factor, eps;

  int c, base, j, other;
  bool turned;
  int64_t tn[8];
  float w[8];

  __device__ __forceinline__ int first_of(int i) const {     // the first piece of pair i
    return INTER ? 2 * i : i < rot / 16 ? i : rot / 8 + 2 * (i - rot / 16);
  }
  __device__ __forceinline__ void init(int piece, int lane) {
    c = piece;
    base = lane - c;
    if (INTER || c >= rot / 8) {
      j = INTER ? c / 2 : rot / 16 + (c - rot / 8) / 2;
      // (pairs of pieces that pass through begin at rot / 8, an even piece or an odd one)
      other = INTER ? c ^ 1 : rot / 8 + ((c - rot / 8) ^ 1);
    } else {
      j = c < rot / 16 ? c : c - rot / 16;
      other = c < rot / 16 ? c + rot / 16 : c - rot / 16;
    }
    turned = j < rot / 16;
    if (turned) {
#pragma unroll
      for (int i = 0; i < (INTER ? 4 : 8); ++i) tn[i] = turns[(INTER ? 4 * c : 8 * j) + i];
    }
    if (wk) unpack8(*reinterpret_cast<const uint4*>(wk + 8 * c), w);
  }
  __device__ __forceinline__ uint4 operator()(int x, int64_t t, uint4 in) const {
    if (x) return in;
    float own[8], pair[8];
    unpack8(in, own);
    const int from = base + other;
    const uint4 pw = make_uint4(__shfl(in.x, from), __shfl(in.y, from), __shfl(in.z, from), __shfl(in.w, from));
    unpack8(pw, pair);
    const bool first = c < other;
    if (wk) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) { const float y = first ? own[i] : pair[i]; ss += y * y; }
#pragma unroll
      for (int i = 0; i < 8; ++i) { const float y = first ? pair[i] : own[i]; ss += y * y; }
#pragma unroll
      for (int d = D / 32; d >= 1; d >>= 1) ss += __shfl(ss, base + first_of(j ^ d));
      const float n = 1.0f / __builtin_sqrtf(ss * (1.0f / D) + eps);
#pragma unroll
      for (int i = 0; i < 8; ++i) own[i] = own[i] * n * w[i];
      if (!INTER) {       // the other piece as its lane has it
#pragma unroll
        for (int i = 0; i < 8; ++i) pair[i] = __shfl(own[i], from);
      }
    }
    if (turned) {
      const int64_t at = pos[t];
      if constexpr (INTER) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 r = cos_sin(at, tn[i], factor);
          const float p = own[2 * i], q = own[2 * i + 1];
          own[2 * i] = p * r.x - q * r.y;
          own[2 * i + 1] = q * r.x + p * r.y;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 r = cos_sin(at, tn[i], factor);
          const float p = first ? own[i] : pair[i], q = first ? pair[i] : own[i];
          own[i] = first ? p * r.x - q * r.y : q * r.x + p * r.y;
        }
      }
    }
    return pack8(own);
  }
};

// Work-groups [0, writers) write K and V, the rest turn Q rows.
template <int D, bool INTER, int kHold>
__global__ __launch_bounds__(kThreads, 2) void rope_append_fp8_kernel(AppendArgs a, WriteArgs w, int grid_x, int writers, int parts) {
  __shared__ float2 cs[D / 2];
  const int bid = blockIdx.x;
  if (bid >= writers) {
    turn_token<D, INTER, false>(a, (bid - writers) / parts, (bid - writers) % parts, cs);
    return;
  }
  TurnedRows<D, INTER> rows{a.pos, a.turns, a.wk, a.rot, a.factor, a.eps};
  kv_write_fp8_body<D, true, kHold, 2>(w, rows, grid_x, bid % grid_x, bid / grid_x);
}

template <int D, bool INTER>
__global__ __launch_bounds__(kThreads) void rope_append_fp8_small_kernel(AppendArgs a, WriteArgs w, int grid_x, int writers, int parts) {
  __shared__ float2 cs[D / 2];
  const int bid = blockIdx.x;
  if (bid >= writers) {
    turn_token<D, INTER, false>(a, (bid - writers) / parts, (bid - writers) % parts, cs);
    return;
  }
  TurnedRows<D, INTER> rows{a.pos, a.turns, a.wk, a.rot, a.factor, a.eps};
  kv_write_fp8_small_body<D, true, 2>(w, rows, grid_x, bid % grid_x, bid / grid_x);
}

}  // namespace

extern "C" int aia_rope_append(const void* qkv, int64_t qkv_token_stride, int32_t num_tokens,
                               int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                               const int64_t* positions, const int64_t* turns, int32_t rotary_dim,
                               float factor, int32_t interleaved, const void* q_norm_weight,
                               const void* k_norm_weight, float eps, void* q_out,
                               int64_t q_out_token_stride, void* key_cache, void* value_cache,
                               void* key_scale, void* value_scale, const int32_t* slot_mapping,
                               int32_t block_size, int64_t num_slots, int32_t flags, void* stream) {
  using namespace aia;
  if (head_dim != 128 && head_dim != 64)
    return fail(AIA_ERR_UNSUPPORTED, "aia_rope_append: head_dim %d (128 or 64)", head_dim);
  if (rotary_dim <= 0 || rotary_dim > head_dim || rotary_dim % 16)
    return fail(AIA_ERR_UNSUPPORTED, "aia_rope_append: rotary_dim %d (a multiple of 16 up to head_dim %d)",
                rotary_dim, head_dim);
  if (num_tokens < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads > (1 << 20) ||
      num_kv_heads > 65535 || block_size <= 0 || num_slots < 0 || num_slots % block_size || num_slots > INT32_MAX)
    return fail(AIA_ERR_INVALID, "aia_rope_append: bad sizes (tokens %d, heads %d / %d, block %d, slots %lld)",
                num_tokens, num_q_heads, num_kv_heads, block_size, (long long)num_slots);
  if (flags & ~AIA_ATTN_KV_NZ) return fail(AIA_ERR_INVALID, "aia_rope_append: unknown flags %d", flags);
  if ((q_norm_weight == nullptr) != (k_norm_weight == nullptr))
    return fail(AIA_ERR_INVALID, "aia_rope_append: q and k norm weights go together");
  if ((key_scale == nullptr) != (value_scale == nullptr))
    return fail(AIA_ERR_INVALID, "aia_rope_append: key_scale and value_scale go together");
  if (key_scale && flags) return fail(AIA_ERR_UNSUPPORTED, "aia_rope_append: 8-bit caches have no NZ layout");
  if (key_scale && block_size > kMaxBlock)
    return fail(AIA_ERR_UNSUPPORTED, "aia_rope_append: block_size %d (at most %d in 8-bit caches)", block_size, kMaxBlock);
  if (num_tokens == 0) return AIA_OK;
  if (!qkv || !positions || !turns || !q_out || !key_cache || !value_cache || !slot_mapping)
    return fail(AIA_ERR_INVALID, "aia_rope_append: null pointer argument");
  const int64_t nq = (int64_t)num_q_heads * head_dim, nk = (int64_t)num_kv_heads * head_dim;
  auto aligned = [](const void* p) { return ((uintptr_t)p & 15u) == 0; };
  if (qkv_token_stride < nq + 2 * nk || q_out_token_stride < nq || qkv_token_stride % 8 ||
      q_out_token_stride % 8 || !aligned(qkv) || !aligned(q_out) || !aligned(key_cache) || !aligned(value_cache) ||
      !aligned(q_norm_weight) || !aligned(k_norm_weight))
    return fail(AIA_ERR_INVALID, "aia_rope_append: tensors must be 16-byte aligned with token strides a multiple "
                "of 8 that hold a token's heads");
  // Q rows are read and written by the same lanes; any other overlap with the
  // projection would be read after it was written.
  const uint16_t* in = static_cast<const uint16_t*>(qkv);
  const uint16_t* qo = static_cast<const uint16_t*>(q_out);
  const bool in_place = qo == in && (num_tokens == 1 || q_out_token_stride == qkv_token_stride);
  if (!in_place && qo < in + (num_tokens - 1) * qkv_token_stride + nq + 2 * nk &&
      in < qo + (num_tokens - 1) * q_out_token_stride + nq)
    return fail(AIA_ERR_INVALID, "aia_rope_append: q_out overlaps the qkv rows (in place: q_out = qkv, with its "
                "token stride)");
  AppendArgs a;
  a.qkv = in; a.ts = qkv_token_stride;
  a.hq = num_q_heads; a.hkv = num_kv_heads; a.rot = rotary_dim; a.bs = block_size; a.nz = flags & AIA_ATTN_KV_NZ;
  a.pos = positions; a.turns = turns; a.factor = factor; a.eps = eps;
  a.wq = static_cast<const uint16_t*>(q_norm_weight);
  a.wk = static_cast<const uint16_t*>(k_norm_weight);
  a.q_out = static_cast<uint16_t*>(q_out); a.q_ts = q_out_token_stride;
  a.kc = static_cast<uint16_t*>(key_cache); a.vc = static_cast<uint16_t*>(value_cache);
  a.slots = slot_mapping; a.num_slots = num_slots;
  const int rows_per = kThreads / (head_dim / 16);
  if (!key_scale) {
    const int parts = (num_q_heads + 2 * num_kv_heads + rows_per - 1) / rows_per;
    auto* kernel = head_dim == 128 ? (interleaved ? rope_append_kernel<128, true> : rope_append_kernel<128, false>)
                                   : (interleaved ? rope_append_kernel<64, true> : rope_append_kernel<64, false>);
    kernel<<<dim3((unsigned)num_tokens, (unsigned)parts), kThreads, 0, (hipStream_t)stream>>>(a);
    return check_hip(hipGetLastError(), "aia_rope_append launch");
  }
  WriteArgs w;
  w.src[0] = in + nq; w.src[1] = in + nq + nk;
  w.ts[0] = w.ts[1] = qkv_token_stride;
  w.cache[0] = static_cast<uint8_t*>(key_cache); w.cache[1] = static_cast<uint8_t*>(value_cache);
  w.scale[0] = static_cast<uint8_t*>(key_scale); w.scale[1] = static_cast<uint8_t*>(value_scale);
  w.slots = slot_mapping;
  w.tokens = num_tokens; w.hkv = num_kv_heads; w.bs = block_size; w.num_slots = num_slots;
  set_division(w, block_size);
  const WriteGrid g = cut_write(w, head_dim);
  const int parts = (num_q_heads + rows_per - 1) / rows_per;
  const int64_t writers = (int64_t)g.x * g.y, groups = writers + (int64_t)num_tokens * parts;
  if (groups > INT32_MAX) return fail(AIA_ERR_UNSUPPORTED, "aia_rope_append: too many rows in one call");
  auto pick = [&](auto d, auto inter) {
    constexpr int D = decltype(d)::value;
    constexpr bool I = decltype(inter)::value;
    return g.small         ? rope_append_fp8_small_kernel<D, I>
           : g.passes <= 4 ? rope_append_fp8_kernel<D, I, 4>
                           : rope_append_fp8_kernel<D, I, 8>;
  };
  using d128 = std::integral_constant<int, 128>;
  using d64 = std::integral_constant<int, 64>;
  auto* kernel = head_dim == 128 ? (interleaved ? pick(d128{}, std::true_type{}) : pick(d128{}, std::false_type{}))
                                 : (interleaved ? pick(d64{}, std::true_type{}) : pick(d64{}, std::false_type{}));
  kernel<<<(unsigned)groups, kThreads, g.lds, (hipStream_t)stream>>>(a, w, g.x, (int)writers, parts);
  return check_hip(hipGetLastError(), "aia_rope_append launch");
}
