// Rotary positions of a packed qkv projection from the positions themselves,
// with an optional per-head RMSNorm in front: pair i of a head's rotated part
// turns by position * freq_i; the rest of the head passes through.
//
// Angles of far positions: freq_i comes as a 64-bit fraction of a turn, so
// position * freq_i modulo one turn is one wrapping 64-bit product, exact to
// 2^-64 turns per position, at any (also negative) position.  The top 32 bits
// go to v_sin / v_cos, which take turns.
//
// A work-group takes one token: its first lanes compute the token's cos / sin
// once into LDS, then D / 16 lanes own one (token, head) row, two 8-value
// chunks each: chunks j and j + rotary / 16 of the rotated part in the
// half-split layout (pair i = dims i and i + rotary / 2), two neighbouring
// ones otherwise (pair i = dims 2 i and 2 i + 1, or dims that pass through), so
// a pair never crosses lanes.  Everything is fp32 until one rounding at the
// end.
//
// Bound by memory: each row is read and written once.  8,192 tokens of 28/4
// heads of 128, half of each head turned, into other tensors: 28.1 us on the
// GPU, 4.8 TB/s (a large copy: 5.1).  16 tokens: 3.2 us, a launch and one memory round trip.
#include <algorithm>

#include "common.h"

namespace {

constexpr int kThreads = 256;

struct Args {
  const uint16_t* qkv;
  int64_t ts;
  int32_t hq, hkv, rot;
  const int64_t* pos;
  const int64_t* turns;
  float factor, eps;
  const uint16_t* wq;
  const uint16_t* wk;
  uint16_t* q_out;
  int64_t q_ts;
  uint16_t* k_out;
  int64_t k_ts;
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

template <int D, bool INTER>
__global__ __launch_bounds__(kThreads) void rope_qk_kernel(Args a) {
  constexpr int kLanes = D / 16, kRows = kThreads / kLanes;
  __shared__ float2 cs[D / 2];
  const int t = blockIdx.x, tid = threadIdx.x;
  const int j = tid % kLanes, slot = tid / kLanes;
  const int half = a.rot / 2;
  if (tid < half) {
    const uint64_t turn = (uint64_t)a.pos[t] * (uint64_t)a.turns[tid];
    const float x = (float)(int32_t)(turn >> 32) * 0x1p-32f;
    cs[tid] = make_float2(__builtin_amdgcn_cosf(x) * a.factor, __builtin_amdgcn_sinf(x) * a.factor);
  }
  const bool turned = j < a.rot / 16;
  const int c0 = INTER ? 2 * j : turned ? j : a.rot / 8 + 2 * (j - a.rot / 16);
  const int c1 = !INTER && turned ? j + a.rot / 16 : c0 + 1;
  float wq[16], wk[16];
  if (a.wq) {
    unpack8(*reinterpret_cast<const uint4*>(a.wq + 8 * c0), wq);
    unpack8(*reinterpret_cast<const uint4*>(a.wq + 8 * c1), wq + 8);
    unpack8(*reinterpret_cast<const uint4*>(a.wk + 8 * c0), wk);
    unpack8(*reinterpret_cast<const uint4*>(a.wk + 8 * c1), wk + 8);
  }
  __syncthreads();
  float2 r[8];
  if (turned) {
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = cs[8 * j + i];
  }
  const uint16_t* row = a.qkv + t * a.ts;
  for (int h = slot; h < a.hq + a.hkv; h += kRows) {
    const bool isq = h < a.hq;
    float x[16];
    unpack8(*reinterpret_cast<const uint4*>(row + h * D + 8 * c0), x);
    unpack8(*reinterpret_cast<const uint4*>(row + h * D + 8 * c1), x + 8);
    if (a.wq) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) ss += x[i] * x[i];
#pragma unroll
      for (int d = kLanes / 2; d >= 1; d >>= 1) ss += __shfl_xor(ss, d, kLanes);
      const float n = 1.0f / __builtin_sqrtf(ss * (1.0f / D) + a.eps);
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = x[i] * n * (isq ? wq[i] : wk[i]);
    }
    if (turned) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int u = INTER ? 2 * i : i, v = INTER ? 2 * i + 1 : i + 8;
        const float p = x[u], q = x[v];
        x[u] = p * r[i].x - q * r[i].y;
        x[v] = q * r[i].x + p * r[i].y;
      }
    }
    uint16_t* o = isq ? a.q_out + t * a.q_ts + h * D : a.k_out + t * a.k_ts + (h - a.hq) * D;
    *reinterpret_cast<uint4*>(o + 8 * c0) = pack8(x);
    *reinterpret_cast<uint4*>(o + 8 * c1) = pack8(x + 8);
  }
}

// Rows of a token (16-bit elements) in memory.
struct Rows {
  const void* at;
  int64_t len, stride;
};

// Whether the rows of n tokens share memory.  Rows of one stride may interleave
// (columns of one wider tensor): with d the distance modulo the stride, [0, len)
// and [d, d + other len) must not meet.  Rows of different strides whose spans
// meet count as sharing.
bool share_memory(const Rows& a, const Rows& b, int64_t n) {
  const int64_t a0 = (int64_t)((uintptr_t)a.at / 2), b0 = (int64_t)((uintptr_t)b.at / 2);
  if (a0 >= b0 + (n - 1) * b.stride + b.len || b0 >= a0 + (n - 1) * a.stride + a.len) return false;
  if (n == 1 || a.stride != b.stride) return true;
  const int64_t d = ((b0 - a0) % a.stride + a.stride) % a.stride;
  return d < a.len || d + b.len > a.stride;
}

}  // namespace

extern "C" int aia_rope_qk(const void* qkv, int64_t qkv_token_stride, int32_t num_tokens,
                           int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                           const int64_t* positions, const int64_t* turns, int32_t rotary_dim,
                           float factor, int32_t interleaved, const void* q_norm_weight,
                           const void* k_norm_weight, float eps, void* q_out,
                           int64_t q_out_token_stride, void* k_out, int64_t k_out_token_stride,
                           void* stream) {
  using namespace aia;
  if (head_dim != 128 && head_dim != 64)
    return fail(AIA_ERR_UNSUPPORTED, "aia_rope_qk: head_dim %d (128 or 64)", head_dim);
  if (rotary_dim <= 0 || rotary_dim > head_dim || rotary_dim % 16)
    return fail(AIA_ERR_UNSUPPORTED, "aia_rope_qk: rotary_dim %d (a multiple of 16 up to head_dim %d)",
                rotary_dim, head_dim);
  if (num_tokens < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads > (1 << 20) ||
      num_kv_heads > (1 << 20))
    return fail(AIA_ERR_INVALID, "aia_rope_qk: bad sizes (tokens %d, heads %d / %d)", num_tokens,
                num_q_heads, num_kv_heads);
  if ((q_norm_weight == nullptr) != (k_norm_weight == nullptr))
    return fail(AIA_ERR_INVALID, "aia_rope_qk: q and k norm weights go together");
  if (num_tokens == 0) return AIA_OK;
  if (!qkv || !positions || !turns || !q_out || !k_out)
    return fail(AIA_ERR_INVALID, "aia_rope_qk: null pointer argument");
  if (qkv_token_stride < (int64_t)(num_q_heads + num_kv_heads) * head_dim ||
      q_out_token_stride < (int64_t)num_q_heads * head_dim ||
      k_out_token_stride < (int64_t)num_kv_heads * head_dim || qkv_token_stride % 8 ||
      q_out_token_stride % 8 || k_out_token_stride % 8 || ((uintptr_t)qkv & 15) ||
      ((uintptr_t)q_out & 15) || ((uintptr_t)k_out & 15) || ((uintptr_t)q_norm_weight & 15) ||
      ((uintptr_t)k_norm_weight & 15))
    return fail(AIA_ERR_INVALID, "aia_rope_qk: tensors must be 16-byte aligned with token strides a "
                "multiple of 8 that hold a token's heads");
  // A row is read and written by the same lanes, so the qkv rows themselves may
  // be the outputs; any other overlap would be read after it was written.
  const int64_t nq = (int64_t)num_q_heads * head_dim, nk = (int64_t)num_kv_heads * head_dim;
  const Rows in{qkv, num_tokens > 1 ? std::min(qkv_token_stride, nq + 2 * nk) : nq + 2 * nk, qkv_token_stride};
  const Rows qo{q_out, nq, q_out_token_stride}, ko{k_out, nk, k_out_token_stride};
  auto in_place = [&](const Rows& o, int64_t col) {
    return o.at == static_cast<const uint16_t*>(qkv) + col && (num_tokens == 1 || o.stride == qkv_token_stride);
  };
  if ((!in_place(qo, 0) && share_memory(qo, in, num_tokens)) ||
      (!in_place(ko, nq) && share_memory(ko, in, num_tokens)) || share_memory(qo, ko, num_tokens))
    return fail(AIA_ERR_INVALID, "aia_rope_qk: the outputs overlap the qkv rows or each other (in place: q_out = "
                "qkv, k_out = qkv + Hq * D, with its token stride)");
  Args a;
  a.qkv = static_cast<const uint16_t*>(qkv); a.ts = qkv_token_stride;
  a.hq = num_q_heads; a.hkv = num_kv_heads; a.rot = rotary_dim;
  a.pos = positions; a.turns = turns; a.factor = factor; a.eps = eps;
  a.wq = static_cast<const uint16_t*>(q_norm_weight);
  a.wk = static_cast<const uint16_t*>(k_norm_weight);
  a.q_out = static_cast<uint16_t*>(q_out); a.q_ts = q_out_token_stride;
  a.k_out = static_cast<uint16_t*>(k_out); a.k_ts = k_out_token_stride;
  auto* kernel = head_dim == 128 ? (interleaved ? rope_qk_kernel<128, true> : rope_qk_kernel<128, false>)
                                 : (interleaved ? rope_qk_kernel<64, true> : rope_qk_kernel<64, false>);
  kernel<<<(unsigned)num_tokens, kThreads, 0, (hipStream_t)stream>>>(a);
  return check_hip(hipGetLastError(), "aia_rope_qk launch");
}
