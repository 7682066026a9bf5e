// Parts of a row's attention that several work-groups computed, and their join.
//
// A part is y = O / c in fp16, c the row's largest finite |O|, with its running maximum m
// (log2 units), sum l and c: half the bytes of float32 at 2^-11 of c at most.  The join
// gives sums the weights exp2(m - M) and values exp2(m - M) c.  (c folded into the maximum,
// m + log2 c and l / c, takes eight bytes a row less, but a part whose values are 2^126
// times another's then takes the other's keys out of the sum.)  An infinity stays with
// its dims.
#pragma once

#include "gqa_attention.h"

namespace {

struct PartHead {
  float m, l, c, pad;
};
__device__ __forceinline__ PartHead no_part(float l) { return PartHead{-INFINITY, l, 1.f, 0.f}; }

__device__ __forceinline__ float inverse_sum(float l) {       // rows without keys: zeros; NaN stays
  return l > 0.f ? 1.f / l : l == 0.f ? 0.f : __builtin_nanf("");
}

// Lane (n, g) holds dims 16 dt + 4 g .. of row n; op: the row.
template <int D>
__device__ __forceinline__ void write_out(uint16_t* op, const float4_t (&o)[D / 16], float l, int g) {
  const float inv = inverse_sum(l);
#pragma unroll
  for (int dt = 0; dt < D / 16; ++dt)
    *reinterpret_cast<uint2*>(op + 16 * dt + 4 * g) =
        make_uint2(aia::pack_bf16x2(o[dt][0] * inv, o[dt][1] * inv), aia::pack_bf16x2(o[dt][2] * inv, o[dt][3] * inv));
}

template <int D>
__device__ __forceinline__ void write_part(uint16_t* part_o, PartHead* part_head, int64_t row, const float4_t (&o)[D / 16],
                                           float m, float l, bool live, int g) {
  float c = 0.f;
#pragma unroll
  for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
    for (int v = 0; v < 4; ++v) c = fmaxf(c, finite_abs(o[dt][v]));
  c = aia::group4_max(c);
  if (!live) return;
  c = fmaxf(c, 0x1p-126f);                   // (zero rows; below it 1 / c leaves float32's range)
  const float ic = 1.f / c;
  uint16_t* pp = part_o + row * D;
#pragma unroll
  for (int dt = 0; dt < D / 16; ++dt)
    *reinterpret_cast<uint2*>(pp + 16 * dt + 4 * g) =
        make_uint2(pack_f16x2(o[dt][0] * ic, o[dt][1] * ic), pack_f16x2(o[dt][2] * ic, o[dt][3] * ic));
  if (g == 0) part_head[row] = PartHead{m, l, c, 0.f};
}

// One row's parts 0 .. count - 1 (at(i): part i's row in the buffers) to op, by W waves
// of 64 lanes: a wave's lanes weigh up to 64 parts at once, then take the parts' values
// 64 / (D / 8) at a time, 8 dims each.  (One thread per 8 dims walking the parts one
// after another: 36 us for 256 rows of 36 parts, a memory round trip each.)  W > 1:
// called by whole work-groups of W waves.
template <int D, int W, class At>
__device__ __forceinline__ void join_row(const uint16_t* part_o, const PartHead* part_head, int count, At at, uint16_t* op) {
  constexpr int LANES = D / 8, GROUPS = 64 / LANES;
  __shared__ float part[W > 1 ? W : 1][LANES][8];
  __shared__ float part_m[W > 1 ? W : 1], part_l[W > 1 ? W : 1];
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane % LANES, sub = lane / LANES;
  float m = -INFINITY, sum = 0.f, o[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = 0.f;
  // this wave's parts
  const int first = W > 1 ? (int)((int64_t)count * wid / W) : 0;
  const int last = W > 1 ? (int)((int64_t)count * (wid + 1) / W) : count;
  for (int p0 = first; p0 < last; p0 += 64) {
    const int n = min(64, last - p0);
    PartHead p = no_part(0.f);
    if (lane < n) p = part_head[at(p0 + lane)];
    float top = p.m;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
    const float mnew = fmaxf(m, top);
    // (a part without keys has -inf and 0; one that saw NaN alone -inf and NaN)
    const bool none = p.m == -INFINITY && p.l == 0.f;
    const float w = none ? 0.f : __builtin_amdgcn_exp2f(p.m - mnew), wc = w * p.c;
    const float alpha = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mnew);   // (nothing but NaN to scale then)
    sum = sum * alpha + w * p.l;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] *= alpha;
    m = mnew;
    const uint64_t some = __ballot(!none);               // parts without keys have no values
#pragma unroll 4
    for (int i0 = 0; i0 < n; i0 += GROUPS) {
      const int i = i0 + sub;
      const float wi = __shfl(wc, min(i, 63));           // (of all lanes: the last round has idle ones)
      if (i >= n || !(some >> i & 1)) continue;
      const uint4 y = *reinterpret_cast<const uint4*>(part_o + at(p0 + i) * D + 8 * c);
      const uint32_t v[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const half2_t h = __builtin_bit_cast(half2_t, v[k]);
        o[2 * k] += wi * (float)h[0];
        o[2 * k + 1] += wi * (float)h[1];
      }
    }
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
#pragma unroll
  for (int d = LANES; d < 64; d <<= 1)
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] += __shfl_xor(o[i], d);
  if (W > 1) {
    if (sub == 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) part[wid][c][i] = o[i];
      if (c == 0) { part_m[wid] = m; part_l[wid] = sum; }
    }
    __syncthreads();
    if (wid != 0) return;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) top = fmaxf(top, part_m[w]);
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float x = part_m[w] == -INFINITY && part_l[w] == 0.f ? 0.f : __builtin_amdgcn_exp2f(part_m[w] - top);
      sum += x * part_l[w];
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] += x * part[w][c][i];
    }
  }
  if (sub != 0) return;
  const float inv = inverse_sum(sum);
  op += 8 * c;
  *reinterpret_cast<uint2*>(op) = make_uint2(aia::pack_bf16x2(o[0] * inv, o[1] * inv), aia::pack_bf16x2(o[2] * inv, o[3] * inv));
  *reinterpret_cast<uint2*>(op + 4) = make_uint2(aia::pack_bf16x2(o[4] * inv, o[5] * inv), aia::pack_bf16x2(o[6] * inv, o[7] * inv));
}

// Rows of a call up to which each is joined by four waves: few rows have many parts.
constexpr int kFewRows = 1024;

}  // namespace
