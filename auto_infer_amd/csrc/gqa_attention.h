// GQA attention kernels (split-K decode / verify ranges, prefill units and
// both in one grid) over a planned step.
#pragma once

#include <math.h>

#include <type_traits>

#include "attn_plan.h"

namespace {

// ---------------------------------------------------------------- attention

// A record is used only if it lies inside the plan (defence against a plan
// read before its planner finished, e.g. from another stream).
__device__ __forceinline__ bool rec_ok(const int* r, int nseg_tiles, int batch, int tokens,
                                       int ngroups, int nhb) {
  return r[0] >= 0 && r[0] < batch && (r[1] & 0xffff) < ngroups && ((r[1] >> 16) & 0x3fff) < nhb &&
         r[2] >= 0 && (r[3] & 0xff) >= 1 && r[2] + (r[3] & 0xff) <= tokens && r[5] >= 0 && r[5] < r[6] &&
         r[6] <= nseg_tiles;
}

using aia::kWaitVmcnt0;

__device__ __forceinline__ short4_t as_s4(uint32_t a, uint32_t b) {
  short4_t r;
  r[0] = (short)(a & 0xffff); r[1] = (short)(a >> 16);
  r[2] = (short)(b & 0xffff); r[3] = (short)(b >> 16);
  return r;
}

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) short4_t lds_short4_t;

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const half2_t v = {(_Float16)lo, (_Float16)hi};
  return __builtin_bit_cast(uint32_t, v);
}


__device__ __forceinline__ u32x4_t as_u4(uint4 v) { return u32x4_t{v.x, v.y, v.z, v.w}; }

__device__ __forceinline__ bf16x8_t as_b8(uint4 v) { return __builtin_bit_cast(bf16x8_t, as_u4(v)); }

// S^T tile (16 keys x 16 rows) += K (16 keys x 32 dims) . Q^T: lane (key n,
// group g) holds dims [32 j + 8 g, +8) of its key in kk and of its row in q.
__device__ __forceinline__ float4_t qk_step(uint4 kk, uint4 q, float4_t acc) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_b8(kk), as_b8(q), acc, 0, 0, 0);
}

// A V tile is staged in LDS key-major (row stride kVStride elements): lane
// (key n, group g) stores its 16-byte pieces at dims 32 j + 8 g.  The
// transposing LDS read works within each 16-lane group: local lane l receives
// element l % 4 of the 8 bytes addressed by local lanes 4 k + l / 4, k = 0..3.
// Lane (n, g) addressing key 4 g + n / 4, dims 16 dt + 4 (n % 4) therefore
// receives V^T[16 dt + n][keys 4 g .. 4 g + 3], the A fragment of the
// 16x16x16 MFMA, in one instruction.  (The stores take vector values: an
// aggregate copy of the tile registers keeps them in a private array, which
// the compiler then places in LDS, serialising the load pipeline.)
template <int KJ>
__device__ __forceinline__ void stage_v(uint16_t* vs, int n, int g, const uint4 (&vv)[KJ]) {
#pragma unroll
  for (int j = 0; j < KJ; ++j) *reinterpret_cast<u32x4_t*>(vs + n * kVStride + 32 * j + 8 * g) = as_u4(vv[j]);
}
template <int STRIDE = kVStride>
__device__ __forceinline__ short4_t vt_frag(const uint16_t* vs, int n, int g, int dt) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (lds_short4_t*)(vs + (4 * g + (n >> 2)) * STRIDE + 16 * dt + 4 * (n & 3)));
}

// Tiles kept in flight per GQA wave (registers: 32 VGPRs per tile).  One is
// fastest: with random blocks, more outstanding tiles per CU lowers the
// delivered bandwidth (measured on config-1 decode: 18.7 us at 1, 20.1 at 2,
// 24.9 at 5), and the planner keeps ranges short instead.
#ifndef AIA_PIPE
#define AIA_PIPE 1
#endif
constexpr int kPipe = AIA_PIPE;

// The row of a query in front of the first key: its products of masked tiles are
// 0 x V, which is not zero where V is not finite.  (Looked for by the rows' limits,
// which a wave knows from the start: a test of the rows' sums at the end cost 0.08
// of 21.7 us on 16 decode rows.)
template <int DT>
__device__ __forceinline__ void clear_row(float4_t (&o)[DT]) {
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = float4_t{0.f, 0.f, 0.f, 0.f};
}

// |x|, and zero for an infinity or NaN.
__device__ __forceinline__ float finite_abs(float x) {
  return __builtin_fabsf(x) < INFINITY ? __builtin_fabsf(x) : 0.f;
}

// End of a segment's range: bf16 output where the range covers all of its
// keys, else an fp16 partial.  CARE: infinities stay with their dims; the
// partial's scale is the largest finite |O|, so the other dims fit fp16.
template <int RB, int D, bool CARE>
__device__ __forceinline__ void write_segment(const AttnArgs& a, float4_t (&o)[RB][D / 16], float (&m)[RB],
                                              float (&lsum)[RB], const bool (&rv)[RB],
                                              const int (&qi)[RB], int n, int g, int qtok0, int head,
                                              int wid, int w, int tpw, int tile_begin, int tile_end,
                                              int part_base) {
  constexpr int DT = D / 16;
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    lsum[r] = aia::group4_sum(lsum[r]);
  }
  const int first_wave = tile_begin / tpw;
  const int nparts = (tile_end - 1) / tpw - first_wave + 1;
  constexpr int seg_rows = RB * kRows;
  if (nparts == 1) {
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      if (!rv[r]) continue;
      const float inv = lsum[r] > 0.f ? 1.f / lsum[r] : 0.f;
      uint16_t* op = a.out + (int64_t)(qtok0 + qi[r]) * a.o_ts + (int64_t)head * a.o_hs;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        uint2 wv;
        wv.x = aia::pack_bf16x2(o[r][dt][0] * inv, o[r][dt][1] * inv);
        wv.y = aia::pack_bf16x2(o[r][dt][2] * inv, o[r][dt][3] * inv);
        *reinterpret_cast<uint2*>(op + 16 * dt + 4 * g) = wv;
      }
    }
  } else {
    // fp16 partial y = O / c, c = the row's largest |O| (1 for a zero row),
    // with (m + log2 c, l / c) in place of (m, l): the merge's weights
    // exp2(m - M) carry c back, so y folds exactly as O would
    const int part = part_base + (w - first_wave);
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      float cmax = 0.f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) cmax = fmaxf(cmax, CARE ? finite_abs(o[r][dt][i]) : fabsf(o[r][dt][i]));
      cmax = aia::group4_max(cmax);
      if (!rv[r]) continue;
      const float c = cmax > 0.f ? cmax : 1.f;
      const float inv = 1.f / c;
      const int64_t prow = ((int64_t)part * a.nw + wid) * seg_rows + r * kRows + n;
      uint16_t* pp = a.part_o + prow * D;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        uint2 hv;
        hv.x = pack_f16x2(o[r][dt][0] * inv, o[r][dt][1] * inv);
        hv.y = pack_f16x2(o[r][dt][2] * inv, o[r][dt][3] * inv);
        *reinterpret_cast<uint2*>(pp + 16 * dt + 4 * g) = hv;
      }
      if (g == 0) a.part_ml[prow] = make_float2(m[r] + __log2f(c), lsum[r] * inv);
    }
  }
}

// What is done to a raw dot product: nothing (the scale goes into the
// exponent), nothing but a prefix to see, a cap, a bias, both, or what the call's
// ScoreArgs say at run time.  Decode rows wait for memory, so one run-time form
// serves them all (64 requests of up to 4096 keys, 32/8 heads: 120.5 us with a
// cap, 119.4 without); prefill units wait for the VALU and have a form each.
constexpr int kPlain = 0, kPrefixOnly = 1, kCap = 2, kBias = 3, kCapBias = 4, kAnyScore = 5;

// A capped score of at most three quarters of the cap: x times a polynomial in
// (x scale / cap)^2, within 2^-22 of the cap and 2^-18 of the score, under caps
// of any size.  (The exponential's form is within 2^-21 of the cap at any score,
// which is too far for small scores under a large cap.)
__device__ __forceinline__ float cap_poly(float x, float u, const float (&c)[5]) {
  float y = __builtin_fmaf(u, c[4], c[3]);
  y = __builtin_fmaf(u, y, c[2]);
  y = __builtin_fmaf(u, y, c[1]);
  return x * __builtin_fmaf(u, y, c[0]);
}
__device__ __forceinline__ float capped_small(float x, const ScoreArgs& s) {
  const float z = x * s.cap_unit;
  return cap_poly(x, z * z, s.cap_poly);
}

// Modified scores in log2 units (see ScoreArgs); far = query position - key
// position.
template <int SC>
struct ScoreMod {
  const ScoreArgs& args;
  float scale, cap_in, cap_out;
  bool cap, bias;
  __device__ __forceinline__ ScoreMod(const ScoreArgs& s, float scale_log2)
      : args(s), scale(scale_log2), cap_in(s.cap_in), cap_out(s.cap_out),
        cap(SC == kAnyScore ? s.cap_out > 0.f : SC == kCap || SC == kCapBias),
        bias(SC == kAnyScore ? s.slopes != nullptr : SC == kBias || SC == kCapBias) {}
  __device__ __forceinline__ float capped(float x) const {
    const float t = __builtin_amdgcn_exp2f(x * cap_in);
    return __builtin_fmaf(-2.f * cap_out, __builtin_amdgcn_rcpf(t + 1.f), cap_out);
  }
  __device__ __forceinline__ float operator()(float x, float far, float slope) const {
    float y = x * scale;
    if (cap) y = __builtin_fabsf(x) <= args.cap_small ? capped_small(x, args) : capped(x);
    if (bias) y = __builtin_fmaf(-slope, __builtin_fabsf(far), y);
    return y;
  }
};
constexpr float kLog2e = 1.4426950408889634f;

// Non-finite values.  P is zero where a row does not see a key, but 0 x V is not
// where V is an infinity or NaN, so the matrix product of a masked tile would
// carry them into every row of the tile.  The kernels for modified scores and
// 8-bit caches look through V in masked tiles (the diagonal and the sequence's
// end) and multiply those that hold such a value key by key, leaving out what
// a row does not see.
__device__ __forceinline__ uint32_t not_finite_bf16(uint32_t w, uint32_t acc) {   // bits 15 and 31
  return ((w & 0x7fff7fffu) + 0x00800080u) | acc;
}
__device__ __forceinline__ uint32_t not_finite_bf16(uint4 w, uint32_t acc) {
  return not_finite_bf16(w.x, not_finite_bf16(w.y, not_finite_bf16(w.z, not_finite_bf16(w.w, acc))));
}
__device__ __forceinline__ uint32_t nan_fp8(uint4 w, uint32_t acc) {              // bits 7, 15, ...
  const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) acc |= (x[i] & 0x7f7f7f7fu) + 0x01010101u;
  return acc;
}
// Row n's weight of key k, from packed weights: the word of k's pair, held by the
// lane of group (k % 16) / 4 with row n.
__device__ __forceinline__ float weight_of(uint32_t word, int n, int k) {
  const uint32_t w = __shfl(word, n + 16 * ((k & 15) >> 2));
  return k & 1 ? aia::bf16_hi(w) : aia::bf16_lo(w);
}
// o += p * (this lane's 4 dims of each 16 of a V row)
template <int DT, class At>
__device__ __forceinline__ void add_key(float4_t (&o)[DT], float p, At at) {
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    const uint2 w = *reinterpret_cast<const uint2*>(at(dt));
    o[dt][0] = __builtin_fmaf(p, aia::bf16_lo(w.x), o[dt][0]);
    o[dt][1] = __builtin_fmaf(p, aia::bf16_hi(w.x), o[dt][1]);
    o[dt][2] = __builtin_fmaf(p, aia::bf16_lo(w.y), o[dt][2]);
    o[dt][3] = __builtin_fmaf(p, aia::bf16_hi(w.y), o[dt][3]);
  }
}

// Keys of request b that all its rows see.
__device__ __forceinline__ int prefix_keys(const ScoreArgs& s, int b) {
  return s.prefix ? max(0, min(s.prefix[b], s.kvlen[b])) : 0;
}

// Cache layouts.  ND: (num_blocks, block_size, Hkv, D), a token slot's heads
// contiguous.  NZ: the 16-wide fractal layout of the reference's graph-mode
// caches (gqa.py:163,202-226): each block viewed (Hkv D / 16, block_size,
// 16), so 16 dims of all of a block's tokens are contiguous.  kv_piece gives
// the 16-byte index of piece p (8 dims) of head h of (block, offset).
template <int KV>
__device__ __forceinline__ int64_t kv_piece(int64_t blk, int off, int bs, int row_elems, int h,
                                            int D, int p) {
  if (KV != aia::kKvNz) return (((blk * bs + off) * row_elems + (int64_t)h * D) >> 3) + p;
  return ((blk * bs * row_elems) >> 3) +
         (((int64_t)(h * (D / 16) + (p >> 1)) * bs + off) << 1) + (p & 1);
}

// Processes key tiles [lt0, lt1) of one segment; rec = the segment record.
// A segment holds RB blocks of 16 query rows: block r has the segment's
// query tokens [r qb, r qb + qb), row n being token n / hb, head n % hb
// (qb = 16 / hb).  Every K/V tile is loaded once and used by all blocks, so a
// prefill chunk reads its keys 1/RB as often; blocks past the segment's last
// token are skipped (a uniform branch), so a decode segment costs one block.
template <int RB, int D, int KV, int SC>
__device__ __forceinline__ void gqa_segment(const AttnArgs& a, const int* rec, int s, int lt0,
                                            int lt1, int w, int tpw, uint16_t* vt, int lane,
                                            int wid, bool use_pre, int pre) {
  constexpr int KJ = D / 32;   // 32-dim MFMA k-steps = 16-byte chunks per lane and row
  constexpr int DT = D / 16;   // 16-dim output tiles
  const int n = lane & 15, g = lane >> 4;
  const int b = rec[0], kvh = (rec[1] & 0xffff) * a.nw + wid, hbi = (rec[1] >> 16) & 0x3fff;
  const int qtok0 = rec[2], nq = rec[3] & 0xff, q0 = rec[3] >> 8, lim_base = rec[4];
  const int tile_begin = rec[5], tile_end = rec[6], part_base = rec[7];
  const int qb = kRows / a.hb;
  const int nt = n / a.hb, hh = n - nt * a.hb;
  const int nblk = (nq + qb - 1) / qb;               // row blocks holding tokens
  const int head = kvh * a.group + hbi * a.hb + hh;
  int qi[RB], lim[RB];
  bool rv[RB];
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    qi[r] = r * qb + nt;
    rv[r] = nt < qb && qi[r] < nq && hbi * a.hb + hh < a.group;
    lim[r] = rv[r] ? lim_base + qi[r] : -1;
  }
  int visible = max(0, lim_base + nq);
  const ScoreMod<SC> mod(a.sc, a.scale_log2);
  float slope[RB];
  if (SC != kPlain) {
    const int pre = prefix_keys(a.sc, b);
    visible = max(visible, pre);
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      if (rv[r]) lim[r] = max(lim[r], pre - 1);
      slope[r] = mod.bias && rv[r] ? a.sc.slopes[head] * kLog2e : 0.f;
    }
  }
  // smallest key limit of the valid rows (wave-uniform)
  int lim_lo = 0x7fffffff;
#pragma unroll
  for (int r = 0; r < RB; ++r) lim_lo = rv[r] ? min(lim_lo, lim[r]) : lim_lo;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) lim_lo = min(lim_lo, __shfl_xor(lim_lo, d));
  const int row_elems = a.hkv * D;
  // this step's new keys sit at positions [new_start, Lk); the request's last
  // query block (head block 0) owns writing them into the cache.  (A segment
  // without keys reads slot 0 in their place: the new row of position 0 would
  // be the one behind the request's rows.)
  const int new_start = a.kn && visible > 0 ? lim_base - q0 : 0x7fffffff;
  const int q_begin = qtok0 - q0;
  const bool writer = a.kn && ((rec[1] >> 30) & 1) && hbi == 0;

  const int32_t* btrow = a.bt + (int64_t)b * a.bt_stride;
  const int nblk_vis = (visible + a.bs - 1) / a.bs;
  const int last_key = max(visible - 1, 0);   // (a segment without keys has one masked tile)
  int blk_base = 0, btv = 0, w1 = 0;
  // 16-byte pieces between MFMA k-steps j and j + 1 of a cached key (4 pieces
  // on in ND; two 16-dim chunks of block_size x 16 on in NZ)
  const int64_t jstride = KV == aia::kKvNz ? 4 * (int64_t)a.bs : 4;

  uint4 qf[RB][KJ];
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    if (rv[r]) {
      const uint4* qp = reinterpret_cast<const uint4*>(
          a.q + (int64_t)(qtok0 + qi[r]) * a.q_ts + (int64_t)head * a.q_hs);
#pragma unroll
      for (int j = 0; j < KJ; ++j) qf[r][j] = qp[4 * j + g];
    } else {
#pragma unroll
      for (int j = 0; j < KJ; ++j) qf[r][j] = make_uint4(0, 0, 0, 0);
    }
  }

  float4_t o[RB][DT];
  float m[RB], lsum[RB];
#pragma unroll
  for (int r = 0; r < RB; ++r) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[r][dt] = float4_t{0.f, 0.f, 0.f, 0.f};
    m[r] = -1e30f;
    lsum[r] = 0.f;
  }

  // Block ids are held one per lane for a window of 64 logical blocks; the
  // window is (re)loaded only between pipelined runs, so the per-tile address
  // shuffle never waits on an outstanding global load.
  // Loads are issued unconditionally (tiles past the window read the
  // window's first key row, K and V, again: an L1 hit, and a different row
  // for every range, so no memory channel is hammered) so the load stream is
  // straight-line and the compiler can wait for each tile with an exact count.
  auto load = [&](int lt, uint4 (&kk)[KJ], uint4 (&vv)[KJ], int64_t& wdst) {
    const bool live = lt < w1;
    const int tok = live ? min(lt * kTile + n, last_key) : blk_base * a.bs;
    const int bi = tok / a.bs;
    // block ids outside the pool are clamped so a bad table cannot fault
    const int blk = min(max(__shfl(btv, bi - blk_base), 0), a.nb - 1);
    const int off = tok - bi * a.bs;
    // 16-byte index of this lane's first piece (4 g + 0) in the cache; piece
    // 4 j + g is jstride further on in either layout
    const int64_t base = kv_piece<KV>(blk, off, a.bs, row_elems, kvh, D, g);
    const bool fresh = live && tok >= new_start;
    const int64_t nrow = (int64_t)(q_begin + tok - new_start);
    const uint4* kp = fresh ? reinterpret_cast<const uint4*>(a.kn + nrow * a.kn_ts + (int64_t)kvh * D) + g
                            : reinterpret_cast<const uint4*>(a.kc) + base;
    const uint4* vp = fresh ? reinterpret_cast<const uint4*>(a.vn + nrow * a.vn_ts + (int64_t)kvh * D) + g
                            : reinterpret_cast<const uint4*>(a.vc) + base;
    const int64_t js = fresh ? 4 : jstride;
    // cache slot this lane writes after the tile arrives (-1: nothing)
    wdst = (writer && fresh && lt * kTile + n < visible) ? base : (int64_t)-1;
#pragma unroll
    for (int j = 0; j < KJ; ++j) kk[j] = kp[j * js];
#pragma unroll
    for (int j = 0; j < KJ; ++j) vv[j] = vp[j * js];
  };

  auto compute = [&](int lt, const uint4 (&kk)[KJ], const uint4 (&vv)[KJ], int64_t wdst) {
    if (wdst >= 0) {   // KV slot write of a new row (its bytes just arrived)
      uint4* kd = reinterpret_cast<uint4*>(a.kc) + wdst;
      uint4* vd = reinterpret_cast<uint4*>(a.vc) + wdst;
#pragma unroll
      for (int j = 0; j < KJ; ++j) { kd[j * jstride] = kk[j]; vd[j * jstride] = vv[j]; }
    }
    float4_t acc[RB];
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      acc[r] = float4_t{0.f, 0.f, 0.f, 0.f};
      if (r == 0 || r < nblk) {
#pragma unroll
        for (int j = 0; j < KJ; ++j) acc[r] = qk_step(kk[j], qf[r][j], acc[r]);
      }
    }
    stage_v(vt, n, g, vv);
    const int tb = lt * kTile + 4 * g;
    // keys past a valid row's limit exist only in tiles that reach past the
    // smallest limit (causal diagonal, sequence end); rows that are not valid
    // are never written, so their scores need no mask
    const bool masked = lt * kTile + kTile - 1 > lim_lo;
    short4_t pb[RB];
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      // raw scores; scale (> 0) is applied inside the exponent
      float sv[4];
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const float x = SC != kPlain ? mod(acc[r][v], (float)(lim_base + qi[r] - tb - v), slope[r]) : acc[r][v];
        sv[v] = (!masked || tb + v <= lim[r]) ? x : -INFINITY;
      }
      float tmax = fmaxf(fmaxf(sv[0], sv[1]), fmaxf(sv[2], sv[3]));
      tmax = aia::group4_max(tmax);
      const float sl = SC != kPlain ? 1.f : a.scale_log2;
      const float mnew = fmaxf(m[r], tmax * sl);
      float p[4];
#pragma unroll
      for (int v = 0; v < 4; ++v) p[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[v], sl, -mnew));
      const float psum = (p[0] + p[1]) + (p[2] + p[3]);
      if (__any(mnew > m[r])) {   // rescale only when some row's max grew
        const float alpha = __builtin_amdgcn_exp2f(m[r] - mnew);
        lsum[r] = lsum[r] * alpha + psum;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[r][dt] *= alpha;
      } else {
        lsum[r] += psum;
      }
      m[r] = mnew;
      pb[r] = as_s4(aia::pack_bf16x2(p[0], p[1]), aia::pack_bf16x2(p[2], p[3]));
    }
    __builtin_amdgcn_wave_barrier();
    if (SC != kPlain && masked) {
      uint32_t odd = 0;
#pragma unroll
      for (int j = 0; j < KJ; ++j) odd = not_finite_bf16(vv[j], odd);
      if (__any(odd & 0x80008000u)) {
        for (int k = 0; k < kTile; ++k) {
#pragma unroll
          for (int r = 0; r < RB; ++r) {
            const uint2 w = __builtin_bit_cast(uint2, pb[r]);
            const float p = weight_of(k & 2 ? w.y : w.x, n, k);
            if (lt * kTile + k <= lim[r])
              add_key(o[r], p, [&](int dt) { return vt + k * kVStride + 16 * dt + 4 * g; });
          }
        }
        __builtin_amdgcn_wave_barrier();
        return;
      }
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const short4_t va = vt_frag(vt, n, g, dt);
#pragma unroll
      for (int r = 0; r < RB; ++r)
        if (r == 0 || r < nblk)
          o[r][dt] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(va, pb[r], o[r][dt], 0, 0, 0);
    }
    __builtin_amdgcn_wave_barrier();
  };

  uint4 kbuf[kPipe][KJ], vbuf[kPipe][KJ];
  int64_t wbuf[kPipe];
  for (int w0 = lt0; w0 < lt1;) {
    blk_base = (w0 * kTile) / a.bs;
    // tiles whose keys all fall inside blocks [blk_base, blk_base + win);
    // the first window of a range uses the block ids of its work record
    const int win = use_pre ? kRecBlocks : 64;
    w1 = min(lt1, ((blk_base + win) * a.bs - kTile) / kTile + 1);
    if (use_pre) btv = lane < kRecBlocks ? pre : 0;
    else btv = blk_base + lane < nblk_vis ? btrow[blk_base + lane] : 0;
    use_pre = false;
#pragma unroll
    for (int i = 0; i < kPipe; ++i) {
      load(w0 + i, kbuf[i], vbuf[i], wbuf[i]);
      __builtin_amdgcn_sched_barrier(0);
    }
    for (int base = w0; base < w1; base += kPipe) {
#pragma unroll
      for (int i = 0; i < kPipe; ++i) {
        const int lt = base + i;
        if (lt < w1) compute(lt, kbuf[i], vbuf[i], wbuf[i]);
        load(lt + kPipe, kbuf[i], vbuf[i], wbuf[i]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    w0 = w1;
  }

  if (SC == kPlain && lim_base < 0) {
#pragma unroll
    for (int r = 0; r < RB; ++r)
      if (lim[r] < 0) clear_row(o[r]);
  }
  write_segment<RB, D, SC != kPlain>(a, o, m, lsum, rv, qi, n, g, qtok0, head, wid, w, tpw, tile_begin, tile_end, part_base);
}

// ---- 8-bit caches

// Four packed e4m3 values times 2^(e - 127) as four bf16, exactly (an e4m3
// value has four significant bits; the product stays in bf16's normal range for
// the scales that aia_kv_write_fp8 writes, but for 256 * 2^120 = 2^128, which
// magnitudes from 1.9375 * 2^127 on round to: it becomes infinite).
__device__ __forceinline__ uint2 fp8x4_to_bf16(uint32_t w, float scale) {
  uint2 r;
  r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false));
  r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true));
  return r;
}
// 16 consecutive values, e the block's e8m0 scale.
__device__ __forceinline__ void fp8_to_bf16(uint4 w, uint32_t e, uint4 (&out)[2]) {
  const float scale = __uint_as_float(e << 23);
  const uint2 a = fp8x4_to_bf16(w.x, scale), b = fp8x4_to_bf16(w.y, scale);
  const uint2 c = fp8x4_to_bf16(w.z, scale), d = fp8x4_to_bf16(w.w, scale);
  out[0] = make_uint4(a.x, a.y, b.x, b.y);
  out[1] = make_uint4(c.x, c.y, d.x, d.y);
}

// gqa_segment over 8-bit caches.  A row is half as long, so a step takes two
// of the planner's 16-key tiles: the bytes a wave keeps in flight stay those
// of one bf16 tile, and PV uses the 32-key MFMA (operand position 8 g + i
// holds key 4 g + i of the first tile, i < 4, or key 4 g + i - 4 of the
// second, where the two S^T accumulators leave P).  Lane (key n, group g)
// loads the 16-byte chunks g (and g + 4) of its key's rows; chunk c's two
// halves are the operands of k-steps 2 (c / 4) and 2 (c / 4) + 1, and Q is read in
// the same order.  Values become bf16 in registers with their block's scale,
// so the scores need no further factor.  The scales are held like the block
// ids, one logical block per lane.  Bound by memory: 128 single tokens over 1K to
// 8K keys, 64/8 heads of 128, blocks of 16: 219 us a call, 5.5 TB/s (a large
// read: 6.0).
template <int RB, int D, int SC>
__device__ __forceinline__ void gqa_segment_fp8(const AttnArgs& a, const int* rec, int s, int lt0,
                                                int lt1, int w, int tpw, uint16_t* vt0, uint16_t* vt1,
                                                int lane, int wid, bool use_pre, int pre_id) {
  constexpr int KJ = D / 32;   // 32-dim MFMA k-steps
  constexpr int CH = D / 64;   // 16-byte chunks per lane and row
  constexpr int DT = D / 16;   // 16-dim output tiles
  const int n = lane & 15, g = lane >> 4;
  const int b = rec[0], kvh = (rec[1] & 0xffff) * a.nw + wid, hbi = (rec[1] >> 16) & 0x3fff;
  const int qtok0 = rec[2], nq = rec[3] & 0xff, lim_base = rec[4];
  const int tile_begin = rec[5], tile_end = rec[6], part_base = rec[7];
  const int qb = kRows / a.hb;
  const int nt = n / a.hb, hh = n - nt * a.hb;
  const int nblk = (nq + qb - 1) / qb;               // row blocks holding tokens
  const int head = kvh * a.group + hbi * a.hb + hh;
  const int row_bytes = a.hkv * D;
  const ScoreMod<SC> mod(a.sc, a.scale_log2);
  int visible = max(0, lim_base + nq);
  int pre = 0;
  if (SC != kPlain) {
    pre = prefix_keys(a.sc, b);
    visible = max(visible, pre);
  }
  int qi[RB], lim[RB];
  bool rv[RB];
  float slope[RB];
  int lim_lo = 0x7fffffff;         // smallest key limit of the valid rows (wave-uniform)
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    qi[r] = r * qb + nt;
    rv[r] = nt < qb && qi[r] < nq && hbi * a.hb + hh < a.group;
    lim[r] = rv[r] ? max(lim_base + qi[r], pre - 1) : -1;
    lim_lo = rv[r] ? min(lim_lo, lim[r]) : lim_lo;
    slope[r] = SC != kPlain && mod.bias && rv[r] ? a.sc.slopes[head] * kLog2e : 0.f;
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) lim_lo = min(lim_lo, __shfl_xor(lim_lo, d));

  const int32_t* btrow = a.bt + (int64_t)b * a.bt_stride;
  const int nblk_vis = (visible + a.bs - 1) / a.bs;
  const int last_key = max(visible - 1, 0);   // (a segment without keys has one masked tile)
  const uint8_t* kc = reinterpret_cast<const uint8_t*>(a.kc) + (int64_t)kvh * D + 16 * g;
  const uint8_t* vc = reinterpret_cast<const uint8_t*>(a.vc) + (int64_t)kvh * D + 16 * g;
  int blk_base = 0, btv = 0, w1 = 0;
  int sev = 0;                       // this lane's block: K scale | V scale << 8

  uint4 qf[RB][KJ];
#pragma unroll
  for (int r = 0; r < RB; ++r)
#pragma unroll
    for (int j = 0; j < KJ; ++j) {
      qf[r][j] = make_uint4(0, 0, 0, 0);
      if (rv[r])
        qf[r][j] = reinterpret_cast<const uint4*>(
            a.q + (int64_t)(qtok0 + qi[r]) * a.q_ts + (int64_t)head * a.q_hs)[8 * (j >> 1) + 2 * g + (j & 1)];
    }

  float4_t o[RB][DT];
  float m[RB], lsum[RB];
#pragma unroll
  for (int r = 0; r < RB; ++r) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[r][dt] = float4_t{0.f, 0.f, 0.f, 0.f};
    m[r] = -1e30f;
    lsum[r] = 0.f;
  }

  // One 16-key tile's loads (tiles past the window re-read its first row, as
  // in gqa_segment); bi = the lane's logical block in the window.
  auto load = [&](int lt, uint4 (&kk)[CH], uint4 (&vv)[CH], int& bi) {
    const int tok = lt < w1 ? min(lt * kTile + n, last_key) : blk_base * a.bs;
    const int bl = tok / a.bs;
    bi = bl - blk_base;
    const int blk = min(max(__shfl(btv, bi), 0), a.nb - 1);
    const int64_t e = (int64_t)(blk * a.bs + (tok - bl * a.bs)) * row_bytes;
#pragma unroll
    for (int j = 0; j < CH; ++j) kk[j] = *reinterpret_cast<const uint4*>(kc + e + 64 * j);
#pragma unroll
    for (int j = 0; j < CH; ++j) vv[j] = *reinterpret_cast<const uint4*>(vc + e + 64 * j);
  };

  auto compute = [&](int lt, const uint4 (&kk)[2][CH], const uint4 (&vv)[2][CH], const int (&bi)[2]) {
    float4_t acc[RB][2];
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const int e = __shfl(sev, bi[st]);
      uint4 kf[KJ];
#pragma unroll
      for (int j = 0; j < CH; ++j) {
        uint4 x[2];
        fp8_to_bf16(kk[st][j], e & 0xff, x);
        kf[2 * j] = x[0];
        kf[2 * j + 1] = x[1];
        fp8_to_bf16(vv[st][j], (e >> 8) & 0xff, x);
        uint16_t* vs = (st ? vt1 : vt0) + n * kVStride + 64 * j + 16 * g;
        *reinterpret_cast<u32x4_t*>(vs) = as_u4(x[0]);
        *reinterpret_cast<u32x4_t*>(vs + 8) = as_u4(x[1]);
      }
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        acc[r][st] = float4_t{0.f, 0.f, 0.f, 0.f};
        if (r == 0 || r < nblk) {
#pragma unroll
          for (int j = 0; j < KJ; ++j) acc[r][st] = qk_step(kf[j], qf[r][j], acc[r][st]);
        }
      }
    }
    const int tb = lt * kTile + 4 * g;
    const int past = min(lt + 2, w1) * kTile;      // the window's keys end here
    const bool masked = lt * kTile + 2 * kTile - 1 > lim_lo || lt + 1 >= w1;
    uint4 pb[RB];
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      float sv[2][4];
      float tmax = -INFINITY;
      const int last = min(lim[r], past - 1) - tb;
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const int k = 16 * st + v;
          const float x = SC != kPlain ? mod(acc[r][st][v], (float)(lim_base + qi[r] - tb - k), slope[r]) : acc[r][st][v];
          sv[st][v] = (!masked || k <= last) ? x : -INFINITY;
          tmax = fmaxf(tmax, sv[st][v]);
        }
      tmax = aia::group4_max(tmax);
      const float sl = SC != kPlain ? 1.f : a.scale_log2;
      const float mnew = fmaxf(m[r], tmax * sl);
      float p[2][4];
      float psum = 0.f;
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          p[st][v] = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[st][v], sl, -mnew));
          psum += p[st][v];
        }
      if (__any(mnew > m[r])) {   // rescale only when some row's max grew
        const float alpha = __builtin_amdgcn_exp2f(m[r] - mnew);
        lsum[r] = lsum[r] * alpha + psum;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[r][dt] *= alpha;
      } else {
        lsum[r] += psum;
      }
      m[r] = mnew;
      pb[r] = make_uint4(aia::pack_bf16x2(p[0][0], p[0][1]), aia::pack_bf16x2(p[0][2], p[0][3]),
                         aia::pack_bf16x2(p[1][0], p[1][1]), aia::pack_bf16x2(p[1][2], p[1][3]));
    }
    __builtin_amdgcn_wave_barrier();
    if (masked) {
      uint32_t odd = 0;
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int j = 0; j < CH; ++j) odd = nan_fp8(vv[st][j], odd);
      if (__any(odd & 0x80808080u)) {
        for (int k = 0; k < 2 * kTile; ++k) {
          const uint16_t* vs = (k < kTile ? vt0 : vt1) + (k & 15) * kVStride + 4 * g;
#pragma unroll
          for (int r = 0; r < RB; ++r) {
            const uint32_t lo = k < kTile ? pb[r].x : pb[r].z, hi = k < kTile ? pb[r].y : pb[r].w;
            const float p = weight_of(k & 2 ? hi : lo, n, k);
            if (lt * kTile + k <= min(lim[r], past - 1)) add_key(o[r], p, [&](int dt) { return vs + 16 * dt; });
          }
        }
        __builtin_amdgcn_wave_barrier();
        return;
      }
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const bf16x8_t va = __builtin_bit_cast(
          bf16x8_t, __builtin_shufflevector(vt_frag(vt0, n, g, dt), vt_frag(vt1, n, g, dt), 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
      for (int r = 0; r < RB; ++r)
        if (r == 0 || r < nblk)
          o[r][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, as_b8(pb[r]), o[r][dt], 0, 0, 0);
    }
    __builtin_amdgcn_wave_barrier();
  };

  uint4 kbuf[2][CH], vbuf[2][CH];
  int bi[2];
  for (int w0 = lt0; w0 < lt1;) {
    blk_base = (w0 * kTile) / a.bs;
    const int win = use_pre ? kRecBlocks : 64;
    w1 = min(lt1, ((blk_base + win) * a.bs - kTile) / kTile + 1);
    if (use_pre) btv = lane < kRecBlocks ? pre_id : 0;
    else btv = blk_base + lane < nblk_vis ? btrow[blk_base + lane] : 0;
    use_pre = false;
    {
      const int64_t se = (int64_t)min(max(btv, 0), a.nb - 1) * a.hkv + kvh;
      sev = a.sc.ks[se] | a.sc.vs[se] << 8;
    }
#pragma unroll
    for (int st = 0; st < 2; ++st) load(w0 + st, kbuf[st], vbuf[st], bi[st]);
    __builtin_amdgcn_sched_barrier(0);
    // a step's second tile past the window is left for the next one
    for (int lt = w0; lt < w1; lt += 2) {
      compute(lt, kbuf, vbuf, bi);
#pragma unroll
      for (int st = 0; st < 2; ++st) load(lt + 2 + st, kbuf[st], vbuf[st], bi[st]);
      __builtin_amdgcn_sched_barrier(0);
    }
    w0 = w1;
  }
  write_segment<RB, D, true>(a, o, m, lsum, rv, qi, n, g, qtok0, head, wid, w, tpw, tile_begin, tile_end, part_base);
}

// One work-group per key range, one wave per kv head of the segment's group.
// D: head dim, 128 or 64.
template <int NW, int RB, int D, int KV, int SC>
#ifndef AIA_GQA_WAVES_PER_EU
#define AIA_GQA_WAVES_PER_EU 2
#endif
__device__ __forceinline__ void gqa_attn_body(const AttnArgs& a, int bid,
                                              uint16_t (*vt_all)[kTile * kVStride],
                                              uint16_t (*vt_all1)[kTile * kVStride]) {
  const int lane = threadIdx.x & 63;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (bid >= a.waves) return;
  // the planner placed the ranges in the slots, spread over the XCDs
  const int* wr = a.wave_rec + (int64_t)bid * kRecInts;
  const int pre = wr[16 + (lane & (kRecBlocks - 1))];   // issued with the header
  const int nseg = a.hdr[0], total_tiles = a.hdr[1];
  const int ngroups = (a.hkv + NW - 1) / NW, nhb = (a.group + a.hb - 1) / a.hb;
  int s = wr[0];
  int t = wr[1];
  const int t_end = wr[2], tpw = wr[3], s_last = wr[13];
  if (s < 0 || s >= nseg || t < 0 || t >= t_end || t_end > total_tiles || tpw < 1 ||
      s_last < s || s_last >= nseg)
    return;
  const int w = t / tpw;                                  // the range's index
  int rec[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) rec[i] = wr[4 + i];
  uint16_t* vt = vt_all[wid];
  bool first = true;
  while (true) {
    if (!rec_ok(rec, total_tiles, a.batch, a.tokens, ngroups, nhb)) return;
    if (rec[6] > t) {
      const int chunk_end = min(t_end, rec[6]);
      if ((rec[1] & 0xffff) * NW + wid < a.hkv)
      {
        if constexpr (KV == aia::kKvFp8)
          gqa_segment_fp8<RB, D, SC>(a, rec, s, t - rec[5], chunk_end - rec[5], w, tpw, vt, vt_all1[wid],
                                      lane, wid, first, pre);
        else
          gqa_segment<RB, D, KV, SC>(a, rec, s, t - rec[5], chunk_end - rec[5], w, tpw, vt, lane, wid,
                                      first, pre);
      }
      first = false;
      t = chunk_end;
      if (t >= t_end) break;
    }
    if (++s > s_last) return;
    const int* r = a.seg + (int64_t)s * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) rec[i] = r[i];
  }
}

template <int NW, int RB, int D, int KV, int SC>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(AIA_GQA_WAVES_PER_EU, AIA_GQA_WAVES_PER_EU)))
void gqa_attn_kernel(AttnArgs a) {
  __shared__ __attribute__((aligned(16))) uint16_t vt_all[NW][kTile * kVStride];
  if constexpr (KV == aia::kKvFp8) {       // a step is two 16-key tiles
    __shared__ __attribute__((aligned(16))) uint16_t vt_all1[NW][kTile * kVStride];
    gqa_attn_body<NW, RB, D, KV, SC>(a, blockIdx.x, vt_all, vt_all1);
  } else {
    gqa_attn_body<NW, RB, D, KV, SC>(a, blockIdx.x, vt_all, nullptr);
  }
}

// ---------------------------------------------------------------- prefill

// LDS rows of the staged K and V tiles are 2 D bytes, unpadded: the direct
// loads write whole 1 KB runs, so the chunks of each row are swizzled
// instead (see the loader).
constexpr int kKStride = kHeadDim;   // the mixed kernel's (D = 128) buffer rows
#ifndef AIA_PF_LAZY
#define AIA_PF_LAZY 8.0f
#endif
// Instruction order of the QK^T and PV blocks (sched_group_barrier): LDS
// reads kept kPfQkAhead 16-key sub-tiles (QK^T) and kPfPvAhead V^T fragments
// (PV) ahead of their MFMAs.  Left to itself the scheduler reuses one V^T
// fragment's registers and waits for each batch of reads before two MFMAs.
// (configs[1] prefill chunks, µs per call: 48.2 unordered; QK 2 / PV 4 46.0;
// PV 2, 6 or 8 and QK 3 or 4 the same within 0.1; QK 1 46.9; PV 16 46.6.)
constexpr int kPfQkAhead = 2;
constexpr int kPfPvAhead = 4;
constexpr int kSgMfma = 0x008, kSgDsRead = 0x100;    // sched_group_barrier masks
constexpr float kLazyLog2 = AIA_PF_LAZY;              // max growth (log2) before a rescale

// Prefill attention: one work-group per (prefill item, kv head).  An item is
// kPfRows consecutive rows of one request's (query token, group head) row
// list, row = token * group + head-in-group; each of the 4 waves owns 32
// rows (two 16-row MFMA tiles).  The work-group walks the keys its rows can
// see in tiles of 64: every K/V tile is loaded once (straight into one of
// two LDS buffers, one barrier per tile) and used by all 128 rows.
//   S^T = K Q^T   v_mfma_f32_16x16x32_bf16, K fragments ds_read_b128 from LDS
//                 (lane (key n, group g) reads dims 32 j + 8 g of key n), Q^T
//                 fragments held in registers for the whole item;
//   O^T += V^T P^T  v_mfma_f32_16x16x32_bf16 over 32 keys taken from two
//                 16-key sub-tiles s0, s1: operand position 8 g + i holds key
//                 16 s0 + 4 g + i (i < 4) or 16 s1 + 4 g + i - 4, which is
//                 exactly where the S^T accumulators of s0 and s1 leave P,
//                 and V^T comes from two transposing LDS reads.
// Online softmax per row with the scale inside exp2; masks only in tiles
// that reach past a wave's smallest row limit.  Outputs bf16 directly (a
// work-group covers all keys of its rows).  With new K/V rows, keys at this
// step's new positions are read from them, and the work-group writes the new
// rows of the tokens whose first row it holds into the cache.
#ifndef AIA_PF_WPE
#define AIA_PF_WPE 2
#endif
template <bool ONE_BLOCK, bool FUSED, int D, int KV, int SC>
__device__ __forceinline__ void gqa_prefill_body(const PrefillArgs& a, int wg,
                                                 uint16_t* k0, uint16_t* k1,
                                                 uint16_t* v0, uint16_t* v1, int* odd_tile) {
  constexpr int KJ = D / 32;        // 32-dim MFMA k-steps
  constexpr int DT = D / 16;        // 16-dim output tiles
  constexpr int RC = D / 8;         // 16-byte chunks per K / V row
  // The planner writes work-group b's record at dealt[b] (the grid is as long
  // as the list can be); it is loaded beside the header rather than after it.
  const int4* rec = a.dealt + 3 * (int64_t)wg;
  const int4 it = rec[0], iq = rec[1], uk = rec[2];
  const int count = a.hdr[6];
  if (wg >= count * a.hkv) return;
  const int unit = uk.x, kvh = uk.y;
  if (unit < 0 || unit >= count) return;
  const int b = it.x, row0 = it.y, t0 = it.z, t1 = it.w;
  if (b < 0 || b >= a.batch || kvh < 0 || kvh >= a.hkv) return;
  const int q_begin = iq.x, lq = iq.y, lk = iq.z, bid0 = iq.w;
  const int G = a.group;
  const int nrows = lq * G;
  if (row0 < 0 || row0 >= nrows || q_begin < 0 || q_begin + lq > a.tokens) return;
  const int ctx0 = lk - lq;                       // position of the first query token
  const int row_end = min(nrows, row0 + kPfRows);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int row_elems = a.hkv * D;
  const int32_t* btrow = a.bt + (int64_t)b * a.bt_stride;

  // new K/V rows of the tokens whose first row lies in this item (written by
  // the item's first chunk)
  if (FUSED && t0 == 0) {
    const int t_lo = (row0 + G - 1) / G, t_hi = min(lq, (row_end - 1) / G + 1);
    for (int e = tid; e < (t_hi - t_lo) * RC; e += kPfWaves * 64) {
      const int t = t_lo + e / RC, c = e % RC;
      const int p = ctx0 + t;
      if (p < 0) continue;
      const int blk = min(max(btrow[p / a.bs], 0), a.nb - 1);
      const int64_t dst = kv_piece<KV>(blk, p % a.bs, a.bs, row_elems, kvh, D, c);
      const int64_t tok = q_begin + t;
      reinterpret_cast<uint4*>(a.kc)[dst] =
          reinterpret_cast<const uint4*>(a.kn + tok * a.kn_ts + (int64_t)kvh * D)[c];
      reinterpret_cast<uint4*>(a.vc)[dst] =
          reinterpret_cast<const uint4*>(a.vn + tok * a.vn_ts + (int64_t)kvh * D)[c];
    }
  }

  const int pre = SC != kPlain ? prefix_keys(a.sc, b) : 0;
  const ScoreMod<SC> mod(a.sc, a.scale_log2);
  float slope[kPfRt];
  // this wave's rows
  int lim[kPfRt], tokr[kPfRt], headr[kPfRt];
  bool rv[kPfRt];
  int wlim_lo = 0x7fffffff, wlim_hi = -1;
#pragma unroll
  for (int rt = 0; rt < kPfRt; ++rt) {
    const int row = row0 + (wid * kPfRt + rt) * kRows + n;
    rv[rt] = row < row_end;
    tokr[rt] = row / G;
    headr[rt] = kvh * G + (row - tokr[rt] * G);
    lim[rt] = rv[rt] ? min(SC == kPlain ? ctx0 + tokr[rt] : max(ctx0 + tokr[rt], pre - 1), lk - 1) : -1;
    // a bias without a cap starts the accumulators, in units of raw products
    if (SC == kBias || SC == kCapBias)
      slope[rt] = rv[rt] ? a.sc.slopes[headr[rt]] * (SC == kBias ? kLog2e / a.scale_log2 : kLog2e) : 0.f;
    if (rv[rt]) { wlim_lo = min(wlim_lo, lim[rt]); wlim_hi = max(wlim_hi, lim[rt]); }
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    wlim_lo = min(wlim_lo, __shfl_xor(wlim_lo, d));
    wlim_hi = max(wlim_hi, __shfl_xor(wlim_hi, d));
  }
  uint4 qf[kPfRt][KJ];
#pragma unroll
  for (int rt = 0; rt < kPfRt; ++rt) {
    if (rv[rt]) {
      const uint4* qp = reinterpret_cast<const uint4*>(
          a.q + (int64_t)(q_begin + tokr[rt]) * a.q_ts + (int64_t)headr[rt] * a.q_hs);
#pragma unroll
      for (int j = 0; j < KJ; ++j) qf[rt][j] = qp[4 * j + g];
    } else {
#pragma unroll
      for (int j = 0; j < KJ; ++j) qf[rt][j] = make_uint4(0, 0, 0, 0);
    }
  }

  // keys the work-group's last row sees
  const int kend = max(pre, min(lk, ctx0 + (row_end - 1) / G + 1));
  const int ntiles = (kend + kPfKeys - 1) / kPfKeys;
  // this unit's tiles [t0, t1) of the item's [0, ntiles); a unit that does
  // not cover them all writes a partial
  if (t0 < 0 || t1 < t0 || t1 > ntiles) return;
  const bool whole = t0 == 0 && t1 == ntiles;
  const bool wide = unit < a.hdr[11];
  if (!whole && unit >= a.part_units) return;

  // Loader: thread tid moves 16-byte chunk (tid % RC) of keys kLdKeys i + tid / RC
  // (RC = D / 8 chunks per row) straight from global memory into LDS (no
  // registers, no LDS stores).  Each wave's load writes one 1 KB run, 1024 /
  // (2 D) key rows of 2 D bytes with lane l at byte 16 l; lane l fetches the
  // chunk whose swizzled place that is: K chunk c of key r sits at
  // c ^ (r % RC) and V chunk c at c ^ 2 (r % (RC / 2)), so the K fragment
  // reads (16 keys, one chunk each) and the V^T transposing reads (8 keys, 32
  // bytes each) spread over the banks without padded rows.
  // When the block size is a multiple of the tile, a tile lies in one block
  // and a key's address is one multiply-add: lane l of every wave holds the
  // block id of tile tb + l, fetched 64 tiles at a time, and a tile takes its
  // id with one readlane.  (Fetched per tile, the id's load was waited for at
  // once to move it into a scalar register: a memory round trip every tile.)
  // Other block sizes fetch each key's id one tile ahead, so those loads are
  // in flight during a tile's math.  Keys past the last visible one re-read
  // it (never a slot that may hold stale bytes); keys at this step's new
  // positions come from the new rows.
  //   8-bit caches: the thread's chunks (16 values) of the next tile wait in
  // registers during a tile's math, then become bf16 (exactly: an e4m3 value
  // times a power of two) on their way to the same places in LDS, so each value
  // is converted once per work-group.
  constexpr bool F8 = KV == aia::kKvFp8;
  constexpr int RCL = F8 ? D / 16 : RC;                // loaded chunks per row
  const int lkey = tid / RCL, lc = tid % RCL;
  const int64_t kvoff = (int64_t)kvh * D;
  const uint16_t* kcb = a.kc + kvoff;
  const uint16_t* vcb = a.vc + kvoff;
  const uint16_t* knb = FUSED ? a.kn + kvoff : nullptr;
  const uint16_t* vnb = FUSED ? a.vn + kvoff : nullptr;
  constexpr int kWaveKeys = 64 / RCL;                  // key rows per wave per round
  constexpr int kLdKeys = kPfWaves * kWaveKeys;        // keys per loader round
  constexpr int kLdRounds = kPfKeys / kLdKeys;
  static_assert(kLdKeys % 16 == 0 && kPfKeys % kLdKeys == 0,
                "loader rounds of whole 16-key swizzle groups");
  int bid[kLdRounds];
  int tb = -64, vbid = 0;
  auto fetch_ids = [&](int t) {
    if (!ONE_BLOCK) {
#pragma unroll
      for (int i = 0; i < kLdRounds; ++i) bid[i] = btrow[min(t * kPfKeys + kLdKeys * i + lkey, kend - 1) / a.bs];
    }
  };
  auto tile_bid = [&](int t) {
    if (t == t0) return bid0;      // from the unit record
    if (t - tb >= 64) {
      tb = t;
      vbid = btrow[min((t + lane) * kPfKeys, kend - 1) / a.bs];
    }
    return __builtin_amdgcn_readlane(vbid, t - tb);
  };
  // key at position p, in block blk at offset boff
  auto load_row = [&](int i, int p, int blk, int boff, uint16_t* kdst, uint16_t* vdst) {
    // (rounds start at multiples of 16 keys, so lkey stands for the key mod RC)
    const int ck = lc ^ (lkey & (RC - 1)), cv = lc ^ (2 * (lkey & (RC / 2 - 1)));
    const uint16_t* kp;
    const uint16_t* vp;
    if (KV == aia::kKvNz) {
      kp = a.kc + 8 * kv_piece<KV>(blk, boff, a.bs, row_elems, kvh, D, ck);
      vp = a.vc + 8 * kv_piece<KV>(blk, boff, a.bs, row_elems, kvh, D, cv);
    } else {
      // (the slot in 32 bits: the entry points reject pools of 2^31 slots
      // or more, as the int32 slot_mapping cannot address them; the 64-bit
      // form of this address cost the 32K-key prefill 7%)
      const int64_t e = (int64_t)(blk * a.bs + boff) * row_elems;
      kp = kcb + e + 8 * ck;
      vp = vcb + e + 8 * cv;
    }
    if (FUSED) {
      const bool fresh = p >= ctx0;
      const int64_t tok = q_begin + (p - ctx0);
      kp = fresh ? knb + tok * a.kn_ts + 8 * ck : kp;
      vp = fresh ? vnb + tok * a.vn_ts + 8 * cv : vp;
    }
    const int rb = (kLdKeys * i + kWaveKeys * wid) * D;     // the wave's first row
    aia::lds_load16(kp, kdst + rb);
    aia::lds_load16(vp, vdst + rb);
  };
  uint4 kr[F8 ? kLdRounds : 1], vr[F8 ? kLdRounds : 1];
  uint32_t ke[F8 ? kLdRounds : 1], ve[F8 ? kLdRounds : 1];
  auto load_fp8 = [&](int i, int blk, int boff) {
    const int64_t e = (int64_t)(blk * a.bs + boff) * row_elems + kvoff + 16 * lc;
    const int64_t se = (int64_t)blk * a.hkv + kvh;
    kr[i] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(a.kc) + e);
    vr[i] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(a.vc) + e);
    ke[i] = a.sc.ks[se];
    ve[i] = a.sc.vs[se];
  };
  auto store_fp8 = [&](auto buf_tag) {
    constexpr int B = decltype(buf_tag)::value;
    uint16_t* kdst = B ? k1 : k0;
    uint16_t* vdst = B ? v1 : v0;
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
  auto load = [&](int t, auto buf_tag) {
    constexpr int B = decltype(buf_tag)::value;
    uint16_t* kdst = B ? k1 : k0;
    uint16_t* vdst = B ? v1 : v0;
    const int kb = t * kPfKeys;
    if (ONE_BLOCK) {
      const int blk = min(max(tile_bid(t), 0), a.nb - 1);
      const int boff0 = kb % a.bs;
      const int last = kend - 1 - kb;
#pragma unroll
      for (int i = 0; i < kLdRounds; ++i) {
        const int off = min(kLdKeys * i + lkey, last);
        if constexpr (F8) load_fp8(i, blk, boff0 + off);
        else load_row(i, kb + off, blk, boff0 + off, kdst, vdst);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kLdRounds; ++i) {
        const int p = min(kb + kLdKeys * i + lkey, kend - 1);
        const int blk = min(max(bid[i], 0), a.nb - 1);
        if constexpr (F8) load_fp8(i, blk, p % a.bs);
        else load_row(i, p, blk, p % a.bs, kdst, vdst);
      }
    }
  };

  float4_t o[kPfRt][DT];
  float m[kPfRt], lsum[kPfRt];
#pragma unroll
  for (int rt = 0; rt < kPfRt; ++rt) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[rt][dt] = float4_t{0.f, 0.f, 0.f, 0.f};
    m[rt] = -INFINITY;
    lsum[rt] = 0.f;
  }

  // issue_next() issues the next tile's loads after the QK^T MFMAs, so that
  // the load addresses and issue overlap the MFMAs' execution: 0-1% faster
  // than issuing them first.  (A raised wave priority around each MFMA block,
  // 3% faster with register-staged loads, made this order 1-2% slower, and
  // either order is as fast without it, so no priority is set: but for modified
  // scores and 8-bit caches, whose waves spend longer between the blocks.
  // 8-bit, 512 tokens behind 32K, 28/4 heads: 281.9 -> 274.8 us, with a cap 360
  // -> 354.5; prefix and cap, 3 prompts of 600 to 2000: 106.4 -> 104.7.)
  constexpr bool PRIO = F8 || SC != kPlain, CARE = PRIO;
  auto compute = [&](int t, auto buf_tag, auto mask_tag, auto issue_next) {
    constexpr bool MASK = decltype(mask_tag)::value;
    constexpr int B = decltype(buf_tag)::value;
    const int kbase = t * kPfKeys;
    if (MASK && kbase > wlim_hi) {               // no row of this wave sees these keys
      issue_next();
      return;
    }
    const uint16_t* kt = B ? k1 : k0;
    const uint16_t* vt = B ? v1 : v0;
    constexpr int kSt = kPfKeys / 16;      // 16-key sub-tiles
    float4_t acc[kPfRt][kSt];
    float far[kPfRt];                      // the rows' distances from the lane's first key
#pragma unroll
    for (int rt = 0; rt < kPfRt; ++rt) far[rt] = (float)(ctx0 + tokr[rt] - kbase - 4 * g);
    if (PRIO) __builtin_amdgcn_s_setprio(1);
    __builtin_amdgcn_sched_barrier(0);     // the block below is scheduled on its own
#pragma unroll
    for (int st = 0; st < kSt; ++st) {
      uint4 kf[KJ];
#pragma unroll
      for (int j = 0; j < KJ; ++j)
        kf[j] = *reinterpret_cast<const uint4*>(kt + (16 * st + n) * D + 8 * ((4 * j + g) ^ (n & (RC - 1))));
#pragma unroll
      for (int rt = 0; rt < kPfRt; ++rt) {
        // (a row tile with no valid row computes rows that are never written)
        acc[rt][st] = float4_t{0.f, 0.f, 0.f, 0.f};
        if (SC == kBias) {
#pragma unroll
          for (int v = 0; v < 4; ++v)
            acc[rt][st][v] = -slope[rt] * __builtin_fabsf(far[rt] - (float)(16 * st + v));
        }
#pragma unroll
        for (int j = 0; j < KJ; ++j) acc[rt][st] = qk_step(kf[j], qf[rt][j], acc[rt][st]);
      }
    }
    __builtin_amdgcn_sched_group_barrier(kSgDsRead, KJ * kPfQkAhead, 0);
#pragma unroll
    for (int st = 0; st < kSt; ++st) {
      __builtin_amdgcn_sched_group_barrier(kSgMfma, KJ * kPfRt, 0);
      if (st + kPfQkAhead < kSt) __builtin_amdgcn_sched_group_barrier(kSgDsRead, KJ, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (PRIO) __builtin_amdgcn_s_setprio(0);
    issue_next();
    uint4 pb[kPfRt][kSt / 2];
#pragma unroll
    for (int rt = 0; rt < kPfRt; ++rt) {
      float sv[kSt][4];
      float tmax = -INFINITY;
      if (SC == kCap || SC == kCapBias) {
        // The VALU is what these units wait for, and the cap's exponential and
        // reciprocal are a quarter as fast as other instructions: tiles whose
        // scores all stay below three quarters of the cap take a polynomial
        // (six multiply-adds) instead, of the raw products where its factors fit
        // float32 (scaled ones, a multiplication more, cost prefix and cap, 3
        // prompts of 600 to 2000, 2 of 98 us).
        float big = 0.f;
#pragma unroll
        for (int st = 0; st < kSt; ++st)
#pragma unroll
          for (int v = 0; v < 4; ++v) big = fmaxf(big, __builtin_fabsf(acc[rt][st][v]));
        auto each = [&](auto f) {
#pragma unroll
          for (int st = 0; st < kSt; ++st)
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              const float y = f(acc[rt][st][v]);
              acc[rt][st][v] = SC == kCapBias
                  ? __builtin_fmaf(-slope[rt], __builtin_fabsf(far[rt] - (float)(16 * st + v)), y) : y;
            }
        };
        if (__any(big > a.sc.cap_small)) each([&](float x) { return mod.capped(x); });
        else if (a.sc.cap_raw[0] != 0.f) each([&](float x) { return cap_poly(x, x * x, a.sc.cap_raw); });
        else each([&](float x) { return capped_small(x, a.sc); });
      }
      if (MASK) {     // causal diagonal / sequence end: per-key limits
        const int rel = lim[rt] - kbase - 4 * g;
#pragma unroll
        for (int st = 0; st < kSt; ++st)
#pragma unroll
          for (int v = 0; v < 4; ++v) sv[st][v] = 16 * st + v <= rel ? acc[rt][st][v] : -INFINITY;
      } else {
#pragma unroll
        for (int st = 0; st < kSt; ++st)
#pragma unroll
          for (int v = 0; v < 4; ++v) sv[st][v] = acc[rt][st][v];
      }
#pragma unroll
      for (int st = 0; st < kSt; ++st)
#pragma unroll
        for (int v = 0; v < 4; ++v) tmax = fmaxf(tmax, sv[st][v]);
      tmax = aia::group4_max(tmax);
      // Lazy rescale: the running max m only moves when some row's tile max
      // exceeds it by more than kLazyLog2, so P stays below 2^kLazyLog2 and O
      // and l (which share m) need no rescale on most tiles.  m = -inf until
      // a row sees a key; exp2(-inf) = 0 then.
      const float sl = SC == kCap || SC == kCapBias ? 1.f : a.scale_log2;
      const float tm = tmax * sl;
      const bool grow = __any(tm > m[rt] + kLazyLog2);
      const float mnew = grow ? fmaxf(m[rt], tm) : m[rt];
      const float msub = mnew == -INFINITY ? 0.f : mnew;
      float p[kSt][4];
      float psum = 0.f;
#pragma unroll
      for (int st = 0; st < kSt; ++st)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          p[st][v] = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[st][v], sl, -msub));
          psum += p[st][v];
        }
      if (grow) {
        const float alpha = __builtin_amdgcn_exp2f(m[rt] - msub);
        lsum[rt] = lsum[rt] * alpha + psum;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[rt][dt] *= alpha;
      } else {
        lsum[rt] += psum;
      }
      m[rt] = mnew;
#pragma unroll
      for (int pp = 0; pp < kSt / 2; ++pp) {
        pb[rt][pp].x = aia::pack_bf16x2(p[2 * pp][0], p[2 * pp][1]);
        pb[rt][pp].y = aia::pack_bf16x2(p[2 * pp][2], p[2 * pp][3]);
        pb[rt][pp].z = aia::pack_bf16x2(p[2 * pp + 1][0], p[2 * pp + 1][1]);
        pb[rt][pp].w = aia::pack_bf16x2(p[2 * pp + 1][2], p[2 * pp + 1][3]);
      }
    }
    __builtin_amdgcn_sched_barrier(0);     // the block below is scheduled on its own
    if (CARE && MASK && *reinterpret_cast<volatile int*>(odd_tile + B) == t) {
      for (int k = 0; k < kPfKeys; ++k) {
        const uint16_t* vs = vt + k * D + 4 * (g & 1);
        const int sw = 2 * (k & (RC / 2 - 1));
#pragma unroll
        for (int rt = 0; rt < kPfRt; ++rt) {
          uint32_t word = 0;
#pragma unroll
          for (int w = 0; w < kSt * 2; ++w) {       // word w: keys 16 (w / 2) + 4 g + 2 (w % 2), + 1
            const uint4 q = pb[rt][w >> 2];
            const uint32_t x = (w & 3) == 0 ? q.x : (w & 3) == 1 ? q.y : (w & 3) == 2 ? q.z : q.w;
            word = w == 2 * (k >> 4) + ((k >> 1) & 1) ? x : word;
          }
          const float p = weight_of(word, n, k);
          if (kbase + k <= lim[rt])
            add_key(o[rt], p, [&](int dt) { return vs + 8 * ((2 * dt + (g >> 1)) ^ sw); });
        }
      }
      return;
    }
    if (PRIO) __builtin_amdgcn_s_setprio(1);
    // PV over V^T fragments f = (32-key pair pp, 16 dims dt), read kPfPvAhead
    // fragments ahead of their MFMAs.  Lane (n, g) reads keys 4 g + n / 4
    // (+ 16), dims 16 dt + 4 (n % 4), at their swizzled place (the
    // transposing read as in vt_frag).
    const int vrow = 4 * g + (n >> 2);
#pragma unroll
    for (int f = 0; f < kSt / 2 * DT; ++f) {
      const int pp = f / DT, dt = f % DT;
      const int vsw = 16 * (dt ^ (vrow & (RC / 2 - 1)));
      const short4_t x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_short4_t*)(vt + (32 * pp + vrow) * D + vsw + 4 * (n & 3)));
      const short4_t x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_short4_t*)(vt + (32 * pp + 16 + vrow) * D + vsw + 4 * (n & 3)));
      const bf16x8_t va = __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
      for (int rt = 0; rt < kPfRt; ++rt)
        o[rt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, as_b8(pb[rt][pp]), o[rt][dt], 0, 0, 0);
    }
    __builtin_amdgcn_sched_group_barrier(kSgDsRead, 2 * kPfPvAhead, 0);
#pragma unroll
    for (int f = 0; f < kSt / 2 * DT; ++f) {
      __builtin_amdgcn_sched_group_barrier(kSgMfma, kPfRt, 0);
      if (f + kPfPvAhead < kSt / 2 * DT) __builtin_amdgcn_sched_group_barrier(kSgDsRead, 2, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (PRIO) __builtin_amdgcn_s_setprio(0);
  };

  // Tiles from t_care on are masked for some of the work-group's rows.  As such a
  // tile's bytes arrive, each thread looks through the V values that it loaded
  // and names the tile in odd_tile[its buffer] where one is not finite.
  const int t_care = max(t0, min(t1, (min(max(ctx0 + row0 / G, pre - 1), lk - 1) + 1) / kPfKeys));
  auto look = [&](int t, auto buf_tag) {
    constexpr int B = decltype(buf_tag)::value;
    if (!CARE || t < t_care || t >= t1) return;
    bool odd;
    if constexpr (F8) {
      uint32_t x = 0;
#pragma unroll
      for (int i = 0; i < kLdRounds; ++i) x = nan_fp8(vr[i], x);
      odd = x & 0x80808080u;
    } else {
      asm volatile("" ::: "memory");       // after the wait for this wave's direct loads
      uint32_t x = 0;
      const uint16_t* vt = (B ? v1 : v0) + (kWaveKeys * wid) * D + 8 * lane;
#pragma unroll
      for (int i = 0; i < kLdRounds; ++i)
        x = not_finite_bf16(*reinterpret_cast<const uint4*>(vt + kLdKeys * i * D), x);
      odd = x & 0x80008000u;
    }
    if (odd) odd_tile[B] = t;
  };

  if (t1 > t0) {
    using buf0 = std::integral_constant<int, 0>;
    using buf1 = std::integral_constant<int, 1>;
    if (ONE_BLOCK) {   // the next 64 tiles' ids, in flight beside the first tile
      tb = t0;
      vbid = btrow[min((t0 + lane) * kPfKeys, kend - 1) / a.bs];
    }
    fetch_ids(t0);
    load(t0, buf0{});
    fetch_ids(t0 + 1);
    if constexpr (CARE) {
      if (tid < 2) odd_tile[tid] = -1;
      __syncthreads();
    }
    if constexpr (F8) store_fp8(buf0{});
    else __builtin_amdgcn_s_waitcnt(kWaitVmcnt0);
    look(t0, buf0{});
    __syncthreads();
    // Tiles below the wave's smallest row limit need no mask; the two runs
    // together take every tile, so all waves pass the same barriers.  The
    // buffer of each step is a compile-time choice (separate LDS arrays), so
    // the compiler sees that a step's reads and the next tile's direct loads
    // touch different memory and holds no read back for those loads; with a
    // buffer index chosen at run time it waits for the loads before each read.
    // The loop keeps one copy of each buffer's step (unrolled copies cost more
    // in instruction fetch than they save).
    const int t_um = max(t0, min(t1, (wlim_lo + 1) / kPfKeys));
    auto step = [&](int t, auto buf_tag, auto mask_tag) {
      constexpr int B = decltype(buf_tag)::value;
      using other = std::integral_constant<int, B ^ 1>;
      auto issue_next = [&]() {
        if (t + 1 < t1) {
          load(t + 1, other{});
          fetch_ids(t + 2);
        }
      };
      compute(t, buf_tag, mask_tag, issue_next);
      if constexpr (F8) {
        if (t + 1 < t1) store_fp8(other{});
      } else {
        __builtin_amdgcn_s_waitcnt(kWaitVmcnt0);
      }
      look(t + 1, other{});
      __syncthreads();
    };
    auto run = [&](int t, int t_end, auto mask_tag) {
      bool odd = ((t - t0) & 1) != 0;
#pragma clang loop unroll(disable)
      while (t < t_end) {
        if (!odd) {
          step(t, buf0{}, mask_tag);
          if (++t >= t_end) break;
        }
        step(t, buf1{}, mask_tag);
        ++t;
        odd = false;
      }
    };
    run(t0, t_um, std::false_type{});
    run(t_um, t1, std::true_type{});
  }

  const bool front = __builtin_amdgcn_readfirstlane(wlim_lo) < 0;
#pragma unroll
  for (int rt = 0; rt < kPfRt; ++rt) {
    lsum[rt] = aia::group4_sum(lsum[rt]);
    if (!CARE && front && lim[rt] < 0) clear_row(o[rt]);
    // a unit that does not cover all of its item's keys writes a partial:
    // y = O / c in fp16, c = the row's largest |O| (1 for an all-zero row; with
    // CARE the largest finite one, so that an infinity leaves the other dims in
    // range), with (m + log2 c, l / c) in place of (m, l).  The merge's
    // log-sum-exp rule then folds c back exactly (its weights are exp2(m - M)),
    // and the partials take half the bytes of fp32 ones.  The first hdr[11] units
    // of the list keep O and (m, l) as they are, in fp32 (see the planner).
    float cmax = 0.f;
    if (!whole && !wide) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int v = 0; v < 4; ++v)
          cmax = fmaxf(cmax, CARE ? finite_abs(o[rt][dt][v]) : fabsf(o[rt][dt][v]));
      cmax = aia::group4_max(cmax);
    }
    if (!rv[rt]) continue;
    if (!whole && wide) {
      const int64_t prow = ((int64_t)unit * a.hkv + kvh) * kPfRows + (wid * kPfRt + rt) * kRows + n;
      float* pp = reinterpret_cast<float*>(a.part_o) + prow * D;      // its block, whole
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<float4_t*>(pp + 16 * dt + 4 * g) = o[rt][dt];
      if (g == 0) a.part_ml[prow] = make_float2(m[rt], lsum[rt]);
      continue;
    }
    if (!whole) {
      const float c = cmax > 0.f ? cmax : 1.f, ic = 1.f / c;
      const int64_t blk = (int64_t)unit * a.hkv + kvh, r = (wid * kPfRt + rt) * kRows + n;
      uint16_t* pp = a.part_o + (2 * blk * kPfRows + r) * D;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        uint2 hv;
        hv.x = pack_f16x2(o[rt][dt][0] * ic, o[rt][dt][1] * ic);
        hv.y = pack_f16x2(o[rt][dt][2] * ic, o[rt][dt][3] * ic);
        *reinterpret_cast<uint2*>(pp + 16 * dt + 4 * g) = hv;
      }
      if (g == 0) a.part_ml[blk * kPfRows + r] = make_float2(m[rt] + __log2f(c), lsum[rt] * ic);
      continue;
    }
    const float inv = lsum[rt] > 0.f ? 1.f / lsum[rt] : 0.f;
    uint16_t* op = a.out + (int64_t)(q_begin + tokr[rt]) * a.o_ts + (int64_t)headr[rt] * a.o_hs;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      uint2 wv;
      wv.x = aia::pack_bf16x2(o[rt][dt][0] * inv, o[rt][dt][1] * inv);
      wv.y = aia::pack_bf16x2(o[rt][dt][2] * inv, o[rt][dt][3] * inv);
      *reinterpret_cast<uint2*>(op + 16 * dt + 4 * g) = wv;
    }
  }
}

template <bool ONE_BLOCK, bool FUSED, int D, int KV, int SC>
__global__ __launch_bounds__(kPfWaves * 64) __attribute__((amdgpu_waves_per_eu(AIA_PF_WPE, AIA_PF_WPE)))
void gqa_prefill_kernel(PrefillArgs a) {
  __shared__ __attribute__((aligned(16))) uint16_t k0[kPfKeys * D];
  __shared__ __attribute__((aligned(16))) uint16_t k1[kPfKeys * D];
  __shared__ __attribute__((aligned(16))) uint16_t v0[kPfKeys * D];
  __shared__ __attribute__((aligned(16))) uint16_t v1[kPfKeys * D];
  if constexpr (KV == aia::kKvFp8 || SC != kPlain) {
    __shared__ int odd_tile[2];
    gqa_prefill_body<ONE_BLOCK, FUSED, D, KV, SC>(a, blockIdx.x, k0, k1, v0, v1, odd_tile);
  } else {
    gqa_prefill_body<ONE_BLOCK, FUSED, D, KV, SC>(a, blockIdx.x, k0, k1, v0, v1, nullptr);
  }
}

// Mixed steps (prefill items beside split-K decode ranges) in one grid, for
// kPfWaves-wave decode groups (Hkv = kPfWaves).  Launched separately, the
// two kernels barely share a CU: one prefill wave (212-232 VGPRs, allocated
// in blocks of 8) plus two decode waves (2 x 144) fill or exceed a SIMD's
// 512, so the second kernel mostly waits for the first to drain.  In one grid every
// work-group gets the prefill budget and does one job or the other, so the
// compute-bound prefill runs while the HBM-bound decode streams beside it.
// The decode role stages its V^T tiles in the first K buffer (over 8-bit
// caches, whose steps are two tiles, in both).
constexpr int kMixedK0 = kPfWaves * kTile * kVStride > kPfKeys * kKStride
                             ? kPfWaves * kTile * kVStride : kPfKeys * kKStride;
template <bool ONE_BLOCK, bool FUSED, int KV, int SC>
__global__ __launch_bounds__(kPfWaves * 64) __attribute__((amdgpu_waves_per_eu(AIA_PF_WPE, AIA_PF_WPE)))
void gqa_mixed_kernel(AttnArgs a, PrefillArgs pa, int npf) {
  __shared__ __attribute__((aligned(16))) uint16_t k0[kMixedK0];
  __shared__ __attribute__((aligned(16))) uint16_t k1[KV == aia::kKvFp8 ? kMixedK0 : kPfKeys * kKStride];
  __shared__ __attribute__((aligned(16))) uint16_t v0[kPfKeys * kKStride];
  __shared__ __attribute__((aligned(16))) uint16_t v1[kPfKeys * kKStride];
  // Prefill units take the first npf block ids and the decode ranges the
  // rest: the units are dealt out first, one or two per CU, and the ranges
  // fill the remaining slots and every slot a unit frees.  (Alternating the
  // roles by block id measured slower: 590 us against 449 on configs[1] in
  // runs of 8 ids, 459-462 in runs of 64; runs of 256 matched.)
  const int b = blockIdx.x;
  const bool prefill = b < npf;
  const int idx = prefill ? b : b - npf;
  int* odd = nullptr;
  if constexpr (KV == aia::kKvFp8 || SC != kPlain) {
    __shared__ int odd_tile[2];
    odd = odd_tile;
  }
  if (prefill)
    gqa_prefill_body<ONE_BLOCK, FUSED, kHeadDim, KV, SC>(pa, idx, k0, k1, v0, v1, odd);
  else
    gqa_attn_body<kPfWaves, 1, kHeadDim, KV, SC == kPlain ? kPlain : kAnyScore>(a, idx,
                                         reinterpret_cast<uint16_t(*)[kTile * kVStride]>(&k0[0]),
                                         reinterpret_cast<uint16_t(*)[kTile * kVStride]>(&k1[0]));
}

// The attention launches of one call, for one cache format.  SC: the prefill
// units' scores; the split-K ranges take any.  (8-bit caches have no fused
// write: pa.kn is null.)
template <int KV, int SC>
int launch_prefill(const PrefillArgs& pa, const Layout& L, const Geometry& g, int32_t head_dim,
                   bool one_block, hipStream_t s) {
  constexpr bool FUSE = KV != aia::kKvFp8;
  const bool fused = FUSE && pa.kn;
  const dim3 grid((unsigned)(L.pf_unit_cap * g.hkv));
#define AIA_PF_LAUNCH(D)                                                                             \
  (one_block && fused ? gqa_prefill_kernel<true, FUSE, D, KV, SC><<<grid, kPfWaves * 64, 0, s>>>(pa)    \
   : one_block        ? gqa_prefill_kernel<true, false, D, KV, SC><<<grid, kPfWaves * 64, 0, s>>>(pa)   \
   : fused            ? gqa_prefill_kernel<false, FUSE, D, KV, SC><<<grid, kPfWaves * 64, 0, s>>>(pa)   \
                      : gqa_prefill_kernel<false, false, D, KV, SC><<<grid, kPfWaves * 64, 0, s>>>(pa))
  if (head_dim == 64) AIA_PF_LAUNCH(64);
  else AIA_PF_LAUNCH(kHeadDim);
#undef AIA_PF_LAUNCH
  return aia::check_hip(hipGetLastError(), "gqa_prefill_kernel launch");
}

template <int KV, int SC>
int launch_mixed(const AttnArgs& a, const PrefillArgs& pa, const Layout& L, const Geometry& g,
                 int32_t waves, bool one_block, hipStream_t s) {
  constexpr bool FUSE = KV != aia::kKvFp8;
  const bool fused = FUSE && pa.kn;
  const int npf = (int)(L.pf_unit_cap * g.hkv);
  const dim3 grid((unsigned)(npf + waves));
  if (one_block && fused) gqa_mixed_kernel<true, FUSE, KV, SC><<<grid, kPfWaves * 64, 0, s>>>(a, pa, npf);
  else if (one_block) gqa_mixed_kernel<true, false, KV, SC><<<grid, kPfWaves * 64, 0, s>>>(a, pa, npf);
  else if (fused) gqa_mixed_kernel<false, FUSE, KV, SC><<<grid, kPfWaves * 64, 0, s>>>(a, pa, npf);
  else gqa_mixed_kernel<false, false, KV, SC><<<grid, kPfWaves * 64, 0, s>>>(a, pa, npf);
  return aia::check_hip(hipGetLastError(), "gqa_mixed_kernel launch");
}

template <int KV, bool SCORED>
int launch_gqa(const AttnArgs& a, const PrefillArgs& pa, const Layout& L, const Geometry& g,
               int32_t head_dim, int32_t waves, bool one_block, hipStream_t s) {
  constexpr int DEC = SCORED ? kAnyScore : kPlain;
  const bool cap = a.sc.cap_out > 0.f, bias = a.sc.slopes != nullptr;
  if (mixed_grid(g, head_dim)) {
    if constexpr (!SCORED) return launch_mixed<KV, kPlain>(a, pa, L, g, waves, one_block, s);
    else
      return cap && bias ? launch_mixed<KV, kCapBias>(a, pa, L, g, waves, one_block, s)
             : cap       ? launch_mixed<KV, kCap>(a, pa, L, g, waves, one_block, s)
             : bias      ? launch_mixed<KV, kBias>(a, pa, L, g, waves, one_block, s)
                         : launch_mixed<KV, kPrefixOnly>(a, pa, L, g, waves, one_block, s);
  }
#define AIA_GQA_LAUNCH_D(NW, D)                                                         \
  (g.rb == 2 ? gqa_attn_kernel<NW, 2, D, KV, DEC><<<waves, 64 * NW, 0, s>>>(a)             \
             : gqa_attn_kernel<NW, 1, D, KV, DEC><<<waves, 64 * NW, 0, s>>>(a))
#define AIA_GQA_LAUNCH(NW)                                                        \
  (head_dim == 64 ? AIA_GQA_LAUNCH_D(NW, 64) : AIA_GQA_LAUNCH_D(NW, kHeadDim))
  switch (g.nw) {
    case 1: AIA_GQA_LAUNCH(1); break;
    case 2: AIA_GQA_LAUNCH(2); break;
    case 3: AIA_GQA_LAUNCH(3); break;
    case 4: AIA_GQA_LAUNCH(4); break;
    case 5: AIA_GQA_LAUNCH(5); break;
    case 6: AIA_GQA_LAUNCH(6); break;
    case 7: AIA_GQA_LAUNCH(7); break;
    default: AIA_GQA_LAUNCH(8); break;
  }
#undef AIA_GQA_LAUNCH
#undef AIA_GQA_LAUNCH_D
  if (int rc = aia::check_hip(hipGetLastError(), "gqa_attn_kernel launch")) return rc;
  if (L.pf_cap <= 0) return AIA_OK;
  if constexpr (!SCORED) return launch_prefill<KV, kPlain>(pa, L, g, head_dim, one_block, s);
  else
    return cap && bias ? launch_prefill<KV, kCapBias>(pa, L, g, head_dim, one_block, s)
           : cap       ? launch_prefill<KV, kCap>(pa, L, g, head_dim, one_block, s)
           : bias      ? launch_prefill<KV, kBias>(pa, L, g, head_dim, one_block, s)
                       : launch_prefill<KV, kPrefixOnly>(pa, L, g, head_dim, one_block, s);
}

}  // namespace
