// One wave's attention of up to 16 query rows to a run of listed cache blocks: the inner loop of the block-sparse kernel and of the shared-prefix
// kernel's narrow units.  (Two row blocks per wave took 250 registers against 124, and
// 28 us against 24 for 16 requests behind 4096 shared keys: two waves that share a
// tile's bytes through the caches are the better use of a tile for 32 rows.)
//
// Keys are numbered by their place in the list (place p: block p / bs of the list,
// offset p % bs).  A wave takes them in tiles of 16: S^T = K Q^T with K straight
// from memory to the MFMA's operand registers, an online softmax per row, and
// O^T += V^T P^T with V staged in the wave's own LDS for the transposing reads.
// No barriers: waves drift, so some load while others compute.  The next tile's
// loads are in flight during a tile's math.
#pragma once

#include "gqa_attention.h"

namespace {

// A layer's caches, as the attention kernels take them.
struct CacheArgs {
  const uint16_t* kc;        // (num_blocks, bs, hkv, D) bf16, or e4m3 bytes
  const uint16_t* vc;
  const uint8_t* ks;         // e8m0 scales (num_blocks, hkv) of 8-bit caches
  const uint8_t* vs;
  int32_t hkv, group, bs, nb;
  float scale_log2;          // score factor times log2(e)
};

// What a wave keeps of its rows: lane (n, g) holds row n's dims 16 dt + 4 g + (0..3);
// m in log2 units (-inf: no key seen), l this lane's share of the sum until finish().
template <int D>
struct RowState {
  float4_t o[D / 16];
  float m, l;
  __device__ __forceinline__ void clear() {
    clear_row(o);
    m = -INFINITY;
    l = 0.f;
  }
  __device__ __forceinline__ void finish() { l = aia::group4_sum(l); }
};

// Q operands: row n from qp (null: zeros), in the order that
// attend() reads keys of the cache format in.
template <int D, bool F8>
__device__ __forceinline__ void load_q(const uint16_t* qp, int g, uint4 (&qf)[D / 32]) {
#pragma unroll
  for (int j = 0; j < D / 32; ++j) {
    qf[j] = make_uint4(0, 0, 0, 0);
    if (qp) qf[j] = reinterpret_cast<const uint4*>(qp)[F8 ? 8 * (j >> 1) + 2 * g + (j & 1) : 4 * j + g];
  }
}

// The softmax of one tile of NT x 16 keys: scores x (masked ones -inf) to weights.
template <int NT, int DT>
__device__ __forceinline__ void soften(float (&x)[NT][4], float scale_log2, float& m, float& l,
                                       float4_t (&o)[DT]) {
  float top = -INFINITY;
#pragma unroll
  for (int st = 0; st < NT; ++st)
#pragma unroll
    for (int v = 0; v < 4; ++v) top = fmaxf(top, x[st][v]);
  top = aia::group4_max(top);
  const float mnew = fmaxf(m, top * scale_log2);
  const float sub = mnew == -INFINITY ? 0.f : mnew;
  float sum = 0.f;
#pragma unroll
  for (int st = 0; st < NT; ++st)
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      x[st][v] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[st][v], scale_log2, -sub));
      sum += x[st][v];
    }
  if (__any(mnew > m)) {     // rescale only when some row's max grew
    const float alpha = __builtin_amdgcn_exp2f(m - sub);
    l = l * alpha + sum;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
  } else {
    l += sum;
  }
  m = mnew;
}

// Attends places [p0, p1) (p0 a multiple of 16) with rows qf; row n sees places up to
// lim (lim_lo: the smallest of the valid rows', wave-uniform; places from p1 on are
// seen by none).  id(i): the block id of list entry i, called with different i per
// lane, 0 <= i < entries.  vt: kTile * kVStride values of the wave's own LDS (8-bit
// caches: twice that).
//
// Values that are not finite: weights of masked keys are zero, but 0 x V is not
// where V is an infinity or NaN.  Places from p1 on are replaced by zeros, and with
// CARE (rows of different limits) a masked tile that holds such a value is
// multiplied key by key.
template <int D, bool F8, bool CARE, class Id>
__device__ __forceinline__ void attend(const CacheArgs& a, int kvh, const uint4 (&qf)[D / 32], int lim,
                                       int lim_lo, int p0, int p1, int entries, Id id, uint16_t* vt,
                                       int lane, RowState<D>& s) {
  constexpr int KJ = D / 32, DT = D / 16, CH = D / 64;
  constexpr int NT = F8 ? 2 : 1;             // 16-key tiles per step
  constexpr int LD = F8 ? CH : KJ;           // 16-byte loads per key row and lane
  const int n = lane & 15, g = lane >> 4;
  if (p0 >= p1) return;
  const int64_t row_elems = (int64_t)a.hkv * D;
  int base = 0, bend = 0, ids = 0, sev = 0;  // list entries held by the lanes: [base, bend)

  auto load = [&](int tile, uint4 (&kk)[LD], uint4 (&vv)[LD], int& at) {
    // (tiles past the window read its first row again: an L1 hit)
    const int place = tile * kTile < p1 && tile * kTile < bend * a.bs ? min(tile * kTile + n, p1 - 1) : base * a.bs;
    const int e = place / a.bs;
    at = e - base;
    const int blk = __shfl(ids, at);
    const int64_t row = ((int64_t)blk * a.bs + (place - e * a.bs)) * row_elems + (int64_t)kvh * D;
    if constexpr (F8) {
      const uint8_t* kp = reinterpret_cast<const uint8_t*>(a.kc) + row + 16 * g;
      const uint8_t* vp = reinterpret_cast<const uint8_t*>(a.vc) + row + 16 * g;
#pragma unroll
      for (int j = 0; j < LD; ++j) kk[j] = *reinterpret_cast<const uint4*>(kp + 64 * j);
#pragma unroll
      for (int j = 0; j < LD; ++j) vv[j] = *reinterpret_cast<const uint4*>(vp + 64 * j);
    } else {
      const uint4* kp = reinterpret_cast<const uint4*>(a.kc + row) + g;
      const uint4* vp = reinterpret_cast<const uint4*>(a.vc + row) + g;
#pragma unroll
      for (int j = 0; j < LD; ++j) kk[j] = kp[4 * j];
#pragma unroll
      for (int j = 0; j < LD; ++j) vv[j] = vp[4 * j];
    }
  };

  auto compute = [&](int tile, const uint4 (&kk)[NT][LD], uint4 (&vv)[NT][LD], const int (&at)[NT], int end) {
    const int tb = tile * kTile;
    const bool masked = tb + NT * kTile - 1 > lim_lo || tb + NT * kTile > end;
    uint32_t odd = 0;
    if (masked) {
#pragma unroll
      for (int st = 0; st < NT; ++st)
#pragma unroll
        for (int j = 0; j < LD; ++j) {
          if (tb + kTile * st + n >= end) vv[st][j] = make_uint4(0, 0, 0, 0);
          if (CARE) odd = F8 ? nan_fp8(vv[st][j], odd) : not_finite_bf16(vv[st][j], odd);
        }
      odd &= F8 ? 0x80808080u : 0x80008000u;
    }
    float4_t acc[NT];
#pragma unroll
    for (int st = 0; st < NT; ++st) {
      uint4 kf[KJ];
      if constexpr (F8) {
        const int e = __shfl(sev, at[st]);
#pragma unroll
        for (int j = 0; j < CH; ++j) {
          uint4 x[2];
          fp8_to_bf16(kk[st][j], e & 0xff, x);
          kf[2 * j] = x[0];
          kf[2 * j + 1] = x[1];
          fp8_to_bf16(vv[st][j], (e >> 8) & 0xff, x);
          uint16_t* to = vt + (st * kTile + n) * kVStride + 64 * j + 16 * g;
          *reinterpret_cast<u32x4_t*>(to) = as_u4(x[0]);
          *reinterpret_cast<u32x4_t*>(to + 8) = as_u4(x[1]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < KJ; ++j) kf[j] = kk[st][j];
        stage_v(vt + st * kTile * kVStride, n, g, vv[st]);
      }
      acc[st] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < KJ; ++j) acc[st] = qk_step(kf[j], qf[j], acc[st]);
    }
    uint2 pb[NT];
    float x[NT][4];
    const int last = min(lim, end - 1) - tb - 4 * g;
#pragma unroll
    for (int st = 0; st < NT; ++st)
#pragma unroll
      for (int v = 0; v < 4; ++v) x[st][v] = !masked || kTile * st + v <= last ? acc[st][v] : -INFINITY;
    soften<NT, DT>(x, a.scale_log2, s.m, s.l, s.o);
#pragma unroll
    for (int st = 0; st < NT; ++st)
      pb[st] = make_uint2(aia::pack_bf16x2(x[st][0], x[st][1]), aia::pack_bf16x2(x[st][2], x[st][3]));
    __builtin_amdgcn_wave_barrier();
    if (CARE && masked && __any(odd)) {
      for (int k = 0; k < NT * kTile; ++k) {
        const uint2 w = NT == 1 || k < kTile ? pb[0] : pb[NT - 1];
        const float p = weight_of(k & 2 ? w.y : w.x, n, k);
        if (tb + k <= lim && tb + k < end)
          add_key(s.o, p, [&](int dt) { return vt + k * kVStride + 16 * dt + 4 * g; });
      }
      __builtin_amdgcn_wave_barrier();
      return;
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const short4_t v0 = vt_frag(vt, n, g, dt);
      if constexpr (F8) {
        const short4_t v1 = vt_frag(vt + kTile * kVStride, n, g, dt);
        const bf16x8_t va = __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
        s.o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            va, as_b8(make_uint4(pb[0].x, pb[0].y, pb[1].x, pb[1].y)), s.o[dt], 0, 0, 0);
      } else {
        s.o[dt] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(v0, as_s4(pb[0].x, pb[0].y), s.o[dt], 0, 0, 0);
      }
    }
    __builtin_amdgcn_wave_barrier();
  };

  uint4 kbuf[NT][LD], vbuf[NT][LD];
  int at[NT];
  for (int t0 = p0 / kTile, t_end = (p1 + kTile - 1) / kTile; t0 < t_end;) {
    base = t0 * kTile / a.bs;
    bend = min(base + 64, entries);
    // tiles whose places all fall into the window (the last: up to p1)
    const int t1 = bend >= entries ? t_end : min(t_end, bend * a.bs / kTile);
    const int end = min(p1, t1 * kTile);
    // ids outside the pool are clamped, so that a bad table cannot fault
    ids = base + lane < bend ? min(max(id(base + lane), 0), a.nb - 1) : 0;
    if constexpr (F8) {
      const int64_t se = (int64_t)ids * a.hkv + kvh;
      sev = a.ks[se] | a.vs[se] << 8;
    }
#pragma unroll
    for (int st = 0; st < NT; ++st) load(t0 + st, kbuf[st], vbuf[st], at[st]);
    __builtin_amdgcn_sched_barrier(0);
    for (int t = t0; t < t1; t += NT) {
      compute(t, kbuf, vbuf, at, end);
#pragma unroll
      for (int st = 0; st < NT; ++st) load(t + NT + st, kbuf[st], vbuf[st], at[st]);
      __builtin_amdgcn_sched_barrier(0);
    }
    t0 = t1;
  }
}

}  // namespace
