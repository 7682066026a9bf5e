// One wave's attention of up to 16 query rows to a run of listed cache blocks: the
// inner loop of the block-sparse kernels.
//
// Keys are numbered by their place in the list (place p: block p / bs of the list,
// offset p % bs).  A wave takes them in steps of NT tiles of 16: S^T = K Q^T, an online
// softmax per row, O^T += V^T P^T.  No barriers: waves drift, so some load while others
// compute.  K of the next step is loaded behind the staging of this one's, V likewise,
// so a step's bytes are in flight during the math of the one before.
//
// Rows come in whole (neighbouring lanes take neighbouring 16-byte pieces) and pass
// through the wave's own LDS, K and V after each other in the same place, to where the
// MFMA wants them.  Loaded straight into K's operand registers, neighbouring lanes have
// different keys, and the L1 takes each lane's 16 bytes for an access of its own: it
// then delivers 16 bytes a clock, 9 TB/s on the chip, which caps what the L2 holds.
//
// What a step costs beyond its bytes is the softmax's bookkeeping and addresses, so it
// takes several tiles, and blocks of whole tiles (bs a multiple of 16) have their
// addresses in scalar registers.
#pragma once

#include "row_parts.h"

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

// Q operands: row n from qp (null: zeros).
template <int D>
__device__ __forceinline__ void load_q(const uint16_t* qp, int g, uint4 (&qf)[D / 32]) {
#pragma unroll
  for (int j = 0; j < D / 32; ++j) {
    qf[j] = make_uint4(0, 0, 0, 0);
    if (qp) qf[j] = reinterpret_cast<const uint4*>(qp)[4 * j + g];
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

// Attends places [p0, p1) (p0 a multiple of 16) with rows qf, which all see them all.
// id(i): the block id of list entry i, called with different i per lane, 0 <= i <
// entries.  lds: kStep values of the wave's own.  V behind p1 counts as zeros: a
// weight of zero times an infinity or NaN there would not be zero.
constexpr int kNt = 2;                           // tiles per step
constexpr int kStep = kNt * kTile * kVStride;        // K or V values of a step in LDS

template <int D, bool F8, bool WHOLE, class Id>
__device__ __forceinline__ void attend(const CacheArgs& a, int kvh, const uint4 (&qf)[D / 32], int p0, int p1,
                                       int entries, Id id, uint16_t* lds, int lane, RowState<D>& s) {
  constexpr int KJ = D / 32, DT = D / 16, CELL = F8 ? 1 : 2;
  constexpr int CPR = D * CELL / 16;         // 16-byte pieces of a key
  constexpr int RPL = 64 / CPR, LD = kTile / RPL;      // keys per load of the wave, loads per tile
  const int n = lane & 15, g = lane >> 4;
  const int lr = lane / CPR, lc = lane % CPR;          // this lane's key and piece of a load
  p0 = __builtin_amdgcn_readfirstlane(p0);
  p1 = __builtin_amdgcn_readfirstlane(p1);
  entries = __builtin_amdgcn_readfirstlane(entries);
  if (p0 >= p1) return;
  const int block_tiles = a.bs / kTile;      // of whole blocks
  const int row_bytes = a.hkv * D * CELL, head_bytes = kvh * D * CELL;
  const uint8_t* kc = reinterpret_cast<const uint8_t*>(a.kc) + head_bytes;
  const uint8_t* vc = reinterpret_cast<const uint8_t*>(a.vc) + head_bytes;
  int base = 0, bend = 0, ids = 0, sev = 0;  // list entries held by the lanes: [base, bend)
  int end = 0;                               // places of the window

  uint4 kk[kNt][LD], vv[kNt][LD];
  int64_t at[kNt][WHOLE ? 1 : LD];           // byte offsets of the rows being loaded
  uint32_t off[kNt][WHOLE ? LD : 1];
  uint32_t full[LD];                         // this lane's offsets in a tile
#pragma unroll
  for (int i = 0; i < LD; ++i) full[i] = (uint32_t)((i * RPL + lr) * row_bytes + 16 * lc);
  int le = 0, lt = 0;                        // whole blocks: the next tile's entry from base on, its place there
  int ek[kNt][WHOLE ? 1 : LD], ev[kNt][WHOLE ? 1 : LD];      // 8-bit caches: scales of the keys in kk, vv
  // Tiles behind the window read its first row again (an L1 hit); keys behind the end
  // the last one (never a slot that may hold stale bytes).
  auto load_k = [&](int t) {
#pragma unroll
    for (int st = 0; st < kNt; ++st) {
      const int first = (t + st) * kTile;
      const bool in = first < end;
      if (WHOLE) {
        const int e = in ? le : 0, blk = __builtin_amdgcn_readlane(ids, e);
        if (F8) ek[st][0] = __builtin_amdgcn_readlane(sev, e);
        at[st][0] = ((int64_t)blk * a.bs + (in ? lt * kTile : 0)) * row_bytes;
        // (the least of the offsets is that of the least of the rows)
        const uint32_t last = (uint32_t)((in ? min(end - 1 - first, kTile - 1) : 0) * row_bytes + 16 * lc);
#pragma unroll
        for (int i = 0; i < LD; ++i) {
          off[st][i] = min(full[i], last);
          kk[st][i] = *reinterpret_cast<const uint4*>(kc + at[st][0] + off[st][i]);
        }
        if (++lt == block_tiles) { lt = 0; ++le; }
      } else {
#pragma unroll
        for (int i = 0; i < LD; ++i) {
          const int p = in ? min(first + i * RPL + lr, end - 1) : base * a.bs, e = p / a.bs;
          const int blk = __shfl(ids, e - base);
          if (F8) ek[st][i] = __shfl(sev, e - base);
          at[st][i] = ((int64_t)blk * a.bs + (p - e * a.bs)) * row_bytes + 16 * lc;
          kk[st][i] = *reinterpret_cast<const uint4*>(kc + at[st][i]);
        }
      }
    }
  };
  auto load_v = [&]() {
#pragma unroll
    for (int st = 0; st < kNt; ++st)
#pragma unroll
      for (int i = 0; i < LD; ++i) {
        if (F8) ev[st][WHOLE ? 0 : i] = ek[st][WHOLE ? 0 : i];
        vv[st][i] = *reinterpret_cast<const uint4*>(vc + at[st][WHOLE ? 0 : i] + (WHOLE ? off[st][i] : 0));
      }
  };
  // rows of a tile into LDS, as bf16
  auto stage = [&](int st, const uint4 (&w)[LD], const int (&e8)[WHOLE ? 1 : LD], int shift) {
#pragma unroll
    for (int i = 0; i < LD; ++i) {
      uint16_t* to = lds + (st * kTile + i * RPL + lr) * kVStride;
      if constexpr (F8) {
        uint4 x[2];
        fp8_to_bf16(w[i], (e8[WHOLE ? 0 : i] >> shift) & 0xff, x);
        *reinterpret_cast<u32x4_t*>(to + 16 * lc) = as_u4(x[0]);
        *reinterpret_cast<u32x4_t*>(to + 16 * lc + 8) = as_u4(x[1]);
      } else {
        *reinterpret_cast<u32x4_t*>(to + 8 * lc) = as_u4(w[i]);
      }
    }
  };

  for (int t0 = p0 / kTile, t_end = (p1 + kTile - 1) / kTile; t0 < t_end;) {
    base = t0 * kTile / a.bs;
    bend = min(base + 64, entries);
    // tiles whose places all fall into the window (the last: up to p1)
    const int t1 = bend >= entries ? t_end : min(t_end, (int)((int64_t)bend * a.bs / kTile));
    end = min(p1, t1 * kTile);
    // ids outside the pool are clamped, so that a bad table cannot fault
    ids = base + lane < bend ? min(max(id(base + lane), 0), a.nb - 1) : 0;
    if (F8) {
      const int64_t se = (int64_t)ids * a.hkv + kvh;
      sev = a.ks[se] | a.vs[se] << 8;
    }
    le = 0;
    lt = WHOLE ? t0 - base * block_tiles : 0;
    load_k(t0);
    load_v();
    for (int t = t0; t < t1; t += kNt) {
      const int tb = t * kTile;
      const bool masked = tb + kNt * kTile > end;
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int st = 0; st < kNt; ++st) stage(st, kk[st], ek[st], 0);
      const bool more = t + kNt < t1;
      if (more) load_k(t + kNt);
      __builtin_amdgcn_wave_barrier();
      float4_t acc[kNt];
#pragma unroll
      for (int st = 0; st < kNt; ++st) {
        acc[st] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < KJ; ++j)
          acc[st] = qk_step(*reinterpret_cast<const uint4*>(lds + (st * kTile + n) * kVStride + 32 * j + 8 * g), qf[j], acc[st]);
      }
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int st = 0; st < kNt; ++st) {
        if (masked) {
#pragma unroll
          for (int i = 0; i < LD; ++i)
            if (tb + kTile * st + i * RPL + lr >= end) vv[st][i] = make_uint4(0, 0, 0, 0);
        }
        stage(st, vv[st], ev[st], 8);
      }
      if (more) load_v();
      __builtin_amdgcn_sched_barrier(0);
      float x[kNt][4];
      const int last = end - 1 - tb - 4 * g;
#pragma unroll
      for (int st = 0; st < kNt; ++st)
#pragma unroll
        for (int v = 0; v < 4; ++v) x[st][v] = !masked || kTile * st + v <= last ? acc[st][v] : -INFINITY;
      soften<kNt, DT>(x, a.scale_log2, s.m, s.l, s.o);
      uint4 pb[kNt / 2];
#pragma unroll
      for (int p = 0; p < kNt / 2; ++p)
        pb[p] = make_uint4(aia::pack_bf16x2(x[2 * p][0], x[2 * p][1]), aia::pack_bf16x2(x[2 * p][2], x[2 * p][3]),
                           aia::pack_bf16x2(x[2 * p + 1][0], x[2 * p + 1][1]), aia::pack_bf16x2(x[2 * p + 1][2], x[2 * p + 1][3]));
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int p = 0; p < kNt / 2; ++p)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const short4_t v0 = vt_frag(lds + 2 * p * kTile * kVStride, n, g, dt);
          const short4_t v1 = vt_frag(lds + (2 * p + 1) * kTile * kVStride, n, g, dt);
          const bf16x8_t va = __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
          s.o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, as_b8(pb[p]), s.o[dt], 0, 0, 0);
        }
    }
    t0 = t1;
  }
}

}  // namespace
