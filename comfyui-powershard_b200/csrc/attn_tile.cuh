// What the dense (attention.cu) and the block-sparse (sparse_attn.cu) forward
// kernels share: tile sizes, bounded waits, the UMMAs of a key tile and the
// online softmax of one query row (attention.cu's head describes both).
#pragma once

#include "ptx.cuh"
#include "ps_b200.h"
#include "internal.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace psb {
namespace attn {

constexpr int kBlockM = 128;
constexpr int kBlockN = 128;
constexpr int kHeadDim = 128;
constexpr int kKStages = 2;                          // K ring
constexpr int kVStages = 2;                          // V ring
constexpr int kTileBytes = kBlockN * kHeadDim * 2;   // 32 KiB: one Q, K or V tile
constexpr int kHalfTile = kTileBytes / 2;            // one 64-column SW128 half
constexpr int kThreads = 320;                        // 10 warps
constexpr int kSmemQ = 2 * kTileBytes;
constexpr int kSmemK = kKStages * kTileBytes;
constexpr int kSmemV = kVStages * kTileBytes;
// P_t is released to the PV UMMAs in kPParts parts of 128/kPParts keys, so
// the tensor pipe starts on the first keys while the softmax writes the rest.
#ifndef PSB_P_PARTS
#define PSB_P_PARTS 2
#endif
constexpr int kPParts = PSB_P_PARTS;
static_assert(kPParts == 1 || kPParts == 2 || kPParts == 4, "P parts: 1, 2 or 4");
constexpr int kChunksPerPart = 4 / kPParts;  // 32-key chunks per part

// Device status codes written on a bounded-wait timeout (first error wins).
enum Err : int {
  kErrQ = 101,
  kErrEmpty = 102,
  kErrFull = 103,
  kErrP = 104,
  kErrS = 105,
  kErrO = 106,
  kErrDrain = 107,
};

// Bounded wait whose outcome is uniform across the warp (a lane that timed
// out drags the whole warp out, so .sync.aligned tcgen05 ops stay converged).
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag,
                                          int* status, int code) {
  bool ok = mbar_wait(bar, parity, abort_flag, status, code);
  return __all_sync(0xffffffffu, ok);
}

// Wait used only while tearing down: ignores the abort flag (copies/UMMAs in
// flight must land before shared memory / TMEM is released) but is bounded.
__device__ __forceinline__ void drain_wait(uint32_t bar, uint32_t parity, int* status) {
  const uint64_t t0 = globaltimer();
  while (!mbar_try_wait(bar, parity)) {
    if (globaltimer() - t0 > kWaitLimitNs) {
      if (status) atomicCAS(status, 0, kErrDrain);
      return;
    }
  }
}

template <bool kFp16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  return kFp16 ? pack_f16x2(lo, hi) : pack_bf16x2(lo, hi);
}

__device__ __forceinline__ float row_max128(const float (&s)[128]) {
  float mx0 = -INFINITY, mx1 = -INFINITY, mx2 = -INFINITY, mx3 = -INFINITY;
#pragma unroll
  for (int j = 0; j < 128; j += 8) {
    mx0 = fmax3(mx0, s[j], s[j + 1]);
    mx1 = fmax3(mx1, s[j + 2], s[j + 3]);
    mx2 = fmax3(mx2, s[j + 4], s[j + 5]);
    mx3 = fmax3(mx3, s[j + 6], s[j + 7]);
  }
  return fmaxf(fmax3(mx0, mx1, mx2), mx3);
}

// The UMMAs of one key tile, for the issuing thread.
struct TileMma {
  uint32_t tmem, id_qk, id_pv;
  uint64_t dq0, dq1, dk, dv;
  // Descriptor bases; per-UMMA offsets are added to the start-address field
  // (all shared addresses stay below 256 KiB, so the 14-bit field never carries).
  template <bool kFp16>
  __device__ __forceinline__ static TileMma make(uint32_t tmem, const uint8_t* sQ, const uint8_t* sK, const uint8_t* sV) {
    TileMma m;
    m.tmem = tmem;
    m.id_qk = idesc_f16(kBlockM, kBlockN, !kFp16, false, false);
    m.id_pv = idesc_f16(kBlockM, kHeadDim, !kFp16, false, true);
    m.dq0 = sdesc_sw128(smem_u32(sQ), 16, 1024);
    m.dq1 = sdesc_sw128(smem_u32(sQ + kTileBytes), 16, 1024);
    m.dk = sdesc_sw128(smem_u32(sK), 16, 1024);
    m.dv = sdesc_sw128(smem_u32(sV), kHalfTile, 1024);
    return m;
  }
  // S_t = Q_q K^T with the K tile of stage st.
  __device__ __forceinline__ void s(int t, int st) const { s(t, t, st); }
  __device__ __forceinline__ void s(int t, int q, int st) const {
    const uint64_t dq = q ? dq1 : dq0;
    const uint64_t dks = dk + static_cast<uint64_t>(st * (kTileBytes >> 4));
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      const uint32_t off = ((s >> 2) * kHalfTile + (s & 3) * 32) >> 4;
      umma_ss(tmem + 128 * t, dq + off, dks + off, id_qk, s > 0);
    }
  }
  // O_t (+)= P_t V for the keys of part q (8/kPParts UMMAs of K=16).
  __device__ __forceinline__ void pv(int t, int st, int q, bool accumulate) const {
    const uint64_t dvs = dv + static_cast<uint64_t>(st * (kTileBytes >> 4));
#pragma unroll
    for (int k = 0; k < 8 / kPParts; ++k) {
      const int s = (8 / kPParts) * q + k;
      umma_ts(tmem + 256 + 128 * t, tmem + 128 * t + s * 8, dvs + ((s * 2048) >> 4), id_pv,
              (accumulate || s > 0) ? 1u : 0u);
    }
  }
};

// Online softmax of one query row over the 128 scores of a key tile: updates
// the running max m and sum l, writes P over S and rescales O when the max
// rose.  bar_ph: first of the barriers of the leading parts of P, bar_p: of P.
// Scaling and sums go in pairs (the same bits with half the instructions:
// 1.0-1.4 % of a launch at the power limit, nothing of a short one).
// kQuarter: every fourth pair of exponentials is computed on the FMA pipe, which
// is idle next to the MUFU (8 cycles a warp and exponential, as many cycles a
// key tile as its UMMAs): 7 % of a launch, in steps 1/8 4 %, 5/16 6 %, 3/8 3 %,
// 1/2 -4 %.  Its relative error, 7.5e-5, lies below the rounding of P (half a
// step: 2^-8 of bf16, 2^-11 of fp16).
template <bool kFp16, bool kMasked, bool kQuarter>
__device__ __forceinline__ void softmax_row(const float (&s)[128], bool first, float scale_log2,
                                            uint32_t s_addr, uint32_t o_addr, uint32_t bar_ph, uint32_t bar_p,
                                            float& m, float& l) {
  float alpha = 1.f, sum;
  bool rescale = false;
  // Row max first (lazy running max: raised warp-uniformly only when it
  // grew by > 8), then the exponentials.
  const float m_tile = row_max128(s) * scale_log2;
  if (first) {
    // A tile without a key in use (kMasked only) leaves every score at -inf: a
    // finite maximum makes its exponentials 0 instead of NaN.
    m = kMasked ? fmaxf(m_tile, -1e30f) : m_tile;
  } else if (__any_sync(0xffffffffu, m_tile - m > 8.f)) {
    const float m_new = fmaxf(m, m_tile);
    alpha = ex2_approx(m - m_new);
    m = m_new;
    rescale = true;
  }
  {
    float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      uint32_t pk[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        float x0, x1;
        fma2(x0, x1, s[32 * c + 2 * j], s[32 * c + 2 * j + 1], scale_log2, -m);
        float p0, p1;
        if (kQuarter && j % 4 == 2) {
          ex2_pair(p0, p1, x0, x1);
        } else {
          p0 = ex2_approx(x0);
          p1 = ex2_approx(x1);
        }
        add2(sum0, sum1, p0, p1);
        pk[j] = pack2<kFp16>(p0, p1);
      }
      tmem_st16(s_addr + 16 * c, pk);
      if (c == (kPParts > 1 ? kChunksPerPart - 1 : 3)) {
        // The rare O rescale goes here, before the first PV part of this
        // tile is released (O_t's last update completed before S_t was
        // signalled); the row's first chunks are dead by now.
        if (rescale) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t o[32];
            tmem_ld32(o_addr + 32 * q, o);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
            tmem_st32(o_addr + 32 * q, o);
          }
        }
      }
      if ((c + 1) % kChunksPerPart == 0 && c < 3) {  // part (c+1)/kChunksPerPart - 1 written
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(bar_ph + 8 * ((c + 1) / kChunksPerPart - 1));
      }
    }
    sum = sum0 + sum1;
  }
  l = fmaf(l, alpha, sum);
  tmem_wait_st();
  tc_fence_before();
  mbar_arrive(bar_p);
}

// Merges the parts of split unit u for 8 columns from c of row r of its query
// tile t: acc = sum_p w_p o_p with w_p = 2^(m_p - max m) l_p, or 2^(lse_p - max lse) where
// the parts hold their logarithm; returns 1 / sum_p w_p.
__device__ __forceinline__ float merge_parts(const AttnArgs& args, int u, int t, int r, int c, float (&acc)[8]) {
  const int S = args.split;
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[j] = 0.f;
  float mx = -INFINITY;
  auto m_and_l = [&](int p) {
    const int at = ((u * S + p) * 2 + t) * kBlockM + r;
    return args.ws_ml ? args.ws_ml[at] : make_float2(args.ws_lse[at], 1.f);
  };
#pragma unroll 4
  for (int p = 0; p < S; ++p) mx = fmaxf(mx, m_and_l(p).x);
  float wsum = 0.f;
#pragma unroll 4
  for (int p = 0; p < S; ++p) {
    const float2 ml = m_and_l(p);
    const float w = ml.x == -INFINITY ? 0.f : ex2_approx(ml.x - mx) * ml.y;
    wsum += w;
    const float4* src = reinterpret_cast<const float4*>(
        args.ws_o + ((static_cast<int64_t>(u * S + p) * 2 + t) * kBlockM + r) * kHeadDim + c);
    const float4 a0 = src[0], a1 = src[1];
    acc[0] = fmaf(w, a0.x, acc[0]);
    acc[1] = fmaf(w, a0.y, acc[1]);
    acc[2] = fmaf(w, a0.z, acc[2]);
    acc[3] = fmaf(w, a0.w, acc[3]);
    acc[4] = fmaf(w, a1.x, acc[4]);
    acc[5] = fmaf(w, a1.y, acc[5]);
    acc[6] = fmaf(w, a1.z, acc[6]);
    acc[7] = fmaf(w, a1.w, acc[7]);
  }
  return wsum > 0.f ? 1.f / wsum : 0.f;
}

}  // namespace attn
}  // namespace psb
