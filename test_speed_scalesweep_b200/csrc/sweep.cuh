// The scale sweep of one 16-element block, shared by every kernel that
// quantizes: candidate errors, the window's argmin, block amax and the tables
// of E4M3 scales they read; and division by a launch constant.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "ptx.cuh"
#include "quant.cuh"

namespace ssw {

constexpr int kLower = -3;       // bench_kernel/scalesweep_mse_nvfp4_utils.py:17
constexpr int kWindow = 11;      // UPPER_BOUND - LOWER_BOUND + 1 (:17-18, :452-454)
constexpr int kMaxRaw = 126;     // REF_MAX_SCALE_RAW (:20)
constexpr int kWindowTab = 128 + kWindow;  // window positions j = code + 3, code in [-3, 134]

struct ScaleEntry {
  float inv;  // 1 / s, IEEE (equals the reference's Triton 1.0 / s for every code)
  float s2;   // s * s (exact)
};

__device__ __forceinline__ int clamp_raw(int r) { return r < 1 ? 1 : (r > kMaxRaw ? kMaxRaw : r); }

// Squared error of the 16 values for two candidate reciprocals at once.
// Returns {sse_a, sse_b} packed.
template <int kVariant>
__device__ __forceinline__ uint64_t sse_pair(const uint64_t (&vp)[8], float inv_a, float inv_b) {
  const uint64_t ia = pack2(inv_a, inv_a), ib = pack2(inv_b, inv_b);
  if constexpr (kVariant == kVariantMse) {
    uint64_t acc = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      float xa0, xa1, xb0, xb1, da0, da1, db0, db1;
      unpack2(mul2(vp[k], ia), xa0, xa1);
      unpack2(mul2(vp[k], ib), xb0, xb1);
      e2m1_delta2(xa0, xa1, da0, da1);
      e2m1_delta2(xb0, xb1, db0, db1);
      const uint64_t d0 = pack2(da0, db0), d1 = pack2(da1, db1);
      acc = (k == 0) ? mul2(d0, d0) : fma2(d0, d0, acc);
      acc = fma2(d1, d1, acc);
    }
    return acc;
  } else if constexpr (kVariant == kVariantWeighted) {
    // Squares rounded on their own, then summed in element order (importance
    // weights of 1: fma(d^2, 1, acc) == add(d^2, acc)).  Scalar mul.rn /
    // add.rn on purpose: a packed f32x2 multiply feeding a packed add may be
    // fused into one FMA, which rounds differently from the reference.
    float acc_a = 0.0f, acc_b = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      float xa0, xa1, xb0, xb1, da0, da1, db0, db1;
      unpack2(mul2(vp[k], ia), xa0, xa1);
      unpack2(mul2(vp[k], ib), xb0, xb1);
      e2m1_delta2(xa0, xa1, da0, da1);
      e2m1_delta2(xb0, xb1, db0, db1);
      const float sa0 = mul_rn(da0, da0), sa1 = mul_rn(da1, da1);
      const float sb0 = mul_rn(db0, db0), sb1 = mul_rn(db1, db1);
      acc_a = (k == 0) ? add_rn(sa1, sa0) : add_rn(sa1, add_rn(sa0, acc_a));
      acc_b = (k == 0) ? add_rn(sb1, sb0) : add_rn(sb1, add_rn(sb0, acc_b));
    }
    return pack2(acc_a, acc_b);
  } else {
    uint64_t s[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      float xa0, xa1, xb0, xb1, da0, da1, db0, db1;
      unpack2(mul2(vp[k], ia), xa0, xa1);
      unpack2(mul2(vp[k], ib), xb0, xb1);
      e2m1_delta2(xa0, xa1, da0, da1);
      e2m1_delta2(xb0, xb1, db0, db1);
      const uint64_t d0 = pack2(da0, db0), d1 = pack2(da1, db1);
      s[k] = fma2(d1, d1, mul2(d0, d0));
    }
    return add2(add2(add2(s[0], s[1]), add2(s[2], s[3])), add2(add2(s[4], s[5]), add2(s[6], s[7])));
  }
}

// Single-candidate squared error (the odd candidate of the 11-wide window).
template <int kVariant>
__device__ __forceinline__ float sse_one(const uint64_t (&vp)[8], float inv) {
  const uint64_t i2 = pack2(inv, inv);
  if constexpr (kVariant == kVariantMse) {
    float acc = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      float x0, x1, d0, d1;
      unpack2(mul2(vp[k], i2), x0, x1);
      e2m1_delta2(x0, x1, d0, d1);
      acc = (k == 0) ? mul_rn(d0, d0) : fma_rn(d0, d0, acc);
      acc = fma_rn(d1, d1, acc);
    }
    return acc;
  } else if constexpr (kVariant == kVariantWeighted) {
    float acc = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      float x0, x1, d0, d1;
      unpack2(mul2(vp[k], i2), x0, x1);
      e2m1_delta2(x0, x1, d0, d1);
      const float s0 = mul_rn(d0, d0), s1 = mul_rn(d1, d1);
      acc = (k == 0) ? add_rn(s1, s0) : add_rn(s1, add_rn(s0, acc));
    }
    return acc;
  } else {
    float s[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      float x0, x1, d0, d1;
      unpack2(mul2(vp[k], i2), x0, x1);
      e2m1_delta2(x0, x1, d0, d1);
      s[k] = fma_rn(d1, d1, mul_rn(d0, d0));
    }
    return add_rn(add_rn(add_rn(s[0], s[1]), add_rn(s[2], s[3])),
                  add_rn(add_rn(s[4], s[5]), add_rn(s[6], s[7])));
  }
}

__device__ __forceinline__ void consider(float mse, int raw, float& best, int& best_raw) {
  // strict '<': NaN never wins and ties keep the earlier (lower-index) candidate
  if (mse < best) {
    best = mse;
    best_raw = raw;
  }
}

__device__ __forceinline__ void consider_pair(uint64_t sse, float s2a, float s2b, int ra, int rb,
                                              float& best, int& best_raw) {
  float ma, mb;
  unpack2(mul2(sse, pack2(s2a, s2b)), ma, mb);
  consider(ma, ra, best, best_raw);
  consider(mb, rb, best, best_raw);
}

// Block |x| maximum straight from the 16-bit inputs.  max.xorsign.abs.{bf16,f16}x2
// keeps the larger magnitude of each lane and ignores NaN operands, like the
// reference's tl.maximum(tl.abs(a), tl.abs(b)).  Because rounding is
// monotonic, max_j |RN(x_j * g)| == RN(max_j |x_j| * |g|) for every block
// whose normalised values hold no NaN; a block holding a NaN has a NaN
// squared error for every candidate, so its scale does not depend on amax.
template <int kDType>
__device__ __forceinline__ float block_absmax_raw(const uint32_t (&w)[8]) {
  uint32_t a[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (kDType == kDTypeBF16)
      asm("max.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(a[j]) : "r"(w[2 * j]), "r"(w[2 * j + 1]));
    else
      asm("max.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(a[j]) : "r"(w[2 * j]), "r"(w[2 * j + 1]));
  }
  uint32_t b0, b1, c;
  if constexpr (kDType == kDTypeBF16) {
    asm("max.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(b0) : "r"(a[0]), "r"(a[1]));
    asm("max.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(b1) : "r"(a[2]), "r"(a[3]));
    asm("max.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(c) : "r"(b0), "r"(b1));
    const float lo = __uint_as_float((c & 0x7FFFu) << 16);
    const float hi = __uint_as_float(c & 0x7FFF0000u);
    return fmaxf(lo, hi);
  } else {
    asm("max.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(b0) : "r"(a[0]), "r"(a[1]));
    asm("max.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(b1) : "r"(a[2]), "r"(a[3]));
    asm("max.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(c) : "r"(b0), "r"(b1));
    const float lo = __half2float(__ushort_as_half((unsigned short)(c & 0x7FFFu)));
    const float hi = __half2float(__ushort_as_half((unsigned short)((c >> 16) & 0x7FFFu)));
    return fmaxf(lo, hi);
  }
}

// Unsigned 32-bit division by the per-launch constant bpc_out:
// q = (umulhi(n, magic) + n) >> shift (Granlund & Montgomery 1994, round-up
// multiplier; the 33-bit sum is formed in 64 bits).
__device__ __forceinline__ uint32_t div_bpc(uint32_t n, uint32_t magic, uint32_t shift) {
  return (uint32_t)(((uint64_t)__umulhi(n, magic) + n) >> shift);
}

// Lexicographic (mse, index) minimum of two partial sweeps; index -1 = no
// winner.  Merging the per-lane winners of disjoint candidate subsets this way
// gives the sequential strict-'<' scan's result: the smallest mse, the lowest
// index among equal ones, NaN and +inf never winning.
__device__ __forceinline__ void merge_best(float& best, int& bi, float ob, int oi) {
  if (oi >= 0 && (bi < 0 || ob < best || (ob == best && oi < bi))) {
    best = ob;
    bi = oi;
  }
}

// The window's winner for a block of normalised values: the E4M3 code among
// base - 3 .. base + 7 (clamped to 1..126) with the smallest mean squared
// error, the lowest on ties, 0 when none wins (a NaN in the block).  With
// kLanes > 1 each of the block's lanes passes its own `sub` and evaluates the
// candidates i = sub, sub + kLanes, ...; all of the warp must call.
template <int kVariant, int kLanes>
__device__ __forceinline__ int window_best(const uint64_t (&vp)[8], int base_raw,
                                           const ScaleEntry* tabw, uint32_t sub) {
  const ScaleEntry* wt = tabw + base_raw;  // candidate i -> wt[i]
  float best = __uint_as_float(0x7F800000u);
  int bi = -1;
  if constexpr (kLanes > 1) {
    constexpr int kSlots = (kWindow + kLanes - 1) / kLanes;  // 3 (4 lanes) or 6 (2 lanes)
#pragma unroll
    for (int t = 0; t + 1 < kSlots; t += 2) {
      // the last lane's final slot may fall past the window: evaluated, never considered
      const int ia = (int)sub + t * kLanes, ib = (int)sub + (t + 1) * kLanes;
      const ScaleEntry ea = wt[min(ia, kWindow - 1)], eb = wt[min(ib, kWindow - 1)];
      float ma, mb;
      unpack2(mul2(sse_pair<kVariant>(vp, ea.inv, eb.inv), pack2(ea.s2, eb.s2)), ma, mb);
      if (ia < kWindow) consider(ma, ia, best, bi);
      if (ib < kWindow) consider(mb, ib, best, bi);
    }
    if constexpr (kSlots % 2) {
      const int i = (int)sub + (kSlots - 1) * kLanes;
      const ScaleEntry e = wt[min(i, kWindow - 1)];
      const float mm = mul_rn(sse_one<kVariant>(vp, e.inv), e.s2);
      if (i < kWindow) consider(mm, i, best, bi);
    }
#pragma unroll
    for (int off = 1; off < kLanes; off <<= 1)
      merge_best(best, bi, __shfl_xor_sync(0xFFFFFFFFu, best, off),
                 __shfl_xor_sync(0xFFFFFFFFu, bi, off));
  } else {
#pragma unroll
    for (int i = 0; i + 1 < kWindow; i += 2) {
      const ScaleEntry ea = wt[i], eb = wt[i + 1];
      consider_pair(sse_pair<kVariant>(vp, ea.inv, eb.inv), ea.s2, eb.s2, i, i + 1, best, bi);
    }
    const ScaleEntry e = wt[kWindow - 1];
    consider(mul_rn(sse_one<kVariant>(vp, e.inv), e.s2), kWindow - 1, best, bi);
  }
  return bi < 0 ? 0 : clamp_raw(base_raw + kLower + bi);
}

}  // namespace ssw
