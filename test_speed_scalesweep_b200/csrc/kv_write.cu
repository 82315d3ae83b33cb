// Rotary positions and the scale-sweep quantization of keys and values into
// the pages of an NVFP4 cache (layout in kv.cuh), and the reverse gather.
//
//   rotary, pairs (a, b) = (x[i], x[i + r/2]) or (x[2i], x[2i + 1]), i < r/2:
//     a' = a cos - b sin,  b' = b cos + a sin
//   formed in binary32 (both products and their sum rounded) and rounded once
//   to the input type: the bytes of the cache are those that the scalesweep_mse
//   quantizer writes for the rotated 16-bit keys.
//
// Two kinds of CTAs share one launch, spread evenly over the grid, since they
// are bound by different things: the quantizing ones by the FP32 and conversion
// pipes (35 operations per element, as in quant.cu), the query ones by HBM.
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "kv.cuh"
#include "ptx.cuh"
#include "quant.cuh"
#include "sweep.cuh"

namespace ssw {
namespace kv {
namespace {

constexpr int kThreads = 256;  // the shared tables rely on it

__device__ __forceinline__ uint4 ld16(const uint16_t* p) {
  return *reinterpret_cast<const uint4*>(p);
}

template <int kDType>
__device__ __forceinline__ void widen(uint32_t w, float& lo, float& hi) {
  if constexpr (kDType == kDTypeBF16) {
    lo = __uint_as_float(w << 16);
    hi = __uint_as_float(w & 0xFFFF0000u);
  } else {
    lo = __half2float(__ushort_as_half((unsigned short)(w & 0xFFFF)));
    hi = __half2float(__ushort_as_half((unsigned short)(w >> 16)));
  }
}

template <int kDType>
__device__ __forceinline__ uint32_t narrow(float lo, float hi) {
  if constexpr (kDType == kDTypeBF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// own * cos + sign * other * sin for 8 elements of the half layout: sign -1 in
// the first half of the rotated part, +1 in the second.
template <int kDType>
__device__ __forceinline__ void rotate_half8(uint4& own, const uint4& other, const float* cs,
                                             int half, bool first) {
  uint32_t* o = reinterpret_cast<uint32_t*>(&own);
  const uint32_t* t = reinterpret_cast<const uint32_t*>(&other);
  float c[8], s[8];
  *reinterpret_cast<float4*>(c) = *reinterpret_cast<const float4*>(cs);
  *reinterpret_cast<float4*>(c + 4) = reinterpret_cast<const float4*>(cs)[1];
  *reinterpret_cast<float4*>(s) = *reinterpret_cast<const float4*>(cs + half);
  *reinterpret_cast<float4*>(s + 4) = reinterpret_cast<const float4*>(cs + half)[1];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float a0, a1, b0, b1;
    widen<kDType>(o[j], a0, a1);
    widen<kDType>(t[j], b0, b1);
    float p0 = mul_rn(b0, s[2 * j]), p1 = mul_rn(b1, s[2 * j + 1]);
    if (first) {
      p0 = -p0;
      p1 = -p1;
    }
    o[j] = narrow<kDType>(add_rn(mul_rn(a0, c[2 * j]), p0), add_rn(mul_rn(a1, c[2 * j + 1]), p1));
  }
}

// 8 pairs with the cosines and sines at hand: (x[j], y[j]) in the half layout,
// neighbours within x, then within y, in the interleaved one.
template <int kDType, bool kNeox>
__device__ __forceinline__ void rotate_pairs(uint4& x, uint4& y, const float (&c)[8],
                                             const float (&s)[8]) {
  uint32_t* a = reinterpret_cast<uint32_t*>(&x);
  uint32_t* b = reinterpret_cast<uint32_t*>(&y);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (kNeox) {
      float a0, a1, b0, b1;
      widen<kDType>(a[j], a0, a1);
      widen<kDType>(b[j], b0, b1);
      const float c0 = c[2 * j], c1 = c[2 * j + 1], s0 = s[2 * j], s1 = s[2 * j + 1];
      a[j] = narrow<kDType>(add_rn(mul_rn(a0, c0), -mul_rn(b0, s0)),
                            add_rn(mul_rn(a1, c1), -mul_rn(b1, s1)));
      b[j] = narrow<kDType>(add_rn(mul_rn(b0, c0), mul_rn(a0, s0)),
                            add_rn(mul_rn(b1, c1), mul_rn(a1, s1)));
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t* w = h ? b : a;
        float u, v;
        widen<kDType>(w[j], u, v);
        w[j] = narrow<kDType>(add_rn(mul_rn(u, c[4 * h + j]), -mul_rn(v, s[4 * h + j])),
                              add_rn(mul_rn(v, c[4 * h + j]), mul_rn(u, s[4 * h + j])));
      }
    }
  }
}

// 4 interleaved pairs.
template <int kDType>
__device__ __forceinline__ void rotate_pairs4(uint4& x, const float* cs, int half) {
  uint32_t* w = reinterpret_cast<uint32_t*>(&x);
  float c[4], s[4];
  *reinterpret_cast<float4*>(c) = *reinterpret_cast<const float4*>(cs);
  *reinterpret_cast<float4*>(s) = *reinterpret_cast<const float4*>(cs + half);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float a, b;
    widen<kDType>(w[j], a, b);
    w[j] = narrow<kDType>(add_rn(mul_rn(a, c[j]), -mul_rn(b, s[j])),
                          add_rn(mul_rn(b, c[j]), mul_rn(a, s[j])));
  }
}

// Query heads per thread: they share the position's cosines and sines (64
// bytes for 32 bytes of a head), and their loads are in flight together (8192
// tokens of 32 + 8 heads of 128: 69.7 us with one, 61.4 with two, 59.4 with four).
constexpr int kQHeads = 4;

struct KernelArgs {
  WriteArgs a;
  uint32_t kv_ctas, q_ctas;
  uint32_t kv_units, q_units;             // 16-element units: of keys and values, of queries
  uint32_t kv_magic, kv_shift;            // division by a token's kv units
  uint32_t q_magic, q_shift;              // division by a token's query units
  uint32_t kv_per_token, q_per_token;
  int d16_shift, page_shift;              // log2(head_size / 16), log2(page_size)
};

template <int kDType, bool kNeox, int kLanes>
__device__ __forceinline__ void quantize_units(const KernelArgs& g, uint32_t cta,
                                               const ScaleEntry* tab, const ScaleEntry* tabw) {
  const WriteArgs& p = g.a;
  const int half = p.rotary_dim >> 1;
  const uint32_t sub = threadIdx.x % kLanes;
  const float mult_k = *p.cache.multiplier, mult_v = p.cache.multiplier[1];
  // Whole warps stay in the loop: the lanes of a shared unit exchange winners.
  constexpr uint32_t kPerCta = kThreads / kLanes;
  const uint32_t warp_first = (threadIdx.x & ~31u) / kLanes;
  for (uint64_t first = (uint64_t)cta * kPerCta; first + warp_first < g.kv_units;
       first += (uint64_t)g.kv_ctas * kPerCta) {
    const uint64_t u64 = first + threadIdx.x / kLanes;
    const bool in = u64 < g.kv_units;
    const uint32_t u = in ? (uint32_t)u64 : 0;
    const uint32_t token = div_bpc(u, g.kv_magic, g.kv_shift);
    uint32_t r = u - token * g.kv_per_token;
    const uint32_t block = r & ((1u << g.d16_shift) - 1);
    r >>= g.d16_shift;
    const bool is_value = r >= (uint32_t)p.cache.kv_heads;
    const uint32_t head = is_value ? r - p.cache.kv_heads : r;
    const int64_t slot = p.slots[token];
    const int64_t pos = p.positions[token];
    const bool write = in && slot >= 0 && (slot >> g.page_shift) < p.cache.num_pages &&
                       (uint64_t)pos < (uint64_t)p.max_position;
    uint4 x[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
    if (write) {
      const Heads& h = is_value ? p.v : p.k;
      const uint16_t* src = h.p + (int64_t)token * h.token_stride + (int64_t)head * h.head_stride;
      const int e0 = (int)block * 16;
      x[0] = ld16(src + e0);
      x[1] = ld16(src + e0 + 8);
      if (!is_value) {
        const float* cs = p.cos_sin + pos * p.rotary_dim;
        if constexpr (kNeox) {
          uint4 other[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int e = e0 + 8 * j;
            if (e < p.rotary_dim) other[j] = ld16(src + (e < half ? e + half : e - half));
          }
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int e = e0 + 8 * j;
            if (e < p.rotary_dim)
              rotate_half8<kDType>(x[j], other[j], cs + (e < half ? e : e - half), half, e < half);
          }
        } else if (e0 < p.rotary_dim) {
          rotate_pairs4<kDType>(x[0], cs + e0 / 2, half);
          rotate_pairs4<kDType>(x[1], cs + e0 / 2 + 4, half);
        }
      }
    }
    const uint32_t w[8] = {x[0].x, x[0].y, x[0].z, x[0].w, x[1].x, x[1].y, x[1].z, x[1].w};
    const float mult = is_value ? mult_v : mult_k;
    const uint64_t m2 = pack2(mult, mult);
    uint64_t vp[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float lo, hi;
      widen<kDType>(w[j], lo, hi);
      vp[j] = mul2(pack2(lo, hi), m2);
    }
    const float amax = mul_rn(block_absmax_raw<kDType>(w), fabsf(mult));
    const int base_raw = min((int)e4m3_code(mul_rn(amax, (float)(1.0 / 6.0))), 127);
    const int best_raw = window_best<kVariantMse, kLanes>(vp, base_raw, tabw, sub);
    const float inv = tab[best_raw].inv;
    const uint64_t i2 = pack2(inv, inv);
    float y[16];
#pragma unroll
    for (int j = 0; j < 8; ++j) unpack2(mul2(vp[j], i2), y[2 * j], y[2 * j + 1]);
    const uint32_t lo_word = e2m1x8(y[0], y[1], y[2], y[3], y[4], y[5], y[6], y[7]);
    const uint32_t hi_word = e2m1x8(y[8], y[9], y[10], y[11], y[12], y[13], y[14], y[15]);
    if (write && sub == 0) {
      const int64_t page = slot >> g.page_shift;
      const int64_t row =
          (((int64_t)(is_value ? p.cache.kv_heads : 0) + head) << g.page_shift) +
          (slot & ((1 << g.page_shift) - 1));
      const int64_t at = (row << g.d16_shift) + block;
      st_v2(p.cache.codes + page * p.cache.codes_page_stride + at * 8, lo_word, hi_word);
      p.cache.scales[page * p.cache.scales_page_stride + at] = (uint8_t)best_raw;
    }
  }
}

// One unit: 8 pairs of the rotated part (or 16 elements behind it) of kQHeads heads.
template <int kDType, bool kNeox>
__device__ __forceinline__ void rotate_query_unit(const KernelArgs& g, uint32_t cta) {
  const WriteArgs& p = g.a;
  const uint64_t u64 = (uint64_t)cta * kThreads + threadIdx.x;
  if (u64 >= g.q_units) return;
  const uint32_t u = (uint32_t)u64;
  const uint32_t token = div_bpc(u, g.q_magic, g.q_shift);
  const uint32_t r = u - token * g.q_per_token;
  const int unit = (int)(r & ((1u << g.d16_shift) - 1));
  const int head = (int)(r >> g.d16_shift) * kQHeads;
  const int half = p.rotary_dim >> 1;
  const bool turn = unit * 16 < p.rotary_dim;
  const int o1 = kNeox && turn ? unit * 8 : unit * 16;
  const int o2 = kNeox && turn ? o1 + half : o1 + 8;
  const uint16_t* src =
      p.q.p + (int64_t)token * p.q.token_stride + (int64_t)head * p.q.head_stride;
  uint16_t* dst = p.q_out.p + (int64_t)token * p.q_out.token_stride +
                  (int64_t)head * p.q_out.head_stride;
  const int64_t pos = p.positions[token];
  const bool known = (uint64_t)pos < (uint64_t)p.max_position;
  // plain loads: the output may be the query itself
  uint4 x[kQHeads], y[kQHeads];
#pragma unroll
  for (int h = 0; h < kQHeads; ++h)
    if (head + h < p.q_heads) {
      x[h] = *reinterpret_cast<const uint4*>(src + h * p.q.head_stride + o1);
      y[h] = *reinterpret_cast<const uint4*>(src + h * p.q.head_stride + o2);
    }
  float c[8], s[8];
  if (turn && known) {
    // in the half layout pair i's angle is the table's i; in the interleaved
    // one elements 2i and 2i + 1 are pair i
    const float* cs = p.cos_sin + pos * p.rotary_dim + (kNeox ? o1 : o1 / 2);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      *reinterpret_cast<float4*>(c + 4 * j) = reinterpret_cast<const float4*>(cs)[j];
      *reinterpret_cast<float4*>(s + 4 * j) = reinterpret_cast<const float4*>(cs + half)[j];
    }
  }
#pragma unroll
  for (int h = 0; h < kQHeads; ++h)
    if (head + h < p.q_heads) {
      if (!known)
        x[h] = y[h] = make_uint4(0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu);  // NaN in both types
      else if (turn)
        rotate_pairs<kDType, kNeox>(x[h], y[h], c, s);
      *reinterpret_cast<uint4*>(dst + h * p.q_out.head_stride + o1) = x[h];
      *reinterpret_cast<uint4*>(dst + h * p.q_out.head_stride + o2) = y[h];
    }
}

template <int kDType, bool kNeox, int kLanes>
__global__ void __launch_bounds__(kThreads, 4) write_kernel(const KernelArgs g) {
  // CTA b is the query's when the evenly spread count of query CTAs steps at b
  const uint64_t total = (uint64_t)g.kv_ctas + g.q_ctas;
  const uint32_t before = (uint32_t)((uint64_t)blockIdx.x * g.q_ctas / total);
  const uint32_t after = (uint32_t)(((uint64_t)blockIdx.x + 1) * g.q_ctas / total);
  if (after != before) {
    wait_for_predecessor();
    let_successor_start();
    rotate_query_unit<kDType, kNeox>(g, before);
    return;
  }
  __shared__ ScaleEntry tab[128];
  __shared__ ScaleEntry tabw[kWindowTab];
  const uint32_t c = threadIdx.x;
  if (c < 128) {
    const float mag = e4m3_value(c);
    float inv;
    asm("rcp.rn.f32 %0, %1;" : "=f"(inv) : "f"(mag));
    tab[c] = ScaleEntry{inv, mul_rn(mag, mag)};
  }
  if (c < kWindowTab) {
    const float s = e4m3_value((uint32_t)clamp_raw((int)c + kLower));
    float inv;
    asm("rcp.rn.f32 %0, %1;" : "=f"(inv) : "f"(s));
    tabw[c] = ScaleEntry{inv, mul_rn(s, s)};
  }
  __syncthreads();
  wait_for_predecessor();
  let_successor_start();
  quantize_units<kDType, kNeox, kLanes>(g, blockIdx.x - before, tab, tabw);
}

// One thread reads one block (8 bytes of codes, a scale) of one token, head and
// side and writes 16 values: RN16(RN32(code * RN32(scale / multiplier))).  One
// division per block: one per element made the kernel twice as long as its
// bytes (32 us for 8192 tokens of 8 heads of 128).
template <int kDType>
__global__ void __launch_bounds__(kThreads) gather_kernel(const GatherArgs p, uint32_t units,
                                                          uint32_t per_token, uint32_t magic,
                                                          uint32_t shift, int d16_shift,
                                                          int page_shift) {
  wait_for_predecessor();
  let_successor_start();
  const uint64_t u64 = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
  if (u64 >= units) return;
  const uint32_t u = (uint32_t)u64;
  const uint32_t token = div_bpc(u, magic, shift);
  const uint32_t r = u - token * per_token;
  const uint32_t block = r & ((1u << d16_shift) - 1);
  const uint32_t side_head = r >> d16_shift;
  const bool is_value = side_head >= (uint32_t)p.cache.kv_heads;
  const uint32_t head = is_value ? side_head - p.cache.kv_heads : side_head;
  const int64_t slot = p.slots[token];
  uint32_t w[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (slot >= 0 && (slot >> page_shift) < p.cache.num_pages) {
    const int64_t page = slot >> page_shift;
    const int64_t row = ((int64_t)side_head << page_shift) + (slot & ((1 << page_shift) - 1));
    const int64_t at = (row << d16_shift) + block;
    const uint2 c = *reinterpret_cast<const uint2*>(
        p.cache.codes + page * p.cache.codes_page_stride + at * 8);
    uint32_t s2;  // the scale as f16, exact
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;"
        : "=r"(s2)
        : "h"((uint16_t)p.cache.scales[page * p.cache.scales_page_stride + at]));
    const float s = __fdiv_rn(__low2float(*reinterpret_cast<const __half2*>(&s2)),
                              p.cache.multiplier[is_value ? 1 : 0]);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint32_t h[4];
      e2m1_h2x4(j ? c.y : c.x, h);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const __half2 h2 = *reinterpret_cast<const __half2*>(&h[k]);
        w[4 * j + k] = narrow<kDType>(mul_rn(__low2float(h2), s), mul_rn(__high2float(h2), s));
      }
    }
  }
  uint16_t* dst = (is_value ? p.value : p.key) +
                  ((((int64_t)token * p.cache.kv_heads + head) << d16_shift) + block) * 16;
  reinterpret_cast<uint4*>(dst)[0] = make_uint4(w[0], w[1], w[2], w[3]);
  reinterpret_cast<uint4*>(dst)[1] = make_uint4(w[4], w[5], w[6], w[7]);
}

int log2i(int v) {
  int s = 0;
  while ((1 << s) < v) ++s;
  return s;
}

template <int kDType, bool kNeox>
cudaError_t launch_lanes(const KernelArgs& g, int lanes, cudaStream_t stream) {
  return launch_dependent(lanes == 4 ? write_kernel<kDType, kNeox, 4> : write_kernel<kDType, kNeox, 1>,
                          dim3(g.kv_ctas + g.q_ctas), kThreads, 0, stream, g);
}

}  // namespace

cudaError_t launch_write(const WriteArgs& a, int device_sms, cudaStream_t stream) {
  KernelArgs g;
  g.a = a;
  const uint32_t d16 = (uint32_t)a.cache.head_size / 16;
  g.d16_shift = log2i((int)d16);
  g.page_shift = log2i(a.cache.page_size);
  g.kv_per_token = 2u * (uint32_t)a.cache.kv_heads * d16;
  g.q_per_token = (uint32_t)((a.q_heads + kQHeads - 1) / kQHeads) * d16;
  g.kv_units = (uint32_t)(a.tokens * g.kv_per_token);
  g.q_units = (uint32_t)(a.tokens * g.q_per_token);
  make_divider(g.kv_per_token, &g.kv_magic, &g.kv_shift);
  make_divider(g.q_per_token, &g.q_magic, &g.q_shift);
  // Four lanes share a unit's candidates while that still leaves every SM at
  // most one CTA (the rule and the reason of the quantizer's).
  const int lanes = (uint64_t)g.kv_units * 4 <= (uint64_t)device_sms * kThreads ? 4 : 1;
  const uint64_t want = ((uint64_t)g.kv_units * lanes + kThreads - 1) / kThreads;
  const uint64_t cap = (uint64_t)device_sms * 16;
  g.kv_ctas = (uint32_t)(want < cap ? want : cap);
  g.q_ctas = (uint32_t)(((uint64_t)g.q_units + kThreads - 1) / kThreads);
  if (a.dtype == kDTypeBF16)
    return a.neox ? launch_lanes<kDTypeBF16, true>(g, lanes, stream)
                  : launch_lanes<kDTypeBF16, false>(g, lanes, stream);
  return a.neox ? launch_lanes<kDTypeF16, true>(g, lanes, stream)
                : launch_lanes<kDTypeF16, false>(g, lanes, stream);
}

cudaError_t launch_gather(const GatherArgs& a, int device_sms, cudaStream_t stream) {
  (void)device_sms;
  const uint32_t d16 = (uint32_t)a.cache.head_size / 16;
  const uint32_t per_token = 2u * (uint32_t)a.cache.kv_heads * d16;
  const uint32_t units = (uint32_t)(a.tokens * per_token);
  uint32_t magic, shift;
  make_divider(per_token, &magic, &shift);
  const unsigned grid = (unsigned)(((uint64_t)units + kThreads - 1) / kThreads);
  return launch_dependent(
      a.dtype == kDTypeBF16 ? gather_kernel<kDTypeBF16> : gather_kernel<kDTypeF16>, dim3(grid),
      kThreads, 0, stream, a, units, per_token, magic, shift, log2i((int)d16),
      log2i(a.cache.page_size));
}

}  // namespace kv
}  // namespace ssw
