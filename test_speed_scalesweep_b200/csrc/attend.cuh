// What the attention kernels share: launch parameters, the rows and keys of a
// tile, waits, copies and the exact conversions of codes and scales to f16.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "kv.cuh"
#include "ptx.cuh"
#include "quant.cuh"

namespace ssw {
namespace kv {

constexpr int kKeys = 32;        // keys of a decode stage; splits begin at multiples of it
constexpr float kShift = 10.f;  // log2 of the scale of P
constexpr float kSlack = 5.f;   // the maximum may grow by 2^kSlack before O is rescaled
constexpr uint32_t kWaitLimit = 1u << 22;  // bounded spin
constexpr float kLn2 = 0.6931471805599453f, kLog2e = 1.4426950408889634f;

struct Params {
  AttendArgs a;
  int group;       // query heads of a kv head
  int tiles;       // row tiles of the longest query
  int min_rows, max_rows;  // sequences with other numbers of rows are another kernel's
  int splits;      // CTAs that share a tile's keys
  int beside;      // 1: decode_kernel launched while a prompt kernel may still run
  int chunk;       // keys of a split, a multiple of 128
  int page_shift;
  // Partial results: [split][part_rows][head_size], and [..][2] of maximum and sum
  float* part_o;
  float* part_ml;
  int64_t part_rows;
  int part_seq_rows;  // rows kept per sequence and kv head; 0: a row per token and query head
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
               : "memory");
}
// Bounded wait for the phase with the given parity; false = gave up.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity) {
  for (uint32_t i = 0; i < kWaitLimit; ++i) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    if (done) return true;
  }
  return false;
}
// Of a whole warp, whose lanes stay together: false if any of them gave up.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity) {
  return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity));
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes,
                                          uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::
          "r"(dst),
      "l"(src), "r"(bytes), "r"(bar)
      : "memory");
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t mul_h2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t e4m3_h2(uint32_t two) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)two));
  return r;
}
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The rows and keys of one tile.
struct Tile {
  int row0, rows;        // first of the sequence's rows, rows here
  int first_token;       // global token of the sequence's token 0
  int offset;            // position of the sequence's token 0
  int beg, end;          // keys that any of its rows sees
  int all_beg, all_end;  // keys that all of its rows see
};

__device__ __forceinline__ bool tile_of(const Params& p, int seq, int tile, int tile_rows,
                                        Tile& t) {
  const AttendArgs& a = p.a;
  const int q0 = a.query_start[seq];
  int len = a.query_start[seq + 1] - q0;
  if (q0 < 0 || len <= 0 || q0 >= a.tokens) return false;
  if (len > a.tokens - q0) len = (int)(a.tokens - q0);
  // (the bound that max_seq_len has: key numbers and their sums stay in 32 bits)
  const int kv = min(max(0, a.seq_lens[seq]), 1 << 30);
  t.offset = kv - len;
  const int64_t rows64 = (int64_t)len * p.group;
  if (rows64 < p.min_rows || rows64 > p.max_rows) return false;
  const int rows = (int)rows64;
  t.row0 = tile * tile_rows;
  if (t.row0 >= rows) return false;
  t.rows = min(tile_rows, rows - t.row0);
  t.first_token = q0;
  const int lo = t.offset + t.row0 / p.group;
  const int hi = t.offset + (t.row0 + t.rows - 1) / p.group;
  const int room = (int)min((int64_t)a.table_columns << p.page_shift, (int64_t)kv);
  t.end = a.causal ? min(room, hi + 1) : room;
  t.all_end = a.causal ? min(room, lo + 1) : room;
  t.beg = a.window >= 0 ? max(0, lo - a.window) : 0;
  t.all_beg = a.window >= 0 ? max(0, hi - a.window) : 0;
  t.end = max(t.end, 0);
  return true;
}

// Where split `split` of row `row` of a sequence (row `out_row` of the batch) keeps its partial result.
__device__ __forceinline__ int64_t part_row(const Params& p, int split, int seq, int head, int row,
                                            int64_t out_row) {
  return split * p.part_rows +
         (p.part_seq_rows
              ? ((int64_t)seq * p.a.cache.kv_heads + head) * p.part_seq_rows + row
              : out_row);
}

// Splits of a tile that hold keys (at least one, which then writes zeros).  A
// sequence longer than the caller's max_seq_len has no more than were launched.
__device__ __forceinline__ int used_splits(const Params& p, const Tile& t) {
  const int n = t.end - (t.beg & ~(kKeys - 1));
  return min(max(1, (n + p.chunk - 1) / p.chunk), p.splits);
}

// How a row is finished.  It saw no key where its maximum m is -inf and its sum l
// of weights 0, a masked key's weight.  A NaN score makes l NaN and leaves m alone.
// A row whose scores so far are all -inf has m = -inf and a positive l (in
// decode_kernel the keys that it saw), which is dropped (times 2^-inf) when a
// larger score comes.

// 1 / (l * multiplier); 0 for a row that saw no key, whose result is zero; NaN
// where every score is -inf, the weights being 0 / 0.  NaN, too, from |m| = 2^28
// on: m and m - kShift are each off by up to half a step of m, so the largest
// weight is 2^kShift times 2^-32 to 2^32 there, and below 2^-24 times that it
// would be lost to f16, silently.  (From 2^23 on it may pass f16's largest, and the
// result is infinite.)
__device__ __forceinline__ float row_inverse(float m, float l, float inv_mult) {
  return fabsf(m) < 0x1p28f            ? inv_mult / l
         : m == -INFINITY && l == 0.0f ? 0.0f
                                       : NAN;
}
// Natural log-sum-exp: -inf for a row that saw no key (-inf + log2 0).
__device__ __forceinline__ float row_lse(float m, float l) { return (m - kShift + log2f(l)) * kLn2; }
// The weight of a partial result with the maximum x where the joint one is m.
__device__ __forceinline__ float part_weight(float x, float m) { return x == m ? 1.0f : ex2(x - m); }

__device__ __forceinline__ void store16(uint16_t* dst, const float* v, int dtype) {  // 2 values
  if (dtype == kDTypeBF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v[0], v[1]);
    *reinterpret_cast<__nv_bfloat162*>(dst) = h;
  } else {
    *reinterpret_cast<__half2*>(dst) = __floats2half2_rn(v[0], v[1]);
  }
}

// Long queries, on the tensor cores' own memory (kv_prompt.cu): rows of a tile.
constexpr int prompt_rows(int head_size) { return head_size == 256 ? 128 : 256; }
cudaError_t launch_prompt(const Params& p, cudaStream_t stream);

}  // namespace kv
}  // namespace ssw
