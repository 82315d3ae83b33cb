// Attention over an NVFP4 cache for long queries (see kv_attend.cu for the
// operator): tiles of 256 (token, head) rows of one kv head, 128 keys a block,
// on the 5th-generation tensor cores.
//
//   S = Q K^T  (tcgen05.mma kind::f16, Q and K from shared memory, S in TMEM)
//   P = 2^(scale S - m + kShift)  (f16, written over S in TMEM)
//   O += P V   (P from TMEM, V from shared memory, O in TMEM)
//
// One CTA per SM.  The two 128-row halves of a tile take turns: while the
// tensor cores work on one half's P V and next Q K^T, a warpgroup forms the
// other half's softmax.  Warps:
//   0-3, 4-7  softmax of half 0 / 1, one row per thread; also Q's load and the
//             result's store
//   8-11      dequantization: thread i turns key i of a block from codes and
//             scales (prefetched one block ahead in registers) into f16 rows,
//             once for all 256 rows, in a ring of four tiles (K, V, K, V)
//   12        issues the MMAs.  It meets the others on hardware named barriers
//             only: a shared-memory access by the issuing warp would wait for
//             its queued MMAs to drain.
// A row's O is rescaled only when its maximum grows by more than 2^kSlack
// (P keeps that much room below f16's largest), so almost never after the first
// blocks, and by the softmax threads: the P V before it has completed when the
// next S has (MMAs complete in order), and the next one waits for this P.
//
// Every mbarrier wait is bounded; after one that gave up the roles keep their
// barrier protocol, so no partner is left waiting (see bar_tell), MMAs in flight
// are waited for, with a limit, the rows that may be wrong become NaN and *status
// is set.
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "attend.cuh"
#include "kv.cuh"
#include "ptx.cuh"
#include "quant.cuh"

namespace ssw {
namespace kv {
namespace {

constexpr int kPThreads = 16 * 32;
constexpr int kBlock = 128;  // keys of a block
constexpr int kWarpDequant = 8, kWarpMma = 12;
constexpr int kMaskRing = 4;
// Registers: the launch gives every thread 128.  The softmax threads hold a
// whole row of S (128) and take what the others can spare:
// 256 x 184 + 128 x 96 + 128 x 40 = 64512 of the launch's 65536.
constexpr int kRegsSoftmax = 184, kRegsDequant = 96, kRegsMma = 40;
// Heads of 256: 128 x 216 + 256 x 120 + 128 x 40 = 63488.
constexpr int kRegsWideSoftmax = 216, kRegsWideDequant = 120;
template <int kRegs>
__device__ __forceinline__ void more_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
}
template <int kRegs>
__device__ __forceinline__ void fewer_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}

// Named barriers, 16 of hardware: the tiles that K and V are dequantized into
// are full, P is there, Q is loaded.  A warp that only tells the MMA warp arrives
// and goes on, so it may be ahead of it by as many of its arrivals as its waits
// for the MMAs allow.  Each kind therefore has a barrier more for every arrival
// that may be outstanding where such a wait gives up, used in turn: from then on
// the warp waits at its barriers too (bar_tell), and so it can never arrive twice
// at one before the MMA warp has, which would end that barrier's phase without
// it and leave it waiting for good.
//   prompt_kernel: K (V) of a block waits for the MMAs that read its slot, two
//   blocks before: the last three arrivals may be outstanding, 8 barriers for 4
//   slots; P waits for scores issued behind the P before the last: 2 a half.
//   prompt_wide_kernel: K and V wait for the MMAs of the block before: 2 each; P
//   waits for scores issued behind the P before the last two: 4.
constexpr int kBarSlot = 1, kBarP = 9, kBarQ = 13;
constexpr int kBarWideK = 1, kBarWideV = 3, kBarWideP = 5;

template <int kD>
struct PromptShape {
  static constexpr int kHalf = 128 * 128;             // bytes: 128 rows x 64 f16
  static constexpr int kTile = kHalf * (kD / 64);     // 128 rows x kD f16
  static constexpr int kSmem = 2 * kTile + 4 * kTile + 256 + 1024;
  static constexpr uint32_t kS = 0, kO = 256;         // TMEM columns: S0, S1, then O0, O1
  static constexpr uint32_t kIdescQK = (1u << 4) | ((uint32_t)(kBlock >> 3) << 17) | (8u << 24);
  // B (V) is contiguous along N
  static constexpr uint32_t kIdescPV =
      (1u << 4) | (1u << 16) | ((uint32_t)(kD >> 3) << 17) | (8u << 24);
};

struct Control {
  uint64_t empty[4];
  uint64_t s_full[2];
  uint64_t mask_full[kMaskRing];
  uint32_t mask[kMaskRing][4];  // bit i: key i of the block is there
  uint64_t drained;             // after a wait that gave up: every MMA has completed
  uint32_t tmem;
  uint32_t gave_up;
};

__device__ __forceinline__ void bar_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ void bar_arrive(int id, int threads) {
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
// The same `ok` in all of the warp.
__device__ __forceinline__ void bar_tell(bool ok, int id, int threads) {
  if (ok)
    bar_arrive(id, threads);
  else
    bar_sync(id, threads);
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
      : "memory");
}
// Shared-memory matrix descriptor: 128-byte swizzle, version 1.
__device__ __forceinline__ uint64_t smem_desc(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)((lbo >> 4) & 0x3FFF) << 16) |
         ((uint64_t)((sbo >> 4) & 0x3FFF) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accum));
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                       uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accum));
}
// 32 columns of the warp's 32 lanes; the caller waits with tmem_wait_ld.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, "
      "%10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, "
      "%26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
        "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]),
        "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]),
        "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]),
        "=r"(v[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_ld() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
      "%11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
      "%11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, "
      "%28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
      "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]),
      "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]),
      "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]),
      "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void st_shared16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c,
                                            uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c),
               "r"(d)
               : "memory");
}
__device__ __forceinline__ void ld_shared16(uint32_t addr, uint32_t (&x)[4]) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
               : "r"(addr)
               : "memory");
}
// Byte offset of 16-byte chunk c of row r in a 128-row tile of 64-wide halves,
// 128-byte swizzle: K-major for Q and K, N-major for V.
__device__ __forceinline__ uint32_t tile_offset(int r, int c) {
  return (uint32_t)((c >> 3) * 16384 + (r >> 3) * 1024 + (r & 7) * 128 + (((c ^ r) & 7) << 4));
}

// Codes and scales of one key or value row.
template <int kD>
struct RowRegs {
  alignas(16) uint32_t codes[kD / 8];
  alignas(16) uint32_t scales[kD / 64];
};

template <int kD>
__device__ __forceinline__ void load_row(RowRegs<kD>& r, const uint8_t* codes,
                                         const uint8_t* scales, bool there) {
  if (there) {
#pragma unroll
    for (int j = 0; j < kD / 32; ++j)
      *reinterpret_cast<uint4*>(&r.codes[4 * j]) = reinterpret_cast<const uint4*>(codes)[j];
    if constexpr (kD == 64) {
      r.scales[0] = *reinterpret_cast<const uint32_t*>(scales);
    } else if constexpr (kD == 128) {
      *reinterpret_cast<uint2*>(r.scales) = *reinterpret_cast<const uint2*>(scales);
    } else {
      *reinterpret_cast<uint4*>(r.scales) = *reinterpret_cast<const uint4*>(scales);
    }
  } else {  // what lies behind the last key may hold anything, NaN scales too
#pragma unroll
    for (int j = 0; j < kD / 8; ++j) r.codes[j] = 0;
#pragma unroll
    for (int j = 0; j < kD / 64; ++j) r.scales[j] = 0;
  }
}

template <int kD>
__device__ __forceinline__ void store_row(const RowRegs<kD>& r, uint32_t tile, int row) {
#pragma unroll
  for (int b = 0; b < kD / 16; ++b) {
    const uint32_t two = e4m3_h2(r.scales[b / 4] >> (16 * ((b / 2) & 1)));
    const uint32_t f = __byte_perm(two, two, b & 1 ? 0x3232 : 0x1010);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t x[4];
      e2m1_h2x4(r.codes[2 * b + h], x);
      st_shared16(tile + tile_offset(row, 2 * b + h), mul_h2(x[0], f), mul_h2(x[1], f),
                  mul_h2(x[2], f), mul_h2(x[3], f));
    }
  }
}

// One softmax thread's row: its place, and the scale that turns scores into log2.
struct Row {
  bool live;
  int64_t out_row;      // of lse and of the partial results
  const uint16_t* src;  // of the query
  uint16_t* dst;
  int hi_key, lo_key;   // keys it sees
  float scale;
};

__device__ __forceinline__ Row row_of(const Params& p, const Tile& tile, int head, int row_in) {
  const AttendArgs& a = p.a;
  Row w;
  w.live = row_in < tile.rows;
  const int row = tile.row0 + row_in, token = row / p.group, qh = head * p.group + row % p.group;
  const int64_t at = tile.first_token + token;
  w.out_row = at * a.q_heads + qh;
  w.src = a.q.p + at * a.q.token_stride + (int64_t)qh * a.q.head_stride;
  w.dst = a.out.p + at * a.out.token_stride + (int64_t)qh * a.out.head_stride;
  const int pos = tile.offset + token;
  w.hi_key = !w.live ? -1 : a.causal ? pos : 0x7FFFFFFF;
  w.lo_key = a.window >= 0 ? pos - a.window : 0;
  return w;
}

// A pointer that lane `from` holds.
template <typename T>
__device__ __forceinline__ T* shfl_pointer(T* p, int from) {
  return reinterpret_cast<T*>(
      __shfl_sync(0xFFFFFFFFu, reinterpret_cast<unsigned long long>(p), from));
}

// The warp's 32 rows of Q, as they are, into rows r0 .. r0 + 31 of the swizzled
// tile: asynchronous copies, neighbouring lanes taking neighbouring parts of a
// row; zeros for a row that is not there.
template <int kD>
__device__ __forceinline__ void copy_queries(const Params& p, const Row& w, uint32_t tile, int r0) {
  constexpr int kLanes = kD / 8;     // lanes of a row
  constexpr int kPer = 32 / kLanes;  // rows of a warp's copy
  const int lane = threadIdx.x & 31, part = lane % kLanes;
  const uint16_t* const mine = w.live ? w.src : nullptr;
#pragma unroll 2
  for (int i = lane / kLanes; i < 32; i += kPer) {
    const uint16_t* src = shfl_pointer(mine, i);
    const uint32_t bytes = src ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                     tile + tile_offset(r0 + i, part)),
                 "l"((src ? src : p.a.q.p) + part * 8), "r"(bytes)
                 : "memory");
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncwarp();
}

// A row of 16-byte chunks of bf16 pairs times `down` as f16, in place; the
// largest magnitude in each half of the result, as bf16 bits.
template <int kD>
__device__ __forceinline__ uint32_t convert_row(uint32_t tile, int r, float down) {
  uint32_t big = 0;
#pragma unroll 4
  for (int j = 0; j < kD / 8; ++j) {
    uint32_t x[4];
    const uint32_t at = tile + tile_offset(r, j);
    ld_shared16(at, x);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      big = __vmaxu2(big, x[c] & 0x7FFF7FFFu);
      x[c] = pack_h2(__uint_as_float(x[c] << 16) * down,
                     __uint_as_float(x[c] & 0xFFFF0000u) * down);
    }
    st_shared16(at, x[0], x[1], x[2], x[3]);
  }
  return big;
}

// The warp's 32 rows of Q as f16 into the swizzled tile; w.scale.  Short loops:
// this code runs once per CTA, mostly from a cold instruction cache.
//
// A bf16 row whose largest magnitude lies in [2^-6, 2^15) is converted as it is:
// no overflow, and what f16 rounds off its small elements is below 2^-19 of the
// largest.  Other rows are fetched again and scaled by a power of two, as in
// decode_kernel.
template <int kD>
__device__ __forceinline__ void load_queries(const Params& p, Row& w, uint32_t tile, int r0) {
  const AttendArgs& a = p.a;
  const int r = r0 + (threadIdx.x & 31);
  copy_queries<kD>(p, w, tile, r0);
  const float signed_log2 = a.softmax_scale * kLog2e / *a.cache.multiplier;
  const float sign = signed_log2 < 0.0f ? -1.0f : 1.0f;  // the maximum is taken before scaling
  float scale = fabsf(signed_log2);
  if (a.dtype == kDTypeBF16) {
    const uint32_t big = convert_row<kD>(tile, r, sign);
    const uint32_t top = max(big & 0xFFFFu, big >> 16);
    const int e = (int)(top >> 7);  // exponent; zero, subnormal and non-finite rows stay as they are
    const bool resize = (e >= 1 && e < 121) || (e > 141 && e <= 253);
    if (__any_sync(0xFFFFFFFFu, resize)) {
      __syncwarp();
      copy_queries<kD>(p, w, tile, r0);
      float down = sign;
      if (resize) {
        down *= __uint_as_float((uint32_t)(254 - e) << 23);
        scale *= __uint_as_float((uint32_t)e << 23);
      }
      convert_row<kD>(tile, r, down);
    }
  } else if (sign < 0.0f) {
#pragma unroll 1
    for (int j = 0; j < kD / 8; ++j) {
      uint32_t x[4];
      const uint32_t at = tile + tile_offset(r, j);
      ld_shared16(at, x);
      st_shared16(at, x[0] ^ 0x80008000u, x[1] ^ 0x80008000u, x[2] ^ 0x80008000u,
                  x[3] ^ 0x80008000u);
    }
  }
  w.scale = fmaxf(scale, 1e-37f);  // never zero, or a masked score would be NaN
}

// Which keys of the block from k0 the row sees; false: all of them, for every
// row of the warp.
__device__ __forceinline__ bool block_mask(const Control* ctl, int j, int k0, const Row& w,
                                           uint32_t (&mask)[4]) {
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    mask[x] = *reinterpret_cast<const volatile uint32_t*>(&ctl->mask[j % kMaskRing][x]);
    const int first = k0 + 32 * x;
    const int lo = w.lo_key - first, hi = w.hi_key - first;
    const uint32_t above = lo <= 0 ? 0xFFFFFFFFu : lo > 31 ? 0u : 0xFFFFFFFFu << lo;
    const uint32_t below = hi >= 31 ? 0xFFFFFFFFu : hi < 0 ? 0u : 0xFFFFFFFFu >> (31 - hi);
    mask[x] &= above & below;
  }
  return __any_sync(0xFFFFFFFFu, (mask[0] & mask[1] & mask[2] & mask[3]) != 0xFFFFFFFFu);
}

// Softmax of the 128 scores at s_addr: updates the row's maximum and sum,
// rescales O (kD columns at o_addr) where the maximum has grown by more than
// the slack, and writes P over the scores.  `before_rescale` runs before O is
// touched.  `saw` becomes nonzero where the row sees a key.
template <int kD, typename F>
__device__ __forceinline__ void softmax_block(uint32_t s_addr, uint32_t o_addr, bool masked,
                                              const uint32_t (&mask)[4], float scale, bool first,
                                              float& m, float& l, uint32_t& saw,
                                              F&& before_rescale) {
  uint32_t v[128];
#pragma unroll
  for (int c = 0; c < 4; ++c)
    tmem_ld32(s_addr + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(v + 32 * c));
  tmem_wait_ld();
  if (masked) {
#pragma unroll
    for (int x = 0; x < 128; ++x)
      if (!((mask[x / 32] >> (x % 32)) & 1u)) v[x] = 0xFF800000u;
    saw |= mask[0] | mask[1] | mask[2] | mask[3];
  } else {
    saw = 1;
  }
  float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int x = 0; x < 128; x += 8)
#pragma unroll
    for (int y = 0; y < 4; ++y)
      top[y] = fmaxf(fmaxf(top[y], __uint_as_float(v[x + 2 * y])), __uint_as_float(v[x + 2 * y + 1]));
  const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * scale;
  if (__any_sync(0xFFFFFFFFu, mx > m + kSlack)) {
    const float mn = fmaxf(m, mx);
    const float f = mn == -INFINITY ? 1.0f : ex2(m - mn);
    m = mn;
    l *= f;
    if (!first) {  // nothing is in O before the first block
      before_rescale();
#pragma unroll 1
      for (int c = 0; c < kD / 32; ++c) {
        uint32_t o[32];
        tmem_ld32(o_addr + 32 * c, o);
        tmem_wait_ld();
#pragma unroll
        for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
        tmem_st32(o_addr + 32 * c, o);
      }
    }
  }
  const float ms = m == -INFINITY ? 0.0f : m - kShift;
  const uint64_t scale2 = pack2(scale, scale), ms2 = pack2(-ms, -ms);
  uint64_t sums[2] = {0, 0};
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint32_t w[16];
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      const int at = 32 * c + 2 * x;
      float e0, e1;
      unpack2(fma2(pack2(__uint_as_float(v[at]), __uint_as_float(v[at + 1])), scale2, ms2), e0, e1);
      const float p0 = ex2(e0), p1 = ex2(e1);
      sums[x & 1] = add2(sums[x & 1], pack2(p0, p1));
      w[x] = pack_h2(p0, p1);
    }
    tmem_st16(s_addr + 16 * c, w);
  }
  float sum[4];
  unpack2(sums[0], sum[0], sum[1]);
  unpack2(sums[1], sum[2], sum[3]);
  l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
  asm volatile("tcgen05.fence::before_thread_sync;");
}

// 128 bytes of each of the warp's 32 rows, held a row per thread, to `dst` (each
// thread's own row, null: none), through 4 KB of shared memory: eight lanes
// store a row's 128 bytes (16 bytes per row and instruction took 7000 cycles
// for a tile of heads of 128).
__device__ __forceinline__ void store_rows(uint32_t stage, const uint32_t (&v)[32], uint8_t* dst) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int c = 0; c < 8; ++c)
    st_shared16(stage + lane * 128 + (((c ^ lane) & 7) << 4), v[4 * c], v[4 * c + 1], v[4 * c + 2],
                v[4 * c + 3]);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = 4 * i + (lane >> 3), c = lane & 7;
    uint32_t x[4];
    ld_shared16(stage + row * 128 + (((c ^ row) & 7) << 4), x);
    uint8_t* to = shfl_pointer(dst, row);
    if (to) *reinterpret_cast<uint4*>(to + 16 * c) = make_uint4(x[0], x[1], x[2], x[3]);
  }
  __syncwarp();
}

// A wait has given up.  Said before the warp touches a tile that an MMA may still
// read: who sees that MMA's result sees this as well, and makes its rows NaN.
__device__ __forceinline__ void give_up(Control* ctl) {
  *reinterpret_cast<volatile uint32_t*>(&ctl->gave_up) = 1;
}
__device__ __forceinline__ bool gave_up(const Control* ctl) {
  return *reinterpret_cast<const volatile uint32_t*>(&ctl->gave_up) != 0;
}

// The MMA warp, behind the last barrier: where a wait gave up, MMAs may still be
// in flight, which read shared memory, write TMEM and arrive on barriers.  Waits
// for them, with a limit as well, before TMEM is freed and the CTA ends.
__device__ __forceinline__ void drain_after_giving_up(Control* ctl) {
  if (!gave_up(ctl)) return;
  if ((threadIdx.x & 31) == 0) mma_commit(smem_u32(&ctl->drained));
  mbar_wait(smem_u32(&ctl->drained), 0);
  __syncwarp();
}

// The rows' results from O (kD columns at o_addr): out, or a split's partial;
// this thread's is row `row_in` of the tile.
// `stage`: 4 KB of shared memory of the warp's own.
template <int kD>
__device__ __forceinline__ void store_result(const Params& p, const Row& w, int row_in,
                                             uint32_t o_addr, uint32_t stage, bool any, float m,
                                             float l) {
  const AttendArgs& a = p.a;
  const bool seen = any && !(m == -INFINITY && l == 0.0f);  // a row that saw no key is zero
  if (p.splits == 1) {
    const float inv = row_inverse(m, l, 1.0f / a.cache.multiplier[1]);
#pragma unroll 1
    for (int c = 0; c < kD / 64; ++c) {
      uint32_t h[32];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint32_t v[32];
        if (any) {
          tmem_ld32(o_addr + 64 * c + 32 * k, v);
          tmem_wait_ld();
        }
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          const float lo = seen ? __uint_as_float(v[2 * x]) * inv : 0.0f;
          const float hi = seen ? __uint_as_float(v[2 * x + 1]) * inv : 0.0f;
          if (a.dtype == kDTypeBF16) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
            h[16 * k + x] = *reinterpret_cast<const uint32_t*>(&b);
          } else {
            h[16 * k + x] = pack_h2(lo, hi);
          }
        }
      }
      store_rows(stage, h, w.live ? reinterpret_cast<uint8_t*>(w.dst + 64 * c) : nullptr);
    }
    if (w.live && a.lse) a.lse[w.out_row] = row_lse(m, l);
  } else {
    // from the launch's coordinates, which are at hand here: carried through the
    // blocks, the place costs the softmax threads registers
    const int tile = p.tiles - 1 - blockIdx.x % p.tiles;
    const int64_t part = part_row(p, blockIdx.y, blockIdx.x / p.tiles, blockIdx.z,
                                  tile * prompt_rows(kD) + row_in, w.out_row);
#pragma unroll 1
    for (int c = 0; c < kD / 32; ++c) {
      uint32_t v[32];
      if (any) {
        tmem_ld32(o_addr + 32 * c, v);
        tmem_wait_ld();
      }
#pragma unroll
      for (int x = 0; x < 32; ++x) v[x] = seen ? v[x] : 0;
      store_rows(stage, v,
                 w.live ? reinterpret_cast<uint8_t*>(p.part_o + part * kD + 32 * c) : nullptr);
    }
    if (w.live) *reinterpret_cast<float2*>(p.part_ml + part * 2) = make_float2(m, l);
  }
}

template <int kD>
__global__ void __launch_bounds__(kPThreads, 1) prompt_kernel(const Params p) {
  using S = PromptShape<kD>;
  extern __shared__ uint8_t smem_raw[];
  wait_for_predecessor();
  let_successor_start();
  const AttendArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int seq = blockIdx.x / p.tiles, head = blockIdx.z, split = blockIdx.y;
  // the last tiles see the most keys: they start first
  Tile tile;
  if (!tile_of(p, seq, p.tiles - 1 - blockIdx.x % p.tiles, prompt_rows(kD), tile)) return;
  const int base = tile.beg & ~(kKeys - 1);
  if (split > 0 && base + (int64_t)split * p.chunk >= tile.end) return;
  const int c0 = base + split * p.chunk;
  const int c1 = (int)min((int64_t)tile.end, (int64_t)c0 + p.chunk);
  const int blocks = c1 > c0 ? (c1 - c0 + kBlock - 1) / kBlock : 0;
  const bool two = tile.rows > 128;

  const uint32_t smem = (smem_u32(smem_raw) + 1023) & ~1023u;
  const uint32_t q_tile = smem, ring = smem + 2 * S::kTile;
  Control* ctl =
      reinterpret_cast<Control*>(smem_raw + (ring + 4 * S::kTile - smem_u32(smem_raw)));
  static_assert(sizeof(Control) <= 256, "control block");
  if (threadIdx.x == 0) {
    for (int i = 0; i < 4; ++i) mbar_init(smem_u32(&ctl->empty[i]), 1);
    for (int i = 0; i < 2; ++i) mbar_init(smem_u32(&ctl->s_full[i]), 1);
    for (int i = 0; i < kMaskRing; ++i) mbar_init(smem_u32(&ctl->mask_full[i]), 4);
    mbar_init(smem_u32(&ctl->drained), 1);
    ctl->gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kWarpMma) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&ctl->tmem)),
                 "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  asm volatile("tcgen05.fence::before_thread_sync;");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;");
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&ctl->tmem);
  bool ok = true;
  auto wait = [&](uint32_t bar, uint32_t parity) {
    if (ok && !warp_wait(bar, parity)) {
      ok = false;
      give_up(ctl);
      __syncwarp();
    }
  };

  if (warp >= kWarpMma) {
    fewer_registers<kRegsMma>();
    if (warp == kWarpMma) {
    bar_sync(kBarQ, 256 + 32);
    auto qk = [&](int half, int slot) {
      if (lane == 0) {
#pragma unroll
        for (int j = 0; j < kD / 16; ++j) {
          const uint32_t off = (j / 4) * S::kHalf + 32 * (j % 4);
          mma_ss(tmem + S::kS + 128 * half, smem_desc(q_tile + half * S::kTile + off, 16, 1024),
                 smem_desc(ring + slot * S::kTile + off, 16, 1024), S::kIdescQK, j != 0);
        }
        mma_commit(smem_u32(&ctl->s_full[half]));
      }
    };
    auto pv = [&](int half, int slot, bool first) {
      if (lane == 0) {
#pragma unroll
        for (int j = 0; j < kBlock / 16; ++j)
          mma_ts(tmem + S::kO + kD * half, tmem + S::kS + 128 * half + 8 * j,
                 smem_desc(ring + slot * S::kTile + 2048 * j, S::kHalf, 1024), S::kIdescPV,
                 !(first && j == 0));
      }
    };
    if (blocks > 0) {
      bar_sync(kBarSlot, 128 + 32);  // K of block j: kBarSlot + 2j mod 8, V: the next
      asm volatile("tcgen05.fence::after_thread_sync;");
      qk(0, 0);
      if (two) qk(1, 0);
      // a slot's release is committed only where it is waited for: no arrival
      // may be in flight when the CTA ends
      if (lane == 0 && blocks > 2) mma_commit(smem_u32(&ctl->empty[0]));
      for (int j = 0; j < blocks; ++j) {
        const int v_slot = (2 * j + 1) & 3, k_slot = (2 * j + 2) & 3;
        const bool more = j + 1 < blocks;
        bar_sync(kBarSlot + ((2 * j + 1) & 7), 128 + 32);
        if (more) bar_sync(kBarSlot + ((2 * j + 2) & 7), 128 + 32);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (half == 1 && !two) break;
          bar_sync(kBarP + 2 * half + (j & 1), 128 + 32);
          asm volatile("tcgen05.fence::after_thread_sync;");
          pv(half, v_slot, j == 0);
          if (more)
            qk(half, k_slot);
          else if (lane == 0)
            mma_commit(smem_u32(&ctl->s_full[half]));  // the last P V
        }
        if (lane == 0 && j + 2 < blocks) mma_commit(smem_u32(&ctl->empty[v_slot]));
        if (lane == 0 && j + 3 < blocks) mma_commit(smem_u32(&ctl->empty[k_slot]));
      }
    }
    __syncwarp();
    }
  } else if (warp >= kWarpDequant) {
    fewer_registers<kRegsDequant>();
    const int i = threadIdx.x - kWarpDequant * 32;  // this thread's key of a block
    const int page_mask = (1 << p.page_shift) - 1;
    const int32_t* table = a.block_table + (int64_t)seq * a.table_stride;
    const int64_t side = (int64_t)a.cache.kv_heads << p.page_shift;
    auto page_of = [&](int j) -> int {
      const int key = c0 + j * kBlock + i;
      if (key >= c1 || key < tile.beg) return -1;
      const int pg = table[key >> p.page_shift];
      return (uint32_t)pg < (uint32_t)a.cache.num_pages ? pg : -1;
    };
    auto fetch = [&](RowRegs<kD>& r, int j, int pg, int value) {
      const int key = c0 + j * kBlock + i;
      const int64_t row = value * side + ((int64_t)head << p.page_shift) + (key & page_mask);
      load_row<kD>(r, a.cache.codes + pg * a.cache.codes_page_stride + row * (kD / 2),
                   a.cache.scales + pg * a.cache.scales_page_stride + row * (kD / 16), pg >= 0);
    };
    RowRegs<kD> k, v;
    int pg = page_of(0), pg_next = page_of(1);
    fetch(k, 0, pg, 0);
    fetch(v, 0, pg, 1);
    for (int j = 0; j < blocks; ++j) {
      const int k_slot = (2 * j) & 3, v_slot = k_slot + 1;
      const uint32_t there = __ballot_sync(0xFFFFFFFFu, pg >= 0);
      // slots are used every second block
      if (j >= 2) wait(smem_u32(&ctl->empty[k_slot]), ((j >> 1) - 1) & 1);
      if (lane == 0) {
        ctl->mask[j % kMaskRing][warp - kWarpDequant] = there;
        mbar_arrive(smem_u32(&ctl->mask_full[j % kMaskRing]));
      }
      store_row<kD>(k, ring + k_slot * S::kTile, i);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      bar_tell(ok, kBarSlot + ((2 * j) & 7), 128 + 32);
      pg = pg_next;
      pg_next = page_of(j + 2);
      fetch(k, j + 1, pg, 0);
      if (j >= 2) wait(smem_u32(&ctl->empty[v_slot]), ((j >> 1) - 1) & 1);
      store_row<kD>(v, ring + v_slot * S::kTile, i);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      bar_tell(ok, kBarSlot + ((2 * j + 1) & 7), 128 + 32);
      fetch(v, j + 1, pg, 1);
    }
  } else {
    more_registers<kRegsSoftmax>();
    const int half = warp >> 2, r = (warp & 3) * 32 + lane;
    Row w = row_of(p, tile, head, half * 128 + r);
    load_queries<kD>(p, w, q_tile + half * S::kTile, (warp & 3) * 32);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    bar_arrive(kBarQ, 256 + 32);

    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lanes + S::kS + 128 * half;
    const uint32_t o_addr = tmem + lanes + S::kO + kD * half;
    float m = -INFINITY, l = 0.0f;
    uint32_t saw = 0;
    const bool work = half == 0 || two;
    for (int j = 0; work && j < blocks; ++j) {
      wait(smem_u32(&ctl->mask_full[j % kMaskRing]), (j / kMaskRing) & 1);
      uint32_t mask[4];
      const bool masked = block_mask(ctl, j, c0 + j * kBlock, w, mask);
      wait(smem_u32(&ctl->s_full[half]), j & 1);
      asm volatile("tcgen05.fence::after_thread_sync;");
      // the P V before this S was issued before it, and has completed with it
      softmax_block<kD>(s_addr, o_addr, masked, mask, w.scale, j == 0, m, l, saw, [] {});
      bar_tell(ok, kBarP + 2 * half + (j & 1), 128 + 32);
    }
    if (work && blocks > 0) wait(smem_u32(&ctl->s_full[half]), blocks & 1);
    asm volatile("tcgen05.fence::after_thread_sync;");
    if (saw && m == -INFINITY && l == 0.0f) l = 1.0f;  // all its scores are -inf: see row_inverse
    if (!ok || gave_up(ctl)) l = NAN;
    // this half's MMAs are done with its Q, which becomes the staging area
    store_result<kD>(p, w, half * 128 + r, o_addr, q_tile + half * S::kTile + (warp & 3) * 4096,
                     work && blocks > 0, m, l);
  }
  if (!ok && a.status && lane == 0) atomicCAS(a.status, 0, 1);
  asm volatile("tcgen05.fence::before_thread_sync;");
  __syncthreads();
  if (warp == kWarpMma) {
    asm volatile("tcgen05.fence::after_thread_sync;");
    drain_after_giving_up(ctl);
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
  }
}

// Heads of 256: a tile of 128 rows, one K tile and one V tile of 64 KB beside
// Q's, and two score buffers in TMEM beside O's 256 columns.  The next block's
// Q K^T is issued before this block's P V, so that the softmax has both to hide
// behind; K and V are dequantized by a warpgroup each, into the tile that the
// tensor cores have just finished with.  Warps 0-3: softmax; 4-7: V; 8-11: K;
// 12: MMAs.
struct WideControl {
  uint64_t s_full[2];  // scores are in buffer 0 / 1 (and K's tile is free)
  uint64_t o_done;     // a P V before the last has completed (and V's tile is free)
  uint64_t o_last;     // the last one has
};
static_assert(sizeof(WideControl) <= sizeof(uint64_t) * 6, "fits in front of Control's masks");

__global__ void __launch_bounds__(kPThreads, 1) prompt_wide_kernel(const Params p) {
  constexpr int kD = 256, kTile = 16384 * (kD / 64);
  constexpr uint32_t kO = 256;  // TMEM: score buffers at 0 and 128, O from 256
  constexpr uint32_t kIdescQK = (1u << 4) | ((uint32_t)(kBlock >> 3) << 17) | (8u << 24);
  constexpr uint32_t kIdescPV = (1u << 4) | (1u << 16) | ((uint32_t)(kD >> 3) << 17) | (8u << 24);
  extern __shared__ uint8_t smem_raw[];
  wait_for_predecessor();
  let_successor_start();
  const AttendArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int seq = blockIdx.x / p.tiles, head = blockIdx.z, split = blockIdx.y;
  Tile tile;
  if (!tile_of(p, seq, p.tiles - 1 - blockIdx.x % p.tiles, prompt_rows(kD), tile)) return;
  const int base = tile.beg & ~(kKeys - 1);
  if (split > 0 && base + (int64_t)split * p.chunk >= tile.end) return;
  const int c0 = base + split * p.chunk;
  const int c1 = (int)min((int64_t)tile.end, (int64_t)c0 + p.chunk);
  const int blocks = c1 > c0 ? (c1 - c0 + kBlock - 1) / kBlock : 0;

  const uint32_t smem = (smem_u32(smem_raw) + 1023) & ~1023u;
  const uint32_t q_tile = smem, k_tile = smem + kTile, v_tile = smem + 2 * kTile;
  Control* ctl = reinterpret_cast<Control*>(smem_raw + (smem + 3 * kTile - smem_u32(smem_raw)));
  WideControl* wide = reinterpret_cast<WideControl*>(ctl);  // over empty[] and s_full[]
  const uint32_t s_full[2] = {smem_u32(&wide->s_full[0]), smem_u32(&wide->s_full[1])};
  const uint32_t o_done = smem_u32(&wide->o_done), o_last = smem_u32(&wide->o_last);
  if (threadIdx.x == 0) {
    mbar_init(s_full[0], 1);
    mbar_init(s_full[1], 1);
    mbar_init(o_done, 1);
    mbar_init(o_last, 1);
    for (int i = 0; i < kMaskRing; ++i) mbar_init(smem_u32(&ctl->mask_full[i]), 4);
    mbar_init(smem_u32(&ctl->drained), 1);
    ctl->gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kWarpMma) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&ctl->tmem)),
                 "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  asm volatile("tcgen05.fence::before_thread_sync;");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;");
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&ctl->tmem);
  bool ok = true;
  auto wait = [&](uint32_t bar, uint32_t parity) {
    if (ok && !warp_wait(bar, parity)) {
      ok = false;
      give_up(ctl);
      __syncwarp();
    }
  };

  if (warp >= kWarpMma) {
    fewer_registers<kRegsMma>();
    if (warp == kWarpMma) {
      bar_sync(kBarQ, 128 + 32);
      auto qk = [&](int j) {
        bar_sync(kBarWideK + (j & 1), 128 + 32);
        asm volatile("tcgen05.fence::after_thread_sync;");
        if (lane == 0) {
#pragma unroll
          for (int i = 0; i < kD / 16; ++i) {
            const uint32_t off = (i / 4) * 16384 + 32 * (i % 4);
            mma_ss(tmem + 128 * (j & 1), smem_desc(q_tile + off, 16, 1024),
                   smem_desc(k_tile + off, 16, 1024), kIdescQK, i != 0);
          }
          mma_commit(s_full[j & 1]);
        }
      };
      if (blocks > 0) qk(0);
      for (int j = 0; j < blocks; ++j) {
        if (j + 1 < blocks) qk(j + 1);
        bar_sync(kBarWideV + (j & 1), 128 + 32);
        bar_sync(kBarWideP + (j & 3), 128 + 32);
        asm volatile("tcgen05.fence::after_thread_sync;");
        if (lane == 0) {
#pragma unroll
          for (int i = 0; i < kBlock / 16; ++i)
            mma_ts(tmem + kO, tmem + 128 * (j & 1) + 8 * i, smem_desc(v_tile + 2048 * i, 16384, 1024),
                   kIdescPV, (j | i) != 0);
          mma_commit(j + 1 < blocks ? o_done : o_last);
        }
      }
      __syncwarp();
    }
  } else if (warp >= 4) {
    fewer_registers<kRegsWideDequant>();
    const bool value = warp < kWarpDequant;
    const int i = threadIdx.x & 127;  // this thread's key of a block
    const int page_mask = (1 << p.page_shift) - 1;
    const int32_t* table = a.block_table + (int64_t)seq * a.table_stride;
    const int64_t side = value ? (int64_t)a.cache.kv_heads << p.page_shift : 0;
    auto page_of = [&](int j) -> int {
      const int key = c0 + j * kBlock + i;
      if (key >= c1 || key < tile.beg) return -1;
      const int pg = table[key >> p.page_shift];
      return (uint32_t)pg < (uint32_t)a.cache.num_pages ? pg : -1;
    };
    auto fetch = [&](RowRegs<kD>& r, int j, int pg) {
      const int key = c0 + j * kBlock + i;
      const int64_t row = side + ((int64_t)head << p.page_shift) + (key & page_mask);
      load_row<kD>(r, a.cache.codes + pg * a.cache.codes_page_stride + row * (kD / 2),
                   a.cache.scales + pg * a.cache.scales_page_stride + row * (kD / 16), pg >= 0);
    };
    RowRegs<kD> r;
    int pg = page_of(0), pg_next = page_of(1);
    fetch(r, 0, pg);
    for (int j = 0; j < blocks; ++j) {
      const uint32_t there = __ballot_sync(0xFFFFFFFFu, pg >= 0);
      if (j > 0) {
        if (value)
          wait(o_done, (j - 1) & 1);
        else
          wait(s_full[(j - 1) & 1], ((j - 1) >> 1) & 1);
      }
      if (!value && lane == 0) {
        ctl->mask[j % kMaskRing][warp - kWarpDequant] = there;
        mbar_arrive(smem_u32(&ctl->mask_full[j % kMaskRing]));
      }
      store_row<kD>(r, value ? v_tile : k_tile, i);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      bar_tell(ok, (value ? kBarWideV : kBarWideK) + (j & 1), 128 + 32);
      pg = pg_next;
      pg_next = page_of(j + 2);
      fetch(r, j + 1, pg);
    }
  } else {
    more_registers<kRegsWideSoftmax>();
    const int r = threadIdx.x;
    Row w = row_of(p, tile, head, r);
    load_queries<kD>(p, w, q_tile, warp * 32);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    bar_arrive(kBarQ, 128 + 32);
    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    float m = -INFINITY, l = 0.0f;
    uint32_t saw = 0;
    for (int j = 0; j < blocks; ++j) {
      wait(smem_u32(&ctl->mask_full[j % kMaskRing]), (j / kMaskRing) & 1);
      uint32_t mask[4];
      const bool masked = block_mask(ctl, j, c0 + j * kBlock, w, mask);
      wait(s_full[j & 1], (j >> 1) & 1);
      asm volatile("tcgen05.fence::after_thread_sync;");
      // these scores were issued before the last P V, which O's rescaling must
      // wait for
      softmax_block<kD>(tmem + lanes + 128 * (j & 1), tmem + lanes + kO, masked, mask, w.scale,
                        j == 0, m, l, saw, [&] {
                          wait(o_done, (j - 1) & 1);
                          asm volatile("tcgen05.fence::after_thread_sync;");
                        });
      // The next scores may be there before this P V is issued, so the softmax
      // can be one block ahead of the MMA warp.  It cannot be two ahead, the
      // scores after the next being issued behind this P V.
      bar_tell(ok, kBarWideP + (j & 3), 128 + 32);
    }
    // The last P V has a barrier of its own.  On o_done a warp would have to wait
    // for the one before it first, since a parity wait may not skip a phase, and
    // the last could complete before that wait looks: the phase that it waits for
    // would be gone, and the wait run out.
    if (blocks > 0) wait(o_last, 0);
    asm volatile("tcgen05.fence::after_thread_sync;");
    if (saw && m == -INFINITY && l == 0.0f) l = 1.0f;
    if (!ok || gave_up(ctl)) l = NAN;
    store_result<kD>(p, w, r, tmem + lanes + kO, q_tile + warp * 4096, blocks > 0, m, l);
  }
  if (!ok && a.status && lane == 0) atomicCAS(a.status, 0, 1);
  asm volatile("tcgen05.fence::before_thread_sync;");
  __syncthreads();
  if (warp == kWarpMma) {
    asm volatile("tcgen05.fence::after_thread_sync;");
    drain_after_giving_up(ctl);
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
  }
}

cudaError_t launch_wide(const Params& p, cudaStream_t stream) {
  constexpr int kSmem = 3 * 65536 + 256 + 1024;
  const cudaError_t e = cudaFuncSetAttribute(prompt_wide_kernel,
                                             cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (e != cudaSuccess) return e;
  const dim3 grid((unsigned)(p.a.seqs * p.tiles), p.splits, p.a.cache.kv_heads);
  return launch_dependent(prompt_wide_kernel, grid, kPThreads, kSmem, stream, p);
}

template <int kD>
cudaError_t launch_d(const Params& p, cudaStream_t stream) {
  constexpr int kSmem = PromptShape<kD>::kSmem;
  static_assert(kSmem <= 227 * 1024, "shared memory");
  cudaError_t e = cudaFuncSetAttribute(prompt_kernel<kD>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (e != cudaSuccess) return e;
  const dim3 grid((unsigned)(p.a.seqs * p.tiles), p.splits, p.a.cache.kv_heads);
  return launch_dependent(prompt_kernel<kD>, grid, kPThreads, kSmem, stream, p);
}

}  // namespace

cudaError_t launch_prompt(const Params& p, cudaStream_t stream) {
  if (p.a.cache.head_size == 64) return launch_d<64>(p, stream);
  if (p.a.cache.head_size == 128) return launch_d<128>(p, stream);
  return launch_wide(p, stream);
}

}  // namespace kv
}  // namespace ssw
