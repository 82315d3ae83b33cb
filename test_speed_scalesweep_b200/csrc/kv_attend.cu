// Attention over an NVFP4 cache (layout in kv.cuh), one pass over its bytes:
//
//   O[r] = sum_j softmax_j(scale / mult_k * q[r] . K[j]) V[j] / mult_v
//
// for the query rows r of a sequence and the keys j that the causal order and
// the window let r see; K and V are code * scale, which 16-bit floats (f16)
// hold exactly (6 significant bits, 2^-10 .. 2688).
//
// All of a kv head's query heads share the dequantized keys, so the rows of a
// tile are (token, head of the group) pairs, r = token * group + head.
//
// decode_kernel: tiles of 8, 16 or 32 rows, for single tokens and short
// queries.  It is bound by the cache's bytes, so the products are laid out for
// the cheapest dequantization, not for the tensor cores' rate: mma.sync with
// the *cache* as its 16-row operand (S^T = K Q^T, O^T = V^T P^T) spends one
// instruction per 256 cache elements however few rows the query has.
//   - A contraction may visit its index in any order, so a thread's share of a
//     key row is the contiguous quarter that one vector load gives, and Q is
//     permuted to match; a thread needs the scales of its own quarter only.
//   - For V the keys are contracted: two keys' codes are paired nibble by
//     nibble (4 logic operations per 16 codes) and converted together.
//   - Each warp takes every kWarps-th group of 32 keys of its CTA's share of
//     the sequence with its own running maximum and sum, fetched by bulk copies
//     into a ring of its own: no barrier between warps until the end.
// Softmax statistics and both accumulators are binary32.  P is rounded to f16
// (relative 2^-11, finer than a bf16 result) scaled by 2^kShift, so that
// weights down to 2^-(14 + kShift) of the largest keep full precision.
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "attend.cuh"
#include "kv.cuh"
#include "quant.cuh"

namespace ssw {
namespace kv {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;

template <int kD>
struct Shape {
  static constexpr int kCodeRow = kD / 2, kScaleRow = kD / 16;
  static constexpr int kKCodes = kKeys * kCodeRow, kKScales = kKeys * kScaleRow;
  static constexpr int kStage = 2 * (kKCodes + kKScales);
  static constexpr int kStages = kD == 256 ? 2 : 3;
  static constexpr int kRing = kStages * kStage;           // of a warp
  static constexpr int kKSteps = kD / 16;
};

// Shared memory: the warps' rings, then their barriers.  The rings are reused
// for the warps' partial results, kNT * 8 rows of kD + 2 floats each.
template <int kD, int kNT>
constexpr int smem_bytes() {
  constexpr int ring = kWarps * Shape<kD>::kRing;
  constexpr int merge = kWarps * kNT * 8 * (kD + 2) * 4;
  return (ring > merge ? ring : merge) + kWarps * Shape<kD>::kStages * 8;
}

template <bool kOn>
struct Flag {
  static constexpr bool value = kOn;
};

template <int kD, int kNT>
__device__ __forceinline__ void decode_tile(const Params& p) {
  using S = Shape<kD>;
  constexpr int kRows = kNT * 8;
  constexpr int kQuarter = kD / 4;             // elements of a key row per thread
  constexpr int kKWords = kD / 32;             // 32-bit words of codes per thread and key row
  constexpr int kVWords = kD / 64 < 1 ? 1 : kD / 64;  // words of codes per thread and value row
  extern __shared__ __align__(128) uint8_t smem[];
  const AttendArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int split = blockIdx.y, head = blockIdx.z;
  const int seq = blockIdx.x / p.tiles;
  Tile tile;
  if (!tile_of(p, seq, blockIdx.x % p.tiles, kRows, tile)) return;
  const int base = tile.beg & ~(kKeys - 1);
  if (split > 0 && base + (int64_t)split * p.chunk >= tile.end) return;
  const int c0 = base + split * p.chunk;
  const int c1 = min((int64_t)tile.end, (int64_t)c0 + p.chunk);

  constexpr int kBarOff = smem_bytes<kD, kNT>() - kWarps * S::kStages * 8;
  const uint32_t ring = smem_u32(smem) + warp * S::kRing;
  const uint32_t bars = smem_u32(smem) + kBarOff + warp * S::kStages * 8;
  if (lane == 0) {
    for (int s = 0; s < S::kStages; ++s) mbar_init(bars + 8 * s, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncwarp();

  // ---- this warp's stages: keys c0 + 32 (warp + 4 i)
  const int n_stages = c1 > c0 + warp * kKeys ? (c1 - c0 - warp * kKeys + kKeys * kWarps - 1) /
                                                    (kKeys * kWarps)
                                              : 0;
  const int32_t* table = a.block_table + (int64_t)seq * a.table_stride;
  const int page_rows = 1 << p.page_shift;
  const int piece = min(page_rows, kKeys);   // keys of one copy
  const int pieces = kKeys / piece;          // 1 or 2
  const int64_t side_code = (int64_t)a.cache.kv_heads * page_rows * S::kCodeRow;
  const int64_t side_scale = (int64_t)a.cache.kv_heads * page_rows * S::kScaleRow;
  // lane l < 4 * pieces copies part l & 3 (K codes, K scales, V codes, V scales) of piece l >> 2
  const int part = lane & 3, my_piece = lane >> 2;
  const bool copies = my_piece < pieces;
  const bool scales_part = part & 1, value_part = part & 2;
  const int row_bytes = scales_part ? S::kScaleRow : S::kCodeRow;
  const uint32_t copy_bytes = piece * row_bytes;
  const int64_t page_stride = scales_part ? a.cache.scales_page_stride : a.cache.codes_page_stride;
  const uint8_t* copy_src =
      (scales_part ? a.cache.scales + (value_part ? side_scale : 0)
                   : a.cache.codes + (value_part ? side_code : 0)) +
      (int64_t)head * page_rows * row_bytes;
  const uint32_t copy_dst = ring + (value_part ? S::kKCodes + S::kKScales : 0) +
                            (scales_part ? S::kKCodes : 0) + my_piece * copy_bytes;
  const int copy_key = c0 + warp * kKeys + my_piece * piece;  // of stage 0
  const int copy_end = copies ? min((int64_t)tile.end, (int64_t)c0 + p.chunk) : 0;
  // The table's entry for this lane's piece of stage i, or -1; looked at only
  // where it is used, a stage later.
  auto page_of = [&](int i) -> int {
    const int k = copy_key + i * (kWarps * kKeys);
    return k < copy_end ? table[k >> p.page_shift] : -1;
  };
  // Starts stage i's copies into ring slot `slot`; which lanes' pieces exist.
  auto issue = [&](int i, int slot, int pg) -> uint32_t {
    const uint32_t bar = bars + 8 * slot;
    const bool there = (uint32_t)pg < (uint32_t)a.cache.num_pages;
    const uint32_t live = __ballot_sync(0xFFFFFFFFu, there);
    if (lane == 0)
      mbar_expect_tx(bar, (uint32_t)(__popc(live) / 4) * (uint32_t)(S::kStage / kKeys * piece));
    __syncwarp();
    if (there) {
      const int k = copy_key + i * (kWarps * kKeys);
      bulk_load(copy_dst + slot * S::kStage,
                copy_src + pg * page_stride + (k & (page_rows - 1)) * row_bytes, copy_bytes, bar);
    }
    return live;
  };
  // Which pieces of a stage in flight came, two bits a stage (bit 0: piece 0).
  uint32_t present = 0;
  auto note = [&](int slot, uint32_t live) {
    const int at = 2 * slot;
    present = (present & ~(3u << at)) | (((live & 1u) | ((live >> 3) & 2u)) << at);
  };
  for (int i = 0; i < S::kStages && i < n_stages; ++i) note(i, issue(i, i, page_of(i)));
  int next_page = page_of(S::kStages);

  // ---- queries: B fragments of f16, permuted as the keys are
  uint32_t q[kNT][S::kKSteps][2];
  float scale[kNT][2];
  int lo_key[kNT][2], hi_key[kNT][2];
  float acc[kNT][kD / 16][4], m[kNT][2], l[kNT][2];
  // the sign of the scale goes into Q, so that a larger score is a larger weight
  const float signed_log2 = a.softmax_scale * kLog2e / *a.cache.multiplier;
  const float to_log2 = fabsf(signed_log2);
  const bool flip = signed_log2 < 0.0f;
#pragma unroll
  for (int n = 0; n < kNT; ++n) {
    const int r = n * 8 + g;
    uint32_t w[kQuarter / 2];
    const bool live = r < tile.rows;
    if (live) {
      const int row = tile.row0 + r, token = row / p.group, hh = row - token * p.group;
      const uint16_t* src = a.q.p + (int64_t)(tile.first_token + token) * a.q.token_stride +
                            (int64_t)(head * p.group + hh) * a.q.head_stride + t * kQuarter;
#pragma unroll
      for (int j = 0; j < kQuarter / 8; ++j)
        *reinterpret_cast<uint4*>(&w[4 * j]) = *(reinterpret_cast<const uint4*>(src) + j);
    } else {
#pragma unroll
      for (int j = 0; j < kQuarter / 2; ++j) w[j] = 0;
    }
    float row_scale = to_log2;
    if (a.dtype == kDTypeBF16) {
      // bf16 has a wider range than f16: scale the row by a power of two that
      // brings its largest element into [1, 2); elements above 2^-17 of it
      // stay exact, the others are off by less than 2^-25 of it.
      uint32_t big = 0;
#pragma unroll
      for (int j = 0; j < kQuarter / 2; ++j)
        big = max(big, max((w[j] << 16) & 0x7FFFFFFFu, w[j] & 0x7FFF0000u));
      big = max(big, __shfl_xor_sync(0xFFFFFFFFu, big, 1));
      big = max(big, __shfl_xor_sync(0xFFFFFFFFu, big, 2));
      const int e = (int)(big >> 23);
      // exponents 1..253: 2^(127 - e) is a normal number; zero, subnormal, the
      // largest and non-finite rows are left as they are
      const bool sized = e >= 1 && e <= 253;
      const float size = sized ? __uint_as_float((uint32_t)(254 - e) << 23) : 1.0f;
      const float down = flip ? -size : size;
      row_scale = sized ? to_log2 * __uint_as_float((uint32_t)e << 23) : to_log2;
#pragma unroll
      for (int j = 0; j < kQuarter / 2; ++j)
        w[j] = pack_h2(__uint_as_float(w[j] << 16) * down,
                       __uint_as_float(w[j] & 0xFFFF0000u) * down);
    } else if (flip) {
#pragma unroll
      for (int j = 0; j < kQuarter / 2; ++j) w[j] ^= 0x80008000u;
    }
#pragma unroll
    for (int j = 0; j < S::kKSteps; ++j) {
      q[n][j][0] = w[2 * j];
      q[n][j][1] = w[2 * j + 1];
    }
    // columns 2t, 2t + 1 of the score tile are rows n * 8 + 2t, + 1
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      // never zero, or a masked score would be NaN
      scale[n][c] = fmaxf(__shfl_sync(0xFFFFFFFFu, row_scale, (2 * t + c) * 4), 1e-37f);
      const int rr = n * 8 + 2 * t + c;
      const int pos = tile.offset + (tile.row0 + rr) / p.group;
      const bool there = rr < tile.rows;
      hi_key[n][c] = !there ? -1 : a.causal ? min(pos, tile.end - 1) : tile.end - 1;
      lo_key[n][c] = a.window >= 0 ? pos - a.window : 0;
      m[n][c] = -INFINITY;
      l[n][c] = 0.0f;
    }
#pragma unroll
    for (int d = 0; d < kD / 16; ++d)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[n][d][c] = 0.0f;
  }

  // ---- one pass over this warp's stages
  // Row rho of a 16-key group's tile is key pi(rho): pi(2u) = u, pi(2u + 1) =
  // u + 4, pi(8 + 2u) = u + 8, pi(9 + 2u) = u + 12, so that the values a
  // thread pairs lie in rows t, t + 4, t + 8, t + 12.
  const int key_a = (g >> 1) + (g & 1) * 4;  // pi(g); pi(g + 8) = pi(g) + 8
  bool ok = true;
  int slot = 0;
  uint32_t phase = 0;
  for (int i = 0; i < n_stages; ++i) {
    const int k0 = c0 + (warp + i * kWarps) * kKeys;
    const int page_ahead = next_page;
    next_page = page_of(i + 1 + S::kStages);
    if (!warp_wait(bars + 8 * slot, phase)) {
      // give up: the copies still in flight get their (bounded) time to land
      for (int j = i; j < n_stages && j < i + S::kStages; ++j)
        warp_wait(bars + 8 * (j % S::kStages), (j / S::kStages) & 1);
      ok = false;
      break;
    }
    const uint8_t* st = smem + warp * S::kRing + slot * S::kStage;
    const uint8_t* kc = st;
    const uint8_t* ks = st + S::kKCodes;
    const uint8_t* vc = st + S::kKCodes + S::kKScales;
    const uint8_t* vs = vc + S::kKCodes;
    const uint32_t came = (present >> (2 * slot)) & 3u;
    const bool masked = k0 < tile.all_beg || k0 + kKeys > tile.all_end || k0 + kKeys > c1 ||
                        came != (pieces == 2 ? 3u : 1u);

    // One stage; without masks where every row of the tile sees all its keys.
    auto attend = [&](auto mask_tag) {
    constexpr bool masked = decltype(mask_tag)::value;
    // S^T = K Q^T
    float s[2][kNT][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t kw[2][kKWords], sc[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = h * 16 + key_a + 8 * r;
        const uint8_t* src = kc + row * S::kCodeRow + t * (kQuarter / 2);
        if constexpr (kKWords == 2) {
          *reinterpret_cast<uint2*>(kw[r]) = *reinterpret_cast<const uint2*>(src);
          sc[r] = ks[row * S::kScaleRow + t];
        } else {
#pragma unroll
          for (int j = 0; j < kKWords / 4; ++j)
            *reinterpret_cast<uint4*>(&kw[r][4 * j]) = *(reinterpret_cast<const uint4*>(src) + j);
          if constexpr (kKWords == 4)
            sc[r] = *reinterpret_cast<const uint16_t*>(ks + row * S::kScaleRow + 2 * t);
          else
            sc[r] = *reinterpret_cast<const uint32_t*>(ks + row * S::kScaleRow + 4 * t);
        }
      }
#pragma unroll
      for (int n = 0; n < kNT; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[h][n][c] = 0.0f;
      // two chains of accumulation, for the products' latency
      float s2[kNT][4] = {};
#pragma unroll
      for (int w = 0; w < kKWords; ++w) {
        // a word holds two steps of the same block; its scale, twice
        uint32_t x[2][4];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint32_t two = e4m3_h2(sc[r] >> (16 * (w / 4)));
          const uint32_t f = __byte_perm(two, two, (w / 2) & 1 ? 0x3232 : 0x1010);
          e2m1_h2x4(kw[r][w], x[r]);
#pragma unroll
          for (int b = 0; b < 4; ++b) x[r][b] = mul_h2(x[r][b], f);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int n = 0; n < kNT; ++n)
            mma16816(u ? s2[n] : s[h][n], x[0][2 * u], x[1][2 * u], x[0][2 * u + 1],
                     x[1][2 * u + 1], q[n][2 * w + u][0], q[n][2 * w + u][1]);
      }
#pragma unroll
      for (int n = 0; n < kNT; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[h][n][c] += s2[n][c];
    }

    // softmax over this stage's keys, in units of log2
    uint32_t pt[2][kNT][2];  // P^T as B fragments
    bool grow = false;
#pragma unroll
    for (int n = 0; n < kNT; ++n) {
      float mx[2] = {-INFINITY, -INFINITY}, seen[2] = {4.0f, 4.0f};
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float v = s[h][n][c];
          if constexpr (masked) {
            const int key = k0 + h * 16 + key_a + 8 * (c >> 1);
            const bool here = (came >> (pieces == 2 ? h : 0)) & 1u;
            if (!here || key >= c1 || key > hi_key[n][c & 1] || key < lo_key[n][c & 1]) {
              v = -INFINITY;
              seen[c & 1] -= 1.0f;
            }
          }
          s[h][n][c] = v;
          mx[c & 1] = fmaxf(mx[c & 1], v);
        }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        mx[c] = fmaxf(mx[c], __shfl_xor_sync(0xFFFFFFFFu, mx[c], 4));
        mx[c] = fmaxf(mx[c], __shfl_xor_sync(0xFFFFFFFFu, mx[c], 8));
        mx[c] = fmaxf(mx[c], __shfl_xor_sync(0xFFFFFFFFu, mx[c], 16));
        mx[c] *= scale[n][c];
        grow |= mx[c] > m[n][c] + kSlack;
      }
      if (__any_sync(0xFFFFFFFFu, grow)) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float mn = fmaxf(m[n][c], mx[c]);
          const float f = mn == -INFINITY ? 1.0f : ex2(m[n][c] - mn);
          m[n][c] = mn;
          l[n][c] *= f;
#pragma unroll
          for (int d = 0; d < kD / 16; ++d) {
            acc[n][d][c] *= f;
            acc[n][d][c + 2] *= f;
          }
        }
      }
      const float m0 = m[n][0] == -INFINITY ? 0.0f : m[n][0] - kShift;
      const float m1 = m[n][1] == -INFINITY ? 0.0f : m[n][1] - kShift;
#pragma unroll
      for (int c = 0; c < 2; ++c)  // keys seen whose scores are all -inf: see row_inverse
        if (m[n][c] == -INFINITY) l[n][c] += seen[c];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float p0 = ex2(fmaf(s[h][n][0], scale[n][0], -m0));
        const float p1 = ex2(fmaf(s[h][n][1], scale[n][1], -m1));
        const float p2 = ex2(fmaf(s[h][n][2], scale[n][0], -m0));
        const float p3 = ex2(fmaf(s[h][n][3], scale[n][1], -m1));
        l[n][0] += p0 + p2;
        l[n][1] += p1 + p3;
        pt[h][n][0] = transpose8(pack_h2(p0, p1));
        pt[h][n][1] = transpose8(pack_h2(p2, p3));
      }
    }

    // O^T += V^T P^T
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t vw[4][kVWords], sc[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = h * 16 + t + 4 * r;
        const uint8_t* src = vc + row * S::kCodeRow + g * (kD / 16);
        if constexpr (kD == 64) {
          vw[r][0] = *reinterpret_cast<const uint32_t*>(src);
          sc[r] = vs[row * S::kScaleRow + (g >> 1)];
        } else if constexpr (kD == 128) {
          *reinterpret_cast<uint2*>(vw[r]) = *reinterpret_cast<const uint2*>(src);
          sc[r] = vs[row * S::kScaleRow + g];
        } else {
          *reinterpret_cast<uint4*>(vw[r]) = *reinterpret_cast<const uint4*>(src);
          sc[r] = *reinterpret_cast<const uint16_t*>(vs + row * S::kScaleRow + 2 * g);
        }
        // what lies behind the last key may hold anything, NaN scales too
        if constexpr (masked) {
          const int key = k0 + row;
          const bool here = (came >> (pieces == 2 ? h : 0)) & 1u;
          if (!here || key >= c1 || key < tile.beg) sc[r] = 0;
        }
      }
      // scales of key pairs (t, t + 4) and (t + 8, t + 12)
      uint32_t f[2][kD == 256 ? 2 : 1];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        f[u][0] = e4m3_h2((sc[2 * u] & 0xFF) | ((sc[2 * u + 1] & 0xFF) << 8));
        if constexpr (kD == 256) f[u][1] = e4m3_h2((sc[2 * u] >> 8) | (sc[2 * u + 1] & 0xFF00));
      }
#pragma unroll
      for (int w = 0; w < kVWords; ++w) {
        uint32_t even[2], odd[2];  // bytes (code of the first key, code of the second) of even / odd d
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint32_t x = vw[2 * u][w], y = vw[2 * u + 1][w];
          even[u] = (x & 0x0F0F0F0Fu) | ((y << 4) & 0xF0F0F0F0u);
          odd[u] = ((x >> 4) & 0x0F0F0F0Fu) | (y & 0xF0F0F0F0u);
        }
        const int fi = kD == 256 ? w / 2 : 0;
        uint32_t he[2][4], ho[2][4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          e2m1_h2x4(even[u], he[u]);
          e2m1_h2x4(odd[u], ho[u]);
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            he[u][b] = mul_h2(he[u][b], f[u][fi]);
            ho[u][b] = mul_h2(ho[u][b], f[u][fi]);
          }
        }
        // tile w * 4 + b: row g is d = g * D/8 + 8 w + 2 b, row g + 8 the next
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
          for (int n = 0; n < kNT; ++n)
            mma16816(acc[n][w * 4 + b], he[0][b], ho[0][b], he[1][b], ho[1][b], pt[h][n][0],
                     pt[h][n][1]);
      }
    }
    };
    if (masked)
      attend(Flag<true>());
    else
      attend(Flag<false>());
    __syncwarp();  // every lane has read the stage before it is filled again
    if (i + S::kStages < n_stages) note(slot, issue(i + S::kStages, slot, page_ahead));
    if (++slot == S::kStages) {
      slot = 0;
      phase ^= 1;
    }
  }
  if (!ok) {  // unfinished rows are NaN
    if (lane == 0 && a.status) atomicCAS(a.status, 0, 1);
#pragma unroll
    for (int n = 0; n < kNT; ++n) l[n][0] = l[n][1] = NAN;
  }

  // ---- merge the warps through shared memory
#pragma unroll
  for (int n = 0; n < kNT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      l[n][c] += __shfl_xor_sync(0xFFFFFFFFu, l[n][c], 4);
      l[n][c] += __shfl_xor_sync(0xFFFFFFFFu, l[n][c], 8);
      l[n][c] += __shfl_xor_sync(0xFFFFFFFFu, l[n][c], 16);
    }
  __syncthreads();  // the rings are free
  float* mine = reinterpret_cast<float*>(smem) + warp * kRows * (kD + 2);
#pragma unroll
  for (int n = 0; n < kNT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float* row = mine + (n * 8 + 2 * t + c) * (kD + 2);
      if (g == 0) {
        row[kD] = m[n][c];
        row[kD + 1] = l[n][c];
      }
#pragma unroll
      for (int d = 0; d < kD / 16; ++d) {
        row[g * (kD / 8) + 2 * d] = acc[n][d][c];
        row[g * (kD / 8) + 2 * d + 1] = acc[n][d][c + 2];
      }
    }
  __syncthreads();
  const float inv_mult = 1.0f / a.cache.multiplier[1];
  const float* all = reinterpret_cast<const float*>(smem);
  constexpr int kStride = kRows * (kD + 2);
  for (int at = threadIdx.x; at < tile.rows * (kD / 2); at += kThreads) {
    const int r = at / (kD / 2), d = (at % (kD / 2)) * 2;
    const float* x = all + r * (kD + 2);
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, x[w * kStride + kD]);
    float o[2] = {0.0f, 0.0f}, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = part_weight(x[w * kStride + kD], mm);
      sum += f * x[w * kStride + kD + 1];
      o[0] += f * x[w * kStride + d];
      o[1] += f * x[w * kStride + d + 1];
    }
    const int row = tile.row0 + r, token = tile.first_token + row / p.group;
    const int qh = head * p.group + row % p.group;
    const int64_t out_row = (int64_t)token * a.q_heads + qh;
    if (p.splits == 1) {
      const float inv = row_inverse(mm, sum, inv_mult);
      o[0] *= inv;
      o[1] *= inv;
      store16(a.out.p + (int64_t)token * a.out.token_stride + (int64_t)qh * a.out.head_stride + d,
              o, a.dtype);
      if (d == 0 && a.lse)
        a.lse[out_row] = row_lse(mm, sum);
    } else {
      const int64_t at_row = part_row(p, split, seq, head, row, out_row);
      *reinterpret_cast<float2*>(p.part_o + at_row * kD + d) = make_float2(o[0], o[1]);
      if (d == 0) *reinterpret_cast<float2*>(p.part_ml + at_row * 2) = make_float2(mm, sum);
    }
  }
}

template <int kD, int kNT>
__global__ void __launch_bounds__(kThreads, kNT == 1 && kD <= 128 ? 4 : 1)
    decode_kernel(const Params p) {
  // Beside a prompt kernel, which this grid does not read from and which has
  // waited for everything before: it only ends after that one, so that what
  // follows finds both done.  Without a wait of its own at the start, fences
  // keep its loads from lines that the SM's cache had before, and order its bulk
  // copies behind what was written by plain stores.
  if (p.beside) {
    __threadfence();
    asm volatile("fence.proxy.async.global;" ::: "memory");
  } else {
    wait_for_predecessor();
  }
  let_successor_start();
  decode_tile<kD, kNT>(p);
  if (p.beside) wait_for_predecessor();
}

// Joins the splits of a row, always in the same order: of the row's kPerRow
// warps, warp w takes splits w, w + kPerRow, ..., then the warps' results are
// joined.  One warp is enough for few splits (64 sequences, 6 splits: 91 us with
// four warps per row, 89 with one), four for many.
template <int kD, int kPerRow>
__global__ void __launch_bounds__(kThreads) join_kernel(const Params p, int tile_rows) {
  constexpr int kPer = kD / 32;  // elements of a lane
  const AttendArgs& a = p.a;
  const int warp = (threadIdx.x >> 5) % kPerRow, lane = threadIdx.x & 31;
  const int head = blockIdx.z, seq = blockIdx.x / p.tiles;
  const int r = blockIdx.y * (kWarps / kPerRow) + (threadIdx.x >> 5) / kPerRow;
  // Everything that does not read the other grid's results comes before the
  // wait (behind it, 64 sequences took 95 us against 94): the other grid or,
  // beside prompts, the one before it let this one start after waiting for what
  // wrote the inputs, and writes none of them; the fence keeps these loads from
  // lines that the SM's cache had before.  CTAs without a row wait too, so that
  // this grid does not end first.
  __threadfence();
  Tile tile;
  if (!tile_of(p, seq, blockIdx.x % p.tiles, tile_rows, tile) || r >= tile.rows) {
    wait_for_predecessor();
    return;
  }
  const int splits = used_splits(p, tile);
  const int row = tile.row0 + r, token = tile.first_token + row / p.group;
  const int qh = head * p.group + row % p.group;
  const int64_t out_row = (int64_t)token * a.q_heads + qh;
  const int64_t step = p.part_rows, first_part = part_row(p, 0, seq, head, row, out_row);
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + first_part;
  const float* po = p.part_o + first_part * kD + lane * kPer;
  const float inv_mult = 1.0f / a.cache.multiplier[1];
  wait_for_predecessor();
  let_successor_start();
  // one pass with a running maximum, kBatch splits' loads in flight
  constexpr int kBatch = 4;
  float mm = -INFINITY, sum = 0.0f, acc[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) acc[j] = 0.0f;
#pragma unroll 1
  for (int first = warp; first < splits; first += kPerRow * kBatch) {
    float2 x[kBatch];
    float v[kBatch][kPer];
    float top = mm;
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int s = first + b * kPerRow;
      x[b] = make_float2(-INFINITY, 0.0f);
      if (s < splits) {
        x[b] = ml[s * step];
#pragma unroll
        for (int j = 0; j < kPer / 2; ++j)
          *reinterpret_cast<float2*>(v[b] + 2 * j) =
              *reinterpret_cast<const float2*>(po + s * step * kD + 2 * j);
      } else {
#pragma unroll
        for (int j = 0; j < kPer; ++j) v[b][j] = 0.0f;
      }
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) top = fmaxf(top, x[b].x);
    const float keep = part_weight(mm, top);
    mm = top;
    sum *= keep;
#pragma unroll
    for (int j = 0; j < kPer; ++j) acc[j] *= keep;
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const float f = part_weight(x[b].x, mm);
      sum += f * x[b].y;
#pragma unroll
      for (int j = 0; j < kPer; ++j) acc[j] += f * v[b][j];
    }
  }
  uint16_t* dst = a.out.p + (int64_t)token * a.out.token_stride + (int64_t)qh * a.out.head_stride;
  if constexpr (kPerRow == 1) {
    const float inv = row_inverse(mm, sum, inv_mult);
#pragma unroll
    for (int j = 0; j < kPer; j += 2) {
      const float v[2] = {acc[j] * inv, acc[j + 1] * inv};
      store16(dst + lane * kPer + j, v, a.dtype);
    }
    if (lane == 0 && a.lse) a.lse[out_row] = row_lse(mm, sum);
  } else {
    static_assert(kPerRow == kWarps, "the CTA's row");
    __shared__ float part[kWarps][kD];
    __shared__ float part_m[kWarps], part_l[kWarps];
#pragma unroll
    for (int j = 0; j < kPer; ++j) part[warp][lane * kPer + j] = acc[j];
    if (lane == 0) {
      part_m[warp] = mm;
      part_l[warp] = sum;
    }
    __syncthreads();
    float all = part_m[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) all = fmaxf(all, part_m[w]);
    float f[kWarps], total = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      f[w] = part_weight(part_m[w], all);
      total += f[w] * part_l[w];
    }
    const float inv = row_inverse(all, total, inv_mult);
    for (int d = threadIdx.x * 2; d < kD; d += kThreads * 2) {
      float v[2] = {0.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        v[0] += f[w] * part[w][d];
        v[1] += f[w] * part[w][d + 1];
      }
      v[0] *= inv;
      v[1] *= inv;
      store16(dst + d, v, a.dtype);
    }
    if (threadIdx.x == 0 && a.lse) a.lse[out_row] = row_lse(all, total);
  }
}

int log2i(int v) {
  int s = 0;
  while ((1 << s) < v) ++s;
  return s;
}

// How one kernel cuts the batch.
struct Cut {
  int rows;    // of a tile; 0: not launched
  int prompt;  // 1: the kernels of kv_prompt.cu
  int tiles, splits, chunk;
  int min_rows, max_rows;
};
struct Plan {
  Cut decode, prompt;
};

// `most` rows at most per sequence.  The keys are cut so that `wave` CTAs fill
// the GPU once or, where `fine` is more, into that many as far as splits keep
// `floor` keys; never below `min_chunk`.
Cut cut_of(const AttendArgs& a, int tile_rows, int64_t most, int64_t wave, int64_t fine,
           int64_t floor, int64_t min_chunk) {
  Cut c = {};
  c.rows = tile_rows;
  c.tiles = (int)((most + tile_rows - 1) / tile_rows);
  const int group = a.q_heads / a.cache.kv_heads;
  const int64_t tokens = (tile_rows + group - 1) / group + 1;  // that a tile's rows touch
  // a window bounds a tile's keys from both sides in the causal order only
  int64_t span = a.max_seq_len;
  if (a.causal && a.window >= 0 && span > (int64_t)a.window + tokens + kKeys)
    span = (int64_t)a.window + tokens + kKeys;
  const int64_t units = (int64_t)a.seqs * c.tiles * a.cache.kv_heads;
  auto chunk_for = [&](int64_t ctas) {
    const int64_t splits = ctas / units < 1 ? 1 : ctas / units;
    return ((span + splits - 1) / splits + 127) / 128 * 128;
  };
  int64_t chunk = chunk_for(wave);
  if (fine > wave) {
    const int64_t finer = chunk_for(fine) < floor ? floor : chunk_for(fine);
    if (chunk > finer) chunk = finer;
  }
  // Two stages per warp cost less than the second launch (one sequence of 256
  // keys: 5.8 us in one CTA per head, 6.2 split; of 300 keys 7.0 and 6.3).
  if (span <= 256 && tile_rows <= 8) chunk = 256;
  if (chunk < min_chunk) chunk = min_chunk;
  c.chunk = (int)chunk;
  // the first key of a windowed tile is rounded down to a stage
  c.splits = (int)((span + (a.window >= 0 ? kKeys - 1 : 0) + chunk - 1) / chunk);
  return c;
}

// A start and a partial result are what a split costs, so the keys are cut into
// one wave of CTAs: 4 per SM with 8 rows and heads up to 128, else 2 (8
// sequences of 4096 keys: 16.2 us, cut into two waves 18.9, into six 24).
// Sequences of several lengths are cut finer, into up to 24 CTAs per SM, so that
// the longest do not run on alone (64 of up to 8192 keys: 89 us, 98 with 12 per
// SM), but not below 1024 keys (16 of up to 8192: 27 us, 30 with 512) or, two
// per SM, 2048 (16 rows, 64 of up to 8192: 78 us, 82 with 1024).  A single
// sequence takes 3 and 2 CTAs per SM (131072 keys: 45 us, 60 with 4; with 16
// rows 36 us, 50 with 3).
Cut decode_cut(const AttendArgs& a, int tile_rows, int64_t most, int64_t sms) {
  const bool four = tile_rows == 8 && a.cache.head_size <= 128;
  if (a.seqs == 1) {
    const int64_t wave = sms * (four ? 3 : 2);
    return cut_of(a, tile_rows, most, wave, wave, 0, 128);
  }
  return cut_of(a, tile_rows, most, sms * (four ? 4 : 2), sms * 24, four ? 1024 : 2048, 128);
}

Plan plan_of(const AttendArgs& a, int device_sms) {
  const int group = a.q_heads / a.cache.kv_heads;
  const int64_t rows = (int64_t)a.max_query_len * group;
  // Rows up to which decode_kernel is the faster one (32 sequences of 8192 keys, 8
  // kv heads, 32 rows: heads of 64 in one tile 142 us, 234 on the tensor cores'
  // own memory; heads of 128 in two tiles of 16 226 and 274; heads of 256 so 422
  // and 371).
  const int most = a.cache.head_size == 256 ? 16 : 32;
  const int64_t sms = device_sms;
  Plan pl = {};
  if (rows <= most) {
    const int tile_rows = rows <= 8 ? 8 : rows <= 16 || a.cache.head_size == 128 ? 16 : 32;
    pl.decode = decode_cut(a, tile_rows, rows, sms);
    pl.decode.max_rows = 0x7FFFFFFF;
    return pl;
  }
  // One wave of CTAs, one per SM.  What a split costs (a launch, partial results
  // of all its rows) pays down to 256 keys where one tile holds all rows (64
  // queries, 2048 keys: 15.3 us, 18.1 with 512), else to 512 (512 queries, 512
  // keys: 15.7, 20.8 with 256).  Several such sequences are cut finer, to even
  // out their lengths (16 queries each of 4 of up to 65536 keys: 180 us, 235 in
  // one wave), those of more rows are not (500 each of 8 of up to 4096: 184, 243
  // with splits of 2048).
  const int tile_rows = prompt_rows(a.cache.head_size);
  const bool one = rows <= tile_rows;
  pl.prompt = cut_of(a, tile_rows, rows, sms, one && a.seqs > 1 ? sms * 4 : sms, 2048,
                     one ? 256 : 512);
  pl.prompt.prompt = 1;
  pl.prompt.max_rows = 0x7FFFFFFF;
  if (a.seqs > 1) {  // single tokens among prompts (how many is not known here: as if all were)
    const int few = group <= 8 ? 8 : 16;
    pl.decode = decode_cut(a, few, few, sms);
    pl.decode.max_rows = few;
    pl.prompt.min_rows = pl.decode.rows + 1;
  }
  return pl;
}

// The rows of one cut's partial results, for each of its splits: those of the
// batch or, where that is less, as many per sequence as the cut takes (single
// tokens among the rows of prompts; a query tensor padded far past its rows).
// The two cuts' kernels follow each other where both are split, so they share
// the memory.
struct Parts {
  int64_t rows;  // of a split; 0: not split
  int seq_rows;  // Params::part_seq_rows
};
Parts parts_of(const AttendArgs& a, const Cut& c) {
  if (c.rows == 0 || c.splits == 1) return {0, 0};
  const int64_t all = a.tokens * a.q_heads, seq_rows = (int64_t)c.tiles * c.rows;
  const int64_t some = (int64_t)a.seqs * a.cache.kv_heads * seq_rows;
  return some < all ? Parts{some, (int)seq_rows} : Parts{all, 0};
}

int64_t part_rows(const AttendArgs& a, const Cut& c) { return parts_of(a, c).rows * c.splits; }

template <int kD, int kNT>
cudaError_t launch_decode(const Params& p, cudaStream_t stream) {
  constexpr int kSmem = smem_bytes<kD, kNT>();
  static_assert(kSmem <= 227 * 1024, "shared memory");
  // One sequence is cut for three CTAs per SM.  A grid set up while its
  // predecessor still holds some SMs would put four on others and wait for
  // those (131072 keys: 54 us against 46), so with long splits it asks for a
  // third of the shared memory.
  constexpr int kThird = 60 * 1024;
  constexpr int kMost = kSmem < kThird ? kThird : kSmem;
  const int bytes = p.a.seqs == 1 && p.chunk >= 1024 ? kMost : kSmem;
  // always the same limit: another thread may be between this and its launch
  const cudaError_t e = cudaFuncSetAttribute(
      decode_kernel<kD, kNT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost);
  if (e != cudaSuccess) return e;
  return launch_dependent(
      decode_kernel<kD, kNT>,
      dim3((unsigned)(p.a.seqs * p.tiles), p.splits, p.a.cache.kv_heads), kThreads, bytes, stream, p);
}

template <int kD>
cudaError_t launch_rows(const Params& p, int rows, cudaStream_t stream) {
  if (rows == 8) return launch_decode<kD, 1>(p, stream);
  if (rows == 16) return launch_decode<kD, 2>(p, stream);
  if constexpr (kD == 64) return launch_decode<kD, 4>(p, stream);
  return cudaErrorInvalidValue;
}

template <int kD>
cudaError_t launch_join(const Params& p, int tile_rows, cudaStream_t stream) {
  const int64_t longest = (int64_t)p.a.max_query_len * p.group;  // rows of a sequence
  const unsigned rows = (unsigned)(longest < tile_rows ? longest : tile_rows);
  const bool few = p.splits <= 8;
  const dim3 grid((unsigned)(p.a.seqs * p.tiles), few ? (rows + kWarps - 1) / kWarps : rows,
                  p.a.cache.kv_heads);
  return launch_dependent(few ? join_kernel<kD, 1> : join_kernel<kD, kWarps>, grid, kThreads, 0,
                          stream, p, tile_rows);
}

cudaError_t launch_cut(Params p, const Cut& c, cudaStream_t stream) {
  if (c.rows == 0) return cudaSuccess;
  p.tiles = c.tiles;
  p.splits = c.splits;
  p.chunk = c.chunk;
  p.min_rows = c.min_rows;
  p.max_rows = c.max_rows;
  const Parts parts = parts_of(p.a, c);
  p.part_rows = parts.rows;
  p.part_seq_rows = parts.seq_rows;
  p.part_o = p.a.workspace;
  p.part_ml = p.a.workspace + parts.rows * c.splits * p.a.cache.head_size;
  const int d = p.a.cache.head_size;
  cudaError_t e = c.prompt   ? launch_prompt(p, stream)
                  : d == 64  ? launch_rows<64>(p, c.rows, stream)
                  : d == 128 ? launch_rows<128>(p, c.rows, stream)
                             : launch_rows<256>(p, c.rows, stream);
  if (e != cudaSuccess || c.splits == 1) return e;
  return d == 64    ? launch_join<64>(p, c.rows, stream)
         : d == 128 ? launch_join<128>(p, c.rows, stream)
                    : launch_join<256>(p, c.rows, stream);
}

}  // namespace

int64_t attend_workspace_bytes(const AttendArgs& a, int device_sms) {
  const Plan pl = plan_of(a, device_sms);
  const int64_t x = part_rows(a, pl.decode), y = part_rows(a, pl.prompt);
  return (x > y ? x : y) * (a.cache.head_size + 2) * (int64_t)sizeof(float);
}

cudaError_t launch_attend(const AttendArgs& a, int device_sms, cudaStream_t stream) {
  const Plan pl = plan_of(a, device_sms);
  Params p = {};
  p.a = a;
  if (a.window > (1 << 30)) p.a.window = 1 << 30;  // positions stay below it
  p.group = a.q_heads / a.cache.kv_heads;
  p.page_shift = log2i(a.cache.page_size);
  const cudaError_t e = launch_cut(p, pl.prompt, stream);
  if (e != cudaSuccess) return e;
  // Single tokens do not depend on the prompts: their kernel may start while the
  // last prompt tiles run.
  p.beside = pl.prompt.rows && pl.prompt.splits == 1;
  return launch_cut(p, pl.decode, stream);
}

}  // namespace kv
}  // namespace ssw
