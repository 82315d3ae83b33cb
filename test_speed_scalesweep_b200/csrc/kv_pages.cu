// Pages of an NVFP4 cache: taking, sharing, releasing, compacting and copying
// them with all state on the device, so that a step neither waits for the host
// nor leaves a CUDA graph.
//
//   refcount [pages], block_table [max_seqs, columns] (-1: no page), seq_lens
//
// A call that allocates decides everything in one CTA (`plan` kernels: a scan
// over the requests and one over the reference counts, a few microseconds for
// a pool of tens of thousands of pages) and leaves a list of (source,
// destination) pages for a wide kernel that moves the bytes and the table rows.
// Pages are taken lowest first and in the order of the requests, so results do
// not depend on timing.  A call that cannot be served changes nothing and
// leaves a code in `status`.
#include <cstdint>
#include <cuda_runtime.h>

#include "kv.cuh"
#include "quant.cuh"
#include "sweep.cuh"

namespace ssw {
namespace kv {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kCopyThreads = 256;
constexpr int kChunk = kCopyThreads * 2 * 16;  // bytes that a CTA moves per item

// Exclusive scan over the CTA (1024 threads); *total gets the sum.
__device__ __forceinline__ int block_scan(int v, int* total) {
  __shared__ int sums[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xFFFFFFFFu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // sums may still be read from the call before
  if (lane == 31) sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int s = sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xFFFFFFFFu, s, o);
      if (lane >= o) s += y;
    }
    sums[lane] = s;
  }
  __syncthreads();
  *total = sums[31];
  return x - v + (warp ? sums[warp - 1] : 0);
}

// The `need` lowest pages without references, into `fresh`; how many there are (at most need).
__device__ int find_free(const int32_t* refcount, int num_pages, int need, int32_t* fresh) {
  int found = 0;
  for (int base = 0; base < num_pages && found < need; base += kPlanThreads * 4) {
    const int p0 = base + threadIdx.x * 4;
    int f[4], n = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[j] = p0 + j < num_pages && refcount[p0 + j] == 0;
      n += f[j];
    }
    int total;
    int at = found + block_scan(n, &total);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (f[j]) {
        if (at < need) fresh[at] = p0 + j;
        ++at;
      }
    found += total;
  }
  return min(found, need);
}

__device__ __forceinline__ void report(int32_t* status, int code) {
  if (status && threadIdx.x == 0) atomicCAS(status, 0, code);
}

// Workspace of the plans (32-bit words):
//   [0] pairs to copy  [1] 1 = the call goes ahead
//   then per plan: see PagesWork.
struct PagesWork {
  int32_t* head;    // [4]
  int32_t* len;     // [n] lengths before the call
  int32_t* first;   // [n + 1] first fresh page (fork), or first token (extend), of a request
  int32_t* fresh;   // free pages taken
  int32_t* source;  // pages to copy from
  int32_t* target;  // and to
  int32_t* remap;   // [num_pages] (compact)
};

__device__ __host__ __forceinline__ PagesWork work_of(int32_t* w, int64_t n, int64_t pages) {
  PagesWork k;
  k.head = w;
  k.len = w + 4;
  k.first = k.len + n;
  k.fresh = k.first + n + 1;
  k.source = k.fresh + pages;
  k.target = k.source + pages;
  k.remap = k.target + pages;
  return k;
}

// ---- fork: the full pages are shared, a part-filled last page is copied
__global__ void __launch_bounds__(kPlanThreads) fork_plan(const PagesArgs a, int32_t* ws) {
  wait_for_predecessor();
  let_successor_start();
  const PagesWork w = work_of(ws, a.n, a.n);
  const int page_mask = (1 << a.page_shift) - 1;
  int bad = 0, need = 0;
  for (int base = 0; base < a.n; base += kPlanThreads) {
    const int i = base + threadIdx.x;
    int part = 0;
    if (i < a.n) {
      const int parent = a.seqs[i], child = a.other[i];
      int len = 0;
      if ((uint32_t)parent >= (uint32_t)a.max_seqs || (uint32_t)child >= (uint32_t)a.max_seqs) {
        bad = 1;
      } else {
        len = a.seq_lens[parent];
        if (len < 0 || ((int64_t)len + page_mask) >> a.page_shift > a.columns) bad = 1;
      }
      w.len[i] = len;
      part = (len & page_mask) != 0;
    }
    int total;
    const int at = block_scan(part, &total);
    if (i < a.n) w.first[i] = need + at;
    need += total;
  }
  bad = __syncthreads_or(bad);
  // Every child has to be an empty sequence, named once: claim it by -1.
  int twice = 0;
  if (!bad) {
    for (int i = threadIdx.x; i < a.n; i += kPlanThreads)
      if (atomicCAS(&a.seq_lens[a.other[i]], 0, -1) != 0) twice = 1;
    twice = __syncthreads_or(twice);
    if (twice) {  // back to what it was: only claims made here are negative
      for (int i = threadIdx.x; i < a.n; i += kPlanThreads) {
        atomicCAS(&a.seq_lens[a.other[i]], -1, 0);
      }
      __syncthreads();
    }
  }
  const int found = bad || twice ? 0 : find_free(a.refcount, a.num_pages, need, w.fresh);
  __syncthreads();
  const bool go = !bad && !twice && found == need;
  if (!go) {
    if (!bad && !twice)
      for (int i = threadIdx.x; i < a.n; i += kPlanThreads) a.seq_lens[a.other[i]] = 0;
    report(a.status, bad || twice ? kPagesBadIndex : kPagesExhausted);
    if (threadIdx.x == 0) {
      w.head[0] = 0;
      w.head[1] = 0;
    }
    return;
  }
  for (int i = threadIdx.x; i < a.n; i += kPlanThreads) {
    const int len = w.len[i];
    a.seq_lens[a.other[i]] = len;
    if (len & page_mask) {
      const int at = w.first[i];
      w.source[at] = a.block_table[a.seqs[i] * a.table_stride + (len >> a.page_shift)];
      w.target[at] = w.fresh[at];
      a.refcount[w.fresh[at]] = 1;
    }
  }
  if (threadIdx.x == 0) {
    w.head[0] = need;
    w.head[1] = 1;
  }
}

// Moves kChunk bytes of page pair k's layer: items number pairs * layers *
// chunks (below 2^32: a pool's bytes over kChunk).  Divisions by multiplication:
// 64-bit ones took as long as the copy.
__device__ __forceinline__ void copy_item(const PoolArgs& c, const int32_t* source,
                                          const int32_t* target, uint32_t item) {
  const uint32_t per_page = c.code_chunks + c.scale_chunks;
  const uint32_t pair_layer = div_bpc(item, c.page_magic, c.page_shift);
  const int chunk = (int)(item - pair_layer * per_page);
  const uint32_t pair = div_bpc(pair_layer, c.layer_magic, c.layer_shift);
  const uint32_t layer = pair_layer - pair * c.layers;
  const int src = source[pair], dst = target[pair];
  if ((uint32_t)src >= (uint32_t)c.num_pages || (uint32_t)dst >= (uint32_t)c.num_pages) return;
  const bool codes = chunk < c.code_chunks;
  uint8_t* base = codes ? c.codes + layer * c.codes_layer_stride : c.scales + layer * c.scales_layer_stride;
  const int64_t stride = codes ? c.codes_page_stride : c.scales_page_stride;
  const int64_t off = (int64_t)(codes ? chunk : chunk - c.code_chunks) * kChunk + threadIdx.x * 16;
  const int64_t size = codes ? c.codes_page_bytes : c.scales_page_bytes;
  const uint8_t* from = base + src * stride + off;
  uint8_t* to = base + dst * stride + off;
  uint4 v[2];
#pragma unroll
  for (int j = 0; j < 2; ++j)
    if (off + j * kCopyThreads * 16 < size)
      v[j] = *reinterpret_cast<const uint4*>(from + j * kCopyThreads * 16);
#pragma unroll
  for (int j = 0; j < 2; ++j)
    if (off + j * kCopyThreads * 16 < size)
      *reinterpret_cast<uint4*>(to + j * kCopyThreads * 16) = v[j];
}

__device__ __forceinline__ void copy_pairs(const PoolArgs& c, const int32_t* source,
                                           const int32_t* target, int64_t pairs, int first, int step) {
  const int64_t items = pairs * c.layers * (c.code_chunks + c.scale_chunks);
  for (int64_t i = first; i < items; i += step) copy_item(c, source, target, (uint32_t)i);
}

// CTAs 0 .. n - 1 write the children's rows, the others copy.
__global__ void __launch_bounds__(kCopyThreads) fork_apply(const PagesArgs a, const PoolArgs c,
                                                           int32_t* ws) {
  const PagesWork w = work_of(ws, a.n, a.n);
  wait_for_predecessor();
  let_successor_start();
  if (w.head[1] == 0) return;
  const int i = blockIdx.x;
  if (i >= a.n) {
    copy_pairs(c, w.source, w.target, w.head[0], i - a.n, gridDim.x - a.n);
    return;
  }
  const int page_mask = (1 << a.page_shift) - 1;
  const int len = w.len[i], full = len >> a.page_shift;
  const int32_t* from = a.block_table + a.seqs[i] * a.table_stride;
  int32_t* to = a.block_table + a.other[i] * a.table_stride;
  if (len == 0) return;  // the child's row is empty already
  for (int col = threadIdx.x; col < a.columns; col += kCopyThreads) {
    int pg = -1;
    if (col < full) {
      pg = from[col];
      if ((uint32_t)pg < (uint32_t)a.num_pages) atomicAdd(&a.refcount[pg], 1);
    } else if (col == full && (len & page_mask)) {
      pg = w.fresh[w.first[i]];
    }
    to[col] = pg;
  }
}

// ---- free: one CTA per sequence; a sequence named twice is freed once.  Every CTA
// looks at all the indices first (at most a few reads per thread), so that with
// one out of range none frees anything.
__global__ void __launch_bounds__(kCopyThreads) free_kernel(const PagesArgs a) {
  wait_for_predecessor();
  let_successor_start();
  __shared__ int old;
  int bad = 0;
  for (int i = threadIdx.x; i < a.n; i += kCopyThreads)
    bad |= (uint32_t)a.seqs[i] >= (uint32_t)a.max_seqs;
  if (__syncthreads_or(bad)) {
    if (blockIdx.x == 0) report(a.status, kPagesBadIndex);
    return;
  }
  const int s = a.seqs[blockIdx.x];
  if (threadIdx.x == 0) old = atomicExch(&a.seq_lens[s], 0);
  __syncthreads();
  const int page_mask = (1 << a.page_shift) - 1;
  const int pages = min(a.columns, (int)(((int64_t)old + page_mask) >> a.page_shift));
  int32_t* row = a.block_table + s * a.table_stride;
  for (int col = threadIdx.x; col < pages; col += kCopyThreads) {
    const int pg = row[col];
    if ((uint32_t)pg < (uint32_t)a.num_pages) atomicSub(&a.refcount[pg], 1);
    row[col] = -1;
  }
}

// The last of n ascending starts that is at most k (the first is 0): the range
// that k lies in, empty ranges skipped.
__device__ __forceinline__ int last_at_most(const int32_t* starts, int n, int k) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (starts[mid] <= k) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// ---- extend: pages for new tokens, and their slots
__global__ void __launch_bounds__(kPlanThreads) extend_plan(const PagesArgs a, int64_t total_tokens,
                                                            int64_t most_pages, int32_t* ws) {
  wait_for_predecessor();
  let_successor_start();
  const PagesWork w = work_of(ws, a.n, most_pages);
  const int page_mask = (1 << a.page_shift) - 1;
  __shared__ unsigned long long asked;  // in 64 bits: the scan's 32 could wrap
  if (threadIdx.x == 0) asked = 0;
  __syncthreads();
  int bad = 0, longer = 0;
  int64_t tokens = 0;
  // claim every sequence (a length becomes ~length): none may be named twice
  for (int base = 0; base < a.n; base += kPlanThreads) {
    const int i = base + threadIdx.x;
    int more = 0, len = -1;
    if (i < a.n) {
      const int s = a.seqs[i];
      more = a.other[i];
      if ((uint32_t)s >= (uint32_t)a.max_seqs || more < 0 || more > total_tokens) {
        bad = 1;
        more = 0;
      } else {
        len = a.seq_lens[s];
        if (len < 0 || atomicCAS(&a.seq_lens[s], len, ~len) != len) {
          bad = 1;
          len = -1;  // not claimed here
        } else if (((int64_t)len + more + page_mask) >> a.page_shift > a.columns) {
          longer = 1;
        }
      }
      w.len[i] = len;
      if (more) atomicAdd(&asked, (unsigned long long)more);
    }
    int total;
    const int at = block_scan(more, &total);
    if (i < a.n) w.first[i] = (int)min(tokens + at, (int64_t)0x7FFFFFFF);
    tokens += total;
  }
  if (threadIdx.x == 0) w.first[a.n] = (int)min(tokens, (int64_t)0x7FFFFFFF);
  __syncthreads();
  if (asked != (unsigned long long)total_tokens) bad = 1;
  bad = __syncthreads_or(bad);
  longer = __syncthreads_or(longer);
  // pages each request needs, in order
  int need = 0;
  if (!bad && !longer) {
    for (int base = 0; base < a.n; base += kPlanThreads) {
      const int i = base + threadIdx.x;
      int grow = 0;
      if (i < a.n) {
        const int64_t len = w.len[i], after = len + a.other[i];
        grow = (int)(((after + page_mask) >> a.page_shift) - ((len + page_mask) >> a.page_shift));
      }
      int total;
      const int at = block_scan(grow, &total);
      if (i < a.n) w.source[i] = need + at;
      need += total;
    }
  }
  const int found = bad || longer ? -1 : find_free(a.refcount, a.num_pages, need, w.fresh);
  __syncthreads();
  const bool go = found == need;
  for (int i = threadIdx.x; i < a.n; i += kPlanThreads) {
    const int len = w.len[i];
    if (!go) {
      if (len >= 0) a.seq_lens[a.seqs[i]] = len;
      continue;
    }
    a.seq_lens[a.seqs[i]] = len + a.other[i];
  }
  for (int k = threadIdx.x; go && k < need; k += kPlanThreads) {
    const int i = last_at_most(w.source, a.n, k);  // the request that page k is for
    const int have = (int)(((int64_t)w.len[i] + page_mask) >> a.page_shift);
    a.block_table[a.seqs[i] * a.table_stride + have + (k - w.source[i])] = w.fresh[k];
    a.refcount[w.fresh[k]] = 1;
  }
  if (!go) report(a.status, bad ? kPagesBadIndex : longer ? kPagesTooLong : kPagesExhausted);
  if (threadIdx.x == 0) w.head[1] = go;
}

__global__ void __launch_bounds__(kCopyThreads) extend_slots(const PagesArgs a, int64_t total_tokens,
                                                             int64_t most_pages, int32_t* ws,
                                                             int64_t* slots) {
  const PagesWork w = work_of(ws, a.n, most_pages);
  const int64_t t = (int64_t)blockIdx.x * kCopyThreads + threadIdx.x;
  wait_for_predecessor();
  let_successor_start();
  if (t >= total_tokens) return;
  if (w.head[1] == 0) {
    slots[t] = -1;
    return;
  }
  const int lo = last_at_most(w.first, a.n, (int)t);  // the request that token t is of
  const int64_t pos = w.len[lo] + (t - w.first[lo]);
  const int pg = a.block_table[a.seqs[lo] * a.table_stride + (pos >> a.page_shift)];
  slots[t] = pg < 0 ? -1 : ((int64_t)pg << a.page_shift) + (pos & ((1 << a.page_shift) - 1));
}

// ---- compact: the live pages above the live count move into the holes below it
__global__ void __launch_bounds__(kPlanThreads) compact_plan(const PagesArgs a, int32_t* ws) {
  wait_for_predecessor();
  let_successor_start();
  const PagesWork w = work_of(ws, 0, a.num_pages);
  int live = 0;
  for (int p = threadIdx.x; p < a.num_pages; p += kPlanThreads) live += a.refcount[p] != 0;
  int n_live;
  block_scan(live, &n_live);
  int holes = 0, highs = 0;
  for (int base = 0; base < a.num_pages; base += kPlanThreads * 4) {
    const int p0 = base + threadIdx.x * 4;
    int take[4], n = 0;  // a hole below the count, or a live page above it
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int p = p0 + j;
      take[j] = p < a.num_pages && (p < n_live) == (a.refcount[p] == 0);
      // one scan for both: holes in the low half, high pages in the high half
      n += take[j] ? (p < n_live ? 1 : 0x10000) : 0;
      if (p < a.num_pages) w.remap[p] = p;
    }
    int total;
    const int at = block_scan(n, &total);
    int h = holes + (at & 0xFFFF), g = highs + (at >> 16);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (take[j]) {
        if (p0 + j < n_live) w.target[h++] = p0 + j;
        else w.source[g++] = p0 + j;
      }
    holes += total & 0xFFFF;
    highs += total >> 16;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < holes; i += kPlanThreads) {
    const int from = w.source[i], to = w.target[i];
    w.remap[from] = to;
    a.refcount[to] = a.refcount[from];
    a.refcount[from] = 0;
  }
  if (threadIdx.x == 0) w.head[0] = holes;
}

__global__ void __launch_bounds__(kCopyThreads) compact_apply(const PagesArgs a, const PoolArgs c,
                                                              int32_t* ws) {
  const PagesWork w = work_of(ws, 0, a.num_pages);
  wait_for_predecessor();
  let_successor_start();
  const int pairs = w.head[0];
  if (pairs == 0) return;
  copy_pairs(c, w.source, w.target, pairs, blockIdx.x, gridDim.x);
  const int64_t entries = (int64_t)a.max_seqs * a.columns;
  for (int64_t i = (int64_t)blockIdx.x * kCopyThreads + threadIdx.x; i < entries;
       i += (int64_t)gridDim.x * kCopyThreads) {
    int32_t* e = a.block_table + (i / a.columns) * a.table_stride + i % a.columns;
    const int pg = *e;
    if ((uint32_t)pg < (uint32_t)a.num_pages) {
      const int to = w.remap[pg];
      if (to != pg) *e = to;
    }
  }
}

__global__ void __launch_bounds__(kCopyThreads) copy_kernel(const PoolArgs c, const int32_t* source,
                                                            const int32_t* target, int64_t pairs) {
  wait_for_predecessor();
  let_successor_start();
  copy_pairs(c, source, target, pairs, blockIdx.x, gridDim.x);
}

PoolArgs with_chunks(PoolArgs c) {
  c.code_chunks = (int)((c.codes_page_bytes + kChunk - 1) / kChunk);
  c.scale_chunks = (int)((c.scales_page_bytes + kChunk - 1) / kChunk);
  make_divider((uint32_t)(c.code_chunks + c.scale_chunks), &c.page_magic, &c.page_shift);
  make_divider((uint32_t)c.layers, &c.layer_magic, &c.layer_shift);
  return c;
}

unsigned copy_grid(const PoolArgs& c, int64_t pairs, int device_sms) {
  const int64_t items = pairs * c.layers * (c.code_chunks + c.scale_chunks);
  const int64_t cap = (int64_t)device_sms * 8;
  return (unsigned)(items < 1 ? 1 : items < cap ? items : cap);
}

}  // namespace

int64_t pages_workspace_words(int64_t n, int64_t pages, int64_t num_pages_for_remap) {
  return 4 + n + n + 1 + 3 * (pages > n ? pages : n) + num_pages_for_remap;
}

cudaError_t launch_fork(const PagesArgs& a, const PoolArgs& pool, int32_t* ws, int device_sms,
                        cudaStream_t stream) {
  const PoolArgs c = with_chunks(pool);
  const cudaError_t e = launch_dependent(fork_plan, dim3(1), kPlanThreads, 0, stream, a, ws);
  if (e != cudaSuccess) return e;
  return launch_dependent(fork_apply, dim3(a.n + copy_grid(c, a.n, device_sms)), kCopyThreads, 0,
                          stream, a, c, ws);
}

cudaError_t launch_free(const PagesArgs& a, cudaStream_t stream) {
  return launch_dependent(free_kernel, dim3(a.n), kCopyThreads, 0, stream, a);
}

cudaError_t launch_extend(const PagesArgs& a, int64_t total_tokens, int64_t most_pages,
                          int64_t* slots, int32_t* ws, cudaStream_t stream) {
  const cudaError_t e = launch_dependent(extend_plan, dim3(1), kPlanThreads, 0, stream, a,
                                         total_tokens, most_pages, ws);
  if (e != cudaSuccess || total_tokens == 0) return e;
  return launch_dependent(extend_slots,
                          dim3((unsigned)((total_tokens + kCopyThreads - 1) / kCopyThreads)),
                          kCopyThreads, 0, stream, a, total_tokens, most_pages, ws, slots);
}

cudaError_t launch_compact(const PagesArgs& a, const PoolArgs& pool, int32_t* ws, int device_sms,
                           cudaStream_t stream) {
  const PoolArgs c = with_chunks(pool);
  const cudaError_t e = launch_dependent(compact_plan, dim3(1), kPlanThreads, 0, stream, a, ws);
  if (e != cudaSuccess) return e;
  return launch_dependent(compact_apply, dim3(copy_grid(c, a.num_pages / 2 + 1, device_sms)),
                          kCopyThreads, 0, stream, a, c, ws);
}

cudaError_t launch_copy(const PoolArgs& pool, const int32_t* source, const int32_t* target,
                        int64_t pairs, int device_sms, cudaStream_t stream) {
  const PoolArgs c = with_chunks(pool);
  return launch_dependent(copy_kernel, dim3(copy_grid(c, pairs, device_sms)), kCopyThreads, 0, stream,
                          c, source, target, pairs);
}

}  // namespace kv
}  // namespace ssw
