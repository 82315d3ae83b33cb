// Internal launch interface of the NVFP4 KV-cache kernels (not part of the C ABI).
//
// A cache page holds `page_size` tokens of every kv head:
//   codes  [pages, 2 (key, value), kv_heads, page_size, head_size / 2]   E2M1, element 2j in the low nibble
//   scales [pages, 2 (key, value), kv_heads, page_size, head_size / 16]  E4M3, one per 16 elements
// The pages may lie any multiple of 16 bytes apart (a layer of a cache that
// holds all layers); inside a page everything is contiguous.  A value is
// code * scale / multiplier, the multiplier being one float each for the keys
// and the values of a layer.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

namespace ssw {
namespace kv {

// Every kernel of the cache's operators is launched as a programmatic dependent
// of what precedes it on the stream, so that a chain of short kernels does not
// pay each launch in full.  Its first step is to wait for that grid, in all
// CTAs (a grid never ends before its predecessor, and what precedes the
// predecessor is done as well) before it reads anything; only then may its own
// successor be set up.  Inputs are read by plain loads: a non-coherent one asks
// that its memory stays unwritten while the grid lives, and the grid lives
// before its predecessor has written.  What reads inputs without a wait
// (join_kernel's tile, decode_kernel beside a prompt kernel) has a predecessor
// that waited for their writers and writes none of them, and fences first.
__device__ __forceinline__ void wait_for_predecessor() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
__device__ __forceinline__ void let_successor_start() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

template <typename... Params, typename... Args>
cudaError_t launch_dependent(void (*kernel)(Params...), dim3 grid, unsigned threads, size_t smem,
                             cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

struct Cache {
  uint8_t* codes;
  uint8_t* scales;
  int64_t codes_page_stride;   // bytes
  int64_t scales_page_stride;  // bytes
  const float* multiplier;     // [2]: keys, values
  int64_t num_pages;
  int32_t page_size;           // 16, 32, 64 or 128
  int32_t kv_heads;
  int32_t head_size;           // 64, 128 or 256
};

// A [tokens, heads, head_size] tensor of 16-bit floats: strides in elements,
// multiples of 8; the last dimension is contiguous.
struct Heads {
  uint16_t* p;
  int64_t token_stride;
  int64_t head_stride;
};

struct WriteArgs {
  Cache cache;
  Heads q, k, v, q_out;
  const int64_t* positions;  // [tokens]
  const float* cos_sin;      // [max_position, rotary_dim]: cos, then sin
  int64_t max_position;
  const int64_t* slots;      // [tokens]: page * page_size + row, < 0 = padding
  int64_t tokens;
  int32_t q_heads;
  int32_t rotary_dim;        // a multiple of 16, <= head_size
  int32_t neox;              // 1: pairs (i, i + rotary_dim / 2); 0: pairs (2i, 2i + 1)
  int32_t dtype;             // kDTypeBF16 / kDTypeF16
};
cudaError_t launch_write(const WriteArgs& a, int device_sms, cudaStream_t stream);

struct GatherArgs {
  Cache cache;
  const int64_t* slots;  // [tokens]
  int64_t tokens;
  uint16_t* key;         // [tokens, kv_heads, head_size]
  uint16_t* value;
  int32_t dtype;
};
cudaError_t launch_gather(const GatherArgs& a, int device_sms, cudaStream_t stream);

struct AttendArgs {
  Cache cache;
  Heads q, out;
  const int32_t* block_table;  // [seqs, table_columns] of page ids
  int64_t table_stride;        // elements
  const int32_t* seq_lens;     // [seqs]: keys of a sequence, its new tokens' included
  const int32_t* query_start;  // [seqs + 1]: first query token of a sequence
  float* lse;                  // [tokens, q_heads] or null
  float* workspace;            // partial results of split sequences
  int32_t* status;             // or null
  int64_t tokens;              // rows of q and out
  int32_t seqs, table_columns, q_heads, max_query_len, max_seq_len;
  int32_t causal, window;      // window < 0: none
  int32_t dtype;
  float softmax_scale;
};
int64_t attend_workspace_bytes(const AttendArgs& a, int device_sms);
cudaError_t launch_attend(const AttendArgs& a, int device_sms, cudaStream_t stream);

enum { kPagesExhausted = 1, kPagesBadIndex = 2, kPagesTooLong = 3 };

// The page tables of a cache and one request list.
struct PagesArgs {
  int32_t* refcount;     // [num_pages]
  int32_t* block_table;  // [max_seqs, columns]
  int64_t table_stride;  // elements
  int32_t* seq_lens;     // [max_seqs]
  int32_t* status;       // or null
  int32_t num_pages, max_seqs, columns, page_shift;
  const int32_t* seqs;   // [n]: parents, or sequences
  const int32_t* other;  // [n]: children, or numbers of new tokens
  int32_t n;
};

// The bytes of a cache's pages, over all its layers.
struct PoolArgs {
  uint8_t* codes;
  uint8_t* scales;
  int64_t codes_layer_stride, scales_layer_stride;  // bytes
  int64_t codes_page_stride, scales_page_stride;
  int64_t codes_page_bytes, scales_page_bytes;      // multiples of 16
  int64_t num_pages;
  int32_t layers;
  int32_t code_chunks, scale_chunks;                // filled at launch, as these
  uint32_t page_magic, page_shift, layer_magic, layer_shift;  // divisions by chunks, by layers
};

int64_t pages_workspace_words(int64_t n, int64_t pages, int64_t num_pages_for_remap);
cudaError_t launch_fork(const PagesArgs& a, const PoolArgs& pool, int32_t* ws, int device_sms,
                        cudaStream_t stream);
cudaError_t launch_free(const PagesArgs& a, cudaStream_t stream);
cudaError_t launch_extend(const PagesArgs& a, int64_t total_tokens, int64_t most_pages,
                          int64_t* slots, int32_t* ws, cudaStream_t stream);
cudaError_t launch_compact(const PagesArgs& a, const PoolArgs& pool, int32_t* ws, int device_sms,
                           cudaStream_t stream);
cudaError_t launch_copy(const PoolArgs& pool, const int32_t* source, const int32_t* target,
                        int64_t pairs, int device_sms, cudaStream_t stream);

}  // namespace kv
}  // namespace ssw
