// C ABI of the NVFP4 KV-cache operators: argument validation and error
// reporting.  Declarations and contracts live in include/scalesweep_b200.h.
#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include <cuda_runtime.h>

#include "../../include/scalesweep_b200.h"
#include "kv.cuh"
#include "quant.cuh"

namespace ssw {
void set_last_error(const char* msg);
}

namespace {

int fail(int status, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  ssw::set_last_error(buf);
  return status;
}

int cuda_fail(cudaError_t e, const char* what) {
  return fail(SSW_ERR_CUDA, "%s: %s (%s)", what, cudaGetErrorName(e), cudaGetErrorString(e));
}

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

// Streaming multiprocessors of the current device; -1 on failure.
int device_sms() {
  static int cache[64] = {0};
  int dev = 0, v = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return -1;
  if (dev >= 0 && dev < 64 && cache[dev] > 0) return cache[dev];
  if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return -1;
  if (dev >= 0 && dev < 64) cache[dev] = v;
  return v;
}

int check_cache(const char* name, const ssw_kv_cache* c, ssw::kv::Cache* out) {
  if (!c) return fail(SSW_ERR_INVALID_ARGUMENT, "%s: null cache", name);
  if (c->head_size != 64 && c->head_size != 128 && c->head_size != 256)
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: head_size must be 64, 128 or 256 (got %d)", name,
                c->head_size);
  if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128)
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: page_size must be 16, 32, 64 or 128 (got %d)", name,
                c->page_size);
  if (c->kv_heads < 1 || c->kv_heads > 1024)
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: kv_heads must be in 1..1024 (got %d)", name,
                c->kv_heads);
  if (c->num_pages < 0 || c->num_pages >= (1ll << 31))
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: num_pages must be in 0..2^31-1 (got %lld)", name,
                (long long)c->num_pages);
  const int64_t page = 2ll * c->kv_heads * c->page_size * c->head_size;
  if (c->num_pages > 1 && (c->codes_page_stride < page / 2 || c->scales_page_stride < page / 16))
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: the pages overlap (strides %lld and %lld bytes)",
                name, (long long)c->codes_page_stride, (long long)c->scales_page_stride);
  if (c->codes_page_stride % 16 || c->scales_page_stride % 16)
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: page strides must be multiples of 16 bytes", name);
  if (c->num_pages > 0 && (!c->codes || !c->scales))
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
  if (!aligned(c->codes, 16) || !aligned(c->scales, 16) || !aligned(c->input_scale, 4))
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: codes and scales must be 16-byte aligned", name);
  out->codes = c->codes;
  out->scales = c->scales;
  out->codes_page_stride = c->codes_page_stride;
  out->scales_page_stride = c->scales_page_stride;
  out->multiplier = c->input_scale;
  out->num_pages = c->num_pages;
  out->page_size = c->page_size;
  out->kv_heads = c->kv_heads;
  out->head_size = c->head_size;
  return SSW_OK;
}

int check_heads(const char* name, const char* which, const ssw_kv_heads* h, ssw::kv::Heads* out) {
  if (!h || !h->data) return fail(SSW_ERR_INVALID_ARGUMENT, "%s: null %s", name, which);
  if (!aligned(h->data, 16) || h->token_stride % 8 || h->head_stride % 8)
    return fail(SSW_ERR_INVALID_ARGUMENT,
                "%s: %s must be 16-byte aligned, its strides multiples of 8 elements", name, which);
  out->p = static_cast<uint16_t*>(h->data);
  out->token_stride = h->token_stride;
  out->head_stride = h->head_stride;
  return SSW_OK;
}

int check_dtype(const char* name, int dtype) {
  if (dtype != SSW_DTYPE_BF16 && dtype != SSW_DTYPE_F16)
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: dtype must be bf16 or f16 (got %d)", name, dtype);
  return SSW_OK;
}

}  // namespace

extern "C" {

int ssw_rotary_scalesweep_mse_nvfp4_kv_write(const ssw_kv_cache* cache, int dtype, int64_t tokens,
                                             int q_heads, const ssw_kv_heads* query,
                                             const ssw_kv_heads* key, const ssw_kv_heads* value,
                                             const ssw_kv_heads* query_out,
                                             const int64_t* positions, const float* cos_sin_cache,
                                             int64_t max_position, int rotary_dim, int is_neox,
                                             const int64_t* slot_mapping, void* stream) {
  const char* name = "rotary_scalesweep_mse_nvfp4_kv_write";
  ssw::set_last_error("");
  ssw::kv::WriteArgs a;
  int st = check_cache(name, cache, &a.cache);
  if (st == SSW_OK) st = check_dtype(name, dtype);
  if (st != SSW_OK) return st;
  if (tokens < 0 || q_heads < 1 || q_heads > 65536)
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: bad sizes tokens=%lld q_heads=%d", name,
                (long long)tokens, q_heads);
  if (rotary_dim < 16 || rotary_dim % 16 || rotary_dim > cache->head_size)
    return fail(SSW_ERR_INVALID_ARGUMENT,
                "%s: rotary_dim must be a multiple of 16 up to head_size (got %d)", name,
                rotary_dim);
  if (max_position < 1)
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: the cos/sin table is empty", name);
  const int64_t widest = q_heads > 2 * cache->kv_heads ? q_heads : 2 * cache->kv_heads;
  if (tokens > 0 && tokens >= (1ll << 32) / (widest * (cache->head_size / 16)))
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: too many tokens for one call (%lld)", name,
                (long long)tokens);
  if (tokens == 0) return SSW_OK;
  if ((st = check_heads(name, "query", query, &a.q)) != SSW_OK) return st;
  if ((st = check_heads(name, "key", key, &a.k)) != SSW_OK) return st;
  if ((st = check_heads(name, "value", value, &a.v)) != SSW_OK) return st;
  if ((st = check_heads(name, "query_out", query_out, &a.q_out)) != SSW_OK) return st;
  if (!positions || !cos_sin_cache || !slot_mapping || !cache->input_scale)
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
  if (!aligned(positions, 8) || !aligned(slot_mapping, 8) || !aligned(cos_sin_cache, 16))
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: misaligned positions, slots or cos/sin table", name);
  const int sms = device_sms();
  if (sms < 0) return fail(SSW_ERR_CUDA, "%s: no CUDA device", name);
  a.positions = positions;
  a.cos_sin = cos_sin_cache;
  a.max_position = max_position;
  a.slots = slot_mapping;
  a.tokens = tokens;
  a.q_heads = q_heads;
  a.rotary_dim = rotary_dim;
  a.neox = is_neox ? 1 : 0;
  a.dtype = dtype;
  const cudaError_t e = ssw::kv::launch_write(a, sms, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? SSW_OK : cuda_fail(e, name);
}

int ssw_nvfp4_kv_gather(const ssw_kv_cache* cache, int dtype, int64_t tokens,
                        const int64_t* slot_mapping, void* key, void* value, void* stream) {
  const char* name = "nvfp4_kv_gather";
  ssw::set_last_error("");
  ssw::kv::GatherArgs a;
  int st = check_cache(name, cache, &a.cache);
  if (st == SSW_OK) st = check_dtype(name, dtype);
  if (st != SSW_OK) return st;
  if (tokens < 0) return fail(SSW_ERR_INVALID_ARGUMENT, "%s: negative size", name);
  if (tokens > 0 && tokens >= (1ll << 32) / (2 * cache->kv_heads * (cache->head_size / 16)))
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: too many tokens for one call (%lld)", name,
                (long long)tokens);
  if (tokens == 0) return SSW_OK;
  if (!slot_mapping || !key || !value || !cache->input_scale)
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
  if (!aligned(slot_mapping, 8) || !aligned(key, 16) || !aligned(value, 16))
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: misaligned slots, key or value", name);
  const int sms = device_sms();
  if (sms < 0) return fail(SSW_ERR_CUDA, "%s: no CUDA device", name);
  a.slots = slot_mapping;
  a.tokens = tokens;
  a.key = static_cast<uint16_t*>(key);
  a.value = static_cast<uint16_t*>(value);
  a.dtype = dtype;
  const cudaError_t e = ssw::kv::launch_gather(a, sms, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? SSW_OK : cuda_fail(e, name);
}


namespace {

int attend_args(const char* name, const ssw_kv_cache* cache, const ssw_kv_attention* x, int dtype,
                ssw::kv::AttendArgs* a) {
  int st = check_cache(name, cache, &a->cache);
  if (st == SSW_OK) st = check_dtype(name, dtype);
  if (st != SSW_OK) return st;
  if (!x) return fail(SSW_ERR_INVALID_ARGUMENT, "%s: null arguments", name);
  if (x->q_heads < 1 || x->q_heads > 65536 || x->q_heads % cache->kv_heads)
    return fail(SSW_ERR_INVALID_ARGUMENT,
                "%s: q_heads must be a multiple of the cache's %d kv heads (got %d)", name,
                cache->kv_heads, x->q_heads);
  if (x->tokens < 0 || x->tokens >= (1ll << 31) / x->q_heads || x->seqs < 0)
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: bad sizes tokens=%lld seqs=%d", name,
                (long long)x->tokens, x->seqs);
  if (x->max_query_len < 1 || x->max_seq_len < 1 || x->max_seq_len > (1 << 30) ||
      x->max_query_len > (1 << 30) / (x->q_heads / cache->kv_heads))
    return fail(SSW_ERR_INVALID_ARGUMENT,
                "%s: max_query_len and max_seq_len must be positive and below 2^30 rows (got %d, %d)",
                name, x->max_query_len, x->max_seq_len);
  if (x->block_table_columns < 1 || x->block_table_stride < x->block_table_columns)
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: bad block table (%d columns, stride %lld)", name,
                x->block_table_columns, (long long)x->block_table_stride);
  if (!(x->softmax_scale == x->softmax_scale) || x->softmax_scale - x->softmax_scale != 0.0f)
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: softmax_scale must be finite", name);
  a->block_table = x->block_table;
  a->table_stride = x->block_table_stride;
  a->seq_lens = x->seq_lens;
  a->query_start = x->query_start;
  a->lse = x->lse;
  a->status = x->status;
  a->tokens = x->tokens;
  a->seqs = x->seqs;
  a->table_columns = x->block_table_columns;
  a->q_heads = x->q_heads;
  a->max_query_len = x->max_query_len;
  a->max_seq_len = x->max_seq_len;
  a->causal = x->causal ? 1 : 0;
  a->window = x->window;
  a->dtype = dtype;
  a->softmax_scale = x->softmax_scale;
  return SSW_OK;
}

}  // namespace

int64_t ssw_nvfp4_paged_attention_workspace_bytes(const ssw_kv_cache* cache,
                                                  const ssw_kv_attention* args, int dtype) {
  ssw::kv::AttendArgs a;
  ssw::set_last_error("");
  const int sms = device_sms();
  if (sms < 0 || attend_args("nvfp4_paged_attention", cache, args, dtype, &a) != SSW_OK) return -1;
  if (a.tokens == 0 || a.seqs == 0) return 0;
  return ssw::kv::attend_workspace_bytes(a, sms);
}

int ssw_nvfp4_paged_attention(const ssw_kv_cache* cache, const ssw_kv_attention* args, int dtype,
                              const ssw_kv_heads* query, const ssw_kv_heads* out, void* workspace,
                              int64_t workspace_bytes, void* stream) {
  const char* name = "nvfp4_paged_attention";
  ssw::set_last_error("");
  ssw::kv::AttendArgs a;
  int st = attend_args(name, cache, args, dtype, &a);
  if (st != SSW_OK) return st;
  if (a.tokens == 0 || a.seqs == 0) return SSW_OK;
  if ((st = check_heads(name, "query", query, &a.q)) != SSW_OK) return st;
  if ((st = check_heads(name, "out", out, &a.out)) != SSW_OK) return st;
  if (!a.block_table || !a.seq_lens || !a.query_start || !cache->input_scale)
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
  if (!aligned(a.block_table, 4) || !aligned(a.seq_lens, 4) || !aligned(a.query_start, 4) ||
      !aligned(a.lse, 4) || !aligned(workspace, 16))
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: misaligned pointer", name);
  const int sms = device_sms();
  if (sms < 0) return fail(SSW_ERR_CUDA, "%s: no CUDA device", name);
  const int64_t need = ssw::kv::attend_workspace_bytes(a, sms);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: the workspace must hold %lld bytes", name,
                (long long)need);
  a.workspace = static_cast<float*>(workspace);
  const cudaError_t e = ssw::kv::launch_attend(a, sms, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? SSW_OK : cuda_fail(e, name);
}

}  // extern "C"
