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
  // a launch has a CTA column per sequence and 8 rows of the longest query
  if ((int64_t)x->seqs * ((int64_t)x->max_query_len * (x->q_heads / cache->kv_heads) / 8 + 1) >=
      (1ll << 31))
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: %d sequences of up to %d queries are too many", name,
                x->seqs, x->max_query_len);
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

namespace {

int check_pool(const char* name, const ssw_kv_pool* p, ssw::kv::PoolArgs* out) {
  if (!p) return fail(SSW_ERR_INVALID_ARGUMENT, "%s: null pool", name);
  if (p->layers < 1 || p->num_pages < 1 || p->num_pages >= (1ll << 31))
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: bad sizes layers=%d num_pages=%lld", name, p->layers,
                (long long)p->num_pages);
  if (p->codes_page_bytes < 16 || p->scales_page_bytes < 16 || p->codes_page_bytes % 16 ||
      p->scales_page_bytes % 16 || p->codes_page_bytes > (1ll << 30) ||
      p->scales_page_bytes > (1ll << 30))
    return fail(SSW_ERR_INVALID_ARGUMENT,
                "%s: a page's bytes must be a multiple of 16 up to 2^30 (got %lld and %lld)", name,
                (long long)p->codes_page_bytes, (long long)p->scales_page_bytes);
  if (p->codes_page_stride % 16 || p->scales_page_stride % 16 || p->codes_layer_stride % 16 ||
      p->scales_layer_stride % 16 || p->codes_page_stride < p->codes_page_bytes ||
      p->scales_page_stride < p->scales_page_bytes)
    return fail(SSW_ERR_INVALID_ARGUMENT,
                "%s: strides must be multiples of 16 bytes and pages must not overlap", name);
  if (!p->codes || !p->scales || !aligned(p->codes, 16) || !aligned(p->scales, 16))
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: codes and scales must be 16-byte aligned, not null",
                name);
  // items of a copy are counted in 32 bits
  if (p->num_pages * p->layers >
      (int64_t)((1ll << 32) / ((p->codes_page_bytes + p->scales_page_bytes) / 8192 + 2)))
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: %lld pages in %d layers are too many", name,
                (long long)p->num_pages, p->layers);
  out->codes = p->codes;
  out->scales = p->scales;
  out->codes_layer_stride = p->codes_layer_stride;
  out->scales_layer_stride = p->scales_layer_stride;
  out->codes_page_stride = p->codes_page_stride;
  out->scales_page_stride = p->scales_page_stride;
  out->codes_page_bytes = p->codes_page_bytes;
  out->scales_page_bytes = p->scales_page_bytes;
  out->num_pages = p->num_pages;
  out->layers = p->layers;
  return SSW_OK;
}

int check_pages(const char* name, const ssw_kv_pages* t, int64_t n, const int32_t* seqs,
                const int32_t* other, bool two, ssw::kv::PagesArgs* a) {
  if (!t) return fail(SSW_ERR_INVALID_ARGUMENT, "%s: null page tables", name);
  if (t->page_size != 16 && t->page_size != 32 && t->page_size != 64 && t->page_size != 128)
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: page_size must be 16, 32, 64 or 128 (got %d)", name,
                t->page_size);
  if (t->num_pages < 1 || t->num_pages > (1 << 30) || t->max_seqs < 1 || t->columns < 1 ||
      t->table_stride < t->columns)
    return fail(SSW_ERR_INVALID_ARGUMENT,
                "%s: bad sizes num_pages=%d max_seqs=%d columns=%d stride=%lld", name, t->num_pages,
                t->max_seqs, t->columns, (long long)t->table_stride);
  if (n < 0 || n > t->max_seqs)
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: %lld sequences named, the table has %d", name,
                (long long)n, t->max_seqs);
  if (!t->refcount || !t->block_table || !t->seq_lens || (n > 0 && (!seqs || (two && !other))))
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
  if (!aligned(t->refcount, 4) || !aligned(t->block_table, 4) || !aligned(t->seq_lens, 4) ||
      !aligned(t->status, 4) || !aligned(seqs, 4) || !aligned(other, 4))
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: misaligned pointer", name);
  a->refcount = t->refcount;
  a->block_table = t->block_table;
  a->table_stride = t->table_stride;
  a->seq_lens = t->seq_lens;
  a->status = t->status;
  a->num_pages = t->num_pages;
  a->max_seqs = t->max_seqs;
  a->columns = t->columns;
  a->page_shift = 4;
  while ((1 << a->page_shift) < t->page_size) ++a->page_shift;
  a->seqs = seqs;
  a->other = other;
  a->n = (int32_t)n;
  return SSW_OK;
}

int check_workspace(const char* name, void* workspace, int64_t have, int64_t words) {
  if (!workspace || !aligned(workspace, 4) || have < words * 4)
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: the workspace must hold %lld bytes", name,
                (long long)(words * 4));
  return SSW_OK;
}

int64_t most_new_pages(int64_t n, int64_t tokens, int page_size) { return n + tokens / page_size; }

}  // namespace

int64_t ssw_kv_pages_workspace_bytes(int64_t n, int64_t total_tokens, int page_size,
                                     int64_t num_pages) {
  if (n < 0 || total_tokens < 0 || page_size < 1 || num_pages < 0) return -1;
  const int64_t pages = most_new_pages(n, total_tokens, page_size);
  return 4 * ssw::kv::pages_workspace_words(n, pages > num_pages ? pages : num_pages, num_pages);
}

int ssw_kv_pages_fork(const ssw_kv_pages* tables, const ssw_kv_pool* pool, int64_t n,
                      const int32_t* parents, const int32_t* children, void* workspace,
                      int64_t workspace_bytes, void* stream) {
  const char* name = "kv_pages_fork";
  ssw::set_last_error("");
  ssw::kv::PagesArgs a;
  ssw::kv::PoolArgs c;
  int st = check_pages(name, tables, n, parents, children, true, &a);
  if (st == SSW_OK) st = check_pool(name, pool, &c);
  if (st != SSW_OK) return st;
  if (pool->num_pages != tables->num_pages)
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: the pool has %lld pages, the tables %d", name,
                (long long)pool->num_pages, tables->num_pages);
  if (n == 0) return SSW_OK;
  st = check_workspace(name, workspace, workspace_bytes, ssw::kv::pages_workspace_words(n, n, 0));
  if (st != SSW_OK) return st;
  const int sms = device_sms();
  if (sms < 0) return fail(SSW_ERR_CUDA, "%s: no CUDA device", name);
  const cudaError_t e = ssw::kv::launch_fork(a, c, static_cast<int32_t*>(workspace), sms,
                                             static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? SSW_OK : cuda_fail(e, name);
}

int ssw_kv_pages_free(const ssw_kv_pages* tables, int64_t n, const int32_t* seqs, void* stream) {
  const char* name = "kv_pages_free";
  ssw::set_last_error("");
  ssw::kv::PagesArgs a;
  int st = check_pages(name, tables, n, seqs, nullptr, false, &a);
  if (st != SSW_OK || n == 0) return st;
  const cudaError_t e = ssw::kv::launch_free(a, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? SSW_OK : cuda_fail(e, name);
}

int ssw_kv_pages_extend(const ssw_kv_pages* tables, int64_t n, const int32_t* seqs,
                        const int32_t* new_tokens, int64_t total_tokens, int64_t* slot_mapping,
                        void* workspace, int64_t workspace_bytes, void* stream) {
  const char* name = "kv_pages_extend";
  ssw::set_last_error("");
  ssw::kv::PagesArgs a;
  int st = check_pages(name, tables, n, seqs, new_tokens, true, &a);
  if (st != SSW_OK) return st;
  if (total_tokens < 0 || total_tokens >= (1ll << 30) || (n == 0 && total_tokens > 0))
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: bad number of new tokens (%lld)", name,
                (long long)total_tokens);
  if (n == 0) return SSW_OK;
  if (total_tokens > 0 && (!slot_mapping || !aligned(slot_mapping, 8)))
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: null or misaligned slot_mapping", name);
  const int64_t most = most_new_pages(n, total_tokens, tables->page_size);
  st = check_workspace(name, workspace, workspace_bytes, ssw::kv::pages_workspace_words(n, most, 0));
  if (st != SSW_OK) return st;
  const cudaError_t e = ssw::kv::launch_extend(a, total_tokens, most, slot_mapping,
                                               static_cast<int32_t*>(workspace),
                                               static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? SSW_OK : cuda_fail(e, name);
}

int ssw_kv_pages_compact(const ssw_kv_pages* tables, const ssw_kv_pool* pool, void* workspace,
                         int64_t workspace_bytes, void* stream) {
  const char* name = "kv_pages_compact";
  ssw::set_last_error("");
  ssw::kv::PagesArgs a;
  ssw::kv::PoolArgs c;
  int st = check_pages(name, tables, 0, nullptr, nullptr, false, &a);
  if (st == SSW_OK) st = check_pool(name, pool, &c);
  if (st != SSW_OK) return st;
  if (pool->num_pages != tables->num_pages)
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: the pool has %lld pages, the tables %d", name,
                (long long)pool->num_pages, tables->num_pages);
  st = check_workspace(name, workspace, workspace_bytes,
                       ssw::kv::pages_workspace_words(0, tables->num_pages, tables->num_pages));
  if (st != SSW_OK) return st;
  const int sms = device_sms();
  if (sms < 0) return fail(SSW_ERR_CUDA, "%s: no CUDA device", name);
  const cudaError_t e = ssw::kv::launch_compact(a, c, static_cast<int32_t*>(workspace), sms,
                                                static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? SSW_OK : cuda_fail(e, name);
}

int ssw_kv_pages_copy(const ssw_kv_pool* pool, int64_t n, const int32_t* source,
                      const int32_t* target, void* stream) {
  const char* name = "kv_pages_copy";
  ssw::set_last_error("");
  ssw::kv::PoolArgs c;
  int st = check_pool(name, pool, &c);
  if (st != SSW_OK) return st;
  if (n < 0 || n > pool->num_pages)
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: bad size, %lld pairs of %lld pages", name,
                (long long)n, (long long)pool->num_pages);
  if (n == 0) return SSW_OK;
  if (!source || !target || !aligned(source, 4) || !aligned(target, 4))
    return fail(SSW_ERR_INVALID_ARGUMENT, "%s: null or misaligned page list", name);
  const int sms = device_sms();
  if (sms < 0) return fail(SSW_ERR_CUDA, "%s: no CUDA device", name);
  const cudaError_t e = ssw::kv::launch_copy(c, source, target, n, sms,
                                             static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? SSW_OK : cuda_fail(e, name);
}

}  // extern "C"
