// awq_layer_capi.cu -- extern "C" entry points of the operators between a layer's products:
// rotary positions, the paged 4-bit key/value cache and attention over it (declared in
// include/awq_b200.h).  Validation only; the kernels are in awq_rope.cu, awq_kv4_cache.cu,
// awq_kv4_attn.cu and awq_kv4_prefill.cu.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "../../include/awq_b200.h"
#include "awq_internal.h"

namespace {

int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return awq::set_last_error(code, buf);
}
int fail_cuda(cudaError_t e, const char* what) {
  return fail(AWQ_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}
bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int check_shape(int64_t num_pages, int64_t kv_heads, int64_t head_dim, int64_t group_size,
                int64_t page_size, awq::Kv4Shape* c) {
  if (head_dim != 64 && head_dim != 128)
    return fail(AWQ_ERR_UNSUPPORTED, "head_dim=%lld must be 64 or 128", (long long)head_dim);
  if ((group_size != 32 && group_size != 64 && group_size != 128) || group_size > head_dim)
    return fail(AWQ_ERR_UNSUPPORTED, "group_size=%lld must be 32, 64 or 128 and at most head_dim=%lld",
                (long long)group_size, (long long)head_dim);
  if (page_size < 16 || page_size > 1024 || (page_size & (page_size - 1)))
    return fail(AWQ_ERR_UNSUPPORTED, "page_size=%lld must be a power of two from 16 to 1024",
                (long long)page_size);
  if (num_pages < 1 || num_pages > 0x7fffffffLL || kv_heads < 1 || kv_heads > 4096)
    return fail(AWQ_ERR_INVALID_ARG, "num_pages=%lld or kv_heads=%lld out of range",
                (long long)num_pages, (long long)kv_heads);
  c->num_pages = num_pages;
  c->heads = (int)kv_heads;
  c->dim = (int)head_dim;
  c->group = (int)group_size;
  c->page = (int)page_size;
  return AWQ_OK;
}

}  // namespace

extern "C" {

size_t awq_kv4_page_bytes(int64_t kv_heads, int64_t head_dim, int64_t group_size, int64_t page_size) {
  awq::Kv4Shape c;
  if (check_shape(1, kv_heads, head_dim, group_size, page_size, &c)) return 0;
  return (size_t)kv_heads * (page_size / 16) * (16 * head_dim + 128 * (head_dim / group_size));
}

int awq_kv4_append(const void* k, int64_t k_token_stride, int64_t k_head_stride, const void* v,
                   int64_t v_token_stride, int64_t v_head_stride, const int64_t* slots,
                   int64_t tokens, void* cache, int64_t num_pages, int64_t kv_heads,
                   int64_t head_dim, int64_t group_size, int64_t page_size, void* stream) {
  awq::Kv4Shape c;
  int rc = check_shape(num_pages, kv_heads, head_dim, group_size, page_size, &c);
  if (rc) return rc;
  if (tokens < 0 || tokens > (int64_t)1 << 31) return fail(AWQ_ERR_INVALID_ARG, "tokens=%lld out of range", (long long)tokens);
  if (tokens == 0) return AWQ_OK;
  if (!k || !v || !slots || !cache) return fail(AWQ_ERR_INVALID_ARG, "null k, v, slots or cache");
  if (!aligned(k, 2) || !aligned(v, 2) || !aligned(slots, 8) || !aligned(cache, 16))
    return fail(AWQ_ERR_INVALID_ARG, "k and v must be 2-byte, slots 8-byte and cache 16-byte aligned");
  int sms = 0, *status = nullptr;
  if ((rc = awq::device_context(&sms, &status))) return rc;
  const cudaError_t e = awq::launch_kv4_append(c, k, k_token_stride, k_head_stride, v, v_token_stride,
                                               v_head_stride, slots, tokens, cache, sms, status,
                                               static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail_cuda(e, "kv4 append launch");
  return AWQ_OK;
}

int awq_kv4_gather(const void* cache, int64_t num_pages, int64_t kv_heads, int64_t head_dim,
                   int64_t group_size, int64_t page_size, const int64_t* slots, int64_t tokens,
                   void* out_k, void* out_v, void* stream) {
  awq::Kv4Shape c;
  int rc = check_shape(num_pages, kv_heads, head_dim, group_size, page_size, &c);
  if (rc) return rc;
  if (tokens < 0 || tokens > (int64_t)1 << 31) return fail(AWQ_ERR_INVALID_ARG, "tokens=%lld out of range", (long long)tokens);
  if (tokens == 0) return AWQ_OK;
  if (!cache || !slots || !out_k || !out_v) return fail(AWQ_ERR_INVALID_ARG, "null cache, slots or output");
  if (!aligned(cache, 16) || !aligned(slots, 8) || !aligned(out_k, 16) || !aligned(out_v, 16))
    return fail(AWQ_ERR_INVALID_ARG, "cache, out_k and out_v must be 16-byte, slots 8-byte aligned");
  int sms = 0, *status = nullptr;
  if ((rc = awq::device_context(&sms, &status))) return rc;
  const cudaError_t e = awq::launch_kv4_gather(c, cache, slots, tokens, out_k, out_v, sms, status,
                                               static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail_cuda(e, "kv4 gather launch");
  return AWQ_OK;
}

int awq_kv4_pages_step(int32_t* block_table, int64_t table_stride, int64_t max_blocks, int32_t* held,
                       int32_t* free_pages, int64_t free_capacity, int32_t* free_count,
                       const int32_t* kv_lens, const int32_t* new_tokens, const uint8_t* reset,
                       int64_t requests, int64_t page_size, int64_t* slots, int32_t* positions,
                       int64_t max_tokens, int32_t* cu_q, int32_t* new_lens, int32_t* step_status,
                       void* stream) {
  if (requests < 0 || requests > awq::kKv4MaxRows)
    return fail(AWQ_ERR_UNSUPPORTED, "requests=%lld must be at most %d", (long long)requests, awq::kKv4MaxRows);
  if (max_blocks < 0 || max_blocks > (1 << 30) || table_stride < max_blocks || max_tokens < 0 ||
      max_tokens > (1 << 30) || free_capacity < 0 || free_capacity > (1 << 30) || page_size < 1 ||
      page_size > (1 << 20))
    return fail(AWQ_ERR_INVALID_ARG, "max_blocks, table_stride, max_tokens, free_capacity or page_size out of range");
  if (!free_count || !cu_q || !step_status ||
      (requests && (!block_table || !held || !kv_lens || !new_tokens || !new_lens)) ||
      (max_tokens && (!slots || !positions)) || (free_capacity && !free_pages))
    return fail(AWQ_ERR_INVALID_ARG, "null pointer");
  for (const void* p : {(const void*)block_table, (const void*)held, (const void*)free_pages,
                        (const void*)free_count, (const void*)kv_lens, (const void*)new_tokens,
                        (const void*)positions, (const void*)cu_q, (const void*)new_lens,
                        (const void*)step_status})
    if (!aligned(p, 4)) return fail(AWQ_ERR_INVALID_ARG, "an int32 pointer is not 4-byte aligned");
  if (!aligned(slots, 8)) return fail(AWQ_ERR_INVALID_ARG, "slots must be 8-byte aligned");
  awq::Kv4PagesCall c = {};
  c.table = block_table, c.table_rs = table_stride, c.held = held;
  c.free_pages = free_pages, c.free_count = free_count;
  c.lens = kv_lens, c.new_tokens = new_tokens, c.reset = reset;
  c.slots = slots, c.positions = positions, c.cu_q = cu_q, c.new_lens = new_lens;
  c.status = step_status, c.max_tokens = max_tokens;
  c.rows = (int)requests, c.width = (int)max_blocks, c.capacity = (int)free_capacity;
  c.page = (int)page_size;
  int sms = 0, *status = nullptr, rc;
  if ((rc = awq::device_context(&sms, &status))) return rc;
  const cudaError_t e = awq::launch_kv4_pages(c, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail_cuda(e, "kv4 pages launch");
  return AWQ_OK;
}

size_t awq_kv4_attention_workspace_bytes(int64_t head_dim, int64_t max_rows) {
  int sms = 0, *status = nullptr;
  if ((head_dim != 64 && head_dim != 128) || awq::device_context(&sms, &status)) return 0;
  return awq::kv4_attention_workspace((int)head_dim, max_rows, sms);
}

int awq_kv4_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, int64_t tokens,
                      int64_t q_heads, const void* cache, int64_t num_pages, int64_t kv_heads,
                      int64_t head_dim, int64_t group_size, int64_t page_size,
                      const int32_t* block_table, int64_t table_stride, int64_t max_blocks,
                      const int32_t* kv_lens, const int32_t* cu_q, int64_t requests, int64_t max_q,
                      float scale, void* out, int64_t out_token_stride, int64_t out_head_stride,
                      void* workspace, size_t workspace_bytes, void* stream) {
  awq::Kv4AttnCall a = {};
  int rc = check_shape(num_pages, kv_heads, head_dim, group_size, page_size, &a.cache);
  if (rc) return rc;
  if (requests < 0 || requests > awq::kKv4MaxRows)
    return fail(AWQ_ERR_UNSUPPORTED, "requests=%lld must be at most %d", (long long)requests, awq::kKv4MaxRows);
  if (tokens < 0 || tokens > (1 << 30) || max_blocks < 0 || max_blocks > (1 << 30) ||
      table_stride < max_blocks)
    return fail(AWQ_ERR_INVALID_ARG, "tokens, max_blocks or table_stride out of range");
  if (q_heads < 1 || q_heads % kv_heads)
    return fail(AWQ_ERR_INVALID_ARG, "q_heads=%lld is not a multiple of kv_heads=%lld", (long long)q_heads, (long long)kv_heads);
  if (max_q < 1) return fail(AWQ_ERR_INVALID_ARG, "max_q=%lld must be at least 1", (long long)max_q);
  if (!cu_q && (tokens != requests || max_q != 1))
    return fail(AWQ_ERR_INVALID_ARG, "without cu_q every request has one query token: tokens=%lld requests=%lld max_q=%lld",
                (long long)tokens, (long long)requests, (long long)max_q);
  if (!std::isfinite(scale)) return fail(AWQ_ERR_INVALID_ARG, "scale must be finite");
  if (requests == 0 || tokens == 0) return AWQ_OK;
  if (!q || !cache || !kv_lens || !out || (max_blocks && !block_table))
    return fail(AWQ_ERR_INVALID_ARG, "null q, cache, block_table, kv_lens or out");
  if (!aligned(q, 16) || q_token_stride % 8 || q_head_stride % 8)
    return fail(AWQ_ERR_INVALID_ARG, "q must be 16-byte aligned with strides that are multiples of 8 elements");
  if (!aligned(out, 8) || out_token_stride % 4 || out_head_stride % 4)
    return fail(AWQ_ERR_INVALID_ARG, "out must be 8-byte aligned with strides that are multiples of 4 elements");
  if (!aligned(cache, 16)) return fail(AWQ_ERR_INVALID_ARG, "cache must be 16-byte aligned");
  if (!aligned(block_table, 4) || !aligned(kv_lens, 4) || !aligned(cu_q, 4))
    return fail(AWQ_ERR_INVALID_ARG, "block_table, kv_lens and cu_q must be 4-byte aligned");
  // the list of (request, kv head, row tile, 32-token tile) is counted in 32 bits
  const double tiles = (double)max_blocks * (double)page_size / 32 + 1;
  const double rows = (double)tokens * (double)(q_heads / kv_heads) / 8 + (double)requests;
  if (tiles * rows * (double)kv_heads > 2147000000.0 || (double)max_blocks * page_size > 2147000000.0 ||
      tokens * (q_heads / kv_heads) > 2147000000)
    return fail(AWQ_ERR_UNSUPPORTED, "tokens x max_blocks x page_size is too large for one call");
  int sms = 0, *status = nullptr;
  if ((rc = awq::device_context(&sms, &status))) return rc;
  a.max_q = (int)(max_q < tokens ? max_q : tokens);
  const size_t need = awq::kv4_attention_workspace((int)head_dim, (int64_t)a.max_q * (q_heads / kv_heads), sms);
  if (!workspace || workspace_bytes < need)
    return fail(AWQ_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need, workspace_bytes);
  if (!aligned(workspace, 16)) return fail(AWQ_ERR_INVALID_ARG, "workspace must be 16-byte aligned");
  a.data = cache, a.q = q, a.q_ts = q_token_stride, a.q_hs = q_head_stride;
  a.out = out, a.o_ts = out_token_stride, a.o_hs = out_head_stride;
  a.table = block_table, a.table_rs = table_stride, a.lens = kv_lens, a.cu_q = cu_q;
  a.tokens = tokens, a.rows = (int)requests, a.width = (int)max_blocks, a.q_heads = (int)q_heads;
  a.scale = scale, a.workspace = workspace;
  const cudaError_t e = awq::launch_kv4_attention(a, sms, status, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail_cuda(e, "kv4 attention launch");
  return AWQ_OK;
}

int awq_rope_axes(const void* q, int64_t q_token_stride, int64_t q_head_stride, int64_t q_heads,
                  const void* k, int64_t k_token_stride, int64_t k_head_stride, int64_t k_heads,
                  int64_t tokens, int64_t head_dim, const void* positions, int positions_are_64bit,
                  int64_t axis_stride, const float* inv_freq, const int32_t* sections, int axes,
                  int interleaved, void* out_q, int64_t out_q_token_stride, int64_t out_q_head_stride,
                  void* out_k, int64_t out_k_token_stride, int64_t out_k_head_stride, void* stream) {
  if (axes < 1 || axes > awq::kRopeMaxAxes || !sections)
    return fail(AWQ_ERR_INVALID_ARG, "axes=%d must be 1 to %d, with a section each", axes, awq::kRopeMaxAxes);
  if (tokens < 0 || tokens > (1 << 30) || q_heads < 0 || k_heads < 0 || q_heads > 65536 || k_heads > 65536 ||
      head_dim < 2 || head_dim > 512)
    return fail(AWQ_ERR_INVALID_ARG, "tokens, heads or head_dim (at most 512) out of range");
  awq::RopeCall c = {};
  int64_t half = 0;
  for (int i = 0; i < axes; ++i) {
    if (sections[i] < 0 || sections[i] > 256) return fail(AWQ_ERR_INVALID_ARG, "section %d is %d", i, sections[i]);
    c.sections[i] = sections[i];
    half += sections[i];
  }
  if (half < 1 || 2 * half > head_dim)
    return fail(AWQ_ERR_INVALID_ARG, "the sections rotate 2 x %lld of %lld channels", (long long)half, (long long)head_dim);
  if (tokens == 0 || q_heads + k_heads == 0) return AWQ_OK;
  if (!positions || !inv_freq || (q_heads && (!q || !out_q)) || (k_heads && (!k || !out_k)))
    return fail(AWQ_ERR_INVALID_ARG, "null pointer");
  if (!aligned(q, 2) || !aligned(k, 2) || !aligned(out_q, 2) || !aligned(out_k, 2) || !aligned(inv_freq, 4) ||
      !aligned(positions, positions_are_64bit ? 8 : 4))
    return fail(AWQ_ERR_INVALID_ARG, "a pointer is not aligned to its element size");
  c.q = q, c.k = k, c.q_ts = q_token_stride, c.q_hs = q_head_stride, c.k_ts = k_token_stride, c.k_hs = k_head_stride;
  c.out_q = out_q, c.out_k = out_k, c.oq_ts = out_q_token_stride, c.oq_hs = out_q_head_stride;
  c.ok_ts = out_k_token_stride, c.ok_hs = out_k_head_stride;
  c.positions = positions, c.pos_is_64 = positions_are_64bit, c.pos_as = axis_stride, c.inv_freq = inv_freq;
  c.T = tokens, c.q_heads = (int)q_heads, c.k_heads = (int)k_heads, c.dim = (int)head_dim;
  c.half = (int)half, c.axes = axes, c.interleaved = interleaved;
  int sms = 0, *status = nullptr, rc;
  if ((rc = awq::device_context(&sms, &status))) return rc;
  const cudaError_t e = awq::launch_rope(c, sms, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail_cuda(e, "rope launch");
  return AWQ_OK;
}

}  // extern "C"
