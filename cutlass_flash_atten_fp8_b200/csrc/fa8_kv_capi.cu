// C-ABI layer of the paged fp8 cache: argument validation and launch.  Declared in
// include/fa8_kv_cache.h.  No torch types, no exceptions, no exit().
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "fa8_kernel.h"
#include "fa8_kv.h"
#include "fa8_kv_cache.h"

namespace {

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

constexpr int64_t kMost = 0x7fffff00;     // positions of a sequence, rows
constexpr int32_t kMostHeads = 65536;

// Checks of a cache description, and the kernels' form of it.
int check_cache(const fa8_kv_cache* c, fa8::KvArgs* a) {
  if (!c || !c->k || !c->v || !c->k_descale || !c->v_descale || !c->page_table || !c->seqlens) return FA8_ERR_BAD_ARG;
  if (c->num_pages <= 0 || c->heads_kv <= 0 || c->batch <= 0 || c->table_width <= 0 || c->tokens < 0) return FA8_ERR_BAD_ARG;
  if (c->table_stride < c->table_width && c->batch > 1) return FA8_ERR_BAD_ARG;
  if (c->fp8_format != FA8_FP8_E4M3 && c->fp8_format != FA8_FP8_E5M2) return FA8_ERR_BAD_ARG;
  if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_descale, 4) || !aligned(c->v_descale, 4)) return FA8_ERR_BAD_ARG;
  if (!aligned(c->page_table, 4) || !aligned(c->seqlens, 4) || !aligned(c->cu_seqlens, 4) || !aligned(c->status_word, 4))
    return FA8_ERR_BAD_ARG;
  if (c->head_dim < 32 || c->head_dim > 256 || c->head_dim % 32 != 0) return FA8_ERR_UNSUPPORTED;
  int shift = 4;
  while (shift < 7 && (1 << shift) != c->page_size) ++shift;
  if ((1 << shift) != c->page_size) return FA8_ERR_UNSUPPORTED;
  // positions and rows are 32-bit numbers, also when rounded up to whole blocks
  if (static_cast<int64_t>(c->table_width) * c->page_size > kMost || c->tokens > kMost || c->heads_kv > kMostHeads) return FA8_ERR_UNSUPPORTED;
  if (static_cast<int64_t>(c->num_pages) * c->heads_kv > 0x7fffffff) return FA8_ERR_UNSUPPORTED;
  if (!c->cu_seqlens && c->tokens % c->batch != 0) return FA8_ERR_BAD_ARG;
  a->k = static_cast<uint8_t*>(c->k);
  a->v = static_cast<uint8_t*>(c->v);
  a->k_descale = c->k_descale;
  a->v_descale = c->v_descale;
  a->num_pages = c->num_pages;
  a->heads = c->heads_kv;
  a->page_shift = shift;
  a->head_dim = c->head_dim;
  a->table = c->page_table;
  a->table_width = c->table_width;
  a->table_stride = c->table_stride;
  a->seqlens = c->seqlens;
  a->cu = c->cu_seqlens;
  a->even = c->cu_seqlens ? 0 : c->tokens / c->batch;
  a->batch = c->batch;
  a->tokens = c->tokens;
  return FA8_OK;
}

// Rows of half-precision vectors that are loaded sixteen bytes at a time.
bool rows_ok(const void* x, int64_t token_stride, int64_t head_stride) {
  return x && aligned(x, 16) && token_stride >= 0 && head_stride >= 0 && token_stride % 8 == 0 && head_stride % 8 == 0;
}

// What an earlier launch left, then the words this one reports into.
int begin(const fa8_kv_cache* c, fa8::KvArgs* a, cudaStream_t stream) {
  if (const int rc = fa8::earlier_failure(c->status_word, stream)) return rc;
  int* word = nullptr;
  fa8::status_words(&word, &a->host_status);
  a->status = c->status_word ? c->status_word : word;
  return FA8_OK;
}

int64_t workspace_of(const fa8::KvAttendSizes& z, int sms) {
  return fa8::kv_prefill_takes(z) ? fa8::kv_prefill_workspace(z, sms) : fa8::kv_attend_workspace(z, sms);
}

int launched(cudaError_t e) {
  if (e == cudaSuccess) return FA8_OK;
  fa8::set_error_detail("kernel launch", cudaGetErrorString(e));
  return FA8_ERR_CUDA;
}

}  // namespace

extern "C" {

int fa8_kv_version(void) { return 100; }

int fa8_kv_append(const fa8_kv_cache* cache, const void* k, int64_t k_token_stride, int64_t k_head_stride, const void* v,
                  int64_t v_token_stride, int64_t v_head_stride, int32_t dtype, void* cuda_stream) {
  fa8::clear_error_detail();
  fa8::KvArgs a{};
  if (const int rc = check_cache(cache, &a)) return rc;
  if (dtype != FA8_DTYPE_FP16 && dtype != FA8_DTYPE_BF16) return FA8_ERR_BAD_ARG;
  if (a.tokens == 0) return FA8_OK;
  if (!rows_ok(k, k_token_stride, k_head_stride) || !rows_ok(v, v_token_stride, v_head_stride)) return FA8_ERR_BAD_ARG;
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  if (const int rc = begin(cache, &a, stream)) return rc;
  return launched(fa8::launch_kv_append(a, {k, k_token_stride, k_head_stride}, {v, v_token_stride, v_head_stride},
                                        dtype == FA8_DTYPE_BF16, cache->fp8_format == FA8_FP8_E5M2, stream));
}

int fa8_kv_read(const fa8_kv_cache* cache, void* k_out, void* v_out, int32_t dtype, void* cuda_stream) {
  fa8::clear_error_detail();
  fa8::KvArgs a{};
  if (const int rc = check_cache(cache, &a)) return rc;
  if (dtype != FA8_DTYPE_FP16 && dtype != FA8_DTYPE_BF16) return FA8_ERR_BAD_ARG;
  if (a.tokens == 0) return FA8_OK;
  if (!rows_ok(k_out, 0, 0) || !rows_ok(v_out, 0, 0)) return FA8_ERR_BAD_ARG;
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  if (const int rc = begin(cache, &a, stream)) return rc;
  return launched(fa8::launch_kv_read(a, k_out, v_out, dtype == FA8_DTYPE_BF16, cache->fp8_format == FA8_FP8_E5M2, stream));
}

int64_t fa8_kv_attention_workspace(int32_t batch, int32_t tokens, int32_t heads, int32_t heads_kv, int32_t head_dim,
                                   int32_t page_size, int32_t table_width, int32_t sm_count) {
  if (batch <= 0 || tokens < 0 || heads <= 0 || heads_kv <= 0 || heads % heads_kv != 0 || head_dim <= 0 || page_size <= 0 ||
      table_width <= 0 || sm_count <= 0)
    return FA8_ERR_BAD_ARG;
  if (head_dim > 256) return FA8_ERR_UNSUPPORTED;
  if (tokens == 0) return 0;
  // evenly divided or not: the larger of what either needs
  int64_t most = 0;
  for (const bool ragged : {false, true})
    most = std::max(most, workspace_of({batch, tokens, heads, heads_kv, head_dim, ragged, static_cast<int64_t>(table_width) * page_size}, sm_count));
  return most;
}

int fa8_kv_attention(const fa8_kv_attention_params* p, void* cuda_stream) {
  fa8::clear_error_detail();
  if (!p) return FA8_ERR_BAD_ARG;
  fa8::KvAttendArgs a{};
  if (const int rc = check_cache(&p->cache, &a.c)) return rc;
  if (p->dtype != FA8_DTYPE_FP16 && p->dtype != FA8_DTYPE_BF16) return FA8_ERR_BAD_ARG;
  if (p->heads <= 0 || p->heads % p->cache.heads_kv != 0) return FA8_ERR_BAD_ARG;
  if (!(p->softmax_scale > 0.f) || !std::isfinite(p->softmax_scale)) return FA8_ERR_BAD_ARG;
  if (!aligned(p->lse, 4)) return FA8_ERR_BAD_ARG;
  if (static_cast<int64_t>(a.c.tokens) * p->heads > kMost) return FA8_ERR_UNSUPPORTED;
  if (a.c.tokens == 0) return FA8_OK;
  if (!rows_ok(p->q, p->q_token_stride, p->q_head_stride) || !rows_ok(p->o, 0, 0)) return FA8_ERR_BAD_ARG;
  a.q = {p->q, p->q_token_stride, p->q_head_stride};
  a.o = p->o;
  a.lse = p->lse;
  a.heads_q = p->heads;
  a.group = p->heads / p->cache.heads_kv;
  a.causal = p->is_causal != 0;
  a.bf16 = p->dtype == FA8_DTYPE_BF16;
  a.scale_log2 = p->softmax_scale * 1.4426950408889634f;
  cudaError_t e = cudaSuccess;
  const int sms = fa8::current_sm_count(&e);
  if (sms <= 0) {
    fa8::set_error_detail("SM count", cudaGetErrorString(e));
    return FA8_ERR_CUDA;
  }
  const fa8::KvAttendSizes z{a.c.batch, a.c.tokens, a.heads_q, a.c.heads, a.c.head_dim, a.c.cu != nullptr,
                             static_cast<int64_t>(a.c.table_width) << a.c.page_shift};
  const int64_t need = workspace_of(z, sms);
  if (need > 0 && (!p->workspace || !aligned(p->workspace, 256) || p->workspace_bytes < need)) return FA8_ERR_BAD_ARG;
  // The pool's tensor maps depend on its address and shape, and on what the kernel copies at a time: a thread keeps those of its last call.
  struct Maps {
    const void *k, *v;
    int64_t slices;
    int32_t page_size, head_dim, keys;
    bool valid;
    CUtensorMap tk, tv;
  };
  thread_local Maps m{};
  const fa8_kv_cache& c = p->cache;
  const bool prefill = fa8::kv_prefill_takes(z);
  const int64_t slices = static_cast<int64_t>(c.num_pages) * c.heads_kv;
  const int32_t keys = std::min(c.page_size, prefill ? fa8::kv_prefill_copy_keys(c.head_dim <= 128 ? 128 : 256) : fa8::kv_attend_step_keys(z));
  if (!(m.valid && m.k == c.k && m.v == c.v && m.slices == slices && m.page_size == c.page_size && m.head_dim == c.head_dim && m.keys == keys)) {
    m.valid = false;
    const uint64_t row = static_cast<uint64_t>(fa8::kv_map_bytes(c.head_dim)), rows = static_cast<uint64_t>(c.page_size) * c.head_dim / row;
    const uint32_t inner = static_cast<uint32_t>(fa8::kv_box_bytes(c.head_dim)), box = static_cast<uint32_t>(keys * c.head_dim / row);
    if (!fa8::make_byte_map(&m.tk, c.k, row, rows, slices, inner, box)) return FA8_ERR_CUDA;
    if (!fa8::make_byte_map(&m.tv, c.v, row, rows, slices, inner, box)) return FA8_ERR_CUDA;
    m.k = c.k;
    m.v = c.v;
    m.slices = slices;
    m.page_size = c.page_size;
    m.head_dim = c.head_dim;
    m.keys = keys;
    m.valid = true;
  }
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  if (const int rc = begin(&p->cache, &a.c, stream)) return rc;
  const bool e5m2 = c.fp8_format == FA8_FP8_E5M2;
  return launched(prefill ? fa8::launch_kv_prefill(m.tk, m.tv, a, z, p->workspace, e5m2, sms, stream)
                          : fa8::launch_kv_attend(m.tk, m.tv, a, z, p->workspace, e5m2, sms, stream));
}

}  // extern "C"
