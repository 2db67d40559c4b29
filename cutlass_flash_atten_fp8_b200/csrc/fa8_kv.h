// Internal interface between the C-ABI layer of the paged fp8 cache (fa8_kv_capi.cu) and its
// kernels.  Not installed; callers use include/fa8_kv_cache.h.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace fa8 {

// By-value description of the cache and of the tokens a call is about (struct fa8_kv_cache).
struct KvArgs {
  uint8_t* k;                     // [num_pages, heads, page_size, head_dim]
  uint8_t* v;
  float* k_descale;               // [num_pages, heads]
  float* v_descale;
  int num_pages;
  int heads;
  int page_shift;                 // log2(page_size)
  int head_dim;
  const int* table;               // [batch, table_width], rows table_stride apart
  int table_width;
  int table_stride;
  const int* seqlens;             // [batch]
  const int* cu;                  // [batch + 1] or null: `even` new tokens each
  int even;
  int batch;
  int tokens;
  int* status;                    // device word and mapped host word that an index out of range is reported into
  int* host_status;
};

// Code of an index out of range in the status words (codes of expired waits are others).
constexpr int kBadIndex = 0xbad1;

// Token-major tensors in and out: element strides.
struct KvRows {
  const void* x;
  int64_t token_stride;
  int64_t head_stride;
};

cudaError_t launch_kv_append(const KvArgs& a, const KvRows& k, const KvRows& v, bool bf16, bool e5m2, cudaStream_t stream);
cudaError_t launch_kv_read(const KvArgs& a, void* k_out, void* v_out, bool bf16, bool e5m2, cudaStream_t stream);

struct KvAttendArgs {
  KvArgs c;
  KvRows q;
  void* o;                        // [tokens, heads_q, head_dim]
  float* lse;                     // optional [tokens, heads_q]
  int heads_q;
  int group;                      // heads_q / heads
  int causal;
  float scale_log2;               // softmax_scale * log2(e)
};
cudaError_t launch_kv_attend(const KvAttendArgs& a, bool bf16, bool e5m2, cudaStream_t stream);

// fa8_capi.cu: the library's status words on the current device (null where there are none), a
// failure that an earlier launch left there (0 = none, an FA8_ERR code otherwise, words cleared), and
// the detail string of the calling thread.
void status_words(int** dev_word, int** host_word);
int earlier_failure(int32_t* caller_word, cudaStream_t stream);
void clear_error_detail();
void set_error_detail(const char* what, const char* msg);

}  // namespace fa8
