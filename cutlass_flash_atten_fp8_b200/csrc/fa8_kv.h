// Internal interface between the C-ABI layer of the paged fp8 cache (fa8_kv_capi.cu) and its
// kernels.  Not installed; callers use include/fa8_kv_cache.h.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "fa8_kernel.h"

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

// Token-major tensors in and out: element strides.
struct KvRows {
  const void* x;
  int64_t token_stride;
  int64_t head_stride;
};

cudaError_t launch_kv_append(const KvArgs& a, const KvRows& k, const KvRows& v, bool bf16, bool e5m2, cudaStream_t stream);
cudaError_t launch_kv_read(const KvArgs& a, void* k_out, void* v_out, bool bf16, bool e5m2, cudaStream_t stream);

// Of an item that several CTAs share, written by the one that has its last part (first_cta -1: there is none).
struct alignas(32) KvRecord {
  int first_cta;
  int first;                      // the sequence's first new token
  int row0, n_rows, head;         // rows of the block; K/V head
};

struct KvAttendArgs {
  KvArgs c;
  KvRows q;
  void* o;                        // [tokens, heads_q, head_dim]
  float* lse;                     // optional [tokens, heads_q]
  int heads_q;
  int group;                      // heads_q / heads
  int causal;
  int bf16;                       // of q and o; fp16 otherwise
  float scale_log2;               // softmax_scale * log2(e)
  // Filled in by launch_kv_attend (see fa8_kv_attend.cu): CTAs of the cluster that has an item (0: shares of all steps), new tokens
  // of an item; in the workspace the rest.
  int n_split;
  int block_tokens;
  int unit_shift;                 // log2 of the steps that work is dealt out by
  struct KvRecord* records;       // one per CTA
  float* partial;
};
struct KvAttendSizes {
  int batch, tokens, heads_q, heads, head_dim;
  bool ragged;                    // cu_seqlens given
  int64_t keys_most;              // that a sequence can have: table_width * page_size
};
// tk, tv: the pools as 3-D byte tensors {kv_map_bytes, page_size * head_dim / kv_map_bytes, num_pages * heads} with a box of
// kv_box_bytes x min(page_size, the kernel's keys) x 1, swizzled over the box's row.
cudaError_t launch_kv_attend(const CUtensorMap& tk, const CUtensorMap& tv, KvAttendArgs a, const KvAttendSizes& z, void* workspace,
                             bool e5m2, int sms, cudaStream_t stream);
int64_t kv_attend_workspace(const KvAttendSizes& z, int sms);

// Many rows per sequence and K/V head (fa8_kv_prefill.cu).
struct KvPrefillPlan {
  int64_t items;                  // sequence, block of new tokens, K/V head, part
  int block_tokens;
  int parts;                      // that an item's keys are cut into
  float* partial_o;               // [parts, tokens, heads_q, head_dim]
  float* partial_ml;              // [parts, tokens, heads_q, 2]
};
KvPrefillPlan kv_prefill_plan(const KvAttendSizes& z, int sms);
int64_t kv_prefill_workspace(const KvAttendSizes& z, int sms);
cudaError_t launch_kv_prefill(const CUtensorMap& tk, const CUtensorMap& tv, const KvAttendArgs& a, const KvAttendSizes& z, void* workspace,
                              bool e5m2, int sms, cudaStream_t stream);
// Whether a call is one for launch_kv_prefill.
bool kv_prefill_takes(const KvAttendSizes& z);
// Bytes of a row of the pools' maps (rows of 64 bytes are taken two at a time) and of a box; keys of a box: those that a kernel copies at a
// time (a step of the kernel for few rows, 32 or, at head dims above 128, 16 in the other), or a page's.
#ifdef __CUDACC__
#define FA8_HD __host__ __device__
#else
#define FA8_HD
#endif
FA8_HD constexpr int kv_map_bytes(int head_dim) { return head_dim == 64 ? 128 : head_dim; }
FA8_HD constexpr int kv_box_bytes(int head_dim) { return head_dim < 64 ? 64 : 128; }
// Keys of a step of the kernel for few rows, built for head dims up to `width` and blocks of `rows` rows: what the registers hold.
FA8_HD constexpr int kv_step_keys(int width, int rows) { return width == 256 || (width == 128 && rows == 32) ? 16 : 32; }
FA8_HD constexpr int kv_prefill_copy_keys(int width) { return width == 256 ? 16 : 32; }
int kv_attend_step_keys(const KvAttendSizes& z);

// fa8_capi.cu: a 3-D byte tensor {inner, mid, outer} with a {box_inner, box_mid, 1} tile, swizzled over
// box_inner bytes (64 or 128).  False, with the detail string set, on failure.
bool make_byte_map(CUtensorMap* out, const void* base, uint64_t inner, uint64_t mid, uint64_t outer, uint32_t box_inner, uint32_t box_mid);

// fa8_capi.cu: the library's status words on the current device (null where there are none), a
// failure that an earlier launch left there (0 = none, an FA8_ERR code otherwise, words cleared), and
// the detail string of the calling thread.
void status_words(int** dev_word, int** host_word);
int earlier_failure(int32_t* caller_word, cudaStream_t stream);
void clear_error_detail();
void set_error_detail(const char* what, const char* msg);

}  // namespace fa8
