/*
 * fa8_kv_cache.h - C ABI of the paged fp8 key/value cache (libfa8_b200.so, sm_100a): writing it,
 * reading it back and attending over it.  Beside fa8_b200.h, whose conventions it follows: plain
 * pointers and sizes, a CUDA stream handle as void*, an int status as the return value; calls are
 * enqueued on the caller's stream, allocate nothing and do not synchronise.
 *
 * The reference has no counterpart: its one operator attends over contiguous K and V of one length
 * for the whole batch (include/attention_api.h:10-11), which cannot be kept up while tokens are
 * appended one at a time to sequences of different lengths.
 *
 * The cache.  Keys and values of all sequences live in a pool of pages of `page_size` tokens:
 *   k, v                  fp8 [num_pages, heads_kv, page_size, head_dim], contiguous
 *   k_descale, v_descale  fp32 [num_pages, heads_kv]: a scale for each block of page_size tokens and
 *                         head, x = descale * x8; 0 or from 2^-64 to 2^64 (as fa8_kv_append leaves
 *                         them; no powers of two are needed) where a token of the page is held
 * Sequence b has seqlens[b] tokens, those that the call is about included; its token p lies in slot
 * p % page_size of page page_table[b][p / page_size].  A call is about the last n_b tokens of each
 * sequence ("new" ones): rows cu_seqlens[b] .. cu_seqlens[b+1]-1 of the token-major tensors, or
 * tokens / batch rows each when cu_seqlens is NULL.  So the same three tensors describe the append
 * of new tokens and the attention of the same tokens' queries.  Table entries past a sequence's last
 * page are not looked at.  Rows of token-major tensors before cu_seqlens[0] and from
 * cu_seqlens[batch] on are neither read nor written.
 *
 * Numbers out of range - a page outside the pool, a length that is negative, above what a table row
 * can hold or below n_b (append, read), token ranges that decrease or leave the tensor - reach the
 * device only, so the kernels check them: such a page or sequence is left out (read: zeros;
 * attention: its keys do not count), nothing outside the tensors is touched, and FA8_ERR_BAD_INDEX
 * is reported the way expired waits are, by fa8_check_status and by the next call on the device, be it
 * of this header or fa8_fwd.  Calls that were enqueued before are computed.
 *
 * Limits (FA8_ERR_UNSUPPORTED past them): table_width * page_size, tokens and tokens * heads up to
 * 2^31 - 256, num_pages * heads_kv up to 2^31 - 1, 65536 heads_kv.
 */
#ifndef FA8_KV_CACHE_H_
#define FA8_KV_CACHE_H_

#include <stdint.h>

#include "fa8_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct fa8_kv_cache {
  void* k;                   /* 16-byte aligned, as v */
  void* v;
  float* k_descale;
  float* v_descale;
  int32_t num_pages;
  int32_t heads_kv;
  int32_t page_size;         /* 16, 32, 64 or 128 */
  int32_t head_dim;          /* a multiple of 32 up to 256 */
  int32_t fp8_format;        /* FA8_FP8_E4M3 or FA8_FP8_E5M2 */
  int32_t batch;
  const int32_t* page_table; /* [batch, table_width], rows table_stride entries apart */
  int32_t table_width;
  int32_t table_stride;
  const int32_t* seqlens;    /* [batch], new tokens included */
  const int32_t* cu_seqlens; /* [batch + 1] or NULL: tokens / batch new tokens each */
  int32_t tokens;            /* rows of the token-major tensors */
  int32_t* status_word;      /* as in fa8_fwd_params; NULL = the library's own */
} fa8_kv_cache;

/* Writes new keys and values into the pages.  k, v: fp16 or bf16 (FA8_DTYPE_*) [tokens, heads_kv,
 * head_dim], rows of head_dim contiguous elements, token and head strides in elements (multiples of
 * 8; bases 16-byte aligned), so both may be views of a fused projection's output.
 *
 * Per touched page and head, for K and V apart: a = max |x| over the page's new finite values and
 * e = the smallest exponent in [-64, 64] with a <= MAX * 2^e (a = 0: -64; above all of them: 64, and
 * what does not fit becomes +-MAX), MAX = 448 (e4m3) or 57344 (e5m2).  If the page's first slot is among the new tokens the page starts anew with descale
 * 2^e.  Otherwise its descale d becomes max(d, 2^e), and if that is larger the older tokens of the
 * page are rounded anew, x8 = fp8(x8 * d_old / d_new).  New tokens: x8 = fp8(x / d), to the nearest,
 * ties to even; infinities become +-MAX, NaN stays NaN.  Scales are powers of two: fp8 keeps its
 * relative precision whatever the scale, x / d is exact, and rounding anew changes only values that
 * become subnormal.
 * No two touched pages of a call may be the same page (sequences may share pages they only read). */
int fa8_kv_append(const fa8_kv_cache* cache, const void* k, int64_t k_token_stride, int64_t k_head_stride,
                  const void* v, int64_t v_token_stride, int64_t v_head_stride, int32_t dtype, void* cuda_stream);

/* Reads the last n_b tokens of every sequence back: k_out, v_out fp16 or bf16 [tokens, heads_kv,
 * head_dim], contiguous and 16-byte aligned, x8 * descale rounded once. */
int fa8_kv_read(const fa8_kv_cache* cache, void* k_out, void* v_out, int32_t dtype, void* cuda_stream);

typedef struct fa8_kv_attention_params {
  fa8_kv_cache cache;
  const void* q;           /* fp16 or bf16 [tokens, heads, head_dim], strides as for fa8_kv_append */
  int64_t q_token_stride;
  int64_t q_head_stride;
  void* o;                 /* the same type, contiguous [tokens, heads, head_dim], 16-byte aligned */
  float* lse;              /* optional [tokens, heads]: log(sum_j exp(s_j)); -inf for a row without keys */
  int32_t dtype;           /* FA8_DTYPE_FP16 or FA8_DTYPE_BF16, of q and o */
  int32_t heads;           /* a multiple of heads_kv; head h reads K/V head h / (heads / heads_kv) */
  int32_t is_causal;       /* 1: new token i of n_b sees the keys up to its own position seqlens[b] - n_b + i;
                              0: every key of its sequence.  A row that sees no key is zeros. */
  float softmax_scale;     /* > 0; s_j = softmax_scale * (q . k_j) */
  void* workspace;         /* fa8_kv_attention_workspace bytes, 256-byte aligned, this call's own until it
                              has run (graphs that run at once: one each); NULL where that is 0 */
  int64_t workspace_bytes;
} fa8_kv_attention_params;

/* Attention of the new tokens' queries over their sequences' pages.  What a row does not see does not
 * count, whatever is held there.  A NaN of V reaches the rows that see its key, in the columns that hold it; an infinity (e5m2; not
 * from fa8_kv_append) too, as an infinity or, where a row's probability of the key is too small for the products, as a NaN. */
int fa8_kv_attention(const fa8_kv_attention_params* params, void* cuda_stream);

/* Bytes of workspace for a call of these sizes on a device of `sm_count` SMs; host arithmetic only.
 * Negative: an error code. */
int64_t fa8_kv_attention_workspace(int32_t batch, int32_t tokens, int32_t heads, int32_t heads_kv, int32_t head_dim,
                                   int32_t page_size, int32_t table_width, int32_t sm_count);

/* ABI version of this header: major*100 + minor. */
int fa8_kv_version(void);

#ifdef __cplusplus
}
#endif
#endif /* FA8_KV_CACHE_H_ */
