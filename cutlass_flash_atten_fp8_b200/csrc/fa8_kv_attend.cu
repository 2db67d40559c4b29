// Attention of new tokens' queries over the pages of the fp8 cache, sm_100a.
//
//   s_j = c (q . k8_j) dk[page of j],   O = sum_j 2^(s_j - m) v8_j dv[page of j] / sum_j 2^(s_j - m),   c = softmax_scale log2(e)
//
// The simplest form: a warp to a row (token and query head), a key at a time, the lanes side by side
// along head_dim, fp32 throughout.  It is bound by its own instructions (a shuffle reduction per key).
#include <cuda_runtime.h>

#include "fa8_kernel.h"
#include "fa8_kv.h"
#include "kv_common.cuh"

namespace fa8 {

namespace {

constexpr int kWarps = 4;

template <bool kBf16, bool kE5M2>
__global__ void __launch_bounds__(32 * kWarps) kv_attend_kernel(const KvAttendArgs a) {
  start_after_predecessor();
  let_successor_start();
  const int lane = threadIdx.x & 31;
  if (blockIdx.x == 0)                                    // a bad range has no rows that would find it
    for (int i = threadIdx.x; i < a.c.batch; i += blockDim.x)
      if (kv_seq(a.c, i).bad) report_bad_index(a.c);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int token = static_cast<int>(row / a.heads_q), head = static_cast<int>(row - static_cast<int64_t>(token) * a.heads_q);
  if (token >= a.c.tokens) return;
  // slots of one token each: the sequence whose range the token is in
  int b, j;
  if (a.c.cu == nullptr) {
    b = token / a.c.even;
  } else {
    b = -1;
    for (int i = lane; i < a.c.batch; i += 32)
      if (ld_int(a.c.cu + i) <= token && token < ld_int(a.c.cu + i + 1)) b = i;
    b = __reduce_max_sync(0xffffffffu, b);
    if (b < 0) return;
  }
  const KvSeq s = kv_seq(a.c, b);
  if (token < s.first || token >= s.first + s.n) return;
  const int i = token - s.first;
  const int seen = a.causal ? min(s.len, s.len - s.n + i + 1) : s.len;
  const int D = a.c.head_dim, per = D >> 5, h = head / a.group;
  float q[8], o[8];
  for (int e = 0; e < 8; ++e) q[e] = o[e] = 0.f;
  const uint16_t* qp = static_cast<const uint16_t*>(a.q.x) + token * a.q.token_stride + head * a.q.head_stride;
  for (int e = 0; e < per; ++e) q[e] = half_pair<kBf16>(ld_global(qp + lane + 32 * e)).x;
  float m = -INFINITY, l = 0.f, l_page = 0.f;             // row sum of the pages before, and of this one: short sums lose little
  int page = -1;
  float kd = 0.f, vd = 0.f;
  for (j = 0; j < seen; ++j) {
    if ((j & ((1 << a.c.page_shift) - 1)) == 0) {
      page = kv_page(a.c, b, j >> a.c.page_shift);
      l += l_page;
      l_page = 0.f;
      if (page >= 0) {
        kd = ld_global(a.c.k_descale + static_cast<int64_t>(page) * a.c.heads + h);
        vd = ld_global(a.c.v_descale + static_cast<int64_t>(page) * a.c.heads + h);
      }
    }
    if (page < 0) continue;
    const int64_t at = (((static_cast<int64_t>(page) * a.c.heads + h) << a.c.page_shift) + (j & ((1 << a.c.page_shift) - 1))) * D;
    auto fp8 = [&](const uint8_t* p) {
      uint32_t lo, hi;
      fp8_to_half4<kE5M2>(*reinterpret_cast<const volatile uint8_t*>(p), lo, hi);
      return half_pair<false>(lo).x;
    };
    float dot = 0.f;
    for (int e = 0; e < per; ++e) dot = fmaf(q[e], fp8(a.c.k + at + lane + 32 * e), dot);
    for (int w = 16; w > 0; w >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, w);
    const float x = dot * (a.scale_log2 * kd);
    const float mn = fmaxf(m, x);
    const float alpha = exp2f(m - mn), p = exp2f(x - mn);
    l *= alpha;
    l_page = l_page * alpha + p;
    for (int e = 0; e < per; ++e) o[e] = o[e] * alpha + p * vd * fp8(a.c.v + at + lane + 32 * e);
    m = mn;
  }
  l += l_page;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint16_t* op = static_cast<uint16_t*>(a.o) + row * D;
  for (int e = 0; e < per; ++e) op[lane + 32 * e] = static_cast<uint16_t>(pack_pair<kBf16>(o[e] * inv, 0.f));
  if (a.lse != nullptr && lane == 0) a.lse[row] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

}  // namespace

cudaError_t launch_kv_attend(const KvAttendArgs& a, bool bf16, bool e5m2, cudaStream_t stream) {
  cudaLaunchConfig_t cfg{};
  const int64_t ctas = (static_cast<int64_t>(a.c.tokens) * a.heads_q + kWarps - 1) / kWarps;
  if (ctas > 0x7fffffff) return cudaErrorInvalidConfiguration;
  cfg.gridDim = dim3(static_cast<unsigned>(ctas), 1, 1);
  cfg.blockDim = dim3(32 * kWarps, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1] = {overlap_attribute()};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  auto kernel = bf16 ? (e5m2 ? &kv_attend_kernel<true, true> : &kv_attend_kernel<true, false>)
                     : (e5m2 ? &kv_attend_kernel<false, true> : &kv_attend_kernel<false, false>);
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

}  // namespace fa8
