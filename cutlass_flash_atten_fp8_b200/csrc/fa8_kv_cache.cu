// Writing new keys and values into the pages of the fp8 cache, and reading them back.
//
// A unit of work is what one sequence's new tokens touch of one page and head, of K or of V: at most
// page_size rows of head_dim.  Units own their page, head and scale, so the scale can be raised and
// the page's older tokens rounded anew by the unit alone, with no atomics.
//
//   a = max |x| of the new rows,  2^e = the smallest power of two with a <= MAX 2^e,
//   d = 2^e in a page that starts anew, max(d, 2^e) otherwise;  older x8 <- fp8(x8 d_old / d),  x8 = fp8(x / d)
//
// Bound by memory: two bytes in and one out per element (append; the reverse for read).  Measured: 16 prompts, 257 MB, 49 us, 5.3 TB/s,
// against 39 at the rate of a copy; read of 8 x 8192 tokens at head dim 64, 201 MB, 36 us against 31; a token of each of 128 sequences
// 3.4 us and of one 2.4, a launch's latency and a chain of loads (where the token is, its page, its old scale).
#include <cuda_runtime.h>

#include "fa8_kernel.h"
#include "fa8_kv.h"
#include "kv_common.cuh"

namespace fa8 {

namespace {

constexpr int kVec = 8;                 // elements of a vector: 16 bytes of half precision, 8 of fp8
constexpr int kHold = 8;                // vectors that a thread keeps in registers (1 where units have no more)
constexpr int kWarpWork = 32 * kHold * kVec;
constexpr int kMaxThreads = 512;
constexpr int kWarpsPerCta = 4;        // units of a CTA where a warp takes one

// Units past the last look at the sequences, a thread each: one that is out of range may have no unit that finds it.  (Asked by the
// units themselves the prompts of append took 50 to 53 us for 47.)
__device__ __forceinline__ void check_sequence(const KvArgs& a, int64_t b) {
  if (kv_bad(a, b, true)) report_bad_index(a);
}

// The part of a page that a unit is about.
struct Unit {
  int head;
  bool of_v;
  int page;                            // as the table has it; -1: nothing to do, or (read) zeros are due
  int off, rows;                       // slots off .. off + rows - 1; off -1: of a sequence that is out of range
  int row0;                            // first row of the token-major tensors
};

template <bool kRead>
__device__ __forceinline__ Unit find_unit(const KvArgs& a, int64_t u) {
  Unit r{};
  const int64_t slot = u / (2 * a.heads);
  const int i = static_cast<int>(u - slot * (2 * a.heads));
  r.of_v = i >= a.heads;
  r.head = r.of_v ? i - a.heads : i;
  r.page = -1;
  int b, j;
  kv_find_slot(a, slot, 1 << a.page_shift, 2, &b, &j);
  const KvSeq s = kv_seq(a, b);
  const int P = 1 << a.page_shift;
  if (s.bad || s.n > s.len) {
    const int64_t lo = static_cast<int64_t>(j) * P;
    if (kRead && lo < s.n) {
      r.off = -1;
      r.rows = min(P, s.n - static_cast<int>(lo));
      r.row0 = s.first + static_cast<int>(lo);
    }
    return r;
  }
  const int start = s.len - s.n;
  const int64_t pi = static_cast<int64_t>(start >> a.page_shift) + j;
  const int64_t lo = max(static_cast<int64_t>(start), pi * P), hi = min(static_cast<int64_t>(s.len), (pi + 1) * P);
  if (lo >= hi) return r;
  r.off = static_cast<int>(lo) & (P - 1);
  r.rows = static_cast<int>(hi - lo);
  r.row0 = s.first + static_cast<int>(lo - start);
  r.page = ld_int(a.table + static_cast<int64_t>(b) * a.table_stride + pi);      // looked at once the rows are on their way
  return r;
}

// Row of vector i where a row has `per_row` <= 32 vectors, i <= 4096: magic = 2^20 / per_row + 1.
__device__ __forceinline__ int row_of(int i, uint32_t magic) { return static_cast<int>((static_cast<uint32_t>(i) * magic) >> 20); }

// A page number from the table, -1 (reported) if it is out of range.
__device__ __forceinline__ int checked(const KvArgs& a, int page) {
  if (static_cast<unsigned>(page) < static_cast<unsigned>(a.num_pages)) return page;
  report_bad_index(a);
  return -1;
}

template <bool kE5M2>
__device__ __forceinline__ float scale_for(float amax) {
  // MAX = 1.75 * 2^8 (e4m3) or 1.75 * 2^15 (e5m2): the exponent follows from amax's own and whether
  // its significand is above 1.75
  const uint32_t bits = __float_as_uint(amax);
  int e = static_cast<int>(bits >> 23) - 127 - (kE5M2 ? 15 : 8) + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = min(max(e, -64), 64);
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

__device__ __forceinline__ uint32_t pair_max(uint32_t m, uint32_t w, bool bf16) {
  w &= 0x7fff7fffu;                                       // max drops NaN
  if (bf16) asm("max.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(w));
  else asm("max.f16x2 %0, %0, %1;" : "+r"(m) : "r"(w));
  return m;
}

template <bool kBf16>
__device__ __forceinline__ float abs_max(const uint4& x) {
  uint32_t m = 0;
  m = pair_max(m, x.x, kBf16);
  m = pair_max(m, x.y, kBf16);
  m = pair_max(m, x.z, kBf16);
  m = pair_max(m, x.w, kBf16);
  const float2 f = half_pair<kBf16>(m);
  float r = fmaxf(f.x, f.y);
  if (r == INFINITY) {                                    // infinities saturate and do not count
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    r = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = half_pair<kBf16>(w[i] & 0x7fff7fffu);
      if (p.x < INFINITY) r = fmaxf(r, p.x);
      if (p.y < INFINITY) r = fmaxf(r, p.y);
    }
  }
  return r;
}

template <bool kBf16, bool kE5M2>
__device__ __forceinline__ uint2 to_fp8x8(const uint4& x, float inv) {
  const float2 a = half_pair<kBf16>(x.x), b = half_pair<kBf16>(x.y), c = half_pair<kBf16>(x.z), d = half_pair<kBf16>(x.w);
  return make_uint2(fp8_pair<kE5M2>(a.x * inv, a.y * inv) | (fp8_pair<kE5M2>(b.x * inv, b.y * inv) << 16),
                    fp8_pair<kE5M2>(c.x * inv, c.y * inv) | (fp8_pair<kE5M2>(d.x * inv, d.y * inv) << 16));
}
// x / d to fp32's precision, for any d: 1 / d is taken as hi + lo, lo from the remainder 1 - d hi (0 for powers of two), and x hi with its rounding
// error; both are exact by a fused multiplication.
__device__ __forceinline__ float quotient(float x, float hi, float lo) {
  const float p = x * hi;
  return fabsf(p) < INFINITY ? p + fmaf(x, lo, fmaf(x, hi, -p)) : p;
}
template <bool kBf16, bool kE5M2>
__device__ __forceinline__ uint32_t divided_to_fp8x4(uint32_t x, uint32_t y, float hi, float lo) {
  const float2 a = half_pair<kBf16>(x), b = half_pair<kBf16>(y);
  return fp8_pair<kE5M2>(quotient(a.x, hi, lo), quotient(a.y, hi, lo)) | (fp8_pair<kE5M2>(quotient(b.x, hi, lo), quotient(b.y, hi, lo)) << 16);
}

// kWarp: a unit to a warp, several a CTA; otherwise a unit to a CTA, of which two of 512 threads are to fit an SM (64 registers; with the 76
// that the compiler would take, 16 x 2000 tokens at head dim 256 took 116 us for 80).
template <bool kBf16, bool kE5M2, bool kWarp, int kHold>
__global__ void __launch_bounds__(kWarp ? 32 * kWarpsPerCta : kMaxThreads, kWarp ? 0 : 2) kv_append_kernel(const KvArgs a, const KvRows kin, const KvRows vin,
                                                                                            int64_t units, uint32_t magic) {
  __shared__ float part[kMaxThreads / 32];
  start_after_predecessor();
  let_successor_start();
  const int tid = kWarp ? threadIdx.x & 31 : threadIdx.x, n_threads = kWarp ? 32 : blockDim.x;
  const int64_t u = kWarp ? static_cast<int64_t>(blockIdx.x) * kWarpsPerCta + (threadIdx.x >> 5) : blockIdx.x;
  if (u >= units) return check_sequence(a, (u - units) * n_threads + tid);
  const Unit w = find_unit<false>(a, u);
  if (w.rows == 0) return;                                // the same for all threads of the unit, as below
  const int D = a.head_dim, per_row = D / kVec, n = w.rows * per_row;
  const KvRows& in = w.of_v ? vin : kin;
  const uint16_t* x = static_cast<const uint16_t*>(in.x) + w.row0 * in.token_stride + w.head * in.head_stride;
  auto src = [&](int i) {
    const int r = row_of(i, magic);
    return reinterpret_cast<const uint4*>(x + r * in.token_stride + kVec * (i - r * per_row));
  };
  uint4 hold[kHold];
#pragma unroll
  for (int h = 0; h < kHold; ++h) {
    const int i = tid + h * n_threads;
    hold[h] = make_uint4(0u, 0u, 0u, 0u);
    if (i < n) hold[h] = ld_global(src(i));
  }
  const int page = checked(a, w.page);
  if (page < 0) return;
  const int64_t page_head = static_cast<int64_t>(page) * a.heads + w.head;
  uint8_t* const y = (w.of_v ? a.v : a.k) + (page_head << a.page_shift) * D;
  float* const descale = (w.of_v ? a.v_descale : a.k_descale) + page_head;
  const float old = w.off > 0 ? ld_global(descale) : 0.f;
  float amax = 0.f;
#pragma unroll
  for (int h = 0; h < kHold; ++h)
    amax = fmaxf(amax, abs_max<kBf16>(hold[h]));
  for (int i = tid + kHold * n_threads; i < n; i += n_threads) amax = fmaxf(amax, abs_max<kBf16>(ld_global(src(i))));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if (!kWarp) {
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = amax;
    __syncthreads();
    for (int i = 0; i < (blockDim.x >> 5); ++i) amax = fmaxf(amax, part[i]);
  }
  float d = scale_for<kE5M2>(amax);
  if (w.off > 0) {
    d = fmaxf(old, d);
    if (d > old) {
      const float f = old / d;
      uint4* const older = reinterpret_cast<uint4*>(y);
      for (int i = tid; i < w.off * (D / 16); i += n_threads) {
        const uint4 c = ld_global(older + i);
        const uint32_t in4[4] = {c.x, c.y, c.z, c.w};
        uint32_t out4[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t lo, hi;
          fp8_to_half4<kE5M2>(in4[k], lo, hi);
          const float2 p = half_pair<false>(lo), q = half_pair<false>(hi);
          out4[k] = fp8_pair<kE5M2>(p.x * f, p.y * f) | (fp8_pair<kE5M2>(q.x * f, q.y * f) << 16);
        }
        older[i] = make_uint4(out4[0], out4[1], out4[2], out4[3]);
      }
    }
  }
  if (tid == 0) *descale = d;                             // every thread has read the old one: the reduction lies between
  uint2* const dst = reinterpret_cast<uint2*>(y + w.off * D);
  // Scales of pages that were filled in another way need not be powers of two, and x (1 / d) rounds twice: such pages' rows are read again.
  const float inv = 1.f / d;
  const bool exact = (__float_as_uint(d) & 0x7fffffu) == 0u;
  const int n_held = exact ? n : 0;
#pragma unroll
  for (int h = 0; h < kHold; ++h) {
    const int i = tid + h * n_threads;
    if (i < n_held) dst[i] = to_fp8x8<kBf16, kE5M2>(hold[h], inv);
  }
  const float lo = exact ? 0.f : fmaf(-d, inv, 1.f) * inv;
  for (int i = tid + (exact ? kHold * n_threads : 0); i < n; i += n_threads) {
    const uint4 v = ld_global(src(i));
    dst[i] = make_uint2(divided_to_fp8x4<kBf16, kE5M2>(v.x, v.y, inv, lo), divided_to_fp8x4<kBf16, kE5M2>(v.z, v.w, inv, lo));
  }
}

template <bool kBf16, bool kE5M2, bool kWarp, int kHold>
__global__ void __launch_bounds__(kWarp ? 32 * kWarpsPerCta : kMaxThreads) kv_read_kernel(const KvArgs a, uint16_t* k_out, uint16_t* v_out,
                                                                                          int64_t units, uint32_t magic) {
  start_after_predecessor();
  let_successor_start();
  const int tid = kWarp ? threadIdx.x & 31 : threadIdx.x, n_threads = kWarp ? 32 : blockDim.x;
  const int64_t u = kWarp ? static_cast<int64_t>(blockIdx.x) * kWarpsPerCta + (threadIdx.x >> 5) : blockIdx.x;
  if (u >= units) return check_sequence(a, (u - units) * n_threads + tid);
  const Unit w = find_unit<true>(a, u);
  if (w.rows == 0) return;
  const int D = a.head_dim, per_row = D / kVec, n = w.rows * per_row;
  const int page = w.page == -1 && w.off < 0 ? -1 : checked(a, w.page);
  const int64_t page_head = static_cast<int64_t>(max(page, 0)) * a.heads + w.head;
  const uint8_t* x = (w.of_v ? a.v : a.k) + ((page_head << a.page_shift) + max(w.off, 0)) * D;
  const float d = page < 0 ? 0.f : ld_global((w.of_v ? a.v_descale : a.k_descale) + page_head);
  const int64_t row = static_cast<int64_t>(a.heads) * D;
  uint16_t* const y = (w.of_v ? v_out : k_out) + w.row0 * row + static_cast<int64_t>(w.head) * D;
  for (int i0 = tid; i0 < n; i0 += kHold * n_threads) {
    uint2 c[kHold];
#pragma unroll
    for (int h = 0; h < kHold; ++h) {
      const int i = i0 + h * n_threads;
      c[h] = i < n && page >= 0 ? ld_stream8(x + kVec * static_cast<int64_t>(i)) : make_uint2(0u, 0u);
    }
#pragma unroll
    for (int h = 0; h < kHold; ++h) {
      const int i = i0 + h * n_threads;
      if (i >= n) continue;
      const uint32_t in2[2] = {c[h].x, c[h].y};
      uint32_t out4[4];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint32_t lo, hi;
        fp8_to_half4<kE5M2>(in2[k], lo, hi);
        const float2 p = half_pair<false>(lo), q = half_pair<false>(hi);
        out4[2 * k] = pack_pair<kBf16>(p.x * d, p.y * d);
        out4[2 * k + 1] = pack_pair<kBf16>(q.x * d, q.y * d);
      }
      const int r = row_of(i, magic);
      st_global_v4(y + r * row + kVec * (i - r * per_row), out4[0], out4[1], out4[2], out4[3]);
    }
  }
}

// Threads of a unit: enough to hold what an average one has to move.
struct UnitPlan {
  int64_t units;
  int threads;                       // of a CTA; a warp's unit below that
  bool warp, one;                    // a unit to a warp; no more than a vector a thread
  uint32_t magic;
  cudaLaunchConfig_t cfg;
};
bool plan_units(const KvArgs& a, cudaStream_t stream, cudaLaunchAttribute* attr, UnitPlan* p) {
  p->units = kv_slots(a.batch, a.tokens, a.even, a.cu != nullptr, 1 << a.page_shift, 2) * 2 * a.heads;
  const int P = 1 << a.page_shift;
  const int mean = a.cu != nullptr ? (a.tokens + a.batch - 1) / a.batch : a.even;
  const int work = (mean < P ? mean : P) * a.head_dim;
  p->warp = work <= kWarpWork;
  p->one = work <= 32 * kVec;
  p->threads = p->warp ? 32 * kWarpsPerCta : (work / (kHold * kVec) + 31) / 32 * 32;
  if (p->threads > kMaxThreads) p->threads = kMaxThreads;
  p->magic = (1u << 20) / static_cast<uint32_t>(a.head_dim / kVec) + 1u;
  const int at_a_time = p->warp ? 32 : p->threads;
  const int64_t all = p->units + (a.batch + at_a_time - 1) / at_a_time;
  const int64_t ctas = p->warp ? (all + kWarpsPerCta - 1) / kWarpsPerCta : all;
  if (ctas > 0x7fffffff) return false;
  p->cfg = cudaLaunchConfig_t{};
  p->cfg.gridDim = dim3(static_cast<unsigned>(ctas), 1, 1);
  p->cfg.blockDim = dim3(static_cast<unsigned>(p->threads), 1, 1);
  p->cfg.stream = stream;
  attr[0] = overlap_attribute();
  p->cfg.attrs = attr;
  p->cfg.numAttrs = 1;
  return true;
}

template <bool kBf16, bool kE5M2>
cudaError_t append(const KvArgs& a, const KvRows& k, const KvRows& v, cudaStream_t stream) {
  cudaLaunchAttribute attr[1];
  UnitPlan p;
  if (!plan_units(a, stream, attr, &p)) return cudaErrorInvalidConfiguration;
  return cudaLaunchKernelEx(&p.cfg, p.one ? &kv_append_kernel<kBf16, kE5M2, true, 1>
                                         : (p.warp ? &kv_append_kernel<kBf16, kE5M2, true, kHold> : &kv_append_kernel<kBf16, kE5M2, false, kHold>), a, k, v,
                            p.units, p.magic);
}

template <bool kBf16, bool kE5M2>
cudaError_t read(const KvArgs& a, void* k_out, void* v_out, cudaStream_t stream) {
  cudaLaunchAttribute attr[1];
  UnitPlan p;
  if (!plan_units(a, stream, attr, &p)) return cudaErrorInvalidConfiguration;
  return cudaLaunchKernelEx(&p.cfg, p.warp ? &kv_read_kernel<kBf16, kE5M2, true, kHold> : &kv_read_kernel<kBf16, kE5M2, false, kHold>, a,
                            static_cast<uint16_t*>(k_out), static_cast<uint16_t*>(v_out), p.units, p.magic);
}

}  // namespace

cudaError_t launch_kv_append(const KvArgs& a, const KvRows& k, const KvRows& v, bool bf16, bool e5m2, cudaStream_t stream) {
  if (bf16) return e5m2 ? append<true, true>(a, k, v, stream) : append<true, false>(a, k, v, stream);
  return e5m2 ? append<false, true>(a, k, v, stream) : append<false, false>(a, k, v, stream);
}

cudaError_t launch_kv_read(const KvArgs& a, void* k_out, void* v_out, bool bf16, bool e5m2, cudaStream_t stream) {
  if (bf16) return e5m2 ? read<true, true>(a, k_out, v_out, stream) : read<true, false>(a, k_out, v_out, stream);
  return e5m2 ? read<false, true>(a, k_out, v_out, stream) : read<false, false>(a, k_out, v_out, stream);
}

}  // namespace fa8
