// Device code shared by the kernels of the paged fp8 cache: which tokens and pages a sequence has,
// with every number that comes from device memory checked, and fp8 conversions.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "fa8_kv.h"
#include "ptx_sm100.cuh"
#include "status_word.cuh"

namespace fa8 {

__device__ __forceinline__ int ld_int(const int* p) {
  int v;
  asm volatile("ld.global.s32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}

__device__ __forceinline__ void report_bad_index(const KvArgs& a) {
  if (a.status != nullptr) atomicCAS(a.status, 0, kBadIndex);
  if (a.host_status != nullptr && *reinterpret_cast<volatile int*>(a.host_status) == 0)
    *reinterpret_cast<volatile int*>(a.host_status) = kBadIndex;
}

// New tokens of sequence b: rows first .. first + n - 1 of the token-major tensors; len tokens in
// all.  A range or length that is out of range is `bad` and comes back as n = 0 (range) or len = 0.
struct KvSeq {
  int first, n, len;
  bool bad;
};
__device__ __forceinline__ KvSeq kv_seq(const KvArgs& a, int b) {
  KvSeq s;
  s.len = ld_int(a.seqlens + b);
  s.bad = false;
  if (a.cu != nullptr) {
    const int lo = ld_int(a.cu + b), hi = ld_int(a.cu + b + 1);
    s.first = lo;
    s.n = hi - lo;
    if (lo < 0 || hi < lo || hi > a.tokens) {
      s.bad = true;
      s.first = s.n = 0;
    }
  } else {
    s.first = b * a.even;
    s.n = a.even;
  }
  if (s.len < 0 || s.len > (static_cast<int64_t>(a.table_width) << a.page_shift)) {
    s.bad = true;
    s.len = 0;
  }
  return s;
}

// Sequence b is out of range (with_len: or has fewer tokens than it is to write or read).  Asked once for every sequence of a call: token
// ranges that decrease can hide a sequence from the search below.
__device__ __forceinline__ bool kv_bad(const KvArgs& a, int64_t b, bool with_len) {
  if (b >= a.batch) return false;
  const KvSeq s = kv_seq(a, static_cast<int>(b));
  return s.bad || (with_len && s.n > s.len);
}

// Work is dealt out in slots of a host-known number, a slot being one block of T tokens of one sequence at most.  Even
// batches have the same number for each.  Otherwise sequence b has the slots from cu[b] / T + extra * b on.  extra = 1 covers blocks counted
// from a sequence's first new token (ceil(n / T) <= floor(cu[b+1] / T) - floor(cu[b] / T) + 1), extra = 2 blocks at fixed places of
// the sequence, which the new tokens may enter and leave in the middle; T = 1 and extra = 0 finds a token's sequence.
__host__ __device__ inline int64_t kv_slots(int batch, int tokens, int even, bool ragged, int T, int extra) {
  if (ragged) return static_cast<int64_t>(tokens) / T + static_cast<int64_t>(extra) * batch;
  return batch * ((static_cast<int64_t>(even) + T - 1) / T + (extra - 1));
}

// Sequence of a slot and the slot's number within it, by the calling warp (all lanes alike).
// A search over 32 places at a time: two rounds of loads up to 1024 sequences.
__device__ __forceinline__ void kv_find_slot(const KvArgs& a, int64_t slot, int T, int extra, int* seq, int* j) {
  if (a.cu == nullptr) {
    const int per_seq = (a.even + T - 1) / T + (extra - 1);
    *seq = static_cast<int>(slot / per_seq);
    *j = static_cast<int>(slot - static_cast<int64_t>(*seq) * per_seq);
    return;
  }
  // largest b in [0, batch) whose first slot is not past `slot` (cu may hold anything: it is clamped,
  // and then checked by kv_seq)
  const int lane = threadIdx.x & 31;
  int lo = 0, n = a.batch;
  while (n > 1) {
    const int step = (n + 31) >> 5;
    const int at = lo + lane * step;
    bool before = false;
    if (at < lo + n) {
      const int t = min(max(ld_int(a.cu + at), 0), a.tokens);
      before = t / T + static_cast<int64_t>(extra) * at <= slot;
    }
    const int count = __popc(__ballot_sync(0xffffffffu, before));
    const int from = lo + max(count - 1, 0) * step;
    n = min(step, lo + n - from);
    lo = from;
  }
  const int t = min(max(ld_int(a.cu + lo), 0), a.tokens);
  *seq = lo;
  const int64_t d = slot - (t / T + static_cast<int64_t>(extra) * lo);
  *j = d < 0 ? 0x3fffffff : static_cast<int>(d < 0x3fffffff ? d : 0x3fffffff);
}

// Page p of sequence b (p < table_width), or -1 with a report.
__device__ __forceinline__ int kv_page(const KvArgs& a, int b, int p) {
  const int page = ld_int(a.table + static_cast<int64_t>(b) * a.table_stride + p);
  if (static_cast<unsigned>(page) < static_cast<unsigned>(a.num_pages)) return page;
  report_bad_index(a);
  return -1;
}

template <bool kBf16>
__device__ __forceinline__ float2 half_pair(uint32_t w) {
  if (kBf16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <bool kBf16>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
  uint32_t r;
  if (kBf16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Four fp8 -> two pairs of fp16, ascending (exact).
template <bool kE5M2>
__device__ __forceinline__ void fp8_to_half4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (kE5M2) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e5m2x2 %0, l;\n\tcvt.rn.f16x2.e5m2x2 %1, h;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
  } else {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
  }
}
// Two fp32 -> two fp8, to the nearest, saturating.
template <bool kE5M2>
__device__ __forceinline__ uint32_t fp8_pair(float lo, float hi) {
  uint16_t r;
  if (kE5M2) asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// From reference m to reference m_new >= m: what sums of P are multiplied by, and a sum of denominators l.  References follow the scales of
// V, which denominators know nothing of, so that the factor may be below fp32's range where l times it is not: l takes it in
// halves.  A reference of -inf (no keys, or scores that are all NaN) leaves nothing but NaNs.
__device__ __forceinline__ float to_reference(float m, float m_new, float& l) {
  const float half = m == -INFINITY ? 0.f : ex2_approx(0.5f * (m - m_new));
  l = l * half * half;
  return half * half;
}

// A product adds 0 * V for keys that a row's mask leaves out, and a NaN or an infinity there would become a NaN.  So where rows of a tile
// see different keys, they are taken out of V's tile before the product, and the rows that do see them get theirs afterwards, in what was
// stored for them (write_specials).  e4m3 has NaN 0x7f and no infinities, e5m2 NaN from 0x7d on and infinity 0x7c.
template <bool kE5M2>
__device__ __forceinline__ bool drop_specials(uint4& x) {
  // sign bits of the bytes that hold one
  auto of = [](uint32_t w) { return ((w & 0x7f7f7f7fu) + (kE5M2 ? 0x04040404u : 0x01010101u)) & 0x80808080u; };
  const uint32_t n[4] = {of(x.x), of(x.y), of(x.z), of(x.w)};
  if ((n[0] | n[1] | n[2] | n[3]) == 0u) return false;
  x.x &= ~((n[0] >> 7) * 0xffu);
  x.y &= ~((n[1] >> 7) * 0xffu);
  x.z &= ~((n[2] >> 7) * 0xffu);
  x.w &= ~((n[3] >> 7) * 0xffu);
  return true;
}
// Calls put(column, value) for the columns col, col + 32 ... below `end` in which a key from lo to hi - 1 of a sequence holds a NaN or an
// infinity: what they add up to.  Goes through the pool byte by byte, but only after one has been met.
template <bool kE5M2, typename Put>
__device__ __forceinline__ void write_specials(const KvArgs& a, int seq, int head, int lo, int hi, int col, int end, Put put) {
#pragma unroll 1
  for (; col < end; col += 32) {
    float sum = 0.f;
#pragma unroll 1
    for (int key = lo; key < hi; ++key) {
      const int page = ld_int(a.table + static_cast<int64_t>(seq) * a.table_stride + (key >> a.page_shift));
      if (static_cast<unsigned>(page) >= static_cast<unsigned>(a.num_pages)) continue;
      const int64_t row = ((static_cast<int64_t>(page) * a.heads + head) << a.page_shift) + (key & ((1 << a.page_shift) - 1));
      const int x = a.v[row * a.head_dim + col];
      if ((x & 0x7f) < (kE5M2 ? 0x7c : 0x7f)) continue;
      sum += kE5M2 && (x & 0x7f) == 0x7c ? (x & 0x80 ? -INFINITY : INFINITY) : NAN;
      if (sum != sum) break;
    }
    if (sum != 0.f) put(col, sum);
  }
}
// What was stored for a row and column, plus such a sum.  (Of the halves, infinities of either sign together are a NaN, all of whose bits are set.)
__device__ __forceinline__ uint16_t with_special(uint16_t old, float sum, bool bf16) {
  const int inf = bf16 ? 0x7f80 : 0x7c00, had = old & 0x7fff;
  const uint16_t sign = sum < 0.f ? 0x8000 : 0;
  if (sum != sum || had > inf || (had == inf && (old & 0x8000) != sign)) return 0x7fff;
  return static_cast<uint16_t>(sign | inf);
}

}  // namespace fa8
