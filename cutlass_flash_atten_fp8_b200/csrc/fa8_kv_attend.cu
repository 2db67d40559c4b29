// Attention of a few new tokens' queries over the pages of the fp8 cache (decoding), sm_100a.
//
//   x_j = c (q . k8_j) dk_j,   m >= x_j + log2 dv_j - 14,   O = sum_j 2^(x_j - m) dv_j v8_j / sum_j 2^(x_j - m)
//
// with c = softmax_scale log2(e) and dk_j, dv_j the scales of key j's page.  The reference m of a row is taken over x + log2 dv,
// so that what is rounded to fp16, P_j = 2^(x_j - m) dv_j, is at most 2^14 whatever the pages' scales; the sum of the
// denominators is of unrounded fp32 numbers.  m starts 6 below the first keys' maximum, so that P has its full precision twenty
// binades down, and is raised to 6 below the maximum so far, and what was summed rescaled, only when some P would pass 2^14.  Keys and queries enter the products exactly: every fp8 value is an
// fp16 value, and bf16 queries are brought into fp16's range by a power of two per row (what that cuts off is below
// 2^-39 of the row's largest).
//
// What bounds it: reading K and V once, 2 * head_dim bytes a key for all query rows that share it.
//   * The rows of a block are the query heads that share a K/V head times the new tokens: 8, 16 or 32 rows.
//   * Work is counted in steps of 32 keys of one sequence, K/V head and row block, and dealt out to the warps of one
//     CTA per SM in equal, contiguous shares whatever the lengths of the sequences are.  A share is worked out from the
//     lengths on the device, so a captured call can be replayed with other lengths.
//   * A warp streams its steps through a ring of its own in shared memory: one lane issues tiled copies (swizzled, so
//     that both operands are read without bank conflicts), page numbers being loaded a step and scales a ring ahead.
//     No warp waits for another.
//   * What a warp computed of an item that others share goes to the workspace, and kv_combine_kernel puts such items
//     together, always in the same order.  How steps are dealt out depends on all lengths of the call, hence so do
//     the last bits.
//
// Operand layouts are those of fa8_decode_sm100.cu: S = Q K^T with the query rows as M (16, eight of them padding
// when there are eight) and eight keys as N, the k index permuted alike in both operands; O^T = V^T P^T with 16 output
// columns as M, the rows as N and 16 keys as k.  tcgen05 would want 128 rows.
#include <cuda_runtime.h>

#include <atomic>

#include "fa8_kernel.h"
#include "fa8_kv.h"
#include "kv_common.cuh"

namespace fa8 {

namespace {

constexpr int kStepKeys = 32;
constexpr float kHeadroom = 6.f, kRaiseBy = 14.f;       // log2 of the largest P under a fresh reference, and at all
constexpr float kLog2Least = -100.f;                   // log2 of the smallest scale of V that the reference m follows
constexpr unsigned long long kLimitNs = 2000000000ull; // bound of every wait

// Head dims up to W run in the instance built for W (the copies fill what is missing with zeros); RB blocks of eight rows.
template <int W, int RB>
struct ACfg {
  static constexpr int kRowBytes = W < 128 ? W : 128;            // of a swizzled tile
  static constexpr int kBlocks = W / kRowBytes;                  // tiles side by side
  static constexpr int kTile = kStepKeys * kRowBytes;
  static constexpr int kStageBytes = 2 * kBlocks * kTile;        // K, then V
  static constexpr int kWarps = W == 256 ? 4 : 8;                // of the one CTA per SM
  static constexpr int kStages = W == 64 ? 6 : 3;                // of each: 192 KB in all
  static constexpr int kChunks = W / 64;                         // 16-byte pieces of a K row per thread
  static constexpr int kSteps = W / 16;                          // k-steps of Q K^T
  static constexpr int kVWords = W == 64 ? 2 : 4;
  static constexpr int kTilesPerBlock = 2 * kVWords;
  static constexpr int kMTiles = W / 16;
  static constexpr int kRows = 8 * RB;
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 ld_shared16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint2 ld_shared8(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}

constexpr int kExpiredWait = 0xa77e;                   // code in the status words

// By the whole warp: waits for the phase with the given parity, at most kLimitNs; whether it came, for all lanes alike.
__device__ __forceinline__ bool wait_copies(uint32_t bar, uint32_t parity) {
  bool here = mbar_try_wait(bar, parity);
  if (!here) {
    const uint64_t t0 = global_timer_ns();
    while (!(here = mbar_try_wait(bar, parity)) && global_timer_ns() - t0 < kLimitNs) {}
  }
  return __all_sync(0xffffffffu, here);
}

// Steps of an item of sequence s, and its row blocks.  An item without keys has a step that finds none: its rows are zeros.
__device__ __forceinline__ int item_steps(const KvSeq& s) { return max(1, (s.len + kStepKeys - 1) / kStepKeys); }
__device__ __forceinline__ int64_t row_blocks(const KvSeq& s, int group, int rows) {
  return (static_cast<int64_t>(s.n) * group + rows - 1) / rows;
}

// Share w of `total` steps among `workers`: [total * w / workers, total * (w + 1) / workers).
__device__ __forceinline__ int64_t share_start(int64_t total, int64_t workers, int64_t w) { return total * w / workers; }
__device__ __forceinline__ int64_t share_of(int64_t total, int64_t workers, int64_t x) {
  return ((x + 1) * workers + total - 1) / total - 1;
}
__device__ __forceinline__ int64_t workers_of(int64_t total, int64_t workers) { return total < workers ? total : workers; }

// All threads of the CTA: the steps of the call, and in s_scan[8 + i] those of the sequences before the i-th thread's part of
// the batch.  `bases` (one CTA only): the first step of every sequence, and the total.
__device__ __forceinline__ void scan_sequences(const KvAttendArgs& a, int rows, int64_t* s_scan, int64_t* bases, int64_t* total) {
  const int t = threadIdx.x, n = blockDim.x;
  const int per = (a.c.batch + n - 1) / n;
  const int b0 = min(t * per, a.c.batch), b1 = min(b0 + per, a.c.batch);
  int64_t sum = 0;
  for (int b = b0; b < b1; ++b) {
    const KvSeq s = kv_seq(a.c, b);
    if (s.bad && blockIdx.x == 0) report_bad_index(a.c);
    sum += row_blocks(s, a.group, rows) * a.c.heads * item_steps(s);
  }
  int64_t x = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
    if ((t & 31) >= o) x += y;
  }
  if ((t & 31) == 31) s_scan[t >> 5] = x;
  __syncthreads();
  int64_t before = 0, all = 0;
  for (int w = 0; w < (n >> 5); ++w) {
    if (w < (t >> 5)) before += s_scan[w];
    all += s_scan[w];
  }
  before += x - sum;
  s_scan[8 + t] = before;
  *total = all;
  if (bases != nullptr) {
    for (int b = b0; b < b1; ++b) {
      bases[b] = before;
      const KvSeq s = kv_seq(a.c, b);
      before += row_blocks(s, a.group, rows) * a.c.heads * item_steps(s);
    }
    if (t == 0) bases[a.c.batch] = all;
  }
  __syncthreads();
}

template <int W, int RB, bool kE5M2>
__global__ void __launch_bounds__(32 * ACfg<W, RB>::kWarps, 1) kv_attend_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                                                                   const KvAttendArgs a) {
  using C = ACfg<W, RB>;
  constexpr int kWarps = C::kWarps;
  extern __shared__ uint8_t smem_raw[];
  __shared__ int64_t s_scan[8 + 32 * kWarps];
  __shared__ __align__(8) uint64_t s_bar[kWarps * C::kStages];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t ring = ((smem_u32(smem_raw) + 1023u) & ~1023u) + warp * C::kStages * C::kStageBytes;
  const uint32_t bars = smem_u32(s_bar) + 8u * warp * C::kStages;
  if (lane == 0) {
    for (int i = 0; i < C::kStages; ++i) mbar_init(bars + 8 * i, 1);
    fence_mbar_init();
    fence_proxy_async_smem();
    if (warp == 0) {
      prefetch_tensormap(&tk);
      prefetch_tensormap(&tv);
    }
  }
  start_after_predecessor();
  let_successor_start();
  int64_t total;
  scan_sequences(a, C::kRows, s_scan, blockIdx.x == 0 ? a.bases : nullptr, &total);
  const int64_t workers = workers_of(total, static_cast<int64_t>(gridDim.x) * kWarps);
  const int64_t me = static_cast<int64_t>(warp) * gridDim.x + blockIdx.x;         // neighbours on different SMs
  if (me >= workers) return;
  int64_t pos = share_start(total, workers, me);
  const int64_t end = share_start(total, workers, me + 1);

  // The sequence that pos is in: the last thread's part whose exclusive sum is not past it, then by steps of one.
  int seq, per = (a.c.batch + 32 * kWarps - 1) / (32 * kWarps);
  int64_t at;                                            // first step of `seq`
  {
    int part = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      const int64_t v = s_scan[8 + 32 * i + lane];
      part += __popc(__ballot_sync(0xffffffffu, v <= pos));
    }
    at = s_scan[8 + part - 1];
    seq = (part - 1) * per;
  }

  const int P = 1 << a.c.page_shift;
  const int boxes = P < kStepKeys ? 2 : 1;               // copies per step and tile
  int stage = 0;
  uint32_t phase = 0;

  KvSeq s = kv_seq(a.c, seq);
  int steps = item_steps(s);
  int64_t items = row_blocks(s, a.group, C::kRows) * a.c.heads;
  while (pos < end) {
    while (pos >= at + items * steps) {                  // the next sequence that has items
      at += items * steps;
      s = kv_seq(a.c, ++seq);
      steps = item_steps(s);
      items = row_blocks(s, a.group, C::kRows) * a.c.heads;
    }
    const int64_t item = (pos - at) / steps;
    const int64_t item_at = at + item * steps;
    const int step0 = static_cast<int>(pos - item_at);
    const int step1 = static_cast<int>(min(static_cast<int64_t>(steps), end - item_at));
    const int rb = static_cast<int>(item / a.c.heads), h = static_cast<int>(item - static_cast<int64_t>(rb) * a.c.heads);
    const int row0 = rb * C::kRows, n_rows = min(C::kRows, s.n * a.group - row0);
    // keys that the block's last row sees; of the others, seen(row)
    auto seen = [&](int row) { return a.causal ? max(0, min(s.len, s.len - s.n + row / a.group + 1)) : s.len; };
    const int vis = seen(row0 + n_rows - 1);
    const int least = seen(row0);
    const int last = min(step1, (vis + kStepKeys - 1) / kStepKeys);     // steps past it see nothing

    // ---- filling the ring ----
    // Page of key `key` (of the two halves of a step, by lane & 1): loaded ahead, checked when it is used.
    const int* const table = a.c.table + static_cast<int64_t>(seq) * a.c.table_stride;
    auto load_page = [&](int step) {
      const int key = step * kStepKeys + (lane & 1) * 16;
      return step < last && key < vis ? ld_int(table + (key >> a.c.page_shift)) : -2;
    };
    // Copies of `step` into `st`; returns this lane's scale: of K (lanes 0, 1 mod 4) or V, of its half.
    auto fill = [&](int step, int page, int st) {
      const bool ok = static_cast<unsigned>(page) < static_cast<unsigned>(a.c.num_pages);
      if (!ok && page != -2) report_bad_index(a.c);
      float d = 0.f;
      if (ok) d = ld_global(((lane & 2) ? a.c.v_descale : a.c.k_descale) + static_cast<int64_t>(page) * a.c.heads + h);
      else d = -1.f;                                      // no such keys
      const int p1 = __shfl_sync(0xffffffffu, ok ? page : -1, 1);
      const int p0 = __shfl_sync(0xffffffffu, ok ? page : -1, 0);
      if (lane == 0) {
        const uint32_t bar = bars + 8 * st, dst = ring + st * C::kStageBytes;
        const int in_page = (step * kStepKeys) & (P - 1);
        const int loads = (p0 >= 0) + (boxes == 2 && p1 >= 0);
        constexpr uint32_t kBoxRow = 2 * C::kBlocks * C::kRowBytes;
        mbar_arrive_expect_tx(bar, loads * kBoxRow * (boxes == 2 ? 16 : kStepKeys));
        for (int i = 0; i < boxes; ++i) {
          const int p = i == 0 ? p0 : p1;
          if (p < 0) continue;
          const int slice = p * a.c.heads + h, row = i == 0 ? in_page : 0;
#pragma unroll
          for (int c = 0; c < C::kBlocks; ++c) {
            tma_load_3d(dst + c * C::kTile + i * 16 * C::kRowBytes, &tk, bar, c * 128, row, slice);
            tma_load_3d(dst + (C::kBlocks + c) * C::kTile + i * 16 * C::kRowBytes, &tv, bar, c * 128, row, slice);
          }
        }
      }
      return d;
    };
    float scales[C::kStages];
    int page_next = load_page(step0);
    {
      int st = stage;
#pragma unroll
      for (int i = 0; i < C::kStages; ++i) {
        scales[i] = -1.f;
        if (step0 + i < last) {
          const int page = page_next;
          page_next = load_page(step0 + i + 1);
          scales[i] = fill(step0 + i, page, st);
        }
        if (++st == C::kStages) st = 0;
      }
    }

    // ---- the rows of Q as A operands ----
    // Thread (g, t) takes columns 16 kChunks t ... of a block of 128 (64): the bytes of K that it reads below.
    uint32_t qa[C::kSteps][RB][2];
    float c_row[RB], m_row[RB], nm[RB], l_row[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      const int r = row0 + 8 * b + g;
      const bool in = 8 * b + g < n_rows;
      const int token = s.first + (in ? r / a.group : 0), head = h * a.group + (in ? r % a.group : 0);
      const uint16_t* p = static_cast<const uint16_t*>(a.q.x) + token * a.q.token_stride + head * a.q.head_stride;
      uint4 x[C::kChunks][2];
#pragma unroll
      for (int c = 0; c < C::kChunks; ++c) {
        constexpr int kPer = C::kChunks < 2 ? C::kChunks : 2;            // chunks of a block
        const int col = 128 * (c / 2) + 16 * (kPer * t + c % 2);
        const bool read = in && col < a.c.head_dim;
        x[c][0] = read ? ld_global(reinterpret_cast<const uint4*>(p + col)) : make_uint4(0u, 0u, 0u, 0u);
        x[c][1] = read ? ld_global(reinterpret_cast<const uint4*>(p + col + 8)) : make_uint4(0u, 0u, 0u, 0u);
      }
      float back = 1.f;
      if (a.bf16) {
        // into fp16: times the power of two that brings the row's largest to 2^14 ... 2^15
        float big = 0.f;
#pragma unroll
        for (int c = 0; c < C::kChunks; ++c)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t w[4] = {x[c][i].x, x[c][i].y, x[c][i].z, x[c][i].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 f = half_pair<true>(w[e] & 0x7fff7fffu);
              big = fmaxf(big, fmaxf(f.x, f.y));
            }
          }
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
        // 2^e <= big: times 2^(14 - e); kept where both it and its inverse are normal numbers
        const int e = min(max(static_cast<int>(__float_as_uint(big) >> 23) - 127, -100), 126);
        const float f = __uint_as_float(static_cast<uint32_t>(14 - e + 127) << 23);
        back = __uint_as_float(static_cast<uint32_t>(e - 14 + 127) << 23);
#pragma unroll
        for (int c = 0; c < C::kChunks; ++c)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t w[4] = {x[c][i].x, x[c][i].y, x[c][i].z, x[c][i].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float2 v = half_pair<true>(w[k]);
              w[k] = pack_half2(v.x * f, v.y * f);
            }
            x[c][i] = make_uint4(w[0], w[1], w[2], w[3]);
          }
      }
#pragma unroll
      for (int c = 0; c < C::kChunks; ++c) {
        qa[4 * c][b][0] = x[c][0].x; qa[4 * c][b][1] = x[c][0].y;
        qa[4 * c + 1][b][0] = x[c][0].z; qa[4 * c + 1][b][1] = x[c][0].w;
        qa[4 * c + 2][b][0] = x[c][1].x; qa[4 * c + 2][b][1] = x[c][1].y;
        qa[4 * c + 3][b][0] = x[c][1].z; qa[4 * c + 3][b][1] = x[c][1].w;
      }
      c_row[b] = a.scale_log2 * back;
      m_row[b] = -INFINITY;
      nm[b] = 0.f;
      l_row[b] = 0.f;
    }

    float o[C::kMTiles][RB][4];
#pragma unroll
    for (int j = 0; j < C::kMTiles; ++j)
#pragma unroll
      for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][b][e] = 0.f;

    // ---- the steps ----
    for (int step = step0; step < last; ++step) {
      const int page = page_next;
      page_next = load_page(step + C::kStages + 1);
      const float mine = scales[0];
      float kd[2], vd[2];
      kd[0] = __shfl_sync(0xffffffffu, mine, 0); kd[1] = __shfl_sync(0xffffffffu, mine, 1);
      vd[0] = __shfl_sync(0xffffffffu, mine, 2); vd[1] = __shfl_sync(0xffffffffu, mine, 3);
#pragma unroll
      for (int i = 0; i + 1 < C::kStages; ++i) scales[i] = scales[i + 1];
      scales[C::kStages - 1] = -1.f;
      if (!wait_copies(bars + 8 * stage, phase)) {
        // Give up: report, wait (with a limit each) for the copies in flight, which write to this CTA's memory.
        if (lane == 0) {
          if (a.c.status != nullptr) atomicCAS(a.c.status, 0, kExpiredWait);
          if (a.c.host_status != nullptr) *reinterpret_cast<volatile int*>(a.c.host_status) = kExpiredWait;
        }
        for (int i = step; i < min(step + C::kStages, last); ++i) {
          wait_copies(bars + 8 * stage, phase);
          if (++stage == C::kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        return;
      }
      const uint32_t sk = ring + stage * C::kStageBytes, sv = sk + C::kBlocks * C::kTile;
      // a step that holds keys past some row's last, or of a page that is out of range
      const int key0 = step * kStepKeys;
      const bool whole = key0 + kStepKeys <= least && kd[0] != -1.f && kd[1] != -1.f;

      float x[4][RB][2];                                  // score tile, row block, its two keys: x_j
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        constexpr int kPairs = (RB + 1) / 2;
        float sc[kPairs][4];
#pragma unroll
        for (int b = 0; b < kPairs; ++b) sc[b][0] = sc[b][1] = sc[b][2] = sc[b][3] = 0.f;
        const int row = 8 * j + g;
#pragma unroll
        for (int c = 0; c < C::kChunks; ++c) {
          uint32_t at_row;
          if constexpr (W == 64) at_row = sk + row * 64 + ((t ^ ((row >> 1) & 3)) << 4);
          else at_row = sk + (c / 2) * C::kTile + row * 128 + (((2 * t + c % 2) ^ (row & 7)) << 4);
          const uint4 kr = ld_shared16(at_row);
          const uint32_t w[4] = {kr.x, kr.y, kr.z, kr.w};
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            uint32_t b0, b1;
            fp8_to_half4<kE5M2>(w[u], b0, b1);
            const auto& qw = qa[4 * c + u];
#pragma unroll
            for (int b = 0; b < kPairs; ++b)
              mma_f16(sc[b], qw[2 * b][0], RB > 1 ? qw[RB > 1 ? 2 * b + 1 : 0][0] : 0u, qw[2 * b][1], RB > 1 ? qw[RB > 1 ? 2 * b + 1 : 0][1] : 0u, b0, b1);
          }
        }
#pragma unroll
        for (int b = 0; b < RB; ++b) {
          const float c = c_row[b] * kd[j >> 1];
          x[j][b][0] = sc[b / 2][2 * (b & 1)] * c;
          x[j][b][1] = sc[b / 2][2 * (b & 1) + 1] * c;
        }
      }
      if (!whole) {
#pragma unroll
        for (int b = 0; b < RB; ++b) {
          const int lim = seen(row0 + min(8 * b + g, n_rows - 1));
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (key0 + 8 * j + 2 * t + e >= lim || kd[j >> 1] == -1.f) x[j][b][e] = -INFINITY;
        }
      }
      const float lv[2] = {fmaxf(__log2f(vd[0]), kLog2Least), fmaxf(__log2f(vd[1]), kLog2Least)};
      bool calm = true;
      float top[RB];
#pragma unroll
      for (int b = 0; b < RB; ++b) {
        const float t0 = fmaxf(fmaxf(x[0][b][0], x[0][b][1]), fmaxf(x[1][b][0], x[1][b][1])) + lv[0];
        const float t1 = fmaxf(fmaxf(x[2][b][0], x[2][b][1]), fmaxf(x[3][b][0], x[3][b][1])) + lv[1];
        top[b] = fmaxf(t0, t1);
        calm = calm && !(top[b] > m_row[b] + kRaiseBy);
      }
      if (!__all_sync(0xffffffffu, calm)) {
#pragma unroll
        for (int b = 0; b < RB; ++b) {
          float mx = fmaxf(top[b], __shfl_xor_sync(0xffffffffu, top[b], 1));
          mx = fmaxf(fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2)) - kHeadroom, m_row[b]);
          const float nm_new = mx == -INFINITY ? 0.f : -mx;
          const float alpha = m_row[b] == -INFINITY ? 0.f : ex2_approx(nm_new - nm[b]);
          l_row[b] *= alpha;
          // rows 2t and 2t + 1 of the row block are the columns of O^T this thread holds
          const float a0 = __shfl_sync(0xffffffffu, alpha, 8 * t), a1 = __shfl_sync(0xffffffffu, alpha, 8 * t + 4);
#pragma unroll
          for (int j = 0; j < C::kMTiles; ++j) {
            o[j][b][0] *= a0; o[j][b][2] *= a0;
            o[j][b][1] *= a1; o[j][b][3] *= a1;
          }
          m_row[b] = mx;
          nm[b] = nm_new;
        }
      }
      uint32_t pb[RB][4];
#pragma unroll
      for (int b = 0; b < RB; ++b) {
        float p[8];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) p[2 * j + e] = ex2_approx(x[j][b][e] + nm[b]);
        l_row[b] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
#pragma unroll
        for (int j = 0; j < 4; ++j) pb[b][j] = pack_half2(p[2 * j] * vd[j >> 1], p[2 * j + 1] * vd[j >> 1]);
      }
      if (!whole) {                                       // nothing of keys that do not count, not even a NaN times zero
#pragma unroll
        for (int b = 0; b < RB; ++b)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (kd[j >> 1] == -1.f) pb[b][j] = 0u;
      }
#pragma unroll
      for (int blk = 0; blk < C::kBlocks; ++blk) {
        uint32_t vr[8][C::kVWords];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int row = 16 * (i >> 2) + 8 * ((i >> 1) & 1) + 2 * t + (i & 1);
          if constexpr (W == 64) {
            const uint2 v = ld_shared8(sv + row * 64 + (((g >> 1) ^ ((row >> 1) & 3)) << 4) + 8 * (g & 1));
            vr[i][0] = v.x; vr[i][1] = v.y;
          } else {
            const uint4 v = ld_shared16(sv + blk * C::kTile + row * 128 + ((g ^ (row & 7)) << 4));
            vr[i][0] = v.x; vr[i][1] = v.y; vr[i][C::kVWords - 2] = v.z; vr[i][C::kVWords - 1] = v.w;
          }
          if (!whole && (key0 + row >= vis || kd[row >> 4] == -1.f)) {
#pragma unroll
            for (int w = 0; w < C::kVWords; ++w) vr[i][w] = 0u;
          }
        }
#pragma unroll
        for (int w = 0; w < C::kVWords; ++w) {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint32_t* v = &vr[4 * u][w];
            constexpr int kKey = C::kVWords;
            uint32_t am[4][2];
            fp8_to_half4<kE5M2>(__byte_perm(v[0], v[kKey], 0x5140), am[0][0], am[1][0]);
            fp8_to_half4<kE5M2>(__byte_perm(v[2 * kKey], v[3 * kKey], 0x5140), am[0][1], am[1][1]);
            fp8_to_half4<kE5M2>(__byte_perm(v[0], v[kKey], 0x7362), am[2][0], am[3][0]);
            fp8_to_half4<kE5M2>(__byte_perm(v[2 * kKey], v[3 * kKey], 0x7362), am[2][1], am[3][1]);
#pragma unroll
            for (int b = 0; b < RB; ++b) {
              mma_f16(o[blk * C::kTilesPerBlock + 2 * w][b], am[0][0], am[1][0], am[0][1], am[1][1], pb[b][2 * u], pb[b][2 * u + 1]);
              mma_f16(o[blk * C::kTilesPerBlock + 2 * w + 1][b], am[2][0], am[3][0], am[2][1], am[3][1], pb[b][2 * u], pb[b][2 * u + 1]);
            }
          }
        }
      }
      __syncwarp();                                       // every lane has read the stage
      if (step + C::kStages < last) scales[C::kStages - 1] = fill(step + C::kStages, page, stage);
      if (++stage == C::kStages) {
        stage = 0;
        phase ^= 1u;
      }
    }
    // ---- what the segment gave ----
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      l_row[b] += __shfl_xor_sync(0xffffffffu, l_row[b], 1);
      l_row[b] += __shfl_xor_sync(0xffffffffu, l_row[b], 2);
    }
    const bool alone = step0 == 0 && step1 == steps;
    const int D = a.c.head_dim;
    // slot 2 w: the segment that share w begins with; 2 w + 1: one that begins an item and ends the share
    const int64_t slot = 2 * me + (step0 == 0 ? 1 : 0);
    float* const part = a.partial + slot * C::kRows * (D + 2);
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      if (t == 0 && 8 * b + g < n_rows) {
        const int r = row0 + 8 * b + g;
        if (alone) {
          if (a.lse != nullptr)
            a.lse[static_cast<int64_t>(s.first + r / a.group) * a.heads_q + h * a.group + r % a.group] =
                l_row[b] == 0.f ? -INFINITY : (m_row[b] + __log2f(l_row[b])) * 0.6931471805599453f;
        } else {
          part[C::kRows * D + 8 * b + g] = m_row[b];
          part[C::kRows * (D + 1) + 8 * b + g] = l_row[b];
        }
      }
      const float inv = l_row[b] == 0.f ? 0.f : 1.f / l_row[b];
      float f[2];
      f[0] = __shfl_sync(0xffffffffu, inv, 8 * t);
      f[1] = __shfl_sync(0xffffffffu, inv, 8 * t + 4);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int in = 8 * b + 2 * t + e;
        if (in >= n_rows) continue;
#pragma unroll
        for (int blk = 0; blk < C::kBlocks; ++blk) {
          const int col = 128 * blk + 4 * C::kVWords * g;
          if (col >= D) continue;
          float v[2 * C::kTilesPerBlock];
#pragma unroll
          for (int j = 0; j < C::kTilesPerBlock; ++j) {
            v[2 * j] = o[blk * C::kTilesPerBlock + j][b][e];
            v[2 * j + 1] = o[blk * C::kTilesPerBlock + j][b][2 + e];
          }
          if (alone) {
            const int r = row0 + in;
            uint16_t* const p = static_cast<uint16_t*>(a.o) + (static_cast<int64_t>(s.first + r / a.group) * a.heads_q + h * a.group + r % a.group) * D + col;
#pragma unroll
            for (int j = 0; j < 2 * C::kTilesPerBlock; j += 8) {
              uint32_t w[4];
#pragma unroll
              for (int i = 0; i < 4; ++i)
                w[i] = a.bf16 ? pack_pair<true>(v[j + 2 * i] * f[e], v[j + 2 * i + 1] * f[e]) : pack_pair<false>(v[j + 2 * i] * f[e], v[j + 2 * i + 1] * f[e]);
              st_global_v4(p + j, w[0], w[1], w[2], w[3]);
            }
          } else {
            float4* const p = reinterpret_cast<float4*>(part + in * D + col);
#pragma unroll
            for (int j = 0; j < 2 * C::kTilesPerBlock; j += 4) p[j / 4] = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
          }
        }
      }
    }
    pos = item_at + step1;
  }
}

// Rows (token and query head) whose item several warps shared: kParts warps to a row, of the CTA's eight.
constexpr int kCombineWarps = 8;
template <int kParts>
__global__ void __launch_bounds__(32 * kCombineWarps) kv_combine_kernel(const KvAttendArgs a, int rows, int64_t workers_most) {
  __shared__ float4 s_acc[kParts > 1 ? kCombineWarps : 1][64];
  __shared__ float s_l[kCombineWarps];
  start_after_predecessor();
  let_successor_start();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = warp % kParts;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kCombineWarps / kParts) + warp / kParts;
  const int token = static_cast<int>(row / a.heads_q), head = static_cast<int>(row - static_cast<int64_t>(token) * a.heads_q);
  if (token >= a.c.tokens) return;                        // kParts > 1: the returns are the whole CTA's
  int b, unused;
  if (a.c.cu == nullptr) b = token / a.c.even;
  else kv_find_slot(a.c, token, 1, 0, &b, &unused);
  const KvSeq s = kv_seq(a.c, b);
  if (token < s.first || token >= s.first + s.n) return;
  const volatile int64_t* bases = a.bases;
  const int64_t total = bases[a.c.batch], base = bases[b];
  const int64_t workers = workers_of(total, workers_most);
  const int h = head / a.group;
  const int64_t r = static_cast<int64_t>(token - s.first) * a.group + head % a.group, rb = r / rows;
  const int in = static_cast<int>(r - rb * rows);
  const int steps = item_steps(s);
  const int64_t first = base + (rb * a.c.heads + h) * steps;
  const int64_t w0 = share_of(total, workers, first), w1 = share_of(total, workers, first + steps - 1);
  if (w0 == w1) return;
  const int D = a.c.head_dim;
  // the item begins at the end of share w0 and goes on at the beginning of the next
  auto part_of = [&](int64_t w) { return a.partial + (2 * w + (w == w0 ? 1 : 0)) * rows * (D + 2); };
  float m = -INFINITY;
#pragma unroll 4
  for (int64_t w = w0 + lane; w <= w1; w += 32) m = fmaxf(m, ld_global(part_of(w) + rows * D + in));
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, i));
  float l = 0.f;
  const int quads = D >> 2;                               // a lane has quads lane and lane + 32
  float4 acc[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
#pragma unroll 8
  for (int64_t w = w0 + part; w <= w1; w += kParts) {
    const float* p = part_of(w);
    const float mw = ld_global(p + rows * D + in);
    const float f = mw == -INFINITY ? 0.f : ex2_approx(mw - m);
    l += ld_global(p + rows * (D + 1) + in) * f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int q = lane + 32 * i;
      if (q < quads) {
        const uint4 u = ld_global(reinterpret_cast<const uint4*>(p + in * D) + q);
        acc[i].x += __uint_as_float(u.x) * f; acc[i].y += __uint_as_float(u.y) * f;
        acc[i].z += __uint_as_float(u.z) * f; acc[i].w += __uint_as_float(u.w) * f;
      }
    }
  }
  if (kParts > 1) {
    s_acc[warp][lane] = acc[0];
    s_acc[warp][lane + 32] = acc[1];
    if (lane == 0) s_l[warp] = l;
    __syncthreads();
    if (warp != 0) return;
#pragma unroll
    for (int w = 1; w < kParts; ++w) {
      l += s_l[w];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float4 v = s_acc[w][lane + 32 * i];
        acc[i].x += v.x; acc[i].y += v.y; acc[i].z += v.z; acc[i].w += v.w;
      }
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint2* const out = reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.o) + row * D);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int q = lane + 32 * i;
    if (q >= quads) continue;
    const float4 v = acc[i];
    out[q] = a.bf16 ? make_uint2(pack_pair<true>(v.x * inv, v.y * inv), pack_pair<true>(v.z * inv, v.w * inv))
                    : make_uint2(pack_pair<false>(v.x * inv, v.y * inv), pack_pair<false>(v.z * inv, v.w * inv));
  }
  if (a.lse != nullptr && lane == 0) a.lse[row] = l == 0.f ? -INFINITY : (m + __log2f(l)) * 0.6931471805599453f;
}

int width_of(int head_dim) { return head_dim <= 64 ? 64 : (head_dim <= 128 ? 128 : 256); }

// Rows of a block: as many as the mean sequence has, up to what the registers hold.
int block_rows(const KvAttendSizes& z) {
  const int64_t mean = (static_cast<int64_t>(z.tokens) + z.batch - 1) / z.batch * (z.heads_q / z.heads);
  if (mean <= 8) return 8;
  return mean <= 16 || width_of(z.head_dim) == 256 ? 16 : 32;
}

template <int W, int RB, bool kE5M2>
cudaError_t launch_attend(const CUtensorMap& tk, const CUtensorMap& tv, const KvAttendArgs& a, int sms, cudaStream_t stream) {
  using C = ACfg<W, RB>;
  auto kernel = &kv_attend_kernel<W, RB, kE5M2>;
  constexpr int smem = C::kWarps * C::kStages * C::kStageBytes + 1024;
  static std::atomic<bool> ready[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const bool cached = dev >= 0 && dev < 64;
  if (!cached || !ready[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    if (cached) ready[dev].store(true, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(sms), 1, 1);
  cfg.blockDim = dim3(32 * C::kWarps, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1] = {overlap_attribute()};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kernel, tk, tv, a);
  if (e != cudaSuccess) return e;
  // Up to kWideRows rows a CTA takes one: an item of a long sequence has a part from every warp that shared it.
  constexpr int64_t kWideRows = 8192;
  const int64_t n = static_cast<int64_t>(a.c.tokens) * a.heads_q;
  const int64_t ctas = n <= kWideRows ? n : (n + kCombineWarps - 1) / kCombineWarps;
  if (ctas > 0x7fffffff) return cudaErrorInvalidConfiguration;
  cfg.gridDim = dim3(static_cast<unsigned>(ctas), 1, 1);
  cfg.blockDim = dim3(32 * kCombineWarps, 1, 1);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, n <= kWideRows ? &kv_combine_kernel<kCombineWarps> : &kv_combine_kernel<1>, a, C::kRows,
                            static_cast<int64_t>(sms) * C::kWarps);
}

template <bool kE5M2>
cudaError_t launch_fmt(const CUtensorMap& tk, const CUtensorMap& tv, const KvAttendArgs& a, int sms, int rows, cudaStream_t stream) {
  switch (width_of(a.c.head_dim)) {
    case 64:
      return rows == 8 ? launch_attend<64, 1, kE5M2>(tk, tv, a, sms, stream)
                       : (rows == 16 ? launch_attend<64, 2, kE5M2>(tk, tv, a, sms, stream) : launch_attend<64, 4, kE5M2>(tk, tv, a, sms, stream));
    case 128:
      return rows == 8 ? launch_attend<128, 1, kE5M2>(tk, tv, a, sms, stream)
                       : (rows == 16 ? launch_attend<128, 2, kE5M2>(tk, tv, a, sms, stream) : launch_attend<128, 4, kE5M2>(tk, tv, a, sms, stream));
    default:
      return rows == 8 ? launch_attend<256, 1, kE5M2>(tk, tv, a, sms, stream) : launch_attend<256, 2, kE5M2>(tk, tv, a, sms, stream);
  }
}

int64_t round256(int64_t n) { return (n + 255) / 256 * 256; }

}  // namespace

int64_t kv_attend_workspace(const KvAttendSizes& z, int sms) {
  const int64_t slots = 2ll * sms * (width_of(z.head_dim) == 256 ? ACfg<256, 1>::kWarps : ACfg<128, 1>::kWarps);
  return round256((static_cast<int64_t>(z.batch) + 1) * 8) + slots * block_rows(z) * (z.head_dim + 2) * 4;
}

cudaError_t launch_kv_attend(const CUtensorMap& tk, const CUtensorMap& tv, KvAttendArgs a, const KvAttendSizes& z, void* workspace, bool e5m2, int sms,
                             cudaStream_t stream) {
  a.bases = static_cast<int64_t*>(workspace);
  a.partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + round256((static_cast<int64_t>(a.c.batch) + 1) * 8));
  const int rows = block_rows(z);
  return e5m2 ? launch_fmt<true>(tk, tv, a, sms, rows, stream) : launch_fmt<false>(tk, tv, a, sms, rows, stream);
}

}  // namespace fa8
