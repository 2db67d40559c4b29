// Attention of a few new tokens' queries over the pages of the fp8 cache (decoding), sm_100a.
//
//   x_j = c (q . k8_j) dk_j,   m >= x_j + [log2 dv_j] - 14,   O = sum_j 2^(x_j - m) dv_j v8_j / sum_j 2^(x_j - m)
//
// with c = softmax_scale log2(e), dk_j and dv_j the scales of key j's page, [] the whole part.  The reference m of a row is taken over x + [log2 dv],
// so that what is rounded to fp16, P_j = 2^(x_j - m) dv_j, is below 2^15 whatever the pages' scales; the sum of the
// denominators is of unrounded fp32 numbers.  m starts 6 below the first keys' maximum, so that P has its full precision twenty
// binades down, and is raised to 6 below the maximum so far, and what was summed rescaled, only when some P might pass 2^15.  Keys and
// queries enter the products exactly: every fp8 value is an fp16 value, and bf16 queries are brought into fp16's range by a power
// of two per row (what that cuts off is below 2^-39 of the row's largest).
//
// What bounds it: reading K and V once, 2 * head_dim bytes a key for all query rows that share it.
//   * The rows of a block are the query heads that share a K/V head times the new tokens: 8, 16 or 32 rows.
//   * Work is counted in steps of 32 or 16 keys of one sequence, K/V head and row block (an item), and dealt out to one CTA per SM, and in
//     it to its warps, in equal, contiguous shares whatever the lengths of the sequences are.  A share is worked out from the
//     lengths on the device, so a captured call can be replayed with other lengths.
//   * A warp streams its steps through a ring of its own in shared memory: one lane issues tiled copies (swizzled, so
//     that both operands are read without bank conflicts), page numbers and scales being loaded 32 pages ahead.
//     No warp waits for another until its share is through.
//   * The warps' parts of an item are added up in shared memory.  What a CTA has of an item that others share goes to the workspace, and
//     kv_combine_kernel puts such items together by a record that the CTA with the item's end leaves, always in the same order.  How steps
//     are dealt out depends on all lengths of the call, hence so do the last bits.
//   * Few short items go to a cluster of one to eight CTAs each (lone_split), which adds up over distributed shared memory: one launch.
//
// Measured at head dim 128, 32 heads over 8 (GPU time): 16 sequences of 8192 keys 52.6 us, 5.1 TB/s, of which 36 us are the steps, at
// 7.5 TB/s, and the rest what goes before and after them: lengths 1.3 us, page numbers 1.2, the first pages 1, adding up 1.5, the combining
// kernel 2.  One of 131072 keys 54 us; one of 600 keys 7 us.  At head dim 64, 64 sequences of 20 to 8000 keys, 36 us: 58 % of the issue slots, the rest
// mostly instructions that wait for the one before (a key's 64 bytes cost as many to convert and multiply whatever the rows).
//
// Operand layouts are those of fa8_decode_sm100.cu: S = Q K^T with the query rows as M (16, eight of them padding
// when there are eight) and eight keys as N, the k index permuted alike in both operands; O^T = V^T P^T with 16 output
// columns as M, the rows as N and 16 keys as k.  tcgen05 would want 128 rows.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <atomic>

#include "fa8_kernel.h"
#include "fa8_kv.h"
#include "kv_common.cuh"

namespace fa8 {

namespace {

namespace cg = cooperative_groups;

constexpr float kHeadroom = 6.f, kRaiseBy = 14.f;       // log2 of the largest P, as by the whole part of log2 dv, under a fresh reference, and at all
// log2 of the smallest scale of V that the reference m follows: exponentials reach 2^(kRaiseBy + 80), of which fp32 adds up 2^31
constexpr float kLog2Least = -80.f;
constexpr unsigned long long kLimitNs = 2000000000ull; // bound of every wait
constexpr int kExpiredWait = 0xa77e;                   // code in the status words

// Head dims up to W run in the instance built for W (the copies fill what is missing with zeros); RB blocks of eight rows.
template <int W, int RB>
struct ACfg {
  static constexpr int kStepKeys = kv_step_keys(W, 8 * RB);      // of a step: 4 or 8 KB of K and V
  static constexpr int kHalves = kStepKeys / 16;                 // of a step: sixteen keys lie in one page
  static constexpr int kRowBytes = W < 128 ? W : 128;            // of a swizzled tile
  static constexpr int kBlocks = W / kRowBytes;                  // tiles side by side
  static constexpr int kTile = kStepKeys * kRowBytes;
  static constexpr int kStageBytes = 2 * kBlocks * kTile;        // K, then V
  // Warps of the one CTA per SM: what the register file holds at this instance's registers per thread (a quarter of the warps
  // share a quarter of it), and stages of each: 180 to 192 KB in all, which is more than the 7.5 TB/s times the latency
  // of some 1.5 us ask of an SM (76 KB).
  static constexpr int kWarps = W == 64 && RB == 1 ? 16 : (W == 64 && RB == 2 ? 12 : 8);
  static constexpr int kStages = kWarps == 16 ? 3 : (kWarps == 12 ? 4 : (kStageBytes == 4096 ? 6 : 3));
  static constexpr int kRingBytes = kStages * kStageBytes;
  static constexpr int kChunks = W / 64;                         // 16-byte pieces of a K row per thread
  static constexpr int kSteps = W / 16;                          // k-steps of Q K^T
  static constexpr int kVWords = W == 64 ? 2 : 4;
  static constexpr int kTilesPerBlock = 2 * kVWords;
  static constexpr int kMTiles = W / 16;
  static constexpr int kRows = 8 * RB;
  static constexpr int kORow = W + 4;                            // floats per row of a partial sum in shared memory
  static constexpr int kPartBytes = kRows * (kORow + 2) * 4;
  static_assert(kPartBytes <= kRingBytes, "a warp's partial sum lies in its ring");
  static constexpr int kSmem = kWarps * kRingBytes + 1024;
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
__device__ __forceinline__ int item_steps(const KvSeq& s, int step_keys) { return max(1, (s.len + step_keys - 1) / step_keys); }
__device__ __forceinline__ int row_blocks(const KvSeq& s, int group, int rows) { return (s.n * group + rows - 1) / rows; }

// What an item counts for when work is dealt out, in units of 2^unit_shift steps: its steps, and kStartUnits for what a segment costs
// before its first step (a chain of loads: page number, page).
constexpr int kStartUnits = 2;
__device__ __forceinline__ int item_units(const KvAttendArgs& a, int steps) { return ((steps - 1) >> a.unit_shift) + 1 + kStartUnits; }
__device__ __forceinline__ int seq_units(const KvAttendArgs& a, const KvSeq& s, int rows, int step_keys) {
  return row_blocks(s, a.group, rows) * a.c.heads * item_units(a, item_steps(s, step_keys));
}

// Item of a warp's last segment.
struct Segment {
  int first, row0, n_rows, head;         // first new token of the sequence, rows of the block, K/V head
  bool begins, ends;                     // the CTA's share has the item's first step, its last
};

// kLone: a cluster to an item, its CTAs and their warps sharing the item's steps; otherwise shares of all steps of the call.
template <int W, int RB, bool kE5M2, bool kLone>
__global__ void __launch_bounds__(32 * ACfg<W, RB>::kWarps, 1) kv_attend_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                                                                                const KvAttendArgs a) {
  using C = ACfg<W, RB>;
  constexpr int kWarps = C::kWarps, kStepKeys = C::kStepKeys, kHalves = C::kHalves;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t s_bar[kWarps * C::kStages];
  // Scales of K of the step's halves (-1: no page), then those of V.  (What is static, 1 KB of the system's and the rings are to fit 196 KB: past
  // that the L1 cache gives up 32 KB more.  With sixteen bytes more a stage, for log2 of V's, 8 sequences of 4000 keys and 32 rows at
  // head dim 128 took 46 us for 43.)
  __shared__ __align__(16) float s_scale[kWarps * C::kStages][4];
  // the first unit of the item that a warp's last, and (where it had several) its first segment is of; -1: whole items only
  __shared__ int s_last[kWarps], s_head[kWarps];
  __shared__ bool s_single[kWarps], s_special[kWarps];       // (s_special: NaNs or infinities were taken out of the segment's V)
  __shared__ Segment s_item[kLone ? 1 : kWarps];
  __shared__ float s_m[C::kRows], s_l[C::kRows];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t ring0 = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t ring = ring0 + warp * C::kRingBytes;
  const uint32_t bars = smem_u32(s_bar) + 8u * warp * C::kStages;
  // partial sums of warp w: [row][column], then the rows' references and sums
  auto part_of = [&](int w) { return reinterpret_cast<float*>(smem_raw + (ring0 - smem_u32(smem_raw)) + w * C::kRingBytes); };
  if (lane == 0) {
    s_special[warp] = false;
    for (int i = 0; i < C::kStages; ++i) mbar_init(bars + 8 * i, 1);
    fence_mbar_init();
    fence_proxy_async_smem();
    if (warp == 0) {
      prefetch_tensormap(&tk);
      prefetch_tensormap(&tv);
    }
  }
  __syncwarp();
  start_after_predecessor();
  let_successor_start();
  const int P = 1 << a.c.page_shift;
  const int boxes = P < kStepKeys ? 2 : 1;               // copies per step and tile
  const int D = a.c.head_dim;
  // Rows of 64 bytes come two to a swizzled line of 128 (D = 64; a copy moves a line at a time, whatever its length), rows of 32 padded to
  // 64: in the first the halves of every other four lines are exchanged.
  const uint32_t flip = W == 64 && D == 64 ? 64u : 0u;

  // ---- what this warp has to do: units [pos, end) of the call's (kLone: steps of the item's) ----
  int pos, end, at = 0, cta_lo = 0, cta_hi = 0, share = 1;
  int seq = 0, lone_row0 = 0, lone_head = 0;
  KvSeq s{0, 0, 0, false};
  int steps, items;
  if constexpr (kLone) {
    const int rank = static_cast<int>(blockIdx.x) % a.n_split, id = static_cast<int>(blockIdx.x) / a.n_split;
    const int slot = id / a.c.heads;
    lone_head = id - slot * a.c.heads;
    int j;
    const bool bad = warp == 0 && kv_bad(a.c, blockIdx.x, false);      // there are more CTAs than sequences
    kv_find_slot(a.c, slot, a.block_tokens, 1, &seq, &j);
    s = kv_seq(a.c, seq);
    if (bad) report_bad_index(a.c);
    const int64_t token0 = static_cast<int64_t>(j) * a.block_tokens;
    if (token0 >= s.n) return;                           // the whole cluster
    lone_row0 = static_cast<int>(token0) * a.group;
    steps = item_steps(s, kStepKeys);
    items = 1;
    const int w = rank * kWarps + warp, n = a.n_split * kWarps, each = steps / n, rest = steps - each * n;
    pos = each * w + min(w, rest);
    end = pos + each + (w < rest ? 1 : 0);
  } else {
    // by every warp for itself: 32 sequences at a time, the first of which stay in registers
    const KvSeq mine = lane < a.c.batch ? kv_seq(a.c, lane) : KvSeq{0, 0, 0, false};
    const int units = seq_units(a, mine, C::kRows, kStepKeys);
    int total = units;
    bool bad = mine.bad;
#pragma unroll 4
    for (int b = 32 + lane; b < a.c.batch; b += 32) {
      const KvSeq x = kv_seq(a.c, b);
      bad = bad || x.bad;
      total += seq_units(a, x, C::kRows, kStepKeys);
    }
    total = __reduce_add_sync(0xffffffffu, total);
    if (bad && blockIdx.x == 0 && warp == 0) report_bad_index(a.c);
    if (threadIdx.x == 0) a.records[blockIdx.x].first_cta = -1;
    share = (total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x);
    if (static_cast<int>(blockIdx.x) * static_cast<int64_t>(share) >= total) return;
    cta_lo = blockIdx.x * share;
    cta_hi = min(cta_lo + share, total);
    const int each = (cta_hi - cta_lo) / kWarps, rest = (cta_hi - cta_lo) % kWarps;
    pos = cta_lo + each * warp + min(warp, rest);
    end = pos + each + (warp < rest ? 1 : 0);
    // The sequence that pos is in.  (A warp without steps may stand behind the last one: it looks where the CTA begins.)
    const int from = pos < end ? pos : cta_lo;
    for (int b0 = 0; b0 < a.c.batch; b0 += 32) {
      KvSeq x = mine;
      int u = units;
      if (b0 > 0) {
        x = b0 + lane < a.c.batch ? kv_seq(a.c, b0 + lane) : KvSeq{0, 0, 0, false};
        u = seq_units(a, x, C::kRows, kStepKeys);
      }
      int sum = u;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += y;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, at + sum > from);
      if (past != 0u) {
        const int l = __ffs(past) - 1;
        at += __shfl_sync(0xffffffffu, sum - u, l);
        seq = b0 + l;
        s.first = __shfl_sync(0xffffffffu, x.first, l);
        s.n = __shfl_sync(0xffffffffu, x.n, l);
        s.len = __shfl_sync(0xffffffffu, x.len, l);
        break;
      }
      at += __shfl_sync(0xffffffffu, sum, 31);
    }
    steps = item_steps(s, kStepKeys);
    items = row_blocks(s, a.group, C::kRows) * a.c.heads;
    if (items == 0) end = pos;                           // lengths that changed since they were added up
  }

  // This CTA has the last part of an item that begins at `item_at`: what the combining kernel needs to know.
  auto put_record = [&](int item_at, int first, int row0, int n_rows, int h) {
    a.records[blockIdx.x] = {(item_at + kStartUnits) / share, first, row0, n_rows, h};
  };

  int stage = 0;
  uint32_t phase = 0;
  int last_item = -1, head_item = -1;
  bool single = false;
  bool first = true;
  while (pos < end) {
    int h, row0, n_rows, step0, step1;
    int item_at, item_end;
    if constexpr (kLone) {
      h = lone_head;
      row0 = lone_row0;
      n_rows = min(a.block_tokens * a.group, s.n * a.group - row0);
      item_at = 0;
      item_end = steps;
      step0 = pos;
      step1 = end;
    } else {
      const int units = item_units(a, steps);
      if (pos >= at + items * units) {                     // the next sequence that has items
        at += items * units;
        if (++seq >= a.c.batch) break;                     // lengths that changed since they were added up
        s = kv_seq(a.c, seq);
        steps = item_steps(s, kStepKeys);
        items = row_blocks(s, a.group, C::kRows) * a.c.heads;
        continue;
      }
      const int item = (pos - at) / units;
      item_at = at + item * units;
      item_end = item_at + units;
      // a share that ends before the item's first step leaves the item to the next
      if (end - item_at <= kStartUnits) break;
      step0 = max(0, pos - item_at - kStartUnits) << a.unit_shift;
      step1 = min(steps, (min(item_end, end) - item_at - kStartUnits) << a.unit_shift);
      const int rb = item / a.c.heads;
      h = item - rb * a.c.heads;
      row0 = rb * C::kRows;
      n_rows = min(C::kRows, s.n * a.group - row0);
    }
    // keys that the block's last row sees, and its first
    auto seen = [&](int row) { return a.causal ? max(0, min(s.len, s.len - s.n + row / a.group + 1)) : s.len; };
    const int vis = seen(row0 + n_rows - 1);
    const int least = seen(row0);
    const int last = min(step1, (vis + kStepKeys - 1) / kStepKeys);     // steps past it see nothing

    // The rows of Q: thread (g, t) takes columns 16 kChunks t ... of a block of 128 (64), the bytes of K that it reads below.  Asked
    // for before the pages are: behind those they would wait for as long as a ring takes to fill.
    uint4 q[RB][C::kChunks][2];
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      const bool in = 8 * b + g < n_rows;
      const int r = in ? row0 + 8 * b + g : row0, token = r / a.group;
      const uint16_t* p = static_cast<const uint16_t*>(a.q.x) + (s.first + token) * a.q.token_stride + (h * a.group + (r - token * a.group)) * a.q.head_stride;
#pragma unroll
      for (int c = 0; c < C::kChunks; ++c) {
        constexpr int kPer = C::kChunks < 2 ? C::kChunks : 2;            // chunks of a block
        const int col = 128 * (c / 2) + 16 * (kPer * t + c % 2);
        const bool read = in && col < D;
        q[b][c][0] = read ? ld_global(reinterpret_cast<const uint4*>(p + col)) : make_uint4(0u, 0u, 0u, 0u);
        q[b][c][1] = read ? ld_global(reinterpret_cast<const uint4*>(p + col + 8)) : make_uint4(0u, 0u, 0u, 0u);
      }
    }

    // ---- filling the ring ----
    // Page numbers and scales of 32 pages at a time, a lane each: those of the batch of pages in use, the numbers and scales of the
    // next, the numbers of the one after, so that no load is waited for once the segment has begun.
    const int* const table = a.c.table + static_cast<int64_t>(seq) * a.c.table_stride;
    const int n_pages = (min(vis, last * kStepKeys) + P - 1) >> a.c.page_shift;     // of this segment's keys
    auto load_page = [&](int p) { return p + lane < n_pages ? ld_int(table + p + lane) : -2; };
    auto load_scale = [&](const float* d, int page) {
      return static_cast<unsigned>(page) < static_cast<unsigned>(a.c.num_pages) ? ld_global(d + static_cast<int64_t>(page) * a.c.heads + h) : -1.f;
    };
    int page0 = (step0 * kStepKeys) >> a.c.page_shift;   // the batch's first
    int id = load_page(page0), id1 = load_page(page0 + 32), id2 = load_page(page0 + 64);
    float kd_of = load_scale(a.c.k_descale, id), vd_of = load_scale(a.c.v_descale, id);
    float kd1 = load_scale(a.c.k_descale, id1), vd1 = load_scale(a.c.v_descale, id1);
    auto advance = [&](int step) {
      if (((step * kStepKeys) >> a.c.page_shift) >= page0 + 32) {
        page0 += 32;
        id = id1;
        kd_of = kd1;
        vd_of = vd1;
        id1 = id2;
        kd1 = load_scale(a.c.k_descale, id1);
        vd1 = load_scale(a.c.v_descale, id1);
        id2 = load_page(page0 + 64);
      }
    };
    // Copies of a step, by one lane.  (A batch of 32 pages begins with a step.)
    auto copy = [&](int step, int st) {
      const int key = step * kStepKeys, in_batch = (key >> a.c.page_shift) - page0;
      const int p0 = __shfl_sync(0xffffffffu, id, in_batch);
      const bool ok0 = static_cast<unsigned>(p0) < static_cast<unsigned>(a.c.num_pages);
      int p1 = 0;
      bool ok1 = false, bad = !ok0;
      if (boxes == 2) {
        p1 = __shfl_sync(0xffffffffu, id, in_batch + 1);
        ok1 = static_cast<unsigned>(p1) < static_cast<unsigned>(a.c.num_pages);
        bad = bad || (!ok1 && key + 16 < vis);
      }
      if (bad) report_bad_index(a.c);
      if (lane == 0) {
        const uint32_t bar = bars + 8 * st, dst = ring + st * C::kStageBytes;
        constexpr uint32_t kRow = 2 * C::kBlocks * C::kRowBytes;
        mbar_arrive_expect_tx(bar, boxes == 2 ? (static_cast<int>(ok0) + ok1) * 16 * kRow : (ok0 ? kStepKeys * kRow : 0u));
        if (ok0) {
          const int slice = p0 * a.c.heads + h, row = (key & (P - 1)) >> (flip ? 1 : 0);
#pragma unroll
          for (int c = 0; c < C::kBlocks; ++c) {
            tma_load_3d(dst + c * C::kTile, &tk, bar, c * 128, row, slice);
            tma_load_3d(dst + (C::kBlocks + c) * C::kTile, &tv, bar, c * 128, row, slice);
          }
        }
        if (ok1) {
          const int slice = p1 * a.c.heads + h;
#pragma unroll
          for (int c = 0; c < C::kBlocks; ++c) {
            tma_load_3d(dst + c * C::kTile + 16 * C::kRowBytes, &tk, bar, c * 128, 0, slice);
            tma_load_3d(dst + (C::kBlocks + c) * C::kTile + 16 * C::kRowBytes, &tv, bar, c * 128, 0, slice);
          }
        }
      }
      __syncwarp();
    };
    // Lane l looks after the step's half l & 1: the scale of K (l & 2 = 0), -1 where there is no page, or that of V.
    auto put_scales = [&](int step, int st) {
      const int key = step * kStepKeys + (lane & (kHalves - 1)) * 16;
      const int src = ((key >> a.c.page_shift) - page0) & 31;
      const float kd = __shfl_sync(0xffffffffu, kd_of, src), vd = __shfl_sync(0xffffffffu, vd_of, src);
      if (lane < 4) s_scale[warp * C::kStages + st][lane] = (lane & 2) ? vd : (key < vis ? kd : -1.f);
    };
    // (Code that runs once a launch is kept short: its instructions have to be fetched past the pages that are being read.)
    {
      int st = stage;
#pragma unroll 1
      for (int i = step0; i < min(step0 + C::kStages, last); ++i) {      // at most 32 pages: one batch
        copy(i, st);
        if (++st == C::kStages) st = 0;
      }
    }

    // ---- the rows of Q as A operands ----
    uint32_t qa[C::kSteps][RB][2];
    float c_row[RB], m_row[RB], nm[RB], l_row[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      auto& x = q[b];
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
    {
      int st = stage;
#pragma unroll 1
      for (int i = step0; i < min(step0 + C::kStages, last); ++i) {
        put_scales(i, st);
        if (++st == C::kStages) st = 0;
      }
      __syncwarp();
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
      if (!wait_copies(bars + 8 * stage, phase)) {
        // Give up: report, wait (with a limit each) for the copies in flight, which write to this CTA's memory, and go where the
        // others will be waiting.
        if (lane == 0) report_expired_wait(a.c.status, a.c.host_status, kExpiredWait);
        for (int i = step; i < min(step + C::kStages, last); ++i) {
          wait_copies(bars + 8 * stage, phase);
          if (++stage == C::kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        end = pos;
        break;
      }
      const uint32_t sk = ring + stage * C::kStageBytes, sv = sk + C::kBlocks * C::kTile;
      const float4 scale = *reinterpret_cast<const float4*>(s_scale[warp * C::kStages + stage]);
      const float kd[2] = {scale.x, scale.y}, dv[2] = {scale.z, scale.w};
      // For the reference the whole part of log2 dv will do, which lets P be 2^15: of the exponent e, 2^23 + e + 127 as a float less 2^23 + 127.
      auto log2_of = [](float d) { return fmaxf(__uint_as_float(0x4b000000u | (__float_as_uint(d) >> 23)) - 8388735.f, kLog2Least); };
      const float lv[2] = {log2_of(dv[0]), log2_of(dv[1])};
      // a step that holds keys past some row's last, or of a page that is out of range
      const int key0 = step * kStepKeys;
      const bool whole = key0 + kStepKeys <= least && kd[0] != -1.f && (kHalves == 1 || kd[1] != -1.f);

      float x[2 * kHalves][RB][2];                        // score tile, row block, its two keys: q . k8
#pragma unroll
      for (int j = 0; j < 2 * kHalves; ++j) {
        constexpr int kPairs = (RB + 1) / 2;
        float sc[kPairs][4];
#pragma unroll
        for (int b = 0; b < kPairs; ++b) sc[b][0] = sc[b][1] = sc[b][2] = sc[b][3] = 0.f;
        const int row = 8 * j + g;
#pragma unroll
        for (int c = 0; c < C::kChunks; ++c) {
          uint32_t at_row;
          if constexpr (W == 64) at_row = sk + ((row * 64 + ((t ^ ((row >> 1) & 3)) << 4)) ^ ((j & 1) ? flip : 0u));
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
          x[j][b][0] = sc[b / 2][2 * (b & 1)];
          x[j][b][1] = sc[b / 2][2 * (b & 1) + 1];
        }
      }
      if (!whole) {
#pragma unroll
        for (int b = 0; b < RB; ++b) {
          const int lim = seen(row0 + min(8 * b + g, n_rows - 1));
#pragma unroll
          for (int j = 0; j < 2 * kHalves; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (key0 + 8 * j + 2 * t + e >= lim || kd[j >> 1] == -1.f) x[j][b][e] = -INFINITY;
        }
      }
      bool calm = true;
      float top[RB], c_of[RB][kHalves];
#pragma unroll
      for (int b = 0; b < RB; ++b) {
        top[b] = -INFINITY;
#pragma unroll
        for (int i = 0; i < kHalves; ++i) {
          c_of[b][i] = fmaxf(c_row[b] * kd[i], 0x1p-126f);       // above zero: a masked -inf stays one
          top[b] = fmaxf(top[b], fmaf(fmaxf(fmaxf(x[2 * i][b][0], x[2 * i][b][1]), fmaxf(x[2 * i + 1][b][0], x[2 * i + 1][b][1])), c_of[b][i], lv[i]));
        }
        calm = calm && !(top[b] > m_row[b] + kRaiseBy);
      }
      if (!__all_sync(0xffffffffu, calm)) {
#pragma unroll
        for (int b = 0; b < RB; ++b) {
          float mx = fmaxf(top[b], __shfl_xor_sync(0xffffffffu, top[b], 1));
          mx = fmaxf(fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2)) - kHeadroom, m_row[b]);
          const float nm_new = mx == -INFINITY ? 0.f : -mx;
          const float alpha = to_reference(m_row[b], -nm_new, l_row[b]);
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
      // 2^(x_j - m) for the denominators, P_j = 2^(x_j - m) dv.  (The first from the second, by 1 / dv, would be lost where dv is so small that P_j
      // is nothing beside what other pages add to O.)
      uint32_t pb[RB][2 * kHalves];
#pragma unroll
      for (int b = 0; b < RB; ++b) {
#pragma unroll
        for (int i = 0; i < kHalves; ++i) {
          float p[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) p[e] = ex2_approx(fmaf(x[2 * i + e / 2][b][e & 1], c_of[b][i], nm[b]));
          l_row[b] += (p[0] + p[1]) + (p[2] + p[3]);
          pb[b][2 * i] = pack_half2(p[0] * dv[i], p[1] * dv[i]);
          pb[b][2 * i + 1] = pack_half2(p[2] * dv[i], p[3] * dv[i]);
        }
      }
      if (!whole && least < vis && key0 + kStepKeys > least) {      // only some rows see all these keys
#pragma unroll 1
        for (int i = lane; i < C::kBlocks * C::kTile / 16; i += 32) {
          const int row = W == 64 ? ((16 * i) ^ ((i & 32) ? flip : 0u)) >> 6 : (i >> 3) % kStepKeys;
          if (key0 + row >= vis || (kHalves > 1 && row >= 16 ? kd[1] : kd[0]) == -1.f) continue;
          uint4 v = ld_shared16(sv + 16 * i);
          if (drop_specials<kE5M2>(v)) {
            s_special[warp] = true;
            st_shared_v4(sv + 16 * i, v.x, v.y, v.z, v.w);
            fence_proxy_async_smem();                     // before the next copy to this place
          }
        }
        __syncwarp();
      }
#pragma unroll
      for (int blk = 0; blk < C::kBlocks; ++blk) {
        uint32_t vr[4 * kHalves][C::kVWords];
#pragma unroll
        for (int i = 0; i < 4 * kHalves; ++i) {
          const int row = 16 * (i >> 2) + 8 * ((i >> 1) & 1) + 2 * t + (i & 1);
          if constexpr (W == 64) {
            const uint2 v = ld_shared8(sv + ((row * 64 + (((g >> 1) ^ ((row >> 1) & 3)) << 4) + 8 * (g & 1)) ^ ((i & 2) ? flip : 0u)));
            vr[i][0] = v.x; vr[i][1] = v.y;
          } else {
            const uint4 v = ld_shared16(sv + blk * C::kTile + row * 128 + ((g ^ (row & 7)) << 4));
            vr[i][0] = v.x; vr[i][1] = v.y; vr[i][C::kVWords - 2] = v.z; vr[i][C::kVWords - 1] = v.w;
          }
          // nothing of keys that do not count, not even a NaN or an infinity times zero
          if (!whole && (key0 + row >= vis || kd[i >> 2] == -1.f)) {
#pragma unroll
            for (int w = 0; w < C::kVWords; ++w) vr[i][w] = 0u;
          }
        }
#pragma unroll
        for (int w = 0; w < C::kVWords; ++w) {
#pragma unroll
          for (int u = 0; u < kHalves; ++u) {
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
      if (step + C::kStages < last) {
        advance(step + C::kStages);
        copy(step + C::kStages, stage);
        put_scales(step + C::kStages, stage);
        __syncwarp();
      }
      if (++stage == C::kStages) {
        stage = 0;
        phase ^= 1u;
      }
    }
    if (pos >= end) break;

    // ---- what the segment gave ----
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      l_row[b] += __shfl_xor_sync(0xffffffffu, l_row[b], 1);
      l_row[b] += __shfl_xor_sync(0xffffffffu, l_row[b], 2);
    }
    const bool alone = !kLone && step0 == 0 && step1 == steps;           // the item is this warp's
    // this is not its last segment
    const bool more = !kLone && item_end < end && end - item_end > kStartUnits;
    // Where the sums go: to O; to the ring, which is idle once the last segment is through, to be put together with those of the
    // CTA's other warps; or, of a first segment that others began, to the workspace.
    float* part = nullptr;
    int part_row = C::kORow;
    if (!alone) {
      if (more) {
        part_row = D;
        part = a.partial + (warp == 0 ? 2ll * blockIdx.x : 2ll * gridDim.x + static_cast<int64_t>(blockIdx.x) * kWarps + warp) * (C::kRows * (D + 2));
        head_item = item_at;
        if (warp == 0 && lane == 0) put_record(item_at, s.first, row0, n_rows, h);
      } else {
        part = part_of(warp);
        last_item = item_at;
        single = first;
      }
    }
    float* const part_m = part + C::kRows * part_row;
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      if (t == 0 && 8 * b + g < n_rows) {
        const int r = row0 + 8 * b + g;
        if (alone) {
          if (a.lse != nullptr)
            a.lse[static_cast<int64_t>(s.first + r / a.group) * a.heads_q + h * a.group + r % a.group] =
                l_row[b] == 0.f ? -INFINITY : (m_row[b] + __log2f(l_row[b])) * 0.6931471805599453f;
        } else {
          part_m[8 * b + g] = m_row[b];
          part_m[C::kRows + 8 * b + g] = l_row[b];
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
            float4* const p = reinterpret_cast<float4*>(part + in * part_row + col);
#pragma unroll
            for (int j = 0; j < 2 * C::kTilesPerBlock; j += 4) p[j / 4] = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
          }
        }
      }
    }
    __syncwarp();
    if (s_special[warp]) {
#pragma unroll 1
      for (int in = 0; in < n_rows; ++in) {
        const int r = row0 + in;
        uint16_t* const po = static_cast<uint16_t*>(a.o) + (static_cast<int64_t>(s.first + r / a.group) * a.heads_q + h * a.group + r % a.group) * D;
        write_specials<kE5M2>(a.c, seq, h, max(least / kStepKeys, step0) * kStepKeys, min(seen(r), last * kStepKeys), lane, D, [&](int col, float sum) {
          if (alone) po[col] = with_special(po[col], sum, a.bf16);
          else part[in * part_row + col] += sum;
        });
      }
      __syncwarp();
      s_special[warp] = false;
      __syncwarp();
    }
    if (!more) break;
    pos = item_end;
    first = false;
  }

  if constexpr (kLone) {
    // ---- the item's sum: of this CTA's warps, in the place of warp 0's, then of the cluster ----
    if (lane == 0) s_single[warp] = last_item >= 0;
    __syncthreads();
    const int n_rows = min(a.block_tokens * a.group, s.n * a.group - lone_row0);
    for (int i = threadIdx.x; i < n_rows * (W / 4); i += 32 * kWarps) {
      const int r = i / (W / 4), col = 4 * (i % (W / 4));
      if (col >= D) continue;
      float m = -INFINITY, l = 0.f;
      for (int w = 0; w < kWarps; ++w)
        if (s_single[w]) m = fmaxf(m, part_of(w)[C::kRows * C::kORow + r]);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int w = 0; w < kWarps; ++w) {
        if (!s_single[w]) continue;
        const float* p = part_of(w);
        const float mw = p[C::kRows * C::kORow + r];
        float lw = p[C::kRows * C::kORow + C::kRows + r];
        const float f = to_reference(mw, m, lw);
        const float4 x = *reinterpret_cast<const float4*>(p + r * C::kORow + col);
        acc.x += x.x * f; acc.y += x.y * f; acc.z += x.z * f; acc.w += x.w * f;
        l += lw;
      }
      *reinterpret_cast<float4*>(part_of(0) + r * C::kORow + col) = acc;
      if (col == 0) {
        s_m[r] = m;
        s_l[r] = l;
      }
    }
    cg::cluster_group cluster = cg::this_cluster();
    const int n_split = a.n_split;
    if (n_split > 1) cluster.sync();
    else __syncthreads();
    const int rank = static_cast<int>(blockIdx.x) % n_split;
    for (int i = rank * 32 * kWarps + threadIdx.x; i < n_rows * (W / 4); i += n_split * 32 * kWarps) {
      const int r = i / (W / 4), col = 4 * (i % (W / 4));
      if (col >= D) continue;
      float m = -INFINITY, l = 0.f;
      for (int p = 0; p < n_split; ++p) m = fmaxf(m, n_split > 1 ? *cluster.map_shared_rank(s_m + r, p) : s_m[r]);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int p = 0; p < n_split; ++p) {
        const float *po = part_of(0) + r * C::kORow + col, *pm = s_m + r, *pl = s_l + r;
        if (n_split > 1) {
          po = cluster.map_shared_rank(po, p);
          pm = cluster.map_shared_rank(pm, p);
          pl = cluster.map_shared_rank(pl, p);
        }
        float lp = *pl;
        const float f = to_reference(*pm, m, lp);
        const float4 x = *reinterpret_cast<const float4*>(po);
        acc.x += x.x * f; acc.y += x.y * f; acc.z += x.z * f; acc.w += x.w * f;
        l += lp;
      }
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const int row = lone_row0 + r;
      const int64_t at_row = static_cast<int64_t>(s.first + row / a.group) * a.heads_q + lone_head * a.group + row % a.group;
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.o) + at_row * D + col) =
          a.bf16 ? make_uint2(pack_pair<true>(acc.x * inv, acc.y * inv), pack_pair<true>(acc.z * inv, acc.w * inv))
                 : make_uint2(pack_pair<false>(acc.x * inv, acc.y * inv), pack_pair<false>(acc.z * inv, acc.w * inv));
      if (a.lse != nullptr && col == 0) a.lse[at_row] = l == 0.f ? -INFINITY : (m + __log2f(l)) * 0.6931471805599453f;
    }
    if (n_split > 1) cluster.sync();                       // no CTA leaves while its shared memory is read
    return;
  }

  // ---- items that several of the CTA's warps shared ----
  // All threads go through them: the last segment of the warp that has an item's first part here, those of the warps after it while
  // they had no other, and the first segment of a warp that had several.
  if (lane == 0) {
    s_last[warp] = last_item;
    s_head[warp] = head_item;
    s_single[warp] = single;
    if (last_item >= 0) {                                  // `s` and `steps` are those of the last segment
      const int units = item_units(a, steps), item = (last_item - at) / units, rb = item / a.c.heads;
      s_item[warp] = {s.first, rb * C::kRows, min(C::kRows, s.n * a.group - rb * C::kRows), item - rb * a.c.heads,
                      last_item + kStartUnits >= cta_lo, last_item + units <= cta_hi};
    }
  }
  __syncthreads();
  // lane x holds what warp x has
  const int last_of = lane < kWarps ? s_last[lane] : -1, head_of = lane < kWarps ? s_head[lane] : -1;
  const bool single_of = lane < kWarps && s_single[lane];
  const uint32_t with_parts = __ballot_sync(0xffffffffu, last_of >= 0 || head_of >= 0), before = with_parts & ((1u << lane) - 1u);
  const int previous = __shfl_sync(0xffffffffu, last_of, before != 0u ? 31 - __clz(before) : lane);
  uint32_t starts = __ballot_sync(0xffffffffu, last_of >= 0 && !(single_of && before != 0u && previous == last_of));
  for (; starts != 0u; starts &= starts - 1u) {
    const int w = __ffs(starts) - 1, item = __shfl_sync(0xffffffffu, last_of, w);
    const uint32_t members = __ballot_sync(0xffffffffu, last_of == item && lane >= w && (lane == w || single_of));
    const uint32_t heads = __ballot_sync(0xffffffffu, head_of == item && lane > w);
    const Segment it = s_item[w];
    if (!it.begins && it.ends && threadIdx.x == 0) put_record(item, it.first, it.row0, it.n_rows, it.head);
    float* const part = a.partial + (2ll * blockIdx.x + (it.begins ? 1 : 0)) * (C::kRows * (D + 2));
    const float* const head = a.partial + (2ll * gridDim.x + static_cast<int64_t>(blockIdx.x) * kWarps + (__ffs(heads) - 1)) * (C::kRows * (D + 2));
    for (int i = threadIdx.x; i < it.n_rows * (W / 4); i += 32 * kWarps) {
      const int r = i / (W / 4), col = 4 * (i % (W / 4));
      if (col >= D) continue;
      float mw[kWarps], mh = -INFINITY, lh = 0.f, m = -INFINITY, l = 0.f;
      uint4 u = make_uint4(0u, 0u, 0u, 0u);
      if (heads != 0u) {
        mh = ld_global(head + C::kRows * D + r);
        lh = ld_global(head + C::kRows * (D + 1) + r);
        u = ld_global(reinterpret_cast<const uint4*>(head + r * D + col));
      }
#pragma unroll
      for (int x = 0; x < kWarps; ++x) mw[x] = members >> x & 1u ? part_of(x)[C::kRows * C::kORow + r] : -INFINITY;
#pragma unroll
      for (int x = 0; x < kWarps; ++x) m = fmaxf(m, mw[x]);
      m = fmaxf(m, mh);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      auto add = [&](float mx, float lx, const float4& v) {
        const float f = to_reference(mx, m, lx);
        acc.x += v.x * f; acc.y += v.y * f; acc.z += v.z * f; acc.w += v.w * f;
        l += lx;
      };
#pragma unroll
      for (int x = 0; x < kWarps; ++x) {
        if (!(members >> x & 1u)) continue;
        const float* p = part_of(x);
        add(mw[x], p[C::kRows * C::kORow + C::kRows + r], *reinterpret_cast<const float4*>(p + r * C::kORow + col));
      }
      add(mh, lh, make_float4(__uint_as_float(u.x), __uint_as_float(u.y), __uint_as_float(u.z), __uint_as_float(u.w)));
      if (it.begins && it.ends) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const int row = it.row0 + r, token = row / a.group;
        const int64_t at_row = static_cast<int64_t>(it.first + token) * a.heads_q + it.head * a.group + (row - token * a.group);
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.o) + at_row * D + col) =
            a.bf16 ? make_uint2(pack_pair<true>(acc.x * inv, acc.y * inv), pack_pair<true>(acc.z * inv, acc.w * inv))
                   : make_uint2(pack_pair<false>(acc.x * inv, acc.y * inv), pack_pair<false>(acc.z * inv, acc.w * inv));
        if (a.lse != nullptr && col == 0) a.lse[at_row] = l == 0.f ? -INFINITY : (m + __log2f(l)) * 0.6931471805599453f;
      } else {
        *reinterpret_cast<float4*>(part + r * D + col) = acc;
        if (col == 0) {
          part[C::kRows * D + r] = m;
          part[C::kRows * (D + 1) + r] = l;
        }
      }
    }
  }
}

// Items that several CTAs shared, by the record of the last of them: a warp to a row (token and query head).
constexpr int kCombineWarps = 4;
__global__ void __launch_bounds__(32 * kCombineWarps) kv_combine_kernel(const KvAttendArgs a, int rows) {
  start_after_predecessor();
  let_successor_start();
  const int lane = threadIdx.x & 31, in = static_cast<int>(blockIdx.y) * kCombineWarps + (threadIdx.x >> 5);
  const int* const rec = reinterpret_cast<const int*>(a.records + blockIdx.x);
  const uint4 r4 = ld_global(reinterpret_cast<const uint4*>(rec));
  const int h = ld_int(rec + 4), c0 = static_cast<int>(r4.x), c1 = blockIdx.x;
  if (c0 < 0 || in >= static_cast<int>(r4.w)) return;
  const int r = static_cast<int>(r4.z) + in, token = r / a.group;
  const int64_t row = static_cast<int64_t>(r4.y + token) * a.heads_q + h * a.group + (r - token * a.group);
  const int D = a.c.head_dim;
  // the item begins at the end of share c0 and goes on at the beginning of the next
  auto part_of = [&](int c) { return a.partial + (2ll * c + (c == c0 ? 1 : 0)) * (rows * (D + 2)); };
  const int quads = D >> 2;                               // a lane has quads lane and lane + 32
  float m = -INFINITY, l = 0.f;
  float4 acc[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
  constexpr int kAt = 8;                                  // parts at a time, all loads of which go out together
  for (int c = c0; c <= c1; c += kAt) {
    float mp[kAt], lp[kAt];
    uint4 v[kAt][2];
#pragma unroll
    for (int i = 0; i < kAt; ++i) {
      mp[i] = -INFINITY;
      lp[i] = 0.f;
      v[i][0] = v[i][1] = make_uint4(0u, 0u, 0u, 0u);
      if (c + i <= c1) {
        const float* p = part_of(c + i);
        mp[i] = ld_global(p + rows * D + in);
        lp[i] = ld_global(p + rows * (D + 1) + in);
        if (lane < quads) v[i][0] = ld_global(reinterpret_cast<const uint4*>(p + in * D) + lane);
        if (lane + 32 < quads) v[i][1] = ld_global(reinterpret_cast<const uint4*>(p + in * D) + lane + 32);
      }
    }
    float top = m;
#pragma unroll
    for (int i = 0; i < kAt; ++i) top = fmaxf(top, mp[i]);
    const float back = to_reference(m, top, l);
    m = top;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      acc[k].x *= back; acc[k].y *= back; acc[k].z *= back; acc[k].w *= back;
    }
#pragma unroll
    for (int i = 0; i < kAt; ++i) {
      const float f = to_reference(mp[i], m, lp[i]);
      l += lp[i];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        acc[k].x += __uint_as_float(v[i][k].x) * f; acc[k].y += __uint_as_float(v[i][k].y) * f;
        acc[k].z += __uint_as_float(v[i][k].z) * f; acc[k].w += __uint_as_float(v[i][k].w) * f;
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
int warps_of(const KvAttendSizes& z) {
  const int rows = block_rows(z);
  switch (width_of(z.head_dim)) {
    case 64: return rows == 8 ? ACfg<64, 1>::kWarps : (rows == 16 ? ACfg<64, 2>::kWarps : ACfg<64, 4>::kWarps);
    case 128: return rows == 8 ? ACfg<128, 1>::kWarps : (rows == 16 ? ACfg<128, 2>::kWarps : ACfg<128, 4>::kWarps);
    default: return rows == 8 ? ACfg<256, 1>::kWarps : ACfg<256, 2>::kWarps;
  }
}

int step_keys_of(const KvAttendSizes& z) { return kv_step_keys(width_of(z.head_dim), block_rows(z)); }

// A cluster to an item (no second kernel, no workspace) where that leaves no CTA more than kLoneKeys keys, going by what the page
// table can hold; CTAs of the cluster, or 0.  Clusters of a launch are to run at once: as a cluster lies within a part of the GPU of
// 16 to 20 SMs, and a CTA takes an SM, no more than one of eight per sixteen SMs is counted on (sixteen of them: 27 us, where eight
// take 14 and 32 of four 15: B1 H32 Hk8 D128, 1000 keys), and of four as many as fill seven eighths of the SMs.
constexpr int64_t kLoneKeys = 1024;
int lone_split(const KvAttendSizes& z, int sms) {
  const int group = z.heads_q / z.heads, rows = block_rows(z);
  if (group > rows) return 0;
  const int64_t items = kv_slots(z.batch, z.tokens, z.tokens / z.batch, z.ragged, rows / group, 1) * z.heads;
  const int64_t steps = (z.keys_most + step_keys_of(z) - 1) / step_keys_of(z);
  int split = 1;
  for (const int n : {2, 4, 8})
    if (n * items <= (n == 8 ? sms / 2 : (n == 4 ? sms * 7 / 8 : sms)) && n / 2 * warps_of(z) < steps) split = n;
  return z.keys_most <= kLoneKeys * split && items <= 2 * sms ? split : 0;
}

template <int W, int RB, bool kE5M2, bool kLone>
cudaError_t launch_attend(const CUtensorMap& tk, const CUtensorMap& tv, const KvAttendArgs& a, const KvAttendSizes& z, int sms, cudaStream_t stream) {
  using C = ACfg<W, RB>;
  auto kernel = &kv_attend_kernel<W, RB, kE5M2, kLone>;
  static std::atomic<bool> ready[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const bool cached = dev >= 0 && dev < 64;
  if (!cached || !ready[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e != cudaSuccess) return e;
    if (cached) ready[dev].store(true, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg{};
  cfg.blockDim = dim3(32 * C::kWarps, 1, 1);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2] = {overlap_attribute()};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (kLone) {
    const int64_t items = kv_slots(z.batch, z.tokens, z.tokens / z.batch, z.ragged, a.block_tokens, 1) * z.heads;
    cfg.gridDim = dim3(static_cast<unsigned>(items * a.n_split), 1, 1);
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(a.n_split);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = a.n_split > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, tk, tv, a);
  }
  cfg.gridDim = dim3(static_cast<unsigned>(sms), 1, 1);
  e = cudaLaunchKernelEx(&cfg, kernel, tk, tv, a);
  if (e != cudaSuccess) return e;
  cfg.gridDim = dim3(static_cast<unsigned>(sms), C::kRows / kCombineWarps, 1);
  cfg.blockDim = dim3(32 * kCombineWarps, 1, 1);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, &kv_combine_kernel, a, C::kRows);
}

template <int W, int RB>
cudaError_t launch_rows(const CUtensorMap& tk, const CUtensorMap& tv, const KvAttendArgs& a, const KvAttendSizes& z, bool e5m2, int sms, cudaStream_t stream) {
  if (a.n_split > 0)
    return e5m2 ? launch_attend<W, RB, true, true>(tk, tv, a, z, sms, stream) : launch_attend<W, RB, false, true>(tk, tv, a, z, sms, stream);
  return e5m2 ? launch_attend<W, RB, true, false>(tk, tv, a, z, sms, stream) : launch_attend<W, RB, false, false>(tk, tv, a, z, sms, stream);
}

int64_t records_bytes(int sms) { return (static_cast<int64_t>(sms) * sizeof(KvRecord) + 255) / 256 * 256; }

}  // namespace

int kv_attend_step_keys(const KvAttendSizes& z) { return step_keys_of(z); }

int64_t kv_attend_workspace(const KvAttendSizes& z, int sms) {
  if (lone_split(z, sms) > 0) return 0;
  const int64_t slots = static_cast<int64_t>(sms) * (2 + warps_of(z));
  return records_bytes(sms) + slots * block_rows(z) * (z.head_dim + 2) * 4;
}

cudaError_t launch_kv_attend(const CUtensorMap& tk, const CUtensorMap& tv, KvAttendArgs a, const KvAttendSizes& z, void* workspace, bool e5m2, int sms,
                             cudaStream_t stream) {
  a.records = static_cast<KvRecord*>(workspace);
  a.partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + records_bytes(sms));
  const int rows = block_rows(z);
  a.n_split = lone_split(z, sms);
  // units of all items together are a 31-bit number
  const int step_keys = step_keys_of(z);
  const double items = (static_cast<double>(z.tokens) * a.group / rows + z.batch) * z.heads;
  a.unit_shift = 0;
  while (items * ((static_cast<double>(z.keys_most) / step_keys) / (1 << a.unit_shift) + 2 + kStartUnits) > 1e9 && a.unit_shift < 30) ++a.unit_shift;
  a.block_tokens = rows / a.group;
  switch (width_of(a.c.head_dim)) {
    case 64:
      return rows == 8 ? launch_rows<64, 1>(tk, tv, a, z, e5m2, sms, stream)
                       : (rows == 16 ? launch_rows<64, 2>(tk, tv, a, z, e5m2, sms, stream) : launch_rows<64, 4>(tk, tv, a, z, e5m2, sms, stream));
    case 128:
      return rows == 8 ? launch_rows<128, 1>(tk, tv, a, z, e5m2, sms, stream)
                       : (rows == 16 ? launch_rows<128, 2>(tk, tv, a, z, e5m2, sms, stream) : launch_rows<128, 4>(tk, tv, a, z, e5m2, sms, stream));
    default:
      return rows == 8 ? launch_rows<256, 1>(tk, tv, a, z, e5m2, sms, stream) : launch_rows<256, 2>(tk, tv, a, z, e5m2, sms, stream);
  }
}

}  // namespace fa8
