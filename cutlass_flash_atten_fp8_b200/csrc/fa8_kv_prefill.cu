// Attention of many new tokens' queries over the pages of the fp8 cache (prompts, pieces of prompts), sm_100a.
//
// The formulas and the treatment of scales are those of fa8_kv_attend.cu; here a K/V head's query rows come in tiles of 128, and both
// products run on the tensor cores in fp16 with fp32 accumulators in tensor memory (tcgen05.mma kind::f16): fp8 products would
// need P, and Q, rounded to three bits.  What bounds it: per 128 keys and tile 1024 cycles of products and 1024 of
// exponentials (16 per cycle and SM) at head dim 128, and shared memory: widening a tile of K or V moves as many bytes as a product reads.
//
// A CTA per SM, warps with roles, work items of two tiles (one at head dims above 128) of one sequence and K/V head:
//   producer   looks up items and pages, copies K and V tiles of kN keys from the pages (fp8) into shared memory
//   widening   four warps turn a tile into fp16, in the layout that the products want, times the power of two by which its pages' scales
//              differ from the item's first page; keys past the last one become zeros (a NaN or an infinity there must not meet a zero P).  Eight warps
//              were no faster (330 us for 1024 tokens over 16384 keys where four took 322)
//   issuer     one thread: S = Q K^T into tensor memory, O += P V with P from tensor memory
//   softmax    eight warps a tile, two to 32 rows (four, a row to a thread, took 26 % longer): each has half of a block's keys, P = 2^(c s - m) over
//              S as it lies, and at the end half of O's columns
// Two tiles keep the tensor cores and the exponentials busy in turns; at head dims above 128 O takes half of tensor memory
// and the one tile has two score buffers instead.
//
// The row reference m lies 6 below the maximum over the item's first kN keys, so that P, at 2^6, has its full precision twenty
// binades down, and is raised, and O rescaled, when the sum of P over half a block nears fp16's largest number.  Scales that differ by
// more than fp16 can take in, or are no powers of two, go through a slower form of the softmax that multiplies them in (`residual`).
//
// Measured: 1024 tokens, 32 heads over 8, over 16384 keys, head dim 128: 323 us, 824 TFLOP/s, half of what a plain fp16 product
// reaches on this GPU; four prompts of 4096: 451 us.  A block of 128 keys takes some 4000 cycles for two tiles where the tensor cores are busy for
// 2048: a tile's chain S, softmax (1024 cycles of exponentials alone, 2350 beside the other tile's), P V is longer than the other tile's
// work.  A quarter of the exponentials by a polynomial instead gained 2 % and was left out.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "fa8_kernel.h"
#include "fa8_kv.h"
#include "kv_common.cuh"
#include "kv_turns.h"

namespace fa8 {

namespace {

constexpr int kTileM = 128;
constexpr uint32_t kTmemCols = 512;
constexpr unsigned long long kLimitNs = 2000000000ull;
constexpr float kRaiseAbove = 60000.f;   // below fp16's largest number
constexpr float kHeadroom = 6.f;         // a fresh reference puts the row's largest P at 2^6: fp16 is exact to half a step down to 2^-14
constexpr float kLog2Least = -80.f;      // see fa8_kv_attend.cu
constexpr int kItemSlots = 4;
constexpr int kBlockSlots = 8;           // blocks whose residual scales are kept: the producer is at most four ahead of the softmax

template <int W>
struct PCfg {
  static constexpr int kTiles = W == 256 ? 1 : 2;
  static constexpr int kN = W == 256 ? 64 : 128;               // keys of a block
  // Score buffers, which the blocks of both tiles take in turn: what tensor memory holds beside O.  The scores go out as many turns ahead, one more
  // than the item's tiles at most (kv_turns.h), so a tile whose turn it is finds its next scores ready when there are more buffers than tiles: 8 prompts of 2048 at
  // head dim 64 took 340 us with two, 311 with three (305 since).  (Four of 64 keys would do that at head dim 128, but a product of N = 64 is
  // bound by reading Q from shared memory: 80 cycles a step of 16 against 64 for N = 128.)
  static constexpr int kBufs = W == 64 ? 3 : 2;
  static constexpr int kGroups = kN / 16;                      // of keys that share a page
  static constexpr int kCols = W / 64;                         // column blocks of 64 fp16 (128 bytes)
  static constexpr int kRawRow = W < 128 ? W : 128;            // bytes of a row of a raw (fp8) tile
  static constexpr int kRawBlocks = W / kRawRow;
  static constexpr int kRawBlockBytes = kN * kRawRow;
  static constexpr int kRawBytes = kN * W;
  static constexpr int kRaw = W == 64 ? 4 : 2;                 // raw tiles
  static constexpr int kRing = 4;                              // widened tiles
  static constexpr int kRingBytes = kN * W * 2;
  static constexpr int kQBytes = kTileM * W * 2;               // of a tile
  // Columns of tensor memory: the score buffers (P over them), then O of each tile.
  static constexpr int kOCol = kN * kBufs;
  static constexpr int kSoftWarps = 8 * kTiles;
  static constexpr int kWideWarp0 = kSoftWarps;
  static constexpr int kLoadWarp = kWideWarp0 + 4;
  static constexpr int kMmaWarp = kLoadWarp + 1;
  // Whole warpgroups (two warps stand by), so that registers can be dealt out anew: 512 * 96 + 128 * 48 + 128 * 48 = 768 * 80.  (A thread of
  // the softmax holds 32 scores and 32 pairs of P beside its row: with 88 registers 328 us for 1024 tokens over 16384 keys, 320 with 96.)
  static constexpr bool kDeal = kTiles == 2;
  static constexpr int kThreads = 32 * (kLoadWarp + 4);
  static constexpr uint32_t kSoftRegs = 96, kWideRegs = 48, kOtherRegs = 48;
  static_assert(!kDeal || 32 * kSoftWarps * kSoftRegs + 128 * (kWideRegs + kOtherRegs) <= kThreads * 80, "registers of the launch");
  static constexpr int kRawOffset = kTiles * kQBytes;
  static constexpr int kRingOffset = kRawOffset + kRaw * kRawBytes;
  static constexpr int kSharedOffset = kRingOffset + kRing * kRingBytes;
  static_assert(kOCol + W * kTiles <= 512, "tensor memory");
};

struct Item {
  int seq, head;
  int first, n, len;                     // of the sequence
  int token0, n_tokens;                  // its new tokens in the item
  int blk0, blk1;                        // key blocks
  int vis;                               // keys that the item's last row sees
  int part;                              // of its keys; -1: all of them
};

template <int W>
struct Shared {
  using C = PCfg<W>;
  uint64_t item_full[kItemSlots], item_empty[kItemSlots];
  uint64_t raw_full[C::kRaw], raw_empty[C::kRaw];
  uint64_t ring_full[C::kRing], ring_empty[C::kRing];
  uint64_t s_full[2][2], p_full[C::kBufs];       // by tile and turn, by buffer: kv_turns.h
  uint64_t q_full[2], o_done[2], o_final[2];     // by tile
  uint64_t blk_full[kBlockSlots];
  uint64_t drain, given;
  uint4 answer;                          // to the request for another CTA's item
  Item item[kItemSlots];                 // seq < 0: no more
  int with_special_v[kItemSlots];        // NaNs or infinities of V of keys that only some of the item's rows see were taken out (drop_specials)
  uint32_t factor[C::kRaw][C::kGroups];  // fp16 pair to multiply a group of 16 keys by
  int valid[C::kRaw];                    // rows of the tile that are keys
  int complete[C::kRaw];                 // all are, and of pages that exist
  float residual[kBlockSlots][2][C::kGroups];   // of K and V; K's is -1 for a group without a page
  float ref[kBlockSlots][2];             // reference scales of the item that the block is of
  int flagged[kBlockSlots];              // some residual is not 1
  float row[2][kTileM];                  // by tile and row, between the two warps that have it: what Q was divided by, maxima, sums
  uint32_t tmem;
  int abort;
};

struct Wait {
  volatile int* abort;
  int* status;
  volatile int* host_status;
};
// (Not in line: there are two dozen waits, and the two status words would be held in registers for them.  In line, four prompts of 4096
// at head dim 128 took 478 us and 1024 tokens over 16384 keys 327; so they take 452 and 323.)
__device__ __noinline__ void give_up(const Wait& w, int code) {
  *w.abort = 1;
  report_expired_wait(w.status, w.host_status, code);
}
__device__ __forceinline__ bool wait_bounded(const Wait& w, uint64_t* barrier, uint32_t parity, int code) {
  const uint32_t bar = smem_u32(barrier);
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = global_timer_ns();
  uint32_t spins = 0;
  while (true) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((++spins & 31u) == 0) {
      if (*w.abort) return false;
      if (global_timer_ns() - t0 > kLimitNs) {
        give_up(w, code);
        return false;
      }
    }
  }
}

// Takes over the work of a CTA of this grid that has not started (there is one to an item): the answer arrives at `bar`.
__device__ __forceinline__ void ask_for_cta(uint32_t answer, uint32_t bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(answer), "r"(bar) : "memory");
}
// Its number, or -1: all have started or been taken, and there must be no further request.
__device__ __forceinline__ int taken_cta(uint32_t answer) {
  uint32_t id;
  asm volatile("{\n\t.reg .pred p;\n\t.reg .b128 a;\n\tld.shared.b128 a, [%1];\n\t"
               "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, a;\n\tmov.u32 %0, 0xffffffff;\n\t"
               "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, a;\n\t}" : "=r"(id) : "r"(answer) : "memory");
  return static_cast<int>(id);
}

// kind::f16 products: D[tmem] (+)= A B, fp16 operands, fp32 sums.
__device__ __forceinline__ void mma_f16_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n"
               ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n"
               ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
// Shared-memory matrix descriptors, 128-byte swizzle: low word (address, leading offset) and high word (stride offset 1024 bytes
// between groups of eight rows, version 1, swizzle mode 2), all in units of 16 bytes.
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t leading) { return ((addr & 0x3ffffu) >> 4) | ((leading >> 4) << 16); }
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint64_t desc(uint32_t lo) { return (static_cast<uint64_t>(kDescHi) << 32) | lo; }
// Instruction descriptor: fp16 x fp16 -> fp32; bit 16: B with its columns (head dim) contiguous.
__host__ __device__ constexpr uint32_t idesc(int n, bool b_mn) {
  return (1u << 4) | (b_mn ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(kTileM >> 4) << 24);
}

__device__ __forceinline__ void st_shared16(uint32_t addr, const uint4& v) { st_shared_v4(addr, v.x, v.y, v.z, v.w); }
__device__ __forceinline__ uint4 ld_shared16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Sixteen fp8 -> fp16, times a pair of factors.
template <bool kE5M2>
__device__ __forceinline__ void widen16(const uint4& x, uint32_t f, uint4& lo, uint4& hi) {
  uint32_t r[8];
  fp8_to_half4<kE5M2>(x.x, r[0], r[1]);
  fp8_to_half4<kE5M2>(x.y, r[2], r[3]);
  fp8_to_half4<kE5M2>(x.z, r[4], r[5]);
  fp8_to_half4<kE5M2>(x.w, r[6], r[7]);
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = hmul2(r[i], f);
  lo = make_uint4(r[0], r[1], r[2], r[3]);
  hi = make_uint4(r[4], r[5], r[6], r[7]);
}

// Parts that an item of n_blk blocks is cut into, at most `most`.
constexpr int kPartBlocks = 4;
__device__ __forceinline__ int parts_of(int n_blk, int most) { return max(1, min(most, n_blk / kPartBlocks)); }

// What the softmax of a row carries from block to block.
struct Row {
  float c;                               // scale_log2 * reference scale of K * what Q was scaled by
  float m, nm, l;                        // reference (log2 units), its negative (0 while there is none), row sum
  float most;                            // sum of P over a half above which the reference is raised: 0 while there is none
  int lim;                               // keys that the row sees
};

// P of 32 keys from their scores s, into pk as fp16 pairs; returns the sum of P and adds that of the denominators to *l.  General:
// keys from `lim` on are masked, the residual scales of the two groups of sixteen keys are multiplied in.
template <bool kGeneral>
__device__ __forceinline__ float exponentials(const uint32_t (&s)[32], float c, float nm, int lim, const float* rk, const float* rv,
                                              uint32_t* pk, float* l) {
  if (kGeneral) {
    float sum = 0.f, sum_l = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float k = rk[h], v = rv[h], ck = c * k;
#pragma unroll
      for (int i = 16 * h; i < 16 * h + 16; i += 2) {
        float x0 = fmaf(__uint_as_float(s[i]), ck, nm), x1 = fmaf(__uint_as_float(s[i + 1]), ck, nm);
        if (i >= lim || k == -1.f) x0 = -INFINITY;
        if (i + 1 >= lim || k == -1.f) x1 = -INFINITY;
        const float e0 = ex2_approx(x0), e1 = ex2_approx(x1), p0 = e0 * v, p1 = e1 * v;
        sum_l += e0 + e1;
        sum += p0 + p1;
        pk[i / 2] = pack_half2(p0, p1);
      }
    }
    *l += sum_l;
    return sum;
  }
  f32x2_t sum[2] = {pack2(0.f, 0.f), pack2(0.f, 0.f)};
  const f32x2_t c2 = pack2(c, c), nm2 = pack2(nm, nm);
#pragma unroll
  for (int i = 0; i < 32; i += 2) {
    float x0, x1;
    unpack2(fma2(pack2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), c2, nm2), x0, x1);
    const float e0 = ex2_approx(x0), e1 = ex2_approx(x1);
    sum[(i >> 1) & 1] = add2(sum[(i >> 1) & 1], pack2(e0, e1));
    pk[i / 2] = pack_half2(e0, e1);
  }
  float a, b;
  unpack2(add2(sum[0], sum[1]), a, b);
  *l += a + b;
  return a + b;
}

// Largest c s + log2(scale of V) of 32 keys.
template <bool kGeneral>
__device__ __forceinline__ float largest(const uint32_t (&s)[32], float c, int lim, const float* rk, const float* rv) {
  float m = -INFINITY;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float x = -INFINITY;
    if (kGeneral) {
      const float k = rk[h];
#pragma unroll
      for (int i = 16 * h; i < 16 * h + 16; ++i)
        if (i < lim && k != -1.f) x = fmaxf(x, __uint_as_float(s[i]) * (c * k));
      m = fmaxf(m, x + fmaxf(__log2f(rv[h]), kLog2Least));
    } else {
#pragma unroll
      for (int i = 16 * h; i < 16 * h + 16; ++i) x = fmaxf(x, __uint_as_float(s[i]));
      m = fmaxf(m, x * c);
    }
  }
  return m;
}

// Columns of tensor memory times alpha.
__device__ __noinline__ void rescale(uint32_t t, int columns, float alpha) {
#pragma unroll 1
  for (int c = 0; c < columns; c += 16) {
    uint32_t x[16];
    tmem_ld_32x32b_x16(t + c, x);
    tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * alpha);
    tmem_st_32x32b_x16(t + c, x);
  }
  tmem_wait_st();
}

template <int W, bool kE5M2>
__global__ void __launch_bounds__(PCfg<W>::kThreads, 1) kv_prefill_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                                                                          const KvAttendArgs a, const KvPrefillPlan plan) {
  using C = PCfg<W>;
  // (No static shared memory, so this lies at a multiple of 1024 bytes, which the swizzled tiles need.)
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t base = smem_u32(smem_raw);
  Shared<W>& sh = *reinterpret_cast<Shared<W>*>(smem_raw + C::kSharedOffset);
  const uint32_t s_q = base, s_raw = base + C::kRawOffset, s_ring = base + C::kRingOffset;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Wait wctx{&sh.abort, a.c.status, a.c.host_status};
  if (threadIdx.x == 0) {
    auto init = [](uint64_t* b, int n, int count) {
      for (int i = 0; i < n; ++i) mbar_init(smem_u32(b + i), count);
    };
    init(sh.item_full, kItemSlots, 1);
    init(sh.item_empty, kItemSlots, C::kSoftWarps + 4 + 1);
    init(sh.raw_full, C::kRaw, 1);
    init(sh.raw_empty, C::kRaw, 4);
    init(sh.ring_full, C::kRing, 4);
    init(sh.ring_empty, C::kRing, 1);
    init(sh.q_full, 2, 8);
    init(&sh.s_full[0][0], 4, 1);
    init(sh.p_full, C::kBufs, 8);
    init(sh.o_done, 2, 1);
    init(sh.o_final, 2, 1);
    init(sh.blk_full, kBlockSlots, 1);
    init(&sh.drain, 1, 1);
    init(&sh.given, 1, 1);
    sh.abort = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  if (warp == C::kLoadWarp && lane == 0) {
    prefetch_tensormap(&tk);
    prefetch_tensormap(&tv);
  }
  if (warp == C::kMmaWarp) {
    tmem_alloc(smem_u32(&sh.tmem), kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  start_after_predecessor();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&sh.tmem);
  if (threadIdx.x == 0 && (base & 1023u) != 0u) {            // never seen; the tiles would be garbage, and it is reported
    sh.abort = 1;
    report_expired_wait(wctx.status, wctx.host_status, 0xb000);
  }

  // rows of 64 bytes lie two to a swizzled line of 128: the halves of every other four lines are exchanged
  const uint32_t flip = W == 64 && a.c.head_dim == 64 ? 64u : 0u;
  const int group = a.group, tile_tokens = kTileM / group;       // a token's rows lie in one tile
  const int over_group = (65536 + group - 1) / group;            // r / group = (r * over_group) >> 16 for r < 128
  // Consumers of the item ring: the next item (false: no more, or a wait ran out).
  int n_items = 0;
  auto next_item = [&](Item& it) {
    const int slot = n_items % kItemSlots;
    if (!wait_bounded(wctx, &sh.item_full[slot], (n_items / kItemSlots) & 1, 0xb100)) return false;
    it = sh.item[slot];
    return true;
  };
  // From the block of this key on NaNs and infinities of V are left to the end: the item's rows do not all see its keys.
  auto apart = [&](const Item& i) { return a.causal ? max(0, min(i.len, i.len - i.n + i.token0 + 1)) / C::kN : 0x7fffffff; };
  auto item_read = [&] { mbar_arrive(smem_u32(&sh.item_empty[n_items++ % kItemSlots])); };

  __syncwarp();
  if (warp >= C::kLoadWarp) {
    if constexpr (C::kDeal) setmaxnreg_dec<C::kOtherRegs>();
    if (warp == C::kLoadWarp) {
      // ---------------------------------------------------------------- producer
      uint32_t tiles = 0, blocks = 0;                              // raw tiles and blocks filled so far
      // once a wait has run out, the CTAs that are still to come have nothing to do
      bool ok = true, more = !wait_has_expired(a.c.status), asked = false;
      auto push = [&](const Item& it) {
        const int slot = n_items % kItemSlots;
        ok = wait_bounded(wctx, &sh.item_empty[slot], ((n_items / kItemSlots) & 1) ^ 1, 0xb200);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) return;
        if (lane == 0) {
          sh.item[slot] = it;
          sh.with_special_v[slot] = 0;
          mbar_arrive(smem_u32(&sh.item_full[slot]));
        }
        ++n_items;
      };
      auto load_item = [&](int64_t id) {
        Item it;
        const int64_t sh_id = id / plan.parts;
        it.part = static_cast<int>(id - sh_id * plan.parts);
        const int64_t slot = sh_id / a.c.heads;
        it.head = static_cast<int>(sh_id - slot * a.c.heads);
        int j;
        kv_find_slot(a.c, slot, plan.block_tokens, 1, &it.seq, &j);
        const KvSeq s = kv_seq(a.c, it.seq);
        const int tiles_of = (s.n + plan.block_tokens - 1) / plan.block_tokens;
        if (j >= tiles_of) return;
        it.first = s.first;
        it.n = s.n;
        it.len = s.len;
        it.token0 = (tiles_of - 1 - j) * plan.block_tokens;
        it.n_tokens = min(plan.block_tokens, s.n - it.token0);
        it.vis = a.causal ? max(0, min(s.len, s.len - s.n + it.token0 + it.n_tokens)) : s.len;
        const int n_blk = max(1, (it.vis + C::kN - 1) / C::kN);
        const int parts = parts_of(n_blk, plan.parts);
        if (it.part >= parts) return;
        it.blk0 = static_cast<int>(static_cast<int64_t>(n_blk) * it.part / parts);
        it.blk1 = static_cast<int>(static_cast<int64_t>(n_blk) * (it.part + 1) / parts);
        if (parts == 1) it.part = -1;
        push(it);
        if (!ok) return;

        // Lane g < kGroups looks after the g-th sixteen keys of a block: page numbers are loaded two blocks ahead, scales one.
        const int* const table = a.c.table + static_cast<int64_t>(it.seq) * a.c.table_stride;
        auto load_page = [&](int blk) {
          const int64_t key = static_cast<int64_t>(blk) * C::kN + 16 * lane;
          return lane < C::kGroups && blk < it.blk1 && key < it.vis ? ld_int(table + (key >> a.c.page_shift)) : -2;
        };
        auto in_pool = [&](int page) { return static_cast<unsigned>(page) < static_cast<unsigned>(a.c.num_pages); };
        auto load_scale = [&](const float* d, int page) { return in_pool(page) ? ld_global(d + static_cast<int64_t>(page) * a.c.heads + it.head) : 1.f; };
        int page = load_page(it.blk0), page1 = load_page(it.blk0 + 1);
        float kd = load_scale(a.c.k_descale, page), vd = load_scale(a.c.v_descale, page);
        // The item's reference scales: its first page's, or 1 where that is so far out that another page's, from 2^-64 to 2^64, might be
        // infinite or nothing relative to it; times what keeps e5m2 (up to 2^15.8) away from fp16's ends.
        const float margin = kE5M2 ? 16.f : 1.f;
        auto reference = [&](float d) {
          d = __shfl_sync(0xffffffffu, d, 0);
          return (d >= 0x1p-32f && d <= 0x1p32f ? d : 1.f) * margin;
        };
        const float kref = reference(kd), vref = reference(vd);
        for (int blk = it.blk0; blk < it.blk1 && ok; ++blk) {
          const int page2 = load_page(blk + 2);
          const float kd1 = load_scale(a.c.k_descale, page1), vd1 = load_scale(a.c.v_descale, page1);
          const bool here = in_pool(page);
          if (!here && page != -2) report_bad_index(a.c);
          // factor 2^e that fp16 takes in exactly: e4m3 2^-15 ... 2^7, e5m2 2^-8 ... 1; the rest is residual
          auto split = [&](float d, float ref, float* rest) {
            const float f = d / ref;
            const uint32_t bits = __float_as_uint(f);
            const int e = static_cast<int>(bits >> 23) - 127;
            const bool exact = (bits & 0x7fffffu) == 0 && e >= (kE5M2 ? -8 : -15) && e <= (kE5M2 ? 0 : 7);
            const float take = exact ? f : (kE5M2 ? 0x1p-4f : 1.f);
            *rest = exact ? 1.f : d / ref / take;
            const uint32_t h = pack_half2(take, take);
            return h;
          };
          const uint32_t n = blocks % kBlockSlots;
          float rk = 1.f, rv = 1.f;
          const uint32_t fk = split(kd, kref, &rk), fv = split(vd, vref, &rv);
          if (!here) {
            rv = 1.f;
            rk = page == -2 ? 1.f : -1.f;                          // past the last key: masked by the row's limit
          }
          if (lane < C::kGroups) {
            sh.residual[n][0][lane] = rk;
            sh.residual[n][1][lane] = rv;
          }
          const bool flagged = __any_sync(0xffffffffu, lane < C::kGroups && (rk != 1.f || rv != 1.f));
          if (lane == 0) {
            sh.ref[n][0] = kref;
            sh.ref[n][1] = vref;
            sh.flagged[n] = flagged;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&sh.blk_full[n]));
          ++blocks;
          // one copy per page part of the block (box_keys keys) and 128 columns
          const int box_keys = min(1 << a.c.page_shift, kv_prefill_copy_keys(W));
          const bool issues = here && (16 * lane) % box_keys == 0;
          const int boxes = __popc(__ballot_sync(0xffffffffu, issues));
          const bool all_here = __all_sync(0xffffffffu, here || lane >= C::kGroups);
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            const int st = tiles % C::kRaw;
            ok = __all_sync(0xffffffffu, wait_bounded(wctx, &sh.raw_empty[st], ((tiles / C::kRaw) & 1) ^ 1, 0xb300 + st));
            if (!ok) break;
            if (lane < C::kGroups) sh.factor[st][lane] = here ? (kv ? fv : fk) : 0u;
            if (lane == 0) {
              sh.valid[st] = max(0, min(C::kN, it.vis - blk * C::kN));
              sh.complete[st] = all_here && it.vis >= (blk + 1) * C::kN;
            }
            __syncwarp();
            const uint32_t bar = smem_u32(&sh.raw_full[st]);
            if (lane == 0) mbar_arrive_expect_tx(bar, boxes * box_keys * C::kRawRow * C::kRawBlocks);
            __syncwarp();
            if (issues) {
              const int row = ((blk * C::kN + 16 * lane) & ((1 << a.c.page_shift) - 1)) >> (flip ? 1 : 0);
#pragma unroll
              for (int b = 0; b < C::kRawBlocks; ++b)
                tma_load_3d(s_raw + st * C::kRawBytes + b * C::kRawBlockBytes + 16 * lane * C::kRawRow, kv ? &tv : &tk, bar, 128 * b, row,
                            page * a.c.heads + it.head);
            }
            ++tiles;
          }
          page = page1;
          page1 = page2;
          kd = kd1;
          vd = vd1;
        }
      };
      uint32_t answers = 0;
      // A CTA to an item is launched; those on the GPU take over the others, one after another, as they get through their own, so that
      // all end together whatever the items' lengths (dealt out in turns, 148 CTAs differed by a fifth at 2048 and 4096 new tokens).
      for (int64_t id = blockIdx.x; ok && more;) {
        if (id == 0)                                               // a bad range has no rows that would find it
          for (int b = lane; b < a.c.batch; b += 32)
            if (kv_seq(a.c, b).bad) report_bad_index(a.c);
        load_item(id);
        // One item waits while one is worked on, no more: others may be through before.
        if (ok && n_items > 0) ok = wait_bounded(wctx, &sh.item_empty[(n_items - 1) % kItemSlots], ((n_items - 1) / kItemSlots) & 1, 0xb200);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0) {
          fence_proxy_async_smem();                                // the last answer has been read
          mbar_arrive_expect_tx(smem_u32(&sh.given), 16);
          ask_for_cta(smem_u32(&sh.answer), smem_u32(&sh.given));
        }
        asked = true;
        ok = __all_sync(0xffffffffu, wait_bounded(wctx, &sh.given, answers & 1, 0xb210));
        if (!ok) break;
        asked = false;
        ++answers;
        id = taken_cta(smem_u32(&sh.answer));
        more = id >= 0;
        __syncwarp();
      }
      if (ok) {
        Item none{};
        none.seq = -1;
        push(none);
      }
      if (!ok) {
        // copies in flight, and an answer, land before the CTA's memory is given back (a wait each, with a limit)
        if (asked) {
          const uint64_t t0 = global_timer_ns();
          while (!mbar_try_wait(smem_u32(&sh.given), answers & 1) && global_timer_ns() - t0 < 20000000ull) {}
        }
        for (uint32_t i = tiles > C::kRaw ? tiles - C::kRaw : 0; i < tiles; ++i) {
          const uint64_t t0 = global_timer_ns();
          while (!mbar_try_wait(smem_u32(&sh.raw_full[i % C::kRaw]), (i / C::kRaw) & 1) && global_timer_ns() - t0 < 20000000ull) {}
        }
      }
    } else if (warp == C::kMmaWarp) {
      // ---------------------------------------------------------------- issuer
      if (elect_one()) {
        constexpr uint32_t kIdescQK = idesc(C::kN, false), kIdescPV = idesc(W, true);
        constexpr uint32_t kColQ = kTileM * 128 / 16, kColK = C::kN * 128 / 16;     // column blocks of Q and K in 16 bytes
        const uint32_t q_lo = desc_lo(s_q, 16), k_lo = desc_lo(s_ring, 16), v_lo = desc_lo(s_ring, C::kN * 128);
        bool ok = true;
        uint32_t ld = 0;                                           // widened tiles used so far: K, V, K, V ...
        uint32_t qn[2] = {0, 0};                                   // q_full phases by tile
        uint32_t turns = 0;                                        // of the score buffers, before this item
        uint32_t scored = 0;                                       // bit i: parity of tile i's own turns whose scores have been issued
        auto ring_wait = [&](uint32_t i) { return wait_bounded(wctx, &sh.ring_full[i % C::kRing], (i / C::kRing) & 1, 0xb400); };
        auto ring_release = [&](uint32_t i) { tc_commit(smem_u32(&sh.ring_empty[i % C::kRing])); };
        auto issue_qk = [&](int tile, uint32_t b, uint32_t i) {
          const uint32_t kk = k_lo + (i % C::kRing) * (C::kRingBytes / 16), qq = q_lo + tile * (C::kQBytes / 16);
#pragma unroll
          for (int k = 0; k < W / 16; ++k)
            mma_f16_ss(tmem + C::kN * b, desc(qq + (k >> 2) * kColQ + 2 * (k & 3)), desc(kk + (k >> 2) * kColK + 2 * (k & 3)), kIdescQK, k > 0);
          tc_commit(smem_u32(&sh.s_full[tile][score_barrier(scored >> tile)]));
          scored ^= 1u << tile;
        };
        auto issue_pv = [&](int tile, uint32_t b, uint32_t i, bool more) {
          const uint32_t vv = v_lo + (i % C::kRing) * (C::kRingBytes / 16);
#pragma unroll
          for (int k = 0; k < C::kN / 16; ++k)
            mma_f16_ts(tmem + C::kOCol + W * tile, tmem + C::kN * b + 8 * k, desc(vv + k * 128), kIdescPV, more || k > 0);
        };
        Item it;
        while (ok && (ok = next_item(it))) {
          item_read();
          if (it.seq < 0) break;
          const int n = it.blk1 - it.blk0;
          const int nt = C::kTiles == 2 && it.n_tokens > tile_tokens ? 2 : 1;
          // Turn t is block t / nt of tile t % nt; the scores run `ahead` turns ahead, into a buffer that P V (t), or one before it, was the last to read.
          const int ahead = turns_ahead<C::kBufs>(nt);
          int tile_v = 0, blk_v = 0, tile_k = 0, blk_k = 0;
          for (int t = -ahead; t < n * nt && ok; ++t) {
            if (t >= 0) {
              const uint32_t turn = turns + t, b = turn_buffer<C::kBufs>(turn), lv = ld + 2 * blk_v + 1;
              if (tile_v == 0) ok = ring_wait(lv);
              if (ok) ok = wait_bounded(wctx, &sh.p_full[b], turn_parity<C::kBufs>(turn), 0xb600 + b);
              if (!ok) break;
              tc_fence_after();
              issue_pv(tile_v, b, lv, blk_v > 0);
              tc_commit(smem_u32(&sh.o_done[tile_v]));
              if (blk_v + 1 == n) tc_commit(smem_u32(&sh.o_final[tile_v]));
              if (++tile_v == nt) {
                ring_release(lv);
                tile_v = 0;
                ++blk_v;
              }
            }
            if (blk_k < n) {
              const uint32_t b = turn_buffer<C::kBufs>(turns + t + ahead), lk = ld + 2 * blk_k;
              if (blk_k == 0) ok = wait_bounded(wctx, &sh.q_full[tile_k], qn[tile_k]++ & 1, 0xb500 + tile_k);
              if (ok && tile_k == 0) ok = ring_wait(lk);
              if (!ok) break;
              tc_fence_after();
              issue_qk(tile_k, b, lk);
              if (++tile_k == nt) {
                ring_release(lk);
                tile_k = 0;
                ++blk_k;
              }
            }
          }
          turns += n * nt;
          ld += 2 * n;
        }
        {
          // products in flight, and their arrivals, end before tensor and shared memory are freed (with a limit)
          tc_commit(smem_u32(&sh.drain));
          const uint64_t t0 = global_timer_ns();
          while (!mbar_try_wait(smem_u32(&sh.drain), 0) && global_timer_ns() - t0 < 20000000ull) {}
        }
      }
      __syncwarp();
    }
  } else if (warp >= C::kWideWarp0) {
    // ---------------------------------------------------------------- widening
    if constexpr (C::kDeal) setmaxnreg_dec<C::kWideRegs>();
    const int w = warp - C::kWideWarp0;
    uint32_t tiles = 0;
    Item it;
    bool ok = true;
    while (ok && (ok = next_item(it))) {
      __syncwarp();
      if (lane == 0) item_read();
      else ++n_items;
      if (it.seq < 0) break;
      const int n_tiles = 2 * (it.blk1 - it.blk0), apart_blk = apart(it);
      for (int i = 0; i < n_tiles && ok; ++i, ++tiles) {
        const uint32_t st = tiles % C::kRaw, rg = tiles % C::kRing;
        ok = wait_bounded(wctx, &sh.raw_full[st], (tiles / C::kRaw) & 1, 0xb700 + st);
        if (ok) ok = wait_bounded(wctx, &sh.ring_empty[rg], ((tiles / C::kRing) & 1) ^ 1, 0xb800 + rg);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const int valid = sh.valid[st];
        const uint32_t src = s_raw + st * C::kRawBytes, dst = s_ring + rg * C::kRingBytes;
        // A warp takes eight rows and 64 columns at a time: eight lanes side by side read and write eight rows of one 16-byte
        // column, which the swizzles spread over all banks.
        constexpr int kParts = (C::kN / 8) * C::kCols, kMine = kParts / 4;
        const int q = lane >> 3, r8 = lane & 7;
        auto from = [&](int p) {
          const int cb = p % C::kCols, r = (p / C::kCols) * 8 + r8;
          if constexpr (W == 64) return src + ((r * 64 + ((q ^ ((r >> 1) & 3)) << 4)) ^ ((r & 8) ? flip : 0u));
          else return src + (cb >> 1) * C::kRawBlockBytes + r * 128 + (((4 * (cb & 1) + q) ^ r8) << 4);
        };
        auto put = [&](int p, const uint4& lo, const uint4& hi) {
          const uint32_t to = dst + (p % C::kCols) * (C::kN * 128) + ((p / C::kCols) * 8 + r8) * 128;
          st_shared16(to + (((2 * q) ^ r8) << 4), lo);
          st_shared16(to + (((2 * q + 1) ^ r8) << 4), hi);
        };
        if ((i & 1) && it.blk0 + (i >> 1) >= apart_blk) {
#pragma unroll 1
          for (int p = w; p < kParts; p += 4) {
            if (sh.factor[st][p / C::kCols / 2] == 0u || (p / C::kCols) * 8 + r8 >= valid) continue;
            uint4 x = ld_shared16(from(p));
            if (drop_specials<kE5M2>(x)) {
              st_shared16(from(p), x);
              sh.with_special_v[(n_items - 1) % kItemSlots] = 1;
            }
          }
          __syncwarp();
        }
        if (sh.complete[st]) {
          // four loads go out before the first is used
#pragma unroll
          for (int k0 = 0; k0 < kMine; k0 += 4) {
            uint4 x[4];
            uint32_t f[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int p = w + 4 * (k0 + k);
              x[k] = ld_shared16(from(p));
              f[k] = sh.factor[st][p / C::kCols / 2];
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              uint4 lo, hi;
              widen16<kE5M2>(x[k], f[k], lo, hi);
              put(w + 4 * (k0 + k), lo, hi);
            }
          }
        } else {
#pragma unroll 1
          for (int p = w; p < kParts; p += 4) {
            const uint32_t f = sh.factor[st][p / C::kCols / 2];
            uint4 lo = make_uint4(0u, 0u, 0u, 0u), hi = lo;
            if (f != 0u && (p / C::kCols) * 8 + r8 < valid) widen16<kE5M2>(ld_shared16(from(p)), f, lo, hi);
            put(p, lo, hi);
          }
        }
        fence_proxy_async_smem();                                // what was written is for the products to read
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(smem_u32(&sh.ring_full[rg]));
          mbar_arrive(smem_u32(&sh.raw_empty[st]));
        }
      }
    }
  } else {
    // ---------------------------------------------------------------- softmax
    if constexpr (C::kDeal) setmaxnreg_inc<C::kSoftRegs>();
    // Two warps to 32 rows (lanes of tensor memory): each takes half of a block's keys, of O's columns and of the rows of Q.
    const int tile = warp / 8, sub = warp % 4, part = warp / 4 % 2;
    const uint32_t lanes = static_cast<uint32_t>(32 * sub) << 16;
    const uint32_t t_o = tmem + lanes + C::kOCol + W * tile + part * (W / 2);
    constexpr int kMyKeys = C::kN / 2, kMyCols = W / 2;
    const int r = 32 * sub + lane;                               // this thread's row
    const int pair_bar = 1 + tile * 4 + sub;
    // (Tensor-memory instructions and barriers want whole warps: lanes that left a wait at different times meet before each.)
    auto pair_sync = [&] {
      __syncwarp();
      asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory");
    };
    auto pair_any = [&](bool x) {
      __syncwarp();
      uint32_t y;
      asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, %2, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}\n"
                   : "=r"(y) : "r"(static_cast<uint32_t>(x)), "r"(pair_bar) : "memory");
      return y != 0u;
    };
    // The other warp's value for this row.
    auto exchange = [&](float x) {
      float* const p = &sh.row[tile][r];
      if (part == 0) *p = x;
      pair_sync();
      float y = 0.f;
      if (part == 1) {
        y = *p;
        *p = x;
      }
      pair_sync();
      return part == 1 ? y : *p;
    };
    uint32_t blocks = 0;                                         // of all items (the residual ring), also those this tile sits out
    uint32_t turns = 0;                                          // of the score buffers, before this item
    uint32_t own = 0;                                            // of this tile's turns
    uint32_t taken = 0;                                          // items this tile took part in
    Item it;
    bool ok = true;
    while (true) {
      // A warp whose wait ran out takes the other of its pair along: neither waits for one that has left.
      ok = !pair_any(!next_item(it));
      if (!ok) break;
      if (lane == 0) item_read();
      else ++n_items;
      if (it.seq < 0) break;
      const int nb = it.blk1 - it.blk0;
      const int tok0 = it.token0 + tile * tile_tokens;
      const int n_rows = min(tile_tokens, it.n_tokens - tile * tile_tokens) * group;
      const int nt = C::kTiles == 2 && it.n_tokens > tile_tokens ? 2 : 1;
      if (n_rows <= 0) {
        blocks += nb;
        turns += nb;
        continue;
      }
      const int D = a.c.head_dim;
      // ---- Q: sixteen rows into shared memory, fp16 ----
      {
        constexpr int kLanes = W / 8, kRowsAt = 32 / kLanes, kTimes = 16 / kRowsAt;     // lanes of a row (8 columns each), rows at a time
        const int col = lane % kLanes, row0 = 32 * sub + 16 * part + lane / kLanes;
        uint4 x[kTimes];                                         // all of them under way at once
        const uint16_t* const q0 = static_cast<const uint16_t*>(a.q.x) + (static_cast<int64_t>(it.first) + tok0) * a.q.token_stride +
                                   static_cast<int64_t>(it.head) * group * a.q.head_stride + 8 * col;
#pragma unroll
        for (int k = 0; k < kTimes; ++k) {
          const int q = row0 + k * kRowsAt, token = (q * over_group) >> 16;
          x[k] = make_uint4(0u, 0u, 0u, 0u);
          if (q < n_rows && 8 * col < D)
            x[k] = ld_global(reinterpret_cast<const uint4*>(q0 + token * a.q.token_stride + (q - token * group) * a.q.head_stride));
        }
#pragma unroll
        for (int k = 0; k < kTimes; ++k) {
          const int q = row0 + k * kRowsAt;
          float back = 1.f;
          if (a.bf16) {
            float big = 0.f;
            uint32_t v[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 f = half_pair<true>(v[e] & 0x7fff7fffu);
              big = fmaxf(big, fmaxf(f.x, f.y));
            }
#pragma unroll
            for (int o = kLanes / 2; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
            const int e = min(max(static_cast<int>(__float_as_uint(big) >> 23) - 127, -100), 126);
            const float f = __uint_as_float(static_cast<uint32_t>(14 - e + 127) << 23);
            back = __uint_as_float(static_cast<uint32_t>(e - 14 + 127) << 23);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 y = half_pair<true>(v[i]);
              v[i] = pack_half2(y.x * f, y.y * f);
            }
            x[k] = make_uint4(v[0], v[1], v[2], v[3]);
          }
          if (col == 0) sh.row[tile][q] = back;
          st_shared16(s_q + tile * C::kQBytes + (col >> 3) * (kTileM * 128) + q * 128 + (((col & 7) ^ (q & 7)) << 4), x[k]);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sh.q_full[tile]));
      pair_sync();                                               // the other warp's rows of sh.row
      const float back = sh.row[tile][r];
      pair_sync();

      Row row{};
      row.m = -INFINITY;
      const int my_token = tok0 + ((min(r, n_rows - 1) * over_group) >> 16);
      row.lim = a.causal ? max(0, min(it.len, it.len - it.n + my_token + 1)) : it.len;
      const int least = a.causal ? max(0, min(it.len, it.len - it.n + tok0 + 1)) : it.len;       // of the tile's first row
      float vref = 1.f;
      for (int j = 0; j < nb && ok; ++j, ++own) {
        const uint32_t buf = turn_buffer<C::kBufs>(turns + j * nt + tile);
        const uint32_t n = (blocks + j) % kBlockSlots;
        const uint32_t t_p = tmem + lanes + C::kN * buf, t_s = t_p + part * kMyKeys;
        ok = wait_bounded(wctx, &sh.blk_full[n], ((blocks + j) / kBlockSlots) & 1, 0xb900);
        if (ok) ok = wait_bounded(wctx, &sh.s_full[tile][score_barrier(own)], score_parity(own), 0xba00 + buf);
        __syncwarp();
        tc_fence_after();
        const int key0 = (it.blk0 + j) * C::kN, lim = row.lim - key0 - part * kMyKeys;
        const bool general = sh.flagged[n] != 0 || key0 + C::kN > least;
        const float *rk = sh.residual[n][0] + part * (kMyKeys / 16), *rv = sh.residual[n][1] + part * (kMyKeys / 16);
        // the largest score of this warp's keys
        auto top_of = [&] {
          float m = -INFINITY;
#pragma unroll 1
          for (int k = 0; k < kMyKeys; k += 32) {
            uint32_t x[32];
            tmem_ld_32x32b_x32(t_s + k, x);
            tmem_wait_ld();
            m = fmaxf(m, general ? largest<true>(x, row.c, lim - k, rk + k / 16, rv + k / 16) : largest<false>(x, row.c, 0, nullptr, nullptr));
          }
          return m;
        };
        if (j == 0) {
          row.c = a.scale_log2 * back * sh.ref[n][0];
          vref = sh.ref[n][1];
          float m = top_of();                                    // exact for the first block
          m = fmaxf(m, exchange(m));
          row.m = m - kHeadroom;
          row.nm = m == -INFINITY ? 0.f : -row.m;
          row.most = m == -INFINITY ? 0.f : kRaiseAbove;
        }
        // P of the block; the scores are left as they are until no reference has to be raised for them.
        uint32_t pk[kMyKeys / 2];
        float l = 0.f;
        bool raised = false;
        while (true) {
          float sum = 0.f;
          l = 0.f;
#pragma unroll
          for (int q = 0; q < kMyKeys / 32; ++q) {
            uint32_t x[32];
            tmem_ld_32x32b_x32(t_s + 32 * q, x);
            tmem_wait_ld();
            sum += general ? exponentials<true>(x, row.c, row.nm, lim - 32 * q, rk + 2 * q, rv + 2 * q, pk + 16 * q, &l)
                           : exponentials<false>(x, row.c, row.nm, 0, nullptr, nullptr, pk + 16 * q, &l);
          }
          // (also: the other warp has read what P is about to be written over)
          const bool over = !(sum <= row.most);
          const bool any = pair_any(over || !ok);
          if (any && pair_any(!ok)) {
            ok = false;
            break;
          }
          if (!any || raised) break;
          // Some row has outgrown its reference (or holds a NaN): take this block's maximum in and rescale O, for which the products
          // before have to be done.
          raised = true;
          const float mine_top = top_of() - kHeadroom, top = over ? mine_top : -INFINITY;
          const float m = fmaxf(fmaxf(row.m, top), exchange(top));
          const float nm = m == -INFINITY ? 0.f : -m;
          const float alpha = to_reference(row.m, -nm, row.l);
          row.m = m;
          row.nm = nm;
          row.most = m == -INFINITY ? 0.f : kRaiseAbove;
          if (j > 0) {
            ok = wait_bounded(wctx, &sh.o_done[tile], done_parity(own), 0xbb00 + tile) && ok;
            __syncwarp();
            tc_fence_after();
            rescale(t_o, kMyCols, alpha);
          }
        }
        if (!ok) break;
        row.l += l;
        if constexpr (kMyKeys == 64) tmem_st_32x32b_x32(t_p + part * 32, pk);       // over the scores
        else tmem_st_32x32b_x16(t_p + part * 16, pk);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.p_full[buf]));
      }
      blocks += nb;
      turns += nb * nt;
      if (!ok) break;

      // ---- O ----
      const bool whole = it.part < 0;
      row.l += exchange(row.l);
      ok = !pair_any(!wait_bounded(wctx, &sh.o_final[tile], taken & 1, 0xbc00 + tile));
      if (!ok) break;
      ++taken;
      tc_fence_after();
      const float inv = (row.l == 0.f ? 0.f : (whole ? 1.f / row.l : 1.f)) * vref;
      const int token = (r * over_group) >> 16;
      const int64_t row0 = (static_cast<int64_t>(it.first) + tok0) * a.heads_q + it.head * group;
      const int64_t out_row = row0 + token * a.heads_q + (r - token * group);
      if (r < n_rows && part == 0) {
        if (whole) {
          if (a.lse != nullptr) a.lse[out_row] = row.l == 0.f ? -INFINITY : (row.m + __log2f(row.l)) * 0.6931471805599453f;
        } else {
          float* const ml = plan.partial_ml + 2 * (static_cast<int64_t>(it.part) * a.c.tokens * a.heads_q + out_row);
          ml[0] = row.m;
          ml[1] = row.l;
        }
      }
      float* const po = whole ? nullptr : plan.partial_o + (static_cast<int64_t>(it.part) * a.c.tokens * a.heads_q + out_row) * D;
      // through these rows and columns of Q's shared memory, which the last scores have been made from: 16 bytes a lane side by side
      const uint32_t stage = s_q + tile * C::kQBytes;
#pragma unroll 1
      for (int c = 0; c < kMyCols; c += 32) {
        __syncwarp();
        uint32_t o[32];
        tmem_ld_32x32b_x32(t_o + c, o);
        tmem_wait_ld();
        const int col = part * kMyCols + c;
        if (col >= D) continue;
        if (whole) {
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            uint32_t v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float x = __uint_as_float(o[i + 2 * k]) * inv, y = __uint_as_float(o[i + 2 * k + 1]) * inv;
              v[k] = a.bf16 ? pack_pair<true>(x, y) : pack_pair<false>(x, y);
            }
            const int ch = (col + i) >> 3;
            st_shared_v4(stage + (ch >> 3) * (kTileM * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4), v[0], v[1], v[2], v[3]);
          }
        } else if (r < n_rows) {
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            float4 v;
            v.x = __uint_as_float(o[i]) * inv; v.y = __uint_as_float(o[i + 1]) * inv;
            v.z = __uint_as_float(o[i + 2]) * inv; v.w = __uint_as_float(o[i + 3]) * inv;
            *reinterpret_cast<float4*>(po + col + i) = v;
          }
        }
      }
      tc_fence_before();
      if (whole) {
        __syncwarp();
        constexpr int kLanes = kMyCols / 8, kRowsAt = 32 / kLanes;       // lanes of half a row, rows at a time
        const int ch = part * kLanes + lane % kLanes;
#pragma unroll 4
        for (int q = 32 * sub + lane / kLanes; q < 32 * sub + 32; q += kRowsAt) {
          const int t = (q * over_group) >> 16;
          if (q < n_rows && 8 * ch < D) {
            const uint4 v = ld_shared16(stage + (ch >> 3) * (kTileM * 128) + q * 128 + (((ch & 7) ^ (q & 7)) << 4));
            st_global_v4(static_cast<uint16_t*>(a.o) + (row0 + t * a.heads_q + (q - t * group)) * D + 8 * ch, v.x, v.y, v.z, v.w);
          }
        }
      }
      pair_sync();                                               // both warps are through with these rows of Q's memory
      const int slot = (n_items - 1) % kItemSlots;               // still this item's: no more than one other waits
      if (*static_cast<volatile int*>(&sh.with_special_v[slot]) != 0) {
        const Item i = sh.item[slot];
        const int token0 = i.token0 + tile * tile_tokens, rows = min(tile_tokens, i.n_tokens - tile * tile_tokens) * group;
#pragma unroll 1
        for (int q = 32 * sub; q < min(32 * sub + 32, rows); ++q) {
          const int t = (q * over_group) >> 16;
          const int64_t to = ((static_cast<int64_t>(i.first) + token0 + t) * a.heads_q + i.head * group + (q - t * group)) * a.c.head_dim;
          float* const partial = plan.partial_o + static_cast<int64_t>(i.part) * a.c.tokens * a.heads_q * a.c.head_dim;
          write_specials<kE5M2>(a.c, i.seq, i.head, max(apart(i), i.blk0) * C::kN, min(i.len - i.n + token0 + t + 1, i.blk1 * C::kN),
                            part * kMyCols + lane, min(a.c.head_dim, (part + 1) * kMyCols), [&](int col, float sum) {
            if (i.part < 0) {
              uint16_t* const p = static_cast<uint16_t*>(a.o) + to + col;
              *p = with_special(*p, sum, a.bf16);
            } else {
              partial[to + col] += sum;
            }
          });
        }
        __syncwarp();
      }
    }
  }
  let_successor_start();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == C::kMmaWarp) tmem_dealloc(tmem, kTmemCols);
}

// Rows whose keys were cut into parts: a warp to a row.
__global__ void __launch_bounds__(256) kv_join_kernel(const KvAttendArgs a, const KvPrefillPlan plan, int block_keys) {
  start_after_predecessor();
  let_successor_start();
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int token = static_cast<int>(row / a.heads_q);
  if (token >= a.c.tokens) return;
  int b, unused;
  if (a.c.cu == nullptr) b = token / a.c.even;
  else kv_find_slot(a.c, token, 1, 0, &b, &unused);
  const KvSeq s = kv_seq(a.c, b);
  if (token < s.first || token >= s.first + s.n) return;
  const int token0 = (token - s.first) / plan.block_tokens * plan.block_tokens;
  const int n_tokens = min(plan.block_tokens, s.n - token0);
  const int vis = a.causal ? max(0, min(s.len, s.len - s.n + token0 + n_tokens)) : s.len;
  const int parts = parts_of(max(1, (vis + block_keys - 1) / block_keys), plan.parts);
  if (parts == 1) return;
  const int D = a.c.head_dim, quads = D >> 2;
  const int64_t rows = static_cast<int64_t>(a.c.tokens) * a.heads_q;
  float m = -INFINITY;
  for (int p = 0; p < parts; ++p) m = fmaxf(m, ld_global(plan.partial_ml + 2 * (p * rows + row)));
  float l = 0.f;
  float4 acc[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
#pragma unroll 4
  for (int p = 0; p < parts; ++p) {
    const float* ml = plan.partial_ml + 2 * (p * rows + row);
    const float mp = ld_global(ml);
    float lp = ld_global(ml + 1);
    const float f = to_reference(mp, m, lp);
    l += lp;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int q = lane + 32 * i;
      if (q < quads) {
        const uint4 u = ld_global(reinterpret_cast<const uint4*>(plan.partial_o + (p * rows + row) * D) + q);
        acc[i].x += __uint_as_float(u.x) * f; acc[i].y += __uint_as_float(u.y) * f;
        acc[i].z += __uint_as_float(u.z) * f; acc[i].w += __uint_as_float(u.w) * f;
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

template <int W, bool kE5M2>
cudaError_t launch_one(const CUtensorMap& tk, const CUtensorMap& tv, const KvAttendArgs& a, const KvPrefillPlan& plan, cudaStream_t stream) {
  using C = PCfg<W>;
  auto kernel = &kv_prefill_kernel<W, kE5M2>;
  constexpr int smem = C::kSharedOffset + static_cast<int>(sizeof(Shared<W>));
  static_assert(smem <= 227 * 1024, "shared memory");
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
  cfg.gridDim = dim3(static_cast<unsigned>(plan.items), 1, 1);      // below 2^28: kv_prefill_takes wants 17 rows of a sequence
  cfg.blockDim = dim3(C::kThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1] = {overlap_attribute()};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kernel, tk, tv, a, plan);
  if (e != cudaSuccess || plan.parts == 1) return e;
  const int64_t ctas = (static_cast<int64_t>(a.c.tokens) * a.heads_q + 7) / 8;
  cfg.gridDim = dim3(static_cast<unsigned>(ctas), 1, 1);
  cfg.blockDim = dim3(256, 1, 1);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, &kv_join_kernel, a, plan, C::kN);
}

}  // namespace

// The kernel for few rows reads a K/V head's keys once for every 32 rows (16 at head dims above 128), so its time goes with blocks of rows
// times keys, a block counting for some 400 keys more: about 10 us, and 1 us per 9300 of these at head dim 128, per 19000 at 64 and per 9300 of
// the smaller blocks at 256.  This kernel reads them once for 256 (128) rows, but starts later.  Measured, few rows / this one, us
// (H = 4 Hk; 8 K/V heads at head dim 128, otherwise 4):
//   rows of a sequence      32             64             128            32, D 64   64      128      32, D 256  64      128
//   1 x 16000 keys          32 / 30        42 / 33        65 / 35        17 / 25  19 / 25  25 / 26   30 / 42  43 / 43  70 / 47
//   8 x  4000               43 / 44        68 / 46       119 / 51        17 / 24  24 / 26  37 / 26   43 / 42  71 / 45 129 / 48
//  32 x  1000               49 / 49        80 / 51       141 / 55        19 / 21  29 / 22  44 / 24   47 / 39  80 / 40 150 / 42
//   1 x  1000               13 / 20        15 / 21        15 / 24        10 / 16  10 / 17  10 / 18   13 / 20  14 / 22  15 / 26
// and 16 sequences of 17 to 300 new tokens and up to 512 keys, a row a token, 48 / 27.  They meet near 300000 blocks times keys (sooner where one
// long sequence is all there is).  The host knows how many keys the page table can hold, and takes that.
//
// The rule goes by the mean sequence, since the host does not know the lengths, so that a call of many single tokens and one long piece runs in the kernel
// for few rows as a whole: 255 tokens over 4096 keys with 1024 tokens over 16384, head dim 128, take 2480 us, in two calls 360 + 270.
constexpr int64_t kFewRowsMost = 128, kFewRowsKeys = 300000, kBlockKeys = 400;
bool kv_prefill_takes(const KvAttendSizes& z) {
  const int64_t group = z.heads_q / z.heads, rows = (z.tokens * group + z.batch - 1) / z.batch, block = width_of(z.head_dim) == 256 ? 16 : 32;
  if (group > kTileM || rows <= block) return false;
  return rows > kFewRowsMost || z.batch * z.heads * ((rows + block - 1) / block) * (z.keys_most + kBlockKeys) > kFewRowsKeys;
}

constexpr int kPartsMost = 16;
KvPrefillPlan kv_prefill_plan(const KvAttendSizes& z, int sms) {
  KvPrefillPlan p{};
  const int width = width_of(z.head_dim), tiles = width == 256 ? 1 : 2;
  p.block_tokens = kTileM / (z.heads_q / z.heads) * tiles;
  p.items = kv_slots(z.batch, z.tokens, z.tokens / z.batch, z.ragged, p.block_tokens, 1) * z.heads;
  // Few items: their keys are cut into as many parts as fill the GPU once, where they have that many (parts_of).  More parts than CTAs at once
  // (to even out sequences of different lengths) helped some and hurt others: 11 short chunks over 500 to 12000 keys 96 -> 73 us, 3
  // over 3000 to 9000 116 -> 136.
  const int64_t block = width == 256 ? PCfg<256>::kN : PCfg<128>::kN, blocks = (z.keys_most + block - 1) / block;
  const int64_t parts = std::min(blocks / kPartBlocks, sms / std::max<int64_t>(1, p.items));
  p.parts = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(kPartsMost, parts)));
  p.items *= p.parts;
  return p;
}

int64_t kv_prefill_workspace(const KvAttendSizes& z, int sms) {
  const KvPrefillPlan p = kv_prefill_plan(z, sms);
  return p.parts == 1 ? 0 : static_cast<int64_t>(p.parts) * z.tokens * z.heads_q * (z.head_dim + 2) * 4;
}

cudaError_t launch_kv_prefill(const CUtensorMap& tk, const CUtensorMap& tv, const KvAttendArgs& a, const KvAttendSizes& z, void* workspace,
                              bool e5m2, int sms, cudaStream_t stream) {
  KvPrefillPlan p = kv_prefill_plan(z, sms);
  if (p.parts > 1) {
    p.partial_o = static_cast<float*>(workspace);
    p.partial_ml = p.partial_o + static_cast<int64_t>(p.parts) * z.tokens * z.heads_q * z.head_dim;
  }
  switch (width_of(a.c.head_dim)) {
    case 64: return e5m2 ? launch_one<64, true>(tk, tv, a, p, stream) : launch_one<64, false>(tk, tv, a, p, stream);
    case 128: return e5m2 ? launch_one<128, true>(tk, tv, a, p, stream) : launch_one<128, false>(tk, tv, a, p, stream);
    default: return e5m2 ? launch_one<256, true>(tk, tv, a, p, stream) : launch_one<256, false>(tk, tv, a, p, stream);
  }
}

}  // namespace fa8
