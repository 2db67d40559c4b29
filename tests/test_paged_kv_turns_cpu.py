"""The waits on the score buffers' barriers of the kernel for many rows over the paged cache (csrc/kv_turns.h, compiled here for
the host as the kernel uses it), in every state that a model of the kernel's warps can reach: each passes exactly when what it is
for has happened, whichever warps are ahead and however far, also where a tile sits out an item that the other works on."""
import os
import shutil
import subprocess

import pytest

from cutlass_flash_atten_fp8_b200.build import CSRC

# The issuer: scores so many turns ahead, then P V of a turn and the next scores.  The tensor core completes what was issued in
# order.  Two warps a tile, each for itself: an item is there for the next read once all have read the one before.
MODEL = r"""
#include <cstdint>
#include <cstdio>
#include <unordered_set>
#include <vector>
#include "kv_turns.h"
struct Item { int blocks, tiles; };
struct Op { bool pv; int turn, tile; bool last; };            // last: with a phase of o_final
enum Kind { kRead, kQ, kScores, kProbs, kFinal, kIssue, kAskProbs, kAskQ };
struct Event { Kind kind; int at, before; uint32_t k; };      // at: item, turn or op; before: the tile's turn before it in the item, or -1; k: own turn, item
static bool passes(uint32_t completed, uint32_t parity) { return ((completed & 1u) ^ 1u) == parity; }

// kAhead 0: as the kernel has it
template <int kTiles, int kBufs, int kAhead = 0>
struct Model {
  std::vector<Op> ops;
  std::vector<int> tile_of, s_op, pv_op;                      // of turns
  std::vector<uint32_t> own_of;
  std::vector<Event> issuer, warp[2];
  long wrong = 0, wrong_shared = 0;                           // wrong_shared: with one barrier a buffer for the scores of both tiles

  explicit Model(const std::vector<Item>& items) {
    int turns = 0, asked[2] = {0, 0};
    uint32_t own[2] = {0, 0}, taken[2] = {0, 0};
    for (int i = 0; i < static_cast<int>(items.size()); ++i) {
      const int n = items[i].blocks, nt = items[i].tiles;
      const int ahead = kAhead > 0 ? kAhead : fa8::turns_ahead<kBufs>(nt);
      for (int t = 0; t < n * nt; ++t) {
        tile_of.push_back(t % nt);
        own_of.push_back(own[t % nt] + t / nt);
      }
      s_op.resize(turns + n * nt);
      pv_op.resize(turns + n * nt);
      issuer.push_back({kRead, i, 0, 0});
      for (int t = -ahead; t < n * nt; ++t) {
        if (t >= 0) {
          issuer.push_back({kAskProbs, turns + t, 0, 0});
          issuer.push_back({kIssue, static_cast<int>(ops.size()), 0, 0});
          pv_op[turns + t] = static_cast<int>(ops.size());
          ops.push_back({true, turns + t, t % nt, t / nt + 1 == n});
        }
        const int s = t + ahead;
        if (s < n * nt) {
          if (s < nt) issuer.push_back({kAskQ, s, asked[s]++, 0});
          issuer.push_back({kIssue, static_cast<int>(ops.size()), 0, 0});
          s_op[turns + s] = static_cast<int>(ops.size());
          ops.push_back({false, turns + s, s % nt, false});
        }
      }
      for (int tile = 0; tile < kTiles; ++tile) {
        auto& w = warp[tile];
        w.push_back({kRead, i, 0, 0});
        if (tile >= nt) continue;                             // sits the item out
        w.push_back({kQ, i, 0, 0});
        for (int j = 0; j < n; ++j) {
          const int turn = turns + j * nt + tile;
          w.push_back({kScores, turn, 0, own[tile]});
          w.push_back({kProbs, turn, j > 0 ? turn - nt : -1, own[tile]++});
        }
        w.push_back({kFinal, turns + (n - 1) * nt + tile, 0, taken[tile]++});
      }
      turns += n * nt;
    }
    // scores go into a buffer after the last product that reads it
    for (int t = kBufs; t < turns; ++t) wrong += !(pv_op[t - kBufs] < s_op[t]);
  }

  struct State { int issuer, done, at[2][2]; };               // places in the lists; operations complete
  static uint64_t key(const State& s) {
    uint64_t k = s.issuer;
    for (const int x : {s.done, s.at[0][0], s.at[0][1], s.at[1][0], s.at[1][1]}) k = k * 256 + x;
    return k;
  }
  bool past(const std::vector<Event>& e, int at, Kind kind, int what) const {
    for (int i = 0; i < at; ++i)
      if (e[i].kind == kind && e[i].at == what) return true;
    return false;
  }
  int issued(const State& s) const {
    int n = 0;
    for (int i = 0; i < s.issuer; ++i) n += issuer[i].kind == kIssue;
    return n;
  }
  bool item_there(const State& s, int i) const {
    if (i == 0) return true;
    if (!past(issuer, s.issuer, kRead, i - 1)) return false;
    for (int t = 0; t < kTiles; ++t)
      for (int w = 0; w < 2; ++w)
        if (!past(warp[t], s.at[t][w], kRead, i - 1)) return false;
    return true;
  }
  bool has_probs(const State& s, int turn) const {
    const int t = tile_of[turn];
    return past(warp[t], s.at[t][0], kProbs, turn) && past(warp[t], s.at[t][1], kProbs, turn);
  }
  bool all_q(const State& s, int tile, int nth) const {       // Q of the tile's nth item
    for (int w = 0; w < 2; ++w) {
      int n = 0;
      for (int i = 0; i < s.at[tile][w]; ++i) n += warp[tile][i].kind == kQ;
      if (n <= nth) return false;
    }
    return true;
  }

  // Whether the warp's next event can happen; checks its wait on the way.
  bool warp_moves(const State& s, int tile, int w) {
    const Event& e = warp[tile][s.at[tile][w]];
    auto completed = [&](auto pick) {
      uint32_t n = 0;
      for (int i = 0; i < s.done; ++i) n += pick(ops[i]);
      return n;
    };
    switch (e.kind) {
      case kRead: return item_there(s, e.at);
      case kScores: {
        const bool have = s_op[e.at] < s.done;
        auto mine = [&](const Op& o) { return !o.pv && o.tile == tile && fa8::score_barrier(own_of[o.turn]) == fa8::score_barrier(e.k); };
        wrong += passes(completed(mine), fa8::score_parity(e.k)) != have;
        auto in_buffer = [&](const Op& o) { return !o.pv && fa8::turn_buffer<kBufs>(o.turn) == fa8::turn_buffer<kBufs>(e.at); };
        wrong_shared += passes(completed(in_buffer), fa8::turn_parity<kBufs>(e.at)) != have;
        return have;
      }
      case kProbs:
        if (e.before >= 0)
          wrong += passes(completed([&](const Op& o) { return o.pv && o.tile == tile; }), fa8::done_parity(e.k)) != (pv_op[e.before] < s.done);
        return true;
      case kFinal: {
        const bool have = pv_op[e.at] < s.done;
        wrong += passes(completed([&](const Op& o) { return o.last && o.tile == tile; }), e.k & 1u) != have;
        return have;
      }
      default: return true;
    }
  }
  bool issuer_moves(const State& s) {
    const Event& e = issuer[s.issuer];
    switch (e.kind) {
      case kRead: return item_there(s, e.at);
      case kAskProbs: {
        const bool have = has_probs(s, e.at);
        uint32_t n = 0;
        for (int t = 0; t < static_cast<int>(tile_of.size()); ++t)
          n += fa8::turn_buffer<kBufs>(t) == fa8::turn_buffer<kBufs>(e.at) && has_probs(s, t);
        wrong += passes(n, fa8::turn_parity<kBufs>(e.at)) != have;
        return have;
      }
      case kAskQ: {
        const bool have = all_q(s, e.at, e.before);
        uint32_t n = 0;
        while (all_q(s, e.at, static_cast<int>(n))) ++n;
        wrong += passes(n, static_cast<uint32_t>(e.before) & 1u) != have;
        return have;
      }
      default: return true;
    }
  }

  bool run() {                                                // whether the end is reached from everywhere
    std::unordered_set<uint64_t> known;
    std::vector<State> next{State{}};
    bool stuck = false;
    while (!next.empty()) {
      const State s = next.back();
      next.pop_back();
      if (!known.insert(key(s)).second) continue;
      const size_t before = next.size();
      auto add = [&](State x) { next.push_back(x); };
      State x = s;
      if (s.issuer < static_cast<int>(issuer.size()) && issuer_moves(s)) { ++x.issuer; add(x); x = s; }
      if (s.done < issued(s)) { ++x.done; add(x); x = s; }
      for (int t = 0; t < kTiles; ++t)
        for (int w = 0; w < 2; ++w)
          if (s.at[t][w] < static_cast<int>(warp[t].size()) && warp_moves(s, t, w)) { ++x.at[t][w]; add(x); x = s; }
      if (next.size() == before) {
        bool end = s.issuer == static_cast<int>(issuer.size()) && s.done == static_cast<int>(ops.size());
        for (int t = 0; t < kTiles; ++t)
          for (int w = 0; w < 2; ++w) end = end && s.at[t][w] == static_cast<int>(warp[t].size());
        stuck = stuck || !end;
      }
    }
    return !stuck;
  }
};

template <int kTiles, int kBufs, int kAhead = 0>
void all() {
  long wrong = 0, shared_two = 0, shared_mixed = 0, stuck = 0, runs = 0;
  std::vector<std::vector<Item>> lists;
  for (int a = 1; a <= 3; ++a)
    for (int at = 1; at <= kTiles; ++at)
      for (int b = 1; b <= 3; ++b)
        for (int bt = 1; bt <= kTiles; ++bt) {
          lists.push_back({{a, at}, {b, bt}});
          if (a < 3 && b < 3)
            for (int ct = 1; ct <= kTiles; ++ct) lists.push_back({{a, at}, {b, bt}, {2, ct}});
        }
  for (const auto& items : lists) {
    Model<kTiles, kBufs, kAhead> m(items);
    stuck += !m.run();
    bool mixed = false;
    for (const Item& i : items) mixed = mixed || i.tiles < kTiles;
    wrong += m.wrong;
    (mixed ? shared_mixed : shared_two) += m.wrong_shared;
    ++runs;
  }
  std::printf("%ld %ld %ld %ld %ld\n", runs, wrong, stuck, shared_two, shared_mixed);
}
int main() {
  all<2, 2>();
  all<2, 3>();
  all<1, 2>();
  all<2, 3, 3>();
  return 0;
}
"""


def test_waits_pass_exactly_when_they_should(tmp_path):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no host compiler")
    src, exe = tmp_path / "model.cpp", str(tmp_path / "model")
    src.write_text(MODEL)
    subprocess.run([cxx, "-std=c++17", "-O2", "-I" + CSRC, str(src), "-o", exe], check=True)
    out = subprocess.run([exe], check=True, capture_output=True, text=True).stdout
    *kernel, far = (tuple(map(int, line.split())) for line in out.splitlines())
    for (runs, wrong, stuck, shared_two, shared_mixed), tiles in zip(kernel, (2, 2, 1)):
        assert runs > 10 and wrong == 0 and stuck == 0
        # a barrier per buffer for both tiles would do only while no tile sits an item out
        assert shared_two == 0 and (shared_mixed > 0) == (tiles == 2)
    # scores three turns ahead, also of one tile, would be too many for these barriers
    assert far[1] > 0



def test_the_kernel_uses_these_rules():
    with open(os.path.join(CSRC, "fa8_kv_prefill.cu")) as f:
        text = f.read()
    for part in ("ahead = turns_ahead<C::kBufs>(nt)", "turn_buffer<C::kBufs>(turns + t + ahead)", "turn_buffer<C::kBufs>(turns + j * nt + tile)",
                 "&sh.s_full[tile][score_barrier(own)], score_parity(own)", "tc_commit(smem_u32(&sh.s_full[tile][score_barrier(scored >> tile)]))",
                 "&sh.p_full[b], turn_parity<C::kBufs>(turn)", "&sh.o_done[tile], done_parity(own)", "&sh.o_final[tile], taken & 1"):
        assert part in text, part
