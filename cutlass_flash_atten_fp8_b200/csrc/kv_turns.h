// Turns of the score buffers in the kernel for many rows over the paged cache (fa8_kv_prefill.cu).
//
// A block of keys and a tile of query rows are a turn; an item's turns go over its tiles block by block, and turn t (counted over all
// items of the CTA) lives in buffer t % kBufs, whichever tile it is of.  An item of one tile has turns of tile 0 only: tile 1 sits it
// out, waits for nothing of it and may be at its first turn of the next item while turns of this one are still to come.
//
// The issuer gives out scores turns_ahead() turns ahead within an item and those of turn t + ahead after the product P V of turn t.
//
// A wait by parity is right only while the number of completed phases is known to be the awaited one's (counted from 0) or one more.
// A tile's own turns are counted over all items, k = 0, 1 ...
//   s_full[tile][k % 2]   a phase when the scores of own turn k are there.  The tile has waited for all before; those of own turn k + 2, 2 tiles
//                     later, come after P V of own turn k (turns_ahead <= 2 tiles), which needs P of every warp of the tile.
//                     (A barrier per buffer, with a phase for every turn, will not do: a tile that sat out an item has not seen the phases of
//                     its turns, and may find the one before the awaited one still to come, which passes, or two gone by, which does not.)
//   o_done[tile]      a phase when P V of own turn k is complete.  Asked for own turn k - 1 once the scores of k are there: they were issued after
//                     P V of k - 2 (turns_ahead <= 2 tiles) if that is of the same item, and if not, after it was awaited (o_final);
//                     P V of k needs P of the tile.  (So with three buffers and one tile the scores must not run three turns ahead.)
//   p_full[b]         a phase for each turn in buffer b, waited for by the issuer, which waits for them all, in their order; a warp adds to it
//                     after its turn's s_full, and that turn's scores were issued after P V of the turn before it in the buffer.
//   o_final[tile]     a phase for each item that the tile is part of, all of which it waits for.
#pragma once
#include <cstdint>

#ifndef FA8_HD
#ifdef __CUDACC__
#define FA8_HD __host__ __device__
#else
#define FA8_HD
#endif
#endif

namespace fa8 {

// How many turns ahead the scores of an item of that many tiles run: one more than its tiles if there are buffers for it.
template <int kBufs>
FA8_HD constexpr int turns_ahead(int tiles) { return tiles < kBufs ? tiles + 1 : kBufs; }

template <int kBufs>
FA8_HD constexpr uint32_t turn_buffer(uint32_t turn) { return turn % kBufs; }
// Parity for a barrier with a phase for every turn in the buffer.
template <int kBufs>
FA8_HD constexpr uint32_t turn_parity(uint32_t turn) { return (turn / kBufs) & 1u; }

// Of own turn k: which of the tile's two barriers its scores have, and the parity to wait for them with.
FA8_HD constexpr uint32_t score_barrier(uint32_t k) { return k & 1u; }
FA8_HD constexpr uint32_t score_parity(uint32_t k) { return (k >> 1) & 1u; }
// Parity to wait with for the product of own turn k - 1.
FA8_HD constexpr uint32_t done_parity(uint32_t k) { return (k - 1u) & 1u; }

}  // namespace fa8
