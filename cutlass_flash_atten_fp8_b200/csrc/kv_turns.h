// Turns of the score buffers in the kernel for many rows over the paged cache (fa8_kv_prefill.cu).
//
// A block of keys and a tile of query rows are a turn; an item's turns go over its tiles block by block, and turn t (counted over all
// items of the CTA) lives in buffer t % kBufs, whichever tile it is of.  An item of one tile has turns of tile 0 only: tile 1 sits it
// out, waits for nothing of it and may be at its first turn of the next item while turns of this one are still to come.
//
// A wait by parity is right only while the number of completed phases is known to be the awaited one's (counted from 0) or one more.
//   s_full[tile][b]   a phase for each turn of the tile's own in buffer b, when its scores are there.  The tile has waited for all before.  The
//                     next such turn's scores are issued after the product P V of this one, which needs P of every warp of the tile.
//                     (A barrier per buffer, with a phase for every turn, will not do: a tile that sat out an item has not seen the phases of
//                     its turns, and may find the one before the awaited one still to come, which passes, or two gone by, which does not.)
//   p_full[b]         a phase for each turn in buffer b, waited for by the issuer, which waits for them all, in their order; a warp adds to it
//                     after its turn's s_full, and that turn's scores were issued after P V of the turn before it in the buffer.
//   o_done[tile][b]   a phase for each turn of the tile's own in buffer b, in items with fewer tiles than buffers (in others the tile's next
//                     scores come after the product), when its product P V is complete.  Asked for the tile's turn before the one whose
//                     scores are there: that turn's own scores, there before, were issued after all earlier products from the buffer, and
//                     the next product from it comes after that of the present turn, which needs P of the tile.
//                     (One barrier for all of a tile's products will not do with three buffers and one tile: the scores of the first three
//                     turns are issued ahead of all products, so that two can be outstanding.)
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

template <int kBufs>
FA8_HD constexpr uint32_t turn_buffer(uint32_t turn) { return turn % kBufs; }

// `seen`: parities of the numbers of phases that a warp of a tile has waited for, or counts as gone by: bit b of s_full[tile][b], bit
// kSeenDone + b of o_done[tile][b], bit kSeenFinal of o_final[tile].
FA8_HD constexpr uint32_t seen_parity(uint32_t seen, uint32_t bit) { return (seen >> bit) & 1u; }
FA8_HD constexpr uint32_t seen_next(uint32_t seen, uint32_t bit) { return seen ^ (1u << bit); }
template <int kBufs> constexpr uint32_t kSeenDone = kBufs;
template <int kBufs> constexpr uint32_t kSeenFinal = 2 * kBufs;

// Parity for a barrier with a phase for every turn in the buffer.
template <int kBufs>
FA8_HD constexpr uint32_t turn_parity(uint32_t turn) { return (turn / kBufs) & 1u; }

}  // namespace fa8
