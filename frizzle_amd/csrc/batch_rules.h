// Where a batch of requests finds its keys and how its work is cut, from
// sizes alone (no HIP, so that a test can compile it by itself).
//
// A request's keys lie in pages: slot s of its key p / page_slots is
// p % page_slots, and the page's number stands in the request's row of the
// table. A row of the batch reads the keys (p - window, p]; those past the
// table's width, or in a page that the pool does not have, are not there.
//
// Attention's work is counted in blocks of 32 keys, which lie by position, a
// row's keys' blocks taken by each of its head blocks (a key-value head with
// up to 16 of its query heads). A row of n blocks is cut into ceil(n / chunk)
// parts, a workgroup each, for one chunk that the whole batch shares: a batch
// of one long and many short requests then keeps every compute unit at work,
// where a cut of so many parts a row would leave the long one last. A part's
// waves take its blocks in turn.

#pragma once

#include <stdint.h>

#if defined(__HIPCC__)
#define FRZ_RULE __host__ __device__ inline
#else
#define FRZ_RULE inline
#endif

namespace frz {
namespace rules {

constexpr uint32_t kNone = 0xFFFFFFFFu;  // no position, no page, no adapter

// ---- pages -------------------------------------------------------------------

// The page that holds a sequence's `index`-th page of keys, or kNone.
FRZ_RULE uint32_t page_at(const uint32_t* table, uint32_t sequences, uint32_t width,
                          uint32_t pages, uint32_t sequence, uint32_t index) {
  if (sequence >= sequences || index >= width) return kNone;
  const uint32_t page = table[(uint64_t)sequence * width + index];
  return page < pages ? page : kNone;
}

// The most keys of a sequence: positions stay below 2^24, which F32 holds.
constexpr uint64_t kMostKeys = 1u << 24;

// ---- attention's parts -------------------------------------------------------

constexpr uint32_t kBlockKeys = 32;
constexpr uint32_t kPartWaves = 4;   // a part's workgroup
constexpr uint32_t kHeadBlock = 16;  // query heads that share a part at most
constexpr uint32_t kMostRows = 512;

// The keys [first, end) that a row at `position` reads of a sequence whose
// table holds `capacity`.
struct KeyRange {
  uint32_t first, end;
};
FRZ_RULE KeyRange key_range(uint32_t position, uint32_t window, uint32_t capacity) {
  KeyRange r;
  const uint32_t after = position + 1;  // position is not kNone
  r.first = after > window ? after - window : 0;
  r.end = after < capacity ? after : capacity;
  if (r.first > r.end) r.first = r.end;
  return r;
}

// Blocks of a row's keys; one where it has none, so that its output is written.
FRZ_RULE uint32_t row_blocks(KeyRange r) {
  if (r.first >= r.end) return 1;
  return (r.end + kBlockKeys - 1) / kBlockKeys - r.first / kBlockKeys;
}

// Blocks of a part: as few as leave no more parts than workgroups run at once.
// A part's time is mostly the same whatever its length (its rows' positions,
// then its pages, then its first keys come one after another), so a second
// round of parts would cost more than longer ones do; and a compute unit takes
// in about 40 GB/s, so few blocks are best spread over as many as there are,
// though three of a workgroup's waves then idle (one request's 5,004 keys: 40
// parts of four blocks 9.6 us, 157 of one 7.6). From four on, in fours. The
// fewest are between the batch's blocks shared out evenly and those shared
// over what the `units` (rows times head blocks) leave, as each has at most one
// part that is not full; `parts` counts a chunk's parts, and six halvings come
// near enough. Where the units alone are more than run at once, an even share
// of half as many parts more, so that what runs last is shorter (300 requests
// of 1,000 to 2,000 keys 112 us by shares of as many, 103 by these; of twice as
// many 113).
FRZ_RULE uint32_t shares(uint32_t units, uint32_t at_once) {
  return units < at_once ? at_once : at_once + at_once / 2;
}
FRZ_RULE uint32_t even_chunk(uint64_t blocks, uint32_t share) {
  const uint64_t even = (blocks + share - 1) / share;
  return (uint32_t)(even <= 2 ? even : (even + kPartWaves - 1) / kPartWaves * kPartWaves);
}
template <typename Count>
FRZ_RULE uint32_t part_chunk(uint64_t blocks, uint32_t units, uint32_t at_once, Count parts) {
  uint32_t low = even_chunk(blocks, shares(units, at_once));
  if (units >= at_once) return low;
  while (low < kPartWaves && parts(low) > at_once) low = low < 2 ? 2 : kPartWaves;
  if (parts(low) <= at_once) return low;
  uint32_t high = even_chunk(blocks, at_once - units);
  for (int i = 0; i < 6 && high - low > kPartWaves; ++i) {
    const uint32_t mid = low + (high - low) / (2 * kPartWaves) * kPartWaves;
    if (parts(mid) <= at_once) high = mid;
    else low = mid;
  }
  return high;
}

// Parts of a row of `blocks`, below 2^20, so that their quotient by the chunk is
// right within one from F32, as a product with each = 1.0f / chunk. (No chunk, of
// a batch without blocks: none.)
FRZ_RULE uint32_t row_parts(uint32_t blocks, uint32_t chunk, float each) {
  uint32_t n = (uint32_t)((float)blocks * each);
  n += n * chunk < blocks;
  n += n * chunk < blocks;
  n -= n > 0 && (n - 1) * chunk >= blocks;
  return n;
}

// The most parts there can be, and the most that belong to rows of several
// parts: such a row has fewer than twice the parts that its blocks fill.
FRZ_RULE uint32_t most_parts(uint32_t units, uint32_t at_once) {
  return units < at_once ? at_once : shares(units, at_once) + units;
}
FRZ_RULE uint32_t most_joined_parts(uint32_t units, uint32_t at_once) {
  return units < at_once ? at_once : 2 * shares(units, at_once);
}

}  // namespace rules
}  // namespace frz
