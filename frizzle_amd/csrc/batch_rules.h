// Where a batch of requests finds its keys and how its work is cut, from
// sizes alone (no HIP, so that a test can compile it by itself).
//
// A request's keys lie in pages: slot s of its key p / page_slots is
// p % page_slots, and the page's number stands in the request's row of the
// table. A row of the batch reads the keys (p - window, p] and its request's
// first `sinks`; those past the table's width, or in a page that the pool does
// not have, are not there. Caches of 8 bits hold a scale for each block of 16
// slots and key-value head.
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

// The keys [first, end) and, apart from them and before, [0, sinks) that a row
// at `position` reads of a sequence whose table holds `capacity`.
struct KeyRange {
  uint32_t first, end, sinks;
};
FRZ_RULE KeyRange key_range(uint32_t position, uint32_t window, uint32_t capacity,
                            uint32_t sinks = 0) {
  KeyRange r;
  const uint32_t after = position + 1;  // position is not kNone
  r.first = after > window ? after - window : 0;
  r.end = after < capacity ? after : capacity;
  if (r.first <= sinks) {  // nothing between
    r.first = r.sinks = 0;
  } else {
    r.sinks = sinks < r.end ? sinks : r.end;
    if (r.first > r.end) r.first = r.end;
  }
  return r;
}

// A row's blocks are counted from its first: those of its sinks, then those of
// [first, end), though the last of the former may be the first of the latter; each
// is looked at for its own keys, so no block has a hole.
struct BlockKeys {
  uint32_t block;       // by position
  uint32_t first, end;  // the keys that its own lie among
};
FRZ_RULE uint32_t sink_blocks(KeyRange r) { return (r.sinks + kBlockKeys - 1) / kBlockKeys; }
FRZ_RULE BlockKeys block_keys(KeyRange r, uint32_t counted) {
  const uint32_t lead = sink_blocks(r);
  BlockKeys b;
  b.block = counted < lead ? counted : counted - lead + r.first / kBlockKeys;
  b.first = counted < lead ? 0 : r.first;
  b.end = counted < lead ? r.sinks : r.end;
  return b;
}

// Blocks of a row's keys; one where it has none, so that its output is written.
FRZ_RULE uint32_t row_blocks(KeyRange r) {
  const uint32_t lead = sink_blocks(r);
  if (r.first >= r.end) return lead ? lead : 1;
  return lead + (r.end + kBlockKeys - 1) / kBlockKeys - r.first / kBlockKeys;
}
// The most blocks of any row.
FRZ_RULE uint64_t most_row_blocks(uint64_t capacity, uint32_t window, uint32_t sinks) {
  const uint64_t held = (capacity + kBlockKeys - 1) / kBlockKeys + (sinks ? 1 : 0);
  const uint64_t seen = (uint64_t)window / kBlockKeys + 2 +
                        ((uint64_t)sinks + kBlockKeys - 1) / kBlockKeys;
  const uint64_t most = held < seen ? held : seen;
  return most ? most : 1;
}

// Whether no row is cut, for their most blocks: up to kFewValues (blocks times head_dim)
// always (64 requests of up to 250 keys, 256 wide, 12.6 us cut, 10.8 whole), to
// kManyValues where the units keep the compute units at work (100 of a window of 512:
// 22.6 and 17.2; but 16: 11.9 and 16.0). No further, though a window leaves rows alike
// that have outgrown it: of those that have not, the longest is still at it when the
// others are done (130 rows of 100 to 2,000 keys, window 2,000, F16, 256 wide, 37 us cut,
// 51 whole; 300 74 and 84), and one more unit than runs at once is a second round.
// A row of 8 bits takes 6 us and 0.3 a block, whatever its width but for the narrowest's
// 0.2, and is then as short as cut ones' two launches (256 wide, whole and cut, of rows
// past the window, of 100 to 2,000 keys, of one of those among some of 100): 32 rows,
// window 400, 10.5 and 10.7, 10.4 and 10.6, 10.0 and 10.3; but window 600 12.0 and 11.3,
// 11.9 and 11.1, 11.2 and 10.3; 100 rows, window 1,000, 17.1 and 19.6, 17.1 and 17.2,
// 15.5 and 14.3; but window 1,400 21.3 and 23.1, 20.9 and 18.8, 19.9 and 14.2.
constexpr uint64_t kFewValues = 2048, kManyValues = 8192;
constexpr uint64_t kFewBlocksI8 = 16, kManyBlocksI8 = 36;
FRZ_RULE bool uncut(uint64_t blocks, uint32_t head_dim, bool i8, uint32_t units,
                    uint32_t compute_units) {
  const bool few = 8ull * units < 3ull * compute_units;
  if (blocks * head_dim <= (few ? kFewValues : kManyValues)) return true;
  return i8 && blocks <= (few ? kFewBlocksI8 : kManyBlocksI8);
}

// ---- caches of 8 bits ----------------------------------------------------------

constexpr uint32_t kScaleSlots = 16;  // tokens that share a scale
constexpr int kMostCode = 127;

// The least power of two, from 2^-126 to 2^121, of which kMostCode reach `most`
// (at least 0, not NaN; past 127 * 2^121 the last), as its F32 bits; 0 for 0.
FRZ_RULE uint32_t block_scale_bits(uint32_t most_bits) {
  if (most_bits == 0) return 0;
  // 1.m * 2^x is 127 * 2^(x - 6) at most where 1.m is 127 / 64 at most.
  const int power = (int)(most_bits >> 23) - 6 + ((most_bits & 0x7FFFFFu) > 0x7E0000u);
  return (uint32_t)(power < 1 ? 1 : power > 248 ? 248 : power) << 23;
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

// Blocks of each part of a row cut into several, the last perhaps fewer: as even as
// fours leave them, not the chunk's and a rest (64 rows of 6,250 keys, 4 key-value
// heads, 256 wide, of 8 bits, a part or two each: 187 us by rests, 155 so).
FRZ_RULE uint32_t row_chunk(uint32_t blocks, uint32_t parts, uint32_t chunk) {
  if (parts < 2 || chunk < kPartWaves) return chunk;
  const uint32_t each = (blocks + parts - 1) / parts;
  return (each + kPartWaves - 1) / kPartWaves * kPartWaves;
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
