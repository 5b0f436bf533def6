// Attention of a batch's rows, one token each, over caches in pages.
//
// A row's keys are cut into parts (batch_rules.h), a workgroup each: one
// key-value head and up to 16 of its query heads. A wave takes every fourth
// of the part's blocks of 32 keys with a running maximum m, sum l and output
// O of its own; the part's waves are joined through LDS, the parts of a row
// that has several by a second launch, in order. Short rows are not cut, and
// many short ones a wave each (launch_shape).
//
// What bounds it is the stream of key and value rows, so nothing of it waits:
// both go from memory to the registers that the matrix instructions read,
// with no LDS between, the next block's keys requested as soon as a block's
// scores are formed, its values as soon as the block's are used.
//   S^T = K q^T   16 keys a tile, A = K: lane (n, g) holds 8 of key n's
//                 values, as they lie in memory. It leaves the lane with the
//                 scores of head n at keys 4g .. 4g + 3.
//   O^T += V^T P  B = P: those same keys, of both of a block's tiles, are
//                 the lane's 8 of the 32 that an instruction sums, so P needs
//                 no move; A = V: the lane's 8 keys' rows at dimensions 8n ..,
//                 paired up two keys a register by v_perm. O^T leaves each
//                 lane one head, so m and l stay a lane's own.
// A row's first keys, where it has them apart from its window's, are blocks of
// their own before the window's, each looked at for its own keys alone.
//
// The matrix cores take 16-bit operands, the cache's type; the query and the
// weights are F32. Each is split into parts that add up to it, hi + lo of F16
// (to one F32 ulp, 2^-23) or three of BF16 (all 24 bits), which are further
// columns of the same instruction where the heads leave some free: columns n and
// n + W belong to one head, W the next of 4, 8 or 16 above the heads. A third
// part of F16 had cost 61 requests of 40 to 8,192 keys 23.2 -> 24.9 us, groups of
// 16 heads up to 19%, for that last ulp, which is less than the scores' sums
// round. A head's query is scaled by a power of two, for F16 to lie below 2^15,
// and its low part by 2^12 more, which that column's scores are divided by: a
// value down to 2^-28 of the head's largest is held to its ulp, and one below
// to 2^-51 of that (as it was, rounded by F16's smallest values to 2^-40). Weights
// are 2^14 at the running maximum, for the same reason, and held to 2^-39 of it.
// For BF16, whose range is F32's, the query lies below 2^-8 (one past 2^104 2^113
// below itself) and weights are at most 2^-24, so that no sum of finite keys' or
// values' products leaves it where scores do not (of scores below 2^23, from which
// on F32 does not hold the maximum 24 above). All scales are exact, products are
// exact in F32, sums F32.
//
// A cache of 8 bits is whole numbers c, -127 to 127, and a scale s of each 16 slots
// of a head, which is half a block, so that both scales are the wave's own numbers:
//   S = (q . c) s_k     on the matrix cores' whole numbers, 64 a turn: keys go in as
//                       they lie in memory, the query as four digits of 8 bits,
//                       columns n, n + W, n + 2W .. of a head, or further tiles. It
//                       is held to 2^-30 of its head's largest; sums are exact.
//   O = (p s_v / t) . c t  on those of F16: a byte and a constant make each c exact,
//                       p s_v / t is split as above. t is the largest s_v so far
//                       (of numbers that are not all 0), the outputs' unit, kept as m
//                       is: weights stay below 2^14, and a part leaves its outputs
//                       over its weights, so that no sum is past F32 where no value
//                       is.
// Values' bytes as F16 are half of a block's 330 vector instructions (256 wide); the
// query's digits spare the keys' as many.
//
// Keys outside the row's range or in no page are never read: their rows are
// zeros, and their scores -inf.
//
// Whole calls, 256 wide, F16 but where said: three requests of 98,001 to
// 131,072 keys over 4 key-value heads (1.4 GB) 235 us, 6.0 TB/s; 61 of 40 to
// 8,192 keys (99 MB) 24.5 us, 4.0 TB/s; 32 of 1 to 4,001 keys, 8 BF16 key-value
// heads of 128 (70 MB), 20.0 us, 3.5 TB/s; one of 5,004 keys (5 MB) 10.1 us,
// two launches of dependent loads. The same of 8 bits: 130 us (702 MB, 5.4 TB/s),
// 16.6, 16.0 and 10.9. 29 requests' first 130 and last 4,000 keys, 8 BF16 heads of
// 128 (491 MB), 99 us, 5.0 TB/s.

#include <type_traits>

#include "batch_rules.h"
#include "kernels.h"
#include "numerics.h"

namespace frz {
namespace {

using namespace rules;

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));

constexpr float kMinusInf = -__builtin_inff();
constexpr float kLargest = 0x1.fffffep127f;
constexpr uint64_t kWaveBlocks = 32;  // of rows that go a wave each: see launch_shape
constexpr int kBufferWord3 = 0x00020000;  // raw 32-bit data
constexpr uint32_t kDies = 8;  // workgroups go to them in turn
constexpr float kLeastTop = 0x1p-126f;
constexpr float kCodeUnit = 1024.0f;  // what a value's number of 8 bits is the 2^-10 of

template <CacheFormat kF>
struct Types;
template <>
struct Types<kCacheF16> {
  typedef half8 vec;
  typedef _Float16 scalar;
  static constexpr int kParts = 2;
  static constexpr int kQueryTop = 14;          // the query's largest lies in [2^14, 2^15)
  static constexpr float kPartScale = 4096.0f;  // of a query's part to the one before
  static constexpr float kWeightScale = 14.0f;  // the running maximum's weight: 2^14
  static __device__ __forceinline__ f32x4 mfma(uint4 a, uint4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a),
                                                  __builtin_bit_cast(half8, b), c, 0, 0, 0);
  }
};
template <>
struct Types<kCacheBf16> {
  typedef bf16x8 vec;
  typedef __bf16 scalar;
  static constexpr int kParts = 3;
  static constexpr int kQueryTop = -9;  // the sum of 256 products of any key is finite
  static constexpr float kPartScale = 1.0f;
  static constexpr float kWeightScale = -24.0f;  // the sum of 2^24 such weights of any value is finite
  static __device__ __forceinline__ f32x4 mfma(uint4 a, uint4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};

// Numbers of 8 bits are F16 to their weights.
constexpr int kDigits = 4;  // of a query
template <>
struct Types<kCacheI8> : Types<kCacheF16> {
  static constexpr int kQueryTop = 29;
  static constexpr int kMostUp = 138;  // the query is at most 2^138 times itself
  static __device__ __forceinline__ i32x4 mfma_digits(uint4 a, uint4 b, i32x4 c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a),
                                                 __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
  }
};

// The shapes a kernel is compiled for.
template <int kD, CacheFormat kF, int kW>
struct Shape {
  static constexpr bool kI8 = kF == kCacheI8;
  static constexpr int kBytes = kI8 ? 1 : 2;                            // of a cached value
  static constexpr int kParts = Types<kF>::kParts;
  static constexpr int kPerTile = 16 / kW;                              // parts a column tile holds
  static constexpr int kTiles = (kParts + kPerTile - 1) / kPerTile;     // column tiles
  static constexpr int kQueryTiles = kI8 ? kDigits / kPerTile : kTiles;
  // Tiles whose query is not scaled alike, and so whose sums are apart.
  static constexpr int kScales = kF == kCacheBf16 ? 1 : kQueryTiles;
  static constexpr bool kSpare = kTiles * kPerTile > kParts;            // columns of no part
  static constexpr int kPiece = 16 / kBytes;                            // of a key row that a lane loads
  static constexpr int kChunks = kD / (4 * kPiece);                     // of a key row
  // Values of a value row that a lane loads at once, and how often.
  static constexpr int kVec = kI8 ? kD / 16 : kD >= 128 ? 8 : 4;
  static constexpr int kSpans = kD / (16 * kVec);
  static constexpr int kWords = (kVec * kBytes + 3) / 4;
};

// Workgroups a compute unit runs at once, by the registers that a shape takes; 256 wide
// of 8 bits one, though two would fit (61 requests 16.4 us, 18.7 by two; long ones 130
// and 134).
template <int kD, CacheFormat kF, int kW>
constexpr int kWorkgroups = kD == 256   ? 1
                            : kD == 128 ? (Shape<kD, kF, kW>::kTiles == 1 ? 3 : 2)
                                        : (Shape<kD, kF, kW>::kTiles <= 2 ? 4 : 3);
template <int kD, CacheFormat kF, int kW>
constexpr bool kFits = kWorkgroups<kD, kF, kW> <= kAttentionWorkgroups &&
                       kWorkgroups<kD, kF, kW> * kD <= kAttentionWidth;

// A column's part of a value: what rounding it left to the parts before, taken
// off (`less` holds -1 for each of those, 0 for the others), rounded in its turn.
template <CacheFormat kF>
struct Column {
  static constexpr bool kBf16 = kF == kCacheBf16;
  typedef typename Types<kF>::scalar T;
  float keep;     // 1; 0 for a column past the format's parts
  float less[2];
  float scale;    // of a query's part
  Column() = default;
  __device__ __forceinline__ explicit Column(int part) {
    keep = part < Types<kF>::kParts ? 1.0f : 0.0f;
    less[0] = part >= 1 ? -1.0f : 0.0f;
    less[1] = part >= 2 ? -1.0f : 0.0f;
    scale = !kBf16 && part == 1 ? Types<kF>::kPartScale : 1.0f;
  }
  __device__ __forceinline__ T part_of(float x) const {
    x = fmaf_(less[0], (float)(T)x, x);
    if constexpr (kBf16) x = fmaf_(less[1], (float)(T)x, x);
    return (T)x;
  }
  __device__ __forceinline__ T scaled_part_of(float x) const {
    if constexpr (kBf16) return part_of(x);
    return (T)(fmaf_(less[0], (float)(T)x, x) * scale);
  }
};

// x of the lanes 32 and 16 away, reduced with the lane's own: every lane of
// the four that share n = lane % 16 gets all four's result.
template <typename Op>
__device__ __forceinline__ float across_groups(float x, Op op) {
  float a = x, b = x;
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b));
  x = op(a, b);
  a = x;
  b = x;
  asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(a), "+v"(b));
  return op(a, b);
}

template <int kShift>
__device__ __forceinline__ float row_rotated(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x),
                                                               0x120 + kShift, 0xF, 0xF, true));
}

// All 64 lanes' x, into each of them: by lanes 32, 16, 8 .. 1 away in turn.
template <typename Op>
__device__ __forceinline__ float across_wave(float x, Op op) {
  x = across_groups(x, op);
  x = op(x, row_rotated<8>(x));
  x = op(x, row_rotated<4>(x));
  x = op(x, row_rotated<2>(x));
  return op(x, row_rotated<1>(x));
}

// A head's columns summed, into each of them.
template <int kW>
__device__ __forceinline__ float across_columns(float x) {
  if constexpr (kW <= 8) x += row_rotated<8>(x);
  if constexpr (kW <= 4) x += row_rotated<4>(x);
  return x;
}

// x of the lanes up to this one, summed (DPP: row_shr 1, 2, 4, 8, then the
// rows' last lanes broadcast to the rows after).
template <int kCtrl, int kRows>
__device__ __forceinline__ uint32_t add_dpp(uint32_t x) {
  return x + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, kCtrl, kRows, 0xF, false);
}
__device__ __forceinline__ uint32_t wave_sum_to(uint32_t x) {
  x = add_dpp<0x111, 0xF>(x);
  x = add_dpp<0x112, 0xF>(x);
  x = add_dpp<0x114, 0xF>(x);
  x = add_dpp<0x118, 0xF>(x);
  x = add_dpp<0x142, 0xA>(x);
  return add_dpp<0x143, 0xC>(x);
}

// Nothing is moved past here: registers hold one block's rows, not two.
__device__ __forceinline__ void hold() { __builtin_amdgcn_sched_barrier(0); }

__device__ __forceinline__ uint32_t lane_of(uint32_t x, int lane) {
  return (uint32_t)__builtin_amdgcn_readlane((int)x, lane);
}

// What a workgroup works on.
struct Part {
  uint32_t row, position, sequence;
  uint32_t unit;          // the row's head block
  uint32_t index, parts;  // of the unit's parts
  uint32_t chunk;
  uint32_t slot;          // the unit's first state, where it has several parts
  uint32_t record;        // the unit's number among those
  uint32_t records;       // of them
};

// The part numbered `want`, found by each wave for itself from the rows'
// positions, kPer rows a lane: the rows' blocks give the chunk, the chunk each
// row's parts, and those the row. False past the last part (but for the
// records' number).
template <int kPer>
__device__ __forceinline__ bool find_part(const PagedAttentionArgs& a, uint32_t want, int lane,
                                          Part* out) {
  const uint32_t capacity = a.cache.width * a.cache.page_slots;
  uint32_t position[kPer], sequence[kPer], blocks[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) position[i] = a.positions[min((uint32_t)lane * kPer + i, a.rows - 1)];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const uint32_t r = min((uint32_t)lane * kPer + i, a.rows - 1);
    sequence[i] = a.sequences ? a.sequences[r] : r;
  }
  uint32_t mine = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if ((uint32_t)lane * kPer + i >= a.rows) position[i] = kNone;
    const uint32_t held = sequence[i] < a.cache.sequences ? capacity : 0;
    blocks[i] =
        position[i] == kNone ? 0 : row_blocks(key_range(position[i], a.window, held, a.sinks));
    mine += blocks[i];
  }
  const uint32_t all = lane_of(wave_sum_to(mine), 63);
  uint32_t parts[kPer], total, joined;
  auto cut = [&](uint32_t chunk) {
    const float each = 1.0f / (float)(chunk ? chunk : 1);
    total = joined = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint32_t n = row_parts(blocks[i], chunk, each);
      parts[i] = n;
      total += n;
      joined += n > 1 ? n + (1u << 20) : 0;  // parts, and rows above them
    }
  };
  const uint32_t chunk =
      part_chunk((uint64_t)all * a.units, a.rows * a.units, a.at_once, [&](uint32_t c) {
        cut(c);
        return lane_of(wave_sum_to(total), 63) * a.units;
      });
  cut(chunk);
  // Sums of rows' parts stay below 2^20, all their parts of one head block.
  const uint32_t to = wave_sum_to(total), joined_to = wave_sum_to(joined);
  out->records = (lane_of(joined_to, 63) >> 20) * a.units;
  const uint64_t owners = __ballot(want < to * a.units);
  if (owners == 0) return false;
  const int leader = __builtin_ctzll(owners);  // the first lane whose parts reach past `want`
  uint32_t rest = want - (to - total) * a.units, joined_before = joined_to - joined;
  uint32_t row = 0, position_ = 0, sequence_ = 0, blocks_ = 0, parts_ = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const bool here = parts_ == 0 && rest < parts[i] * a.units;
    row = here ? lane * kPer + i : row;
    position_ = here ? position[i] : position_;
    sequence_ = here ? sequence[i] : sequence_;
    blocks_ = here ? blocks[i] : blocks_;
    parts_ = here ? parts[i] : parts_;
    const bool past = parts_ == 0;
    rest -= past ? parts[i] * a.units : 0;
    joined_before += past && parts[i] > 1 ? parts[i] + (1u << 20) : 0;
  }
  out->row = lane_of(row, leader);
  out->position = lane_of(position_, leader);
  out->sequence = lane_of(sequence_, leader);
  out->parts = lane_of(parts_, leader);
  rest = lane_of(rest, leader);
  joined_before = lane_of(joined_before, leader);
  out->chunk = row_chunk(lane_of(blocks_, leader), out->parts, chunk);
  // Neighbouring workgroups take the head blocks of the same keys, whose
  // rows lie side by side.
  out->unit = rest % a.units;
  out->index = rest / a.units;
  const uint32_t mask = (1u << 20) - 1;
  out->slot = (joined_before & mask) * a.units + out->unit * out->parts;
  out->record = (joined_before >> 20) * a.units + out->unit;
  return true;
}

template <int kD, CacheFormat kF, int kW, int kWaves, bool kWhole>
__global__ __launch_bounds__(64 * kWaves, (kWorkgroups<kD, kF, kW>))
void paged_attention_kernel(PagedAttentionArgs a) {
  typedef Shape<kD, kF, kW> S;
  typedef Types<kF> T;
  constexpr int kPitch = kD + 8;  // floats a head's outputs take in LDS
  __shared__ __attribute__((aligned(16))) float joined_out[kWaves][kW * kPitch];
  __shared__ float joined_m[kWaves][kW], joined_l[kWaves][kW], joined_top[kWaves];
  // Of 8 bits the waves share the query's digits, a wave every fourth piece of them (61
  // requests 16.4 us, 17.9 by waves of all their own). Of 16 bits, whose parts take
  // fewer instructions, a row of few keys waits longer for it than it spares (one of
  // 5,004 10.1 -> 10.4 us, though 61 24.5 -> 23.8).
  constexpr int kOwn = S::kI8 ? (S::kChunks + kWaves - 1) / kWaves : S::kChunks;
  constexpr bool kShared = S::kI8 && kWaves > 1;
  __shared__ uint4 digits[kShared ? S::kQueryTiles * S::kChunks : 1][64];
  __shared__ float largest[kShared ? kWaves : 1][16];
  const int lane = threadIdx.x & 63;
  const uint32_t wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int n = lane & 15, g = lane >> 4;

  // Head blocks that read the same lines go to one die, whose cache then has each once.
  uint32_t want = blockIdx.x;
  if (a.shared_units > 1) {
    const uint32_t in_die = blockIdx.x / kDies;
    want = (in_die / a.shared_units * kDies + blockIdx.x % kDies) * a.shared_units +
           in_die % a.shared_units;
  }
  Part part;
  if constexpr (kWhole) {
    if (want >= a.rows * a.units) return;
    part.row = want / a.units;
    part.unit = want % a.units;
    part.position = a.positions[part.row];
    if (part.position == kNone) return;
    part.sequence = a.sequences ? a.sequences[part.row] : part.row;
    part.index = 0;
    part.parts = 1;
    part.chunk = kMostKeys / kBlockKeys;
  } else {
    const bool found = a.rows <= 64 ? find_part<1>(a, want, lane, &part)
                                    : find_part<kMostRows / 64>(a, want, lane, &part);
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.record_count = part.records;
    if (!found) return;
  }
  const uint32_t head_blocks = a.units / a.cache.kv_heads;
  const uint32_t kv = part.unit / head_blocks;
  const uint32_t group = a.query_heads / a.cache.kv_heads;
  const uint32_t head0 = kv * group + part.unit % head_blocks * kHeadBlock;
  const uint32_t heads = min(group - part.unit % head_blocks * kHeadBlock, kHeadBlock);

  // The part's keys and the wave's blocks of them.
  const uint32_t held = part.sequence < a.cache.sequences
                            ? a.cache.width * a.cache.page_slots : 0;
  const KeyRange keys = key_range(part.position, a.window, held, a.sinks);
  const uint32_t last_block = min((part.index + 1) * part.chunk, row_blocks(keys));
  const uint32_t first_block = part.index * part.chunk;

  // The wave's next 32 blocks' pages, a lane a half block of 16 keys: where
  // that half's first key lies in the pool, in values, or ~0; of 8 bits its
  // keys' and values' scales too.
  const uint32_t row_values = a.cache.kv_heads * kD, row_bytes = S::kBytes * row_values;
  uint64_t pages = ~0ull;
  float key_scales = 0.0f, value_scales = 0.0f;
  auto find_pages = [&](uint32_t counted) {
    const BlockKeys b = block_keys(keys, counted + kWaves * (lane >> 1));
    const uint32_t key = b.block * kBlockKeys + 16 * (lane & 1);
    pages = ~0ull;
    key_scales = value_scales = 0.0f;
    if (key < b.end && key + 16 > b.first) {
      const uint32_t index = key / a.cache.page_slots;
      const uint32_t page = page_at(a.cache.table, a.cache.sequences, a.cache.width,
                                    a.cache.pages, part.sequence, index);
      if (page != kNone) {
        const uint32_t slot = key - index * a.cache.page_slots;
        pages = page * a.cache.page_stride + (uint64_t)slot * row_values;
        if constexpr (S::kI8) {
          const uint64_t at = page * a.cache.scale_stride +
                              (uint64_t)(slot / kScaleSlots) * a.cache.kv_heads + kv;
          key_scales = a.cache.key_scales[at];
          value_scales = a.cache.value_scales[at];
        }
      }
    }
  };
  uint32_t block = first_block + wave;
  find_pages(block);

  // The query's columns: column n of tile t is part t kPerTile + n / W of
  // head n % W; a column past the heads takes the first one's query.
  const uint32_t head = n % kW;
  Column<kF> columns[S::kTiles];
#pragma unroll
  for (int t = 0; t < S::kTiles; ++t) columns[t] = Column<kF>(t * S::kPerTile + n / kW);
  float x[kOwn][S::kPiece];
  {
    const float* src =
        a.query + (uint64_t)part.row * a.q_stride + (uint64_t)(head0 + (head < heads ? head : 0)) * kD;
#pragma unroll
    for (int c = 0; c < kOwn; ++c)
#pragma unroll
      for (int i = 0; i < S::kPiece; i += 4) {
        // (A wave past the last piece takes that again.)
        const int at = kShared ? min(c * kWaves + (int)wave, S::kChunks - 1) : c;
        const float4 v = *reinterpret_cast<const float4*>(src + S::kPiece * (4 * at + g) + i);
        x[c][i] = v.x;
        x[c][i + 1] = v.y;
        x[c][i + 2] = v.z;
        x[c][i + 3] = v.w;
      }
  }

  const uint32_t head_bytes = S::kBytes * kD * kv;
  const uint8_t* key_pool = static_cast<const uint8_t*>(a.cache.keys) + head_bytes;
  const uint8_t* value_pool = static_cast<const uint8_t*>(a.cache.values) + head_bytes;

  // A block: where the rows that are read of each of its halves begin, and
  // which of its 16 keys these are, [lo, hi).
  struct Block {
    uint64_t at[2];
    int lo[2], hi[2];
    uint32_t turn;  // of those whose pages are known
  };
  auto locate = [&](uint32_t counted, uint32_t turn, Block* k) {
    const BlockKeys b = block_keys(keys, counted);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint64_t page = (uint64_t)lane_of((uint32_t)(pages >> 32), 2 * turn + h) << 32 |
                            lane_of((uint32_t)pages, 2 * turn + h);
      const int key = (int)(b.block * kBlockKeys + 16 * h);
      k->lo[h] = max(0, (int)b.first - key);
      k->hi[h] = page == ~0ull ? 0 : min(16, (int)b.end - key);
      const bool some = k->lo[h] < k->hi[h];
      k->at[h] = some ? page + (uint64_t)k->lo[h] * row_values : 0;
      k->hi[h] = some ? k->hi[h] : k->lo[h];
    }
    k->turn = turn;
    return k->lo[0] < k->hi[0] || k->lo[1] < k->hi[1];
  };
  // Rows come through a buffer of just those that are read: a lane whose row is
  // before its start or past its end gets zeros, and no memory is touched.
  auto rows_of = [&](const uint8_t* pool, const Block& k, int h) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(pool + S::kBytes * k.at[h]), 0,
                                             (k.hi[h] - k.lo[h]) * (int)row_bytes, kBufferWord3);
  };
  // Where a lane's first row would begin, were it the first that is read.
  const int key_at = n * (int)row_bytes + 16 * g;
  const int value_at = 4 * g * (int)row_bytes + S::kBytes * S::kVec * n;
  uint4 key_rows[2][S::kChunks];
  auto load_keys = [&](const Block& k) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const __amdgpu_buffer_rsrc_t rows = rows_of(key_pool, k, h);
      const int at = key_at - k.lo[h] * (int)row_bytes;
#pragma unroll
      for (int c = 0; c < S::kChunks; ++c)
        key_rows[h][c] = __builtin_bit_cast(
            uint4, __builtin_amdgcn_raw_buffer_load_b128(rows, at + 64 * c, 0, 0));
    }
  };
  uint4 value_rows[2][4][S::kSpans];
  auto load_values = [&](const Block& k) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const __amdgpu_buffer_rsrc_t rows = rows_of(value_pool, k, h);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int at = value_at + (e - k.lo[h]) * (int)row_bytes;
#pragma unroll
        for (int s = 0; s < S::kSpans; ++s) {
          if constexpr (S::kWords == 4) {
            value_rows[h][e][s] = __builtin_bit_cast(
                uint4, __builtin_amdgcn_raw_buffer_load_b128(rows, at + 256 * s, 0, 0));
          } else if constexpr (S::kWords == 2) {
            const uint2 v = __builtin_bit_cast(
                uint2, __builtin_amdgcn_raw_buffer_load_b64(rows, at, 0, 0));
            value_rows[h][e][s] = make_uint4(v.x, v.y, 0, 0);
          } else {
            value_rows[h][e][s] = make_uint4(
                __builtin_bit_cast(uint32_t, __builtin_amdgcn_raw_buffer_load_b32(rows, at, 0, 0)),
                0, 0, 0);
          }
        }
      }
    }
  };

  f32x4 out[S::kSpans][S::kVec];
#pragma unroll
  for (int s = 0; s < S::kSpans; ++s)
#pragma unroll
    for (int j = 0; j < S::kVec; ++j) out[s][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float m = kMinusInf, l = 0.0f;  // m less T::kWeightScale, once there is a key
  // Of 8 bits: the largest of the values' scales so far, that the outputs are in.
  float top_scale = kLeastTop, each_top = 1.0f / kLeastTop;

  uint32_t turn = 0;
  Block now, next;
  // The first block from `block` on that holds a key; `turn` counts the
  // blocks whose pages are known.
  auto seek = [&](Block* k) {
    for (; block < last_block; block += kWaves, ++turn) {
      if (turn == 32) {
        find_pages(block);
        turn = 0;
      }
      if (locate(block, turn, k)) return true;
    }
    k->at[0] = k->at[1] = 0;
    k->lo[0] = k->lo[1] = k->hi[0] = k->hi[1] = 0;  // no row
    return false;
  };
  const bool some = seek(&now);
  if (S::kI8 || some) {
    load_keys(now);
    load_values(now);
    hold();
    float scale[S::kQueryTiles];  // what turns the scaled query's products into log2 units
    float key_back = 0.0f, key_rest = 1.0f;  // of 8 bits: the key's scale aside
    uint4 q[S::kQueryTiles][S::kChunks];
    if constexpr (S::kI8) {
      // The query as whole numbers below 2^30, four digits of -128 to 127 each:
      // adding 128 of every digit makes them a word's bytes, 128 too large each,
      // which flipping the bytes' top bits takes off again.
      float most = 0.0f;  // NaN where one is
#pragma unroll
      for (int c = 0; c < kOwn; ++c)
#pragma unroll
        for (int i = 0; i < S::kPiece; ++i)
          most = __builtin_elementwise_maximum(most, __builtin_fabsf(x[c][i]));
      most = across_groups(most, [](float p, float r) { return __builtin_elementwise_maximum(p, r); });
      if constexpr (kShared) {
        if (g == 0) largest[wave][n] = most;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWaves; ++w)
          most = __builtin_elementwise_maximum(most, largest[w][n]);
      }
      int up = 127 + T::kQueryTop - (int)(float_to_bits(most) >> 23);
      up = up > T::kMostUp ? T::kMostUp : up;
      // Of a power below 2^-100 the rest is a factor of its own, so that what meets the
      // blocks' scales, which may make up for it, has all of its bits; it is 0 only
      // where scores are below 2^-70.
      const int power = __builtin_amdgcn_frexp_expf(a.scale_log2e) - up;
      const int here = power < -100 ? -100 : power;
      key_back = __builtin_ldexpf(__builtin_amdgcn_frexp_mantf(a.scale_log2e), here);
      key_rest = __builtin_ldexpf(1.0f, power - here);
      if (!(most <= kLargest)) key_back = __builtin_nanf("");
#pragma unroll
      for (int t = 0; t < S::kQueryTiles; ++t) {
        const uint32_t digit = t * S::kPerTile + n / kW;
        scale[t] = bits_to_float((127 + 8 * digit) << 23);
        // Byte `digit` of two words, next to each other.
        const uint32_t pick = digit | (4 + digit) << 8 | 0x0C0C0000u;
#pragma unroll
        for (int c = 0; c < kOwn; ++c) {
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t z[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
              z[j] = (uint32_t)(int)rint_(__builtin_ldexpf(x[c][4 * i + j], up)) + 0x80808080u;
            w[i] = (__builtin_amdgcn_perm(z[1], z[0], pick) |
                    __builtin_amdgcn_perm(z[3], z[2], pick) << 16) ^ 0x80808080u;
          }
          const uint4 piece = make_uint4(w[0], w[1], w[2], w[3]);
          if constexpr (kShared) {
            const int at = c * kWaves + (int)wave;
            if (at < S::kChunks) digits[t * S::kChunks + at][lane] = piece;
          } else {
            q[t][c] = piece;
          }
        }
      }
      if constexpr (kShared) {
        __syncthreads();
#pragma unroll
        for (int t = 0; t < S::kQueryTiles; ++t)
#pragma unroll
          for (int c = 0; c < S::kChunks; ++c) q[t][c] = digits[t * S::kChunks + c][lane];
      }
    } else {
      float most = 0.0f;
#pragma unroll
      for (int c = 0; c < S::kChunks; ++c)
#pragma unroll
        for (int i = 0; i < S::kPiece; ++i)
          most = __builtin_fmaxf(most, __builtin_fabsf(x[c][i]));
      most = across_groups(most, [](float p, float r) { return __builtin_fmaxf(p, r); });
      // 2^up takes the largest to its place; zeros and the smallest (and for
      // BF16 the largest) values as far as both factors, and the scale with its
      // own (at most 2^13), stay ordinary numbers.
      int up = 127 + T::kQueryTop - (int)(float_to_bits(most) >> 23);
      up = up > 100 ? 100 : up < -113 ? -113 : up;
      const float factor = bits_to_float((uint32_t)(127 + up) << 23);
      const float back = a.scale_log2e * bits_to_float((uint32_t)(127 - up) << 23);
#pragma unroll
      for (int t = 0; t < S::kTiles; ++t) {
        scale[t] = back / columns[t].scale;
        const float kept = factor * columns[t].keep;
#pragma unroll
        for (int c = 0; c < S::kChunks; ++c) {
          typename T::vec v;
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = columns[t].scaled_part_of(x[c][i] * kept);
          q[t][c] = __builtin_bit_cast(uint4, v);
        }
      }
    }
    for (bool more = some; more;) {
      typedef typename std::conditional<S::kI8, i32x4, f32x4>::type Sums;
      Sums scores[2][S::kScales];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 0; i < S::kScales; ++i) scores[h][i] = Sums{0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < S::kChunks; ++c)
#pragma unroll
          for (int t = 0; t < S::kQueryTiles; ++t) {
            Sums& sum = scores[h][t % S::kScales];
            if constexpr (S::kI8) sum = T::mfma_digits(key_rows[h][c], q[t][c], sum);
            else sum = T::mfma(key_rows[h][c], q[t][c], sum);
          }
      }
      hold();
      // The block's scales, before the lanes may take those of further ones; not with
      // its rows' places, which would make the first rows wait for them.
      float key_scale[2], value_scale[2];
      if constexpr (S::kI8) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          key_scale[h] = bits_to_float(lane_of(float_to_bits(key_scales), 2 * now.turn + h));
          value_scale[h] = bits_to_float(lane_of(float_to_bits(value_scales), 2 * now.turn + h));
        }
      }
      // After the last block, of no rows: a branch around the loads would make
      // each wait one for all that are under way.
      block += kWaves;
      ++turn;
      more = seek(&next);
      load_keys(next);
      hold();

      float most = kMinusInf, weight[8];  // scores first
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float back[S::kScales];
#pragma unroll
        for (int i = 0; i < S::kScales; ++i) {
          back[i] = scale[i];
          if constexpr (S::kI8) {
            // A query past F32 by numbers that are all 0 is 0; NaN stays.
            back[i] *= key_back * key_scale[h] * key_rest;
            back[i] = __builtin_elementwise_minimum(
                __builtin_elementwise_maximum(back[i], -kLargest), kLargest);
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float s = (float)scores[h][0][e] * back[0];
#pragma unroll
          for (int i = 1; i < S::kScales; ++i) s = fmaf_((float)scores[h][i][e], back[i], s);
          s = across_columns<kW>(s);
          const bool live = 4 * g + e >= now.lo[h] && 4 * g + e < now.hi[h];
          weight[4 * h + e] = live ? s : kMinusInf;
          most = __builtin_fmaxf(most, weight[4 * h + e]);
        }
      }
      most = across_groups(most, [](float p, float r) { return __builtin_fmaxf(p, r); });
      // A block that is worked on holds a key, so `most` is a number but where
      // scores are not.
      const float to = __builtin_fmaxf(m, most - T::kWeightScale);
      if (__ballot(to > m)) {
        const float old = __builtin_amdgcn_exp2f(m - to);
        l *= old;
#pragma unroll
        for (int s = 0; s < S::kSpans; ++s)
#pragma unroll
          for (int j = 0; j < S::kVec; ++j) out[s][j] *= old;
        m = to;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        weight[i] = __builtin_amdgcn_exp2f(weight[i] - m);
        l += weight[i];
      }
      if constexpr (S::kI8) {
        // A value's weight has its block's scale in it, over the largest so far of a
        // block that is not all zeros to the row: beside the scale of one that is,
        // whose large values are outside the window or gone, the others' would vanish.
        // (0.1 to 0.3 us a call; to look at the first block only once one far below it
        // is there takes as long, and more registers.)
        auto widest = [&] {
          return __builtin_fmaxf(__builtin_fabsf(value_scale[0]),
                                 __builtin_fabsf(value_scale[1]));
        };
        if (__ballot(widest() > top_scale)) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t any = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
              for (int s = 0; s < S::kSpans; ++s) {
                const uint4& r = value_rows[h][e][s];
                any |= r.x | r.y | r.z | r.w;
              }
            if (!__ballot(any != 0)) value_scale[h] = 0.0f;
          }
        }
        const float here = widest();
        if (__ballot(here > top_scale)) {
          const float old = top_scale / here;
#pragma unroll
          for (int s = 0; s < S::kSpans; ++s)
#pragma unroll
            for (int j = 0; j < S::kVec; ++j) out[s][j] *= old;
          top_scale = here;
          each_top = 1.0f / here;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) weight[i] *= value_scale[i / 4] * each_top;
      }
      uint4 w[S::kTiles];
#pragma unroll
      for (int t = 0; t < S::kTiles; ++t) {
        typename T::vec v;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          v[i] = columns[t].part_of(S::kSpare ? weight[i] * columns[t].keep : weight[i]);
        w[t] = __builtin_bit_cast(uint4, v);
      }
      hold();
#pragma unroll
      for (int s = 0; s < S::kSpans; ++s)
#pragma unroll
        for (int j = 0; j < S::kVec; ++j) {
          // The lane's 8 keys at dimension j of its span.
          constexpr int kIn = 4 / S::kBytes;  // values a word holds
          auto word = [&](int h, int e) {
            const uint4& r = value_rows[h][e][s];
            return j / kIn == 0 ? r.x : j / kIn == 1 ? r.y : j / kIn == 2 ? r.z : r.w;
          };
          auto pair = [&](int h, int e) {
            if constexpr (S::kI8) {
              // Bytes of 0 to 255, as F16's smallest values u 2^-24: to (u - 128) 2^-10.
              const uint32_t select = 0x0C040C00u + 0x00010001u * (j % 4);
              const half2v u = __builtin_bit_cast(
                  half2v, __builtin_amdgcn_perm(word(h, e + 1) ^ 0x80808080u,
                                                word(h, e) ^ 0x80808080u, select));
              const _Float16 up = (_Float16)16384.0f, less = (_Float16)-0.125f;
              return __builtin_bit_cast(
                  uint32_t, __builtin_elementwise_fma(u, half2v{up, up}, half2v{less, less}));
            } else {
              const uint32_t select = j & 1 ? 0x07060302u : 0x05040100u;
              return __builtin_amdgcn_perm(word(h, e + 1), word(h, e), select);
            }
          };
          const uint4 v = make_uint4(pair(0, 0), pair(0, 2), pair(1, 0), pair(1, 2));
#pragma unroll
          for (int t = 0; t < S::kTiles; ++t) out[s][j] = T::mfma(v, w[t], out[s][j]);
          if (j & 1) hold();
        }
      hold();
      load_values(next);
      hold();
      now = next;
    }
  }

  // The waves' states joined. Lane (n, g) holds dimensions 16 kVec s +
  // kVec (4g + e) + j of its column.
  l = across_groups(l, [](float p, float r) { return p + r; });
  if (g == 0 && n < kW) {
    joined_m[wave][n] = m;
    joined_l[wave][n] = l;
  }
  if (S::kI8 && lane == 0) joined_top[wave] = top_scale;
#pragma unroll
  for (int s = 0; s < S::kSpans; ++s)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float v[S::kVec];
#pragma unroll
      for (int j = 0; j < S::kVec; ++j) v[j] = across_columns<kW>(out[s][j][e]);
      if (n < kW) {
        float* dst = &joined_out[wave][n * kPitch + 16 * S::kVec * s + S::kVec * (4 * g + e)];
#pragma unroll
        for (int j = 0; j < S::kVec; j += 4)
          *reinterpret_cast<float4*>(dst + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
      }
    }
  __syncthreads();
  const bool whole = kWhole || part.parts == 1;
  for (uint32_t i = threadIdx.x; i < heads * (kD / 4); i += 64 * kWaves) {
    const uint32_t h = i / (kD / 4), d = i % (kD / 4) * 4;
    float top = joined_m[0][h];
#pragma unroll
    for (uint32_t w = 1; w < kWaves; ++w) top = __builtin_fmaxf(top, joined_m[w][h]);
    float widest = joined_top[0];
#pragma unroll
    for (uint32_t w = 1; w < kWaves; ++w) widest = __builtin_fmaxf(widest, joined_top[w]);
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float weights = 0.0f;
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) {
      // A wave without a key holds zeros, and so does a row without one.
      const float f = top == kMinusInf ? 0.0f : __builtin_amdgcn_exp2f(joined_m[w][h] - top);
      const float4 o = *reinterpret_cast<const float4*>(&joined_out[w][h * kPitch + d]);
      weights = fmaf_(joined_l[w][h], f, weights);
      const float by = S::kI8 ? f * (joined_top[w] / widest) : f;
      sum.x = fmaf_(o.x, by, sum.x);
      sum.y = fmaf_(o.y, by, sum.y);
      sum.z = fmaf_(o.z, by, sum.z);
      sum.w = fmaf_(o.w, by, sum.w);
    }
    if (S::kI8 || whole) {
      // (Of 8 bits a part's outputs too: their sums' range is the scales'.)
      const float f = weights == 0.0f ? 0.0f : S::kI8 ? kCodeUnit / weights : 1.0f / weights;
      const float unit = S::kI8 ? widest : 1.0f;
      sum.x = sum.x * f * unit;
      sum.y = sum.y * f * unit;
      sum.z = sum.z * f * unit;
      sum.w = sum.w * f * unit;
    }
    if (whole) {
      *reinterpret_cast<float4*>(a.out + (uint64_t)part.row * a.out_stride +
                                 (uint64_t)(head0 + h) * kD + d) = sum;
    } else {
      const uint64_t state = (uint64_t)(part.slot + part.index) * kHeadBlock + h;
      *reinterpret_cast<float4*>(a.states + state * kD + d) = sum;
      if (d == 0) *reinterpret_cast<float2*>(a.stats + 2 * state) = make_float2(top, weights);
    }
  }
  if (!whole && part.index == 0 && threadIdx.x == 0) {
    a.records[part.record] = make_uint4(part.row, head0 | heads << 16, part.parts, part.slot);
  }
}

// The parts of the rows that have several, joined in order: a workgroup a
// (record, head, 64 dimensions), 16 lanes of it the dimensions, four each,
// and its 16 groups every sixteenth part. Some 2 us, a launch and three loads one
// after another. (The last part's workgroup joining them itself would save the
// launch, but read all of a row's states, 640 KB for 157 parts of four heads,
// through one compute unit: 16 us. Rows of few parts so, which have 16 KB in four,
// were not tried.)
constexpr uint32_t kJoinWaves = 4, kThreads = 64 * kJoinWaves, kJoinGroups = kThreads / 16;
// States that a group asks for with the statistics: of up to 64 parts, and of more
// (few parts take 0.5 us longer where all ask for ten, 157 1.5 where all for four).
constexpr uint32_t kEarly = 10, kFew = 4;
template <int kD, bool kI8>
__global__ __launch_bounds__(kThreads) void paged_attention_join_kernel(PagedAttentionArgs a) {
  __shared__ float wave_top[kJoinWaves], wave_sum[kJoinWaves];
  __shared__ float factors[kMostJoinedParts];
  __shared__ float4 sums[kJoinGroups][16];
  const uint32_t t = threadIdx.x, lane = t & 63, wave = t >> 6, group = t / 16;
  // What is read comes in two steps: the records (any first one, were there none),
  // then the statistics with the first states.
  const uint32_t count = *a.record_count;
  uint4 record = a.records[blockIdx.x];
  for (uint32_t i = blockIdx.x; i < count; i += gridDim.x) {
    if (i != blockIdx.x) record = a.records[i];
    const uint32_t h = blockIdx.y / (kD / 64), d = blockIdx.y % (kD / 64) * 64 + t % 16 * 4;
    const uint32_t parts = record.z;
    if (h >= record.y >> 16) continue;
    const uint64_t first = (uint64_t)record.w * kHeadBlock + h;
    auto stats_of = [&](uint32_t p) {
      return *reinterpret_cast<const float2*>(a.stats + 2 * (first + (uint64_t)p * kHeadBlock));
    };
    auto state_of = [&](uint32_t p) {
      return *reinterpret_cast<const float4*>(a.states + (first + (uint64_t)p * kHeadBlock) * kD + d);
    };
    const float2 mine = stats_of(t < parts ? t : 0);
    float4 early[kEarly];
    auto ask = [&](uint32_t k) {
      const uint32_t p = group + k * kJoinGroups;
      early[k] = state_of(p < parts ? p : 0);
    };
#pragma unroll
    for (uint32_t k = 0; k < kFew; ++k) ask(k);
    if (parts > kFew * kJoinGroups) {
#pragma unroll
      for (uint32_t k = kFew; k < kEarly; ++k) ask(k);
    }
    float top = t < parts ? mine.x : kMinusInf;
    for (uint32_t p = t + kThreads; p < parts; p += kThreads)
      top = __builtin_fmaxf(top, stats_of(p).x);
    top = across_wave(top, [](float p, float r) { return __builtin_fmaxf(p, r); });
    __syncthreads();  // the last record's reads are done
    if (lane == 0) wave_top[wave] = top;
    __syncthreads();
    for (uint32_t w = 0; w < kJoinWaves; ++w) top = __builtin_fmaxf(top, wave_top[w]);
    float weights = 0.0f;
    for (uint32_t p = t; p < parts; p += kThreads) {
      const float2 s = p == t ? mine : stats_of(p);
      const float f = top == kMinusInf ? 0.0f : __builtin_amdgcn_exp2f(s.x - top);
      factors[p] = kI8 ? f * s.y : f;  // of 8 bits a part's outputs are over its weights
      weights = fmaf_(s.y, f, weights);
    }
    weights = across_wave(weights, [](float p, float r) { return p + r; });
    if (lane == 0) wave_sum[wave] = weights;
    __syncthreads();
    const float l = wave_sum[0] + wave_sum[1] + wave_sum[2] + wave_sum[3];
    const float each = kI8 && l != 0.0f ? 1.0f / l : 1.0f;  // so that no sum is past the outputs
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto add = [&](uint32_t p, const float4& o) {
      const float f = kI8 ? factors[p] * each : factors[p];
      sum.x = fmaf_(o.x, f, sum.x);
      sum.y = fmaf_(o.y, f, sum.y);
      sum.z = fmaf_(o.z, f, sum.z);
      sum.w = fmaf_(o.w, f, sum.w);
    };
#pragma unroll
    for (uint32_t k = 0; k < kEarly; ++k)
      if (group + k * kJoinGroups < parts) add(group + k * kJoinGroups, early[k]);
#pragma unroll 8
    for (uint32_t p = group + kEarly * kJoinGroups; p < parts; p += kJoinGroups) add(p, state_of(p));
    sums[group][t % 16] = sum;
    __syncthreads();
    if (t < 64) {
      // A lane a dimension.
      const float* column = reinterpret_cast<const float*>(&sums[0][0]) + t;
      float x = 0.0f;
      for (uint32_t k = 0; k < kJoinGroups; ++k) x += column[64 * k];
      a.out[(uint64_t)record.x * a.out_stride + (uint64_t)((record.y & 0xFFFF) + h) * kD +
            blockIdx.y % (kD / 64) * 64 + t] = l == 0.0f ? 0.0f : kI8 ? x : x / l;
    }
  }
}

template <int kD, CacheFormat kF, int kW>
hipError_t launch_shape(hipStream_t s, PagedAttentionArgs a, uint32_t heads, int compute_units) {
  typedef Shape<kD, kF, kW> S;
  static_assert(kFits<kD, kF, kW>, "the workspace holds their parts");
  const uint32_t units = a.rows * a.units;
  a.at_once = kWorkgroups<kD, kF, kW> * (uint32_t)compute_units;
  // Units side by side that read the same lines: a key-value head's head blocks, and two
  // heads of 64 bytes (four rows of 100,000 keys, 16 heads of 64 in 8 bits, 270 -> 215
  // us). Not all of a row's heads, which cost 256-wide ones 4%, and not where a die's
  // compute units do not take them whole, as one would have a workgroup more to do.
  a.shared_units = a.units / a.cache.kv_heads;
  if (kD * S::kBytes < 128 && a.cache.kv_heads % 2 == 0) a.shared_units *= 2;
  if (a.at_once % (kDies * a.shared_units) != 0) a.shared_units = 1;
  auto grid = [&](uint64_t n) {
    const uint32_t even = a.shared_units > 1 ? kDies * a.shared_units : 1;
    return dim3((uint32_t)((n + even - 1) / even * even));
  };
  // The most blocks that a row can have. Where they are few (uncut), each unit is one
  // workgroup's (kWhole), which then need not find its part, nor leave a state to a
  // second launch. Where more units are there than workgroups run at once, a unit is a
  // wave's: four waves would each have had a block or two of a short row (483 rows of 16
  // to 31 keys, 8 key-value heads, 256 wide, 127 us and 35; 512 of a window of 512 67 and
  // 52; not of 63 blocks, 400 rows of 8 heads 128 wide: 214 by workgroups, 257 by waves).
  // The host knows the table's width and the window, not the rows: short rows in a wide
  // table without a window are cut (those 483 take the 127).
  const uint64_t capacity = (uint64_t)a.cache.width * a.cache.page_slots;
  const uint64_t blocks = most_row_blocks(capacity, a.window, a.sinks);
  // Of 8 bits a workgroup's waves are through a row sooner, so that rows go a wave each
  // only if they have few blocks: one where all units' workgroups run at once, up to 12
  // where nearly every wave that does has a unit, kWaveBlocks from there on (128 requests
  // of 10 to 500 keys, 8 heads of 128, 21.2 us by waves, 15.1 by workgroups; 200 of 1 to
  // 64 8.0 and 10.9).
  uint64_t most = kWaveBlocks;
  if (S::kI8) {
    const uint32_t held = a.at_once * (kD == 256 && kW < 16 ? 2 : 1);  // two fit, though
    if (units < kPartWaves * held)
      most = units > held ? 1 + (uint64_t)kPartWaves * (units - held) / held : 1;
  }
  if (units >= a.at_once && blocks <= most) {
    hipLaunchKernelGGL((paged_attention_kernel<kD, kF, kW, 1, true>), grid(units), dim3(64), 0,
                       s, a);
    return hipGetLastError();
  }
  if (uncut(blocks, kD, S::kI8, units, (uint32_t)compute_units)) {
    hipLaunchKernelGGL((paged_attention_kernel<kD, kF, kW, kPartWaves, true>), grid(units),
                       dim3(64 * kPartWaves), 0, s, a);
    return hipGetLastError();
  }
  // No more parts than the rows have blocks.
  const uint64_t fill = units * blocks;
  const uint64_t bound = most_parts(units, a.at_once);
  hipLaunchKernelGGL((paged_attention_kernel<kD, kF, kW, kPartWaves, false>),
                     grid(fill < bound ? fill : bound), dim3(64 * kPartWaves), 0, s, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const uint32_t joins = most_joined_parts(units, a.at_once) / 2;
  const uint32_t records = units < joins ? units : joins;
  hipLaunchKernelGGL((paged_attention_join_kernel<kD, kF == kCacheI8>),
                     dim3(records < 256 ? records : 256, heads * (kD / 64)), dim3(kThreads), 0, s,
                     a);
  return hipGetLastError();
}

template <int kD>
hipError_t launch_heads(hipStream_t s, PagedAttentionArgs a, int compute_units) {
  const uint32_t group = a.query_heads / a.cache.kv_heads;
  const uint32_t heads = group < kHeadBlock ? group : kHeadBlock;
  a.units = a.cache.kv_heads * ((group + kHeadBlock - 1) / kHeadBlock);
  switch (a.cache.format) {
    case kCacheF16:
      if (heads <= 8) return launch_shape<kD, kCacheF16, 8>(s, a, heads, compute_units);
      return launch_shape<kD, kCacheF16, 16>(s, a, heads, compute_units);
    case kCacheBf16:
      if (heads <= 4) return launch_shape<kD, kCacheBf16, 4>(s, a, heads, compute_units);
      if (heads <= 8) return launch_shape<kD, kCacheBf16, 8>(s, a, heads, compute_units);
      return launch_shape<kD, kCacheBf16, 16>(s, a, heads, compute_units);
    case kCacheI8:
      if (heads <= 4) return launch_shape<kD, kCacheI8, 4>(s, a, heads, compute_units);
      if (heads <= 8) return launch_shape<kD, kCacheI8, 8>(s, a, heads, compute_units);
      return launch_shape<kD, kCacheI8, 16>(s, a, heads, compute_units);
  }
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_paged_attention(hipStream_t s, const PagedAttentionArgs& a, int compute_units) {
  if (a.rows == 0 || a.rows > kMostRows || compute_units <= 0 || compute_units > kMostComputeUnits)
    return hipErrorInvalidValue;
  switch (a.cache.head_dim) {
    case 64: return launch_heads<64>(s, a, compute_units);
    case 128: return launch_heads<128>(s, a, compute_units);
    case 256: return launch_heads<256>(s, a, compute_units);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace frz
