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
// Keys outside the row's range or in no page are never read: their rows are
// zeros, and their scores -inf.
//
// Whole calls, 256 wide, F16 but where said: three requests of 98,001 to
// 131,072 keys over 4 key-value heads (1.4 GB) 235 us, 6.0 TB/s; 61 of 40 to
// 8,192 keys (99 MB) 24.8 us, 4.0 TB/s; 32 of 1 to 4,001 keys, 8 BF16 key-value
// heads of 128 (70 MB), 20.6 us, 3.4 TB/s; one of 5,004 keys (5 MB) 11.0 us,
// two launches of dependent loads.

#include "batch_rules.h"
#include "kernels.h"
#include "numerics.h"

namespace frz {
namespace {

using namespace rules;

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr float kMinusInf = -__builtin_inff();
// Rows of no more blocks than these, or blocks times head_dim, are not cut: see
// launch_shape.
constexpr uint64_t kWaveBlocks = 32, kFewValues = 2048, kManyValues = 8192;
constexpr int kBufferWord3 = 0x00020000;  // raw 32-bit data

template <bool kBf16>
struct Types;
template <>
struct Types<false> {
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
struct Types<true> {
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

// The shapes a kernel is compiled for.
template <int kD, bool kBf16, int kW>
struct Shape {
  static constexpr int kParts = Types<kBf16>::kParts;
  static constexpr int kPerTile = 16 / kW;                              // parts a column tile holds
  static constexpr int kTiles = (kParts + kPerTile - 1) / kPerTile;     // column tiles
  // Tiles whose query is not scaled alike, and so whose sums are apart.
  static constexpr int kScales = kBf16 ? 1 : kTiles;
  static constexpr bool kSpare = kTiles * kPerTile > kParts;            // columns of no part
  static constexpr int kChunks = kD / 32;                               // of a key row
  static constexpr int kVec = kD >= 128 ? 8 : 4;                        // values a lane loads at once
  static constexpr int kSpans = kD / (16 * kVec);                       // of a value row
};

// Workgroups a compute unit runs at once, by the registers that a shape takes.
template <int kD, bool kBf16, int kW>
constexpr int kWorkgroups = kD == 256   ? 1
                            : kD == 128 ? (Shape<kD, kBf16, kW>::kTiles == 1 ? 3 : 2)
                                        : (Shape<kD, kBf16, kW>::kTiles <= 2 ? 4 : 3);
template <int kD, bool kBf16, int kW>
constexpr bool kFits = kWorkgroups<kD, kBf16, kW> <= kAttentionWorkgroups &&
                       kWorkgroups<kD, kBf16, kW> * kD <= kAttentionWidth;

// A column's part of a value: what rounding it left to the parts before, taken
// off (`less` holds -1 for each of those, 0 for the others), rounded in its turn.
template <bool kBf16>
struct Column {
  float keep;     // 1; 0 for a column past the format's parts
  float less[2];
  float scale;    // of a query's part
  Column() = default;
  __device__ __forceinline__ explicit Column(int part) {
    keep = part < Types<kBf16>::kParts ? 1.0f : 0.0f;
    less[0] = part >= 1 ? -1.0f : 0.0f;
    less[1] = part >= 2 ? -1.0f : 0.0f;
    scale = !kBf16 && part == 1 ? Types<kBf16>::kPartScale : 1.0f;
  }
  __device__ __forceinline__ typename Types<kBf16>::scalar part_of(float x) const {
    typedef typename Types<kBf16>::scalar T;
    x = fmaf_(less[0], (float)(T)x, x);
    if constexpr (kBf16) x = fmaf_(less[1], (float)(T)x, x);
    return (T)x;
  }
  __device__ __forceinline__ typename Types<kBf16>::scalar scaled_part_of(float x) const {
    typedef typename Types<kBf16>::scalar T;
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
    blocks[i] = position[i] == kNone ? 0 : row_blocks(key_range(position[i], a.window, held));
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
  uint32_t row = 0, position_ = 0, sequence_ = 0, parts_ = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const bool here = parts_ == 0 && rest < parts[i] * a.units;
    row = here ? lane * kPer + i : row;
    position_ = here ? position[i] : position_;
    sequence_ = here ? sequence[i] : sequence_;
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
  out->chunk = chunk;
  // Neighbouring workgroups take the head blocks of the same keys, whose
  // rows lie side by side.
  out->unit = rest % a.units;
  out->index = rest / a.units;
  const uint32_t mask = (1u << 20) - 1;
  out->slot = (joined_before & mask) * a.units + out->unit * out->parts;
  out->record = (joined_before >> 20) * a.units + out->unit;
  return true;
}

template <int kD, bool kBf16, int kW, int kWaves, bool kWhole>
__global__ __launch_bounds__(64 * kWaves, (kWorkgroups<kD, kBf16, kW>))
void paged_attention_kernel(PagedAttentionArgs a) {
  typedef Shape<kD, kBf16, kW> S;
  typedef Types<kBf16> T;
  constexpr int kPitch = kD + 8;  // floats a head's outputs take in LDS
  __shared__ __attribute__((aligned(16))) float joined_out[kWaves][kW * kPitch];
  __shared__ float joined_m[kWaves][kW], joined_l[kWaves][kW];
  const int lane = threadIdx.x & 63;
  const uint32_t wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int n = lane & 15, g = lane >> 4;

  Part part;
  if constexpr (kWhole) {
    part.row = blockIdx.x / a.units;
    part.unit = blockIdx.x % a.units;
    part.position = a.positions[part.row];
    if (part.position == kNone) return;
    part.sequence = a.sequences ? a.sequences[part.row] : part.row;
    part.index = 0;
    part.parts = 1;
    part.chunk = kMostKeys / kBlockKeys;
  } else {
    const bool found = a.rows <= 64 ? find_part<1>(a, blockIdx.x, lane, &part)
                                    : find_part<kMostRows / 64>(a, blockIdx.x, lane, &part);
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
  const KeyRange keys = key_range(part.position, a.window, held);
  const uint32_t base_block = keys.first / kBlockKeys;
  const uint32_t last_block = base_block + min((part.index + 1) * part.chunk, row_blocks(keys));
  const uint32_t first_block = base_block + part.index * part.chunk;

  // The wave's next 32 blocks' pages, a lane a half block of 16 keys: where
  // that half's first key lies in the pool, in values, or ~0.
  const uint32_t row_values = a.cache.kv_heads * kD, row_bytes = 2 * row_values;
  auto find_pages = [&](uint32_t block) {
    const uint32_t key = (block + kWaves * (lane >> 1)) * kBlockKeys + 16 * (lane & 1);
    uint64_t at = ~0ull;
    if (key < keys.end && key + 16 > keys.first) {
      const uint32_t index = key / a.cache.page_slots;
      const uint32_t page = page_at(a.cache.table, a.cache.sequences, a.cache.width,
                                    a.cache.pages, part.sequence, index);
      if (page != kNone)
        at = page * a.cache.page_stride + (uint64_t)(key - index * a.cache.page_slots) * row_values;
    }
    return at;
  };
  uint32_t block = first_block + wave;
  uint64_t pages = find_pages(block);

  // The query's columns: column n of tile t is part t kPerTile + n / W of
  // head n % W; a column past the heads takes the first one's query.
  const uint32_t head = n % kW;
  Column<kBf16> columns[S::kTiles];
#pragma unroll
  for (int t = 0; t < S::kTiles; ++t) columns[t] = Column<kBf16>(t * S::kPerTile + n / kW);
  float x[S::kChunks][8];
  {
    const float* src =
        a.query + (uint64_t)part.row * a.q_stride + (uint64_t)(head0 + (head < heads ? head : 0)) * kD;
#pragma unroll
    for (int c = 0; c < S::kChunks; ++c) {
      const float4 lo = *reinterpret_cast<const float4*>(src + 32 * c + 8 * g);
      const float4 hi = *reinterpret_cast<const float4*>(src + 32 * c + 8 * g + 4);
      const float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) x[c][i] = v[i];
    }
  }

  const uint16_t* key_pool = a.cache.keys + (uint64_t)kv * kD;
  const uint16_t* value_pool = a.cache.values + (uint64_t)kv * kD;

  // A block: where the rows that are read of each of its halves begin, and
  // which of its 16 keys these are, [lo, hi).
  struct Block {
    uint64_t at[2];
    int lo[2], hi[2];
  };
  auto locate = [&](uint32_t b, uint32_t turn, Block* k) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint64_t page = (uint64_t)lane_of((uint32_t)(pages >> 32), 2 * turn + h) << 32 |
                            lane_of((uint32_t)pages, 2 * turn + h);
      const int key = (int)(b * kBlockKeys + 16 * h);
      k->lo[h] = max(0, (int)keys.first - key);
      k->hi[h] = page == ~0ull ? 0 : min(16, (int)keys.end - key);
      const bool some = k->lo[h] < k->hi[h];
      k->at[h] = some ? page + (uint64_t)k->lo[h] * row_values : 0;
      k->hi[h] = some ? k->hi[h] : k->lo[h];
    }
    return k->lo[0] < k->hi[0] || k->lo[1] < k->hi[1];
  };
  // Rows come through a buffer of just those that are read: a lane whose row is
  // before its start or past its end gets zeros, and no memory is touched.
  auto rows_of = [&](const uint16_t* pool, const Block& k, int h) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(pool + k.at[h]), 0,
                                             (k.hi[h] - k.lo[h]) * (int)row_bytes, kBufferWord3);
  };
  uint4 key_rows[2][S::kChunks];
  auto load_keys = [&](const Block& k) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const __amdgpu_buffer_rsrc_t rows = rows_of(key_pool, k, h);
      const int at = (n - k.lo[h]) * (int)row_bytes + 16 * g;
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
        const int at = (4 * g + e - k.lo[h]) * (int)row_bytes + 2 * S::kVec * n;
#pragma unroll
        for (int s = 0; s < S::kSpans; ++s) {
          if constexpr (S::kVec == 8) {
            value_rows[h][e][s] = __builtin_bit_cast(
                uint4, __builtin_amdgcn_raw_buffer_load_b128(rows, at + 256 * s, 0, 0));
          } else {
            const uint2 v = __builtin_bit_cast(
                uint2, __builtin_amdgcn_raw_buffer_load_b64(rows, at, 0, 0));
            value_rows[h][e][s] = make_uint4(v.x, v.y, 0, 0);
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

  uint32_t turn = 0;
  Block now, next;
  // The first block from `block` on that holds a key; `turn` counts the
  // blocks whose pages are known.
  auto seek = [&](Block* k) {
    for (; block < last_block; block += kWaves, ++turn) {
      if (turn == 32) {
        pages = find_pages(block);
        turn = 0;
      }
      if (locate(block, turn, k)) return true;
    }
    k->at[0] = k->at[1] = 0;
    k->lo[0] = k->lo[1] = k->hi[0] = k->hi[1] = 0;  // no row
    return false;
  };
  if (seek(&now)) {
    load_keys(now);
    load_values(now);
    hold();
    float scale[S::kTiles];  // what turns the scaled query's products into log2 units
    uint4 q[S::kTiles][S::kChunks];
    {
      float most = 0.0f;
#pragma unroll
      for (int c = 0; c < S::kChunks; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) most = __builtin_fmaxf(most, __builtin_fabsf(x[c][i]));
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
    for (bool more = true; more;) {
      f32x4 scores[2][S::kScales];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 0; i < S::kScales; ++i) scores[h][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < S::kChunks; ++c)
#pragma unroll
          for (int t = 0; t < S::kTiles; ++t) {
            f32x4& sum = scores[h][t % S::kScales];
            sum = T::mfma(key_rows[h][c], q[t][c], sum);
          }
      }
      hold();
      // After the last block, of no rows: a branch around the loads would make
      // each wait one for all that are under way.
      block += kWaves;
      ++turn;
      more = seek(&next);
      load_keys(next);
      hold();

      float most = kMinusInf, weight[8];  // scores first
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float s = scores[h][0][e] * scale[0];
#pragma unroll
          for (int i = 1; i < S::kScales; ++i) s = fmaf_(scores[h][i][e], scale[i], s);
          s = across_columns<kW>(s);
          const bool live = 4 * g + e >= now.lo[h] && 4 * g + e < now.hi[h];
          weight[4 * h + e] = live ? s : kMinusInf;
          most = __builtin_fmaxf(most, weight[4 * h + e]);
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
          const uint32_t select = j & 1 ? 0x07060302u : 0x05040100u;
          auto word = [&](int h, int e) {
            const uint4& r = value_rows[h][e][s];
            return (j >> 1) == 0 ? r.x : (j >> 1) == 1 ? r.y : (j >> 1) == 2 ? r.z : r.w;
          };
          auto pair = [&](int h, int e) {
            return __builtin_amdgcn_perm(word(h, e + 1), word(h, e), select);
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
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float weights = 0.0f;
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) {
      // A wave without a key holds zeros, and so does a row without one.
      const float f = top == kMinusInf ? 0.0f : __builtin_amdgcn_exp2f(joined_m[w][h] - top);
      const float4 o = *reinterpret_cast<const float4*>(&joined_out[w][h * kPitch + d]);
      weights = fmaf_(joined_l[w][h], f, weights);
      sum.x = fmaf_(o.x, f, sum.x);
      sum.y = fmaf_(o.y, f, sum.y);
      sum.z = fmaf_(o.z, f, sum.z);
      sum.w = fmaf_(o.w, f, sum.w);
    }
    if (whole) {
      const float f = weights == 0.0f ? 0.0f : 1.0f / weights;
      sum.x *= f;
      sum.y *= f;
      sum.z *= f;
      sum.w *= f;
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
// and its 16 groups every sixteenth part. Some 2 us, a launch and five loads one
// after another. (The last part's workgroup joining them itself would save the
// launch, but read all of a row's states, 640 KB for 157 parts of four heads,
// through one compute unit: 16 us.)
constexpr uint32_t kJoinWaves = 4, kThreads = 64 * kJoinWaves, kJoinGroups = kThreads / 16;
template <int kD>
__global__ __launch_bounds__(kThreads) void paged_attention_join_kernel(PagedAttentionArgs a) {
  __shared__ float wave_top[kJoinWaves], wave_sum[kJoinWaves];
  __shared__ float factors[kMostJoinedParts];
  __shared__ float4 sums[kJoinGroups][16];
  const uint32_t count = *a.record_count;
  const uint32_t t = threadIdx.x, lane = t & 63, wave = t >> 6;
  for (uint32_t i = blockIdx.x; i < count; i += gridDim.x) {
    const uint4 record = a.records[i];
    const uint32_t h = blockIdx.y / (kD / 64), d = blockIdx.y % (kD / 64) * 64 + t % 16 * 4;
    const uint32_t parts = record.z;
    if (h >= record.y >> 16) continue;
    const uint64_t first = (uint64_t)record.w * kHeadBlock + h;
    float top = kMinusInf;
    for (uint32_t p = t; p < parts; p += kThreads)
      top = __builtin_fmaxf(top, a.stats[2 * (first + (uint64_t)p * kHeadBlock)]);
    for (int o = 32; o > 0; o >>= 1) top = __builtin_fmaxf(top, __shfl_xor(top, o));
    __syncthreads();  // the last record's reads are done
    if (lane == 0) wave_top[wave] = top;
    __syncthreads();
    for (uint32_t w = 0; w < kJoinWaves; ++w) top = __builtin_fmaxf(top, wave_top[w]);
    float weights = 0.0f;
    for (uint32_t p = t; p < parts; p += kThreads) {
      const float2 s =
          *reinterpret_cast<const float2*>(a.stats + 2 * (first + (uint64_t)p * kHeadBlock));
      const float f = top == kMinusInf ? 0.0f : __builtin_amdgcn_exp2f(s.x - top);
      factors[p] = f;
      weights = fmaf_(s.y, f, weights);
    }
    for (int o = 32; o > 0; o >>= 1) weights += __shfl_xor(weights, o);
    if (lane == 0) wave_sum[wave] = weights;
    __syncthreads();
    const uint32_t group = t / 16;
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
    for (uint32_t p = group; p < parts; p += kJoinGroups) {
      const float f = factors[p];
      const float4 o = *reinterpret_cast<const float4*>(
          a.states + (first + (uint64_t)p * kHeadBlock) * kD + d);
      sum.x = fmaf_(o.x, f, sum.x);
      sum.y = fmaf_(o.y, f, sum.y);
      sum.z = fmaf_(o.z, f, sum.z);
      sum.w = fmaf_(o.w, f, sum.w);
    }
    sums[group][t % 16] = sum;
    __syncthreads();
    if (t < 64) {
      // A lane a dimension.
      const float* column = reinterpret_cast<const float*>(&sums[0][0]) + t;
      float x = 0.0f;
      for (uint32_t k = 0; k < kJoinGroups; ++k) x += column[64 * k];
      const float l = wave_sum[0] + wave_sum[1] + wave_sum[2] + wave_sum[3];
      a.out[(uint64_t)record.x * a.out_stride + (uint64_t)((record.y & 0xFFFF) + h) * kD +
            blockIdx.y % (kD / 64) * 64 + t] = l == 0.0f ? 0.0f : x / l;
    }
  }
}

template <int kD, bool kBf16, int kW>
hipError_t launch_shape(hipStream_t s, PagedAttentionArgs a, uint32_t heads, int compute_units) {
  static_assert(kFits<kD, kBf16, kW>, "the workspace holds their parts");
  const uint32_t units = a.rows * a.units;
  a.at_once = kWorkgroups<kD, kBf16, kW> * (uint32_t)compute_units;
  // The most blocks that a row can have. Where they are few, each unit is one
  // workgroup's (kWhole), which then need not find its part, nor leave a state
  // to a second launch: always to kFewValues (64 requests of up to 250 keys, 256
  // wide, 12.6 us cut, 10.8 whole), and to kManyValues where enough units are
  // there to keep the compute units at work (100 of a window of 512: 22.6 and
  // 17.2; but 16: 11.9 and 16.0). Where more units are there than workgroups run
  // at once, a unit is a wave's: four waves would each have had a block or two
  // of a short row (483 rows of 16 to 31 keys, 8 key-value heads, 256 wide, 127
  // us and 35; 512 of a window of 512 67 and 52; not of 63 blocks, 400 rows of 8
  // heads 128 wide: 214 by workgroups, 257 by waves). The host knows the table's
  // width and the window, not the rows: short rows in a wide table without a window
  // are cut (those 483 take the 127).
  const uint64_t capacity = (uint64_t)a.cache.width * a.cache.page_slots;
  const uint64_t held = (capacity + kBlockKeys - 1) / kBlockKeys;
  const uint64_t seen = (uint64_t)a.window / kBlockKeys + 2;
  const uint64_t blocks = held < seen ? held : seen;
  if (units >= a.at_once && blocks <= kWaveBlocks) {
    hipLaunchKernelGGL((paged_attention_kernel<kD, kBf16, kW, 1, true>), dim3(units), dim3(64), 0,
                       s, a);
    return hipGetLastError();
  }
  const bool few = 8 * units < 3 * (uint32_t)compute_units;
  if (blocks * kD <= (few ? kFewValues : kManyValues)) {
    hipLaunchKernelGGL((paged_attention_kernel<kD, kBf16, kW, kPartWaves, true>), dim3(units),
                       dim3(64 * kPartWaves), 0, s, a);
    return hipGetLastError();
  }
  // No more parts than the rows have blocks.
  const uint64_t fill = units * blocks;
  const uint64_t bound = most_parts(units, a.at_once);
  hipLaunchKernelGGL((paged_attention_kernel<kD, kBf16, kW, kPartWaves, false>),
                     dim3((uint32_t)(fill < bound ? fill : bound)), dim3(64 * kPartWaves), 0, s, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const uint32_t joins = most_joined_parts(units, a.at_once) / 2;
  const uint32_t records = units < joins ? units : joins;
  hipLaunchKernelGGL(paged_attention_join_kernel<kD>,
                     dim3(records < 256 ? records : 256, heads * (kD / 64)), dim3(kThreads), 0, s,
                     a);
  return hipGetLastError();
}

template <int kD>
hipError_t launch_heads(hipStream_t s, PagedAttentionArgs a, int compute_units) {
  const uint32_t group = a.query_heads / a.cache.kv_heads;
  const uint32_t heads = group < kHeadBlock ? group : kHeadBlock;
  a.units = a.cache.kv_heads * ((group + kHeadBlock - 1) / kHeadBlock);
  if (a.cache.bf16) {
    if (heads <= 4) return launch_shape<kD, true, 4>(s, a, heads, compute_units);
    if (heads <= 8) return launch_shape<kD, true, 8>(s, a, heads, compute_units);
    return launch_shape<kD, true, 16>(s, a, heads, compute_units);
  }
  if (heads <= 8) return launch_shape<kD, false, 8>(s, a, heads, compute_units);
  return launch_shape<kD, false, 16>(s, a, heads, compute_units);
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
