// Caches in pages of 8 bits as a step writes them, and caches read back.
//
// Append. A block's 16 slots of one key-value head share a scale s, a power of
// two, so the step's rows in a block are taken together by one workgroup, which
// the first of them in the step finds itself to be:
//   need = least 2^e with max |x| <= 127 2^e over those rows
//   s'   = need where the block is begun anew, else max(s, need)
//   x    -> rint(x / s'), what the block held -> rint(c s / s')
// As scales grow by a factor of 2 at least, all roundings of a number come to
// s' (1/2 + 1/4 + ...) at most. Of keys, x is the normed and turned row, with
// rope_kernel's arithmetic and order of addition (rope_common.h); a head's D
// values are D / 8 lanes, as in paged_rope.hip, and its rows the workgroup's
// groups of lanes. Queries are turned by workgroups of their own.
//
// What bounds it is a chain of loads: the step's positions, the table, the block's
// scale and rows, between launch and store. A token's kernel takes 4.2 us (2 of it a
// launch's), 61 requests' 5.4, 507 rows of three prompts (32 + 16 heads of 128) 11.5.
// A token of each of 128 requests of 8 key-value heads takes 8.9, of 512 29, where a
// workgroup has four blocks, and so four such chains, one after another.
//
// Read. A thread takes one or two pieces of a row's keys and of its values, 16 bytes of
// output each, all loads under way together; what bounds it is memory: 95,001 rows of
// 8 x 128 as BF16 (585 MB) take 110 us, 5.3 TB/s, where a copy of 2 GiB reaches 4.9; of
// caches of 16 bits (778 MB) 135, 5.7.

#include "batch_rules.h"
#include "kernels.h"
#include "rope_common.h"

namespace frz {
namespace {

using namespace rules;

constexpr uint32_t kRopeThreads = 512;
constexpr uint32_t kRopeWorkgroups = 4;  // that a compute unit runs at once
static_assert(kRopeThreads >= kMostRows, "a thread looks at a row");

// A number of the block's scale, rounded to nearest even; NaN is 0.
__device__ __forceinline__ int code_of(float x) {
  const float top = (float)kMostCode;
  return x == x ? (int)rint_(__builtin_fminf(__builtin_fmaxf(x, -top), top)) : 0;
}
__device__ __forceinline__ uint32_t codes_of(float4 v, float scale) {
  if ((float_to_bits(scale) & 0x7FFFFFu) == 0) {  // a power of two, mostly: its product is the quotient
    const float each = 1.0f / scale;
    v = make_float4(v.x * each, v.y * each, v.z * each, v.w * each);
  } else {
    v = make_float4(v.x / scale, v.y / scale, v.z / scale, v.w / scale);
  }
  return (uint32_t)(code_of(v.x) & 0xFF) | (uint32_t)(code_of(v.y) & 0xFF) << 8 |
         (uint32_t)(code_of(v.z) & 0xFF) << 16 | (uint32_t)code_of(v.w) << 24;
}
// Four numbers by a scale `ratio` times as large (at most 1).
__device__ __forceinline__ uint32_t rescaled(uint32_t codes, float ratio) {
  uint32_t r = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    r |= ((uint32_t)(int)rint_((float)(int8_t)(codes >> 8 * i) * ratio) & 0xFF) << 8 * i;
  return r;
}

__device__ __forceinline__ float most_of(float4 v) {
  return __builtin_fmaxf(
      __builtin_fmaxf(__builtin_fabsf(v.x), __builtin_fabsf(v.y)),
      __builtin_fmaxf(__builtin_fabsf(v.z), __builtin_fabsf(v.w)));
}

// A lane's eight values of a head normed and turned to position p; all lanes of
// a head call it together, those of a head that is not there with zeros.
template <int kD>
__device__ __forceinline__ void norm_and_turn(float4& va, float4& vb, const float* gain,
                                              const float* turns_at, uint32_t l, uint32_t p,
                                              float epsilon) {
  constexpr int kLanes = kD / 8, kHalf = kD / 2;
  const float4 ga = ld4f(gain + 4 * l), gb = ld4f(gain + kHalf + 4 * l);
  const float4 turns = ld4f(turns_at + 4 * l);
  float cosine[4], sine[4];
  rope_angle(turns.x, p, &sine[0], &cosine[0]);
  rope_angle(turns.y, p, &sine[1], &cosine[1]);
  rope_angle(turns.z, p, &sine[2], &cosine[2]);
  rope_angle(turns.w, p, &sine[3], &cosine[3]);
  float squares = rope_lane_squares(va, vb);
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) squares = squares + __shfl_xor(squares, o);
  rope_normalize(va, vb, squares, kD, epsilon, ga, gb);
  rope_rotate(va, vb, 0, cosine, sine);
}

// The last workgroups turn queries. The others take a tile of rows and one
// key-value head, whose keys are half of a workgroup's threads and whose values the
// other half, and of those rows the blocks that they are the first in the step to be
// in, one after another: mostly one or none of a prompt's, of single tokens all.
template <int kD, uint32_t kTileRows>
__global__ __launch_bounds__(kRopeThreads) void paged_rope_i8_kernel(PagedRopeArgs a,
                                                                     uint32_t query_groups,
                                                                     uint32_t tiles) {
  constexpr uint32_t kLanes = kD / 8, kHalf = kD / 2;
  constexpr uint32_t kHeads = kRopeThreads / kLanes;  // of queries, at once
  constexpr uint32_t kGroups = kHeads / 2;            // rows of a block, at once
  constexpr uint32_t kTurns = kGroups < kScaleSlots ? kScaleSlots / kGroups : 1;
  const uint32_t t = threadIdx.x, l = t % kLanes;
  const uint32_t appends = tiles * a.cache.kv_heads;
  if (blockIdx.x >= appends) {
    const uint32_t row = (blockIdx.x - appends) / query_groups;
    const uint32_t h = (blockIdx.x - appends) % query_groups * kHeads + t / kLanes;
    const uint32_t p = a.positions[row];
    if (p == kNone) return;
    const bool active = h < a.query_heads;
    float4 va = make_float4(0.f, 0.f, 0.f, 0.f), vb = va;
    if (active) {
      const float* src = a.query + (uint64_t)row * a.q_stride + (uint64_t)h * kD;
      va = ld4f(src + 4 * l);
      vb = ld4f(src + kHalf + 4 * l);
    }
    norm_and_turn<kD>(va, vb, a.query_gain, a.turns, l, p, a.epsilon);
    if (!active) return;
    float* dst = a.roped + (uint64_t)row * a.roped_stride + (uint64_t)h * kD;
    *reinterpret_cast<float4*>(dst + 4 * l) = va;
    *reinterpret_cast<float4*>(dst + kHalf + 4 * l) = vb;
    return;
  }
  __shared__ uint32_t members[kTileRows][kScaleSlots];  // the row that writes a slot, and 1
  __shared__ uint32_t taken;  // rows of the tile that are not the first of their block
  __shared__ float wave_most[kRopeThreads / 64];
  const uint32_t kv = blockIdx.x % a.cache.kv_heads;
  const uint32_t tile = blockIdx.x / a.cache.kv_heads;
  const uint32_t rows = (a.rows - tile + tiles - 1) / tiles;
  // Each thread holds its row of the step against the tile's.
  auto sequence_of = [&](uint32_t r) { return a.sequences ? a.sequences[r] : r; };
  const uint32_t mine = min(t, a.rows - 1);
  const uint32_t p_mine = t < a.rows ? a.positions[mine] : kNone;
  const uint32_t sequence_mine = sequence_of(mine);
  uint32_t p_tile[kTileRows], sequence_tile[kTileRows];
#pragma unroll
  for (uint32_t k = 0; k < kTileRows; ++k) {
    const uint32_t r = tile + min(k, rows - 1) * tiles;
    p_tile[k] = a.positions[r];
    sequence_tile[k] = sequence_of(r);
  }
  if (t < kTileRows * kScaleSlots) members[t / kScaleSlots][t % kScaleSlots] = 0;
  if (t == 0) taken = 0;
  __syncthreads();
#pragma unroll
  for (uint32_t k = 0; k < kTileRows; ++k) {
    if ((k == 0 || k < rows) && p_mine != kNone && p_tile[k] != kNone && sequence_mine == sequence_tile[k] &&
        p_mine / kScaleSlots == p_tile[k] / kScaleSlots) {
      atomicMax(&members[k][p_mine % kScaleSlots], t + 1);  // of rows at one position the last
      if (t < tile + k * tiles) atomicOr(&taken, 1u << k);
    }
  }
  __syncthreads();
  const uint32_t others = taken;
#pragma unroll 1
  for (uint32_t k = 0; k < rows; ++k) {
    if (others >> k & 1) continue;
    uint32_t p = kNone, sequence = 0;
#pragma unroll
    for (uint32_t i = 0; i < kTileRows; ++i) {
      p = i == k ? p_tile[i] : p;
      sequence = i == k ? sequence_tile[i] : sequence;
    }
    if (p == kNone) continue;
    const uint32_t block = p / kScaleSlots;
    const uint32_t index = p / a.cache.page_slots;
    const uint32_t page = page_at(a.cache.table, a.cache.sequences, a.cache.width, a.cache.pages,
                                  sequence, index);
    if (page == kNone) continue;
    const uint32_t* member = members[k];

    const bool is_value = t >= kRopeThreads / 2;
    const uint32_t group = t % (kRopeThreads / 2) / kLanes;
    const uint32_t first_slot = block * kScaleSlots - index * a.cache.page_slots;
    uint8_t* codes = static_cast<uint8_t*>(is_value ? a.cache.values : a.cache.keys) +
                     page * a.cache.page_stride +
                     ((uint64_t)first_slot * a.cache.kv_heads + kv) * kD;
    float* scale_at = (is_value ? a.cache.value_scales : a.cache.key_scales) +
                      page * a.cache.scale_stride +
                      (uint64_t)(first_slot / kScaleSlots) * a.cache.kv_heads + kv;
    float scale = *scale_at;
    if (member[0] || !(scale > 0.0f) || scale == __builtin_inff()) scale = 0.0f;

    uint32_t from[kTurns];
    float4 va[kTurns], vb[kTurns];
    uint32_t ca[kTurns], cb[kTurns];  // what the block holds
#pragma unroll
    for (uint32_t i = 0; i < kTurns; ++i) {
      const uint32_t slot = i * kGroups + group;
      from[i] = slot < kScaleSlots ? member[slot] : 0;
      va[i] = vb[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      ca[i] = cb[i] = 0;
      if (from[i]) {
        const float* src = (is_value ? a.value : a.key) + (uint64_t)(from[i] - 1) * a.kv_stride +
                           (uint64_t)kv * kD;
        va[i] = ld4f(src + 4 * l);
        vb[i] = ld4f(src + kHalf + 4 * l);
      } else if (slot < kScaleSlots) {
        const uint8_t* src = codes + (uint64_t)slot * a.cache.kv_heads * kD;
        ca[i] = *reinterpret_cast<const uint32_t*>(src + 4 * l);
        cb[i] = *reinterpret_cast<const uint32_t*>(src + kHalf + 4 * l);
      }
    }
    float most = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < kTurns; ++i) {
      const uint32_t slot = i * kGroups + group;
      if (!is_value && __ballot(from[i] != 0))
        norm_and_turn<kD>(va[i], vb[i], a.key_gain, a.turns, l, block * kScaleSlots + slot,
                          a.epsilon);
      if (from[i]) most = __builtin_fmaxf(most, __builtin_fmaxf(most_of(va[i]), most_of(vb[i])));
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) most = __builtin_fmaxf(most, __shfl_xor(most, o));
    if (t % 64 == 0) wave_most[t / 64] = most;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < kRopeThreads / 128; ++w)
      most = __builtin_fmaxf(most, wave_most[is_value * (kRopeThreads / 128) + w]);
    const float need = bits_to_float(block_scale_bits(float_to_bits(most)));
    const float after = __builtin_fmaxf(scale, need);
    const float ratio = after > 0.0f ? scale / after : 0.0f;
    const float by = after > 0.0f ? after : 1.0f;  // all zeros: any
#pragma unroll
    for (uint32_t i = 0; i < kTurns; ++i) {
      const uint32_t slot = i * kGroups + group;
      if (slot >= kScaleSlots || (!from[i] && ratio == 1.0f)) continue;
      uint8_t* dst = codes + (uint64_t)slot * a.cache.kv_heads * kD;
      *reinterpret_cast<uint32_t*>(dst + 4 * l) =
          from[i] ? codes_of(va[i], by) : rescaled(ca[i], ratio);
      *reinterpret_cast<uint32_t*>(dst + kHalf + 4 * l) =
          from[i] ? codes_of(vb[i], by) : rescaled(cb[i], ratio);
    }
    if (t % (kRopeThreads / 2) == 0) *scale_at = after;
    __syncthreads();  // what is shared is read
  }
}

template <int kD>
void launch_rope(hipStream_t s, const PagedRopeArgs& a, int compute_units) {
  constexpr uint32_t kHeads = kRopeThreads / (kD / 8);
  const uint32_t groups = (a.query_heads + kHeads - 1) / kHeads;
  // A tile of one row, or of up to four where workgroups of one would be more than run
  // at once. A tile's rows are an odd number apart, so that neither
  // the first rows of a step nor every sixteenth, which are the first of their blocks
  // where rows lie in any order and in theirs, fall into few tiles. (507 rows in any
  // order, 8 key-value heads: tiles of rows side by side 17 us, these 11.6, of eight
  // such rows 12.5, of one 16.5.)
  const uint32_t at_once = kRopeWorkgroups * (uint32_t)compute_units;
  const uint32_t even = (a.rows * a.cache.kv_heads + at_once - 1) / at_once;
  const uint32_t tile = even < 4 ? even : 4;
  uint32_t tiles = (a.rows + tile - 1) / tile;
  if (tile > 1 && tiles % 2 == 0) ++tiles;
  const dim3 grid(tiles * a.cache.kv_heads + a.rows * groups), threads(kRopeThreads);
  if (tile == 1)
    hipLaunchKernelGGL((paged_rope_i8_kernel<kD, 1>), grid, threads, 0, s, a, groups, tiles);
  else
    hipLaunchKernelGGL((paged_rope_i8_kernel<kD, 4>), grid, threads, 0, s, a, groups, tiles);
}

// ---- reading back --------------------------------------------------------------

constexpr uint32_t kThreads = 256;
// Values that a thread takes at once: 16 bytes of output, so that each of a wave's stores
// fills whole lines. 40,000 rows of 8 x 128 bytes as F32 by 8 values and two stores:
// 153 us; so 60 (6.8 TB/s).
template <int kTo>
constexpr int kPieceOf = kTo == 0 ? 4 : 8;
// Outputs past what the L2 caches hold (8 of 4 MB) go past them too, and a thread then
// takes two pieces, all loads first. 40,000 rows of 8 x 128 as BF16 (160 MB): 54 us by
// one piece, 52 by two, 37 past the caches; 95,001 rows 126, 118 and 110. A window's 512
// of 256, as F16: 3.0 by one piece, 4.0 by two. 10,000 rows as F32: 24.2 us in the caches,
// 16.4 past them.
constexpr uint64_t kCachedBytes = 32u << 20;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// A piece of a cache row.
template <CacheFormat kFrom, int kPiece>
struct Piece {
  static constexpr int kWords = kFrom == kCacheI8 ? kPiece / 4 : kPiece / 2;
  typedef uint32_t Words __attribute__((ext_vector_type(kWords)));
  uint32_t words[kWords];
  float scale;
  __device__ __forceinline__ void load(const void* pool, uint64_t at, const float* scales,
                                       uint64_t scale_at) {
    if constexpr (kFrom == kCacheI8) {
      take(static_cast<const uint8_t*>(pool) + at);
      scale = scales[scale_at];
    } else {
      take(static_cast<const uint16_t*>(pool) + at);
    }
  }
  __device__ __forceinline__ void take(const void* from) {
    const Words w = *static_cast<const Words*>(from);
#pragma unroll
    for (int i = 0; i < kWords; ++i) words[i] = w[i];
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (kFrom == kCacheI8)
      return (float)(int8_t)(words[i / 4] >> 8 * (i % 4)) * scale;
    const uint16_t half = (uint16_t)(words[i / 2 % kWords] >> 16 * (i % 2));
    if constexpr (kFrom == kCacheBf16) return bits_to_float((uint32_t)half << 16);
    return (float)__builtin_bit_cast(_Float16, half);
  }
};

template <int kTo>
__device__ __forceinline__ uint16_t half_of(float x) {
  if constexpr (kTo == 1) return f16_pack_device(x);
  return __builtin_bit_cast(uint16_t, (__bf16)x);
}

template <bool kPast>
__device__ __forceinline__ void put(void* dst, u32x4 v) {
  if constexpr (kPast) __builtin_nontemporal_store(v, static_cast<u32x4*>(dst));
  else *static_cast<u32x4*>(dst) = v;
}

template <CacheFormat kFrom, int kTo, bool kPast>
__device__ __forceinline__ void store(void* to, uint64_t at,
                                      const Piece<kFrom, kPieceOf<kTo>>& piece, bool there) {
  if constexpr (kTo == 0) {
    u32x4 w;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = there ? float_to_bits(piece.get(j)) : 0u;
    put<kPast>(static_cast<float*>(to) + at, w);
  } else {
    u32x4 w;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      w[j] = there ? half_of<kTo>(piece.get(2 * j)) |
                         (uint32_t)half_of<kTo>(piece.get(2 * j + 1)) << 16
                   : 0u;
    put<kPast>(static_cast<uint16_t*>(to) + at, w);
  }
}

// A workgroup takes kPieces * kThreads pieces of whole rows, or a part of one row.
template <CacheFormat kFrom, int kTo, uint32_t kPieces>
__global__ __launch_bounds__(kThreads) void paged_read_kernel(PagedReadArgs a, uint32_t row_pieces,
                                                              uint32_t rows_each) {
  const uint32_t first = blockIdx.x * rows_each;
  const uint32_t count = min(rows_each, a.rows - first) * row_pieces;
  const uint32_t from = blockIdx.y * kPieces * kThreads + threadIdx.x;
  constexpr int kPiece = kPieceOf<kTo>;
  Piece<kFrom, kPiece> key[kPieces], value[kPieces];
  bool there[kPieces], live[kPieces];
  uint32_t row[kPieces], piece[kPieces], p[kPieces], sequence[kPieces];
#pragma unroll
  for (uint32_t k = 0; k < kPieces; ++k) {
    const uint32_t i = from + k * kThreads;
    live[k] = i < count;
    row[k] = first + (live[k] ? i : 0) / row_pieces;
    piece[k] = (live[k] ? i : 0) % row_pieces;
    p[k] = a.positions[row[k]];
    sequence[k] = a.sequences ? a.sequences[row[k]] : row[k];
  }
#pragma unroll
  for (uint32_t k = 0; k < kPieces; ++k) {
    live[k] = live[k] && p[k] != kNone;
    const uint32_t index = p[k] / a.cache.page_slots, slot = p[k] - index * a.cache.page_slots;
    const uint32_t page = page_at(a.cache.table, a.cache.sequences, a.cache.width, a.cache.pages,
                                  sequence[k], index);
    there[k] = live[k] && page != kNone;
    if (!there[k]) continue;
    const uint64_t at = page * a.cache.page_stride +
                        (uint64_t)slot * a.cache.kv_heads * a.cache.head_dim +
                        (uint64_t)piece[k] * kPiece;
    const uint64_t scale = page * a.cache.scale_stride +
                           (uint64_t)(slot / kScaleSlots) * a.cache.kv_heads +
                           piece[k] * kPiece / a.cache.head_dim;
    key[k].load(a.cache.keys, at, a.cache.key_scales, scale);
    value[k].load(a.cache.values, at, a.cache.value_scales, scale);
  }
#pragma unroll
  for (uint32_t k = 0; k < kPieces; ++k) {
    if (!live[k]) continue;
    const uint64_t to = (uint64_t)row[k] * a.stride + (uint64_t)piece[k] * kPiece;
    store<kFrom, kTo, (kPieces > 1)>(a.keys, to, key[k], there[k]);
    store<kFrom, kTo, (kPieces > 1)>(a.values, to, value[k], there[k]);
  }
}

template <CacheFormat kFrom, int kTo, uint32_t kPieces>
void launch_pieces(hipStream_t s, const PagedReadArgs& a) {
  constexpr uint32_t kMost = kPieces * kThreads;
  const uint32_t pieces = a.cache.kv_heads * a.cache.head_dim / kPieceOf<kTo>;
  const uint32_t rows = pieces < kMost ? kMost / pieces : 1;
  hipLaunchKernelGGL((paged_read_kernel<kFrom, kTo, kPieces>),
                     dim3((a.rows + rows - 1) / rows, (pieces + kMost - 1) / kMost),
                     dim3(kThreads), 0, s, a, pieces, rows);
}
template <CacheFormat kFrom, int kTo>
void launch_read(hipStream_t s, const PagedReadArgs& a) {
  const uint64_t bytes = 2ull * a.rows * a.cache.kv_heads * a.cache.head_dim * (kTo == 0 ? 4 : 2);
  if (bytes > kCachedBytes) launch_pieces<kFrom, kTo, 2>(s, a);
  else launch_pieces<kFrom, kTo, 1>(s, a);
}
template <CacheFormat kFrom>
hipError_t launch_read_to(hipStream_t s, const PagedReadArgs& a) {
  switch (a.format) {
    case 0: launch_read<kFrom, 0>(s, a); break;
    case 1: launch_read<kFrom, 1>(s, a); break;
    case 30: launch_read<kFrom, 30>(s, a); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_paged_rope_i8(hipStream_t s, const PagedRopeArgs& a, int compute_units) {
  if (compute_units <= 0) return hipErrorInvalidValue;
  switch (a.cache.head_dim) {
    case 64: launch_rope<64>(s, a, compute_units); break;
    case 128: launch_rope<128>(s, a, compute_units); break;
    case 256: launch_rope<256>(s, a, compute_units); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

hipError_t launch_paged_read(hipStream_t s, const PagedReadArgs& a) {
  if (a.rows == 0) return hipErrorInvalidValue;
  switch (a.cache.format) {
    case kCacheF16: return launch_read_to<kCacheF16>(s, a);
    case kCacheBf16: return launch_read_to<kCacheBf16>(s, a);
    case kCacheI8: return launch_read_to<kCacheI8>(s, a);
  }
  return hipErrorInvalidValue;
}

}  // namespace frz
