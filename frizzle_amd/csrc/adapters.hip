// Low-rank adapters of a batch's tokens beside a shared projection:
// y = base + s U (D x), each token with an adapter of its own.
//
// A call that reads little goes by tokens: one launch on the vector units, each
// token's workgroups forming D x for themselves. A large one goes by runs, in
// two launches: tokens next to each other that share an adapter, up to 16, 32
// or 64 within as many aligned ones, are a run, and an adapter's weights are
// read once a run, from HBM once a launch. Work is counted in runs, which each
// wave finds for itself from the tokens' adapters, so that a batch of one
// adapter and one of an adapter a token both fill the chip.
//
// The products of runs are on the matrix cores: with 16-bit weights, and U's of
// long runs with F32 ones, of parts of 16 bits that add up to the operands, else
// F32's own (v_mfma_f32_16x16x4_f32). Sums are F32 in both forms, and operands
// keep their 24 bits (kDownInParts). The weights are the instruction's A operand, 16
// rows of as many columns as it takes: lane (m, g) holds 8 columns of row m as
// they lie in memory, and of F32's eight instructions the j-th takes the j-th of
// each. Loads are a step ahead of the products, and all of a step's loads are
// requested at once: the kernels are compiled for 1, 2 or 4 (D) and 2, 4 or 8
// (U) tiles of 16 ranks, so that no branch parts them.

#include <type_traits>

#include "batch_rules.h"
#include "kernels.h"
#include "numerics.h"

namespace frz {
namespace {

using namespace rules;

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kDownWaves = 8, kUpWaves = 4;  // of a workgroup
constexpr int kTurnCols = 32 * kDownWaves;   // columns that its waves take a turn
constexpr int kBlockRows = 32 * kUpWaves;    // outputs of a workgroup
// Workgroups that a compute unit runs at once; a launch has no more, and each
// takes every so many items: ones without an item would wait for a place, then
// for the tokens' adapters, after all others.
template <int kTiles>
constexpr uint32_t kDownPlaces = kTiles == 4 ? 1 : 2;  // of the D kernel
template <int kRun>
constexpr uint32_t kUpPlaces = kRun == 16 ? 4 : 3;  // of the U kernel
// Columns from which a workgroup of the D kernel takes four tiles of ranks with
// 16-bit weights, for half of the reads of x: 333 tokens of one adapter, rank 64,
// 6,912 to 1,152, a call 17.7 -> 16.7 us, though 23.2 -> 23.7 of 32 adapters, as
// fewer workgroups run at once (300 of one each, rank 128, 4,096 to 4,096, 171 ->
// 180); 512 tokens, 1,152 columns, rank 128, 21.1 -> 22.7.
constexpr int kLongCols = 4096;
constexpr int kTokenWaves = 8;
constexpr uint32_t kTokenWorkgroups = 256;    // that one launch by tokens is cut into, about
// The most that it reads, and the most of it that is one D: takes_tokens.
constexpr uint64_t kTokenBytes = 128u << 20, kTokenDown = 600u << 10;

// Eight weights as they lie in memory, from element `at` (a multiple of 8).
template <int kFormat>
struct Raw {
  uint4 r[kFormat == 0 ? 2 : 1];
  __device__ __forceinline__ void load(const void* pool, uint64_t at) {
    const uint4* p = reinterpret_cast<const uint4*>(static_cast<const char*>(pool) +
                                                    at * (kFormat == 0 ? 4 : 2));
    r[0] = p[0];
    if constexpr (kFormat == 0) r[1] = p[1];
  }
  __device__ __forceinline__ float at(int i) const {
    const uint4& q = r[kFormat == 0 ? i >> 2 : 0];
    const int word = kFormat == 0 ? i & 3 : i >> 1;
    const uint32_t w = word == 0 ? q.x : word == 1 ? q.y : word == 2 ? q.z : q.w;
    if constexpr (kFormat == 0) return bits_to_float(w);
    if constexpr (kFormat == 1)
      return (float)__builtin_bit_cast(_Float16, (uint16_t)(i & 1 ? w >> 16 : w & 0xFFFF));
    return bits_to_float(i & 1 ? w & 0xFFFF0000u : w << 16);
  }
};

// F32 values as parts of BF16 that add up to them (three hold F32's 24 bits and
// its exponents), each what the parts before left. The first of three is cut, not
// rounded: neither it nor a product of it is infinite where the value's own is not.
// Weights are finite; of an x or a low-rank sum that is infinite or no number, the
// first two parts are finite and the last, which meets the other operand's first
// part alone, is the value.
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
template <bool kFinite>
__device__ __forceinline__ float within(float x, float largest) {
  return kFinite ? x : __builtin_amdgcn_fmed3f(x, -largest, largest);
}
template <bool kFinite>
__device__ __forceinline__ __bf16 first_of_three(float x, float* rest) {
  const uint32_t finite = float_to_bits(within<kFinite>(x, 0x1.FFFFFEp127f));
  *rest = x - bits_to_float(finite & 0xFFFF0000u);
  return __builtin_bit_cast(__bf16, (uint16_t)(finite >> 16));
}
template <bool kFinite>
__device__ __forceinline__ __bf16 second_of_three(float x, float* rest) {
  const __bf16 part = (__bf16)within<kFinite>(x, 0x1p121f);  // what the first leaves is below
  *rest = x - (float)part;
  return part;
}
template <bool kFinite>
__device__ __forceinline__ void split8(const float (&x)[8], bf16x8 (&part)[3]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float rest;
    part[0][j] = first_of_three<kFinite>(x[j], &rest);
    part[1][j] = second_of_three<kFinite>(rest, &rest);
    part[2][j] = (__bf16)rest;
  }
}
// Parts that hold a format's weights exactly: F16's 11 bits take two, BF16's one.
template <int kFormat>
constexpr int kWeightParts = kFormat == 0 ? 3 : kFormat == 1 ? 2 : 1;
__device__ __forceinline__ void split_weights(const float (&x)[8], bf16x8 (&part)[3]) {
  split8<true>(x, part);
}
__device__ __forceinline__ void split_weights(const float (&x)[8], bf16x8 (&part)[2]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    part[0][j] = (__bf16)x[j];
    part[1][j] = (__bf16)(x[j] - (float)part[0][j]);
  }
}
__device__ __forceinline__ void split_weights(const float (&x)[8], bf16x8 (&part)[1]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) part[0][j] = (__bf16)x[j];
}

struct Run {
  uint32_t first, tokens;
  uint32_t adapter;  // kNone: none
};

// The tokens' adapters as a wave holds them, token 64 i + lane a lane, and the
// runs of up to kRun tokens, in kRun aligned ones, that start among them.
constexpr int kTokenGroups = kMostRows / 64;
struct Runs {
  uint32_t id[kTokenGroups];
  uint64_t starts[kTokenGroups];  // a bit a token
  uint32_t count;
};

template <int kRun>
__device__ __forceinline__ Runs find_runs(const AdapterArgs& a, int lane) {
  static_assert(64 % kRun == 0, "a run lies in one group");
  Runs r;
#pragma unroll
  for (int i = 0; i < kTokenGroups; ++i) {
    r.id[i] = a.which[min(64u * i + lane, a.tokens - 1)];
  }
  r.count = 0;
#pragma unroll
  for (int i = 0; i < kTokenGroups; ++i) {
    if (r.id[i] >= a.count) r.id[i] = kNone;
    // The token before, of lane - 1 (DPP wave_shr:1); a group's first starts a
    // run whatever it is.
    const uint32_t last = (uint32_t)__builtin_amdgcn_update_dpp((int)r.id[i], (int)r.id[i], 0x138,
                                                                0xF, 0xF, false);
    r.starts[i] =
        __ballot(64u * i + lane < a.tokens && (lane % kRun == 0 || r.id[i] != last));
    r.count += __popcll(r.starts[i]);
  }
  return r;
}

// Run `want` (below r.count): it ends where the next one starts.
__device__ __forceinline__ Run run_at(const AdapterArgs& a, const Runs& r, uint32_t want) {
  uint32_t group = 0;
  uint64_t starts = r.starts[0];
#pragma unroll
  for (int i = 1; i < kTokenGroups; ++i) {
    const uint32_t before = __popcll(starts);
    if (group == (uint32_t)i - 1 && want >= before) {
      want -= before;
      group = i;
      starts = r.starts[i];
    }
  }
  // The lane whose start has `want` others before it.
  const uint32_t before =
      __builtin_amdgcn_mbcnt_hi((uint32_t)(starts >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)starts, 0));
  const uint64_t at = __ballot(before == want) & starts;
  const int lane = __builtin_ctzll(at);
  Run run;
  run.first = 64 * group + lane;
  run.adapter = kNone;
#pragma unroll
  for (int i = 0; i < kTokenGroups; ++i) {
    // Every group's, then the one: an index that varies would put them in memory.
    const uint32_t id = (uint32_t)__builtin_amdgcn_readlane((int)r.id[i], lane);
    run.adapter = group == (uint32_t)i ? id : run.adapter;
  }
  const uint64_t rest = lane == 63 ? 0 : starts >> (lane + 1);
  run.tokens = rest ? 1 + __builtin_ctzll(rest) : min(64 * (group + 1), a.tokens) - run.first;
  return run;
}

// An adapter's own rank. What a pool holds past it is loaded (it lies in the
// pool) but goes into no sum that is kept.
__device__ __forceinline__ int own_rank(const AdapterArgs& a, const Run& run) {
  const uint32_t own = a.ranks ? a.ranks[run.adapter] : (uint32_t)a.rank;
  return (int)min(own, (uint32_t)a.rank);
}

// Four values of a row of `rows`, from element `at`; one past the row's end
// repeats the last.
__device__ __forceinline__ f32x4 load4(const float* row, int at, int rows) {
  if (at + 4 <= rows) return *reinterpret_cast<const f32x4*>(row + at);
  f32x4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = row[min(at + e, rows - 1)];
  return v;
}
__device__ __forceinline__ void store4(float* row, int at, int rows, f32x4 v) {
  if (at + 4 <= rows) {
    *reinterpret_cast<f32x4*>(row + at) = v;
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (at + e < rows) row[at + e] = v[e];
}

// Outputs [from, to) of tokens without an adapter: base, where y is not base.
__device__ __forceinline__ void copy_base(const AdapterArgs& a, uint32_t first, uint32_t tokens,
                                          int from, int to, int wave, int waves, int lane) {
  if (a.base == a.y) return;
  const int pieces = (to - from + 255) / 256;  // of a token, a wave each
  for (uint32_t i = wave; i < tokens * pieces; i += waves) {
    const uint32_t t = first + i / pieces;
    const int o = from + (int)(i % pieces) * 256 + 4 * lane;
    if (o < to)
      store4(a.y + (uint64_t)t * a.y_stride, o, to,
             load4(a.base + (uint64_t)t * a.base_stride, o, to));
  }
}

// Whether D's products are of parts of x on the 16-bit matrix cores, the
// weights as they lie in memory: 3 instructions of 16 cycles for 32 columns
// where F32's eight take 256. 512 tokens, rank 32, 6,912 to 1,152, F16, of one
// adapter 14.4 -> 13.9 us a call, of one each 109 -> 99; rank 128, 4,096 to
// 4,096, 300 of one each 202 -> 180. Three parts hold all of x's 24 bits; those
// of F16 down to 2^-28 of the largest of a token's columns that a wave takes at
// once, and 2^-51 of it below: x is scaled, token by token, to lie below 2^15,
// and the parts after the first by 2^12 more, in sums of their own, so that F16's
// smallest values do not round them. (F16 weights as parts of BF16, for parts of
// x that need no scale: 333 tokens of 3 adapters, rank 64, 6,912 to 1,152, 16.0 ->
// 17.4 us, and 16.6 so; two parts of 23 bits 16.3.)
template <int kFormat>
constexpr bool kDownInParts = kFormat != 0;
constexpr float kRestScale = 4096.0f;

// A wave's share of D x for a run of up to 16 tokens, over the columns
// [from, to) and kTiles tiles of 16 ranks from `rank0` on: every eighth 32 of
// the columns. sum[t] has, in lane (n, g), token n's ranks rank0 + 16 t + 4 g
// .. + 3.
template <int kFormat, int kTiles>
__device__ __forceinline__ void low_rank(const AdapterArgs& a, const Run& run, int rank0, int from,
                                         int to, int wave, int n, int g, f32x4 (&sum)[kTiles]) {
  // Steps whose loads are in flight at once.
  constexpr int kDepth = kTiles == 1 ? 5 : kTiles == 2 && kFormat != 30 ? 3 : 4;
  Raw<0> x[kDepth];
  Raw<kFormat> w[kDepth][kTiles];
  const float* row =
      a.x + (uint64_t)(run.first + ((uint32_t)n < run.tokens ? n : 0)) * a.x_stride;
  const uint64_t pool = (uint64_t)run.adapter * a.rank * (uint64_t)a.cols;
#pragma unroll
  for (int t = 0; t < kTiles; ++t) sum[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int k0 = from + 32 * wave; k0 < to; k0 += kDepth * kTurnCols) {
#pragma unroll
    for (int i = 0; i < kDepth; ++i) {
      if (k0 + i * kTurnCols >= to) continue;
      // Columns are multiples of 8, and so are splits.
      const int at = k0 + i * kTurnCols + 8 * g, k = at < to ? at : from;
      x[i].load(row, k);
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
        w[i][t].load(a.down,
                     pool + (uint64_t)min(rank0 + 16 * t + n, a.rank - 1) * (uint64_t)a.cols + k);
    }
    float factor = 1.0f, back = 1.0f;
    f32x4 scaled[2][kTiles];  // of F16 parts: the first's sums, the others'
    if constexpr (kFormat == 1) {
      float most = 0.0f;
#pragma unroll
      for (int i = 0; i < kDepth; ++i) {
        if (k0 + i * kTurnCols >= to) continue;
#pragma unroll
        for (int j = 0; j < 8; ++j) most = __builtin_fmaxf(most, __builtin_fabsf(x[i].at(j)));
      }
      most = __builtin_fmaxf(most, __shfl_xor(most, 16));
      most = __builtin_fmaxf(most, __shfl_xor(most, 32));
      // To 2^126, which keeps all of F32's smallest values.
      int up = 141 - (int)(float_to_bits(most) >> 23);
      up = up > 126 ? 126 : up;
      factor = bits_to_float((uint32_t)(127 + up) << 23);
      back = bits_to_float((uint32_t)(127 - up) << 23);
#pragma unroll
      for (int t = 0; t < kTiles; ++t) scaled[0][t] = scaled[1][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
#pragma unroll
    for (int i = 0; i < kDepth; ++i) {
      if (k0 + i * kTurnCols >= to) continue;
      const bool in = k0 + i * kTurnCols + 8 * g < to;
      if constexpr (kDownInParts<kFormat>) {
        float xs[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) xs[j] = in ? x[i].at(j) * factor : 0.0f;
        uint4 weight[kTiles];
#pragma unroll
        for (int t = 0; t < kTiles; ++t) weight[t] = in ? w[i][t].r[0] : make_uint4(0, 0, 0, 0);
        if constexpr (kFormat == 1) {
#pragma unroll
          for (int p = 0; p < 3; ++p) {
            half8 part;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              part[j] = (_Float16)(p < 2 ? within<false>(xs[j], 65504.0f) : xs[j]);
              if (p < 2) xs[j] = (xs[j] - (float)part[j]) * (p == 0 ? kRestScale : 1.0f);
            }
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
              scaled[p > 0][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                  __builtin_bit_cast(half8, weight[t]), part, scaled[p > 0][t], 0, 0, 0);
          }
        } else {
          bf16x8 part[3];
          split8<false>(xs, part);
#pragma unroll
          for (int p = 2; p >= 0; --p)
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
              sum[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                  __builtin_bit_cast(bf16x8, weight[t]), part[p], sum[t], 0, 0, 0);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float xj = in ? x[i].at(j) : 0.0f;
#pragma unroll
          for (int t = 0; t < kTiles; ++t)
            sum[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(in ? w[i][t].at(j) : 0.0f, xj, sum[t],
                                                          0, 0, 0);
        }
      }
    }
    if constexpr (kFormat == 1)
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
        sum[t] += (scaled[0][t] + scaled[1][t] * (1 / kRestScale)) * back;
  }
}

// The low-rank rows of each run: a workgroup an item (run, ranks of kTiles
// tiles, split of K). Workgroups go round the eight dies, and a split stays on
// as few of them as there are: each die's L2 then takes in its own columns of
// x and D alone (D on every die had been most of what the dies read). Bound by
// loads of few steps that a launch, the adapters' search and a sum over the
// waves frame: 333 tokens of three F16 adapters, rank 64, 6,912 columns (12 MB)
// some 8.7 us, 512 tokens of an F32 one, rank 128, 1,152 columns some 6.
template <int kFormat, int kTiles>
__global__ __launch_bounds__(64 * kDownWaves, 2 * kDownPlaces<kTiles>)
void adapter_down_kernel(AdapterArgs a) {
  __shared__ f32x4 sums[kDownWaves][kTiles][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int n = lane & 15, g = lane >> 4;
  const Runs runs = find_runs<16>(a, lane);
  const uint32_t groups = (a.rank + 16 * kTiles - 1) / (16 * kTiles);
  // Splits are a power of two: `beside` of them go round the dies together,
  // with as many runs as the dies then have room for.
  const uint32_t splits = a.splits, beside = min(splits, 8u), rows = 8 / beside;
  const uint32_t items = (runs.count + rows - 1) / rows * rows * groups * splits;
  for (uint32_t item = blockIdx.x; item < items; item += gridDim.x) {
    const uint32_t die = item % 8, piece = item / 8, later = piece / groups;
    const uint32_t split = die % beside + later % (splits / beside) * 8;
    const uint32_t want = later / (splits / beside) * rows + die / beside;
    if (want >= runs.count) continue;
    const Run run = run_at(a, runs, want);
    if (run.adapter == kNone) continue;
    const int rank0 = piece % groups * 16 * kTiles;
    const int from = split * a.split_cols, to = min(from + a.split_cols, a.cols);
    f32x4 acc[kTiles];
    low_rank<kFormat, kTiles>(a, run, rank0, from, to, wave, n, g, acc);
    __syncthreads();  // the last item's sums are read
#pragma unroll
    for (int t = 0; t < kTiles; ++t) sums[wave][t][lane] = acc[t];
    __syncthreads();
    const int r = rank0 + 16 * wave + 4 * g;
    if (wave < kTiles && (uint32_t)n < run.tokens && r < a.rank) {
      f32x4 sum = sums[0][wave][lane];
#pragma unroll
      for (int w = 1; w < kDownWaves; ++w) sum += sums[w][wave][lane];
      *reinterpret_cast<f32x4*>(a.low + ((uint64_t)split * a.tokens + run.first + n) * a.rank + r) =
          sum;
    }
  }
}

// Whether the up products are of BF16 parts on the 16-bit matrix cores, 3, 5 or
// 6 instructions of 16 cycles for 32 ranks where F32's eight take 256. What it
// costs is the parts of U, some 150 cycles for 8 weights a lane of F16 or F32,
// which a run's tiles of tokens share: rank 128, 1,152 to 6,912, 512 tokens of
// one adapter, the call 24.5 -> 21.2 us in F16 and 25.6 -> 23.9 in F32 (449 ->
// 466 of an F32 adapter each); not for F32 in shorter runs: rank 128, 6,912 to
// 1,152, 200 tokens, 21.6 -> 21.8 us.
template <int kFormat, int kRun>
constexpr bool kUpInParts = kFormat != 0 || kRun == 64;

// base + s U times the low-rank rows, as the splits left them: a workgroup an
// item (run of up to kRun tokens, 128 outputs), a wave two tiles of 16 outputs
// by the run's tiles of 16 tokens. U is read once a run. The low-rank rows lie
// in LDS as the matrix instructions take them, as three parts of BF16 or F32.
// Bound by what a compute unit takes in of base, U and the low-rank rows (70 MB
// in all for 512 tokens, rank 128 in F32, 6,912 outputs: 14 us).
template <int kFormat, int kTiles, int kRun>
__global__ __launch_bounds__(64 * kUpWaves, kUpPlaces<kRun>) void adapter_up_kernel(AdapterArgs a) {
  constexpr int kChunks = (kTiles + 1) / 2;
  constexpr int kRunTiles = kRun / 16;
  constexpr bool kInParts = kUpInParts<kFormat, kRun>;
  constexpr int kWeights = kInParts ? kWeightParts<kFormat> : 1;
  typedef typename std::conditional<kInParts, __bf16, float>::type Low;
  typedef Low Low4 __attribute__((ext_vector_type(4)));
  constexpr int kLowParts = kInParts ? 3 : 1;
  // Values that a token's row takes in LDS: 16 bytes past a multiple of 64.
  constexpr int kPitch = 32 * kChunks + 16 / sizeof(Low);
  __shared__ __attribute__((aligned(16))) Low low[kLowParts][kRun][kPitch];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int n = lane & 15, g = lane >> 4;
  const Runs runs = find_runs<kRun>(a, lane);
  // As above, by eights of blocks: a block's runs meet on one die.
  const uint32_t blocks = (a.rows + kBlockRows - 1) / kBlockRows;
  const uint32_t places = blocks < 8 ? blocks : (blocks + 7) / 8 * 8;
  const uint32_t items = runs.count * places;
  for (uint32_t item = blockIdx.x; item < items; item += gridDim.x) {
    if (item % places >= blocks) continue;
    const Run run = run_at(a, runs, item / places);
    const int from = item % places * kBlockRows;
    if (run.adapter == kNone) {
      copy_base(a, run.first, run.tokens, from, min(from + kBlockRows, a.rows), wave, kUpWaves,
                lane);
      continue;
    }
    const int o = from + 32 * wave;  // the wave's outputs: o .. o + 31
    Raw<kFormat> w[2][2];            // of a chunk of 32 ranks and of the next, by turns
    auto load = [&](int c, Raw<kFormat> (&to)[2]) {
      const int r = 32 * c + 8 * g;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        to[i].load(a.up, ((uint64_t)run.adapter * a.rows + min(o + 16 * i + n, a.rows - 1)) *
                                 (uint64_t)a.rank + (r < a.rank ? r : 0));
    };
    load(0, w[0]);
    const int rank = __builtin_amdgcn_readfirstlane(own_rank(a, run));
    const float scale = a.scales ? a.scales[run.adapter] : 1.0f;
    const int run_tiles = (int)((run.tokens + 15) / 16);
    __syncthreads();  // the last item's rows are read
    // Four ranks a thread and piece, several splits of all its pieces asked for
    // together; ranks past the adapter's own are zero, tokens past the run its
    // last one, whose products nothing takes.
    constexpr int kFull = kRun * 8 * kChunks, kPieces = kFull < 256 ? 1 : kFull / (64 * kUpWaves);
    constexpr int kTogether = kPieces <= 2 ? 8 : kPieces <= 4 ? 4 : 2;
    f32x4 piece[kPieces];
    const float* src[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      // A piece past the run or the pool's rank reads another's place.
      const uint32_t at = threadIdx.x + i * 64 * kUpWaves;
      const uint32_t t = min(at / (8 * kChunks), run.tokens - 1);
      const int r = min((int)(at % (8 * kChunks) * 4), a.rank - 4);
      src[i] = a.low + (uint64_t)(run.first + t) * a.rank + r;
      piece[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    for (int s0 = 0; s0 < a.splits; s0 += kTogether) {
      f32x4 part[kTogether][kPieces];
#pragma unroll
      for (int s = 0; s < kTogether; ++s)
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
          part[s][i] = *reinterpret_cast<const f32x4*>(
              src[i] + (uint64_t)min(s0 + s, a.splits - 1) * a.tokens * a.rank);
#pragma unroll
      for (int s = 0; s < kTogether; ++s)
        if (s0 + s < a.splits)
#pragma unroll
          for (int i = 0; i < kPieces; ++i) piece[i] += part[s][i];
    }
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int at = threadIdx.x + i * 64 * kUpWaves;
      const int t = at / (8 * kChunks), r = at % (8 * kChunks) * 4;
      if (kFull < 256 && t >= kRun) break;
      Low4 part[kLowParts];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float rest = r + e < rank ? piece[i][e] * scale : 0.0f;
        if constexpr (kInParts) {
          part[0][e] = first_of_three<false>(rest, &rest);
          part[1][e] = second_of_three<false>(rest, &rest);
        }
        part[kLowParts - 1][e] = (Low)rest;
      }
#pragma unroll
      for (int p = 0; p < kLowParts; ++p) *reinterpret_cast<Low4*>(&low[p][t][r]) = part[p];
    }
    __syncthreads();
    // Lane (n, g): outputs 4 g .. + 3 of each tile, of token n of each 16.
    f32x4 base[2][kRunTiles];
#pragma unroll
    for (int t = 0; t < kRunTiles; ++t) {
      const float* row =
          a.base + (uint64_t)(run.first + min(16u * t + n, run.tokens - 1)) * a.base_stride;
#pragma unroll
      for (int i = 0; i < 2; ++i) base[i][t] = load4(row, o + 16 * i + 4 * g, a.rows);
    }
    f32x4 acc[2][kRunTiles];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int t = 0; t < kRunTiles; ++t) acc[i][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      if (c + 1 < kChunks) load(c + 1, w[(c + 1) & 1]);
      float weight[2][8];
      bf16x8 part[2][kWeights];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          weight[i][j] = 32 * c + 8 * g + j < rank ? w[c & 1][i].at(j) : 0.0f;
        if constexpr (kInParts) split_weights(weight[i], part[i]);
      }
#pragma unroll
      for (int t = 0; t < kRunTiles; ++t) {
        if (t >= run_tiles) break;
        const int at = 32 * c + 8 * g;
        if constexpr (kInParts) {
          // The products of parts down to 2^-16 of the largest: what is left
          // out, 2^-22 of a product at most and some 2^-26 mostly, is as small as
          // F32's rounding.
          bf16x8 h[3];
#pragma unroll
          for (int p = 0; p < 3; ++p)
            h[p] = *reinterpret_cast<const bf16x8*>(&low[p][16 * t + n][at]);
#pragma unroll
          for (int q = kWeights - 1; q >= 0; --q)
#pragma unroll
            for (int p = 2 - q; p >= 0; --p)
#pragma unroll
              for (int i = 0; i < 2; ++i)
                acc[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(part[i][q], h[p], acc[i][t], 0,
                                                                    0, 0);
        } else {
          const f32x4 h0 = *reinterpret_cast<const f32x4*>(&low[0][16 * t + n][at]);
          const f32x4 h1 = *reinterpret_cast<const f32x4*>(&low[0][16 * t + n][at + 4]);
#pragma unroll
          for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i)
              acc[i][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                  weight[i][j], j < 4 ? h0[j & 3] : h1[j & 3], acc[i][t], 0, 0, 0);
        }
      }
    }
#pragma unroll
    for (int t = 0; t < kRunTiles; ++t) {
      if (16u * t + n >= run.tokens) break;
      float* dst = a.y + (uint64_t)(run.first + 16 * t + n) * a.y_stride;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        store4(dst, o + 16 * i + 4 * g, a.rows, base[i][t] + acc[i][t]);
    }
  }
}

// Both products of one token: a workgroup a (token, block of outputs), on the
// vector units. All that it reads first is asked for at once: a wave's rows of
// D, a lane 8 columns of each 512, and rows of U, kLanes lanes a row and 8
// ranks a lane, so that a load is one contiguous piece (a row a lane had been
// 64 lines a load: 20 to 23 us where this takes 13 to 18, rank 64, 1,152 to
// 6,912, 64 tokens). Each of a token's workgroups forms all of D x for itself,
// from L2: workgroups go round the eight dies, and each die takes an eighth of
// the tokens, next to each other, so that they are on one, as are most tokens
// of one adapter (256 tokens of 64 adapters, rank 32, 6,912 to 1,152: 12.7 us,
// with every eighth token on a die 23.7). Bound by latency at few tokens (two
// chains of loads and a launch: 3 us of the call's 6) and by what a compute
// unit takes in, about 40 GB/s, at more: 48 tokens of 41 adapters, BF16, rank
// 32, 1,152 to 6,912 (18.5 MB), 8.9 us a call.
template <int kFormat, int kLanes>
__global__ __launch_bounds__(64 * kTokenWaves, kFormat == 0 ? 2 : 4)
void adapter_token_kernel(AdapterArgs a) {
  constexpr int kTurn = 64 * kTokenWaves / kLanes;  // outputs of a turn
  constexpr int kDepth = kFormat == 0 ? 4 : 8;      // turns whose rows are under way at once
  __shared__ __attribute__((aligned(16))) float low[8 * kLanes];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t places = a.tokens < 8 ? a.tokens : (a.tokens + 7) / 8 * 8;
  const uint32_t spot = blockIdx.x % places;
  const uint32_t token = places < 8 ? spot : spot % 8 * (places / 8) + spot / 8;
  if (token >= a.tokens) return;
  const int from = blockIdx.x / places * a.block_rows, to = min(from + a.block_rows, a.rows);
  const uint32_t adapter = a.which[token];
  if (adapter >= a.count) {
    copy_base(a, token, 1, from, to, wave, kTokenWaves, lane);
    return;
  }
  const int o0 = from + (int)threadIdx.x / kLanes, slice = 8 * ((int)threadIdx.x % kLanes);
  const int held = slice < a.rank ? slice : 0;  // a lane past the pool's rank repeats another
  Raw<kFormat> u[kDepth];
  float add[kDepth];
  const float* base = a.base + (uint64_t)token * a.base_stride;
  auto load_up = [&](int first) {
#pragma unroll
    for (int i = 0; i < kDepth; ++i) {
      if (first + i * kTurn >= to) continue;
      const int o = min(o0 - from + first + i * kTurn, a.rows - 1);
      u[i].load(a.up, ((uint64_t)adapter * a.rows + o) * (uint64_t)a.rank + held);
      add[i] = base[o];
    }
  };
  load_up(from);
  const Run run{token, 1, adapter};
  const int rank = __builtin_amdgcn_readfirstlane(own_rank(a, run));
  const float scale = a.scales ? a.scales[adapter] : 1.0f;
  const float* x = a.x + (uint64_t)token * a.x_stride;
  const uint64_t pool = (uint64_t)adapter * a.rank * (uint64_t)a.cols;
  // Four ranks a wave and turn, 1,536 columns at a time.
  for (int r0 = 4 * wave; r0 < 8 * kLanes; r0 += 4 * kTokenWaves) {
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int k0 = 0; r0 < a.rank && k0 < a.cols; k0 += 1536) {
      Raw<0> xs[3];
      Raw<kFormat> d[3][4];
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        const int at = k0 + 512 * i + 8 * lane, k = at < a.cols ? at : 0;
        if (k0 + 512 * i >= a.cols) continue;
        xs[i].load(x, k);
#pragma unroll
        for (int r = 0; r < 4; ++r)  // ranks come in eights
          d[i][r].load(a.down, pool + (uint64_t)(r0 + r) * a.cols + k);
      }
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        if (k0 + 512 * i + 8 * lane >= a.cols) continue;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int j = 0; j < 8; ++j) sum[r] = fmaf_(d[i][r].at(j), xs[i].at(j), sum[r]);
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      sum[r] = wave_tree(sum[r]);
      if (lane == 0) low[r0 + r] = r0 + r < rank ? sum[r] * scale : 0.0f;
    }
  }
  __syncthreads();
  float h[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) h[j] = low[slice + j];
  float* y = a.y + (uint64_t)token * a.y_stride;
  for (int first = from; first < to; first += kDepth * kTurn) {
    if (first > from) load_up(first);
#pragma unroll
    for (int i = 0; i < kDepth; ++i) {
      if (first + i * kTurn >= to) continue;
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        sum = fmaf_(slice + j < rank ? u[i].at(j) : 0.0f, h[j], sum);
      if constexpr (kLanes > 1) sum += __shfl_xor(sum, 1);
      if constexpr (kLanes > 2) sum += __shfl_xor(sum, 2);
      if constexpr (kLanes > 4) sum += __shfl_xor(sum, 4);
      if constexpr (kLanes > 8) sum += __shfl_xor(sum, 8);
      const int o = o0 - from + first + i * kTurn;
      if (slice == 0 && o < to) y[o] = add[i] + sum;
    }
  }
}

template <int kFormat, int kTiles, int kRun>
hipError_t launch_runs(hipStream_t s, const AdapterArgs& a, uint32_t blocks) {
  constexpr uint32_t kMost = 256 * kUpPlaces<kRun>;
  // As many workgroups as items where every token is a run.
  const uint64_t items = (uint64_t)a.tokens * (blocks < 8 ? blocks : (blocks + 7) / 8 * 8);
  hipLaunchKernelGGL((adapter_up_kernel<kFormat, kTiles, kRun>),
                     dim3((uint32_t)(items < kMost ? items : kMost)), dim3(64 * kUpWaves), 0, s,
                     a);
  return hipGetLastError();
}

template <int kFormat, int kTiles>
hipError_t launch_up(hipStream_t s, const AdapterArgs& a) {
  // Runs of 64 tokens read U half as often as runs of 32; but a compute unit
  // takes in about 40 GB/s, so shorter ones where the long ones' workgroups
  // leave compute units idle (333 tokens, rank 64, 1,152 outputs: runs of 16
  // 3.9 us, of 32 4.3).
  const uint32_t blocks = (a.rows + kBlockRows - 1) / kBlockRows;
  if ((a.tokens + 63) / 64 * blocks >= 256) return launch_runs<kFormat, kTiles, 64>(s, a, blocks);
  if ((a.tokens + 31) / 32 * blocks >= 256) return launch_runs<kFormat, kTiles, 32>(s, a, blocks);
  return launch_runs<kFormat, kTiles, 16>(s, a, blocks);
}

// Sets the splits.
template <int kFormat, int kTiles>
hipError_t launch_down(hipStream_t s, AdapterArgs& a) {
  // So many splits that the runs' workgroups fill the chip, a power of two, of
  // whole steps of a wave and not below a turn of a workgroup's waves; the last
  // may be short, or have no columns.
  const uint32_t groups = (a.rank + 16 * kTiles - 1) / (16 * kTiles);
  const uint32_t wanted = 256 / ((a.tokens + 15) / 16 * groups);
  uint32_t splits = 1;
  while (2 * splits <= wanted && 2 * splits <= kMostAdapterSplits &&
         2 * splits * kTurnCols <= (uint32_t)a.cols)
    splits *= 2;
  a.split_cols = 32 * (((a.cols + 31) / 32 + (int)splits - 1) / (int)splits);
  a.splits = (int)splits;
  constexpr uint32_t kMost = 256 * kDownPlaces<kTiles>;
  const uint64_t items = (uint64_t)((a.tokens + 7) / 8 * 8) * groups * splits;
  hipLaunchKernelGGL((adapter_down_kernel<kFormat, kTiles>),
                     dim3((uint32_t)(items < kMost ? items : kMost)),
                     dim3(64 * kDownWaves), 0, s, a);
  return hipGetLastError();
}

template <int kFormat>
hipError_t launch_down_tiles(hipStream_t s, AdapterArgs& a) {
  if (a.rank <= 16) return launch_down<kFormat, 1>(s, a);
  if constexpr (kFormat != 0)
    if (a.rank > 32 && a.cols >= kLongCols) return launch_down<kFormat, 4>(s, a);
  return launch_down<kFormat, 2>(s, a);
}

// A token's workgroups in adapter_token_kernel, each of so many whole turns of
// outputs that all tokens' workgroups are there at once.
struct TokenBlocks {
  uint32_t rows, count;
};
TokenBlocks token_blocks(const AdapterArgs& a, uint32_t turn) {
  const uint32_t turns = (a.rows + turn - 1) / turn;
  const uint32_t wanted = a.tokens < kTokenWorkgroups ? kTokenWorkgroups / a.tokens : 1;
  const uint32_t each = wanted < turns ? (turns + wanted - 1) / wanted : 1;
  return {each * turn, (turns + each - 1) / each};
}

// Whether it takes a call: where a D, which each of its workgroups reads whole,
// a load after another, stays below kTokenDown (one token, 4,000 outputs, rank
// 128, F16, of 1,152 columns, 295 kB, 9.2 us against 10.7 over runs, of 2,304 12.1
// against 10.8, of 6,912 24.6 against 13.4; rank 32 of 9,216, 590 kB, 10.2 against
// 11.2, of 16,384 15.0 against 11.8), and what all of them read, U with it, below
// kTokenBytes. Against two launches over runs, F16
// weights, tokens of one adapter and of one each, at most 64: rank 64, 1,152 to
// 6,912, 16 tokens (50 MB) 8.5 and 9.0 us against 10.3 and 13.0, 64 (90 MB) 13.3
// and 18.7 against 10.6 and 26.4, 128 (144 MB) 20.1 and 23.6 against 11.4 and
// 26.3; rank 32, 6,912 to 1,152, 128 tokens (117 MB) 9.8 and 11.7 against 11.6
// and 19.1, 512 (252 MB) 18.9 and 19.4 against 13.9 and 18.8; rank 16, 1,152 to
// 1,536, 1 to 256 tokens 7 against 9 to 12.
template <int kFormat, int kLanes>
bool takes_tokens(const AdapterArgs& a) {
  const TokenBlocks b = token_blocks(a, 64 * kTokenWaves / kLanes);
  const uint64_t size = kFormat == 0 ? 4 : 2, down = (uint64_t)a.rank * a.cols * size;
  return down <= kTokenDown &&
         a.tokens * (b.count * down + (uint64_t)a.rank * a.rows * size) <= kTokenBytes;
}

template <int kFormat, int kLanes>
hipError_t launch_token(hipStream_t s, AdapterArgs a) {
  const TokenBlocks b = token_blocks(a, 64 * kTokenWaves / kLanes);
  a.block_rows = (int)b.rows;
  const uint32_t places = a.tokens < 8 ? a.tokens : (a.tokens + 7) / 8 * 8;
  hipLaunchKernelGGL((adapter_token_kernel<kFormat, kLanes>), dim3(places * b.count),
                     dim3(64 * kTokenWaves), 0, s, a);
  return hipGetLastError();
}

template <int kFormat>
hipError_t launch_format(hipStream_t s, AdapterArgs a) {
  if (a.rank <= 16) {
    if (takes_tokens<kFormat, 2>(a)) return launch_token<kFormat, 2>(s, a);
  } else if (a.rank <= 32) {
    if (takes_tokens<kFormat, 4>(a)) return launch_token<kFormat, 4>(s, a);
  } else if (a.rank <= 64) {
    if (takes_tokens<kFormat, 8>(a)) return launch_token<kFormat, 8>(s, a);
  } else if (takes_tokens<kFormat, 16>(a)) {
    return launch_token<kFormat, 16>(s, a);
  }
  const hipError_t e = launch_down_tiles<kFormat>(s, a);
  if (e != hipSuccess) return e;
  if (a.rank <= 32) return launch_up<kFormat, 2>(s, a);
  if (a.rank <= 64) return launch_up<kFormat, 4>(s, a);
  return launch_up<kFormat, 8>(s, a);
}

}  // namespace

hipError_t launch_adapters(hipStream_t s, const AdapterArgs& a) {
  if (a.tokens == 0 || a.tokens > kMostRows || a.rank <= 0 || a.rank > kMostAdapterRank ||
      a.rank % 8 || a.cols <= 0 || a.cols % 8 || a.rows <= 0)
    return hipErrorInvalidValue;
  switch (a.format) {
    case 0: return launch_format<0>(s, a);
    case 1: return launch_format<1>(s, a);
    case 30: return launch_format<30>(s, a);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace frz
