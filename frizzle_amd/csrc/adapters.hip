// Low-rank adapters of a batch's tokens beside a shared projection:
// y = base + s U (D x), each token with an adapter of its own.
//
// Tokens next to each other that share an adapter, up to 16 within 16 aligned
// ones, are a run: an adapter's weights are read once a run, from HBM once a
// launch. Two launches: the low-rank rows D x of each run, K cut over
// workgroups, then U times them, added to base. Work is counted in runs, which
// each wave finds for itself from the tokens' adapters, so that a batch of
// one adapter and one of an adapter a token both fill the chip.
//
// Both products run on the F32 matrix cores (v_mfma_f32_16x16x4_f32), weights
// of any format widened exactly on the way: products and sums are F32, and
// rounded nowhere else. The weights are the instruction's A operand, 16 rows
// by 4 columns: lane (m, g) holds 8 columns of row m as they lie in memory,
// and instruction j of 8 takes the j-th of each.

#include "batch_rules.h"
#include "kernels.h"
#include "numerics.h"

namespace frz {
namespace {

using namespace rules;

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kRunTokens = 16;
constexpr int kRankTiles = kMostAdapterRank / 16;
constexpr int kBlockRows = 256;  // outputs a workgroup

struct Weights {
  float v[8];
};

// Eight weights from element `at` (a multiple of 8).
template <int kFormat>
__device__ __forceinline__ Weights load8(const void* pool, uint64_t at) {
  Weights w;
  if constexpr (kFormat == 0) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(pool) + at);
    const float4 a = p[0], b = p[1];
    w = Weights{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
  } else {
    const uint4 r = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(pool) + at);
    const uint32_t word[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (kFormat == 1) {
        w.v[2 * i] = (float)__builtin_bit_cast(_Float16, (uint16_t)(word[i] & 0xFFFF));
        w.v[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(word[i] >> 16));
      } else {
        w.v[2 * i] = bits_to_float(word[i] << 16);
        w.v[2 * i + 1] = bits_to_float(word[i] & 0xFFFF0000u);
      }
    }
  }
  return w;
}

struct Run {
  uint32_t first, tokens;
  uint32_t adapter;  // kNone: none
  int rank;          // its own
};

// The tokens' adapters as a wave holds them, eight tokens a lane, and the
// runs that start among them.
struct Runs {
  uint32_t id[8];
  uint32_t starts;  // bit i: a run starts at token 8 lane + i
  uint32_t before;  // runs before the lane's
  uint32_t count;
};

__device__ __forceinline__ uint32_t adapter_of(const AdapterArgs& a, uint32_t token) {
  const uint32_t id = a.which[token];
  return id < a.count ? id : kNone;
}

__device__ __forceinline__ Runs find_runs(const AdapterArgs& a, int lane) {
  Runs r;
  r.starts = 0;
  uint32_t last = kNone;
  if (lane > 0 && 8 * lane <= (int)a.tokens) last = adapter_of(a, 8 * lane - 1);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t t = 8 * lane + i;
    r.id[i] = t < a.tokens ? adapter_of(a, t) : kNone;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t t = 8 * lane + i;
    const uint32_t prev = i == 0 ? last : r.id[i > 0 ? i - 1 : 0];
    if (t < a.tokens && (t % kRunTokens == 0 || r.id[i] != prev)) r.starts |= 1u << i;
  }
  uint32_t sum = __popc(r.starts);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t up = __shfl_up(sum, o);
    if (lane >= o) sum += up;
  }
  r.count = __builtin_amdgcn_readfirstlane((int)__shfl(sum, 63));
  r.before = sum - __popc(r.starts);
  return r;
}

// Run `want` (below r.count).
__device__ __forceinline__ Run run_at(const AdapterArgs& a, const Runs& r, uint32_t want,
                                      int lane) {
  const uint32_t mine = __popc(r.starts);
  const uint64_t owners = __ballot(want >= r.before && want < r.before + mine);
  const int leader = __builtin_ctzll(owners);
  uint32_t starts = r.starts;
  for (uint32_t i = r.before; i < want && starts; ++i) starts &= starts - 1;
  const int at = starts ? __builtin_ctz(starts) : 0;
  uint32_t id = kNone;
#pragma unroll
  for (int i = 0; i < 8; ++i) id = i == at ? r.id[i] : id;
  Run run;
  run.first = 8 * leader + (uint32_t)__builtin_amdgcn_readlane(at, leader);
  run.adapter = (uint32_t)__builtin_amdgcn_readlane((int)id, leader);
  // The tokens of its 16 that go on with the same adapter.
  const uint32_t room = min(kRunTokens - run.first % kRunTokens, a.tokens - run.first);
  const bool same = (uint32_t)lane < room && adapter_of(a, run.first + lane) == run.adapter;
  run.tokens = (uint32_t)__builtin_ctzll(~__ballot(same));
  run.rank = a.rank;
  if (run.adapter != kNone && a.ranks) {
    const uint32_t own = a.ranks[run.adapter];
    run.rank = own < (uint32_t)a.rank ? (int)own : a.rank;
  }
  run.rank = __builtin_amdgcn_readfirstlane(run.rank);
  return run;
}

// The low-rank rows of each run over one of K's splits: a workgroup an item
// (run, split), its waves every fourth 32 columns of the split.
template <int kFormat>
__global__ __launch_bounds__(kThreads) void adapter_down_kernel(AdapterArgs a) {
  __shared__ f32x4 sums[kWaves][kRankTiles][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int n = lane & 15, g = lane >> 4;
  const Runs runs = find_runs(a, lane);
  const uint32_t items = runs.count * a.splits;
  for (uint32_t item = blockIdx.x; item < items; item += gridDim.x) {
    const Run run = run_at(a, runs, item / a.splits, lane);
    if (run.adapter == kNone || run.rank == 0) continue;
    const uint32_t split = item % a.splits;
    const int from = split * a.split_cols, to = min(from + a.split_cols, a.cols);
    const int tiles = (run.rank + 15) / 16;
    f32x4 acc[kRankTiles];
#pragma unroll
    for (int t = 0; t < kRankTiles; ++t) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const bool live = (uint32_t)n < run.tokens;
    const float* x = a.x + (uint64_t)(run.first + (live ? n : 0)) * a.x_stride;
    const uint64_t pool = (uint64_t)run.adapter * a.rank * a.cols;
    for (int k0 = from + 32 * wave; k0 < to; k0 += 32 * kWaves) {
      const int k = k0 + 8 * g;
      const bool in = k < to;  // columns are multiples of 8, and so are splits
      const int kc = in ? k : from;
      const Weights xs = load8<0>(x, kc);
#pragma unroll
      for (int t = 0; t < kRankTiles; ++t) {
        if (t >= tiles) break;
        const int r = 16 * t + n;
        const bool held = in && r < run.rank;
        const Weights w = load8<kFormat>(a.down, pool + (uint64_t)min(r, run.rank - 1) * a.cols + kc);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(held ? w.v[j] : 0.0f,
                                                        in && live ? xs.v[j] : 0.0f, acc[t], 0, 0, 0);
      }
    }
    __syncthreads();  // the last item's sums are read
#pragma unroll
    for (int t = 0; t < kRankTiles; ++t)
      if (t < tiles) sums[wave][t][lane] = acc[t];
    __syncthreads();
    // Lane (n, g) of tile t: token n, ranks 16 t + 4 g .. + 3.
    for (int i = threadIdx.x; i < tiles * 64; i += kThreads) {
      const int t = i >> 6, ln = i & 63, token = ln & 15, r = 16 * t + 4 * (ln >> 4);
      if ((uint32_t)token >= run.tokens || r >= run.rank) continue;
      f32x4 sum = sums[0][t][ln];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) sum += sums[w][t][ln];
      *reinterpret_cast<f32x4*>(a.low + ((uint64_t)split * a.tokens + run.first + token) * a.rank + r) =
          sum;
    }
  }
}

// base + s U times the low-rank rows: a workgroup an item (run, 256 outputs),
// a wave 64 of them.
template <int kFormat>
__global__ __launch_bounds__(kThreads) void adapter_up_kernel(AdapterArgs a) {
  constexpr int kPitch = kMostAdapterRank + 4;
  __shared__ __attribute__((aligned(16))) float low[kRunTokens][kPitch];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int n = lane & 15, g = lane >> 4;
  const Runs runs = find_runs(a, lane);
  const uint32_t blocks = (a.rows + kBlockRows - 1) / kBlockRows;
  const uint32_t items = runs.count * blocks;
  for (uint32_t item = blockIdx.x; item < items; item += gridDim.x) {
    const Run run = run_at(a, runs, item / blocks, lane);
    const int out0 = item % blocks * kBlockRows + 64 * wave;
    const bool none = run.adapter == kNone || run.rank == 0;
    if (none && a.base == a.y) continue;
    const int chunks = none ? 0 : (run.rank + 31) / 32;
    __syncthreads();  // the last item's rows are read
    if (!none) {
      const float scale = a.scales ? a.scales[run.adapter] : 1.0f;
      const int width = 32 * chunks;
      for (int i = threadIdx.x; i < kRunTokens * width; i += kThreads) {
        const int t = i / width, r = i % width;
        float sum = 0.0f;
        if ((uint32_t)t < run.tokens && r < run.rank) {
          const float* src = a.low + (uint64_t)(run.first + t) * a.rank + r;
          for (int s = 0; s < a.splits; ++s) sum += src[(uint64_t)s * a.tokens * a.rank];
        }
        low[t][r] = sum * scale;
      }
    }
    __syncthreads();
    const uint64_t pool = (uint64_t)run.adapter * a.rows * a.rank;
#pragma unroll 1
    for (int tile = 0; tile < 4; ++tile) {
      const int o = out0 + 16 * tile;
      if (o >= a.rows) break;
      f32x4 acc = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      const uint64_t at = pool + (uint64_t)min(o + n, a.rows - 1) * a.rank;
      for (int c = 0; c < chunks; ++c) {
        const int r = 32 * c + 8 * g;
        const Weights w = load8<kFormat>(a.up, at + (r < a.rank ? r : 0));
        const Weights h = load8<0>(&low[n][0], r);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          acc = __builtin_amdgcn_mfma_f32_16x16x4f32(r + j < run.rank ? w.v[j] : 0.0f, h.v[j], acc,
                                                     0, 0, 0);
      }
      // Lane (n, g): token n, outputs o + 4 g .. + 3.
      const int first = o + 4 * g;
      if ((uint32_t)n >= run.tokens || first >= a.rows) continue;
      const float* base = a.base + (uint64_t)(run.first + n) * a.base_stride + first;
      float* y = a.y + (uint64_t)(run.first + n) * a.y_stride + first;
      if (first + 4 <= a.rows) {
        *reinterpret_cast<f32x4*>(y) = *reinterpret_cast<const f32x4*>(base) + acc;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (first + e < a.rows) y[e] = base[e] + acc[e];
      }
    }
  }
}

template <int kFormat>
hipError_t launch_format(hipStream_t s, const AdapterArgs& a, uint32_t down, uint32_t up) {
  hipLaunchKernelGGL(adapter_down_kernel<kFormat>, dim3(down), dim3(kThreads), 0, s, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(adapter_up_kernel<kFormat>, dim3(up), dim3(kThreads), 0, s, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_adapters(hipStream_t s, const AdapterArgs& args) {
  AdapterArgs a = args;
  if (a.tokens == 0 || a.tokens > kMostRows || a.rank <= 0 || a.rank > kMostAdapterRank ||
      a.rank % 8 || a.cols <= 0 || a.cols % 8 || a.rows <= 0)
    return hipErrorInvalidValue;
  // Splits of 256 columns, two turns of a workgroup's waves; longer ones past
  // kMostAdapterSplits.
  const int turn = 32 * kWaves;
  const int turns = (a.cols + turn - 1) / turn;
  a.split_cols = turn * (turns <= 2 * kMostAdapterSplits
                             ? 2 : (turns + kMostAdapterSplits - 1) / kMostAdapterSplits);
  a.splits = (a.cols + a.split_cols - 1) / a.split_cols;
  const uint32_t blocks = (a.rows + kBlockRows - 1) / kBlockRows;
  const uint64_t most = 2048;  // workgroups; each takes every so many items
  const uint64_t down = (uint64_t)a.tokens * a.splits, up = (uint64_t)a.tokens * blocks;
  const uint32_t grid_down = (uint32_t)(down < most ? down : most);
  const uint32_t grid_up = (uint32_t)(up < most ? up : most);
  switch (a.format) {
    case 0: return launch_format<0>(s, a, grid_down, grid_up);
    case 1: return launch_format<1>(s, a, grid_down, grid_up);
    case 30: return launch_format<30>(s, a, grid_down, grid_up);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace frz
