// QK-norm, rope and the append to pages of a batch's rows, each at its own
// request's position: rope_kernel's arithmetic and order of addition
// (rope_common.h), so that a row's bits are those of frz_op_rope.
//
// A head of D values is D / 8 lanes of a wave, which holds 512 / D heads: its
// squares are summed by a butterfly, whose every lane forms the halving tree's
// sum, and each lane turns the four pairs that it holds, so a wave shares
// nothing with another and waits for nothing but its loads. Few rows are one
// launch's latency (6 us a call, of which the kernel 1 to 2); 504 rows of 32
// query and 8 key-value heads of 128 (22.7 MB) take 6.8 us, 3.3 TB/s.

#include "batch_rules.h"
#include "kernels.h"
#include "rope_common.h"

namespace frz {
namespace {

using namespace rules;

__device__ __forceinline__ ushort4 pack4_bf16(float4 v) {
  ushort4 o;
  o.x = __builtin_bit_cast(uint16_t, (__bf16)v.x);
  o.y = __builtin_bit_cast(uint16_t, (__bf16)v.y);
  o.z = __builtin_bit_cast(uint16_t, (__bf16)v.z);
  o.w = __builtin_bit_cast(uint16_t, (__bf16)v.w);
  return o;
}

template <int kD>
__global__ __launch_bounds__(256) void paged_rope_kernel(PagedRopeArgs a) {
  constexpr int kLanes = kD / 8, kHalf = kD / 2;
  constexpr uint32_t kWaveHeads = 64 / kLanes;
  const uint32_t row = blockIdx.x;
  const uint32_t wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t lane = threadIdx.x & 63, l = lane % kLanes;
  const uint32_t heads = a.query_heads + 2 * a.cache.kv_heads;
  const uint32_t first = (blockIdx.y * 4 + wave) * kWaveHeads;
  if (first >= heads) return;
  const uint32_t p = a.positions[row];
  if (p == kNone) return;
  const uint32_t h = first + lane / kLanes;
  const bool active = h < heads;
  const bool is_query = h < a.query_heads;
  const bool is_value = h >= a.query_heads + a.cache.kv_heads;
  const uint32_t kv = is_value ? h - a.query_heads - a.cache.kv_heads : h - a.query_heads;
  const float* src = is_query   ? a.query + (uint64_t)row * a.q_stride + (uint64_t)h * kD
                     : is_value ? a.value + (uint64_t)row * a.kv_stride + (uint64_t)kv * kD
                                : a.key + (uint64_t)row * a.kv_stride + (uint64_t)kv * kD;
  float4 va = make_float4(0.f, 0.f, 0.f, 0.f), vb = va, ga = va, gb = va;
  if (active) {
    va = ld4f(src + 4 * l);
    vb = ld4f(src + kHalf + 4 * l);
    const float* gain = is_query ? a.query_gain : a.key_gain;
    ga = ld4f(gain + 4 * l);
    gb = ld4f(gain + kHalf + 4 * l);
  }
  // Where the row's keys and values go. Of rows at one request's position the
  // last is kept: a row looks whether one after it is there too, at all of
  // them at once (each of few loads that wait for one another had taken twice
  // the rest of a full step's kernel).
  uint64_t at = 0;
  bool kept = false;
  if (first + kWaveHeads > a.query_heads) {
    const uint32_t sequence = a.sequences ? a.sequences[row] : row;
    const uint32_t index = p / a.cache.page_slots, slot = p - index * a.cache.page_slots;
    const uint32_t page = page_at(a.cache.table, a.cache.sequences, a.cache.width, a.cache.pages,
                                  sequence, index);
    kept = page != kNone;
    at = page * a.cache.page_stride + (uint64_t)slot * a.cache.kv_heads * kD;
    if (a.sequences) {  // without, each row is its own request
      constexpr int kGroups = kMostRows / 64;
      uint32_t other[kGroups], of[kGroups];
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
        if (row + 1 + 64 * i >= a.rows) continue;
        const uint32_t r = min(row + 1 + 64 * i + lane, a.rows - 1);
        other[i] = a.positions[r];
        of[i] = a.sequences[r];
      }
      bool again = false;
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
        if (row + 1 + 64 * i >= a.rows) continue;
        again |= row + 1 + 64 * i + lane < a.rows && other[i] == p && of[i] == sequence;
      }
      kept = kept && __ballot(again) == 0;
    }
  }
  const float4 turns = ld4f(a.turns + 4 * l);
  float cosine[4], sine[4];
  rope_angle(turns.x, p, &sine[0], &cosine[0]);
  rope_angle(turns.y, p, &sine[1], &cosine[1]);
  rope_angle(turns.z, p, &sine[2], &cosine[2]);
  rope_angle(turns.w, p, &sine[3], &cosine[3]);
  float squares = rope_lane_squares(va, vb);
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) squares = squares + __shfl_xor(squares, o);
  if (!active) return;
  if (!is_value) {
    rope_normalize(va, vb, squares, kD, a.epsilon, ga, gb);
    rope_rotate(va, vb, 0, cosine, sine);
  }
  if (is_query) {
    float* dst = a.roped + (uint64_t)row * a.roped_stride + (uint64_t)h * kD;
    *reinterpret_cast<float4*>(dst + 4 * l) = va;
    *reinterpret_cast<float4*>(dst + kHalf + 4 * l) = vb;
  } else if (kept) {
    uint16_t* dst = (is_value ? a.cache.values : a.cache.keys) + at + (uint64_t)kv * kD;
    *reinterpret_cast<ushort4*>(dst + 4 * l) = a.cache.bf16 ? pack4_bf16(va) : pack4_f16(va);
    *reinterpret_cast<ushort4*>(dst + kHalf + 4 * l) =
        a.cache.bf16 ? pack4_bf16(vb) : pack4_f16(vb);
  }
}

template <int kD>
void launch_heads(hipStream_t s, const PagedRopeArgs& a) {
  constexpr uint32_t kGroupHeads = 4 * 512 / kD;  // heads a workgroup
  const uint32_t heads = a.query_heads + 2 * a.cache.kv_heads;
  hipLaunchKernelGGL(paged_rope_kernel<kD>,
                     dim3(a.rows, (heads + kGroupHeads - 1) / kGroupHeads), dim3(256), 0, s, a);
}

}  // namespace

hipError_t launch_paged_rope(hipStream_t s, const PagedRopeArgs& a) {
  if (a.rows == 0 || a.rows > kMostRows) return hipErrorInvalidValue;
  switch (a.cache.head_dim) {
    case 64: launch_heads<64>(s, a); break;
    case 128: launch_heads<128>(s, a); break;
    case 256: launch_heads<256>(s, a); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace frz
