// Exchanges between the lanes of a wave that need no LDS, and reductions made of them (DPP and permlane swaps: a few cycles a step where a
// __shfl_xor takes an LDS round trip).  Every lane gets the result.
#pragma once
#include "common.h"

__device__ __forceinline__ float as_f(uint32_t u) { return __builtin_bit_cast(float, u); }
__device__ __forceinline__ uint32_t as_u(float f) { return __builtin_bit_cast(uint32_t, f); }

// the pairs (x[l], x[l ^ 16]) and (x[l], x[l ^ 32]) in some order
__device__ __forceinline__ void swap16(float x, float& a, float& b) {
  const auto p = __builtin_amdgcn_permlane16_swap(as_u(x), as_u(x), false, false);
  a = as_f(p[0]);
  b = as_f(p[1]);
}
__device__ __forceinline__ void swap32(float x, float& a, float& b) {
  const auto p = __builtin_amdgcn_permlane32_swap(as_u(x), as_u(x), false, false);
  a = as_f(p[0]);
  b = as_f(p[1]);
}
// maximum / sum over the four 16-lane groups that hold one query's keys
__device__ __forceinline__ float across_max(float x) {
  float a, b;
  swap16(x, a, b);
  swap32(fmaxf(a, b), a, b);
  return fmaxf(a, b);
}
__device__ __forceinline__ float across_sum(float x) {
  float a, b;
  swap16(x, a, b);
  swap32(a + b, a, b);
  return a + b;
}
// value of lane l ^ 1 / l ^ 2 (quad permutes), l + 4 / l + 8 in a ring of 16 (row rotations)
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return as_f((uint32_t)__builtin_amdgcn_mov_dpp((int)as_u(x), CTRL, 0xf, 0xf, true));
}
constexpr int DPP_HALF_MIRROR = 0x141, DPP_MIRROR = 0x140;           // lane 7 - l of eight, 15 - l of sixteen
constexpr int DPP_XOR1 = 0xB1, DPP_XOR2 = 0x4E, DPP_ROR4 = 0x124, DPP_ROR8 = 0x128;
// maximum of an unsigned number over the wave
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
  float a, b;
  x = max(x, as_u(dpp<DPP_XOR1>(as_f(x))));
  x = max(x, as_u(dpp<DPP_XOR2>(as_f(x))));
  x = max(x, as_u(dpp<DPP_ROR4>(as_f(x))));
  x = max(x, as_u(dpp<DPP_ROR8>(as_f(x))));
  swap16(as_f(x), a, b);
  swap32(as_f(max(as_u(a), as_u(b))), a, b);
  return max(as_u(a), as_u(b));
}
// maximum / sum over the wave's sixteen quads, each of which holds one value four times (the sum's last bit may differ from lane to lane)
__device__ __forceinline__ float quads_max(float x) {
  x = fmaxf(x, dpp<DPP_ROR4>(x));
  x = fmaxf(x, dpp<DPP_ROR8>(x));
  return across_max(x);
}
__device__ __forceinline__ float quads_sum(float x) {
  x += dpp<DPP_ROR4>(x);
  x += dpp<DPP_ROR8>(x);
  return across_sum(x);
}
// sum of an unsigned number over the wave
__device__ __forceinline__ uint32_t wave_sum_u(uint32_t x) {
  float a, b;
  x += as_u(dpp<DPP_XOR1>(as_f(x)));
  x += as_u(dpp<DPP_XOR2>(as_f(x)));
  x += as_u(dpp<DPP_ROR4>(as_f(x)));
  x += as_u(dpp<DPP_ROR8>(as_f(x)));
  swap16(as_f(x), a, b);
  swap32(as_f(as_u(a) + as_u(b)), a, b);
  return __builtin_amdgcn_readfirstlane(as_u(a) + as_u(b));
}
// maximum over the wave (NaN counts as nothing)
__device__ __forceinline__ float wave_max(float x) {
  x = fmaxf(x, dpp<DPP_XOR1>(x));
  x = fmaxf(x, dpp<DPP_XOR2>(x));
  return quads_max(x);
}
// sum over the wave, in 64 bits; the same bits in every lane (the rings add in another order in each)
template <int CTRL>
__device__ __forceinline__ double dpp64(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = as_u(dpp<CTRL>(as_f((uint32_t)u))), hi = as_u(dpp<CTRL>(as_f((uint32_t)(u >> 32))));
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double wave_sum64(double x) {
  x += dpp64<DPP_XOR1>(x);
  x += dpp64<DPP_XOR2>(x);
  x += dpp64<DPP_ROR4>(x);
  x += dpp64<DPP_ROR8>(x);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    float l0, l1, h0, h1;
    if (i == 0) {
      swap16(as_f((uint32_t)u), l0, l1);
      swap16(as_f((uint32_t)(u >> 32)), h0, h1);
    } else {
      swap32(as_f((uint32_t)u), l0, l1);
      swap32(as_f((uint32_t)(u >> 32)), h0, h1);
    }
    x = __builtin_bit_cast(double, (uint64_t)as_u(h0) << 32 | as_u(l0)) + __builtin_bit_cast(double, (uint64_t)as_u(h1) << 32 | as_u(l1));
  }
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(u >> 32)), lo = __builtin_amdgcn_readfirstlane((uint32_t)u);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// The least of the maxima of the wave's groups of 2^most lanes: a number that 64 >> most lanes reach at least.  Six exchanges; the K-th largest
// itself takes a search.
__device__ __forceinline__ uint32_t wave_group_bound(uint32_t x, int most) {
  auto pick = [&](int step, uint32_t a, uint32_t b) { return step < most ? max(a, b) : min(a, b); };
  x = pick(0, x, as_u(dpp<DPP_XOR1>(as_f(x))));
  x = pick(1, x, as_u(dpp<DPP_XOR2>(as_f(x))));
  x = pick(2, x, as_u(dpp<DPP_HALF_MIRROR>(as_f(x))));
  x = pick(3, x, as_u(dpp<DPP_MIRROR>(as_f(x))));
  float a, b;
  swap16(as_f(x), a, b);
  x = pick(4, as_u(a), as_u(b));
  swap32(as_f(x), a, b);
  return __builtin_amdgcn_readfirstlane(pick(5, as_u(a), as_u(b)));
}
