// How the sampler's fp32 sums are taken, and how far they may be off.  Plain C++ too, so that a host can try it.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define SWVR_HD __host__ __device__ __forceinline__
#else
#define SWVR_HD inline
#endif

namespace swvr {
namespace sample {

// log2 of the largest score's fixed-point weight: sums of V of them stay below 2^63.
SWVR_HD int lg_one_of(int64_t V) {
  int lg = 0;
  while ((int64_t(1) << lg) < V) ++lg;
  return lg <= 18 ? 44 : 62 - lg;
}

constexpr int kRoughMost = 1 << 20;  // longest row with fp32 sums

// The sum of VEC (a power of two) weights, in a tree: log2(VEC) roundings, where one after another would take VEC - 1.
template <int VEC>
SWVR_HD float tree_sum(float (&v)[VEC]) {
#pragma unroll
  for (int o = VEC / 2; o > 0; o /= 2)
#pragma unroll
    for (int e = 0; e < o; ++e) v[e] += v[e + o];
  return v[0];
}

// How far a partial sum may be from the fixed-point one, in the units of a total, for rows of up to kRoughMost scores:
// 10 2^-24 of the total.  Relatively, and in 2^-24: 0.6 for the rounding of the exponent's rest, 4 for ex2, 3 for sums of eight, up to 2
// for the fixed point itself (half a unit a score: V 2^-(lg_one + 1), most at V = 2^20), 0.2 for cutting sums
// down to units of 2^-40.
SWVR_HD unsigned long long rough_error(unsigned long long total) { return (total >> 21) + (total >> 23) + 1; }

}  // namespace sample
}  // namespace swvr
