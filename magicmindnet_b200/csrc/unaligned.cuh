// Rows that start anywhere, through aligned vector accesses: offsets from a vector's
// start, and elements moved to their place in registers.
#pragma once

#include <cstdint>

namespace mmn {

// Elements of T past the last multiple of V, of an address counted in elements.
template <typename T, int V>
__device__ __forceinline__ int vec_offset(const void* p) {
  return (int)(reinterpret_cast<uintptr_t>(p) / sizeof(T)) & (V - 1);
}

// out = the V elements of T that start `o` (0 <= o < V) elements into the 2 V held
// by w; W = the 32-bit words of V elements.
template <typename T, int V, int W = V * (int)sizeof(T) / 4>
__device__ __forceinline__ void shift_down(const uint32_t (&w)[2 * W], int o, uint32_t (&out)[W]) {
  constexpr bool kHalf = sizeof(T) == 2;
  const int s = kHalf ? o >> 1 : o;
  uint32_t d[2 * W + 1];
#pragma unroll
  for (int i = 0; i < 2 * W; ++i) d[i] = w[i];
  d[2 * W] = 0;
  if constexpr (W >= 4) {
#pragma unroll
    for (int i = 0; i + 2 < 2 * W; ++i) d[i] = s & 2 ? d[i + 2] : d[i];
  }
#pragma unroll
  for (int i = 0; i <= W && i + 1 < 2 * W; ++i) d[i] = s & 1 ? d[i + 1] : d[i];
#pragma unroll
  for (int i = 0; i < W; ++i)
    out[i] = kHalf ? __funnelshift_r(d[i], d[i + 1], (o & 1) * 16) : d[i];
}

// Zeros in place of all but the first n elements.
template <typename T, int V, int W = V * (int)sizeof(T) / 4>
__device__ __forceinline__ void keep_first(uint32_t (&w)[W], int n) {
#pragma unroll
  for (int i = 0; i < W; ++i) {
    if constexpr (sizeof(T) == 2)
      w[i] = 2 * i + 1 < n ? w[i] : (2 * i < n ? w[i] & 0xFFFFu : 0u);
    else
      w[i] = i < n ? w[i] : 0u;
  }
}

}  // namespace mmn
