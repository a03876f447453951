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

// Moves words of T elements down by `o` elements (0 <= o < 16 bytes' worth), in place:
// the first N of d then start there.
template <typename T, int N>
__device__ __forceinline__ void shift_down(uint32_t (&d)[N + 4], int o) {
  constexpr bool kHalf = sizeof(T) == 2;
  const int s = kHalf ? o >> 1 : o;
#pragma unroll
  for (int i = 0; i < N + 2; ++i) d[i] = s & 2 ? d[i + 2] : d[i];
#pragma unroll
  for (int i = 0; i < N + 1; ++i) d[i] = s & 1 ? d[i + 1] : d[i];
  if constexpr (kHalf) {
#pragma unroll
    for (int i = 0; i < N; ++i) d[i] = __funnelshift_r(d[i], d[i + 1], 16 * (o & 1));
  }
}

// Zeros in place of all but the first n elements of N words.
template <typename T, int N, int M>
__device__ __forceinline__ void keep_first(uint32_t (&d)[M], int n) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if constexpr (sizeof(T) == 2)
      d[i] = 2 * i + 1 < n ? d[i] : (2 * i < n ? d[i] & 0xFFFFu : 0u);
    else
      d[i] = i < n ? d[i] : 0u;
  }
}

}  // namespace mmn
