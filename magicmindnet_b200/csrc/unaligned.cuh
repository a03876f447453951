// Rows that start anywhere, through aligned vector accesses: a run of elements that
// straddles two aligned vectors is moved to its place in registers. Beside the
// second access that costs about two instructions an element, where single 2-byte
// accesses cost four times the memory instructions of the whole kernel.
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

// out = the V elements of T that end `o` (0 <= o < V) elements before the end of the
// 2 V held by w.
template <typename T, int V, int W = V * (int)sizeof(T) / 4>
__device__ __forceinline__ void shift_up(const uint32_t (&w)[2 * W], int o, uint32_t (&out)[W]) {
  constexpr bool kHalf = sizeof(T) == 2;
  const int s = kHalf ? o >> 1 : o;
  uint32_t d[2 * W];
#pragma unroll
  for (int i = 0; i < 2 * W; ++i) d[i] = w[i];
  if constexpr (W >= 4) {
#pragma unroll
    for (int i = 2 * W - 1; i >= 2; --i) d[i] = s & 2 ? d[i - 2] : d[i];
  }
#pragma unroll
  for (int i = 2 * W - 1; i >= W - 1 && i >= 1; --i) d[i] = s & 1 ? d[i - 1] : d[i];
#pragma unroll
  for (int i = 0; i < W; ++i)
    out[i] = kHalf ? __funnelshift_l(d[W + i - 1], d[W + i], (o & 1) * 16) : d[W + i];
}

// The V elements at the aligned address p as words; those outside [begin, end) are
// not read (a vector that reaches past either end is read one element at a time).
template <typename T, int V, int W = V * (int)sizeof(T) / 4>
__device__ __forceinline__ void load_within(const T* p, const T* begin, const T* end,
                                            uint32_t* w) {
  if (p >= begin && p + V <= end) {
    if constexpr (W == 4) {
      const uint4 u = *reinterpret_cast<const uint4*>(p);
      w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
    } else {
      const uint2 u = *reinterpret_cast<const uint2*>(p);
      w[0] = u.x, w[1] = u.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = 0;
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (p + j >= begin && p + j < end) {
        if constexpr (sizeof(T) == 2)
          w[j >> 1] |= (uint32_t)*reinterpret_cast<const uint16_t*>(p + j) << (16 * (j & 1));
        else
          w[j] = *reinterpret_cast<const uint32_t*>(p + j);
      }
  }
}

// V elements at any address p; those outside [begin, end) come back as zero.
template <typename T, int V, int W = V * (int)sizeof(T) / 4>
__device__ __forceinline__ void load_unaligned(const T* p, const T* begin, const T* end,
                                               uint32_t (&out)[W]) {
  const int o = vec_offset<T, V>(p);
  uint32_t w[2 * W];
  load_within<T, V>(p - o, begin, end, w);
#pragma unroll
  for (int i = 0; i < W; ++i) w[W + i] = 0;
  if (o) load_within<T, V>(p - o + V, begin, end, w + W);
  shift_down<T, V>(w, o, out);
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
