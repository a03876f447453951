// Layer norm over the last axis, forward and backward, with the reduction of
// the gain's and shift's gradients (the ln1 / ln2 slots of the optimizer step;
// crates/mmn-nn/src/lib.rs LayerNorm is the CPU layer whose grads
// crates/mmn-models/src/chatbot.rs:118-206 hands to AdamW).
//
//   mu = sum x / d, v = sum (x - mu)^2 / d, r = 1 / sqrt(v + eps)
//   h = (x - mu) r,  y = h gamma + beta
//   g = dy gamma, c1 = sum g / d, c2 = sum g h / d, dx = r (g - c1 - h c2)
//   dgamma = sum over rows of dy h, dbeta = sum over rows of dy
//
// Bound by memory: a row is read once, into registers or shared memory, the
// squares are summed about the mean there (so that the variance of a row whose mean
// is large against its spread does not cancel), and the row is written once. All
// statistics and sums are fp32; y and dx are rounded once. The mean is an fp32 sum,
// and (x - mean) r carries its error: 2^-24 |mean| / sigma at least, with the sum's
// own up to some 2^-24 times the additions an element passes through (32 in a
// thread, 10 across) times mean|x| / sigma.
//
// Which kernel takes a call (measured on one B200 with operands that are not in L2,
// fractions of the 6.53 TB/s a copy reaches):
//   forward   ln_fwd_ring_kernel  bf16 rows, many and aligned: 16384 x 4096 in
//                                 44.0 us (0.93), 1.28 times as long with a row per
//                                 block; rows that start anywhere, beyond 1024 columns:
//                                 16384 x 4057 65.0 us (0.63), fp32 96.3 (0.85)
//             ln_fwd_rows_kernel  the rest of the rows that can be read four at a
//                                 time: 16384 x 2048 fp32 to bf16 in 34.5 us (0.89)
//             ln_fwd_kernel       an element at a time, where x and y start differently
//                                 and for fewer columns: 3001 x 1013 fp32 in 11.1
//                                 us (0.34; 6.8 from L2), 16384 x 4057 bf16 132 (0.31)
//             ln_fwd_wide_kernel  rows beyond 16384
//   backward  ln_bwd_ring_kernel  aligned rows of 65 columns to where two rows of x and
//                                 dy (and beyond 8192 columns gamma) no longer fit one SM's
//                                 shared memory: 16384 in bf16, 14080 in mixed types,
//                                 11264 in fp32. 16384 x 4096 bf16 in 75.7 us (0.81) with
//                                 the closing sums, 113 us with the rows loaded into
//                                 registers; rows that start anywhere, beyond 512 columns:
//                                 16384 x 4057 107 us (0.57), fp32 143 (0.85)
//             ln_bwd_kernel       narrow rows, and an element at a time up to 8192
//                                 columns: 3001 x 1013 fp32 15.8 us (12.9 by vectors),
//                                 16384 x 4057 bf16 158
//             ln_bwd_wide_*       the rest: 4096 x 11272 fp32 204 us (11264: 118),
//                                 16384 320
#include <cuda_bf16.h>

#include <algorithm>
#include <mutex>

#include "capi_internal.cuh"
#include "mmn_ptx.cuh"
#include "unaligned.cuh"

namespace mmn {
namespace {

// ------------------------------------------------------------ element access
__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_f32(float& d, float x) { d = x; }
__device__ __forceinline__ void from_f32(__nv_bfloat16& d, float x) { d = __float2bfloat16_rn(x); }

// V consecutive elements as one vector access (V * sizeof(T) a power of two up
// to 16 bytes, or a multiple of 16 bytes).
template <typename T, int V>
struct alignas(V * sizeof(T) < 16 ? V * sizeof(T) : 16) Vec {
  T e[V];
};

template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load_vec(const T* p) {
  return *reinterpret_cast<const Vec<T, V>*>(p);
}

// V elements of gamma or beta, held in fp32 or bf16.
template <int V>
__device__ __forceinline__ void load_param(const void* p, bool bf16, int64_t c, float (&v)[V]) {
  if (bf16) {
    const Vec<__nv_bfloat16, V> u = load_vec<__nv_bfloat16, V>(
        static_cast<const __nv_bfloat16*>(p) + c);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = __bfloat162float(u.e[j]);
  } else {
    const Vec<float, V> u = load_vec<float, V>(static_cast<const float*>(p) + c);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = u.e[j];
  }
}

// Sum over the TR threads of a row (TR <= 32: lanes; else the whole block, with
// `red` a 32-entry shared buffer that the caller alternates between calls).
template <int TR>
__device__ __forceinline__ float2 row_sum(float2 v, float2* red) {
#pragma unroll
  for (int o = (TR < 32 ? TR : 32) / 2; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  if constexpr (TR > 32) {
    constexpr int W = TR / 32;
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[threadIdx.x & (W - 1)];
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) {
      v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
      v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
  }
  return v;
}

struct LnFwd {
  const void* x;
  const void* gamma;
  const void* beta;
  void* y;
  float* mean;
  float* rstd;
  int64_t x_ld, y_ld, rows, cols;
  float eps;
  int param_bf16;
};

struct LnBwd {
  const void* dy;
  const void* x;
  const void* gamma;
  const float* mean;
  const float* rstd;
  void* dx;
  float* partial;  // [blocks][2][cols]: dgamma, dbeta sums of each block's rows
  int64_t dy_ld, x_ld, dx_ld, rows, cols;
  int param_bf16;
};

// ------------------------------------------------------------------- forward
// Rows at any alignment: TR threads hold one row, NE elements each, taken one at a
// time.
template <typename XT, typename YT, int TR, int NE>
__global__ void __launch_bounds__(TR <= 32 ? 128 : TR) ln_fwd_kernel(const LnFwd a) {
  constexpr int kBlock = TR <= 32 ? 128 : TR, RB = kBlock / TR;
  __shared__ float2 red[2][32];
  griddep_wait();
  griddep_launch_dependents();
  const int t = threadIdx.x % TR;
  const int64_t row = (int64_t)blockIdx.x * RB + threadIdx.x / TR;
  const bool ok = row < a.rows;
  const XT* x = static_cast<const XT*>(a.x) + (ok ? row : 0) * a.x_ld;
  float v[NE], s = 0.0f;
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    const int c = i * TR + t;
    v[i] = ok && c < a.cols ? to_f32(x[c]) : 0.0f;
    s += v[i];
  }
  const float n = (float)a.cols;
  const float mean = row_sum<TR>(make_float2(s, 0.0f), red[0]).x / n;
  float q = 0.0f;
#pragma unroll
  for (int i = 0; i < NE; ++i)
    if (i * TR + t < a.cols) {
      const float d = v[i] - mean;
      q += d * d;
    }
  const float var = row_sum<TR>(make_float2(q, 0.0f), red[1]).x / n;
  const float rstd = 1.0f / sqrtf(var + a.eps);
  if (!ok) return;
  if (t == 0) {
    if (a.mean) a.mean[row] = mean;
    if (a.rstd) a.rstd[row] = rstd;
  }
  YT* y = static_cast<YT*>(a.y) + row * a.y_ld;
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    const int c = i * TR + t;
    if (c < a.cols) {
      float ga[1], be[1];
      load_param<1>(a.gamma, a.param_bf16, c, ga);
      load_param<1>(a.beta, a.param_bf16, c, be);
      from_f32(y[c], (v[i] - mean) * rstd * ga[0] + be[0]);
    }
  }
}

// Rows too wide for the registers: one block per row, read three times (the
// second and third time mostly from L1 and L2).
template <typename XT, typename YT>
__global__ void __launch_bounds__(512) ln_fwd_wide_kernel(const LnFwd a) {
  __shared__ float2 red[2][32];
  griddep_wait();
  griddep_launch_dependents();
  const int64_t row = blockIdx.x;
  const XT* x = static_cast<const XT*>(a.x) + row * a.x_ld;
  YT* y = static_cast<YT*>(a.y) + row * a.y_ld;
  const float n = (float)a.cols;
  float s = 0.0f;
  for (int64_t c = threadIdx.x; c < a.cols; c += 512) s += to_f32(x[c]);
  const float mean = row_sum<512>(make_float2(s, 0.0f), red[0]).x / n;
  float q = 0.0f;
  for (int64_t c = threadIdx.x; c < a.cols; c += 512) {
    const float d = to_f32(x[c]) - mean;
    q += d * d;
  }
  const float var = row_sum<512>(make_float2(q, 0.0f), red[1]).x / n;
  const float rstd = 1.0f / sqrtf(var + a.eps);
  if (threadIdx.x == 0) {
    if (a.mean) a.mean[row] = mean;
    if (a.rstd) a.rstd[row] = rstd;
  }
  for (int64_t c = threadIdx.x; c < a.cols; c += 512) {
    float ga[1], be[1];
    load_param<1>(a.gamma, a.param_bf16, c, ga);
    load_param<1>(a.beta, a.param_bf16, c, be);
    from_f32(y[c], (to_f32(x[c]) - mean) * rstd * ga[0] + be[0]);
  }
}

// ------------------------------------------------------- pairs of fp32 values
// sm_100 adds, multiplies and fuses two fp32 values per instruction; each half
// rounds as the scalar instruction does.
typedef unsigned long long f2;
__device__ __forceinline__ f2 pack2(float lo, float hi) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ f2 dup2(float v) { return pack2(v, v); }
__device__ __forceinline__ float2 unpack2(f2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float sum2(f2 v) {
  const float2 f = unpack2(v);
  return f.x + f.y;
}

// V consecutive elements as V / 2 pairs, and back (rounded to T).
template <typename T, int V>
__device__ __forceinline__ void load_pairs(const T* p, f2* v) {
  const Vec<T, V> u = load_vec<T, V>(p);
  if constexpr (sizeof(T) == 2) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&u);
#pragma unroll
    for (int j = 0; j < V / 2; ++j)
      v[j] = pack2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xFFFF0000u));
  } else {
#pragma unroll
    for (int j = 0; j < V / 2; ++j) v[j] = pack2(to_f32(u.e[2 * j]), to_f32(u.e[2 * j + 1]));
  }
}
template <typename T, int V>
__device__ __forceinline__ void store_pairs(T* p, const f2* v) {
  Vec<T, V> u;
#pragma unroll
  for (int j = 0; j < V / 2; ++j) {
    const float2 f = unpack2(v[j]);
    if constexpr (sizeof(T) == 2) {
      reinterpret_cast<__nv_bfloat162*>(&u)[j] = __floats2bfloat162_rn(f.x, f.y);
    } else {
      from_f32(u.e[2 * j], f.x);
      from_f32(u.e[2 * j + 1], f.y);
    }
  }
  *reinterpret_cast<Vec<T, V>*>(p) = u;
}
template <int V>
__device__ __forceinline__ void load_param_pairs(const void* p, bool bf16, int64_t c, f2* v) {
  float u[V];
  load_param<V>(p, bf16, c, u);
#pragma unroll
  for (int j = 0; j < V / 2; ++j) v[j] = pack2(u[2 * j], u[2 * j + 1]);
}

// A row's sum over the TR threads that hold it (red: one entry per warp of the row;
// another buffer for the next call).
template <int TR>
__device__ __forceinline__ float row_sum1(float v, float* red) {
#pragma unroll
  for (int o = (TR < 32 ? TR : 32) / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (TR > 32) {
    constexpr int W = TR / 32;
    if ((threadIdx.x & 31) == 0) red[(threadIdx.x >> 5) & (W - 1)] = v;
    __syncthreads();
    if constexpr (W == 2) {
      v = red[0] + red[1];
    } else {
      v = 0.0f;
#pragma unroll
      for (int w = 0; w < W; w += 4) {
        const float4 u = *reinterpret_cast<const float4*>(red + w);
        v += (u.x + u.y) + (u.z + u.w);
      }
    }
  }
  return v;
}

// Two sums at once: the lanes with bit 4 clear go on with the first, the others
// with the second (5 exchanges a warp in place of 10).
template <int TR>
__device__ __forceinline__ float2 ring_sum2(float x, float y, float2* red) {
  const bool up = (threadIdx.x & 16) != 0;
  float v = (up ? y : x) + __shfl_xor_sync(0xffffffffu, up ? x : y, 16);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (TR == 32) {
    return make_float2(__shfl_sync(0xffffffffu, v, 0), __shfl_sync(0xffffffffu, v, 16));
  } else {
    constexpr int W = TR / 32;
    if ((threadIdx.x & 15) == 0) reinterpret_cast<float*>(red)[(threadIdx.x >> 5) * 2 + (up ? 1 : 0)] = v;
    __syncthreads();
    f2 t = 0;
#pragma unroll
    for (int w = 0; w < W; w += 2) {
      const float4 u = *reinterpret_cast<const float4*>(red + w);
      t = add2(t, add2(pack2(u.x, u.y), pack2(u.z, u.w)));
    }
    return unpack2(t);
  }
}

// Rows that start anywhere (EDGE in the ring kernels). A row's columns are counted
// from the vector that its first element lies in, o columns earlier, so every access
// stays a whole vector and only a row's first and last one need care. That works
// because o repeats every eight rows: a row group takes rows a multiple of eight
// apart, has one o for all of them, and holds gamma and beta (and the sums of their
// gradients) moved by it. All matrices of the call have to agree in o.
//
// The row comes into a 16-byte aligned slot of shared memory, at its offset from 16
// bytes: `n` elements from `from` by bulk copy. Those are all whole vectors that the
// row touches, as long as they lie in the matrix [begin, end); else those inside the
// row, and the issuing thread copies its ends.
struct Hull {
  int from, n;
};
template <typename T>
__device__ __forceinline__ Hull row_hull(uint8_t* slot, const T* row, int cols, const T* begin,
                                         const T* end) {
  constexpr int A = 16 / sizeof(T);
  const int o = vec_offset<T, A>(row), n = (o + cols + A - 1) / A * A;
  if (row - o >= begin && row - o + n <= end) return {-o, n};
  const int lo = o ? A : 0, hi = (o + cols) / A * A;
  T* s = reinterpret_cast<T*>(slot);
  for (int j = o; j < lo; ++j) s[j] = row[j - o];
  for (int j = hi; j < o + cols; ++j) s[j] = row[j - o];
  return {lo - o, hi - lo};
}
template <typename T>
__device__ __forceinline__ void load_hull(uint8_t* slot, const T* row, Hull h, uint64_t* bar) {
  constexpr int A = 16 / sizeof(T);
  bulk_load(slot + (vec_offset<T, A>(row) + h.from) * sizeof(T), row + h.from, h.n * sizeof(T), bar);
}
__host__ __device__ constexpr int hull_bytes(int64_t cols, int es) {
  return (int)((cols * es + 15) / 16 * 16 + 16);
}

// Zeros in place of elements outside [lo, hi) of V.
template <int V>
__device__ __forceinline__ void keep_pairs(f2* v, int lo, int hi) {
#pragma unroll
  for (int j = 0; j < V / 2; ++j) {
    const float2 f = unpack2(v[j]);
    v[j] = pack2(2 * j >= lo && 2 * j < hi ? f.x : 0.0f,
                 2 * j + 1 >= lo && 2 * j + 1 < hi ? f.y : 0.0f);
  }
}

// gamma or beta from column c on; zeros outside [0, cols).
template <int V>
__device__ __forceinline__ void load_param_edge(const void* p, bool bf16, int c, int cols, f2* v) {
  float u[V];
#pragma unroll
  for (int j = 0; j < V; ++j)
    u[j] = c + j < 0 || c + j >= cols ? 0.0f
           : bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[c + j])
                  : static_cast<const float*>(p)[c + j];
#pragma unroll
  for (int j = 0; j < V / 2; ++j) v[j] = pack2(u[2 * j], u[2 * j + 1]);
}

// Bit i: a thread's chunk i holds a row's first or last elements and others.
template <int V, int TR, int NC>
__device__ __forceinline__ uint32_t row_ends(int t, int o, int cols) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = (i * TR + t) * V - o;
    m |= (c < 0 || c + V > cols ? 1u : 0u) << i;
  }
  return m;
}

// Those of the V elements from column c on that lie in [0, cols).
template <typename T, int V>
__device__ __forceinline__ void store_edge(T* row, int c, int cols, const f2* v) {
#pragma unroll
  for (int j = 0; j < V; ++j)
    if (c + j >= 0 && c + j < cols) {
      const float2 f = unpack2(v[j / 2]);
      from_f32(row[c + j], j & 1 ? f.y : f.x);
    }
}

constexpr int kRingMax = 4;  // rows in flight per row group, at most (8 gained nothing)
constexpr int kFwdRing = 2;  // ... in the forward kernel

// A row group whose block has given up a wait: those of its `asked` rows that are still
// on their way land, or run out of time too, before the block leaves its shared
// memory to another. By the thread that issued them; it asks for no more rows once a
// wait has given up (a slot whose row is still on its way must not be asked for another).
__device__ __forceinline__ void ring_drain(uint64_t* bars, int asked, int depth) {
#pragma unroll 1
  for (int k = asked > depth ? asked - depth : 0; k < asked; ++k) {
    const uint64_t start = global_timer_ns();
    while (!mbar_try_wait(&bars[k % depth], (uint32_t)(k / depth) & 1u))
      if (global_timer_ns() - start > kWaitLimitNs) break;
  }
}

// The forward kernel for rows that can be read four elements at a time: TR threads
// hold one row, NE columns each, a block a row (or a few short ones). Chunks of
// four keep every access, the fp32 parameters' too, to whole consecutive lines
// per warp. A block lives 2 to 3 us, most of it waiting, so what is in flight is
// what the blocks on the GPU hold: enough for fp32 rows (16384 x 4096 in 80.9
// us, 6.6 TB/s; 86 us with a third fewer blocks an SM) and not for bf16 ones (54.8 us
// on one set of operands, where ln_fwd_ring_kernel takes 42.9).
__host__ __device__ constexpr int ln_rows_block(int tr) { return tr <= 32 ? 128 : tr; }

template <typename XT, typename YT, int TR, int NE>
__global__ void __launch_bounds__(ln_rows_block(TR), ln_rows_block(TR) > 512 ? 1 : 1536 / ln_rows_block(TR))
    ln_fwd_rows_kernel(const LnFwd a) {
  constexpr int kBlock = ln_rows_block(TR), RB = kBlock / TR, V = 4, NC = NE / V, H = V / 2;
  __shared__ __align__(16) float red[2][RB][32];
  const int t = threadIdx.x % TR, sub = threadIdx.x / TR;
  const int64_t row = (int64_t)blockIdx.x * RB + sub;
  const bool ok = row < a.rows;
  const int cols = ok ? (int)a.cols : 0;
  const XT* x = static_cast<const XT*>(a.x) + row * a.x_ld;
  griddep_wait();
  griddep_launch_dependents();
  f2 v[NE / 2];
  f2 s = 0;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = (i * TR + t) * V;
    if (c < cols) {
      load_pairs<XT, V>(x + c, v + i * H);
    } else {
#pragma unroll
      for (int j = 0; j < H; ++j) v[i * H + j] = 0;
    }
  }
#pragma unroll
  for (int j = 0; j < NE / 2; ++j) s = add2(s, v[j]);
  const float inv_n = 1.0f / (float)a.cols;
  const float mean = row_sum1<TR>(sum2(s), red[0][sub]) * inv_n;
  const f2 nm = dup2(-mean);
  f2 q = 0;
#pragma unroll
  for (int i = 0; i < NC; ++i)
    if ((i * TR + t) * V < cols) {
#pragma unroll
      for (int j = 0; j < H; ++j) {
        v[i * H + j] = add2(v[i * H + j], nm);
        q = fma2(v[i * H + j], v[i * H + j], q);
      }
    }
  const float var = row_sum1<TR>(sum2(q), red[1][sub]) * inv_n;
  const float rstd = 1.0f / sqrtf(var + a.eps);
  if (t == 0 && ok) {
    if (a.mean) a.mean[row] = mean;
    if (a.rstd) a.rstd[row] = rstd;
  }
  const f2 r2 = dup2(rstd);
  YT* y = static_cast<YT*>(a.y) + row * a.y_ld;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = (i * TR + t) * V;
    if (c < cols) {
      f2 ga[H], be[H];
      load_param_pairs<V>(a.gamma, a.param_bf16, c, ga);
      load_param_pairs<V>(a.beta, a.param_bf16, c, be);
#pragma unroll
      for (int j = 0; j < H; ++j) ga[j] = fma2(mul2(v[i * H + j], r2), ga[j], be[j]);
      store_pairs<YT, V>(y + c, ga);
    }
  }
}

// bf16 rows, many of them: blocks walk the rows. gamma and beta stay in registers,
// each row group keeps a ring of rows in flight through bulk copies, and a
// thread takes 32 columns, since the conversions and the two sums across the
// threads cost more instructions than the arithmetic. Rows that start and end on 16
// bytes, or (EDGE) anywhere, then of both types, with 16 columns a thread up to 4096,
// for the ends' sake: 20000 x 2037 bf16 44.7 us, 54.3 with 32.
__host__ __device__ constexpr int ln_ring_block(int tr) { return tr <= 64 ? 128 : tr; }
__host__ __device__ constexpr int ln_ring_blocks(int tr, int ne) {
  return (ne > 16 ? 512 : 768) / ln_ring_block(tr);
}

template <typename XT, typename YT, int TR, int NE, bool EDGE>
__global__ void __launch_bounds__(ln_ring_block(TR), ln_ring_blocks(TR, NE))
    ln_fwd_ring_kernel(const LnFwd a, int depth, int* timeouts) {
  constexpr int V = sizeof(XT) == 2 && sizeof(YT) == 2 ? 8 : 4;
  constexpr int kBlock = ln_ring_block(TR), RB = kBlock / TR, NC = NE / V, H = V / 2;
  extern __shared__ __align__(16) uint8_t dyn[];
  __shared__ __align__(16) float red[2][RB][32];
  __shared__ __align__(8) uint64_t bars[RB][kRingMax];
  __shared__ volatile int abort_flag;
  __shared__ int asked[RB];  // rows that each group has asked for in the end
  const int t = threadIdx.x % TR, sub = threadIdx.x / TR;
  const int cols = (int)a.cols;
  const int rb = EDGE ? hull_bytes(cols, sizeof(XT)) : cols * (int)sizeof(XT);
  uint8_t* ring = dyn + sub * depth * rb;
  const int64_t first = (int64_t)blockIdx.x * RB + sub, step = (int64_t)gridDim.x * RB;
  if (threadIdx.x == 0) {
    for (int g = 0; g < RB; ++g)
      for (int d = 0; d < depth; ++d) mbar_init(&bars[g][d], 1);
    abort_flag = 0;
    fence_barrier_init();
  }
  __syncthreads();
  // rows of this group; the block runs as many trips as its first group has
  const int mine = first < a.rows ? (int)((a.rows - first + step - 1) / step) : 0;
  const int trips = (int)((a.rows - (int64_t)blockIdx.x * RB + step - 1) / step);
  const XT* x = static_cast<const XT*>(a.x) + first * a.x_ld;
  YT* y = static_cast<YT*>(a.y) + first * a.y_ld;
  const int at = EDGE ? vec_offset<XT, 16 / sizeof(XT)>(x) : 0, o = at & (V - 1);
  auto issue = [&](int k, int slot) {  // row k of this group into a slot
    const XT* row = x + k * step * a.x_ld;
    if constexpr (EDGE) {
      const XT* const begin = static_cast<const XT*>(a.x);
      const Hull h = row_hull(ring + slot * rb, row, cols, begin,
                              begin + (a.rows - 1) * a.x_ld + a.cols);
      mbar_arrive_expect_tx(&bars[sub][slot], h.n * (int)sizeof(XT));
      load_hull(ring + slot * rb, row, h, &bars[sub][slot]);
    } else {
      mbar_arrive_expect_tx(&bars[sub][slot], rb);
      bulk_load(ring + slot * rb, row, rb, &bars[sub][slot]);
    }
  };
  griddep_wait();
  griddep_launch_dependents();
  if (t == 0) {
    for (int k = 0; k < depth && k < mine; ++k) issue(k, k);
    asked[sub] = mine;
  }
  f2 ga[NE / 2], be[NE / 2];
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = (i * TR + t) * V - o;
    if constexpr (EDGE) {
      load_param_edge<V>(a.gamma, a.param_bf16, c, cols, ga + i * H);
      load_param_edge<V>(a.beta, a.param_bf16, c, cols, be + i * H);
    } else if (c < cols) {
      load_param_pairs<V>(a.gamma, a.param_bf16, c, ga + i * H);
      load_param_pairs<V>(a.beta, a.param_bf16, c, be + i * H);
    }
  }
  const uint32_t ends = EDGE ? row_ends<V, TR, NC>(t, o, cols) : 0u;
  const float inv_n = 1.0f / (float)cols;
  int slot = 0;
  uint32_t phase = 0;
  for (int k = 0; k < trips; ++k) {
    const bool ok = k < mine;
    const int lim = ok ? cols : -V;  // (below a row's first vector: no row, no columns)
    const XT* sx = reinterpret_cast<const XT*>(ring + slot * rb) + at;
    // (a wait that gives up is counted; the loop runs on so that every
    // barrier is met)
    if (ok) mbar_wait(&bars[sub][slot], phase, &abort_flag);
    f2 v[NE / 2], s = 0;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = (i * TR + t) * V - o;
      if (c < lim) {
        load_pairs<XT, V>(sx + c, v + i * H);
        if (EDGE && (ends >> i & 1)) keep_pairs<V>(v + i * H, -c, cols - c);
#pragma unroll
        for (int j = 0; j < H; ++j) s = add2(s, v[i * H + j]);
      }
    }
    const float mean = row_sum1<TR>(sum2(s), red[0][sub]) * inv_n;
    if constexpr (TR <= 32) __syncwarp();
    // every thread of the group has the row in registers: its slot is free
    if (t == 0 && k + depth < mine) {
      if (!abort_flag)
        issue(k + depth, slot);
      else
        asked[sub] = min(asked[sub], k + depth);
    }
    const f2 nm = dup2(-mean);
    f2 q = 0;
#pragma unroll
    for (int i = 0; i < NC; ++i)
      if (const int c = (i * TR + t) * V - o; c < lim) {
#pragma unroll
        for (int j = 0; j < H; ++j) v[i * H + j] = add2(v[i * H + j], nm);
        if (EDGE && (ends >> i & 1)) keep_pairs<V>(v + i * H, -c, cols - c);
#pragma unroll
        for (int j = 0; j < H; ++j) q = fma2(v[i * H + j], v[i * H + j], q);
      }
    const float var = row_sum1<TR>(sum2(q), red[1][sub]) * inv_n;
    const float rstd = 1.0f / sqrtf(var + a.eps);
    if (t == 0 && ok) {
      if (a.mean) a.mean[first + k * step] = mean;
      if (a.rstd) a.rstd[first + k * step] = rstd;
    }
    const f2 r2 = dup2(rstd);
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = (i * TR + t) * V - o;
      if (c < lim) {
#pragma unroll
        for (int j = 0; j < H; ++j)
          v[i * H + j] = fma2(mul2(v[i * H + j], r2), ga[i * H + j], be[i * H + j]);
        if (EDGE && (ends >> i & 1))
          store_edge<YT, V>(y, c, cols, v + i * H);
        else
          store_pairs<YT, V>(y + c, v + i * H);
      }
    }
    y += step * a.y_ld;
    if (++slot == depth) {
      slot = 0;
      phase ^= 1u;
    }
  }
  if constexpr (TR <= 32) __syncthreads();  // the waits of every group are over
  if (abort_flag) {
    if (t == 0) ring_drain(bars[sub], asked[sub], depth);
    if (threadIdx.x == 0) atomicAdd(timeouts, 1);
  }
}

// ------------------------------------------------------------------ backward
// Blocks walk the rows; a thread owns the same columns in every row and keeps
// their dgamma and dbeta sums in registers, so the rows are read once for both
// results. Each block writes its sums; ln_bwd_sum_kernel adds them in a fixed
// order (no atomics: the result does not depend on timing).
__host__ __device__ constexpr int ln_bwd_block(int tr) {
  return tr == 8 ? 256 : tr == 32 ? 64 : tr;
}
__host__ __device__ constexpr int ln_bwd_min_blocks(int tr) {
  return tr == 8 ? 2 : 512 / ln_bwd_block(tr);
}

template <typename XT, typename DT, int V, int TR, int NE>
__global__ void __launch_bounds__(ln_bwd_block(TR), ln_bwd_min_blocks(TR))
    ln_bwd_kernel(const LnBwd a) {
  constexpr int kBlock = ln_bwd_block(TR), RB = kBlock / TR, NC = NE / V;
  __shared__ float2 red[2][32];
  griddep_wait();
  griddep_launch_dependents();
  const int t = threadIdx.x % TR, sub = threadIdx.x / TR;
  const float inv_n = 1.0f / (float)a.cols;
  float sg[NE], sb[NE];  // dgamma, dbeta of this thread's columns
#pragma unroll
  for (int k = 0; k < NE; ++k) sg[k] = sb[k] = 0.0f;
  int par = 0;
  const int64_t step = (int64_t)gridDim.x * RB;
  // every thread of a warp takes the same trips: the loop runs on the block's first row
  for (int64_t row0 = (int64_t)blockIdx.x * RB; row0 < a.rows; row0 += step) {
    const int64_t row = row0 + sub;
    const bool ok = row < a.rows;
    const XT* x = static_cast<const XT*>(a.x) + (ok ? row : 0) * a.x_ld;
    const DT* dy = static_cast<const DT*>(a.dy) + (ok ? row : 0) * a.dy_ld;
    Vec<XT, V> xr[NC];
    Vec<DT, V> dr[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int64_t c = (int64_t)(i * TR + t) * V;
      if (ok && c < a.cols) {
        xr[i] = load_vec<XT, V>(x + c);
        dr[i] = load_vec<DT, V>(dy + c);
      }
    }
    const float mean = ok ? a.mean[row] : 0.0f, rstd = ok ? a.rstd[row] : 0.0f;
    float h[NE], g[NE];
    float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int64_t c = (int64_t)(i * TR + t) * V;
      if (ok && c < a.cols) {
        float ga[V];
        load_param<V>(a.gamma, a.param_bf16, c, ga);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int k = i * V + j;
          const float d = to_f32(dr[i].e[j]);
          h[k] = (to_f32(xr[i].e[j]) - mean) * rstd;
          g[k] = d * ga[j];
          s.x += g[k];
          s.y += g[k] * h[k];
          sg[k] += d * h[k];
          sb[k] += d;
        }
      }
    }
    s = row_sum<TR>(s, red[par]);
    par ^= 1;
    const float c1 = s.x * inv_n, c2 = s.y * inv_n;
    if (ok) {
      XT* dx = static_cast<XT*>(a.dx) + row * a.dx_ld;
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int64_t c = (int64_t)(i * TR + t) * V;
        if (c < a.cols) {
          Vec<XT, V> o;
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const int k = i * V + j;
            from_f32(o.e[j], rstd * (g[k] - c1 - h[k] * c2));
          }
          *reinterpret_cast<Vec<XT, V>*>(dx + c) = o;
        }
      }
    }
  }
  float* out = a.partial + (int64_t)blockIdx.x * 2 * a.cols;
  if constexpr (RB == 1) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int64_t c = (int64_t)(i * TR + t) * V;
      if (c < a.cols) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          out[c + j] = sg[i * V + j];
          out[a.cols + c + j] = sb[i * V + j];
        }
      }
    }
  } else {
    // the block's RB row groups, added in order
    __shared__ float acc[RB][TR * NE];
#pragma unroll
    for (int pass = 0; pass < 2; ++pass) {
#pragma unroll
      for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j)
          acc[sub][(i * TR + t) * V + j] = pass ? sb[i * V + j] : sg[i * V + j];
      __syncthreads();
      for (int c = threadIdx.x; c < TR * NE && c < a.cols; c += kBlock) {
        float v = 0.0f;
#pragma unroll
        for (int r = 0; r < RB; ++r) v += acc[r][c];
        out[pass * a.cols + c] = v;
      }
      __syncthreads();
    }
  }
}

// The same walk with the rows brought in by bulk copies: every row group keeps a
// ring of `depth` rows of x and dy in flight in shared memory, so the loads of
// the next rows run under the sums, the barrier and the stores of this one
// (16384 x 4096 bf16: 113 us with the rows loaded into registers).
// Rows that start and end on 16 bytes, or (EDGE) anywhere. NE <= 16: gamma, h and g
// live in registers. NE = 32 (rows of 8192 to 16384): gamma is kept in shared memory, and
// the second pass reads the row again.
template <typename XT, typename DT, int V, int TR, int NE, bool EDGE>
__global__ void __launch_bounds__(ln_bwd_block(TR), ln_bwd_min_blocks(TR))
    ln_bwd_ring_kernel(const LnBwd a, int depth, int* timeouts) {
  constexpr int kBlock = ln_bwd_block(TR), RB = kBlock / TR, NC = NE / V, H = V / 2;
  constexpr bool kReread = NE > 16;
  extern __shared__ __align__(16) uint8_t dyn[];
  __shared__ __align__(16) float2 red[2][32];
  __shared__ __align__(8) uint64_t bars[RB][kRingMax];
  __shared__ volatile int abort_flag;
  __shared__ int asked[RB];  // rows that each group has asked for in the end
  const int t = threadIdx.x % TR, sub = threadIdx.x / TR;
  const int cols = (int)a.cols;
  const int xb = EDGE ? hull_bytes(cols, sizeof(XT)) : cols * (int)sizeof(XT);
  const int db = EDGE ? hull_bytes(cols, sizeof(DT)) : cols * (int)sizeof(DT), rb = xb + db;
  const int gb = kReread ? (EDGE ? (cols + 2 * V) / 4 * 16 : cols * 4) : 0;
  float* gs = reinterpret_cast<float*>(dyn);  // gamma (kReread)
  uint8_t* ring = dyn + gb + sub * depth * rb;
  const int64_t first = (int64_t)blockIdx.x * RB + sub, step = (int64_t)gridDim.x * RB;
  const XT* const x0 = static_cast<const XT*>(a.x);
  const DT* const d0 = static_cast<const DT*>(a.dy);
  const int ax = EDGE ? vec_offset<XT, 16 / sizeof(XT)>(x0 + first * a.x_ld) : 0;
  const int ad = EDGE ? vec_offset<DT, 16 / sizeof(DT)>(d0 + first * a.dy_ld) : 0;
  const int o = ax & (V - 1);
  auto issue = [&](int64_t k, int slot) {  // row k of this group into a slot
    const XT* x = x0 + (first + k * step) * a.x_ld;
    const DT* d = d0 + (first + k * step) * a.dy_ld;
    uint8_t* to = ring + slot * rb;
    if constexpr (EDGE) {
      const Hull hx = row_hull(to, x, cols, x0, x0 + (a.rows - 1) * a.x_ld + a.cols);
      const Hull hd = row_hull(to + xb, d, cols, d0, d0 + (a.rows - 1) * a.dy_ld + a.cols);
      mbar_arrive_expect_tx(&bars[sub][slot], hx.n * (int)sizeof(XT) + hd.n * (int)sizeof(DT));
      load_hull(to, x, hx, &bars[sub][slot]);
      load_hull(to + xb, d, hd, &bars[sub][slot]);
    } else {
      mbar_arrive_expect_tx(&bars[sub][slot], rb);
      bulk_load(to, x, xb, &bars[sub][slot]);
      bulk_load(to + xb, d, db, &bars[sub][slot]);
    }
  };
  if (threadIdx.x == 0) {
    for (int g = 0; g < RB; ++g)
      for (int d = 0; d < depth; ++d) mbar_init(&bars[g][d], 1);
    abort_flag = 0;
    fence_barrier_init();
  }
  __syncthreads();
  // rows of this group; the block runs as many trips as its first group has
  const int64_t mine = first < a.rows ? (a.rows - first + step - 1) / step : 0;
  const int64_t first0 = (int64_t)blockIdx.x * RB;
  const int64_t trips = first0 < a.rows ? (a.rows - first0 + step - 1) / step : 0;
  griddep_wait();
  if (t == 0) {
    for (int k = 0; k < depth && k < mine; ++k) issue(k, k);
    asked[sub] = (int)mine;
  }
  f2 ga[kReread ? 1 : NE / 2];
  if constexpr (kReread) {
    for (int k = threadIdx.x; k < gb / 4; k += kBlock) {
      const int c = k - o;
      gs[k] = EDGE && (c < 0 || c >= cols) ? 0.0f
              : a.param_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(a.gamma)[c])
                             : static_cast<const float*>(a.gamma)[c];
    }
    __syncthreads();
  } else {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = (i * TR + t) * V - o;
      if constexpr (EDGE)
        load_param_edge<V>(a.gamma, a.param_bf16, c, cols, ga + i * H);
      else if (c < cols)
        load_param_pairs<V>(a.gamma, a.param_bf16, c, ga + i * H);
    }
  }
  const uint32_t ends = EDGE ? row_ends<V, TR, NC>(t, o, cols) : 0u;
  const float inv_n = 1.0f / (float)cols;
  f2 sg[NE / 2], sb[NE / 2];
#pragma unroll
  for (int k = 0; k < NE / 2; ++k) sg[k] = sb[k] = 0;
  float mean = 0.0f, rstd = 0.0f;
  if (mine > 0) {
    mean = a.mean[first];
    rstd = a.rstd[first];
  }
  int slot = 0, prev = 0;
  uint32_t phase = 0;
  for (int64_t k = 0; k < trips; ++k) {
    const bool ok = k < mine;
    const int64_t row = first + k * step;
    const XT* const sx = reinterpret_cast<const XT*>(ring + slot * rb) + ax;
    const DT* const sd = reinterpret_cast<const DT*>(ring + slot * rb + xb) + ad;
    auto get = [&](int i, int c, f2* x, f2* d) {
      load_pairs<XT, V>(sx + c, x);
      load_pairs<DT, V>(sd + c, d);
      if (EDGE && (ends >> i & 1)) {
        keep_pairs<V>(x, -c, cols - c);
        keep_pairs<V>(d, -c, cols - c);
      }
    };
    float mean2 = 0.0f, rstd2 = 0.0f;  // of the group's next row
    if (k + 1 < mine) {
      mean2 = a.mean[row + step];
      rstd2 = a.rstd[row + step];
    }
    // (a wait that gives up is counted; the loop runs on so that every
    // barrier is met)
    if (ok) mbar_wait(&bars[sub][slot], phase, &abort_flag);
    const f2 nm = dup2(-mean), r2 = dup2(rstd);
    f2 h[kReread ? 1 : NE / 2], g[kReread ? 1 : NE / 2];
    f2 s1 = 0, s2 = 0;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = (i * TR + t) * V - o;
      if (ok && c < cols) {
        f2 x[H], d[H], gm[H];
        get(i, c, x, d);
        if constexpr (kReread) load_pairs<float, V>(gs + o + c, gm);
#pragma unroll
        for (int j = 0; j < H; ++j) {
          const int e = i * H + j;
          const f2 hh = mul2(add2(x[j], nm), r2);
          const f2 gg = mul2(d[j], kReread ? gm[j] : ga[kReread ? 0 : e]);
          s1 = add2(s1, gg);
          s2 = fma2(gg, hh, s2);
          sg[e] = fma2(d[j], hh, sg[e]);
          sb[e] = add2(sb[e], d[j]);
          if constexpr (!kReread) {
            h[e] = hh;
            g[e] = gg;
          }
        }
      }
    }
    const float2 s = ring_sum2<TR>(sum2(s1), sum2(s2), red[k & 1]);
    // every thread of the group is past the previous row: its slot is free
    if (t == 0 && k > 0 && k - 1 + depth < mine) {
      if (!abort_flag)
        issue(k - 1 + depth, prev);
      else
        asked[sub] = min(asked[sub], (int)k - 1 + depth);
    }
    const f2 c1 = dup2(-s.x * inv_n), c2 = dup2(-s.y * inv_n);
    if (ok) {
      XT* dx = static_cast<XT*>(a.dx) + row * a.dx_ld;
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int c = (i * TR + t) * V - o;
        if (c < cols) {
          f2 u[H];
          if constexpr (kReread) {
            f2 x[H], d[H], gm[H];
            get(i, c, x, d);
            load_pairs<float, V>(gs + o + c, gm);
#pragma unroll
            for (int j = 0; j < H; ++j)
              u[j] = mul2(fma2(mul2(add2(x[j], nm), r2), c2, add2(mul2(d[j], gm[j]), c1)), r2);
          } else {
#pragma unroll
            for (int j = 0; j < H; ++j)
              u[j] = mul2(fma2(h[i * H + j], c2, add2(g[i * H + j], c1)), r2);
          }
          if (EDGE && (ends >> i & 1))
            store_edge<XT, V>(dx, c, cols, u);
          else
            store_pairs<XT, V>(dx + c, u);
        }
      }
    }
    mean = mean2;
    rstd = rstd2;
    prev = slot;
    if (++slot == depth) {
      slot = 0;
      phase ^= 1u;
    }
  }
  griddep_launch_dependents();  // ln_bwd_sum_kernel may take its place; it waits for the sums
  if constexpr (TR <= 32) __syncthreads();  // the waits of every group are over
  if (abort_flag) {
    if (t == 0) ring_drain(bars[sub], asked[sub], depth);
    if (threadIdx.x == 0) atomicAdd(timeouts, 1);
  }
  float* out = a.partial + (int64_t)blockIdx.x * 2 * a.cols;
  if constexpr (RB == 1) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = (i * TR + t) * V - o;
      if constexpr (EDGE) {
        store_edge<float, V>(out, c, cols, sg + i * H);
        store_edge<float, V>(out + cols, c, cols, sb + i * H);
      } else if (c < cols) {
#pragma unroll
        for (int j = 0; j < H; ++j) {
          const float2 u = unpack2(sg[i * H + j]), w = unpack2(sb[i * H + j]);
          *reinterpret_cast<float2*>(out + c + 2 * j) = u;
          *reinterpret_cast<float2*>(out + cols + c + 2 * j) = w;
        }
      }
    }
  } else {
    // the block's row groups, added in order; the ring has been read
    float* acc = reinterpret_cast<float*>(dyn);
#pragma unroll
    for (int pass = 0; pass < 2; ++pass) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int c = (i * TR + t) * V - o;
        float* to = acc + sub * TR * NE;
        if constexpr (EDGE)
          store_edge<float, V>(to, c, cols, (pass ? sb : sg) + i * H);
        else
#pragma unroll
          for (int j = 0; j < H; ++j)
            *reinterpret_cast<float2*>(to + c + 2 * j) = unpack2(pass ? sb[i * H + j] : sg[i * H + j]);
      }
      __syncthreads();
      for (int c = threadIdx.x; c < cols; c += kBlock) {
        float v = 0.0f;
#pragma unroll
        for (int r = 0; r < RB; ++r) v += acc[r * TR * NE + c];
        out[pass * cols + c] = v;
      }
    }
  }
}

// Rows too wide for the registers: the column sums first (dx may overwrite dy
// or x), then dx row by row.
template <typename XT, typename DT>
__global__ void __launch_bounds__(128) ln_bwd_wide_cols_kernel(const LnBwd a, int64_t chunk) {
  griddep_wait();
  griddep_launch_dependents();
  const int64_t c = (int64_t)blockIdx.x * 128 + threadIdx.x;
  if (c >= a.cols) return;
  const int64_t r0 = (int64_t)blockIdx.y * chunk, r1 = min(a.rows, r0 + chunk);
  const XT* x = static_cast<const XT*>(a.x) + c;
  const DT* dy = static_cast<const DT*>(a.dy) + c;
  float sg = 0.0f, sb = 0.0f;
  for (int64_t r = r0; r < r1; ++r) {
    const float d = to_f32(dy[r * a.dy_ld]);
    sg += d * ((to_f32(x[r * a.x_ld]) - a.mean[r]) * a.rstd[r]);
    sb += d;
  }
  float* out = a.partial + (int64_t)blockIdx.y * 2 * a.cols;
  out[c] = sg;
  out[a.cols + c] = sb;
}

template <typename XT, typename DT>
__global__ void __launch_bounds__(512) ln_bwd_wide_rows_kernel(const LnBwd a) {
  __shared__ float2 red[32];
  griddep_wait();
  griddep_launch_dependents();
  const int64_t row = blockIdx.x;
  const XT* x = static_cast<const XT*>(a.x) + row * a.x_ld;
  const DT* dy = static_cast<const DT*>(a.dy) + row * a.dy_ld;
  XT* dx = static_cast<XT*>(a.dx) + row * a.dx_ld;
  const float mean = a.mean[row], rstd = a.rstd[row];
  const float inv_n = 1.0f / (float)a.cols;
  float2 s = make_float2(0.0f, 0.0f);
  for (int64_t c = threadIdx.x; c < a.cols; c += 512) {
    float ga[1];
    load_param<1>(a.gamma, a.param_bf16, c, ga);
    const float g = to_f32(dy[c]) * ga[0];
    s.x += g;
    s.y += g * ((to_f32(x[c]) - mean) * rstd);
  }
  s = row_sum<512>(s, red);
  const float c1 = s.x * inv_n, c2 = s.y * inv_n;
  for (int64_t c = threadIdx.x; c < a.cols; c += 512) {
    float ga[1];
    load_param<1>(a.gamma, a.param_bf16, c, ga);
    const float g = to_f32(dy[c]) * ga[0];
    const float h = (to_f32(x[c]) - mean) * rstd;
    from_f32(dx[c], rstd * (g - c1 - h * c2));
  }
}

// dgamma and dbeta from the blocks' sums: 32 columns a block, 32 threads a
// column, each adding every 32nd partial in order (their loads are all in
// flight at once), the 32 added in a fixed tree. Launched as a programmatic
// dependent, so its start overlaps the backward kernel's end.
struct LnSum {
  const float* partial;
  void* dgamma;
  void* dbeta;
  int64_t cols;
  int parts;
  int grad_bf16;
  int accumulate;
};

__global__ void __launch_bounds__(1024) ln_bwd_sum_kernel(const LnSum a) {
  __shared__ float red[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t col = (int64_t)blockIdx.x * 32 + tx;
  griddep_wait();
  float v = 0.0f;
  if (col < a.cols) {
    const float* p = a.partial + (int64_t)blockIdx.y * a.cols + col;
#pragma unroll 10
    for (int k = ty; k < a.parts; k += 32) v += p[(int64_t)k * 2 * a.cols];
  }
  red[ty][tx] = v;
  __syncthreads();
  // warp ty now takes column ty of the block: lane l holds partial sum l
  v = red[tx][ty];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int64_t c = (int64_t)blockIdx.x * 32 + ty;
  if (tx != 0 || c >= a.cols) return;
  void* out = blockIdx.y ? a.dbeta : a.dgamma;
  if (a.grad_bf16) {
    __nv_bfloat16* o = static_cast<__nv_bfloat16*>(out) + c;
    *o = __float2bfloat16_rn(a.accumulate ? __bfloat162float(*o) + v : v);
  } else {
    float* o = static_cast<float*>(out) + c;
    *o = a.accumulate ? *o + v : v;
  }
}

// ------------------------------------------------------------------ dispatch
// How a row is spread: the threads of a row by its width, so that a thread holds 8
// to 32 elements of it.
constexpr int64_t kFwdMaxCols = 16384;
constexpr int64_t kBwdMaxCols = 8192;    // rows in registers
constexpr int64_t kRingMaxCols = 16384;  // rows through shared memory

template <typename XT, typename YT, int TR, int NE>
void fwd_scalar(const LnFwd& a, cudaStream_t s) {
  constexpr int kBlock = TR <= 32 ? 128 : TR, RB = kBlock / TR;
  launch_dependent(ln_fwd_kernel<XT, YT, TR, NE>, dim3((unsigned)((a.rows + RB - 1) / RB)), kBlock,
                   0, s, a);
}

template <typename XT, typename YT, int TR, int NE>
void fwd_rows(const LnFwd& a, cudaStream_t s) {
  constexpr int64_t kRows = ln_rows_block(TR) / TR;
  launch_dependent(ln_fwd_rows_kernel<XT, YT, TR, NE>,
                   dim3((unsigned)((a.rows + kRows - 1) / kRows)), ln_rows_block(TR), 0, s, a);
}

// Shared memory above 48 KB for a kernel, once per device (`done`: the devices
// that have it).
template <typename K>
int raise_smem(K kernel, int device, std::mutex& mu, uint64_t& done) {
  std::lock_guard<std::mutex> lock(mu);
  if (device < 64 && (done >> device) & 1u) return MMN_OK;
  MMN_CUDA_TRY(
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024));
  if (device < 64) done |= uint64_t(1) << device;
  return MMN_OK;
}

template <typename XT, typename YT>
void fwd_width(const LnFwd& a, cudaStream_t s) {
  if (a.cols <= 64)
    fwd_rows<XT, YT, 8, 8>(a, s);
  else if (a.cols <= 256)
    fwd_rows<XT, YT, 32, 8>(a, s);
  else if (a.cols <= 512)
    fwd_rows<XT, YT, 32, 16>(a, s);
  else if (a.cols <= 1024)
    fwd_rows<XT, YT, 128, 8>(a, s);
  else if (a.cols <= 2048)
    fwd_rows<XT, YT, 128, 16>(a, s);
  else if (a.cols <= 4096)
    fwd_rows<XT, YT, 256, 16>(a, s);
  else if (a.cols <= 8192)
    fwd_rows<XT, YT, 512, 16>(a, s);
  else
    fwd_rows<XT, YT, 1024, 16>(a, s);
}

// Blocks of a ring kernel, RB rows at a time. For rows that start anywhere the rows of
// a group lie a multiple of eight apart.
int ring_grid(int64_t rows, int rb, int64_t most, bool edge) {
  int64_t grid = std::min((rows + rb - 1) / rb, most);
  if (edge && grid * rb < rows) grid -= grid % (8 / std::min(rb, 8));
  return (int)grid;
}

// Whether the rows of two matrices start alike, counted modulo v elements.
bool rows_agree(const void* p, int64_t p_ld, size_t p_es, const void* q, int64_t q_ld, size_t q_es,
                int v) {
  const uintptr_t d = reinterpret_cast<uintptr_t>(p) / p_es - reinterpret_cast<uintptr_t>(q) / q_es;
  return d % v == 0 && (p_ld - q_ld) % v == 0;
}

template <typename XT, typename YT, int TR, int NE, bool EDGE>
int ring_fwd_launch(const LnFwd& a, int sms, int device, cudaStream_t s) {
  constexpr int RB = ln_ring_block(TR) / TR, kBlocks = ln_ring_blocks(TR, NE);
  static std::mutex mu;
  static uint64_t done = 0;
  auto* kernel = ln_fwd_ring_kernel<XT, YT, TR, NE, EDGE>;
  int* timeouts = nullptr;
  int rc;
  if ((rc = raise_smem(kernel, device, mu, done)) != MMN_OK) return rc;
  if ((rc = kernel_timeout_word(device, &timeouts)) != MMN_OK) return rc;
  const int64_t row = EDGE ? hull_bytes(a.cols, sizeof(XT)) : a.cols * (int64_t)sizeof(XT);
  // more rows in flight cost bandwidth (16384 x 4096: 43.6 us with 2, 45.6 with 3,
  // 47.2 with 4)
  const int depth = (int)std::min<int64_t>(kFwdRing, (224 * 1024 / kBlocks - 4096) / (row * RB));
  const int64_t grid = ring_grid(a.rows, RB, (int64_t)sms * kBlocks, EDGE);
  launch_dependent(kernel, dim3((unsigned)grid), ln_ring_block(TR), depth * row * RB, s, a, depth,
                   timeouts);
  return MMN_OK;
}

// bf16 rows in whole vectors, many of them.
template <typename XT, typename YT>
int ring_whole(const LnFwd& a, int sms, int device, cudaStream_t s) {
  if (a.cols <= 512) return ring_fwd_launch<XT, YT, 32, 16, false>(a, sms, device, s);
  if (a.cols <= 1024) return ring_fwd_launch<XT, YT, 32, 32, false>(a, sms, device, s);
  if (a.cols <= 2048) return ring_fwd_launch<XT, YT, 64, 32, false>(a, sms, device, s);
  if (a.cols <= 4096) return ring_fwd_launch<XT, YT, 128, 32, false>(a, sms, device, s);
  if (a.cols <= 8192) return ring_fwd_launch<XT, YT, 256, 32, false>(a, sms, device, s);
  return ring_fwd_launch<XT, YT, 512, 32, false>(a, sms, device, s);
}

// Rows that start anywhere; w: the columns and what the start may add.
template <typename XT, typename YT>
int ring_edge(const LnFwd& a, int64_t w, int sms, int device, cudaStream_t s) {
  if (w <= 2048) return ring_fwd_launch<XT, YT, 128, 16, true>(a, sms, device, s);
  if (w <= 4096) return ring_fwd_launch<XT, YT, 256, 16, true>(a, sms, device, s);
  if (w <= 8192) return ring_fwd_launch<XT, YT, 256, 32, true>(a, sms, device, s);
  return ring_fwd_launch<XT, YT, 512, 32, true>(a, sms, device, s);
}

// vec, vec8: rows in whole vectors of four or eight elements; alike: x and y start alike.
template <typename XT, typename YT>
int fwd_types(const LnFwd& a, bool vec, bool vec8, bool alike, int sms, int device, cudaStream_t s) {
  // bf16 rows: with fewer a block of its own per row is quicker
  if constexpr (sizeof(XT) == 2)
    if (vec8 && a.cols > 64 && a.cols <= kFwdMaxCols && a.rows >= 8 * (int64_t)sms)
      return ring_whole<XT, YT>(a, sms, device, s);
  // Rows that start anywhere: vectors with care at the ends, or an element at a time
  // (launches one behind the other). 16384 x 4057 63.4 us and 132, fp32 95.1 and 115; 20000 x
  // 2037 44.8 and 79.0, fp32 60.5 and 68.0; 8 x 4001 2.8 and 5.4. Up to 1024 columns the
  // ends outweigh the rest (32768 x 1013 59.9 and 51.5, fp32 63.9 and 49.8; 16384 x 777 32.2
  // and 22.1, fp32 33.7 and 22.6; 1200 x 1013 6.2 and 4.0; 300 x 600 equal), and so they do
  // for fp32 rows that the start pushes into the next class (16384 x 4095 124 and 116; bf16
  // 102 and 132).
  if (const int64_t w = a.cols + (sizeof(XT) == 2 && sizeof(YT) == 2 ? 7 : 3);
      alike && !vec && a.cols > 1024 && w <= kFwdMaxCols) {
    int64_t cls = 2048;
    while (cls < a.cols) cls *= 2;
    if (sizeof(XT) == 2 || w <= cls) return ring_edge<XT, YT>(a, w, sms, device, s);
  }
  if (a.cols > kFwdMaxCols)
    launch_dependent(ln_fwd_wide_kernel<XT, YT>, dim3((unsigned)a.rows), 512, 0, s, a);
  else if (vec)
    fwd_width<XT, YT>(a, s);
  else if (a.cols <= 64)
    fwd_scalar<XT, YT, 8, 8>(a, s);
  else if (a.cols <= 256)
    fwd_scalar<XT, YT, 32, 8>(a, s);
  else if (a.cols <= 512)
    fwd_scalar<XT, YT, 32, 16>(a, s);
  else if (a.cols <= 1024)
    fwd_scalar<XT, YT, 128, 8>(a, s);
  else if (a.cols <= 2048)
    fwd_scalar<XT, YT, 128, 16>(a, s);
  else if (a.cols <= 4096)
    fwd_scalar<XT, YT, 256, 16>(a, s);
  else if (a.cols <= 8192)
    fwd_scalar<XT, YT, 512, 16>(a, s);
  else
    fwd_scalar<XT, YT, 512, 32>(a, s);
  return MMN_OK;
}

// Threads per row of the backward kernels for a width.
int bwd_tr(int64_t cols) {
  return cols <= 64 ? 8 : cols <= 256 ? 32 : cols <= 512 ? 64 : cols <= 2048 ? 128
         : cols <= 4096 ? 256 : 512;
}

// Blocks of the backward kernel (partial sums to add) for tr threads a row: one per
// row group, at most what the GPU holds at once.
int bwd_parts(int64_t rows, int tr, int sms, bool edge) {
  return ring_grid(rows, ln_bwd_block(tr) / tr, (int64_t)sms * ln_bwd_min_blocks(tr), edge);
}

// ... at most, however the rows start.
int bwd_max_parts(int64_t rows, int64_t cols, int sms) {
  return rows <= 0 || cols <= 0 ? 0 : bwd_parts(rows, bwd_tr(cols), sms, false);
}

template <typename XT, typename DT, int V, int TR, int NE>
void bwd_launch(const LnBwd& a, int parts, cudaStream_t s) {
  launch_dependent(ln_bwd_kernel<XT, DT, V, TR, NE>, dim3(parts), ln_bwd_block(TR), 0, s, a);
}

// Rows of any width up to 8192, one element at a time.
template <typename XT, typename DT>
void bwd_scalar(const LnBwd& a, int parts, cudaStream_t s) {
  switch (bwd_tr(a.cols)) {
    case 8:
      return bwd_launch<XT, DT, 1, 8, 8>(a, parts, s);
    case 32:
      return bwd_launch<XT, DT, 1, 32, 8>(a, parts, s);
    case 64:
      return bwd_launch<XT, DT, 1, 64, 8>(a, parts, s);
    case 128:
      return bwd_launch<XT, DT, 1, 128, 16>(a, parts, s);
    case 256:
      return bwd_launch<XT, DT, 1, 256, 16>(a, parts, s);
    default:
      return bwd_launch<XT, DT, 1, 512, 16>(a, parts, s);
  }
}

// Rows in flight per group with bulk copies: what an SM's 224 KB hold, shared by
// the blocks on it. w: the columns and what an uneven start adds.
template <typename XT, typename DT>
int ring_depth(int64_t cols, int64_t w, bool edge, int* smem) {
  const int tr = bwd_tr(w), rb = ln_bwd_block(tr) / tr;
  const int64_t row = edge ? hull_bytes(cols, sizeof(XT)) + hull_bytes(cols, sizeof(DT))
                           : cols * (int64_t)(sizeof(XT) + sizeof(DT));
  const int64_t gamma = w > kBwdMaxCols ? (edge ? (w + 9) / 4 * 16 : cols * 4) : 0;
  const int64_t budget = 224 * 1024 / ln_bwd_min_blocks(tr) - 4096 - gamma;
  const int depth = (int)std::min<int64_t>(kRingMax, budget / (row * rb));
  // (the closing sums of several groups use the same memory)
  const int64_t acc = rb > 1 ? (int64_t)rb * tr * 8 * 4 : 0;
  *smem = (int)std::max<int64_t>(gamma + depth * row * rb, acc);
  return depth;
}

template <typename XT, typename DT, int TR, int NE, bool EDGE>
int ring_launch(const LnBwd& a, int parts, int depth, int smem, int* timeouts, int device,
                cudaStream_t s) {
  constexpr int V = sizeof(XT) == 2 && sizeof(DT) == 2 ? 8 : 4;
  static std::mutex mu;
  static uint64_t done = 0;
  auto* kernel = ln_bwd_ring_kernel<XT, DT, V, TR, NE, EDGE>;
  const int rc = raise_smem(kernel, device, mu, done);
  if (rc != MMN_OK) return rc;
  launch_dependent(kernel, dim3(parts), ln_bwd_block(TR), smem, s, a, depth, timeouts);
  return MMN_OK;
}

template <typename XT, typename DT, bool EDGE>
int ring_bwd(const LnBwd& a, int64_t w, int parts, int depth, int smem, int device, cudaStream_t s) {
  int* st = nullptr;
  const int rc = kernel_timeout_word(device, &st);
  if (rc != MMN_OK) return rc;
  if constexpr (!EDGE) {
    if (w <= 256) return ring_launch<XT, DT, 32, 8, false>(a, parts, depth, smem, st, device, s);
    if (w <= 512) return ring_launch<XT, DT, 64, 8, false>(a, parts, depth, smem, st, device, s);
  }
  if (w <= 1024) return ring_launch<XT, DT, 128, 8, EDGE>(a, parts, depth, smem, st, device, s);
  if (w <= 2048) return ring_launch<XT, DT, 128, 16, EDGE>(a, parts, depth, smem, st, device, s);
  if (w <= 4096) return ring_launch<XT, DT, 256, 16, EDGE>(a, parts, depth, smem, st, device, s);
  if (w <= 8192) return ring_launch<XT, DT, 512, 16, EDGE>(a, parts, depth, smem, st, device, s);
  return ring_launch<XT, DT, 512, 32, EDGE>(a, parts, depth, smem, st, device, s);
}

// vec: rows in whole vectors; ring: ... of 16 bytes; alike: the rows of all three
// matrices start alike. parts: the blocks launched.
template <typename XT, typename DT>
int bwd_types(const LnBwd& a, int* parts, bool vec, bool ring, bool alike, int sms, int device,
              cudaStream_t s) {
  constexpr int V = sizeof(XT) == 2 && sizeof(DT) == 2 ? 8 : 4;
  const int64_t w = a.cols + (ring ? 0 : V - 1);  // ... and what an uneven start may add
  // Rows that start anywhere: vectors with care at the ends, or an element at a time.
  // 16384 x 4057 106 us and 158, fp32 140 and 184; 32768 x 1013 75.6 and 109, fp32 69.9 and
  // 118. Element-wise where the start pushes the row into the next class (16384 x 4095
  // 205 and 158), for few columns (32768 x 501 47.9 and 36.9) and few bf16 rows (600 x
  // 1013 13.8 and 9.6; fp32 8.7 and 10.1).
  const bool edge = alike && a.cols > 512 && bwd_tr(w) == bwd_tr(a.cols) &&
                    (V == 4 || a.rows >= 8 * (int64_t)sms);
  if (a.cols > 64 && (ring || edge) && w <= kRingMaxCols) {
    int smem = 0;
    const int depth = ring_depth<XT, DT>(a.cols, w, !ring, &smem);
    if (depth >= 2) {
      *parts = bwd_parts(a.rows, bwd_tr(w), sms, !ring);
      return ring ? ring_bwd<XT, DT, false>(a, w, *parts, depth, smem, device, s)
                  : ring_bwd<XT, DT, true>(a, w, *parts, depth, smem, device, s);
    }
  }
  *parts = bwd_parts(a.rows, bwd_tr(a.cols), sms, false);
  if (a.cols > kBwdMaxCols) {
    const int64_t chunk = (a.rows + *parts - 1) / *parts;
    launch_dependent(ln_bwd_wide_cols_kernel<XT, DT>,
                     dim3((unsigned)((a.cols + 127) / 128), (unsigned)*parts), 128, 0, s, a, chunk);
    launch_dependent(ln_bwd_wide_rows_kernel<XT, DT>, dim3((unsigned)a.rows), 512, 0, s, a);
  } else if (vec && a.cols <= 64) {
    bwd_launch<XT, DT, V, 8, 8>(a, *parts, s);
  } else {
    bwd_scalar<XT, DT>(a, *parts, s);
  }
  return MMN_OK;
}

bool bad_dtype(int d) { return d != MMN_DTYPE_F32 && d != MMN_DTYPE_BF16; }
size_t esize(int d) { return d == MMN_DTYPE_BF16 ? 2 : 4; }

int check_extent(int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 0) return fail(MMN_E_INVALID, "negative dimension");
  if (rows > (int64_t(1) << 31) - 1 || cols > (int64_t(1) << 31) - 1)
    return fail(MMN_E_SHAPE, "rows and cols must lie below 2^31");
  return MMN_OK;
}

}  // namespace

}  // namespace mmn

using namespace mmn;

extern "C" int mmn_layer_norm(const void* x, int64_t x_ld, int x_dtype, const void* gamma,
                              const void* beta, int param_dtype, float eps, int64_t rows,
                              int64_t cols, void* y, int64_t y_ld, int y_dtype, float* mean,
                              float* rstd, int device, void* stream) {
  if (bad_dtype(x_dtype) || bad_dtype(y_dtype) || bad_dtype(param_dtype))
    return fail(MMN_E_INVALID, "unknown dtype");
  if (!(eps >= 0.0f) || std::isinf(eps)) return fail(MMN_E_INVALID, "eps must be finite and >= 0");
  int rc, sms = 0;
  if ((rc = check_extent(rows, cols)) != MMN_OK) return rc;
  const bool empty = rows == 0 || cols == 0;
  if (!empty && (!x || !gamma || !beta || !y)) return fail(MMN_E_INVALID, "null pointer");
  if (rows > 1 && (x_ld < cols || y_ld < cols))
    return fail(MMN_E_INVALID, "a row pitch is smaller than cols");
  if (!empty) {
    const MatrixIn mx{x, rows > 1 ? x_ld : cols, rows, cols, esize(x_dtype)};
    const MatrixIn my{y, rows > 1 ? y_ld : cols, rows, cols, esize(y_dtype)};
    const MatrixIn mm{mean, rows, mean ? 1 : 0, rows, 4}, mr{rstd, rows, rstd ? 1 : 0, rows, 4};
    const MatrixIn mg{gamma, cols, 1, cols, esize(param_dtype)};
    const MatrixIn mb{beta, cols, 1, cols, esize(param_dtype)};
    if ((rc = check_out_overlap(my, "y", mx)) != MMN_OK) return rc;
    if (matrices_overlap(my, mg) || matrices_overlap(my, mb))
      return fail(MMN_E_INVALID, "y overlaps gamma or beta");
    if (matrices_overlap(mm, mr)) return fail(MMN_E_INVALID, "mean and rstd overlap");
    for (const MatrixIn& m : {mx, my, mg, mb})
      if (matrices_overlap(mm, m) || matrices_overlap(mr, m))
        return fail(MMN_E_INVALID, "mean or rstd overlaps another buffer");
  }
  if ((rc = percall_device(device, &sms)) != MMN_OK) return rc;
  if (empty) return MMN_OK;
  DeviceGuard guard(device);
  const struct { const void* p; int dt; const char* n; } ptrs[] = {
      {x, x_dtype, "x"}, {gamma, param_dtype, "gamma"}, {beta, param_dtype, "beta"},
      {y, y_dtype, "y"}, {mean, MMN_DTYPE_F32, "mean"}, {rstd, MMN_DTYPE_F32, "rstd"}};
  for (const auto& q : ptrs)
    if (q.p && (rc = check_device_elems(q.p, esize(q.dt), device, q.n)) != MMN_OK) return rc;
  LnFwd a{x, gamma, beta, y, mean, rstd, rows > 1 ? x_ld : cols, rows > 1 ? y_ld : cols, rows, cols,
          eps, param_dtype == MMN_DTYPE_BF16};
  const int v = 4;
  const bool vec = cols % v == 0 && vec_rows(x, a.x_ld, esize(x_dtype), v) &&
                   vec_rows(y, a.y_ld, esize(y_dtype), v) &&
                   vec_rows(gamma, 0, esize(param_dtype), v) &&
                   vec_rows(beta, 0, esize(param_dtype), v);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool xb = x_dtype == MMN_DTYPE_BF16, yb = y_dtype == MMN_DTYPE_BF16;
  const bool vec8 = vec && cols % 8 == 0 && vec_rows(x, a.x_ld, esize(x_dtype), 8) &&
                    vec_rows(y, a.y_ld, esize(y_dtype), 8) &&
                    vec_rows(gamma, 0, esize(param_dtype), 8) &&
                    vec_rows(beta, 0, esize(param_dtype), 8);
  const bool alike = rows_agree(x, a.x_ld, esize(x_dtype), y, a.y_ld, esize(y_dtype),
                                xb && yb ? 8 : 4);
  if (xb && yb)
    rc = fwd_types<__nv_bfloat16, __nv_bfloat16>(a, vec, vec8, alike, sms, device, s);
  else if (xb)
    rc = fwd_types<__nv_bfloat16, float>(a, vec, vec8, alike, sms, device, s);
  else if (yb)
    rc = fwd_types<float, __nv_bfloat16>(a, vec, vec8, alike, sms, device, s);
  else
    rc = fwd_types<float, float>(a, vec, vec8, alike, sms, device, s);
  if (rc != MMN_OK) return rc;
  MMN_CUDA_TRY(cudaGetLastError());
  return MMN_OK;
}

extern "C" int mmn_layer_norm_backward_workspace(int64_t rows, int64_t cols, int device,
                                                 int64_t* bytes) {
  if (!bytes) return fail(MMN_E_INVALID, "null pointer");
  int rc, sms = 0;
  if ((rc = check_extent(rows, cols)) != MMN_OK) return rc;
  if ((rc = percall_device(device, &sms)) != MMN_OK) return rc;
  *bytes = (int64_t)bwd_max_parts(rows, cols, sms) * 2 * cols * 4;
  return MMN_OK;
}

extern "C" int mmn_layer_norm_backward(const void* dy, int64_t dy_ld, int dy_dtype, const void* x,
                                       int64_t x_ld, int x_dtype, const void* gamma,
                                       int param_dtype, const float* mean, const float* rstd,
                                       int64_t rows, int64_t cols, void* dx, int64_t dx_ld,
                                       void* dgamma, void* dbeta, int grad_dtype, int accumulate,
                                       void* workspace, int64_t workspace_bytes, int device,
                                       void* stream) {
  if (bad_dtype(x_dtype) || bad_dtype(dy_dtype) || bad_dtype(param_dtype) || bad_dtype(grad_dtype))
    return fail(MMN_E_INVALID, "unknown dtype");
  int rc, sms = 0;
  if ((rc = check_extent(rows, cols)) != MMN_OK) return rc;
  const bool empty = rows == 0 || cols == 0;
  if (cols > 0 && (!dgamma || !dbeta)) return fail(MMN_E_INVALID, "null pointer");
  if (!empty && (!dy || !x || !gamma || !mean || !rstd || !dx || !workspace))
    return fail(MMN_E_INVALID, "null pointer");
  if (rows > 1 && (x_ld < cols || dy_ld < cols || dx_ld < cols))
    return fail(MMN_E_INVALID, "a row pitch is smaller than cols");
  const MatrixIn mg{dgamma, cols, 1, cols, esize(grad_dtype)};
  const MatrixIn mb{dbeta, cols, 1, cols, esize(grad_dtype)};
  if (matrices_overlap(mg, mb)) return fail(MMN_E_INVALID, "dgamma and dbeta overlap");
  if (!empty) {
    const MatrixIn mdx{dx, rows > 1 ? dx_ld : cols, rows, cols, esize(x_dtype)};
    const MatrixIn mx{x, rows > 1 ? x_ld : cols, rows, cols, esize(x_dtype)};
    const MatrixIn mdy{dy, rows > 1 ? dy_ld : cols, rows, cols, esize(dy_dtype)};
    const MatrixIn small[] = {{gamma, cols, 1, cols, esize(param_dtype)}, {mean, rows, 1, rows, 4},
                              {rstd, rows, 1, rows, 4}};
    if ((rc = check_out_overlap(mdx, "dx", mx)) != MMN_OK ||
        (rc = check_out_overlap(mdx, "dx", mdy)) != MMN_OK)
      return rc;
    for (const MatrixIn& m : small)
      if (matrices_overlap(mdx, m)) return fail(MMN_E_INVALID, "dx overlaps gamma, mean or rstd");
    for (const MatrixIn& m : {mdx, mx, mdy, small[0], small[1], small[2]})
      if (matrices_overlap(mg, m) || matrices_overlap(mb, m))
        return fail(MMN_E_INVALID, "dgamma or dbeta overlaps another buffer");
  }
  if (!empty && reinterpret_cast<uintptr_t>(workspace) % 16)
    return fail(MMN_E_INVALID, "workspace is not 16-byte aligned");
  if ((rc = percall_device(device, &sms)) != MMN_OK) return rc;
  int parts = bwd_max_parts(rows, cols, sms);
  if (workspace_bytes < (int64_t)parts * 2 * cols * 4)
    return fail(MMN_E_INVALID, "workspace is smaller than mmn_layer_norm_backward_workspace gives");
  if (cols == 0) return MMN_OK;
  if (!empty) {
    const MatrixIn mw{workspace, 2 * cols, parts, 2 * cols, 4};
    const MatrixIn others[] = {mg, mb, {dx, rows > 1 ? dx_ld : cols, rows, cols, esize(x_dtype)},
                               {x, rows > 1 ? x_ld : cols, rows, cols, esize(x_dtype)},
                               {dy, rows > 1 ? dy_ld : cols, rows, cols, esize(dy_dtype)},
                               {gamma, cols, 1, cols, esize(param_dtype)},
                               {mean, rows, 1, rows, 4}, {rstd, rows, 1, rows, 4}};
    for (const MatrixIn& m : others)
      if (matrices_overlap(mw, m)) return fail(MMN_E_INVALID, "workspace overlaps another buffer");
  }
  DeviceGuard guard(device);
  const struct { const void* p; int dt; const char* n; } ptrs[] = {
      {dy, dy_dtype, "dy"}, {x, x_dtype, "x"}, {gamma, param_dtype, "gamma"},
      {mean, MMN_DTYPE_F32, "mean"}, {rstd, MMN_DTYPE_F32, "rstd"}, {dx, x_dtype, "dx"},
      {workspace, MMN_DTYPE_F32, "workspace"}, {dgamma, grad_dtype, "dgamma"},
      {dbeta, grad_dtype, "dbeta"}};
  for (const auto& q : ptrs)
    if (q.p && (rc = check_device_elems(q.p, esize(q.dt), device, q.n)) != MMN_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (!empty) {
    LnBwd a{dy, x, gamma, mean, rstd, dx, static_cast<float*>(workspace),
            rows > 1 ? dy_ld : cols, rows > 1 ? x_ld : cols, rows > 1 ? dx_ld : cols, rows, cols,
            param_dtype == MMN_DTYPE_BF16};
    const int v = x_dtype == MMN_DTYPE_BF16 && dy_dtype == MMN_DTYPE_BF16 ? 8 : 4;
    const bool vec = cols % v == 0 && vec_rows(x, a.x_ld, esize(x_dtype), v) &&
                     vec_rows(dy, a.dy_ld, esize(dy_dtype), v) &&
                     vec_rows(dx, a.dx_ld, esize(x_dtype), v) &&
                     vec_rows(gamma, 0, esize(param_dtype), v);
    // dx in place of an input that a later row still reads is no hazard: a row is
    // read before its dx is written, and no other row is touched
    const bool ring = vec && (cols * esize(x_dtype)) % 16 == 0 && (cols * esize(dy_dtype)) % 16 == 0 &&
                      vec_rows(x, a.x_ld, esize(x_dtype), 16) &&
                      vec_rows(dy, a.dy_ld, esize(dy_dtype), 16);
    const bool alike =
        rows_agree(x, a.x_ld, esize(x_dtype), dy, a.dy_ld, esize(dy_dtype), v) &&
        rows_agree(x, a.x_ld, esize(x_dtype), dx, a.dx_ld, esize(x_dtype), v);
    const bool xb = x_dtype == MMN_DTYPE_BF16, db = dy_dtype == MMN_DTYPE_BF16;
    if (xb && db)
      rc = bwd_types<__nv_bfloat16, __nv_bfloat16>(a, &parts, vec, ring, alike, sms, device, s);
    else if (xb)
      rc = bwd_types<__nv_bfloat16, float>(a, &parts, vec, ring, alike, sms, device, s);
    else if (db)
      rc = bwd_types<float, __nv_bfloat16>(a, &parts, vec, ring, alike, sms, device, s);
    else
      rc = bwd_types<float, float>(a, &parts, vec, ring, alike, sms, device, s);
    if (rc != MMN_OK) return rc;
    MMN_CUDA_TRY(cudaGetLastError());
  }
  if (parts == 0 && accumulate) return MMN_OK;  // no rows: the sums are zero
  LnSum su{static_cast<const float*>(workspace), dgamma, dbeta, cols, parts,
           grad_dtype == MMN_DTYPE_BF16, accumulate != 0};
  MMN_CUDA_TRY(launch_dependent(ln_bwd_sum_kernel, dim3((unsigned)((cols + 31) / 32), 2), 1024, 0, s,
                                su));
  return MMN_OK;
}
