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
// Bound by memory: a row is read once into registers, both sums of the
// variance run over the registers (the second about the mean, so that a row
// whose mean is large against its spread loses nothing), and the row is written
// once. All statistics and sums are fp32; y and dx are rounded once.
#include <cuda_bf16.h>

#include <algorithm>

#include "capi_internal.cuh"

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
// TR threads hold one row, NE elements each, in chunks of V.
template <typename XT, typename YT, int V, int TR, int NE>
__global__ void __launch_bounds__(TR <= 32 ? 128 : TR) ln_fwd_kernel(const LnFwd a) {
  constexpr int kBlock = TR <= 32 ? 128 : TR, RB = kBlock / TR, NC = NE / V;
  __shared__ float2 red[2][32];
  const int t = threadIdx.x % TR;
  const int64_t row = (int64_t)blockIdx.x * RB + threadIdx.x / TR;
  const bool ok = row < a.rows;
  const XT* x = static_cast<const XT*>(a.x) + (ok ? row : 0) * a.x_ld;
  float v[NE];
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int64_t c = (int64_t)(i * TR + t) * V;
    if (ok && c < a.cols) {
      const Vec<XT, V> u = load_vec<XT, V>(x + c);
#pragma unroll
      for (int j = 0; j < V; ++j) v[i * V + j] = to_f32(u.e[j]);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) v[i * V + j] = 0.0f;
    }
  }
  const float n = (float)a.cols;
  float s = 0.0f;
#pragma unroll
  for (int k = 0; k < NE; ++k) s += v[k];
  const float mean = row_sum<TR>(make_float2(s, 0.0f), red[0]).x / n;
  float q = 0.0f;
#pragma unroll
  for (int i = 0; i < NC; ++i)
    if ((int64_t)(i * TR + t) * V < a.cols) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = v[i * V + j] - mean;
        q += d * d;
      }
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
  for (int i = 0; i < NC; ++i) {
    const int64_t c = (int64_t)(i * TR + t) * V;
    if (c < a.cols) {
      float ga[V], be[V];
      load_param<V>(a.gamma, a.param_bf16, c, ga);
      load_param<V>(a.beta, a.param_bf16, c, be);
      Vec<YT, V> o;
#pragma unroll
      for (int j = 0; j < V; ++j)
        from_f32(o.e[j], (v[i * V + j] - mean) * rstd * ga[j] + be[j]);
      *reinterpret_cast<Vec<YT, V>*>(y + c) = o;
    }
  }
}

// Rows too wide for the registers: one block per row, read three times (the
// second and third time mostly from L1 and L2).
template <typename XT, typename YT>
__global__ void __launch_bounds__(512) ln_fwd_wide_kernel(const LnFwd a) {
  __shared__ float2 red[2][32];
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

// ------------------------------------------------------------------ backward
// Blocks walk the rows; a thread owns the same columns in every row and keeps
// their dgamma and dbeta sums in registers, so the rows are read once for both
// results. Each block writes its sums; ln_bwd_sum_kernel adds them in a fixed
// order (no atomics: the result does not depend on timing).
__host__ __device__ constexpr int ln_bwd_block(int tr) { return tr <= 32 ? 256 : tr; }
__host__ __device__ constexpr int ln_bwd_min_blocks(int tr) {
  return tr <= 32 ? 2 : tr == 128 ? 4 : tr == 256 ? 2 : 1;
}

template <typename XT, typename DT, int V, int TR, int NE>
__global__ void __launch_bounds__(ln_bwd_block(TR), ln_bwd_min_blocks(TR))
    ln_bwd_kernel(const LnBwd a) {
  constexpr int kBlock = ln_bwd_block(TR), RB = kBlock / TR, NC = NE / V;
  __shared__ float2 red[2][32];
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

// Rows too wide for the registers: the column sums first (dx may overwrite dy
// or x), then dx row by row.
template <typename XT, typename DT>
__global__ void __launch_bounds__(128) ln_bwd_wide_cols_kernel(const LnBwd a, int64_t chunk) {
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

// dgamma and dbeta from the blocks' sums: 32 columns a block, 8 threads a
// column, each adding every eighth partial in order, the eight added in order.
struct LnSum {
  const float* partial;
  void* dgamma;
  void* dbeta;
  int64_t cols;
  int parts;
  int grad_bf16;
  int accumulate;
};

__global__ void __launch_bounds__(256) ln_bwd_sum_kernel(const LnSum a) {
  __shared__ float red[8][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + tx;
  float v = 0.0f;
  if (c < a.cols) {
    const float* p = a.partial + (int64_t)blockIdx.y * a.cols + c;
#pragma unroll 4
    for (int k = ty; k < a.parts; k += 8) v += p[(int64_t)k * 2 * a.cols];
  }
  red[ty][tx] = v;
  __syncthreads();
  if (ty != 0 || c >= a.cols) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) v += red[k][tx];
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
// How a row is spread: the threads of a row by its width, so that a thread
// holds at most 32 elements forward and 16 backward (where x, dy and two sums
// per column are live).
constexpr int64_t kFwdMaxCols = 16384;
constexpr int64_t kBwdMaxCols = 8192;

template <typename XT, typename YT, int V, int TR, int NE>
void fwd_launch(const LnFwd& a, cudaStream_t s) {
  constexpr int kBlock = TR <= 32 ? 128 : TR, RB = kBlock / TR;
  ln_fwd_kernel<XT, YT, V, TR, NE><<<(unsigned)((a.rows + RB - 1) / RB), kBlock, 0, s>>>(a);
}

template <typename XT, typename YT, int V>
void fwd_width(const LnFwd& a, cudaStream_t s) {
  if (a.cols <= 64)
    fwd_launch<XT, YT, V, 8, 8>(a, s);
  else if (a.cols <= 256)
    fwd_launch<XT, YT, V, 32, 8>(a, s);
  else if (a.cols <= 1024)
    fwd_launch<XT, YT, V, 128, 8>(a, s);
  else if (a.cols <= 2048)
    fwd_launch<XT, YT, V, 128, 16>(a, s);
  else if (a.cols <= 4096)
    fwd_launch<XT, YT, V, 256, 16>(a, s);
  else if (a.cols <= 8192)
    fwd_launch<XT, YT, V, 512, 16>(a, s);
  else
    fwd_launch<XT, YT, V, 512, 32>(a, s);
}

template <typename XT, typename YT>
void fwd_types(const LnFwd& a, bool vec, cudaStream_t s) {
  constexpr int V = sizeof(XT) == 2 && sizeof(YT) == 2 ? 8 : 4;
  if (a.cols > kFwdMaxCols)
    ln_fwd_wide_kernel<XT, YT><<<(unsigned)a.rows, 512, 0, s>>>(a);
  else if (vec)
    fwd_width<XT, YT, V>(a, s);
  else
    fwd_width<XT, YT, 1>(a, s);
}

// Threads per row of the backward kernel for a width.
int bwd_tr(int64_t cols) {
  return cols <= 64 ? 8 : cols <= 512 ? 32 : cols <= 2048 ? 128 : cols <= 4096 ? 256 : 512;
}

// Blocks of the backward kernel (partial sums to add): one per row group, at
// most what the GPU holds at once. Wide rows: chunks of rows.
int bwd_parts(int64_t rows, int64_t cols, int sms) {
  if (rows <= 0 || cols <= 0) return 0;
  if (cols > kBwdMaxCols) return (int)std::min<int64_t>(rows, 64);
  const int tr = bwd_tr(cols), rb = ln_bwd_block(tr) / tr;
  return (int)std::min<int64_t>((rows + rb - 1) / rb, (int64_t)sms * ln_bwd_min_blocks(tr));
}

template <typename XT, typename DT, int V, int TR, int NE>
void bwd_launch(const LnBwd& a, int parts, cudaStream_t s) {
  ln_bwd_kernel<XT, DT, V, TR, NE><<<parts, ln_bwd_block(TR), 0, s>>>(a);
}

template <typename XT, typename DT, int V>
void bwd_width(const LnBwd& a, int parts, cudaStream_t s) {
  switch (bwd_tr(a.cols)) {
    case 8:
      return bwd_launch<XT, DT, V, 8, 8>(a, parts, s);
    case 32:
      return bwd_launch<XT, DT, V, 32, 16>(a, parts, s);
    case 128:
      return bwd_launch<XT, DT, V, 128, 16>(a, parts, s);
    case 256:
      return bwd_launch<XT, DT, V, 256, 16>(a, parts, s);
    default:
      return bwd_launch<XT, DT, V, 512, 16>(a, parts, s);
  }
}

template <typename XT, typename DT>
void bwd_types(const LnBwd& a, int parts, bool vec, cudaStream_t s) {
  constexpr int V = sizeof(XT) == 2 && sizeof(DT) == 2 ? 8 : 4;
  if (a.cols > kBwdMaxCols) {
    const int64_t chunk = (a.rows + parts - 1) / parts;
    ln_bwd_wide_cols_kernel<XT, DT>
        <<<dim3((unsigned)((a.cols + 127) / 128), (unsigned)parts), 128, 0, s>>>(a, chunk);
    ln_bwd_wide_rows_kernel<XT, DT><<<(unsigned)a.rows, 512, 0, s>>>(a);
  } else if (vec) {
    bwd_width<XT, DT, V>(a, parts, s);
  } else {
    bwd_width<XT, DT, 1>(a, parts, s);
  }
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

// A rows x cols matrix in memory, for the overlap rule of the caller-buffer calls.
bool matrices_overlap(const void* p, int64_t ld, size_t esz, const void* q, int64_t qld,
                      size_t qesz, int64_t rows, int64_t cols) {
  const uintptr_t p0 = reinterpret_cast<uintptr_t>(p), q0 = reinterpret_cast<uintptr_t>(q);
  const uintptr_t pw = (uintptr_t)cols * esz, qw = (uintptr_t)cols * qesz;
  const uintptr_t ps = (uintptr_t)ld * esz, qs = (uintptr_t)qld * qesz;
  const uintptr_t p1 = p0 + (uintptr_t)(rows - 1) * ps + pw, q1 = q0 + (uintptr_t)(rows - 1) * qs + qw;
  if (p1 <= q0 || q1 <= p0) return false;
  if (ps != qs || ps == 0) return true;
  // same row pitch: column slices of one buffer may interleave
  const uintptr_t d = q0 >= p0 ? (q0 - p0) % ps : (ps - (p0 - q0) % ps) % ps;
  return !(d >= pw && d + qw <= ps);
}

// An output matrix may be one input (same place, pitch and element size) or
// share no element with it.
int check_out_overlap(const void* out, int64_t out_ld, size_t out_esz, const char* what,
                      const void* in, int64_t in_ld, size_t in_esz, int64_t rows, int64_t cols) {
  if (rows == 0 || cols == 0) return MMN_OK;
  if (out == in && out_ld == in_ld && out_esz == in_esz) return MMN_OK;
  if (matrices_overlap(out, out_ld, out_esz, in, in_ld, in_esz, rows, cols))
    return fail(MMN_E_INVALID, std::string(what) + " overlaps an input it does not equal");
  return MMN_OK;
}

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
  if (!empty && (rc = check_out_overlap(y, y_ld, esize(y_dtype), "y", x, x_ld, esize(x_dtype),
                                        rows, cols)) != MMN_OK)
    return rc;
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
  const int v = x_dtype == MMN_DTYPE_BF16 && y_dtype == MMN_DTYPE_BF16 ? 8 : 4;
  const bool vec = cols % v == 0 && vec_rows(x, a.x_ld, esize(x_dtype), v) &&
                   vec_rows(y, a.y_ld, esize(y_dtype), v) &&
                   vec_rows(gamma, cols, esize(param_dtype), v) &&
                   vec_rows(beta, cols, esize(param_dtype), v);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool xb = x_dtype == MMN_DTYPE_BF16, yb = y_dtype == MMN_DTYPE_BF16;
  if (xb && yb)
    fwd_types<__nv_bfloat16, __nv_bfloat16>(a, vec, s);
  else if (xb)
    fwd_types<__nv_bfloat16, float>(a, vec, s);
  else if (yb)
    fwd_types<float, __nv_bfloat16>(a, vec, s);
  else
    fwd_types<float, float>(a, vec, s);
  MMN_CUDA_TRY(cudaGetLastError());
  return MMN_OK;
}

extern "C" int mmn_layer_norm_backward_workspace(int64_t rows, int64_t cols, int device,
                                                 int64_t* bytes) {
  if (!bytes) return fail(MMN_E_INVALID, "null pointer");
  int rc, sms = 0;
  if ((rc = check_extent(rows, cols)) != MMN_OK) return rc;
  if ((rc = percall_device(device, &sms)) != MMN_OK) return rc;
  *bytes = (int64_t)bwd_parts(rows, cols, sms) * 2 * cols * 4;
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
  if (dgamma == dbeta && cols > 0) return fail(MMN_E_INVALID, "dgamma and dbeta are one buffer");
  if (!empty &&
      ((rc = check_out_overlap(dx, dx_ld, esize(x_dtype), "dx", x, x_ld, esize(x_dtype), rows,
                               cols)) != MMN_OK ||
       (rc = check_out_overlap(dx, dx_ld, esize(x_dtype), "dx", dy, dy_ld, esize(dy_dtype), rows,
                               cols)) != MMN_OK))
    return rc;
  if (!empty && reinterpret_cast<uintptr_t>(workspace) % 16)
    return fail(MMN_E_INVALID, "workspace is not 16-byte aligned");
  if ((rc = percall_device(device, &sms)) != MMN_OK) return rc;
  const int parts = bwd_parts(rows, cols, sms);
  if (workspace_bytes < (int64_t)parts * 2 * cols * 4)
    return fail(MMN_E_INVALID, "workspace is smaller than mmn_layer_norm_backward_workspace gives");
  if (cols == 0) return MMN_OK;
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
                     vec_rows(gamma, cols, esize(param_dtype), v);
    const bool xb = x_dtype == MMN_DTYPE_BF16, db = dy_dtype == MMN_DTYPE_BF16;
    if (xb && db)
      bwd_types<__nv_bfloat16, __nv_bfloat16>(a, parts, vec, s);
    else if (xb)
      bwd_types<__nv_bfloat16, float>(a, parts, vec, s);
    else if (db)
      bwd_types<float, __nv_bfloat16>(a, parts, vec, s);
    else
      bwd_types<float, float>(a, parts, vec, s);
    MMN_CUDA_TRY(cudaGetLastError());
  }
  if (parts == 0 && accumulate) return MMN_OK;  // no rows: the sums are zero
  LnSum su{static_cast<const float*>(workspace), dgamma, dbeta, cols, parts,
           grad_dtype == MMN_DTYPE_BF16, accumulate != 0};
  ln_bwd_sum_kernel<<<dim3((unsigned)((cols + 31) / 32), 2), 256, 0, s>>>(su);
  MMN_CUDA_TRY(cudaGetLastError());
  return MMN_OK;
}
