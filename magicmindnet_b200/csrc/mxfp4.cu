// 4-bit microscaled matrices (OCP Microscaling v1.0, MXFP4): quantisation along
// the rows, the columns or both in one pass, the way back, and the products.
//
// A block is 32 consecutive elements of a row. With e = floor(log2 max |x|) over
// the block, its scale is 2^(e - 2) (held as the byte e - 2 + 127, clamped at
// 0), its elements x / scale rounded to the nearest of 0, 1/2, 1, 3/2, 2, 3, 4,
// 6 with ties to the even code, values above 6 becoming 6. The division is by a
// power of two, so it is exact where the result matters and the one rounding is
// the conversion's. A block that holds an Inf or a NaN has the scale byte 255,
// which the format reads as NaN for every element: a non-finite gradient stays
// visible to the step's non-finite scan behind the product.
//
// Layout of a matrix of R rows and K columns: elements row-major, two to a byte
// (the even column in the low half), rows padded with zeros to a multiple of 32;
// scales in blocks of 128 rows x 128 columns, 512 bytes each, byte (r % 32) * 16 +
// (r / 32 % 4) * 4 + (k / 32 % 4), the blocks of one 128-row tile one after the
// other and padded to an even number with zero bytes. That is the form that
// tcgen05 wants its scales in (mxfp4_gemm.cuh).
#include "mxfp4_gemm.cuh"

#include <mutex>
#include <vector>

#include "capi_internal.cuh"
#include "ns_engine.cuh"
#include "unaligned.cuh"

namespace mmn {
namespace {

// -------------------------------------------------------------- conversions
// The values of four 4-bit codes as two pairs of bf16, which hold them: the byte
// permutation looks up the high and the low byte of 0, 1/2, 1, 3/2, 2, 3, 4, 6.
__device__ __forceinline__ uint2 e2m1x4_bf16(uint32_t w) {
  const uint32_t sel = w & 0x7777u;
  const uint32_t hi = __byte_perm(0x3F3F3F00u, 0x40404040u, sel);
  const uint32_t lo = __byte_perm(0xC0800000u, 0xC0804000u, sel);
  return make_uint2(__byte_perm(lo, hi, 0x5140) | ((w & 0x8u) << 12) | ((w & 0x80u) << 24),
                    __byte_perm(lo, hi, 0x7362) | ((w & 0x800u) << 4) | ((w & 0x8000u) << 16));
}

// A scale as a pair of bf16, 2^(s - 127): subnormal for 0, NaN for 255.
__device__ __forceinline__ uint32_t mx_scale_bf16x2(uint32_t s) {
  const uint32_t b = s == 255u ? 0x7FFFu : (s ? s << 7 : 0x0040u);
  return b | (b << 16);
}

__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t x, uint32_t y) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y));
  return r;
}

__device__ __forceinline__ float mx_scale_value(uint32_t s) {
  if (s == 255u) return __uint_as_float(0x7FFFFFFFu);
  return s ? __uint_as_float(s << 23) : __uint_as_float(0x00400000u);
}

// ------------------------------------------------------------- quantisation
struct MxQuantArgs {
  const void* x;
  int64_t ld;
  int rows, cols;
  uint8_t *codes, *scales;      // of x, or null
  uint8_t *codes_t, *scales_t;  // of x transposed, or null
  int64_t pitch, pitch_t;       // bytes of one row of codes
  int ka, ka_t;                 // scale blocks of one 128-row tile
  int nct;                      // column tiles of the grid
};

// The larger magnitudes of two pairs of bf16 (m >= 0); a NaN stays one.
__device__ __forceinline__ uint32_t max_abs2(uint32_t m, uint32_t x) {
  uint32_t r;
  asm("{\n\t.reg .b32 t;\n\t"
      "abs.bf16x2 t, %2;\n\t"
      "max.NaN.bf16x2 %0, %1, t;\n\t}"
      : "=r"(r)
      : "r"(m), "r"(x));
  return r;
}

template <typename T>
struct MxTile {
  static constexpr int kPitch = 128 * sizeof(T) + 16;  // bytes; the skew spreads a column over banks
  static constexpr int kCodePitch = 80;
  static constexpr int kSmem = 128 * kPitch + 1024;
};

__device__ __forceinline__ void cp_async16(void* dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)),
               "l"(__cvta_generic_to_global(src)), "r"(bytes)
               : "memory");
}

// One 128 x 128 tile per block: it goes to shared memory once; threads take its
// blocks of 32 along the rows, then down the columns, whose bytes are collected
// in shared memory so that global memory sees 64 consecutive bytes per row of
// codes. A tile gives exactly one 512-byte block of scales in each direction.
// Operands not in L2: 8192 x 4096 bf16 rows 16.1 us, columns 16.2, both 21.7 (0.81, 0.80
// and 0.73 of a copy's rate); 16384 x 8192 52, 54 and 73 us (1.0, 0.96, 0.87); 14336 x 4096
// fp32, a weight's copies after a step, 44, 45 and 57 us (0.93, 0.91, 0.80). With few waves
// of blocks their loads and their work fall together; within a block "both" is 14
// instructions an element (issue slots 69% busy, the shared-memory pipe 62%).
template <typename T, bool SHIFT>
__global__ void __launch_bounds__(256) mx_quantize_kernel(const MxQuantArgs a) {
  constexpr int kPitch = MxTile<T>::kPitch;
  constexpr bool kBf16 = sizeof(T) == 2, kMove = SHIFT && !kBf16;
  extern __shared__ __align__(16) uint8_t sm[];
  uint8_t* codes_s = sm;  // the transposed codes take the tile's place once it is read
  uint8_t* sf_row = sm + 128 * kPitch;
  uint8_t* sf_col = sf_row + 512;
  const int tid = threadIdx.x;
  griddep_wait();
  griddep_launch_dependents();  // a product's setup overlaps this kernel's end
  const int ct = blockIdx.x % a.nct, rt = blockIdx.x / a.nct;
  const int c0 = ct * 128, r0 = rt * 128;
  const bool in_c = c0 < a.cols, in_r = r0 < a.rows;
  if (!in_c || !in_r) {
    // padding of the scales to an even number of blocks
    if (tid < 32) {
      const uint4 z = make_uint4(0, 0, 0, 0);
      if (in_r && a.scales)
        reinterpret_cast<uint4*>(a.scales + ((int64_t)rt * a.ka + ct) * 512)[tid] = z;
      if (in_c && a.scales_t)
        reinterpret_cast<uint4*>(a.scales_t + ((int64_t)ct * a.ka_t + rt) * 512)[tid] = z;
    }
    return;
  }
  const T* x = static_cast<const T*>(a.x);
  const int nr = min(128, a.rows - r0), nc = min(128, a.cols - c0);
  constexpr int kPer = 16 / sizeof(T), kCh = 128 / kPer;
  // where row r's first element of the tile lies past a vector's start (the same in
  // rows kPer apart)
  const uint32_t e0 = (uint32_t)(reinterpret_cast<uintptr_t>(x) / sizeof(T)) +
                      (uint32_t)r0 * (uint32_t)a.ld + (uint32_t)c0;
  auto offset = [&](int r) {
    return SHIFT ? (int)((e0 + (uint32_t)r * (uint32_t)a.ld) & (kPer - 1)) : 0;
  };
  if constexpr (!SHIFT) {
#pragma unroll
    for (int i = 0; i < 128 * kCh / 256; ++i) {
      const int id = i * 256 + tid, r = id / kCh, c = (id % kCh) * kPer;
      const int bytes = r < nr ? max(0, min(kPer, nc - c)) * (int)sizeof(T) : 0;
      const T* src = bytes ? x + (int64_t)(r0 + r) * a.ld + c0 + c : x;
      cp_async16(sm + r * kPitch + c * sizeof(T), src, bytes);
    }
  } else {
    // Rows that start anywhere arrive in whole vectors, one more a row. bf16 moves to
    // its place within shared memory (44 to 45 us moved as it is read), fp32 as it is
    // read (73 to 75 moved before). 16384 x 4095 bf16 43 us, fp32 68 along the rows and
    // 65 along the columns (80 and 128 with an element a load; 55 and 123 with the
    // vectors moved on their way to shared memory, which leaves fewer loads in flight).
    // Aligned rows take 26 and 48 us: the move is a second pass over shared memory whose
    // instructions count (the shared-memory pipe 67% busy, an instruction issued in 64% of
    // the cycles, DRAM 41%); an uneven row of a tile touches 9 sectors for 8.
    auto copy = [&](int r, int j) {
      const T* row = x + (int64_t)(r0 + r) * a.ld + c0;
      const int c = j * kPer - offset(r);  // the vector's first column
      uint8_t* dst = sm + r * kPitch + j * 16;
      if (r < nr && c + c0 < 0 && row + c < x) {  // the matrix starts inside this vector
        for (int k = 0; k < kPer; ++k)
          if (row + c + k >= x && c + k < nc) reinterpret_cast<T*>(dst)[k] = row[c + k];
      } else {
        const int bytes = r < nr ? max(0, min(kPer, a.cols - c0 - c)) * (int)sizeof(T) : 0;
        cp_async16(dst, bytes ? row + c : x - vec_offset<T, kPer>(x), bytes);
      }
    };
#pragma unroll
    for (int i = 0; i < 128 * kCh / 256; ++i) copy((i * 256 + tid) / kCh, tid % kCh);
    if (tid < 128) copy(tid, kCh);
  }
  asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  if constexpr (SHIFT && kBf16) {
    constexpr int kRows = 256 / kCh;
    static_assert(kRows % kPer == 0, "rows of a thread differ in their offset");
    const int r1 = tid / kCh, j1 = tid % kCh, o = offset(r1);
#pragma unroll
    for (int i = 0; i < 128 / kRows; ++i) {
      // (the lanes of a warp take whole rows)
      uint4* at = reinterpret_cast<uint4*>(sm + (i * kRows + r1) * kPitch) + j1;
      const uint4 u = at[0], v = at[1];
      uint32_t d[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
      shift_down<T, 4>(d, o);
      if (nc < 128) keep_first<T, 4>(d, nc - j1 * kPer);
      __syncwarp();
      at[0] = make_uint4(d[0], d[1], d[2], d[3]);
    }
    __syncthreads();
  }

  if (a.codes) {
    // a thread per block of 32: eight rows at a time read the same columns, so the
    // skewed rows spread over the banks, and a row's four blocks leave together
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = (i * 8 + (tid >> 5)) * 8 + (tid & 7), k4 = (tid >> 3) & 3;
      constexpr int N = 8 * (int)sizeof(T);  // words of a block
      uint32_t d[N + 4], q4[4], s;
#pragma unroll
      for (int q = 0; q < N / 4 + (kMove ? 1 : 0); ++q) {
        const uint4 u =
            *reinterpret_cast<const uint4*>(sm + r * kPitch + k4 * 32 * sizeof(T) + q * 16);
        d[4 * q] = u.x, d[4 * q + 1] = u.y, d[4 * q + 2] = u.z, d[4 * q + 3] = u.w;
      }
      if constexpr (kMove) {
        shift_down<T, N>(d, offset(r));
        if (nc < 128) keep_first<T, N>(d, nc - k4 * 32);
      }
      if constexpr (kBf16) {
        uint32_t mm = 0;
#pragma unroll
        for (int k = 0; k < 16; ++k) mm = max_abs2(mm, d[k]);
        s = mx_scale(max(mm & 0xFFFFu, mm >> 16) << 16);
      } else {
        uint32_t m = 0;
#pragma unroll
        for (int k = 0; k < 32; ++k) m = max(m, d[k] & 0x7FFFFFFFu);
        s = mx_scale(m);
      }
      const float inv = mx_inv_scale(s);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
          v[k] = __uint_as_float(!kBf16  ? d[(q * 8 + k) % N]
                                 : k & 1 ? d[q * 4 + k / 2] & 0xFFFF0000u
                                         : d[q * 4 + k / 2] << 16) *
                 inv;
        q4[q] = e2m1x8(v);
      }
      const int64_t off = (int64_t)ct * 64 + k4 * 16;
      if (r < nr && off < a.pitch)
        *reinterpret_cast<uint4*>(a.codes + (int64_t)(r0 + r) * a.pitch + off) =
            make_uint4(q4[0], q4[1], q4[2], q4[3]);
      sf_row[(r & 31) * 16 + (r >> 5) * 4 + k4] = (uint8_t)s;
    }
  }
  if (a.codes_t) {
    // 64 values per thread: two columns of 32 rows (bf16, read as words), or one
    // column in two blocks of rows
    uint4 o[2];
    uint32_t sb[2];
    if constexpr (kBf16) {
      const int cp = tid & 63, rb = tid >> 6;
      uint32_t w[32], mm = 0;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        w[i] = *reinterpret_cast<const uint32_t*>(sm + (rb * 32 + i) * kPitch + cp * 4);
        mm = max_abs2(mm, w[i]);
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        sb[half] = mx_scale(half ? mm & 0xFFFF0000u : mm << 16);
        const float inv = mx_inv_scale(sb[half]);
        uint32_t q4[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float v[8];
#pragma unroll
          for (int k = 0; k < 8; ++k)
            v[k] = __uint_as_float(half ? w[q * 8 + k] & 0xFFFF0000u : w[q * 8 + k] << 16) * inv;
          q4[q] = e2m1x8(v);
        }
        o[half] = make_uint4(q4[0], q4[1], q4[2], q4[3]);
      }
    } else {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int c = tid & 127, rb = (tid >> 7) + 2 * half;
        float w[32];
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          w[i] = *reinterpret_cast<const float*>(sm + (rb * 32 + i) * kPitch + (c + (kMove ? offset(i) : 0)) * 4);
          if (kMove && c >= nc) w[i] = 0.0f;
          m = max(m, __float_as_uint(w[i]) & 0x7FFFFFFFu);
        }
        sb[half] = mx_scale(m);
        const float inv = mx_inv_scale(sb[half]);
        uint32_t q4[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float v[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] = w[q * 8 + k] * inv;
          q4[q] = e2m1x8(v);
        }
        o[half] = make_uint4(q4[0], q4[1], q4[2], q4[3]);
      }
    }
    __syncthreads();
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int c = kBf16 ? (tid & 63) * 2 + half : tid & 127;
      const int rb = kBf16 ? tid >> 6 : (tid >> 7) + 2 * half;
      *reinterpret_cast<uint4*>(codes_s + c * MxTile<T>::kCodePitch + rb * 16) = o[half];
      sf_col[(c & 31) * 16 + (c >> 5) * 4 + rb] = (uint8_t)sb[half];
    }
  }
  __syncthreads();
  if (a.codes_t) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int id = i * 256 + tid, c = id >> 2, seg = id & 3;
      const int64_t off = (int64_t)rt * 64 + seg * 16;
      if (c < nc && off < a.pitch_t)
        *reinterpret_cast<uint4*>(a.codes_t + (int64_t)(c0 + c) * a.pitch_t + off) =
            *reinterpret_cast<const uint4*>(codes_s + c * MxTile<T>::kCodePitch + seg * 16);
    }
    if (tid >= 32 && tid < 64)
      reinterpret_cast<uint4*>(a.scales_t + ((int64_t)ct * a.ka_t + rt) * 512)[tid - 32] =
          reinterpret_cast<const uint4*>(sf_col)[tid - 32];
  }
  if (a.codes && tid < 32)
    reinterpret_cast<uint4*>(a.scales + ((int64_t)rt * a.ka + ct) * 512)[tid] =
        reinterpret_cast<const uint4*>(sf_row)[tid];
}

// ----------------------------------------------------------- the way back
struct MxDequantArgs {
  const uint8_t *codes, *scales;
  void* out;
  int64_t ld, pitch;
  int rows, cols;
  int ka;
  int nct;  // column tiles
};

__device__ __forceinline__ void store32(void* p, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]),
               "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// 32 rows x 512 (bf16) or 256 (fp32) columns per block. A lane turns the codes of 32
// output bytes into one store, so that every sector is written whole; the loads of
// a lane's rows are issued first, without branches between them (what lies outside
// is read from the edge and not used). 16384 x 4096: 28.1 us to bf16, 48.8 to fp32
// (0.93 and 0.95 of a copy's rate; 29.8 and 49.0 with 16-byte stores).
// SHIFT: output rows that start anywhere. A lane's columns begin where the row's
// memory is aligned, o columns before its codes; the codes are moved by o nibbles,
// and the first o values may belong to the block before. 16384 x 4095: 39.5 and
// 50.3 us (187 and 89 with an element a store); bf16 is bound by instructions (issued
// in 75% of the cycles), the moving and the second scale's selection among them.
template <typename T, bool SHIFT>
__global__ void __launch_bounds__(256) mx_dequantize_kernel(const MxDequantArgs a) {
  constexpr int V = 32 / sizeof(T), W = V / 8, NR = 4;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int ct = blockIdx.x % a.nct, rt = blockIdx.x / a.nct;
  griddep_wait();
  griddep_launch_dependents();
  T* const out = static_cast<T*>(a.out) + (int64_t)(rt * 32 + warp) * a.ld;
  // of a lane's rows, eight apart: V divides 8 or 16 of them
  static_assert(V == 8 || V == 16, "offsets of a lane's rows");
  const int o2[2] = {SHIFT ? vec_offset<T, V>(out) : 0,
                     SHIFT ? vec_offset<T, V>(out + 8 * a.ld) : 0};
  // the lane's codes and those before
  const int at = (ct * 32 + lane) * V, top = (a.cols - 1) / 32 * 32 + 32 - V;
  const int e = min(at, top), f = max(min(at - V, top), 0);
  const uint8_t* const scales = a.scales + (int64_t)(rt >> 2) * a.ka * 512 + (rt & 3) * 4;
  const uint8_t* const se = scales + (int64_t)(e >> 7) * 512 + ((e >> 5) & 3);
  const uint8_t* const sf = scales + (int64_t)(f >> 7) * 512 + ((f >> 5) & 3);
  uint32_t w[NR][2 * W], s[NR], sp[NR];  // w: the codes before, the codes
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int rr = min(rt * 32 + warp + 8 * i, a.rows - 1) & 31;
    const uint32_t* p =
        reinterpret_cast<const uint32_t*>(a.codes + (int64_t)(rt * 32 + rr) * a.pitch);
    if constexpr (W == 2) {
      const uint2 u = *reinterpret_cast<const uint2*>(p + e / 8);
      w[i][2] = u.x, w[i][3] = u.y;
      if constexpr (SHIFT) {
        const uint2 v = *reinterpret_cast<const uint2*>(p + f / 8);
        w[i][0] = v.x, w[i][1] = v.y;
      }
    } else {
      w[i][1] = p[e / 8];
      if constexpr (SHIFT) w[i][0] = p[f / 8];
    }
    s[i] = se[rr * 16];
    if constexpr (SHIFT) sp[i] = sf[rr * 16];
  }
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int r = rt * 32 + warp + 8 * i, o = o2[i & 1], c = at - o;
    if (r >= a.rows) break;
    uint32_t x[W], v[8];
    if constexpr (!SHIFT) {
#pragma unroll
      for (int k = 0; k < W; ++k) x[k] = w[i][W + k];
    } else if constexpr (W == 1) {
      x[0] = __funnelshift_l(w[i][0], w[i][1], 4 * o);
    } else {
      // (the shift counts modulo 32)
      const uint32_t t = __funnelshift_l(w[i][1], w[i][2], 4 * o);
      x[0] = o & 8 ? __funnelshift_l(w[i][0], w[i][1], 4 * o) : t;
      x[1] = o & 8 ? t : __funnelshift_l(w[i][2], w[i][3], 4 * o);
    }
    if constexpr (sizeof(T) == 2) {
      // a value times its scale is a bf16 (down to 2^-128), so the product is exact
      const uint32_t fs = mx_scale_bf16x2(s[i]);
      const uint32_t gs = SHIFT ? mx_scale_bf16x2(sp[i]) : 0u;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint2 p = e2m1x4_bf16(x[k / 2] >> (16 * (k & 1)));
        // columns 4 k to 4 k + 3 of the lane's: those below o take the first scale
        const uint32_t m0 = (o > 4 * k ? 0xFFFFu : 0u) | (o > 4 * k + 1 ? 0xFFFF0000u : 0u);
        const uint32_t m1 = (o > 4 * k + 2 ? 0xFFFFu : 0u) | (o > 4 * k + 3 ? 0xFFFF0000u : 0u);
        v[2 * k] = mul_bf16x2(p.x, (fs & ~m0) | (gs & m0));
        v[2 * k + 1] = mul_bf16x2(p.y, (fs & ~m1) | (gs & m1));
      }
    } else {
      const float fs = mx_scale_value(s[i]), gs = SHIFT ? mx_scale_value(sp[i]) : 0.0f;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint2 p = e2m1x4_bf16(x[0] >> (16 * k));
        const uint32_t u[4] = {p.x << 16, p.x & 0xFFFF0000u, p.y << 16, p.y & 0xFFFF0000u};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          v[4 * k + j] = __float_as_uint(__uint_as_float(u[j]) * (o > 4 * k + j ? gs : fs));
      }
    }
    T* const row = out + (int64_t)(8 * i) * a.ld + c;
    if (c >= 0 && c + V <= a.cols) {
      store32(row, v);
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k)
        if (c + k >= 0 && c + k < a.cols) {
          if constexpr (sizeof(T) == 2)
            reinterpret_cast<uint16_t*>(row)[k] = (uint16_t)(v[k / 2] >> (16 * (k & 1)));
          else
            reinterpret_cast<uint32_t*>(row)[k] = v[k];
        }
    }
  }
}

// An empty sum: zeros, unless they are to be added.
__global__ void __launch_bounds__(256) mx_zero_kernel(void* out, int64_t ld, int64_t rows,
                                                      int64_t cols, int bf16) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * cols;
       i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / cols, o = r * ld + (i - r * cols);
    if (bf16)
      static_cast<__nv_bfloat16*>(out)[o] = __float2bfloat16_rn(0.0f);
    else
      static_cast<float*>(out)[o] = 0.0f;
  }
}

// -------------------------------------------------------------------- host
constexpr int64_t kMaxDim = int64_t(1) << 30;

int64_t code_pitch(int64_t cols) { return (cols + 31) / 32 * 16; }
int64_t scale_blocks(int64_t cols) { return (cols + 255) / 256 * 2; }
int64_t code_bytes(int64_t rows, int64_t cols) { return rows * code_pitch(cols); }
int64_t scale_bytes(int64_t rows, int64_t cols) {
  return (rows + 127) / 128 * scale_blocks(cols) * 512;
}

bool bad_dtype(int d) { return d != MMN_DTYPE_F32 && d != MMN_DTYPE_BF16; }
size_t esize(int d) { return d == MMN_DTYPE_BF16 ? 2 : 4; }

int check_dims(int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 0) return fail(MMN_E_INVALID, "negative dimension");
  if (rows > kMaxDim || cols > kMaxDim)
    return fail(MMN_E_SHAPE, "rows and cols must not exceed 2^30");
  return MMN_OK;
}

// Pointers of a 4-bit matrix before any device is touched.
int check_mx(const mmn_mxfp4* q, const char* what) {
  int rc = check_dims(q->rows, q->cols);
  if (rc != MMN_OK) return rc;
  if (q->rows == 0 || q->cols == 0) return MMN_OK;
  if (!q->codes || !q->scales)
    return fail(MMN_E_INVALID, std::string(what) + ": null codes or scales");
  if (reinterpret_cast<uintptr_t>(q->codes) % 16 || reinterpret_cast<uintptr_t>(q->scales) % 16)
    return fail(MMN_E_INVALID, std::string(what) + ": codes or scales are not 16-byte aligned");
  return MMN_OK;
}

int check_mx_device(const mmn_mxfp4* q, int device, const char* what) {
  if (q->rows == 0 || q->cols == 0) return MMN_OK;
  int rc = check_device_ptr(q->codes, device, what);
  return rc != MMN_OK ? rc : check_device_ptr(q->scales, device, what);
}

struct Range {
  const void* p;
  int64_t bytes;
};

bool ranges_meet(const Range& a, const Range& b) {
  const uintptr_t a0 = reinterpret_cast<uintptr_t>(a.p), b0 = reinterpret_cast<uintptr_t>(b.p);
  return a.bytes > 0 && b.bytes > 0 && a0 < b0 + (uintptr_t)b.bytes && b0 < a0 + (uintptr_t)a.bytes;
}

Range matrix_range(const void* p, int64_t ld, int64_t rows, int64_t cols, size_t esz) {
  return {p, rows && cols ? ((rows - 1) * ld + cols) * (int64_t)esz : 0};
}
Range codes_range(const mmn_mxfp4* q) { return {q->codes, code_bytes(q->rows, q->cols)}; }
Range scales_range(const mmn_mxfp4* q) {
  return {q->scales, q->cols ? scale_bytes(q->rows, q->cols) : 0};
}

template <int BN, int SRC>
int split_setup() {
  MMN_CUDA_TRY(cudaFuncSetAttribute(mx_split_kernel<BN, SRC>,
                                    cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    MxSplit<BN, SRC>::kSmemBytes));
  return MMN_OK;
}

// Shared memory of the kernels above 48 KB, once per device.
int kernel_setup(int device) {
  static std::mutex mu;
  static uint64_t done = 0;
  std::lock_guard<std::mutex> lock(mu);
  if (device < 64 && (done >> device) & 1u) return MMN_OK;
  const auto smem = cudaFuncAttributeMaxDynamicSharedMemorySize;
  MMN_CUDA_TRY(cudaFuncSetAttribute(mx_quantize_kernel<float, false>, smem, MxTile<float>::kSmem));
  MMN_CUDA_TRY(cudaFuncSetAttribute(mx_quantize_kernel<float, true>, smem, MxTile<float>::kSmem));
  int rc;
  if ((rc = split_setup<16, 0>()) != MMN_OK || (rc = split_setup<32, 0>()) != MMN_OK ||
      (rc = split_setup<64, 0>()) != MMN_OK || (rc = split_setup<128, 0>()) != MMN_OK ||
      (rc = split_setup<16, 1>()) != MMN_OK || (rc = split_setup<16, 2>()) != MMN_OK)
    return rc;
  MMN_CUDA_TRY(cudaFuncSetAttribute(mx_gemm_pair_kernel<192>, smem, MxPair<192>::kSmemBytes));
  MMN_CUDA_TRY(cudaFuncSetAttribute(mx_gemm_pair_kernel<256>, smem, MxPair<256>::kSmemBytes));
  if (device < 64) done |= uint64_t(1) << device;
  return MMN_OK;
}

int launch_quantize(const void* x, int64_t ld, int dtype, int64_t rows, int64_t cols,
                    const mmn_mxfp4* q, const mmn_mxfp4* qt, cudaStream_t s) {
  MxQuantArgs a{};
  a.x = x;
  a.ld = ld;
  a.rows = (int)rows;
  a.cols = (int)cols;
  if (q) {
    a.codes = static_cast<uint8_t*>(q->codes);
    a.scales = static_cast<uint8_t*>(q->scales);
  }
  if (qt) {
    a.codes_t = static_cast<uint8_t*>(qt->codes);
    a.scales_t = static_cast<uint8_t*>(qt->scales);
  }
  a.pitch = code_pitch(cols);
  a.pitch_t = code_pitch(rows);
  a.ka = (int)scale_blocks(cols);
  a.ka_t = (int)scale_blocks(rows);
  a.nct = q ? a.ka : (int)((cols + 127) / 128);
  const int64_t nrt = qt ? a.ka_t : (rows + 127) / 128;
  const bool vec = vec_rows(x, ld, esize(dtype), 16);
  const int64_t blocks = nrt * a.nct;
  if (blocks > (int64_t(1) << 31) - 1) return fail(MMN_E_SHAPE, "matrix too large");
  const dim3 grid((unsigned)blocks);
  const bool bf = dtype == MMN_DTYPE_BF16;
  const auto kernel = bf ? (vec ? mx_quantize_kernel<__nv_bfloat16, false>
                                : mx_quantize_kernel<__nv_bfloat16, true>)
                         : (vec ? mx_quantize_kernel<float, false> : mx_quantize_kernel<float, true>);
  MMN_CUDA_TRY(launch_dependent(kernel, grid, 256,
                                bf ? MxTile<__nv_bfloat16>::kSmem : MxTile<float>::kSmem, s, a));
  return MMN_OK;
}

// out = A W^T with A's rows on the N side: A as 4-bit codes (SRC 0) or as rows to
// round (SRC 1: bf16, 2: fp32).
template <int BN, int SRC>
int launch_split(const mmn_mxfp4* a, const MxRows& rows, const mmn_mxfp4* w, int64_t n,
                 MxGemmArgs& g, int sms, cudaStream_t s) {
  CUtensorMap tw, tx;
  std::string err = encode_byte_rows(&tw, w->codes, code_pitch(w->cols), w->rows, 128);
  if (SRC != 0)
    tx = tw;
  else if (err.empty())
    err = encode_byte_rows(&tx, a->codes, code_pitch(a->cols), a->rows, BN);
  if (!err.empty()) return fail(MMN_E_CUDA, err);
  g.sfa = static_cast<const uint8_t*>(w->scales);
  g.sfb = SRC == 0 ? static_cast<const uint8_t*>(a->scales) : nullptr;
  g.ka = (int)scale_blocks(w->cols);
  g.M = (int)w->rows;
  g.N = (int)n;
  g.num_kb = (int)((w->cols + 255) / 256);
  g.tiles_n = (int)((n + BN - 1) / BN);
  const int64_t tiles = (w->rows + 127) / 128 * g.tiles_n;
  // Split K while a split leaves no CTA without an SM: a cluster of 2, 4 or 8 CTAs
  // with at least one stage of K each.
  int splits = 1;
  while (splits < 8 && tiles * splits * 2 <= sms && splits * 2 <= g.num_kb) splits *= 2;
  if (tiles * splits > (int64_t(1) << 31) - 1) return fail(MMN_E_SHAPE, "product too large");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * splits), 1, 1);
  cfg.blockDim = dim3(MxSplit<BN, SRC>::kThreads, 1, 1);
  cfg.dynamicSmemBytes = MxSplit<BN, SRC>::kSmemBytes;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = splits;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  MMN_CUDA_TRY(cudaLaunchKernelEx(&cfg, mx_split_kernel<BN, SRC>, tw, tx, g, rows, splits));
  return MMN_OK;
}

// The CTA pairs that fit on the GPU at once (a persistent grid must not exceed
// them: a pair scheduled late would run its whole tile list after the others).
// One CTA fills an SM, so both tile widths have the same number.
int max_pairs(int sms, int* out) {
  static std::mutex mu;
  static int known_sms = 0, pairs = 0;  // every sm_100 device gives the same for its SM count
  std::lock_guard<std::mutex> lock(mu);
  if (known_sms != sms) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * (sms / 2), 1, 1);
    cfg.blockDim = dim3(MxPair<256>::kThreads, 1, 1);
    cfg.dynamicSmemBytes = MxPair<256>::kSmemBytes;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    MMN_CUDA_TRY(cudaOccupancyMaxActiveClusters(&n, mx_gemm_pair_kernel<256>, &cfg));
    if (n <= 0) return fail(MMN_E_CUDA, "no CTA pair fits on the device");
    pairs = n < sms / 2 ? n : sms / 2;
    known_sms = sms;
  }
  *out = pairs;
  return MMN_OK;
}

template <int BN>
int launch_pair(const mmn_mxfp4* a, const mmn_mxfp4* b, MxGemmArgs& g, int pairs, cudaStream_t s) {
  CUtensorMap ta, tb, tsa, tsb, to;
  const int64_t runs = scale_blocks(a->cols) / 2;
  std::string err = encode_byte_rows(&ta, a->codes, code_pitch(a->cols), a->rows, 128);
  if (err.empty()) err = encode_byte_rows(&tb, b->codes, code_pitch(b->cols), b->rows, BN / 2);
  if (err.empty()) err = encode_scale_runs(&tsa, a->scales, runs, (a->rows + 127) / 128, 1);
  if (err.empty()) err = encode_scale_runs(&tsb, b->scales, runs, (b->rows + 127) / 128, 2);
  // Stores and fp32 additions go through the tensor map where the rows are aligned and
  // end on 16 bytes: TMA clips a store at the matrix's edge in steps of 16 bytes, so it
  // would write up to 15 bytes behind a row that ends inside one.
  // Additions in memory, TMA's and mx_store_block's, flush values below 2^-126 to zero,
  // which the header says; loads, additions in registers and stores keep them and
  // were measured: 4096 x 14336 x 4096 164 us against 139, 8192 x 2048 x 4096 55 against
  // 44, and with rows that start anywhere 4096 x 14335 x 4095 232 against 156, 2048 x
  // 4097 x 4096 68 against 30. bf16 values are added in
  // the epilogue's registers: a TMA addition would round the product to bf16
  // before the sum.
  const int esz = g.out_bf16 ? 2 : 4;
  g.tma_out = g.vec && b->rows * esz % 16 == 0 && !(g.out_bf16 && g.accumulate);
  if (!g.tma_out)
    to = ta;
  else if (err.empty())
    err = encode_store_rows(&to, g.out, a->rows, b->rows, g.ld, esz);
  if (!err.empty()) return fail(MMN_E_CUDA, err);
  g.M = (int)a->rows;
  g.N = (int)b->rows;
  g.num_kb = (int)((a->cols + 255) / 256);
  g.tiles_n = (int)((b->rows + BN - 1) / BN);
  const int64_t tiles_m = (a->rows + 255) / 256, tiles = tiles_m * g.tiles_n;
  if (tiles > (int64_t(1) << 30)) return fail(MMN_E_SHAPE, "product too large");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * (unsigned)(tiles < pairs ? tiles : pairs), 1, 1);
  cfg.blockDim = dim3(MxPair<BN>::kThreads, 1, 1);
  cfg.dynamicSmemBytes = MxPair<BN>::kSmemBytes;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  MMN_CUDA_TRY(cudaLaunchKernelEx(&cfg, mx_gemm_pair_kernel<BN>, ta, tb, tsa, tsb, to, g,
                                  (int)tiles_m, (int)tiles));
  return MMN_OK;
}

int launch_gemm_pair(const mmn_mxfp4* a, const mmn_mxfp4* b, MxGemmArgs& g, int sms,
                     cudaStream_t s) {
  int pairs = 0, rc = max_pairs(sms, &pairs);
  if (rc != MMN_OK) return rc;
  // The tile width whose whole waves take fewer clocks (the measured costs of a k
  // block and of a tile, mxfp4_gemm.cuh): 4096 x 14336 x 4096 165.9 thousand clocks
  // with 192 and 173.4 with 256, 4096 x 2048 x 8192 65.2 and 57.5.
  const int64_t tm = (a->rows + 255) / 256, kb = (a->cols + 255) / 256;
  const int64_t w192 = (tm * ((b->rows + 191) / 192) + pairs - 1) / pairs;
  const int64_t w256 = (tm * ((b->rows + 255) / 256) + pairs - 1) / pairs;
  return w192 * (464 * kb + 2000) < w256 * (591 * kb + 3100) ? launch_pair<192>(a, b, g, pairs, s)
                                                             : launch_pair<256>(a, b, g, pairs, s);
}

int zero_out(void* out, int64_t ld, int64_t rows, int64_t cols, int dtype, cudaStream_t s) {
  mx_zero_kernel<<<256, 256, 0, s>>>(out, ld, rows, cols, dtype == MMN_DTYPE_BF16);
  MMN_CUDA_TRY(cudaGetLastError());
  return MMN_OK;
}

int gemm_out(MxGemmArgs* g, void* out, int64_t ld, int dtype, int accumulate, int device) {
  g->out = out;
  g->ld = ld;
  g->out_bf16 = dtype == MMN_DTYPE_BF16;
  g->accumulate = accumulate != 0;
  g->vec = vec_rows(out, ld, esize(dtype), 8);
  return kernel_timeout_word(device, &g->timeouts);
}

// out (a.rows x b.rows) = A B^T, on checked arguments. early_w: B was complete
// before the stream's previous kernel, one of this file, began.
int product(const mmn_mxfp4* a, const mmn_mxfp4* b, void* out, int64_t ld, int dtype,
            int accumulate, int early_w, int sms, int device, cudaStream_t s) {
  if (a->rows == 0 || b->rows == 0) return MMN_OK;
  if (a->cols == 0) return accumulate ? MMN_OK : zero_out(out, ld, a->rows, b->rows, dtype, s);
  MxGemmArgs g{};
  int rc = gemm_out(&g, out, ld, dtype, accumulate, device);
  if (rc != MMN_OK) return rc;
  g.early_w = early_w;
  // 256 x 256 tiles on CTA pairs once 128 x 128 ones fill two thirds of the SMs
  // (512 x 4096 x 4096, 128 of them: 11.6 us against 12.0; 256 x 4096 x 4096, 64:
  // 11.1 against 10.0; 1000 x 1030 x 4096, 72: 18.8 against 10.3).
  const int64_t tiles = (a->rows + 127) / 128 * ((b->rows + 127) / 128);
  if (a->rows > 128 && tiles * 3 > (int64_t)sms * 2)
    return launch_gemm_pair(a, b, g, sms, s);
  const MxRows none{};
  if (a->rows <= 16) return launch_split<16, 0>(a, none, b, a->rows, g, sms, s);
  if (a->rows <= 32) return launch_split<32, 0>(a, none, b, a->rows, g, sms, s);
  if (a->rows <= 64) return launch_split<64, 0>(a, none, b, a->rows, g, sms, s);
  return launch_split<128, 0>(a, none, b, a->rows, g, sms, s);
}

// out = q(x) W^T for at most MMN_MXFP4_DIRECT_ROWS rows of x, on checked arguments.
int direct_linear(const void* x, int64_t ld, int dtype, int64_t rows, const mmn_mxfp4* w, void* out,
                  int64_t out_ld, int out_dtype, int sms, int device, cudaStream_t s) {
  MxGemmArgs g{};
  int rc = gemm_out(&g, out, out_ld, out_dtype, 0, device);
  if (rc != MMN_OK) return rc;
  const MxRows r{x, ld, (int)w->cols, vec_rows(x, ld, esize(dtype), 16)};
  return dtype == MMN_DTYPE_BF16 ? launch_split<16, 1>(nullptr, r, w, rows, g, sms, s)
                                 : launch_split<16, 2>(nullptr, r, w, rows, g, sms, s);
}

int check_out(const void* out, int64_t ld, int dtype, int64_t rows, int64_t cols,
              const Range* in, int n) {
  if (rows == 0 || cols == 0) return MMN_OK;
  if (!out) return fail(MMN_E_INVALID, "null output");
  if (rows > 1 && ld < cols) return fail(MMN_E_INVALID, "a row pitch is smaller than the row");
  const Range o = matrix_range(out, rows > 1 ? ld : cols, rows, cols, esize(dtype));
  for (int i = 0; i < n; ++i)
    if (ranges_meet(o, in[i])) return fail(MMN_E_INVALID, "the output overlaps an input");
  return MMN_OK;
}

}  // namespace
}  // namespace mmn

using namespace mmn;

extern "C" int mmn_mxfp4_size(int64_t rows, int64_t cols, int64_t* code_bytes_out,
                              int64_t* scale_bytes_out) {
  if (!code_bytes_out || !scale_bytes_out) return fail(MMN_E_INVALID, "null pointer");
  const int rc = check_dims(rows, cols);
  if (rc != MMN_OK) return rc;
  *code_bytes_out = code_bytes(rows, cols);
  *scale_bytes_out = cols ? scale_bytes(rows, cols) : 0;
  return MMN_OK;
}

extern "C" int mmn_mxfp4_quantize(const void* x, int64_t x_ld, int dtype, int64_t rows,
                                  int64_t cols, const mmn_mxfp4* q, const mmn_mxfp4* qt,
                                  int device, void* stream) {
  if (bad_dtype(dtype)) return fail(MMN_E_INVALID, "unknown dtype");
  if (!q && !qt) return fail(MMN_E_INVALID, "neither q nor qt is given");
  int rc, sms = 0;
  if ((rc = check_dims(rows, cols)) != MMN_OK) return rc;
  if (q && (q->rows != rows || q->cols != cols))
    return fail(MMN_E_SHAPE, "q is not a rows x cols matrix");
  if (qt && (qt->rows != cols || qt->cols != rows))
    return fail(MMN_E_SHAPE, "qt is not a cols x rows matrix");
  const bool empty = rows == 0 || cols == 0;
  if (!empty && !x) return fail(MMN_E_INVALID, "null pointer");
  if (rows > 1 && x_ld < cols) return fail(MMN_E_INVALID, "a row pitch is smaller than cols");
  if (q && (rc = check_mx(q, "q")) != MMN_OK) return rc;
  if (qt && (rc = check_mx(qt, "qt")) != MMN_OK) return rc;
  if (!empty) {
    const Range rx = matrix_range(x, rows > 1 ? x_ld : cols, rows, cols, esize(dtype));
    Range r[5] = {rx};
    int n = 1;
    for (const mmn_mxfp4* m : {q, qt})
      if (m) {
        r[n++] = codes_range(m);
        r[n++] = scales_range(m);
      }
    for (int i = 0; i < n; ++i)
      for (int j = i + 1; j < n; ++j)
        if (ranges_meet(r[i], r[j])) return fail(MMN_E_INVALID, "two of the buffers overlap");
  }
  if ((rc = percall_device(device, &sms)) != MMN_OK) return rc;
  if (empty) return MMN_OK;
  DeviceGuard guard(device);
  if ((rc = check_device_elems(x, esize(dtype), device, "x")) != MMN_OK) return rc;
  if (q && (rc = check_mx_device(q, device, "q")) != MMN_OK) return rc;
  if (qt && (rc = check_mx_device(qt, device, "qt")) != MMN_OK) return rc;
  if ((rc = kernel_setup(device)) != MMN_OK) return rc;
  return launch_quantize(x, rows > 1 ? x_ld : cols, dtype, rows, cols, q, qt,
                         static_cast<cudaStream_t>(stream));
}

extern "C" int mmn_mxfp4_dequantize(const mmn_mxfp4* q, void* out, int64_t out_ld, int dtype,
                                    int device, void* stream) {
  if (!q) return fail(MMN_E_INVALID, "null matrix");
  if (bad_dtype(dtype)) return fail(MMN_E_INVALID, "unknown dtype");
  int rc, sms = 0;
  if ((rc = check_mx(q, "q")) != MMN_OK) return rc;
  const Range in[] = {codes_range(q), scales_range(q)};
  if ((rc = check_out(out, out_ld, dtype, q->rows, q->cols, in, 2)) != MMN_OK) return rc;
  if ((rc = percall_device(device, &sms)) != MMN_OK) return rc;
  if (q->rows == 0 || q->cols == 0) return MMN_OK;
  DeviceGuard guard(device);
  if ((rc = check_mx_device(q, device, "q")) != MMN_OK) return rc;
  if ((rc = check_device_elems(out, esize(dtype), device, "out")) != MMN_OK) return rc;
  MxDequantArgs a{};
  a.codes = static_cast<const uint8_t*>(q->codes);
  a.scales = static_cast<const uint8_t*>(q->scales);
  a.out = out;
  a.ld = q->rows > 1 ? out_ld : q->cols;
  a.pitch = code_pitch(q->cols);
  a.rows = (int)q->rows;
  a.cols = (int)q->cols;
  a.ka = (int)scale_blocks(q->cols);
  // 32-byte stores; a row that starts between two has one vector more
  const int64_t v = 32 / (int64_t)esize(dtype);
  const bool vec = reinterpret_cast<uintptr_t>(out) % 32 == 0 && a.ld % v == 0;
  a.nct = (int)((q->cols + (vec ? 0 : v - 1) + 32 * v - 1) / (32 * v));
  const int64_t blocks = (q->rows + 31) / 32 * a.nct;
  if (blocks > (int64_t(1) << 31) - 1) return fail(MMN_E_SHAPE, "matrix too large");
  const auto kernel = dtype == MMN_DTYPE_BF16
                          ? (vec ? mx_dequantize_kernel<__nv_bfloat16, false>
                                 : mx_dequantize_kernel<__nv_bfloat16, true>)
                          : (vec ? mx_dequantize_kernel<float, false>
                                 : mx_dequantize_kernel<float, true>);
  MMN_CUDA_TRY(launch_dependent(kernel, dim3((unsigned)blocks), 256, 0,
                                static_cast<cudaStream_t>(stream), a));
  return MMN_OK;
}

extern "C" int mmn_mxfp4_matmul(const mmn_mxfp4* a, const mmn_mxfp4* b, void* out, int64_t out_ld,
                                int dtype, int accumulate, int device, void* stream) {
  if (!a || !b) return fail(MMN_E_INVALID, "null matrix");
  if (bad_dtype(dtype)) return fail(MMN_E_INVALID, "unknown dtype");
  int rc, sms = 0;
  if ((rc = check_mx(a, "a")) != MMN_OK || (rc = check_mx(b, "b")) != MMN_OK) return rc;
  if (a->cols != b->cols)
    return fail(MMN_E_SHAPE, "a and b differ in cols, the axis that is summed");
  const Range in[] = {codes_range(a), scales_range(a), codes_range(b), scales_range(b)};
  if ((rc = check_out(out, out_ld, dtype, a->rows, b->rows, in, 4)) != MMN_OK) return rc;
  if ((rc = percall_device(device, &sms)) != MMN_OK) return rc;
  if (a->rows == 0 || b->rows == 0) return MMN_OK;
  DeviceGuard guard(device);
  if ((rc = check_mx_device(a, device, "a")) != MMN_OK) return rc;
  if ((rc = check_mx_device(b, device, "b")) != MMN_OK) return rc;
  if ((rc = check_device_elems(out, esize(dtype), device, "out")) != MMN_OK) return rc;
  if ((rc = kernel_setup(device)) != MMN_OK) return rc;
  return product(a, b, out, a->rows > 1 ? out_ld : b->rows, dtype, accumulate, 0,
                 sms, device, static_cast<cudaStream_t>(stream));
}

extern "C" int mmn_mxfp4_linear(const void* x, int64_t x_ld, int x_dtype, int64_t rows,
                                const mmn_mxfp4* w, const mmn_mxfp4* xq, void* out, int64_t out_ld,
                                int out_dtype, int device, void* stream) {
  if (!w) return fail(MMN_E_INVALID, "null matrix");
  if (bad_dtype(x_dtype) || bad_dtype(out_dtype)) return fail(MMN_E_INVALID, "unknown dtype");
  int rc, sms = 0;
  if ((rc = check_dims(rows, w->cols)) != MMN_OK) return rc;
  const int64_t cols = w->cols;
  const bool direct = rows <= MMN_MXFP4_DIRECT_ROWS;
  if (!direct && !xq) return fail(MMN_E_INVALID, "xq is needed for this many rows");
  if (xq && (xq->rows != rows || xq->cols != cols))
    return fail(MMN_E_SHAPE, "xq is not a rows x w.cols matrix");
  if ((rc = check_mx(w, "w")) != MMN_OK) return rc;
  if (xq && (rc = check_mx(xq, "xq")) != MMN_OK) return rc;
  const bool empty = rows == 0 || cols == 0;
  if (!empty && !x) return fail(MMN_E_INVALID, "null pointer");
  if (rows > 1 && x_ld < cols) return fail(MMN_E_INVALID, "a row pitch is smaller than cols");
  const Range none{nullptr, 0};
  const Range in[] = {matrix_range(x, rows > 1 ? x_ld : cols, rows, cols, esize(x_dtype)),
                      codes_range(w), scales_range(w), xq ? codes_range(xq) : none,
                      xq ? scales_range(xq) : none};
  for (int i = 0; i < 3; ++i)
    if (ranges_meet(in[i], in[3]) || ranges_meet(in[i], in[4]))
      return fail(MMN_E_INVALID, "xq overlaps an input");
  if (ranges_meet(in[3], in[4])) return fail(MMN_E_INVALID, "xq's codes and scales overlap");
  if ((rc = check_out(out, out_ld, out_dtype, rows, w->rows, in + 1, 4)) != MMN_OK) return rc;
  // (x and out may be column slices of one buffer)
  if (matrices_overlap({out, rows > 1 ? out_ld : w->rows, rows, w->rows, esize(out_dtype)},
                       {x, rows > 1 ? x_ld : cols, rows, cols, esize(x_dtype)}))
    return fail(MMN_E_INVALID, "the output overlaps x");
  if ((rc = percall_device(device, &sms)) != MMN_OK) return rc;
  if (rows == 0 || w->rows == 0) return MMN_OK;
  DeviceGuard guard(device);
  if (cols && (rc = check_device_elems(x, esize(x_dtype), device, "x")) != MMN_OK) return rc;
  if ((rc = check_mx_device(w, device, "w")) != MMN_OK) return rc;
  if (!direct && (rc = check_mx_device(xq, device, "xq")) != MMN_OK) return rc;
  if ((rc = check_device_elems(out, esize(out_dtype), device, "out")) != MMN_OK) return rc;
  if ((rc = kernel_setup(device)) != MMN_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t ld = rows > 1 ? x_ld : cols, old = rows > 1 ? out_ld : w->rows;
  if (cols == 0) return zero_out(out, old, rows, w->rows, out_dtype, s);
  if (direct)
    return direct_linear(x, ld, x_dtype, rows, w, out, old, out_dtype, sms, device, s);
  if ((rc = launch_quantize(x, ld, x_dtype, rows, cols, xq, nullptr, s)) != MMN_OK) return rc;
  return product(xq, w, out, old, out_dtype, 0, 1, sms, device, s);
}

extern "C" int mmn_kernel_status(int device, void* stream) {
  int rc, sms = 0;
  if ((rc = percall_device(device, &sms)) != MMN_OK) return rc;
  DeviceGuard guard(device);
  int* word = nullptr;
  if ((rc = kernel_timeout_word(device, &word)) != MMN_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int count = 0;
  MMN_CUDA_TRY(cudaMemcpyAsync(&count, word, sizeof(int), cudaMemcpyDeviceToHost, s));
  MMN_CUDA_TRY(cudaStreamSynchronize(s));
  static std::mutex mu;
  static std::vector<int> reported;  // per device
  std::lock_guard<std::mutex> lock(mu);
  if (reported.size() <= (size_t)device) reported.resize((size_t)device + 1, 0);
  return report_timeouts(count, &reported[(size_t)device]);
}
