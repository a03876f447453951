// The product of two 4-bit microscaled matrices on the sm_100a tensor cores:
// out[i, j] = sum_k A[i, k] B[j, k], A and B in MXFP4 (e2m1 elements, one ue8m0
// scale per 32 elements of k), fp32 accumulation, rounded once.
//
// tcgen05.mma kind::mxf4 takes K = 64 per instruction (32 bytes of packed
// elements), so a 128-byte swizzle row is 256 elements: a stage holds 256 of K,
// four MMAs. The scales of 128 rows x 128 elements are one 512-byte block, laid
// out in global memory as TMEM wants them (row r, block k at (r % 32) * 16 +
// (r / 32) * 4 + k), so a stage copies them with one bulk load per 128 rows and
// tcgen05.cp moves them to TMEM. Each stage has its own TMEM columns for its
// scales: they are free again when the stage is, which the commit of its MMAs
// says.
#pragma once
#include <cuda.h>

#include "mmn_ptx.cuh"

namespace mmn {

struct MxGemmArgs {
  const uint8_t* sfa;  // split kernel: scale blocks of the operand on the 128 lanes
  const uint8_t* sfb;  // ... and of the other one
  int ka;              // scale blocks along K of one 128-row tile (even)
  int M, N;            // rows of the two operands (the one on the lanes first)
  int num_kb;          // stages of 256 along K
  int tiles_n;
  void* out;
  long long ld;        // elements between rows of out
  int out_bf16;
  int accumulate;
  int vec;             // out and ld are aligned for 16-byte accesses
  int tma_out;         // the pair kernel stores through its tensor map (rows end on 16 bytes)
  int early_w;         // split kernel: the lanes' operand was complete before the previous kernel
  int* timeouts;       // counts waits that were given up
};

// -------------------------------------------------------- block conversions
// Four e2m1 bytes from eight fp32 values (v[0] in the lowest four bits), to
// nearest even, saturating.
__device__ __forceinline__ uint32_t e2m1x8(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

// Scale byte of a block from the bits of its largest magnitude as fp32 (taken
// as an integer maximum, so that a NaN is not lost in it).
__device__ __forceinline__ uint32_t mx_scale(uint32_t amax_bits) {
  const uint32_t e = amax_bits >> 23;
  return e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
}

// 1 / scale (2^(127 - byte)); for a block without values any finite number.
__device__ __forceinline__ float mx_inv_scale(uint32_t s) {
  return s == 255u ? 1.0f : __uint_as_float((254u - s) << 23);
}

// The codes of one block of 32 values; its scale byte in *scale.
__device__ __forceinline__ uint4 mx_block(const float (&w)[32], uint32_t* scale) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) m = max(m, __float_as_uint(w[i]) & 0x7FFFFFFFu);
  const uint32_t s = mx_scale(m);
  const float inv = mx_inv_scale(s);
  uint32_t q[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = w[i * 8 + k] * inv;
    q[i] = e2m1x8(v);
  }
  *scale = s;
  return make_uint4(q[0], q[1], q[2], q[3]);
}

// ------------------------------------------------------ few rows, split along K
// out^T tiles: 128 rows of B (columns of out) on the TMEM lanes, BN rows of A
// (rows of out) as the N side. With few tiles the GPU would idle and the weight
// stream would be short of loads in flight, so a cluster of up to 8 CTAs shares a
// tile, each taking a part of K; the partial tiles are added in rank order
// through distributed shared memory (the same result in every run).
//
// SRC = 0: A comes as 4-bit codes by TMA. SRC = 1 / 2: A is bf16 / fp32 and each CTA
// rounds its part of K to 4 bits in shared memory while the weights' first
// stages are on their way: a token costs one launch, and no scratch. BN below 128
// takes one tile of A's rows (its scales then start at a block's first row).
//
// Bound by latency at these sizes (operands not in L2): 1 x 8192 x 2048 takes 6.8 us
// (rounded in the kernel: 7.1) where its bytes take 1.4, 48 x 4096 x 4096 8.4 us (1.5),
// 16 x 14336 x 4096 10.8 us (rounded in the kernel: 12.6; 4.9), 333 x 517 x 1030 8 us.
template <int BN, int SRC>
struct MxSplit {
  static constexpr int kABytes = 128 * 128;
  static constexpr int kBBytes = BN * 128;
  static constexpr int kTileBytes = kABytes + (SRC == 0 ? kBBytes : 0);
  static constexpr int kSfBytes = SRC == 0 ? 2048 : 1024;
  static constexpr int kStageBytes = kTileBytes + kSfBytes;
  static constexpr int kStages = 212000 / kStageBytes < 8 ? 212000 / kStageBytes : 8;
  static constexpr int kPairs = SRC == 0 ? 0 : 8;  // pairs of rounded k blocks (SRC != 0)
  static constexpr int kQBytes = 2 * kPairs * (kBBytes + 1024);
  static constexpr int kAccCols = BN < 32 ? 32 : BN;
  static constexpr int kColsUsed = kAccCols + kStages * 16;
  static constexpr int kTmemCols = kColsUsed <= 128 ? 128 : 256;
  static constexpr int kThreads = 64 + 256;
  static constexpr int kSmemBytes = 1024 + kStages * kStageBytes + kQBytes + 512;
  static_assert(kColsUsed <= 256, "TMEM columns");
  static_assert(SRC == 0 || BN == 16, "a thread per block of a pair of k blocks");
  static_assert(kSmemBytes <= 232448, "shared memory per CTA");
  static_assert(kStages * kTileBytes >= BN * 128 * 4, "the partial tile takes the stages' place");
};

struct MxRows {
  const void* x;  // SRC != 0: the rows to round
  long long ld;
  int cols;
  int vec;        // rows are 16-byte aligned
};

// A block of 32 values of a row on its way: bf16 (SRC 1) or fp32 (2) as loaded.
template <int SRC>
struct MxRaw {
  uint4 u[SRC == 2 ? 8 : 4];
  // `have` values exist from (row, col) on; the rest of the block is zero
  __device__ __forceinline__ void load(const MxRows& r, int row, int col, int have) {
    constexpr int kPer = SRC == 2 ? 4 : 8;  // values per 16 bytes
    const char* p = static_cast<const char*>(r.x) + ((long long)row * r.ld + col) * (16 / kPer);
    if (have == 32 && r.vec) {
#pragma unroll
      for (int i = 0; i < 32 / kPer; ++i) u[i] = reinterpret_cast<const uint4*>(p)[i];
    } else {
#pragma unroll
      for (int i = 0; i < 32 / kPer; ++i) {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if constexpr (SRC == 2) {
            w[k] = i * 4 + k < have ? reinterpret_cast<const uint32_t*>(p)[i * 4 + k] : 0u;
          } else {
            const int e = i * 8 + 2 * k;
            const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
            w[k] = (e < have ? (uint32_t)h[e] : 0u) | (e + 1 < have ? (uint32_t)h[e + 1] << 16 : 0u);
          }
        }
        u[i] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
  __device__ __forceinline__ void values(float (&w)[32]) const {
#pragma unroll
    for (int i = 0; i < (SRC == 2 ? 8 : 4); ++i) {
      const uint32_t e[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (SRC == 2) {
          w[i * 4 + k] = __uint_as_float(e[k]);
        } else {
          w[i * 8 + 2 * k] = __uint_as_float(e[k] << 16);
          w[i * 8 + 2 * k + 1] = __uint_as_float(e[k] & 0xFFFF0000u);
        }
      }
    }
  }
};

template <int BN, int SRC>
__global__ void __launch_bounds__(320, 1)
    mx_split_kernel(const __grid_constant__ CUtensorMap tm_w,
                    const __grid_constant__ CUtensorMap tm_x, const MxGemmArgs args,
                    const MxRows rows, int splits) {
  using S = MxSplit<BN, SRC>;
  constexpr int STAGES = S::kStages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* tiles = smem;
  uint8_t* qb = smem + STAGES * S::kTileBytes;    // rounded A: [k block][BN x 128 B], swizzled
  uint8_t* qs = qb + 2 * S::kPairs * S::kBBytes;  // its scales: [k block][1024]
  uint8_t* sfs = qs + 2 * S::kPairs * 1024;
  uint64_t* full = reinterpret_cast<uint64_t*>(sfs + STAGES * S::kSfBytes);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = full + 2 * STAGES;
  uint64_t* bready = tfull + 1;           // a pair of k blocks of A is rounded
  uint64_t* bfree = bready + S::kPairs;   // its MMAs are done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bfree + S::kPairs);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bfree + S::kPairs + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x % splits, tile = blockIdx.x / splits;
  const int tm = tile / args.tiles_n, tn = tile % args.tiles_n;
  const int kb0 = (int)((long long)args.num_kb * rank / splits);
  const int nkb = (int)((long long)args.num_kb * (rank + 1) / splits) - kb0;

  // The loads of a stage: the lanes' operand, then (SRC = 0) the rows.
  auto load_w = [&](int i) {
    const int s = i % STAGES, kb = kb0 + i;
    mbar_arrive_expect_tx(&full[s], S::kStageBytes);
    tma_load_3d(tiles + s * S::kTileBytes, &tm_w, &full[s], kb * 128, tm * 128, 0);
    bulk_load(sfs + s * S::kSfBytes, args.sfa + ((long long)tm * args.ka + kb * 2) * 512, 1024,
              &full[s]);
  };
  auto load_x = [&](int i) {
    const int s = i % STAGES, kb = kb0 + i;
    tma_load_3d(tiles + s * S::kTileBytes + S::kABytes, &tm_x, &full[s], kb * 128, tn * BN, 0);
    bulk_load(sfs + s * S::kSfBytes + 1024,
              args.sfb + ((long long)(tn * BN / 128) * args.ka + kb * 2) * 512, 1024, &full[s]);
  };
  // SRC != 0: a thread rounds one block of 32 of each pair of k blocks (16 rows x 16
  // blocks), its next one already on the way. Pairs go round a ring of kPairs.
  const int et = threadIdx.x - 64, qn = et >> 4, qj = et & 15;
  const int npairs = (nkb + 1) / 2;
  MxRaw<SRC> raw;
  auto fetch = [&](int p) {
    const int row = tn * BN + qn, col = (kb0 + 2 * p) * 256 + qj * 32;
    raw.load(rows, row, col, row < args.N && 2 * p + (qj >> 3) < nkb ? min(32, rows.cols - col) : 0);
  };

  // Launched as a programmatic dependent: barriers and TMEM are set up while the
  // previous kernel ends. Nothing it may have written is read before the wait;
  // early_w says that the lanes' operand is older than it. The first stages are
  // on their way, and the first rows rounded, before the block first meets.
  uint32_t last = 0, issued = 0;  // parity of each stage's last load, stages used
  const int ahead = nkb < STAGES ? nkb : STAGES;
  if (warp == 0) {
    if (elect_one()) {
      tma_prefetch_desc(&tm_w);
      if (SRC == 0) tma_prefetch_desc(&tm_x);
      for (int s = 0; s < STAGES; ++s) {
        mbar_init(&full[s], 1);
        mbar_init(&empty[s], 1);
      }
      mbar_init(tfull, 1);
      for (int p = 0; p < S::kPairs; ++p) {
        mbar_init(&bready[p], 256);
        mbar_init(&bfree[p], 1);
      }
      *abort_flag = 0;
      fence_barrier_init();
      if (!args.early_w) griddep_wait();
      for (int i = 0; i < ahead; ++i) load_w(i);
      if (args.early_w) griddep_wait();
      if (SRC == 0)
        for (int i = 0; i < ahead; ++i) load_x(i);
    }
    __syncwarp();
    issued = (1u << ahead) - 1;
  } else if (warp == 1) {
    tmem_alloc(tmem_slot, S::kTmemCols);
    tmem_relinquish();
  } else {
    griddep_wait();
    if constexpr (SRC != 0) fetch(0);
  }
  griddep_launch_dependents();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    const bool one = elect_one();
    for (int i = ahead; i < nkb; ++i) {
      const int s = i % STAGES;
      const uint32_t ph = (i / STAGES) & 1;
      if (!mbar_wait_warp(&empty[s], ph ^ 1u, abort_flag)) break;
      if (one) {
        load_w(i);
        if (SRC == 0) load_x(i);
      }
      last = (last & ~(1u << s)) | (ph << s);
    }
    // every load lands before the CTA may exit
    for (int s = 0; s < STAGES; ++s)
      if (issued & (1u << s)) {
        const uint64_t t0 = global_timer_ns();
        while (!mbar_try_wait(&full[s], (last >> s) & 1u))
          if (global_timer_ns() - t0 > kWaitLimitNs) {
            *abort_flag = 1;
            break;
          }
      }
  } else if (warp == 1) {
    const bool one = elect_one();
    bool ok = true;
    for (int i = 0; i < nkb; ++i) {
      const int s = i % STAGES;
      if constexpr (SRC != 0) {
        const int p = i >> 1;
        if (!(i & 1) && !mbar_wait_warp(&bready[p % S::kPairs], (p / S::kPairs) & 1, abort_flag)) {
          ok = false;
          break;
        }
      }
      if (!mbar_wait_warp(&full[s], (i / STAGES) & 1, abort_flag)) {
        ok = false;
        break;
      }
      tc_fence_after();
      if (one) {
        const uint32_t t = smem_u32(tiles + s * S::kTileBytes);
        const uint32_t f = smem_u32(sfs + s * S::kSfBytes);
        const int qi = SRC == 0 ? 0 : i % (2 * S::kPairs);
        const uint32_t bt = SRC == 0 ? t + S::kABytes : smem_u32(qb + qi * S::kBBytes);
        const uint32_t bf = SRC == 0 ? f + 1024 : smem_u32(qs + qi * 1024);
        const uint32_t sa = tmem_base + S::kAccCols + s * 16, sb = sa + 8;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          tc_cp_scales(sa + 4 * h, umma_desc_scales(f + 512 * h));
          tc_cp_scales(sb + 4 * h, umma_desc_scales(bf + 512 * h));
        }
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          constexpr uint32_t id0 = umma_idesc_mxf4(128, BN, 0), id1 = umma_idesc_mxf4(128, BN, 1);
          const int h = kk >> 1;
          tc_mma_mxf4(tmem_base, umma_desc_sw128(t + kk * 32, 16, 1024),
                      umma_desc_sw128(bt + kk * 32, 16, 1024), (kk & 1) ? id1 : id0, sa + 4 * h,
                      sb + 4 * h, (i | kk) != 0);
        }
        tc_commit(&empty[s]);
        if (SRC != 0 && (i & 1)) tc_commit(&bfree[(i >> 1) % S::kPairs]);
      }
      __syncwarp();
    }
    if (one) {
      tc_commit(tfull);  // after a time-out too: what was issued ends before TMEM is freed
      if (!ok) {
        const uint64_t t0 = global_timer_ns();
        while (!mbar_try_wait(tfull, 0))
          if (global_timer_ns() - t0 > kWaitLimitNs) break;
      }
    }
    __syncwarp();
  } else {
    if constexpr (SRC != 0) {
      for (int p = 0; p < npairs; ++p) {
        const int slot = p % S::kPairs, q = 2 * slot + (qj >> 3), j = qj & 7;
        if (p >= S::kPairs) mbar_wait(&bfree[slot], (p / S::kPairs - 1) & 1, abort_flag);
        float w[32];
        raw.values(w);
        if (p + 1 < npairs) fetch(p + 1);
        uint32_t sc;
        const uint4 u = mx_block(w, &sc);
        *reinterpret_cast<uint4*>(qb + q * S::kBBytes + qn * 128 + ((j ^ (qn & 7)) << 4)) = u;
        qs[q * 1024 + (j >> 2) * 512 + qn * 16 + (j & 3)] = (uint8_t)sc;
        fence_proxy_async_smem();
        mbar_arrive(&bready[slot]);
      }
    }
    // the partial tile, [row of out][column of out], into the stages' place
    const int sub = warp & 3, half = (warp - 2) >> 2;
    const bool ready = mbar_wait(tfull, 0, abort_flag);
    if (__all_sync(0xffffffffu, ready)) {  // tcgen05.ld is warp-collective
      tc_fence_after();
      float* part = reinterpret_cast<float*>(tiles);
#pragma unroll 1
      for (int ch = half; ch < (BN + 31) / 32; ch += 2) {
        float v[32];
        tmem_ld_32x32b_x32(tmem_base + ((uint32_t)(sub * 32) << 16) + ch * 32, v);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (BN >= 32 || j < BN) part[(ch * 32 + j) * 128 + sub * 32 + lane] = v[j];
      }
      tc_fence_before();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (splits > 1) cluster_sync_all();
  {
    // four consecutive columns of out per thread, the ranks' partials in order
    const uint32_t part = smem_u32(tiles);
    const int total = BN * 32, per = (total + splits - 1) / splits;
    const int e1 = min(total, (rank + 1) * per);
    for (int e = rank * per + threadIdx.x; e < e1; e += 320) {
      const int j = e >> 5, r = (e & 31) * 4;
      const int row = tn * BN + j, col = tm * 128 + r;
      if (row >= args.N || col >= args.M) continue;
      float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (int k = 0; k < splits; ++k) {
        const uint32_t addr = part + (j * 128 + r) * 4;
        const float4 g = splits > 1 ? ld_cluster_f32x4(mapa_shared(addr, k))
                                    : *reinterpret_cast<const float4*>(tiles + (j * 128 + r) * 4);
        f.x += g.x;
        f.y += g.y;
        f.z += g.z;
        f.w += g.w;
      }
      const long long i = (long long)row * args.ld + col;
      const float v[4] = {f.x, f.y, f.z, f.w};
      if (args.vec && col + 4 <= args.M) {
        if (args.out_bf16) {
          uint2* p = reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(args.out) + i);
          float o[4] = {v[0], v[1], v[2], v[3]};
          if (args.accumulate) {
            const uint2 old = *p;
            o[0] += __uint_as_float(old.x << 16);
            o[1] += __uint_as_float(old.x & 0xFFFF0000u);
            o[2] += __uint_as_float(old.y << 16);
            o[3] += __uint_as_float(old.y & 0xFFFF0000u);
          }
          uint2 u;
          *reinterpret_cast<__nv_bfloat162*>(&u.x) = __floats2bfloat162_rn(o[0], o[1]);
          *reinterpret_cast<__nv_bfloat162*>(&u.y) = __floats2bfloat162_rn(o[2], o[3]);
          *p = u;
        } else {
          float4* p = reinterpret_cast<float4*>(static_cast<float*>(args.out) + i);
          if (args.accumulate) {
            const float4 old = *p;
            f.x += old.x;
            f.y += old.y;
            f.z += old.z;
            f.w += old.w;
          }
          *p = f;
        }
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (col + k < args.M) {
            if (args.out_bf16) {
              __nv_bfloat16* p = static_cast<__nv_bfloat16*>(args.out) + i + k;
              *p = __float2bfloat16_rn(args.accumulate ? v[k] + __bfloat162float(*p) : v[k]);
            } else {
              float* p = static_cast<float*>(args.out) + i + k;
              *p = args.accumulate ? *p + v[k] : v[k];
            }
          }
      }
    }
  }
  if (splits > 1) {
    __syncthreads();
    cluster_sync_all();  // every rank has read this one's partial
  }
  if (*abort_flag && threadIdx.x == 0) atomicAdd(args.timeouts, 1);
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, S::kTmemCols);
  }
}

// Writes (or adds) a 32 x 32 block held one row per lane (v[j] = column j) to
// out rows r0.., columns c0.., through the warp's 32 x 33 stage: what cannot go by TMA,
// rows that are not aligned and sums of bf16. 4096 x 14335 x 4095: 119 us bf16, 134
// fp32 (14336: 101 and 117 by TMA; 136 with a bf16 element a lane and a store); added
// to, 176 and 145 (292 and 366 with loads of eight rows before their stores); 14336
// bf16, added to, 125 (161 with a load and a store at a time).
__device__ __forceinline__ void mx_store_block(const MxGemmArgs& a, long long r0, long long c0,
                                               int rows, int cols, const float (&v)[32],
                                               float* tst) {
  const int lane = threadIdx.x & 31;
  if (a.out_bf16 && !a.accumulate) {
    // bf16 rows that start anywhere: each is packed into the words that its memory
    // has (its first element left over where it starts half-way into one), and two rows
    // are stored at a time.
    __nv_bfloat16* const out = static_cast<__nv_bfloat16*>(a.out) + r0 * a.ld + c0;
    const int at = (int)(reinterpret_cast<uintptr_t>(out) >> 1), ld1 = (int)a.ld;
    const int odd = (at + lane * ld1) & 1;
    uint32_t w[17];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const __nv_bfloat162 p = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
      w[j] = *reinterpret_cast<const uint32_t*>(&p);
    }
    w[16] = 0;
    if (odd && lane < rows)
      *reinterpret_cast<uint16_t*>(out + lane * a.ld) = (uint16_t)w[0];
    uint32_t* const ws = reinterpret_cast<uint32_t*>(tst);
#pragma unroll
    for (int j = 0; j < 16; ++j) w[j] = __funnelshift_r(w[j], w[j + 1], 16 * odd);
#pragma unroll
    for (int j = 0; j < 16; j += 4)
      *reinterpret_cast<uint4*>(ws + lane * 20 + j) = make_uint4(w[j], w[j + 1], w[j + 2], w[j + 3]);
    __syncwarp();
    const int h = lane >> 4, j = lane & 15;
    const int o = (at + h * ld1) & 1, c = 2 * j + o;  // (rows two apart start alike)
    __nv_bfloat16* to = out + h * a.ld + c;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint32_t u = ws[(2 * i + h) * 20 + j];
      if (2 * i + h < rows) {
        if (c + 1 < cols)
          *reinterpret_cast<uint32_t*>(to) = u;
        else if (c < cols)
          *reinterpret_cast<uint16_t*>(to) = (uint16_t)u;
      }
      to += 2 * a.ld;
    }
    __syncwarp();
    return;
  }
#pragma unroll
  for (int j = 0; j < 32; ++j) tst[lane * 33 + j] = v[j];
  __syncwarp();
  if (!a.out_bf16) {
    float* to = static_cast<float*>(a.out) + r0 * a.ld + c0 + lane;
    if (a.accumulate) {
      // (one addend per element, so the order is no matter; like TMA's, this addition
      // flushes values below 2^-126 to zero)
#pragma unroll
      for (int r = 0; r < 32; ++r, to += a.ld)
        if (r < rows && lane < cols) atomicAdd(to, tst[r * 33 + lane]);
    } else {
#pragma unroll
      for (int r = 0; r < 32; ++r, to += a.ld)
        if (r < rows && lane < cols) *to = tst[r * 33 + lane];
    }
  } else if (a.vec && cols == 32) {
    const int rs = lane >> 2, c8 = (lane & 3) * 8;
    uint4* const p = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.out) +
                                              (r0 + rs) * a.ld + c0 + c8);
    uint4 old[4];  // all before the first store
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (q * 8 + rs < rows) old[q] = p[q * a.ld];  // (8 rows are ld vectors of 8)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float* f = tst + (q * 8 + rs) * 33 + c8;
      const __nv_bfloat162* o2 = reinterpret_cast<const __nv_bfloat162*>(&old[q]);
      uint4 u;
      __nv_bfloat162* u2 = reinterpret_cast<__nv_bfloat162*>(&u);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        u2[i] = __floats2bfloat162_rn(f[2 * i] + __low2float(o2[i]),
                                      f[2 * i + 1] + __high2float(o2[i]));
      if (q * 8 + rs < rows) p[q * a.ld] = u;
    }
  } else if (lane < cols) {
    // a row per turn, one column per lane; loads of sixteen rows before their stores
    __nv_bfloat16* to = static_cast<__nv_bfloat16*>(a.out) + r0 * a.ld + c0 + lane;
#pragma unroll 1
    for (int r = 0; r < rows; r += 16) {
      __nv_bfloat16 old[16];
#pragma unroll
      for (int k = 0; k < 16; ++k)
        if (r + k < rows) old[k] = to[k * a.ld];
#pragma unroll
      for (int k = 0; k < 16; ++k)
        if (r + k < rows)
          to[k * a.ld] = __float2bfloat16_rn(tst[(r + k) * 33 + lane] + __bfloat162float(old[k]));
      to += 16 * a.ld;
    }
  }
  __syncwarp();
}

// ---------------------------------------------------------------- CTA pairs
// 256 x BN tiles on CTA pairs, persistent: each CTA loads its 128 rows of A and half
// of B's rows, and the scales of its rows of A and of all of B's. TMEM (512
// columns) holds two accumulators and a set of 24 columns of scales per stage (a
// stage that has been loaded again has had its MMAs completed, so its scale
// columns are free too).
//   BN = 192: the accumulators are apart, and no tile's MMAs wait for the epilogue
//             of the one before.
//   BN = 256: they overlap by 120 columns. The epilogue drains the shared columns
//             first and releases them before it stores anything; the wait costs
//             about 1900 clocks a tile, but a stage's operands serve a third more.
// Measured (clocks): a k block 464 and 591, and 2000 and 3100 a tile, for 192 and
// 256; launch_gemm_pair takes the cheaper for the number of waves. What bounds
// them: a stage's operands cross shared memory at nearly its bandwidth (67 KB in
// 512 tensor clocks for 256) and L2 delivers them at 0.85 of the rate measured
// without MMAs; the SM clock settles at 1.65 GHz under the power cap.
template <int BN>
struct MxPair {
  static constexpr int kABytes = 128 * 128;
  static constexpr int kBBytes = BN / 2 * 128;
  static constexpr int kTileBytes = kABytes + kBBytes;
  static constexpr int kSfBytes = 3 * 1024;
  static constexpr int kStageBytes = kTileBytes + kSfBytes;
  static constexpr int kStages = 5;
  static constexpr int kSfCols = 24;
  static constexpr int kSfCol = 512 - kStages * kSfCols;  // first column of the scales
  static constexpr bool kOverlap = 2 * BN > kSfCol;
  static constexpr int kAcc1 = kOverlap ? kSfCol - BN : BN;  // the second accumulator's first column
  static constexpr int kEpiWarps = 8;
  static constexpr int kThreads = 64 + 32 * kEpiWarps;
  static constexpr int kEpiWarpBytes = 4608;  // two 2 KB store boxes, or a 32 x 33 fp32 tile
  static constexpr int kEpiBytes = kEpiWarps * kEpiWarpBytes;
  static constexpr int kSmemBytes = 1024 + kStages * kStageBytes + 512 + kEpiBytes;
  static_assert(BN == 192 || BN == 256, "tile widths");
  static_assert(kEpiWarpBytes >= 32 * 33 * 4 && kEpiWarpBytes % 512 == 0, "epilogue stage");
  static_assert(!kOverlap || BN - kAcc1 <= 128, "the epilogue releases four chunks of 32 first");
  static_assert(kSmemBytes <= 232448, "shared memory per CTA");
};

// Tile order: bands of kBand tile rows, column by column within a band, so that
// the pairs at work share operand tiles in L2.
__device__ __forceinline__ void mx_tile(int tile, int tiles_m, int tiles_n, int& tm, int& tn) {
  constexpr int kBand = 8;
  const int band = tile / (kBand * tiles_n);
  const int h = min(kBand, tiles_m - band * kBand);
  const int r = tile - band * kBand * tiles_n;
  tn = r / h;
  tm = band * kBand + (r - tn * h);
}

// One 32 x 32 block (v[j] = column c0 + j of the lane's row) to out by TMA: rows
// of 64 bytes (all 32 columns in bf16, 16 of fp32) are staged with the 64-byte
// swizzle (conflict-free 16-byte stores) in two buffers that alternate, so a
// store is read out of shared memory while the next is filled. Clipped at the
// matrix edge by the tensor map, whose rows end on 16 bytes. `add` (fp32): added to
// what out holds.
template <bool BF16>
__device__ __forceinline__ void mx_store_tma(const CUtensorMap* map, uint8_t* stage, int c0, int r0,
                                             bool add, const float (&v)[32], int& buf) {
  const int lane = threadIdx.x & 31, sw = (lane >> 1) & 3;
#pragma unroll
  for (int h = 0; h < (BF16 ? 1 : 2); ++h) {
    uint8_t* st = stage + buf * 2048;
    buf ^= 1;
    if (lane == 0) bulk_wait_read_but_one();
    __syncwarp();
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      uint4 u;
      if constexpr (BF16) {
        __nv_bfloat162* u2 = reinterpret_cast<__nv_bfloat162*>(&u);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          u2[i] = __floats2bfloat162_rn(v[c * 8 + 2 * i], v[c * 8 + 2 * i + 1]);
      } else {
        u = make_uint4(__float_as_uint(v[h * 16 + c * 4]), __float_as_uint(v[h * 16 + c * 4 + 1]),
                       __float_as_uint(v[h * 16 + c * 4 + 2]),
                       __float_as_uint(v[h * 16 + c * 4 + 3]));
      }
      *reinterpret_cast<uint4*>(st + lane * 64 + ((c ^ sw) << 4)) = u;
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      if (!BF16 && add)
        tma_add_3d(map, st, c0 + h * 16, r0, 0);
      else
        tma_store_3d(map, st, c0 + h * 16, r0, 0);
      bulk_commit();
    }
  }
}

template <int BN>
__global__ void __launch_bounds__(MxPair<BN>::kThreads, 1)
    mx_gemm_pair_kernel(const __grid_constant__ CUtensorMap tm_a,
                        const __grid_constant__ CUtensorMap tm_b,
                        const __grid_constant__ CUtensorMap tm_sfa,
                        const __grid_constant__ CUtensorMap tm_sfb,
                        const __grid_constant__ CUtensorMap tm_out, const MxGemmArgs args,
                        int tiles_m, int num_tiles) {
  using S = MxPair<BN>;
  constexpr int STAGES = S::kStages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* tiles = smem;
  uint8_t* sfs = smem + STAGES * S::kTileBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(sfs + STAGES * S::kSfBytes);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = full + 2 * STAGES;       // [2] MMA -> epilogue
  uint64_t* tempty = full + 2 * STAGES + 2;  // [2] epilogue -> MMA
  uint64_t* drain = full + 2 * STAGES + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(full + 2 * STAGES + 5);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(full + 2 * STAGES + 6);
  uint8_t* epi = sfs + STAGES * S::kSfBytes + 512;  // 512-byte aligned, as the swizzle needs

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int group = blockIdx.x >> 1, groups = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&tfull[0], 1);
    mbar_init(&tfull[1], 1);
    for (int b = 0; b < 2; ++b)
      mbar_init(&tempty[b], 2 * S::kEpiWarps);  // one lane of every epilogue warp of the pair
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tm_a);
    tma_prefetch_desc(&tm_b);
    tma_prefetch_desc(&tm_sfa);
    tma_prefetch_desc(&tm_sfb);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // the peer's barriers are initialised, both TMEM allocations done
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // Launched as a programmatic dependent: only the setup above overlaps the
  // previous kernel.
  griddep_wait();
  griddep_launch_dependents();

  // The loading and the issuing warp stay converged: all lanes wait, one elected
  // lane issues. (With the waits inside a one-lane branch the scale copies did
  // not overlap the MMAs: 183 instead of 128 clocks per MMA.)
  if (warp == 0) {
    const bool one = elect_one();
    int stage = 0;
    uint32_t phase = 0, issued = 0, last = 0;
    bool ok = true;
    for (int tile = group; ok && tile < num_tiles; tile += groups) {
      int tm, tn;
      mx_tile(tile, tiles_m, args.tiles_n, tm, tn);
      for (int kb = 0; kb < args.num_kb; ++kb) {
        if (!mbar_wait_warp(&empty[stage], phase ^ 1u, abort_flag)) {
          ok = false;
          break;
        }
        if (one) {
          if (leader) mbar_arrive_expect_tx(&full[stage], 2 * S::kStageBytes);
          const uint32_t fb = mapa_shared(smem_u32(&full[stage]), 0);
          uint8_t* t = tiles + stage * S::kTileBytes;
          uint8_t* f = sfs + stage * S::kSfBytes;
          tma_load_3d_pair(t, &tm_a, fb, kb * 128, tm * 256 + (int)rank * 128, 0);
          tma_load_3d_pair(t + S::kABytes, &tm_b, fb, kb * 128, tn * BN + (int)rank * (BN / 2), 0);
          tma_load_3d_pair(f, &tm_sfa, fb, 0, kb, tm * 2 + (int)rank);
          // (two 128-row blocks of scales; an odd tile of 192 starts in the first one's middle)
          tma_load_3d_pair(f + 1024, &tm_sfb, fb, 0, kb, tn * BN / 128);
        }
        issued |= 1u << stage;
        last = (last & ~(1u << stage)) | (phase << stage);
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    // Every load lands before the CTA may exit; the leader's barriers count
    // both CTAs' bytes, and the final cluster barrier holds the peer.
    if (leader)
      for (int s = 0; s < STAGES; ++s)
        if (issued & (1u << s)) {
          const uint64_t t0 = global_timer_ns();
          while (!mbar_try_wait(&full[s], (last >> s) & 1u))
            if (global_timer_ns() - t0 > kWaitLimitNs) {
              *abort_flag = 1;
              break;
            }
        }
  } else if (warp == 1) {
    if (leader) {
      const bool one = elect_one();
      constexpr uint32_t id0 = umma_idesc_mxf4(256, BN, 0),
                         id1 = umma_idesc_mxf4(256, BN, 1);
      int stage = 0, it = 0;  // it: tiles so far
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = group; ok && tile < num_tiles; tile += groups, ++it) {
        // apart: the accumulator's last tile has been read out of TMEM
        if (!S::kOverlap && it > 1 && !mbar_wait_warp(&tempty[it & 1], ((it >> 1) - 1) & 1, abort_flag)) break;
        tc_fence_after();
        const uint32_t acc = tmem_base + (it & 1) * S::kAcc1;
        int tm, tn;
        mx_tile(tile, tiles_m, args.tiles_n, tm, tn);
        // (an odd tile of 192 starts 64 rows, two columns, into its scales)
        const uint32_t sfb_row = BN == 192 && (tn & 1) ? 2 : 0;
        for (int kb = 0; kb < args.num_kb; ++kb) {
          if (!mbar_wait_warp(&full[stage], phase, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t t = smem_u32(tiles + stage * S::kTileBytes);
          const uint32_t f = smem_u32(sfs + stage * S::kSfBytes);
          // [K half][4] for A, [K half][row group][4] for B
          const uint32_t sa = tmem_base + S::kSfCol + stage * S::kSfCols;
          const uint32_t sb = sa + 8;
          if (one) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              tc_cp_scales_pair(sa + 4 * h, umma_desc_scales(f + 512 * h));
              tc_cp_scales_pair(sb + 8 * h, umma_desc_scales(f + 1024 + 512 * h));
              tc_cp_scales_pair(sb + 8 * h + 4, umma_desc_scales(f + 2048 + 512 * h));
            }
          }
          if (S::kOverlap && kb == 0 && it > 0) {
            // the columns that the previous tile's accumulator shares with this one
            __syncwarp();
            if (!mbar_wait_warp(&tempty[0], (it - 1) & 1, abort_flag)) {
              ok = false;
              break;
            }
            tc_fence_after();
          }
          if (one) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
              const int h = kk >> 1;
              tc_mma_mxf4_pair(acc, umma_desc_sw128(t + kk * 32, 16, 1024),
                               umma_desc_sw128(t + S::kABytes + kk * 32, 16, 1024),
                               (kk & 1) ? id1 : id0, sa + 4 * h, sb + 8 * h + sfb_row,
                               (kb | kk) != 0);
            }
            tc_commit_pair_mc(&empty[stage], 0x3);
          }
          __syncwarp();
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        if (one) tc_commit_pair_mc(&tfull[it & 1], 0x3);
        __syncwarp();
      }
      if (one && *abort_flag) {
        // what was issued ends before TMEM is freed
        tc_commit_pair_mc(drain, 0x1);
        const uint64_t t0 = global_timer_ns();
        while (!mbar_try_wait(drain, 0))
          if (global_timer_ns() - t0 > kWaitLimitNs) break;
      }
      __syncwarp();
    }
  } else {
    const int sub = warp & 3, half = (warp - 2) >> 2;
    uint8_t* stg = epi + (warp - 2) * S::kEpiWarpBytes;
    int buf = 0;
    const uint32_t tempty_leader = mapa_shared(smem_u32(tempty), 0);
    int it = 0;
    for (int tile = group; tile < num_tiles; tile += groups, ++it) {
      int tm, tn;
      mx_tile(tile, tiles_m, args.tiles_n, tm, tn);
      const bool ready = mbar_wait(&tfull[it & 1], (it >> 1) & 1, abort_flag);
      if (!__all_sync(0xffffffffu, ready)) break;  // tcgen05.ld is warp-collective
      tc_fence_after();
      const uint32_t acc = tmem_base + ((uint32_t)(sub * 32) << 16) + (it & 1) * S::kAcc1;
      const int m0 = tm * 256 + (int)rank * 128 + sub * 32;
      const int mr = min(32, args.M - m0);
      auto store = [&](int ch, const float (&x)[32]) {
        const int n0 = tn * BN + ch * 32, nr = min(32, args.N - n0);
        if (mr <= 0 || nr <= 0) return;
        if (args.tma_out) {
          if (args.out_bf16)
            mx_store_tma<true>(&tm_out, stg, n0, m0, false, x, buf);
          else
            mx_store_tma<false>(&tm_out, stg, n0, m0, args.accumulate, x, buf);
        } else {
          mx_store_block(args, m0, n0, mr, nr, x, reinterpret_cast<float*>(stg));
        }
      };
      auto release = [&](int b) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(tempty_leader + b * 8);
      };
      if constexpr (S::kOverlap) {
        // The first accumulator shares its last columns with the second, that one
        // its first: the outermost four of the eight 32-column chunks are read
        // first, two a warp, and released.
#pragma unroll 1
        for (int i = 0; i < 4; i += 2) {
          const int o0 = 2 * i + half, o1 = o0 + 2;
          const int ch0 = (it & 1) ? o0 : 7 - o0, ch1 = (it & 1) ? o1 : 7 - o1;
          float v[32], w[32];
          tmem_ld_32x32b_x32(acc + ch0 * 32, v);
          tmem_ld_32x32b_x32(acc + ch1 * 32, w);
          tmem_ld_wait();
          if (i == 0) release(0);
          store(ch0, v);
          store(ch1, w);
        }
      } else {
        constexpr int kChunks = BN / 32 / 2;  // 32-column chunks of a warp
#pragma unroll 1
        for (int i = 0; i < kChunks; ++i) {
          float v[32];
          tmem_ld_32x32b_x32(acc + (half * kChunks + i) * 32, v);
          tmem_ld_wait();
          if (i == kChunks - 1) release(it & 1);
          store(half * kChunks + i, v);
        }
      }
      tc_fence_before();
    }
    if (args.tma_out && lane == 0) bulk_wait_all();  // the stage outlives the stores that read it
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // peer loads landed, remote arrivals done, MMAs retired
  if (*abort_flag && threadIdx.x == 0) atomicAdd(args.timeouts, 1);
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

}  // namespace mmn
