// code2vec_amd — hand-written CDNA4 (gfx950 / MI355X) kernels.
//
// Covers the reference hot-op inventory:
//   K1-K3  fused embedding gather + concat + dropout  (k_gather_concat)
//   K4     MFMA bf16 128x128-tile GEMM w/ tanh epilogue (k_gemm_bt) — the
//          m97 structure from the CDNA4 guide: global_load_lds width-16
//          staging, 16x16x32 bf16 MFMA, 4 waves x (64x64) per block,
//          XCD-aware bijective block swizzle
//   K5-K7  fused masked-softmax attention reduce, fwd+bwd (k_attn_*) —
//          the whole (C,D) context tile for one example stays in LDS
//          (200x384 bf16 = 150 KiB of the 160 KiB/CU)
//   K9     fused large-vocab log-softmax + NLL, fwd+bwd (k_ce_*)
//   K10    dense Adam (TF formulation) + lazy sparse-row Adam for the
//          embedding tables (k_adam_*)
//
// Compute dtype is bf16 with fp32 accumulation; master weights fp32.
// Wavefront size is 64 everywhere (CDNA4), blocks are multiples of 64.

#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>

#include <cstdint>

#include "c2v_device.h"

// ---------------------------------------------------------------------------
// small helpers
// ---------------------------------------------------------------------------

DEVI ushort f2bf(float f) {
  // round-to-nearest-even, NaN-safe enough for our ranges
  union { float f; u32 u; } cvt;
  cvt.f = f;
  u32 u = cvt.u;
  u32 rounded = (u + 0x7FFFu + ((u >> 16) & 1u)) >> 16;
  return (ushort)rounded;
}

DEVI float wave_reduce_sum(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_down(v, off, 64);
  return v;
}

DEVI float wave_reduce_max(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = fmaxf(v, __shfl_down(v, off, 64));
  return v;
}

// ---------------------------------------------------------------------------
// K1-K3: fused gather + concat + dropout
// out (Nrows, 3d) bf16 from two fp32 tables; element (row, off):
//   off <  d   -> tok_table[src[row]][off]
//   off < 2d   -> path_table[path[row]][off-d]
//   else       -> tok_table[tgt[row]][off-2d]
// dropout keep-mask is the splitmix64 counter hash over the flat element
// index (identical to the CPU reference), scaled by 1/keep_prob.
// ---------------------------------------------------------------------------

__global__ void k_gather_concat(
    const float* __restrict__ tok, const float* __restrict__ path,
    const int* __restrict__ src_ids, const int* __restrict__ path_ids,
    const int* __restrict__ tgt_ids, ushort* __restrict__ out,
    int n_rows, int d, float keep_prob, u64 seed_scalar,
    const long* __restrict__ seed_ptr, int apply_dropout) {
  const u64 seed = seed_ptr ? (u64)*seed_ptr : seed_scalar;
  const int slots_per_row = (3 * d) / 8;
  const long total = (long)n_rows * slots_per_row;
  const float inv_keep = 1.0f / keep_prob;
  for (long slot = blockIdx.x * blockDim.x + threadIdx.x; slot < total;
       slot += (long)gridDim.x * blockDim.x) {
    const int row = (int)(slot / slots_per_row);
    const int off = (int)(slot % slots_per_row) * 8;
    const float* base;
    int col;
    if (off < d) {
      base = tok + (long)src_ids[row] * d;
      col = off;
    } else if (off < 2 * d) {
      base = path + (long)path_ids[row] * d;
      col = off - d;
    } else {
      base = tok + (long)tgt_ids[row] * d;
      col = off - 2 * d;
    }
    float4 lo = *reinterpret_cast<const float4*>(base + col);
    float4 hi = *reinterpret_cast<const float4*>(base + col + 4);
    float vals[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    if (apply_dropout) {
      const u64 eidx = (u64)row * (3 * d) + off;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool keep = hash_uniform(seed, eidx + j) < keep_prob;
        vals[j] = keep ? vals[j] * inv_keep : 0.0f;
      }
    }
    ushort outv[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) outv[j] = f2bf(vals[j]);
    *reinterpret_cast<ulonglong2*>(out + (long)row * (3 * d) + off) =
        *reinterpret_cast<ulonglong2*>(outv);
  }
}

// dropout backward: scale d_ctx by the same keep mask (bf16 in/out)
__global__ void k_dropout_bwd(const ushort* __restrict__ g_in,
                              ushort* __restrict__ g_out, long total,
                              float keep_prob, u64 seed_scalar,
                              const long* __restrict__ seed_ptr) {
  const u64 seed = seed_ptr ? (u64)*seed_ptr : seed_scalar;
  const float inv_keep = 1.0f / keep_prob;
  for (long i8 = blockIdx.x * blockDim.x + threadIdx.x; i8 * 8 < total;
       i8 += (long)gridDim.x * blockDim.x) {
    const long e = i8 * 8;
    ulonglong2 packed = *reinterpret_cast<const ulonglong2*>(g_in + e);
    ushort* u = reinterpret_cast<ushort*>(&packed);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const bool keep = hash_uniform(seed, e + j) < keep_prob;
      u[j] = keep ? f2bf(bf2f(u[j]) * inv_keep) : (ushort)0;
    }
    *reinterpret_cast<ulonglong2*>(g_out + e) = packed;
  }
}

// ---------------------------------------------------------------------------
// K4: bf16 MFMA GEMM, C(N,M) = A(N,K) @ Bt(M,K)^T, optional tanh epilogue.
// m97 structure (CDNA4 guide §5): 128x128 tile, BK=32, 256 threads (4 waves,
// 2x2 of 64x64), LDS staging via __builtin_amdgcn_global_load_lds width 16,
// v_mfma_f32_16x16x32_bf16, XCD-aware bijective grid swizzle (m204).
// Ragged N/M handled by clamping staged rows and masking the C-store.
// ---------------------------------------------------------------------------

#define GEMM_BM 128
#define GEMM_BN 128
#define GEMM_BK 32

template <bool TANH, bool DROPOUT = false>
__launch_bounds__(256)
__global__ void k_gemm_bt(const ushort* __restrict__ A,
                          const ushort* __restrict__ Bt,
                          ushort* __restrict__ C, int N, int M, int K,
                          float keep_prob = 1.f, u64 seed_scalar = 0,
                          const long* __restrict__ seed_ptr = nullptr,
                          const long* __restrict__ b_rows = nullptr) {
  // b_rows: optional row-gather on the Bt operand — Bt row r sources table
  // row b_rows[r] (the sampled-softmax candidate GEMM: logits_cand =
  // code @ gather(targets, cand)^T without materializing w_cand)
  const u64 seed = DROPOUT ? (seed_ptr ? (u64)*seed_ptr : seed_scalar) : 0;
  const float inv_keep = DROPOUT ? (1.f / keep_prob) : 1.f;
  __shared__ ushort lds_a[GEMM_BM * GEMM_BK];
  __shared__ ushort lds_b[GEMM_BN * GEMM_BK];

  // XCD-aware bijective swizzle of the (row-tile, col-tile) space
  const int n_tiles = (N + GEMM_BM - 1) / GEMM_BM;
  const int m_tiles = (M + GEMM_BN - 1) / GEMM_BN;
  const int nwg = n_tiles * m_tiles;
  int wg = blockIdx.x;
  {
    const int nxcd = 8;
    const int q = nwg / nxcd, r = nwg % nxcd;
    const int xcd = wg % nxcd, orig = wg / nxcd;
    wg = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + orig;
  }
  const int tile_n = wg / m_tiles;   // row-tile of A
  const int tile_m = wg % m_tiles;   // row-tile of Bt (= col-tile of C)
  const int row0 = tile_n * GEMM_BM;
  const int col0 = tile_m * GEMM_BN;

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wid = tid >> 6;           // 4 waves: 2x2 over (64,64) subtiles
  const int wrow = (wid >> 1) * 64;   // wave's row offset in the tile
  const int wcol = (wid & 1) * 64;    // wave's col offset

  f32x4 acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};

  const int k_steps = K / GEMM_BK;
  for (int ks = 0; ks < k_steps; ++ks) {
    const int k0 = ks * GEMM_BK;
    // ---- stage A and B tiles: each wave issues 2+2 width-16 direct loads.
    // One wave-load covers 1 KiB of LDS = 16 rows x 32 cols bf16; lane i
    // sources row (i>>2), byte-col (i&3)*16 of the 16x64B sub-tile.
    {
      const int sub = wid;                       // wave's 16-row chunk pair
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int r16 = sub * 2 + half;          // 16-row group index (0..7)
        const int lrow = r16 * 16 + (lane >> 2);
        const int kb = (lane & 3) * 8;           // 8 bf16 = 16 B
        {
          const int grow = min(row0 + lrow, N - 1);
          const ushort* gp = A + (long)grow * K + k0 + kb;
          __builtin_amdgcn_global_load_lds(
              (const __attribute__((address_space(1))) u32*)gp,
              (__attribute__((address_space(3))) u32*)(lds_a + r16 * 16 * GEMM_BK),
              16, 0, 0);
        }
        {
          int grow = min(col0 + lrow, M - 1);
          if (b_rows) grow = (int)b_rows[grow];
          const ushort* gp = Bt + (long)grow * K + k0 + kb;
          __builtin_amdgcn_global_load_lds(
              (const __attribute__((address_space(1))) u32*)gp,
              (__attribute__((address_space(3))) u32*)(lds_b + r16 * 16 * GEMM_BK),
              16, 0, 0);
        }
      }
    }
    __syncthreads();

    // ---- fragments + MFMA. a-frag: row (lane&15) of the 16-row block,
    // k = (lane>>4)*8..+8 (contiguous 16 B -> ds_read_b128).
    bf16x8 afrag[4], bfrag[4];
#pragma unroll
    for (int mi = 0; mi < 4; ++mi) {
      const int r = wrow + mi * 16 + (lane & 15);
      afrag[mi] = *reinterpret_cast<const bf16x8*>(
          lds_a + r * GEMM_BK + (lane >> 4) * 8);
    }
#pragma unroll
    for (int ni = 0; ni < 4; ++ni) {
      const int r = wcol + ni * 16 + (lane & 15);
      bfrag[ni] = *reinterpret_cast<const bf16x8*>(
          lds_b + r * GEMM_BK + (lane >> 4) * 8);
    }
#pragma unroll
    for (int mi = 0; mi < 4; ++mi)
#pragma unroll
      for (int ni = 0; ni < 4; ++ni)
        acc[mi][ni] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            afrag[mi], bfrag[ni], acc[mi][ni], 0, 0, 0);
    __syncthreads();
  }

  // ---- epilogue: C/D layout col=lane&15, row=(lane>>4)*4+reg (guide §3)
#pragma unroll
  for (int mi = 0; mi < 4; ++mi) {
#pragma unroll
    for (int ni = 0; ni < 4; ++ni) {
      const int col = col0 + wcol + ni * 16 + (lane & 15);
      if (col >= M) continue;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = row0 + wrow + mi * 16 + (lane >> 4) * 4 + r;
        if (row >= N) continue;
        float v = acc[mi][ni][r];
        if (TANH) v = tanhf(v);
        if (DROPOUT) {
          // fused dropout backward: apply the keep-mask/scale for element
          // (row, col) of the (N, 3d) d_ctx directly in the epilogue
          const bool keep =
              hash_uniform(seed, (u64)row * M + col) < keep_prob;
          v = keep ? v * inv_keep : 0.f;
        }
        C[(long)row * M + col] = f2bf(v);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// K4 v2: 128x128-tile, BK=64, double-buffered (one barrier per k-step,
// bt-kernel pipeline). The single-buffered BK=32 k_gemm_bt pays 2 barriers
// and an exposed staging latency per step — tolerable at java14m's K=384
// for throughput-bound shapes, but the transform GEMMs (K=384 -> only 6
// BK=64 steps) are latency-bound, so prefetching the next tile during
// compute matters. Same epilogue options (TANH / fused dropout mask).
// ---------------------------------------------------------------------------

template <bool TANH, bool DROPOUT = false>
__launch_bounds__(256, 1)
__global__ void k_gemm_bt2(const ushort* __restrict__ A,
                           const ushort* __restrict__ Bt,
                           ushort* __restrict__ C, int N, int M, int K,
                           float keep_prob = 1.f, u64 seed_scalar = 0,
                           const long* __restrict__ seed_ptr = nullptr) {
  const u64 seed = DROPOUT ? (seed_ptr ? (u64)*seed_ptr : seed_scalar) : 0;
  const float inv_keep = DROPOUT ? (1.f / keep_prob) : 1.f;
  // 2 buffers x (A[128][64] + B[128][64]) bf16 = 64 KiB
  extern __shared__ ushort lds2[];
#define L2A(b) (lds2 + (b) * 16384)
#define L2B(b) (lds2 + (b) * 16384 + 8192)

  const int n_tiles = (N + GEMM_BM - 1) / GEMM_BM;
  const int m_tiles = (M + GEMM_BN - 1) / GEMM_BN;
  const int nwg = n_tiles * m_tiles;
  int wg = blockIdx.x;
  {
    const int nxcd = 8;
    const int q = nwg / nxcd, r = nwg % nxcd;
    const int xcd = wg % nxcd, orig = wg / nxcd;
    wg = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + orig;
  }
  const int tile_n = wg / m_tiles;
  const int tile_m = wg % m_tiles;
  const int row0 = tile_n * GEMM_BM;
  const int col0 = tile_m * GEMM_BN;

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wid = tid >> 6;           // 4 waves: 2x2 over (64,64) subtiles
  const int wrow = (wid >> 1) * 64;
  const int wcol = (wid & 1) * 64;

  f32x4 acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};

  // stage one 128x64 tile pair per k-step: 16 KiB per operand, 4 waves x
  // 4 width-16 issues each (one issue = 64 lanes x 16 B = 8 rows of 128 B)
  auto stage = [&](int buf, int ks) {
    const int k0 = ks * 64;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int off = (wid * 4 + q) * 1024 + lane * 16;  // byte in tile
      const int lrow = off >> 7;           // 128 B per row of 64 bf16
      const int lcol = (off & 127) >> 1;
      {
        const int grow = min(row0 + lrow, N - 1);
        const ushort* gp = A + (long)grow * K + k0 + lcol;
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) u32*)gp,
            (__attribute__((address_space(3))) u32*)(L2A(buf) +
                                                     (wid * 4 + q) * 512),
            16, 0, 0);
      }
      {
        const int grow = min(col0 + lrow, M - 1);
        const ushort* gp = Bt + (long)grow * K + k0 + lcol;
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) u32*)gp,
            (__attribute__((address_space(3))) u32*)(L2B(buf) +
                                                     (wid * 4 + q) * 512),
            16, 0, 0);
      }
    }
  };

  const int k_steps = K / 64;
  stage(0, 0);
  __syncthreads();
  int cur = 0;
  for (int ks = 0; ks < k_steps; ++ks) {
    if (ks + 1 < k_steps) stage(cur ^ 1, ks + 1);
    bf16x8 bfrag[4][2];
#pragma unroll
    for (int ni = 0; ni < 4; ++ni)
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const int r = wcol + ni * 16 + (lane & 15);
        bfrag[ni][kk] = *reinterpret_cast<const bf16x8*>(
            L2B(cur) + r * 64 + kk * 32 + (lane >> 4) * 8);
      }
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int mi = 0; mi < 4; ++mi) {
      bf16x8 afrag[2];
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const int r = wrow + mi * 16 + (lane & 15);
        afrag[kk] = *reinterpret_cast<const bf16x8*>(
            L2A(cur) + r * 64 + kk * 32 + (lane >> 4) * 8);
      }
#pragma unroll
      for (int ni = 0; ni < 4; ++ni) {
        acc[mi][ni] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            afrag[0], bfrag[ni][0], acc[mi][ni], 0, 0, 0);
        acc[mi][ni] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            afrag[1], bfrag[ni][1], acc[mi][ni], 0, 0, 0);
      }
    }
    __builtin_amdgcn_s_setprio(0);
    __syncthreads();
    cur ^= 1;
  }

#pragma unroll
  for (int mi = 0; mi < 4; ++mi) {
#pragma unroll
    for (int ni = 0; ni < 4; ++ni) {
      const int col = col0 + wcol + ni * 16 + (lane & 15);
      if (col >= M) continue;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = row0 + wrow + mi * 16 + (lane >> 4) * 4 + r;
        if (row >= N) continue;
        float v = acc[mi][ni][r];
        if (TANH) v = tanhf(v);
        if (DROPOUT) {
          const bool keep =
              hash_uniform(seed, (u64)row * M + col) < keep_prob;
          v = keep ? v * inv_keep : 0.f;
        }
        C[(long)row * M + col] = f2bf(v);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// K4/K8 v2: 256x256-tile bf16 MFMA GEMM (CDNA4 guide §5 template, 2-phase
// double-buffered variant). C(N,M) = A(N,K) @ Bt(M,K)^T.
// 8 waves (512 threads) as 2x4 over (128x64) per-wave outputs; BK=64;
// K-tile staged to LDS via width-16 global_load_lds, double buffered with
// next-tile prefetch issued before the current tile's compute.
// Grid ordering is COLUMN-major with the XCD-bijective swizzle so the blocks
// sharing a Bt panel run on the same XCD back-to-back (Bt streams once per
// XCD from HBM instead of once per row-tile) — that is what makes this
// kernel win on the skinny-N logits shape (N=1024, M=261246).
// ---------------------------------------------------------------------------

#define G256_BM 256
#define G256_BN 256
#define G256_BK 64

// CE_PART: fused CE-forward partials — each (row-tile, col-tile) block also
// emits (rowmax, sumexp) over its 256-col slice into partials[(row)*T+tile_m]
// so the separate 535 MB ce_fwd pass over the logits disappears;
// k_ce_reduce_partials folds the T partials per row into (loss, lse).
template <bool TANH, bool CE_PART = false>
__launch_bounds__(512, 1)
__global__ void k_gemm256_bt(const ushort* __restrict__ A,
                             const ushort* __restrict__ Bt,
                             ushort* __restrict__ C, int N, int M, int K,
                             float* __restrict__ partials = nullptr,
                             int n_col_tiles = 0) {
  // LDS: 2 buffers x (A[256][64] + B[256][64]) bf16 = 128 KiB
  extern __shared__ ushort lds256[];
  // buffer b: A at b*32768, B at b*32768+16384 (ushort units)
#define LDS_A(b) (lds256 + (b) * 32768)
#define LDS_B(b) (lds256 + (b) * 32768 + 16384)

  const int n_tiles = (N + G256_BM - 1) / G256_BM;
  const int m_tiles = (M + G256_BN - 1) / G256_BN;
  const int nwg = n_tiles * m_tiles;
  int wg = blockIdx.x;
  {
    const int nxcd = 8;
    const int q = nwg / nxcd, r = nwg % nxcd;
    const int xcd = wg % nxcd, orig = wg / nxcd;
    wg = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + orig;
  }
  const int tile_m = wg / n_tiles;   // column-major order: Bt panel reuse
  const int tile_n = wg % n_tiles;
  const int row0 = tile_n * G256_BM;
  const int col0 = tile_m * G256_BN;

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wid = tid >> 6;          // 8 waves: 2 (row) x 4 (col)
  const int wrow = (wid >> 2) * 128;
  const int wcol = (wid & 3) * 64;

  f32x4 acc[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};

  // staging: each wave issues 4 width-16 loads for A and 4 for B per K-tile;
  // wave-issue q covers 1 KiB (8 rows of 64 bf16) of the [256][64] tile.
  auto stage = [&](int buf, int ks) {
    const int k0 = ks * G256_BK;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int off = (wid * 4 + q) * 1024 + lane * 16;   // byte in tile
      const int lrow = off >> 7;             // 128 B per row
      const int lcol = (off & 127) >> 1;     // bf16 column
      {
        const int grow = min(row0 + lrow, N - 1);
        const ushort* gp = A + (long)grow * K + k0 + lcol;
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) u32*)gp,
            (__attribute__((address_space(3))) u32*)(LDS_A(buf) + (wid * 4 + q) * 512),
            16, 0, 0);
      }
      {
        const int grow = min(col0 + lrow, M - 1);
        const ushort* gp = Bt + (long)grow * K + k0 + lcol;
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) u32*)gp,
            (__attribute__((address_space(3))) u32*)(LDS_B(buf) + (wid * 4 + q) * 512),
            16, 0, 0);
      }
    }
  };

  const int k_steps = K / G256_BK;
  stage(0, 0);
  __syncthreads();

  int cur = 0;
  for (int ks = 0; ks < k_steps; ++ks) {
    if (ks + 1 < k_steps) stage(cur ^ 1, ks + 1);

    // B fragments for this wave's 64 columns: 4 col-frags x 2 k-frags
    bf16x8 bfrag[4][2];
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const int r = wcol + n * 16 + (lane & 15);
        bfrag[n][kk] = *reinterpret_cast<const bf16x8*>(
            LDS_B(cur) + r * G256_BK + kk * 32 + (lane >> 4) * 8);
      }
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int m = 0; m < 8; ++m) {
      bf16x8 afrag[2];
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const int r = wrow + m * 16 + (lane & 15);
        afrag[kk] = *reinterpret_cast<const bf16x8*>(
            LDS_A(cur) + r * G256_BK + kk * 32 + (lane >> 4) * 8);
      }
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            afrag[0], bfrag[n][0], acc[m][n], 0, 0, 0);
        acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            afrag[1], bfrag[n][1], acc[m][n], 0, 0, 0);
      }
    }
    __builtin_amdgcn_s_setprio(0);
    __syncthreads();
    cur ^= 1;
  }

  // epilogue: C/D layout col=lane&15, row=(lane>>4)*4+reg. The CE variant
  // reduces each row's 64-col slice across its 16-lane group — processed in
  // 4-row-tile HALVES with all 16 shfl chains of a half INTERLEAVED: the
  // original per-(m,r) sequential chains (8 dependent shfls + 4 exps each,
  // 32 chains back-to-back) measured +42% busy / +68% SQ_WAIT over the
  // plain GEMM; batching the chains turns 32 serial latencies into 2.
#pragma unroll
  for (int mh = 0; mh < 2; ++mh) {
    float lmax[4][4], lsum[4][4];
#pragma unroll
    for (int mi = 0; mi < 4; ++mi) {
      const int m = mh * 4 + mi;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = row0 + wrow + m * 16 + (lane >> 4) * 4 + r;
        float lm = -3.0e38f;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const int col = col0 + wcol + n * 16 + (lane & 15);
          float v = acc[m][n][r];
          if (TANH) v = tanhf(v);
          if (col < M && row < N) C[(long)row * M + col] = f2bf(v);
          if (CE_PART && col < M) lm = fmaxf(lm, v);
        }
        lmax[mi][r] = lm;
      }
    }
    if (CE_PART) {
#pragma unroll
      for (int off = 1; off < 16; off <<= 1)
#pragma unroll
        for (int mi = 0; mi < 4; ++mi)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            lmax[mi][r] = fmaxf(lmax[mi][r],
                                __shfl_xor(lmax[mi][r], off, 16));
#pragma unroll
      for (int mi = 0; mi < 4; ++mi)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float ls = 0.f;
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const int col = col0 + wcol + n * 16 + (lane & 15);
            if (col < M)
              ls += __expf(acc[mh * 4 + mi][n][r] - lmax[mi][r]);
          }
          lsum[mi][r] = ls;
        }
#pragma unroll
      for (int off = 1; off < 16; off <<= 1)
#pragma unroll
        for (int mi = 0; mi < 4; ++mi)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            lsum[mi][r] += __shfl_xor(lsum[mi][r], off, 16);
      if ((lane & 15) == 0) {
#pragma unroll
        for (int mi = 0; mi < 4; ++mi)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int row =
                row0 + wrow + (mh * 4 + mi) * 16 + (lane >> 4) * 4 + r;
            if (row >= N) continue;
            // per-wave-column slot: 4 waves cover the 256-col tile, each
            // owns a quarter; (tile, quarter)-major layout so this block's
            // rows land 8 B apart (the row-major layout scattered every
            // store 32 KB apart, one cache line each)
            float* p = partials +
                       2 * (((long)tile_m * 4 + (wid & 3)) * N + row);
            p[0] = lmax[mi][r];
            p[1] = lsum[mi][r];
          }
      }
    }
  }
}

// stage 1: fold the (T, N, 2) partials down to (N, T2, 2) — each thread
// owns one row inside a 256-row block and walks a T-chunk; reads are fully
// coalesced (256 rows x 8 B contiguous per step)
__launch_bounds__(256)
__global__ void k_ce_part_reduce1(const float* __restrict__ partials,
                                  float* __restrict__ out, int N, int T,
                                  int t_chunks) {
  const int row = blockIdx.x * 256 + threadIdx.x;
  const int tc = blockIdx.y;
  if (row >= N) return;
  const int per = (T + t_chunks - 1) / t_chunks;
  const int t0 = tc * per, t1 = min(T, t0 + per);
  float m = -3.0e38f, ssum = 0.f;
  for (int t = t0; t < t1; ++t) {
    const float pm = partials[2 * ((long)t * N + row)];
    const float ps = partials[2 * ((long)t * N + row) + 1];
    if (pm > m) { ssum = ssum * __expf(m - pm) + ps; m = pm; }
    else ssum += ps * __expf(pm - m);
  }
  out[2 * ((long)row * t_chunks + tc)] = m;
  out[2 * ((long)row * t_chunks + tc) + 1] = ssum;
}

// stage 2 (and legacy single-stage path): fold per-(row, chunk) (max,
// sumexp) partials in (N, T, 2) layout into (loss, lse)
__launch_bounds__(256)
__global__ void k_ce_reduce_partials(const float* __restrict__ partials,
                                     const ushort* __restrict__ logits,
                                     const long* __restrict__ labels,
                                     float* __restrict__ loss,
                                     float* __restrict__ lse, int N, int T,
                                     int V) {
  __shared__ float sm[4], ss[4];
  const int row = blockIdx.x;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wid = tid >> 6;
  float m = -3.0e38f, s = 0.f;
  for (int t = tid; t < T; t += blockDim.x) {
    const float pm = partials[2 * ((long)row * T + t)];
    const float psum = partials[2 * ((long)row * T + t) + 1];
    if (pm > m) { s = s * __expf(m - pm) + psum; m = pm; }
    else s += psum * __expf(pm - m);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const float mo = __shfl_down(m, off, 64);
    const float so = __shfl_down(s, off, 64);
    if (mo > m) { s = s * __expf(m - mo) + so; m = mo; }
    else s += so * __expf(mo - m);
  }
  if (lane == 0) { sm[wid] = m; ss[wid] = s; }
  __syncthreads();
  if (tid == 0) {
    float M2 = sm[0], S2 = ss[0];
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      if (sm[w] > M2) { S2 = S2 * __expf(M2 - sm[w]) + ss[w]; M2 = sm[w]; }
      else S2 += ss[w] * __expf(sm[w] - M2);
    }
    const float l = M2 + __logf(S2);
    lse[row] = l;
    loss[row] = l - bf2f(logits[(long)row * V + labels[row]]);
  }
}

// ---------------------------------------------------------------------------
// d_code GEMM (nn operands): C(N,M) = A(N,K) @ B(K,M), A and B ROW-major
// bf16, C fp32. Shaped for dL/dcode = d_logits(B,V) @ target_shadow(V,D):
// N small (batch), M <= 384 (code dim), K huge (vocab) — so the kernel is
// SPLIT-K: the K axis is carved into S chunks, each block accumulates a
// (256 x M) fp32 partial for its chunk, and k_splitk_reduce folds the S
// slices. B fragments need column-major k-runs, so the B tile is staged
// TRANSPOSED into LDS ([col][k], padded stride) from coalesced row-major
// b128 global reads; frag reads are then contiguous b128 like the A side.
// Grid mapping (m204-style): dispatch round-robins blockIdx over the 8 XCDs,
// so we decode (k_chunk, row_tile) such that all row-tiles of one k-chunk
// land on ONE XCD back-to-back — the chunk's B panel (~3 MB) streams from
// HBM once per XCD instead of once per row-tile.
// ---------------------------------------------------------------------------

#define GNN_BM 128
#define GNN_BN 384   // max M (full code dim); cols beyond M are zero-padded
#define GNN_BK 32
// padded LDS strides, chosen for bank spread (32 banks x 4B):
//  A rows stride 36 ushorts (72 B): afrag b64 reads hit 16 distinct bank
//    starts across the 16 lanes of a row group (18*r mod 32 is a bijection
//    on even banks) -> conflict-free;
//  B rows stride 440 ushorts with the row image of k ROTATED right by
//    16*(k/8) cols: b128 stores stay 16 B-aligned and contiguous
//    (conflict-free), and bfrag u16 reads get their four k-groups on
//    disjoint bank quarters via the +16*(k/8) term (bank = 28j + col/2
//    + 8q mod 32) with paired cols sharing a dword (LDS broadcast)
//    -> conflict-free. Two earlier layouts measured worse: a transposed
//    [col][k] tile made the scalar u16 stores 48-way same-bank
//    (SQ_LDS_BANK_CONFLICT ~6x busy cycles, 897 us); an unrotated 386
//    stride fixed the reads but its 4 B stores still hit only 8 banks
//    (conflicts ~1.2x busy, 433 us).
#define GNN_PKA 36
#define GNN_PKB 440
#define GNN_BROT(k) (16 * ((k) >> 3))

// CEB: CE-backward fused into the A staging — A holds LOGITS and each
// staged element becomes d_logit = bf16((exp(l - lse[row]) - onehot)*scale),
// bit-identical to k_ce_bwd's output. CEB=1 keeps d_logits virtual;
// CEB=2 ALSO streams the transformed tiles back to DL (each logits element
// is staged by exactly one block, so coverage is bijective) — that retires
// the separate k_ce_bwd pass (535 MB read + 535 MB write) for the cost of
// one extra 535 MB write here, and d_target's hipBLASLt GEMM still gets a
// materialized d_logits.
template <int CEB = 0>
__launch_bounds__(256, 1)
__global__ void k_gemm_nn_splitk(const ushort* __restrict__ A,
                                 const ushort* __restrict__ B,
                                 float* __restrict__ P,  // (S, N, M) partials
                                 int N, int M, int K, int S,
                                 int ksteps_per_chunk, int row_tiles,
                                 const float* __restrict__ lse = nullptr,
                                 const long* __restrict__ labels = nullptr,
                                 float ce_scale = 1.f,
                                 ushort* __restrict__ DL = nullptr,
                                 const long* __restrict__ b_rows = nullptr) {
  // double-buffered: A[2][128][36] + B[2][32][440] bf16 = 73 KiB dynamic.
  // 256 threads = 4 waves = 1 wave/SIMD: the per-SIMD register pool is 512
  // regs/lane, the only occupancy at which the 192-reg accumulator tile
  // plus staging fits unspilled (the gfx950 compiler does not move MFMA
  // accumulators into the AGPR half of the unified file). Tile-size A/B:
  // BM=32 with 2 blocks/CU amortized per-kstep costs 4x worse (607 us);
  // BM=128 measured 409 us ~= the 2.1 GB HBM bound (B re-read once per
  // row-tile; the XCD-grouped decode lets L2 absorb part of it).
  // Non-temporal A loads / P stores measured worse (449 us) — reverted.
  extern __shared__ ushort ldsnn[];
#define NLDS_A(b) (ldsnn + (b) * (GNN_BM * GNN_PKA))
#define NLDS_B(b) (ldsnn + 2 * GNN_BM * GNN_PKA + (b) * (GNN_BK * GNN_PKB))

  // XCD-aware decode: blocks dispatch round-robin over 8 XCDs, so
  // xcd = bid % 8 and slot = bid / 8 enumerate one XCD's blocks; chunks are
  // dealt to XCDs in groups of row_tiles consecutive slots, so every
  // row-tile of one k-chunk shares that XCD's L2 for the B panel.
  const int bid = blockIdx.x;
  const int xcd = bid & 7;
  const int slot = bid >> 3;
  const int chunk = (slot / row_tiles) * 8 + xcd;
  const int tile_n = slot % row_tiles;
  const int row0 = tile_n * GNN_BM;

  const int total_ksteps = (K + GNN_BK - 1) / GNN_BK;
  const int ks0 = chunk * ksteps_per_chunk;
  const int ks1 = min(total_ksteps, ks0 + ksteps_per_chunk);
  const int ks1_main = min(ks1, K / GNN_BK);  // full 32-k steps only
  // ks0 >= ks1 (empty chunk) still falls through: acc stays zero and the
  // epilogue writes a zero partial slice (the reducer reads every slice)

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wid = tid >> 6;              // 4 waves, one 96-col group each
  const int wcol = wid * 96;

  f32x4 acc[8][6];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 6; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};

  // per-thread staging slices, raw u16 vectors (an arithmetic __bf16 type
  // here would make LDS stores VALUE-convert instead of bit-copy — caught
  // by tools/debug_nn.py: outputs were denormals whose bit patterns equaled
  // the rounded reference values shifted left 16).
  // A tile 128x32 = 512 b128 chunks -> 2/thread; row = idx/4, k8 = idx%4*8
  const int a_row[2] = {(tid + 0) >> 2, (tid + 256) >> 2};
  const int a_k8 = (tid & 3) * 8;
  // B tile 32x384 = 1536 b128 chunks -> 6/thread; krow = idx/48, c8=idx%48*8
  int b_kr[6], b_c8[6];
#pragma unroll
  for (int r = 0; r < 6; ++r) {
    const int idx = tid + r * 256;
    b_kr[r] = idx / 48;
    b_c8[r] = (idx % 48) * 8;
  }

  u16x8 ra[2], rb[6];
  auto ce_map = [&](u16x8 v, int grow, int kbase) -> u16x8 {
    if (CEB == 0) return v;
    const float l = lse[grow];
    const long lab = labels[grow];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float pr = __expf(bf2f(v[j]) - l);
      if (kbase + j == lab) pr -= 1.f;
      v[j] = f2bf(pr * ce_scale);
    }
    return v;
  };
  auto load_ab = [&](int ks) {
    const int k0 = ks * GNN_BK;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int grow = min(row0 + a_row[r], N - 1);
      ra[r] = ce_map(*reinterpret_cast<const u16x8*>(
                         A + (long)grow * K + k0 + a_k8),
                     grow, k0 + a_k8);
      if (CEB == 2 && row0 + a_row[r] < N)
        *reinterpret_cast<u16x8*>(DL + (long)grow * K + k0 + a_k8) = ra[r];
    }
#pragma unroll
    for (int r = 0; r < 6; ++r) {
      long krow = k0 + b_kr[r];
      if (b_rows) krow = b_rows[krow];
      if (b_c8[r] + 8 <= M) {
        rb[r] = *reinterpret_cast<const u16x8*>(
            B + krow * M + b_c8[r]);
      } else {
        const long base = krow * M;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          rb[r][j] = (b_c8[r] + j < M) ? B[base + b_c8[r] + j] : (ushort)0;
      }
    }
  };
  auto store_ab = [&](int buf) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      ushort* p = NLDS_A(buf) + a_row[r] * GNN_PKA + a_k8;
      // 2x b64 (72 B row stride keeps b64 alignment; b128 would misalign
      // on odd rows)
      *reinterpret_cast<u16x4*>(p) =
          u16x4{ra[r][0], ra[r][1], ra[r][2], ra[r][3]};
      *reinterpret_cast<u16x4*>(p + 4) =
          u16x4{ra[r][4], ra[r][5], ra[r][6], ra[r][7]};
    }
#pragma unroll
    for (int r = 0; r < 6; ++r) {
      ushort* p = NLDS_B(buf) + b_kr[r] * GNN_PKB + GNN_BROT(b_kr[r]) +
                  b_c8[r];
      *reinterpret_cast<u16x8*>(p) = rb[r];   // single aligned b128 store
    }
  };

  auto compute = [&](int buf) {
    // bfrag: 8 scalar u16 reads per fragment from the row-major B tile
    // ([k][col], k-stride 386) — the k-groups land on disjoint bank
    // quarters, and paired cols share a dword (LDS broadcast)
    bf16x8 bfrag[6];
#pragma unroll
    for (int n = 0; n < 6; ++n) {
      const int col = wcol + n * 16 + (lane & 15);
      const ushort* bp = NLDS_B(buf) + (lane >> 4) * (8 * GNN_PKB + 16) + col;
      u16x8 t;
#pragma unroll
      for (int j = 0; j < 8; ++j) t[j] = bp[j * GNN_PKB];
      bfrag[n] = __builtin_bit_cast(bf16x8, t);
    }
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int m = 0; m < 8; ++m) {
      const int row = m * 16 + (lane & 15);
      const ushort* ap = NLDS_A(buf) + row * GNN_PKA + (lane >> 4) * 8;
      const u16x4 alo = *reinterpret_cast<const u16x4*>(ap);
      const u16x4 ahi = *reinterpret_cast<const u16x4*>(ap + 4);
      const bf16x8 afrag = __builtin_bit_cast(
          bf16x8, u16x8{alo[0], alo[1], alo[2], alo[3],
                        ahi[0], ahi[1], ahi[2], ahi[3]});
#pragma unroll
      for (int n = 0; n < 6; ++n)
        acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            afrag, bfrag[n], acc[m][n], 0, 0, 0);
    }
    __builtin_amdgcn_s_setprio(0);
  };

  if (ks0 < ks1_main) {
    load_ab(ks0);
    store_ab(0);
    if (ks0 + 1 < ks1_main) load_ab(ks0 + 1);
    __syncthreads();
    for (int ks = ks0; ks < ks1_main; ++ks) {
      const int cur = (ks - ks0) & 1;
      if (ks + 1 < ks1_main) {
        store_ab(cur ^ 1);          // regs loaded one iteration ago
        if (ks + 2 < ks1_main) load_ab(ks + 2);
      }
      compute(cur);
      __syncthreads();
    }
  }

  // partial last k-step (K % 32): cooperative zero-filled manual staging,
  // one guarded iteration outside the hot loop
  if ((K % GNN_BK) && ks1 == total_ksteps && ks0 < ks1) {
    const int k0 = (total_ksteps - 1) * GNN_BK;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int grow = min(row0 + a_row[r], N - 1);
      u16x8 v;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        v[j] = (k0 + a_k8 + j < K) ? A[(long)grow * K + k0 + a_k8 + j]
                                   : (ushort)0;
      if (CEB != 0) {
        const u16x8 m = ce_map(v, grow, k0 + a_k8);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          v[j] = (k0 + a_k8 + j < K) ? m[j] : (ushort)0;
        if (CEB == 2 && row0 + a_row[r] < N) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (k0 + a_k8 + j < K) DL[(long)grow * K + k0 + a_k8 + j] = v[j];
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
        NLDS_A(0)[a_row[r] * GNN_PKA + a_k8 + j] = v[j];
    }
#pragma unroll
    for (int r = 0; r < 6; ++r) {
      const int gk = k0 + b_kr[r];
      const long bk = (gk < K && b_rows) ? b_rows[gk] : gk;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        NLDS_B(0)[b_kr[r] * GNN_PKB + GNN_BROT(b_kr[r]) + b_c8[r] + j] =
            (gk < K && b_c8[r] + j < M) ? B[bk * M + b_c8[r] + j]
                                        : (ushort)0;
    }
    __syncthreads();
    compute(0);
  }

  float* Pc = P + (long)chunk * N * M;
#pragma unroll
  for (int m = 0; m < 8; ++m) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = row0 + m * 16 + (lane >> 4) * 4 + r;
      if (row >= N) continue;
#pragma unroll
      for (int n = 0; n < 6; ++n) {
        const int col = wcol + n * 16 + (lane & 15);
        if (col < M) Pc[(long)row * M + col] = acc[m][n][r];
      }
    }
  }
}

// ---------------------------------------------------------------------------
// d_target GEMM (tn operands): C(V,M) bf16 = A(K,V)^T @ B(K,M), A and B
// ROW-major bf16. Shaped for dL/dtarget = d_logits(B,V)^T @ code(B,M):
// the contraction axis K is the BATCH (small), V is huge -> one block per
// 128-row V-tile (~2041 blocks, no split-K). Neither operand is transposed
// in memory: both tiles stage ROW-major along K with the same rotated
// padded layout as k_gemm_nn_splitk's B tile, and both fragments gather 8
// k-strided u16 scalars (conflict-free: the +16*(k/8) rotation puts the
// four k-groups on disjoint bank quarters). code (K x M, ~768 KB) is read
// by every block and lives in L2; d_logits streams once.
// ---------------------------------------------------------------------------

#define GTN_BV 128   // V rows per block
#define GTN_PKT 184  // padded+rotated stride of the staged d_logits tile

// SPLITK: for tn shapes whose contraction axis is HUGE and output tiny
// (dW = ctx^T @ d_z: K = B*C ~ 205K, out 384x384) — blocks are
// (row-tile, k-chunk) pairs like k_gemm_nn_splitk, accumulate fp32
// partials P[(chunk, V, M)] folded by k_splitk_reduce. C is unused then.
template <bool CEB = false, bool SPLITK = false, int BV = GTN_BV>
__launch_bounds__(4 * BV, 1)
__global__ void k_gemm_tn(const ushort* __restrict__ A,  // d_logits (K, V)
                          const ushort* __restrict__ B,  // code (K, M)
                          ushort* __restrict__ C,        // out (V, M)
                          int V, int M, int K,
                          const float* __restrict__ lse = nullptr,
                          const long* __restrict__ labels = nullptr,
                          float ce_scale = 1.f,
                          float* __restrict__ P = nullptr,
                          int S = 1, int ksteps_per_chunk = 0,
                          int row_tiles = 1) {
  // double-buffered: At[2][32][BV+56] + B[2][32][440] bf16 (78 KiB at
  // BV=128 with one block/CU; 66 KiB at BV=64 with TWO blocks/CU, whose
  // independent barriers overlap each other's load and compute phases)
  extern __shared__ ushort ldstn[];
  constexpr int PKT = BV + 56;          // padded+rotated A-tile stride
  constexpr int TNT = 4 * BV;           // block threads (8 or 4 waves)
  constexpr int NB = 1536 / TNT;        // B-tile b128 chunks per thread
#define TLDS_A(b) (ldstn + (b) * (GNN_BK * PKT))
#define TLDS_B(b) (ldstn + 2 * GNN_BK * PKT + (b) * (GNN_BK * GNN_PKB))

  int v0, chunk = 0, ks0 = 0, ks1;
  const int total_ksteps = (K + GNN_BK - 1) / GNN_BK;
  if (SPLITK) {
    // XCD-aware decode (see k_gemm_nn_splitk)
    const int xcd = blockIdx.x & 7;
    const int slot = blockIdx.x >> 3;
    chunk = (slot / row_tiles) * 8 + xcd;
    v0 = (slot % row_tiles) * BV;
    ks0 = chunk * ksteps_per_chunk;
    ks1 = min(total_ksteps, ks0 + ksteps_per_chunk);
  } else {
    v0 = blockIdx.x * BV;
    ks1 = total_ksteps;
  }
  const int ks1_main = min(ks1, K / GNN_BK);

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wid = tid >> 6;              // 8 waves: 2 (v-rows) x 4 (cols)
  const int wrow = (wid >> 2) * 64;
  const int wcol = (wid & 3) * 96;

  // 512 threads / 64x96 per-wave tile: 96 accumulator regs -> the whole
  // block fits 2 waves/SIMD (the earlier 4-wave/128-row layout needed 192
  // accs and ran 1 wave/SIMD, fully latency-exposed at only 32 k-steps)
  f32x4 acc[4][6];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 6; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};

  // A tile: 32 k-rows x BV v-cols -> 1 b128 chunk/thread
  const int at_kr[1] = {tid / (BV / 8)};
  const int at_c8 = (tid % (BV / 8)) * 8;
  // B tile: 32 k-rows x 384 cols = 1536 b128 chunks -> NB/thread
  int b_kr[NB], b_c8[NB];
#pragma unroll
  for (int r = 0; r < NB; ++r) {
    const int idx = tid + r * TNT;
    b_kr[r] = idx / 48;
    b_c8[r] = (idx % 48) * 8;
  }

  u16x8 ra[1], rb[NB];
  auto ce_map = [&](u16x8 v, int gk, int vbase) -> u16x8 {
    if (!CEB) return v;
    const float l = lse[gk];
    const long lab = labels[gk];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float pr = __expf(bf2f(v[j]) - l);
      if (vbase + j == lab) pr -= 1.f;
      v[j] = f2bf(pr * ce_scale);
    }
    return v;
  };
  auto load_ab = [&](int ks) {
    const int k0 = ks * GNN_BK;
#pragma unroll
    for (int r = 0; r < 1; ++r) {
      const long base = (long)(k0 + at_kr[r]) * V + v0;
      if (v0 + at_c8 + 8 <= V) {
        ra[r] = ce_map(*reinterpret_cast<const u16x8*>(A + base + at_c8),
                       k0 + at_kr[r], v0 + at_c8);
      } else {
        u16x8 v;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          v[j] = (v0 + at_c8 + j < V) ? A[base + at_c8 + j] : (ushort)0;
        const u16x8 m = ce_map(v, k0 + at_kr[r], v0 + at_c8);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          ra[r][j] = (v0 + at_c8 + j < V) ? m[j] : (ushort)0;
      }
    }
#pragma unroll
    for (int r = 0; r < NB; ++r) {
      if (b_c8[r] + 8 <= M) {
        rb[r] = *reinterpret_cast<const u16x8*>(
            B + (long)(k0 + b_kr[r]) * M + b_c8[r]);
      } else {
        const long base = (long)(k0 + b_kr[r]) * M;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          rb[r][j] = (b_c8[r] + j < M) ? B[base + b_c8[r] + j] : (ushort)0;
      }
    }
  };
  auto store_ab = [&](int buf) {
#pragma unroll
    for (int r = 0; r < 1; ++r) {
      ushort* p = TLDS_A(buf) + at_kr[r] * PKT + GNN_BROT(at_kr[r]) +
                  at_c8;
      *reinterpret_cast<u16x8*>(p) = ra[r];  // aligned b128 (368 B stride)
    }
#pragma unroll
    for (int r = 0; r < NB; ++r) {
      ushort* p = TLDS_B(buf) + b_kr[r] * GNN_PKB + GNN_BROT(b_kr[r]) +
                  b_c8[r];
      *reinterpret_cast<u16x8*>(p) = rb[r];
    }
  };

  auto compute = [&](int buf) {
    bf16x8 bfrag[6];
#pragma unroll
    for (int n = 0; n < 6; ++n) {
      const int col = wcol + n * 16 + (lane & 15);
      const ushort* bp = TLDS_B(buf) + (lane >> 4) * (8 * GNN_PKB + 16) + col;
      u16x8 t;
#pragma unroll
      for (int j = 0; j < 8; ++j) t[j] = bp[j * GNN_PKB];
      bfrag[n] = __builtin_bit_cast(bf16x8, t);
    }
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const int row = wrow + m * 16 + (lane & 15);  // v-col inside the tile
      const ushort* ap = TLDS_A(buf) + (lane >> 4) * (8 * PKT + 16) + row;
      u16x8 t;
#pragma unroll
      for (int j = 0; j < 8; ++j) t[j] = ap[j * GTN_PKT];
      const bf16x8 afrag = __builtin_bit_cast(bf16x8, t);
#pragma unroll
      for (int n = 0; n < 6; ++n)
        acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            afrag, bfrag[n], acc[m][n], 0, 0, 0);
    }
    __builtin_amdgcn_s_setprio(0);
  };

  if (ks0 < ks1_main) {
    load_ab(ks0);
    store_ab(0);
    if (ks0 + 1 < ks1_main) load_ab(ks0 + 1);
    __syncthreads();
    for (int ks = ks0; ks < ks1_main; ++ks) {
      const int cur = (ks - ks0) & 1;
      if (ks + 1 < ks1_main) {
        store_ab(cur ^ 1);
        if (ks + 2 < ks1_main) load_ab(ks + 2);
      }
      compute(cur);
      __syncthreads();
    }
  }

  // ragged last rows (K % 32): one zero-filled guarded iteration
  if ((K % GNN_BK) && ks1 == total_ksteps && ks0 < ks1) {
    const int k0 = (total_ksteps - 1) * GNN_BK;
#pragma unroll
    for (int r = 0; r < 1; ++r) {
      const int gk = k0 + at_kr[r];
      u16x8 v;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        v[j] = (gk < K && v0 + at_c8 + j < V)
                   ? A[(long)gk * V + v0 + at_c8 + j] : (ushort)0;
      if (CEB && gk < K) {
        const u16x8 m = ce_map(v, gk, v0 + at_c8);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          v[j] = (v0 + at_c8 + j < V) ? m[j] : (ushort)0;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
        TLDS_A(0)[at_kr[r] * PKT + GNN_BROT(at_kr[r]) + at_c8 + j] = v[j];
    }
#pragma unroll
    for (int r = 0; r < NB; ++r) {
      const int gk = k0 + b_kr[r];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        TLDS_B(0)[b_kr[r] * GNN_PKB + GNN_BROT(b_kr[r]) + b_c8[r] + j] =
            (gk < K && b_c8[r] + j < M) ? B[(long)gk * M + b_c8[r] + j]
                                        : (ushort)0;
    }
    __syncthreads();
    compute(0);
  }

  float* Pc = SPLITK ? P + (long)chunk * V * M : nullptr;
#pragma unroll
  for (int m = 0; m < 4; ++m) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int v = v0 + wrow + m * 16 + (lane >> 4) * 4 + r;
      if (v >= V) continue;
#pragma unroll
      for (int n = 0; n < 6; ++n) {
        const int col = wcol + n * 16 + (lane & 15);
        if (col >= M) continue;
        if (SPLITK) Pc[(long)v * M + col] = acc[m][n][r];
        else C[(long)v * M + col] = f2bf(acc[m][n][r]);
      }
    }
  }
}

// Direct-register tn GEMM: C(V,M) bf16 = A(K,V)^T @ B(K,M), M == 384.
// No LDS, no barriers: both operands are k-major in memory (the transpose
// problem), so instead of staging+transposing tiles through LDS, each lane
// assembles its MFMA fragments with 8 k-strided u16 loads straight from
// global — a wave's 16 consecutive v/col lanes make every load instruction a
// set of 32 B row segments that L1/L2 serve from lines the neighboring
// m/n-tiles complete. Waves run free (register double-buffering only), which
// removes the 32 block-wide barrier pairs that left the staged kernel
// latency-bound at 2 waves/SIMD.
template <bool CEB = false>
__launch_bounds__(512, 1)
__global__ void k_gemm_tn_direct(const ushort* __restrict__ A,
                                 const ushort* __restrict__ B,
                                 ushort* __restrict__ C, int V, int M, int K,
                                 const float* __restrict__ lse = nullptr,
                                 const long* __restrict__ labels = nullptr,
                                 float ce_scale = 1.f) {
  const int v0 = blockIdx.x * 128;
  const int lane = threadIdx.x & 63;
  const int wid = threadIdx.x >> 6;      // 8 waves: 2 (v) x 4 (col)
  const int wrow = (wid >> 2) * 64;
  const int wcol = (wid & 3) * 96;
  const int kg = (lane >> 4) * 8;        // k-offset of this lane's fragment
  const int lr = lane & 15;
  const bool vtail = v0 + 128 > V;

  f32x4 acc[4][6];
#pragma unroll
  for (int m = 0; m < 4; ++m)
#pragma unroll
    for (int n = 0; n < 6; ++n) acc[m][n] = {0.f, 0.f, 0.f, 0.f};

  u16x8 af[2][4], bf[2][6];
  auto ce_map = [&](u16x8 t, int gk0, int v) -> u16x8 {
    if (!CEB) return t;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float pr = __expf(bf2f(t[j]) - lse[gk0 + j]);
      if (v == (int)labels[gk0 + j]) pr -= 1.f;
      t[j] = f2bf(pr * ce_scale);
    }
    return t;
  };
  auto load_step = [&](int ks, int buf) {
    const int k0 = ks * GNN_BK;
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const int v = v0 + wrow + m * 16 + lr;
      const long base = (long)(k0 + kg) * V + v;
      u16x8 t;
      if (!vtail || v < V) {
#pragma unroll
        for (int j = 0; j < 8; ++j) t[j] = A[base + (long)j * V];
        t = ce_map(t, k0 + kg, v);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) t[j] = (ushort)0;
      }
      af[buf][m] = t;
    }
#pragma unroll
    for (int n = 0; n < 6; ++n) {
      const long base = (long)(k0 + kg) * M + wcol + n * 16 + lr;
      u16x8 t;
#pragma unroll
      for (int j = 0; j < 8; ++j) t[j] = B[base + (long)j * M];
      bf[buf][n] = t;
    }
  };
  auto compute = [&](int buf) {
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const bf16x8 afr = __builtin_bit_cast(bf16x8, af[buf][m]);
#pragma unroll
      for (int n = 0; n < 6; ++n)
        acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            afr, __builtin_bit_cast(bf16x8, bf[buf][n]), acc[m][n], 0, 0, 0);
    }
    __builtin_amdgcn_s_setprio(0);
  };

  const int ksteps = K / GNN_BK;
  if (ksteps > 0) {
    load_step(0, 0);
    for (int ks = 0; ks < ksteps; ++ks) {
      const int cur = ks & 1;
      if (ks + 1 < ksteps) load_step(ks + 1, cur ^ 1);
      compute(cur);
    }
  }
  if (K % GNN_BK) {                       // ragged K tail, fully guarded
    const int k0 = ksteps * GNN_BK;
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const int v = v0 + wrow + m * 16 + lr;
      u16x8 t;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        t[j] = (k0 + kg + j < K && v < V) ? A[(long)(k0 + kg + j) * V + v]
                                          : (ushort)0;
      if (CEB && v < V) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (k0 + kg + j >= K) continue;
          float pr = __expf(bf2f(t[j]) - lse[k0 + kg + j]);
          if (v == (int)labels[k0 + kg + j]) pr -= 1.f;
          t[j] = f2bf(pr * ce_scale);
        }
      }
      af[0][m] = t;
    }
#pragma unroll
    for (int n = 0; n < 6; ++n) {
      const int col = wcol + n * 16 + lr;
      u16x8 t;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        t[j] = (k0 + kg + j < K) ? B[(long)(k0 + kg + j) * M + col]
                                 : (ushort)0;
      bf[0][n] = t;
    }
    compute(0);
  }

#pragma unroll
  for (int m = 0; m < 4; ++m) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int v = v0 + wrow + m * 16 + (lane >> 4) * 4 + r;
      if (v >= V) continue;
#pragma unroll
      for (int n = 0; n < 6; ++n) {
        const int col = wcol + n * 16 + lr;
        C[(long)v * M + col] = f2bf(acc[m][n][r]);
      }
    }
  }
}

// fold the S split-K slices: C[i] = sum_s P[s][i] (fp32 out)
__launch_bounds__(256)
__global__ void k_splitk_reduce(const float* __restrict__ P,
                                float* __restrict__ C, int S, long total) {
  for (long i4 = blockIdx.x * blockDim.x + threadIdx.x; i4 * 4 < total;
       i4 += (long)gridDim.x * blockDim.x) {
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    for (int c = 0; c < S; ++c) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(P + c * total + i4 * 4);
      s[0] += v[0]; s[1] += v[1]; s[2] += v[2]; s[3] += v[3];
    }
    *reinterpret_cast<f32x4*>(C + i4 * 4) = s;
  }
}

// elementwise tanh backward: d_z = d_y * (1 - y^2), bf16
__global__ void k_tanh_bwd_mul(const ushort* __restrict__ dy,
                               const ushort* __restrict__ y,
                               ushort* __restrict__ dz, long total) {
  for (long i8 = blockIdx.x * blockDim.x + threadIdx.x; i8 * 8 < total;
       i8 += (long)gridDim.x * blockDim.x) {
    const long e = i8 * 8;
    ulonglong2 pd = *reinterpret_cast<const ulonglong2*>(dy + e);
    ulonglong2 py = *reinterpret_cast<const ulonglong2*>(y + e);
    ushort* ud = reinterpret_cast<ushort*>(&pd);
    ushort* uy = reinterpret_cast<ushort*>(&py);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float yv = bf2f(uy[j]);
      ud[j] = f2bf(bf2f(ud[j]) * (1.0f - yv * yv));
    }
    *reinterpret_cast<ulonglong2*>(dz + e) = pd;
  }
}

// ---------------------------------------------------------------------------
// K5-K7: fused masked-softmax attention (one workgroup per example).
// LDS holds the example's whole (C,D) bf16 tile + the attention vector +
// per-context scores (java14m: 200x384x2B = 150 KiB).
//   scores_c = comb_c . a + log(mask_c);  alpha = softmax_c; code = sum alpha*comb
// All-masked rows produce zeros (reference would NaN).
// ---------------------------------------------------------------------------

// Streaming design (v2): NO whole-tile LDS staging — the 150 KiB tile capped
// occupancy at 1 block/CU and left the kernels 5-7x off the BW floor. LDS
// holds only the per-context scores (C f32) and the D-sized vectors; comb is
// streamed from HBM/L2 with coalesced accesses (contexts row-major: the dot
// pass reads 16 B/lane per context row; the column passes read/write
// thread-per-column so consecutive threads touch consecutive addresses).

extern __shared__ unsigned char smem[];

#define ATTN_THREADS 256

__launch_bounds__(ATTN_THREADS)
__global__ void k_attn_fwd(const ushort* __restrict__ comb,
                           const float* __restrict__ a,
                           const float* __restrict__ mask,
                           float* __restrict__ code,
                           float* __restrict__ alpha_out, int B, int C, int D) {
  float* sc = reinterpret_cast<float*>(smem);  // C f32 scores -> alpha
  const int b = blockIdx.x;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wid = tid >> 6;
  const int n_waves = blockDim.x >> 6;
  const ushort* base = comb + (long)b * C * D;

  // per-lane slice of `a` for the dot pass: lane covers [lane*8, lane*8+8)
  const int d8 = D / 8;  // D % 64 == 0 is checked host-side (so D%8==0)
  float areg[8];
  const bool lane_active = lane < d8;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    areg[j] = lane_active ? a[lane * 8 + j] : 0.f;

  // ---- scores: one context per wave per iteration
  for (int c = wid; c < C; c += n_waves) {
    float dot = 0.f;
    if (lane_active) {
      ulonglong2 packed = *reinterpret_cast<const ulonglong2*>(
          base + (long)c * D + lane * 8);
      const ushort* u = reinterpret_cast<const ushort*>(&packed);
#pragma unroll
      for (int j = 0; j < 8; ++j) dot += bf2f(u[j]) * areg[j];
    }
    dot = wave_reduce_sum(dot);
    if (lane == 0)
      sc[c] = (mask[(long)b * C + c] > 0.f) ? dot : -3.0e38f;
  }
  __syncthreads();

  // ---- softmax over C (single wave; C is at most a few thousand)
  if (wid == 0) {
    float m = -3.0e38f;
    for (int c = lane; c < C; c += 64) m = fmaxf(m, sc[c]);
    m = wave_reduce_max(m);
    m = __shfl(m, 0, 64);
    const bool any_valid = m > -1.0e38f;
    float s = 0.f;
    for (int c = lane; c < C; c += 64) {
      const float e = (any_valid && sc[c] > -1.0e38f) ? __expf(sc[c] - m) : 0.f;
      sc[c] = e;
      s += e;
    }
    s = wave_reduce_sum(s);
    s = __shfl(s, 0, 64);
    const float inv = (s > 0.f) ? 1.0f / s : 0.f;
    for (int c = lane; c < C; c += 64) {
      sc[c] *= inv;
      alpha_out[(long)b * C + c] = sc[c];
    }
  }
  __syncthreads();

  // ---- weighted sum, vectorized: thread owns an 8-col octet x a C-slice
  // (b128 row loads; per-element u16 was issue-bound); slices combine in
  // LDS behind the sc scratch
  float* acc_sh = sc + C;
  for (int col = tid; col < D; col += blockDim.x) acc_sh[col] = 0.f;
  __syncthreads();
  {
    const int octets = D >> 3;
    const int slices = min(8, (int)blockDim.x / octets);
    const int oct = tid % octets;
    const int slice = tid / octets;
    if (slice < slices) {
      const int per = (C + slices - 1) / slices;
      const int c0 = slice * per, c1 = min(C, c0 + per);
      const int col0 = oct * 8;
      float acc8[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) acc8[j] = 0.f;
      for (int c = c0; c < c1; ++c) {
        const float w = sc[c];
        ulonglong2 packed = *reinterpret_cast<const ulonglong2*>(
            base + (long)c * D + col0);
        const ushort* u = reinterpret_cast<const ushort*>(&packed);
#pragma unroll
        for (int j = 0; j < 8; ++j) acc8[j] += w * bf2f(u[j]);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (slices > 1) atomicAdd(acc_sh + col0 + j, acc8[j]);
        else acc_sh[col0 + j] = acc8[j];
    }
  }
  __syncthreads();
  for (int col = tid; col < D; col += blockDim.x)
    code[(long)b * D + col] = acc_sh[col];
}

__launch_bounds__(ATTN_THREADS)
__global__ void k_attn_bwd(const ushort* __restrict__ comb,
                           const float* __restrict__ a,
                           const float* __restrict__ alpha,
                           const float* __restrict__ d_code,
                           ushort* __restrict__ d_comb,
                           float* __restrict__ d_a_partial,  // (grid,D)
                           int B, int C, int D, int fuse_tanh_bwd) {
  float* dal = reinterpret_cast<float*>(smem);  // C f32: d_alpha then d_e
  __shared__ float s_inner;
  const int b = blockIdx.x;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wid = tid >> 6;
  const int n_waves = blockDim.x >> 6;
  const ushort* base = comb + (long)b * C * D;
  const float* alpha_row = alpha + (long)b * C;

  const int d8 = D / 8;
  const bool lane_active = lane < d8;
  float dvreg[8];
#pragma unroll
  for (int j = 0; j < 8; ++j)
    dvreg[j] = lane_active ? d_code[(long)b * D + lane * 8 + j] : 0.f;

  // ---- d_alpha_c = comb_c . dv
  for (int c = wid; c < C; c += n_waves) {
    float dot = 0.f;
    if (lane_active) {
      ulonglong2 packed = *reinterpret_cast<const ulonglong2*>(
          base + (long)c * D + lane * 8);
      const ushort* u = reinterpret_cast<const ushort*>(&packed);
#pragma unroll
      for (int j = 0; j < 8; ++j) dot += bf2f(u[j]) * dvreg[j];
    }
    dot = wave_reduce_sum(dot);
    if (lane == 0) dal[c] = dot;
  }
  __syncthreads();

  // ---- inner = sum alpha*d_alpha ; d_e_c = alpha_c (d_alpha_c - inner)
  if (wid == 0) {
    float inner = 0.f;
    for (int c = lane; c < C; c += 64) inner += alpha_row[c] * dal[c];
    inner = wave_reduce_sum(inner);
    if (lane == 0) s_inner = inner;
  }
  __syncthreads();
  const float inner = s_inner;
  for (int c = tid; c < C; c += blockDim.x)
    dal[c] = alpha_row[c] * (dal[c] - inner);
  __syncthreads();

  // ---- column pass, vectorized: thread owns an 8-col octet x a C-slice;
  // b128 row loads/stores replace the earlier per-element u16 accesses
  // (the scalar version was VALU/issue-bound at ~2.6x the BW floor).
  //   d_comb[c,col] = alpha_c*dv[col] + d_e_c*a[col]
  //   d_a[col]     += sum_c d_e_c * comb[c,col]   (LDS-accumulated)
  float* da_sh = dal + C;          // D floats after the d_e scratch
  for (int col = tid; col < D; col += blockDim.x) da_sh[col] = 0.f;
  __syncthreads();
  const int octets = D >> 3;
  const int slices = min(8, (int)blockDim.x / octets);
  const int oct = tid % octets;
  const int slice = tid / octets;
  if (slice < slices) {
    const int per = (C + slices - 1) / slices;
    const int c0 = slice * per, c1 = min(C, c0 + per);
    const int col0 = oct * 8;
    float av8[8], dv8[8], da8[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      av8[j] = a[col0 + j];
      dv8[j] = d_code[(long)b * D + col0 + j];
      da8[j] = 0.f;
    }
    for (int c = c0; c < c1; ++c) {
      const float de = dal[c];
      const float al = alpha_row[c];
      ulonglong2 packed = *reinterpret_cast<const ulonglong2*>(
          base + (long)c * D + col0);
      ushort* u = reinterpret_cast<ushort*>(&packed);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float y = bf2f(u[j]);
        da8[j] += de * y;
        float g = al * dv8[j] + de * av8[j];
        // fused tanh backward: comb = tanh(z) is already in hand, so emit
        // dL/dz = dL/dcomb * (1 - comb^2) directly (kills the separate
        // 157 MB tanh_bwd_mul pass)
        if (fuse_tanh_bwd) g *= (1.f - y * y);
        u[j] = f2bf(g);
      }
      *reinterpret_cast<ulonglong2*>(
          d_comb + (long)b * C * D + (long)c * D + col0) = packed;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (slices > 1) atomicAdd(da_sh + col0 + j, da8[j]);
      else da_sh[col0 + j] = da8[j];
  }
  __syncthreads();
  for (int col = tid; col < D; col += blockDim.x)
    d_a_partial[(long)blockIdx.x * D + col] = da_sh[col];
}

// ---------------------------------------------------------------------------
// K9: fused CE over the target vocab. One workgroup per row.
// fwd: online max/sum-exp -> (loss, lse). bwd: d = scale*(softmax - onehot).
// ---------------------------------------------------------------------------

__launch_bounds__(256)
__global__ void k_ce_fwd(const ushort* __restrict__ logits,
                         const long* __restrict__ labels,
                         float* __restrict__ loss, float* __restrict__ lse,
                         int B, int V) {
  __shared__ float sm[4], ss[4];
  const int b = blockIdx.x;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wid = tid >> 6;
  const ushort* row = logits + (long)b * V;

  float m = -3.0e38f, s = 0.f;
  const int v8 = V / 8;
  for (int i = tid; i < v8; i += blockDim.x) {
    ulonglong2 packed = *reinterpret_cast<const ulonglong2*>(row + (long)i * 8);
    const ushort* u = reinterpret_cast<const ushort*>(&packed);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float x = bf2f(u[j]);
      if (x > m) { s = s * __expf(m - x) + 1.f; m = x; }
      else s += __expf(x - m);
    }
  }
  for (int i = v8 * 8 + tid; i < V; i += blockDim.x) {
    const float x = bf2f(row[i]);
    if (x > m) { s = s * __expf(m - x) + 1.f; m = x; }
    else s += __expf(x - m);
  }
  // reduce (m, s) across lanes then waves
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const float mo = __shfl_down(m, off, 64);
    const float so = __shfl_down(s, off, 64);
    if (mo > m) { s = s * __expf(m - mo) + so; m = mo; }
    else s += so * __expf(mo - m);
  }
  if (lane == 0) { sm[wid] = m; ss[wid] = s; }
  __syncthreads();
  if (tid == 0) {
    float M = sm[0], S = ss[0];
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      if (sm[w] > M) { S = S * __expf(M - sm[w]) + ss[w]; M = sm[w]; }
      else S += ss[w] * __expf(sm[w] - M);
    }
    const float l = M + __logf(S);
    lse[b] = l;
    loss[b] = l - bf2f(row[labels[b]]);
  }
}

__global__ void k_ce_bwd(const ushort* __restrict__ logits,
                         const float* __restrict__ lse,
                         const long* __restrict__ labels,
                         ushort* __restrict__ d_logits, float scale, int B,
                         int V) {
  const int b = blockIdx.y;
  const float l = lse[b];
  const long lab = labels[b];
  const ushort* row = logits + (long)b * V;
  ushort* drow = d_logits + (long)b * V;
  // 32 B per iteration (2x b128): more loads in flight per thread
  const int v16 = V / 16;
  for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < v16;
       i += gridDim.x * blockDim.x) {
    const long e0 = (long)i * 16;
    ulonglong2 pk0 = *reinterpret_cast<const ulonglong2*>(row + e0);
    ulonglong2 pk1 = *reinterpret_cast<const ulonglong2*>(row + e0 + 8);
    ushort* u0 = reinterpret_cast<ushort*>(&pk0);
    ushort* u1 = reinterpret_cast<ushort*>(&pk1);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float p0 = __expf(bf2f(u0[j]) - l);
      float p1 = __expf(bf2f(u1[j]) - l);
      if (e0 + j == lab) p0 -= 1.f;
      if (e0 + 8 + j == lab) p1 -= 1.f;
      u0[j] = f2bf(p0 * scale);
      u1[j] = f2bf(p1 * scale);
    }
    *reinterpret_cast<ulonglong2*>(drow + e0) = pk0;
    *reinterpret_cast<ulonglong2*>(drow + e0 + 8) = pk1;
  }
  if (blockIdx.x == 0 && threadIdx.x < (V - v16 * 16)) {
    const long e = (long)v16 * 16 + threadIdx.x;
    float p = __expf(bf2f(row[e]) - l);
    if (e == lab) p -= 1.f;
    drow[e] = f2bf(p * scale);
  }
}

// ---------------------------------------------------------------------------
// Sampled softmax CE (training-time). Candidate logits
// L (B, T=B+S): column b is row b's true class, columns B.. are S shared
// log-uniform negatives. Effective per-row set: {L[b,b]-corr_true[b]} ∪
// {L[b,B+j]-corr_samp[j] | sampled[j] != labels[b]} (accidental hits masked).
// ---------------------------------------------------------------------------

// log-uniform sampling correction log(S*q(id)) computed inline instead of
// via ~12 torch elementwise launches/step: q = log((id+2)/(id+1))/log(V+1),
// so log(S*q) = log(s_over_logv1 * log((id+2)/(id+1))) with
// s_over_logv1 = S/log(V+1) precomputed on the host.
__device__ __forceinline__ float lu_corr(long id, float s_over_logv1) {
  return __logf(s_over_logv1 *
                __logf(((float)id + 2.f) / ((float)id + 1.f)));
}

__launch_bounds__(256)
__global__ void k_sampled_ce_fwd(const ushort* __restrict__ L,
                                 const long* __restrict__ labels,
                                 const long* __restrict__ sampled,
                                 float s_over_logv1,
                                 float* __restrict__ loss,
                                 float* __restrict__ lse_out, int B, int S) {
  __shared__ float sm[4], ss[4];
  const int b = blockIdx.x;
  const int T = B + S;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wid = tid >> 6;
  const ushort* row = L + (long)b * T;
  const long lab = labels[b];
  const float z0 = bf2f(row[b]) - lu_corr(lab, s_over_logv1);

  float m = z0, s = 1.f;  // thread 0's stream starts with z0; others -inf
  if (tid != 0) { m = -3.0e38f; s = 0.f; }
  for (int j = tid; j < S; j += blockDim.x) {
    if (sampled[j] == lab) continue;
    const float x = bf2f(row[B + j]) - lu_corr(sampled[j], s_over_logv1);
    if (x > m) { s = s * __expf(m - x) + 1.f; m = x; }
    else s += __expf(x - m);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const float mo = __shfl_down(m, off, 64);
    const float so = __shfl_down(s, off, 64);
    if (mo > m) { s = s * __expf(m - mo) + so; m = mo; }
    else s += so * __expf(mo - m);
  }
  if (lane == 0) { sm[wid] = m; ss[wid] = s; }
  __syncthreads();
  if (tid == 0) {
    float M = sm[0], Ssum = ss[0];
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      if (sm[w] > M) { Ssum = Ssum * __expf(M - sm[w]) + ss[w]; M = sm[w]; }
      else Ssum += ss[w] * __expf(sm[w] - M);
    }
    const float l = M + __logf(Ssum);
    lse_out[b] = l;
    loss[b] = l - z0;
  }
}

__global__ void k_sampled_ce_bwd(const ushort* __restrict__ L,
                                 const long* __restrict__ labels,
                                 const long* __restrict__ sampled,
                                 float s_over_logv1,
                                 const float* __restrict__ lse,
                                 ushort* __restrict__ dL, float scale, int B,
                                 int S) {
  const int b = blockIdx.y;
  const int T = B + S;
  const long lab = labels[b];
  const float l = lse[b];
  const ushort* row = L + (long)b * T;
  ushort* drow = dL + (long)b * T;
  for (int j = blockIdx.x * blockDim.x + threadIdx.x; j < S;
       j += gridDim.x * blockDim.x) {
    float p = 0.f;
    if (sampled[j] != lab)
      p = __expf(bf2f(row[B + j]) - lu_corr(sampled[j], s_over_logv1) - l);
    drow[B + j] = f2bf(p * scale);
  }
  if (blockIdx.x == 0) {
    // the B true-label columns: zero except this row's own (column b)
    for (int j = threadIdx.x; j < B; j += blockDim.x) drow[j] = f2bf(0.f);
    __syncthreads();
    if (threadIdx.x == 0) {
      const float z0 = bf2f(row[b]) - lu_corr(lab, s_over_logv1);
      drow[b] = f2bf((__expf(z0 - l) - 1.f) * scale);
    }
  }
}

// ---------------------------------------------------------------------------
// K10: Adam, TF AdamOptimizer formulation:
//   m <- b1*m + (1-b1)*g ; v <- b2*v + (1-b2)*g^2
//   lr_t = lr*sqrt(1-b2^t)/(1-b1^t) ; p -= lr_t * m/(sqrt(v)+eps)
// Dense kernel optionally refreshes a bf16 shadow. Sparse path: atomic
// row-accumulate into a compact fp32 buffer (dedup'd ids), then per-row
// lazy update of p/m/v.
// ---------------------------------------------------------------------------

// One-thread fusion of the Adam bias-correction scalar chain
// lr_t = lr*sqrt(1-b2^t)/(1-b1^t): the torch version is ~7 elementwise
// launches on 1-element tensors per step inside the captured graph
// (~35 us of serialized ~5 us dispatches in the steady-state trace).
template <typename T>
__global__ void k_adam_lrt(const T* __restrict__ step_t,
                           float* __restrict__ out, float lr, float log_b1,
                           float log_b2) {
  const float t = (float)*step_t;
  out[0] = lr * sqrtf(1.f - __expf(t * log_b2)) / (1.f - __expf(t * log_b1));
}

template <typename G, bool NT = false>
__global__ void k_adam_dense(float* __restrict__ p, const G* __restrict__ g,
                             float* __restrict__ m, float* __restrict__ v,
                             ushort* __restrict__ shadow, long n, float lr_t,
                             float b1, float b2, float eps,
                             const float* __restrict__ lrt_ptr) {
  if (lrt_ptr) lr_t = *lrt_ptr;
  // vectorized x4 main body (p/m/v as float4, g as bf16x4 or float4)
  const long n4 = n / 4;
  for (long i4 = blockIdx.x * blockDim.x + threadIdx.x; i4 < n4;
       i4 += (long)gridDim.x * blockDim.x) {
    const long i = i4 * 4;
    float4 pv = *reinterpret_cast<float4*>(p + i);
    float4 mv = *reinterpret_cast<float4*>(m + i);
    float4 vv = *reinterpret_cast<float4*>(v + i);
    float gv[4];
    if constexpr (sizeof(G) == 2) {
      ulonglong1 packed = *reinterpret_cast<const ulonglong1*>((const ushort*)g + i);
      const ushort* u = reinterpret_cast<const ushort*>(&packed);
#pragma unroll
      for (int j = 0; j < 4; ++j) gv[j] = bf2f(u[j]);
    } else {
      float4 gf = *reinterpret_cast<const float4*>((const float*)g + i);
      gv[0] = gf.x; gv[1] = gf.y; gv[2] = gf.z; gv[3] = gf.w;
    }
    float* pp = &pv.x; float* mp = &mv.x; float* vp = &vv.x;
    ushort sh[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float mi = b1 * mp[j] + (1.f - b1) * gv[j];
      const float vi = b2 * vp[j] + (1.f - b2) * gv[j] * gv[j];
      mp[j] = mi; vp[j] = vi;
      const float pn = pp[j] - lr_t * mi / (sqrtf(vi) + eps);
      pp[j] = pn;
      sh[j] = f2bf(pn);
    }
    if (NT) {
      // streaming stores: p/m/v/shadow are not re-read in this kernel and
      // the tables far exceed L2 — keep them out of the caches.
      // (ext_vector types: HIP_vector_type isn't accepted by the builtin)
      using f32x4v = __attribute__((ext_vector_type(4))) float;
      __builtin_nontemporal_store(*reinterpret_cast<f32x4v*>(&pv),
                                  reinterpret_cast<f32x4v*>(p + i));
      __builtin_nontemporal_store(*reinterpret_cast<f32x4v*>(&mv),
                                  reinterpret_cast<f32x4v*>(m + i));
      __builtin_nontemporal_store(*reinterpret_cast<f32x4v*>(&vv),
                                  reinterpret_cast<f32x4v*>(v + i));
      if (shadow != nullptr)
        __builtin_nontemporal_store(*reinterpret_cast<unsigned long long*>(sh),
                                    reinterpret_cast<unsigned long long*>(shadow + i));
    } else {
      *reinterpret_cast<float4*>(p + i) = pv;
      *reinterpret_cast<float4*>(m + i) = mv;
      *reinterpret_cast<float4*>(v + i) = vv;
      if (shadow != nullptr)
        *reinterpret_cast<ulonglong1*>(shadow + i) =
            *reinterpret_cast<ulonglong1*>(sh);
    }
  }
  // scalar tail
  for (long i = n4 * 4 + blockIdx.x * blockDim.x + threadIdx.x; i < n;
       i += (long)gridDim.x * blockDim.x) {
    float gv;
    if constexpr (sizeof(G) == 2) gv = bf2f(((const ushort*)g)[i]);
    else gv = ((const float*)g)[i];
    const float mi = b1 * m[i] + (1.f - b1) * gv;
    const float vi = b2 * v[i] + (1.f - b2) * gv * gv;
    m[i] = mi;
    v[i] = vi;
    const float pv = p[i] - lr_t * mi / (sqrtf(vi) + eps);
    p[i] = pv;
    if (shadow != nullptr) shadow[i] = f2bf(pv);
  }
}

// Width-2 dense Adam: each thread owns two lane-contiguous float4 chunks per
// iteration with all 8 loads issued before any compute — doubles the
// outstanding-miss count per wave to cover the p/m/v read->write turnaround
// that keeps the width-1 kernel under the streaming floor.
template <typename G, bool NT = false>
__global__ void k_adam_dense_w2(float* __restrict__ p, const G* __restrict__ g,
                                float* __restrict__ m, float* __restrict__ v,
                                ushort* __restrict__ shadow, long n, float lr_t,
                                float b1, float b2, float eps,
                                const float* __restrict__ lrt_ptr) {
  if (lrt_ptr) lr_t = *lrt_ptr;
  const long n4 = n / 4;
  using f32x4v = __attribute__((ext_vector_type(4))) float;
  for (long base = (long)blockIdx.x * blockDim.x * 2; base < n4;
       base += (long)gridDim.x * blockDim.x * 2) {
    long i4s[2];
    float4 pv[2], mv[2], vv[2];
    float gv[2][4];
    bool live[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const long i4 = base + w * blockDim.x + threadIdx.x;
      i4s[w] = i4;
      live[w] = i4 < n4;
      if (!live[w]) continue;
      const long i = i4 * 4;
      pv[w] = *reinterpret_cast<float4*>(p + i);
      mv[w] = *reinterpret_cast<float4*>(m + i);
      vv[w] = *reinterpret_cast<float4*>(v + i);
      if constexpr (sizeof(G) == 2) {
        ulonglong1 packed =
            *reinterpret_cast<const ulonglong1*>((const ushort*)g + i);
        const ushort* u = reinterpret_cast<const ushort*>(&packed);
#pragma unroll
        for (int j = 0; j < 4; ++j) gv[w][j] = bf2f(u[j]);
      } else {
        float4 gf = *reinterpret_cast<const float4*>((const float*)g + i);
        gv[w][0] = gf.x; gv[w][1] = gf.y; gv[w][2] = gf.z; gv[w][3] = gf.w;
      }
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      if (!live[w]) continue;
      const long i = i4s[w] * 4;
      float* pp = &pv[w].x; float* mp = &mv[w].x; float* vp = &vv[w].x;
      ushort sh[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float mi = b1 * mp[j] + (1.f - b1) * gv[w][j];
        const float vi = b2 * vp[j] + (1.f - b2) * gv[w][j] * gv[w][j];
        mp[j] = mi; vp[j] = vi;
        const float pn = pp[j] - lr_t * mi / (sqrtf(vi) + eps);
        pp[j] = pn;
        sh[j] = f2bf(pn);
      }
      if (NT) {
        __builtin_nontemporal_store(*reinterpret_cast<f32x4v*>(&pv[w]),
                                    reinterpret_cast<f32x4v*>(p + i));
        __builtin_nontemporal_store(*reinterpret_cast<f32x4v*>(&mv[w]),
                                    reinterpret_cast<f32x4v*>(m + i));
        __builtin_nontemporal_store(*reinterpret_cast<f32x4v*>(&vv[w]),
                                    reinterpret_cast<f32x4v*>(v + i));
        if (shadow != nullptr)
          __builtin_nontemporal_store(
              *reinterpret_cast<unsigned long long*>(sh),
              reinterpret_cast<unsigned long long*>(shadow + i));
      } else {
        *reinterpret_cast<float4*>(p + i) = pv[w];
        *reinterpret_cast<float4*>(m + i) = mv[w];
        *reinterpret_cast<float4*>(v + i) = vv[w];
        if (shadow != nullptr)
          *reinterpret_cast<ulonglong1*>(shadow + i) =
              *reinterpret_cast<ulonglong1*>(sh);
      }
    }
  }
  // scalar tail
  for (long i = n4 * 4 + blockIdx.x * blockDim.x + threadIdx.x; i < n;
       i += (long)gridDim.x * blockDim.x) {
    float gvs;
    if constexpr (sizeof(G) == 2) gvs = bf2f(((const ushort*)g)[i]);
    else gvs = ((const float*)g)[i];
    const float mi = b1 * m[i] + (1.f - b1) * gvs;
    const float vi = b2 * v[i] + (1.f - b2) * gvs * gvs;
    m[i] = mi;
    v[i] = vi;
    const float pvs = p[i] - lr_t * mi / (sqrtf(vi) + eps);
    p[i] = pvs;
    if (shadow != nullptr) shadow[i] = f2bf(pvs);
  }
}

// Hash-based id dedup (replaces sort-based torch.unique on the sparse-Adam
// path): open-addressing table with atomicCAS claims; a claiming thread takes
// a compact index from a global counter, so inverse mapping and unique list
// come out of one pass with no sort and no host sync.
// Three spin-free passes (an intra-wave publish/spin pair can deadlock under
// the exec-mask divergence model, so claim / compact / lookup are separate
// kernel launches with the stream as the barrier):
//   1. claim: CAS the id into its probe slot
//   2. compact: every occupied slot takes a compact index
//   3. lookup: every input id re-probes and reads its compact index
// Hot-id replica accumulation: ids whose occurrence count crosses HOT_T get
// HOT_R replica accumulator rows; contributions spread across replicas by
// wave id and a fold pass sums them back. Without this, a Zipf-frequent id
// (top java14m token ≈ 9% of a batch) serializes ~39K same-address fp32
// atomics per column — measured 2.2 ms/step at Zipf s=1.1 vs 0.46 ms on
// uniform ids. With replicas the worst per-address chain drops HOT_R-fold.
#define HOT_T 48       // occurrences before an id is treated as hot
#define HOT_R 64       // replica rows per hot id
#define HOT_CAP 2048   // max tracked hot ids (beyond: plain atomics)
#define INV_SINGLE (1 << 30)
#define INV_HOT (1 << 29)
#define INV_IDX 0x1FFFFFFF

template <typename I>
__global__ void k_hash_claim(const I* __restrict__ ids, long n,
                             int* __restrict__ tbl_id, u32 mask_,
                             int* __restrict__ cnt = nullptr) {
  const int lane = threadIdx.x & 63;
  for (long i = blockIdx.x * blockDim.x + threadIdx.x; i < n;
       i += (long)gridDim.x * blockDim.x) {
    const int id = (int)ids[i];
    // run-length wave dedup: duplicate ids are typically CONTIGUOUS in the
    // grad-row stream (the PAD id is ~30% of a batch as row suffixes);
    // without this, hundreds of thousands of threads burst-CAS one address
    // (measured 2.3 ms/step). Lane L-1 is active whenever L is (i grows
    // with lane), so the shuffle is safe at the tail.
    const int prev = __shfl_up(id, 1, 64);
    const bool cont = (lane > 0 && prev == id);
    // occurrence counts: drive the accum single-store fast path (cnt==1)
    // and hot-id detection (cnt>=HOT_T); each run leader adds its run length
    const unsigned long long cmask = __ballot(cont);
    if (cont) continue;                    // leader of each run claims
    int run_len = 1;
    if (cnt) {
      const unsigned long long rest =
          (lane < 63) ? ~(cmask >> (lane + 1)) : ~0ull;
      run_len = 1 + (rest ? __builtin_ctzll(rest) : 64);
    }
    u32 slot = ((u32)id * 2654435761u) & mask_;
    for (;;) {
      const int cur = tbl_id[slot];
      if (cur == id) break;
      if (cur == -1) {
        const int seen = atomicCAS(&tbl_id[slot], -1, id);
        if (seen == -1 || seen == id) break;
      }
      slot = (slot + 1) & mask_;
    }
    if (cnt) {
      // saturating count: adds stop once the hot threshold is reached
      // (read-before-add — an UNCONDITIONAL atomicAdd serialized 136K
      // same-address adds when a hot id appeared as many short runs:
      // 6.2 ms on the 33%-interleaved PAD micro-bench); races may
      // overshoot HOT_T, which only matters as ">= HOT_T". Above the
      // exactness range (1 vs 2+ drives the single-store path) only every
      // 8th leader adds, x8 — cuts the launch-burst same-address adds on a
      // Zipf-hot id 8x while still crossing HOT_T in expectation.
      const int c = cnt[slot];
      if (c < 4) {
        atomicAdd(cnt + slot, run_len);
      } else if (c < HOT_T && ((u32)i & 31u) == 0u) {
        // 1/32 sampling x32: a Zipf-hot id's ~39K leaders would otherwise
        // serialize on this one address; ids with >=~2*32 occurrences still
        // cross HOT_T in expectation, and ids in the 48..64 gray zone that
        // miss the samples just stay on the plain atomic path (bounded by
        // their own occurrence count)
        atomicAdd(cnt + slot, 32 * run_len);
      }
    }
  }
}

__global__ void k_hash_compact(const int* __restrict__ tbl_id,
                               int* __restrict__ tbl_cidx,
                               long* __restrict__ uniq_out,
                               int* __restrict__ n_uniq, u32 cap,
                               const int* __restrict__ occ_cnt = nullptr,
                               int* __restrict__ tbl_hot = nullptr,
                               int* __restrict__ hot2cidx = nullptr,
                               int* __restrict__ n_hot = nullptr) {
  // block-aggregated counter: ballots per wave, one atomicAdd per BLOCK per
  // sweep (a per-wave atomic still serialized ~32K same-address adds/step)
  __shared__ int wave_cnt[4];
  __shared__ int block_base;
  const int lane = threadIdx.x & 63;
  const int wid = threadIdx.x >> 6;
  for (u32 s0 = blockIdx.x * blockDim.x; s0 < cap;
       s0 += gridDim.x * blockDim.x) {
    const u32 s = s0 + threadIdx.x;
    const int id = (s < cap) ? tbl_id[s] : -1;
    const bool occ = id != -1;
    const unsigned long long ball = __ballot(occ);
    const int cnt = __popcll(ball);
    if (lane == 0) wave_cnt[wid] = cnt;
    __syncthreads();
    if (threadIdx.x == 0) {
      const int total = wave_cnt[0] + wave_cnt[1] + wave_cnt[2] + wave_cnt[3];
      block_base = total ? atomicAdd(n_uniq, total) : 0;
    }
    __syncthreads();
    if (occ) {
      int wave_base = block_base;
      for (int w = 0; w < wid; ++w) wave_base += wave_cnt[w];
      const int off = wave_base + __popcll(ball & ((1ull << lane) - 1ull));
      tbl_cidx[s] = off;
      uniq_out[off] = id;
      if (tbl_hot) {
        int h = -1;
        if (occ_cnt[s] >= HOT_T) {
          h = atomicAdd(n_hot, 1);
          if (h < HOT_CAP) hot2cidx[h] = off;
          else h = -1;  // replica table full: plain atomics fallback
        }
        tbl_hot[s] = h;
      }
    }
    __syncthreads();
  }
}

template <typename I>
__global__ void k_hash_lookup(const I* __restrict__ ids, long n,
                              const int* __restrict__ tbl_id,
                              const int* __restrict__ tbl_cidx,
                              int* __restrict__ inverse_out, u32 mask_,
                              const int* __restrict__ cnt = nullptr,
                              const int* __restrict__ tbl_hot = nullptr) {
  for (long i = blockIdx.x * blockDim.x + threadIdx.x; i < n;
       i += (long)gridDim.x * blockDim.x) {
    const int id = (int)ids[i];
    u32 slot = ((u32)id * 2654435761u) & mask_;
    while (tbl_id[slot] != id) slot = (slot + 1) & mask_;
    // bit 30 marks single-occurrence ids (accum stores without atomics);
    // bit 29 marks hot ids (accum spreads over HOT_R replica rows, payload
    // is the hot index)
    int inv = tbl_cidx[slot];
    if (cnt && cnt[slot] == 1) inv |= INV_SINGLE;
    else if (tbl_hot && tbl_hot[slot] >= 0) inv = tbl_hot[slot] | INV_HOT;
    inverse_out[i] = inv;
  }
}

// fold the HOT_R replica rows of each hot id back into its compact acc row
__global__ void k_hot_fold(const float* __restrict__ hot_acc,
                           const int* __restrict__ hot2cidx,
                           const int* __restrict__ n_hot_ptr,
                           float* __restrict__ acc, int d) {
  const int n_hot = min(*n_hot_ptr, HOT_CAP);
  for (long s = blockIdx.x * blockDim.x + threadIdx.x; s < (long)n_hot * d;
       s += (long)gridDim.x * blockDim.x) {
    const int h = (int)(s / d);
    const int col = (int)(s % d);
    float sum = 0.f;
    const float* base = hot_acc + ((long)h * HOT_R) * d + col;
#pragma unroll 4
    for (int r = 0; r < HOT_R; ++r) sum += base[(long)r * d];
    acc[(long)hot2cidx[h] * d + col] += sum;
  }
}

// One-launch init of the hash-build workspace: [-1 x n_neg | 0 x rest].
// Replaces the five torch fills (tbl_id/tbl_cidx full(-1), tbl_cnt/n_hot/
// n_uniq zeros) that cost ~15 launches/step across the three builds.
__global__ void k_hash_ws_init(int* __restrict__ ws, long n_neg, long n_tot) {
  const long n4 = n_neg / 4;
  for (long i4 = blockIdx.x * blockDim.x + threadIdx.x; i4 < n4;
       i4 += (long)gridDim.x * blockDim.x)
    *reinterpret_cast<int4*>(ws + i4 * 4) = int4{-1, -1, -1, -1};
  for (long i = n4 * 4 + blockIdx.x * blockDim.x + threadIdx.x; i < n_neg;
       i += (long)gridDim.x * blockDim.x)
    ws[i] = -1;
  for (long i = n_neg + blockIdx.x * blockDim.x + threadIdx.x; i < n_tot;
       i += (long)gridDim.x * blockDim.x)
    ws[i] = 0;
}

__global__ void k_zero_rows_dyn(float* __restrict__ acc,
                                const int* __restrict__ n_uniq_ptr, int d,
                                int max_rows = 0x7FFFFFFF) {
  // max_rows clamps a counter that may overshoot its buffer (the hot-id
  // counter keeps atomicAdd-ing past HOT_CAP when the table is full)
  const long total = (long)min(*n_uniq_ptr, max_rows) * d;
  const long n4 = total / 4;
  for (long i4 = blockIdx.x * blockDim.x + threadIdx.x; i4 < n4;
       i4 += (long)gridDim.x * blockDim.x)
    *reinterpret_cast<float4*>(acc + i4 * 4) = float4{0.f, 0.f, 0.f, 0.f};
  for (long i = n4 * 4 + blockIdx.x * blockDim.x + threadIdx.x; i < total;
       i += (long)gridDim.x * blockDim.x)
    acc[i] = 0.f;
}

// dynamic-count variant of k_adam_rows: row count read from device memory
// (no host sync on the dedup result)
__global__ void k_adam_rows_dyn(float* __restrict__ p,
                                const long* __restrict__ ids,
                                const float* __restrict__ acc,
                                float* __restrict__ m, float* __restrict__ v,
                                ushort* __restrict__ shadow,
                                const int* __restrict__ n_uniq_ptr, int d,
                                float lr_t, float b1, float b2, float eps,
                                const float* __restrict__ lrt_ptr) {
  const long n_uniq = *n_uniq_ptr;
  if (lrt_ptr) lr_t = *lrt_ptr;
  for (long s = blockIdx.x * blockDim.x + threadIdx.x; s < n_uniq * d;
       s += (long)gridDim.x * blockDim.x) {
    const long u = s / d;
    const int col = (int)(s % d);
    const long off = ids[u] * d + col;
    const float gv = acc[s];
    const float mi = b1 * m[off] + (1.f - b1) * gv;
    const float vi = b2 * v[off] + (1.f - b2) * gv * gv;
    m[off] = mi;
    v[off] = vi;
    const float pv = p[off] - lr_t * mi / (sqrtf(vi) + eps);
    p[off] = pv;
    if (shadow != nullptr) shadow[off] = f2bf(pv);
  }
}

// accumulate token grads straight from the (N,3d) d_ctx layout: logical row
// i < n_per_seg reads d_ctx[i][off0..off0+d); i >= n_per_seg reads
// d_ctx[i-n][off1..) — avoids materializing the 105 MB torch.cat of the
// source/target slices every step
__global__ void k_rows_accum_ctx(const ushort* __restrict__ d_ctx, int ld,
                                 int off0, int off1, long n_per_seg,
                                 int n_seg, const int* __restrict__ inverse,
                                 float* __restrict__ acc, int d,
                                 float* __restrict__ hot_acc = nullptr) {
  const long total = n_per_seg * n_seg * (long)d;
  const int wave = (int)((blockIdx.x * blockDim.x + threadIdx.x) >> 6);
  for (long s = blockIdx.x * blockDim.x + threadIdx.x; s < total;
       s += (long)gridDim.x * blockDim.x) {
    const long r = s / d;
    const int col = (int)(s % d);
    const long src_row = (r < n_per_seg) ? r : r - n_per_seg;
    const int src_off = (r < n_per_seg) ? off0 : off1;
    const float gv = bf2f(d_ctx[src_row * ld + src_off + col]);
    const int inv = inverse[r];
    if (inv & INV_SINGLE) {
      // single-occurrence id (~86% of unique rows on uniform ids): plain
      // store — global atomicAdd throughput was the kernel's bound
      acc[(long)(inv & INV_IDX) * d + col] = gv;
    } else if (gv == 0.f) {
      // masked-context grads are exactly zero: skip the atomic
    } else if (hot_acc && (inv & INV_HOT)) {
      const long h = inv & INV_IDX;
      atomicAdd(hot_acc + (h * HOT_R + (wave & (HOT_R - 1))) * d + col, gv);
    } else {
      atomicAdd(acc + (long)(inv & INV_IDX) * d + col, gv);
    }
  }
}

template <typename G>
__global__ void k_rows_accum(const G* __restrict__ rows,
                             const int* __restrict__ inverse,
                             float* __restrict__ acc, long n_rows, int d,
                             float* __restrict__ hot_acc = nullptr) {
  const int wave = (int)((blockIdx.x * blockDim.x + threadIdx.x) >> 6);
  for (long s = blockIdx.x * blockDim.x + threadIdx.x; s < n_rows * d;
       s += (long)gridDim.x * blockDim.x) {
    const long r = s / d;
    const int col = (int)(s % d);
    float gv;
    if constexpr (sizeof(G) == 2) gv = bf2f(((const ushort*)rows)[s]);
    else gv = ((const float*)rows)[s];
    const int inv = inverse[r];
    if (inv & INV_SINGLE) {
      acc[(long)(inv & INV_IDX) * d + col] = gv;
    } else if (gv == 0.f) {
    } else if (hot_acc && (inv & INV_HOT)) {
      const long h = inv & INV_IDX;
      atomicAdd(hot_acc + (h * HOT_R + (wave & (HOT_R - 1))) * d + col, gv);
    } else {
      atomicAdd(acc + (long)(inv & INV_IDX) * d + col, gv);
    }
  }
}

__global__ void k_adam_rows(float* __restrict__ p, const long* __restrict__ ids,
                            const float* __restrict__ acc, float* __restrict__ m,
                            float* __restrict__ v, ushort* __restrict__ shadow,
                            long n_uniq, int d, float lr_t, float b1, float b2,
                            float eps) {
  for (long s = blockIdx.x * blockDim.x + threadIdx.x; s < n_uniq * d;
       s += (long)gridDim.x * blockDim.x) {
    const long u = s / d;
    const int col = (int)(s % d);
    const long off = ids[u] * d + col;
    const float gv = acc[s];
    const float mi = b1 * m[off] + (1.f - b1) * gv;
    const float vi = b2 * v[off] + (1.f - b2) * gv * gv;
    m[off] = mi;
    v[off] = vi;
    const float pv = p[off] - lr_t * mi / (sqrtf(vi) + eps);
    p[off] = pv;
    if (shadow != nullptr) shadow[off] = f2bf(pv);
  }
}

// ---------------------------------------------------------------------------
// K11: per-row top-k over the target vocabulary (k <= 32).
// One workgroup per row: each thread keeps a sorted local top-k of its
// strided slice in registers, candidates go to LDS, then wave 0 does k
// max-scan passes over the 256*k candidates. Ties resolve to the lower index.
// ---------------------------------------------------------------------------

__launch_bounds__(256)
__global__ void k_topk(const ushort* __restrict__ logits,
                       float* __restrict__ out_vals,
                       long* __restrict__ out_idx, int V, int K) {
  extern __shared__ unsigned char smem_raw[];
  float* cand_v = reinterpret_cast<float*>(smem_raw);          // 256*K
  int* cand_i = reinterpret_cast<int*>(cand_v + blockDim.x * K);

  const int b = blockIdx.x;
  const int tid = threadIdx.x;
  const ushort* row = logits + (long)b * V;

  float lv[32];
  int li[32];
#pragma unroll
  for (int j = 0; j < 32; ++j) { lv[j] = -3.0e38f; li[j] = 0x7FFFFFFF; }

  for (int c = tid; c < V; c += blockDim.x) {
    const float x = bf2f(row[c]);
    if (x > lv[K - 1] || (x == lv[K - 1] && c < li[K - 1])) {
      // insertion into the sorted (desc, then idx asc) local list
      int pos = K - 1;
      while (pos > 0 && (x > lv[pos - 1] ||
                         (x == lv[pos - 1] && c < li[pos - 1]))) {
        lv[pos] = lv[pos - 1];
        li[pos] = li[pos - 1];
        --pos;
      }
      lv[pos] = x;
      li[pos] = c;
    }
  }
  for (int j = 0; j < K; ++j) {
    cand_v[tid * K + j] = lv[j];
    cand_i[tid * K + j] = li[j];
  }
  __syncthreads();

  // k selection passes; all threads participate so __syncthreads is legal.
  __shared__ float red_v[4];
  __shared__ int red_i[4], red_s[4];
  const int n_cand = blockDim.x * K;
  const int lane = tid & 63;
  const int wid = tid >> 6;
  for (int sel = 0; sel < K; ++sel) {
    float m = -3.0e38f;
    int mi = 0x7FFFFFFF;
    int mslot = -1;
    for (int s = tid; s < n_cand; s += blockDim.x) {
      const float x = cand_v[s];
      const int ci = cand_i[s];
      if (x > m || (x == m && ci < mi)) { m = x; mi = ci; mslot = s; }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      const float mo = __shfl_down(m, off, 64);
      const int io = __shfl_down(mi, off, 64);
      const int so = __shfl_down(mslot, off, 64);
      if (mo > m || (mo == m && io < mi)) { m = mo; mi = io; mslot = so; }
    }
    if (lane == 0) { red_v[wid] = m; red_i[wid] = mi; red_s[wid] = mslot; }
    __syncthreads();
    if (tid == 0) {
      float M = red_v[0]; int Mi = red_i[0]; int Ms = red_s[0];
#pragma unroll
      for (int w = 1; w < 4; ++w)
        if (red_v[w] > M || (red_v[w] == M && red_i[w] < Mi)) {
          M = red_v[w]; Mi = red_i[w]; Ms = red_s[w];
        }
      out_vals[(long)b * K + sel] = M;
      out_idx[(long)b * K + sel] = Mi;
      if (Ms >= 0) cand_v[Ms] = -3.0e38f;
    }
    __syncthreads();
  }
}

// ===========================================================================
// host wrappers
// ===========================================================================

namespace {

inline hipStream_t cur_stream() {
  return at::cuda::getCurrentCUDAStream().stream();
}

inline int grid_1d(long total, int block, int cap = 2048) {
  long g = (total + block - 1) / block;
  if (g < 1) g = 1;  // zero-sized work still needs a valid launch config
  return (int)std::min<long>(g, cap);
}

#define CHECK_DEV(t) TORCH_CHECK((t).is_cuda(), #t " must be on GPU")
#define CHECK_CONT(t) TORCH_CHECK((t).is_contiguous(), #t " must be contiguous")

const ushort* bf_ptr(const torch::Tensor& t) {
  return reinterpret_cast<const ushort*>(t.data_ptr<at::BFloat16>());
}
ushort* bf_ptr_mut(torch::Tensor& t) {
  return reinterpret_cast<ushort*>(t.data_ptr<at::BFloat16>());
}

torch::Tensor gather_concat_fwd(torch::Tensor tok, torch::Tensor path,
                                torch::Tensor src, torch::Tensor pth,
                                torch::Tensor tgt, double keep_prob,
                                int64_t seed, bool training,
                                torch::Tensor seed_t) {
  const long* seed_ptr = (seed_t.defined() && seed_t.numel() == 1)
                             ? seed_t.data_ptr<long>() : nullptr;
  CHECK_DEV(tok); CHECK_CONT(tok); CHECK_DEV(path); CHECK_CONT(path);
  CHECK_DEV(src); CHECK_CONT(src);
  TORCH_CHECK(src.scalar_type() == torch::kInt32, "ids must be int32");
  const int d = tok.size(1);
  TORCH_CHECK(d % 8 == 0, "embedding dim must be a multiple of 8");
  const long n_rows = src.numel();
  auto out = torch::empty({n_rows, 3 * (long)d},
                          tok.options().dtype(torch::kBFloat16));
  const bool drop = training && keep_prob < 1.0;
  const long slots = n_rows * (3 * d / 8);
  k_gather_concat<<<grid_1d(slots, 256), 256, 0, cur_stream()>>>(
      tok.data_ptr<float>(), path.data_ptr<float>(), src.data_ptr<int>(),
      pth.data_ptr<int>(), tgt.data_ptr<int>(), bf_ptr_mut(out), (int)n_rows,
      d, (float)keep_prob, (u64)seed, seed_ptr, drop ? 1 : 0);
  return out;
}

torch::Tensor gather_concat_bwd(torch::Tensor d_ctx, double keep_prob,
                                int64_t seed, bool training,
                                torch::Tensor seed_t) {
  CHECK_DEV(d_ctx); CHECK_CONT(d_ctx);
  if (!(training && keep_prob < 1.0)) return d_ctx;
  const long* seed_ptr = (seed_t.defined() && seed_t.numel() == 1)
                             ? seed_t.data_ptr<long>() : nullptr;
  auto out = torch::empty_like(d_ctx);
  const long total = d_ctx.numel();
  TORCH_CHECK(total % 8 == 0);
  k_dropout_bwd<<<grid_1d(total / 8, 256), 256, 0, cur_stream()>>>(
      bf_ptr(d_ctx), bf_ptr_mut(out), total, (float)keep_prob, (u64)seed,
      seed_ptr);
  return out;
}

torch::Tensor gemm_bt(torch::Tensor A, torch::Tensor Bt, bool tanh_epilogue,
                      int variant) {
  CHECK_DEV(A); CHECK_CONT(A); CHECK_DEV(Bt); CHECK_CONT(Bt);
  TORCH_CHECK(A.scalar_type() == torch::kBFloat16 &&
              Bt.scalar_type() == torch::kBFloat16);
  const int N = A.size(0), K = A.size(1), M = Bt.size(0);
  TORCH_CHECK(Bt.size(1) == K, "K mismatch");

  // variant: 0 = auto, 1 = 128x128/BK32 single-buffered,
  // 2 = 256x256/BK64, 3 = 128x128/BK64 double-buffered (K%64==0)
  bool use256 = false;
  if (variant == 2) use256 = true;
  else if (variant == 0)
    use256 = (K % G256_BK == 0) && ((long)N * M >= 4L * 1024 * 1024) &&
             N >= G256_BM;
  if (use256) {
    TORCH_CHECK(K % G256_BK == 0, "256-tile variant needs K%64==0");
  } else if (variant == 3) {
    TORCH_CHECK(K % 64 == 0, "bt2 variant needs K%64==0");
  } else {
    TORCH_CHECK(K % GEMM_BK == 0, "K must be a multiple of 32");
  }

  auto C = torch::empty({N, M}, A.options());
  if (use256) {
    const int n_tiles = (N + G256_BM - 1) / G256_BM;
    const int m_tiles = (M + G256_BN - 1) / G256_BN;
    dim3 grid(n_tiles * m_tiles);
    const size_t lds = 4 * 16384 * 2;  // 128 KiB
    static bool lds_configured = false;
    if (!lds_configured) {
      (void)hipFuncSetAttribute((const void*)k_gemm256_bt<true>,
                                hipFuncAttributeMaxDynamicSharedMemorySize,
                                (int)lds);
      (void)hipFuncSetAttribute((const void*)k_gemm256_bt<false>,
                                hipFuncAttributeMaxDynamicSharedMemorySize,
                                (int)lds);
      lds_configured = true;
    }
    if (tanh_epilogue)
      k_gemm256_bt<true><<<grid, 512, lds, cur_stream()>>>(
          bf_ptr(A), bf_ptr(Bt), bf_ptr_mut(C), N, M, K);
    else
      k_gemm256_bt<false><<<grid, 512, lds, cur_stream()>>>(
          bf_ptr(A), bf_ptr(Bt), bf_ptr_mut(C), N, M, K);
    return C;
  }
  const int n_tiles = (N + GEMM_BM - 1) / GEMM_BM;
  const int m_tiles = (M + GEMM_BN - 1) / GEMM_BN;
  dim3 grid(n_tiles * m_tiles);
  if (variant == 3) {
    const size_t lds = 64 * 1024;
    static bool bt2_cfg = false;
    if (!bt2_cfg) {
      (void)hipFuncSetAttribute((const void*)k_gemm_bt2<true>,
                                hipFuncAttributeMaxDynamicSharedMemorySize,
                                (int)lds);
      (void)hipFuncSetAttribute((const void*)k_gemm_bt2<false>,
                                hipFuncAttributeMaxDynamicSharedMemorySize,
                                (int)lds);
      (void)hipFuncSetAttribute((const void*)k_gemm_bt2<false, true>,
                                hipFuncAttributeMaxDynamicSharedMemorySize,
                                (int)lds);
      bt2_cfg = true;
    }
    if (tanh_epilogue)
      k_gemm_bt2<true><<<grid, 256, lds, cur_stream()>>>(
          bf_ptr(A), bf_ptr(Bt), bf_ptr_mut(C), N, M, K);
    else
      k_gemm_bt2<false><<<grid, 256, lds, cur_stream()>>>(
          bf_ptr(A), bf_ptr(Bt), bf_ptr_mut(C), N, M, K);
    return C;
  }
  if (tanh_epilogue)
    k_gemm_bt<true><<<grid, 256, 0, cur_stream()>>>(
        bf_ptr(A), bf_ptr(Bt), bf_ptr_mut(C), N, M, K);
  else
    k_gemm_bt<false><<<grid, 256, 0, cur_stream()>>>(
        bf_ptr(A), bf_ptr(Bt), bf_ptr_mut(C), N, M, K);
  return C;
}

std::vector<torch::Tensor> logits_ce_fused(torch::Tensor code,
                                           torch::Tensor shadow,
                                           torch::Tensor labels) {
  CHECK_DEV(code); CHECK_CONT(code); CHECK_DEV(shadow); CHECK_CONT(shadow);
  const int N = code.size(0), K = code.size(1), M = shadow.size(0);
  TORCH_CHECK(shadow.size(1) == K && K % G256_BK == 0);
  auto labels_c = labels.contiguous();
  auto C = torch::empty({N, M}, code.options());
  const int n_tiles = (N + G256_BM - 1) / G256_BM;
  const int m_tiles = (M + G256_BN - 1) / G256_BN;
  // (tile, quarter)-major partials (see the CE_PART epilogue comment)
  auto partials = torch::empty({(long)m_tiles * 4, (long)N, 2},
                               code.options().dtype(torch::kFloat32));
  const int t_chunks = 64;
  auto partials2 = torch::empty({(long)N, (long)t_chunks, 2},
                                code.options().dtype(torch::kFloat32));
  auto loss = torch::empty({N}, code.options().dtype(torch::kFloat32));
  auto lse = torch::empty({N}, code.options().dtype(torch::kFloat32));
  const size_t lds = 4 * 16384 * 2;
  static bool configured = false;
  if (!configured) {
    (void)hipFuncSetAttribute((const void*)k_gemm256_bt<false, true>,
                              hipFuncAttributeMaxDynamicSharedMemorySize,
                              (int)lds);
    configured = true;
  }
  k_gemm256_bt<false, true><<<n_tiles * m_tiles, 512, lds, cur_stream()>>>(
      bf_ptr(code), bf_ptr(shadow), bf_ptr_mut(C), N, M, K,
      partials.data_ptr<float>(), m_tiles);
  dim3 rg1((N + 255) / 256, t_chunks);
  k_ce_part_reduce1<<<rg1, 256, 0, cur_stream()>>>(
      partials.data_ptr<float>(), partials2.data_ptr<float>(), N,
      m_tiles * 4, t_chunks);
  k_ce_reduce_partials<<<N, 256, 0, cur_stream()>>>(
      partials2.data_ptr<float>(), bf_ptr(C), labels_c.data_ptr<long>(),
      loss.data_ptr<float>(), lse.data_ptr<float>(), N, t_chunks, M);
  return {C, loss, lse};
}

torch::Tensor transform_tanh_fwd(torch::Tensor ctx, torch::Tensor w_oi) {
  return gemm_bt(ctx, w_oi, true, 1);
}

torch::Tensor gemm_bt_bf16(torch::Tensor A, torch::Tensor Bt) {
  return gemm_bt(A, Bt, false, 1);
}

// Sampled-softmax candidate logits: C (N, n_idx) = A @ gather(table, idx)^T
// — the gather rides the GEMM's B staging (no w_cand materialization).
torch::Tensor gemm_bt_gather(torch::Tensor A, torch::Tensor table,
                             torch::Tensor idx) {
  CHECK_DEV(A); CHECK_CONT(A); CHECK_DEV(table); CHECK_CONT(table);
  TORCH_CHECK(A.scalar_type() == torch::kBFloat16 &&
              table.scalar_type() == torch::kBFloat16);
  auto idx_c = idx.contiguous();
  TORCH_CHECK(idx_c.scalar_type() == torch::kInt64, "idx must be int64");
  const int N = A.size(0), K = A.size(1), M = (int)idx_c.numel();
  TORCH_CHECK(table.size(1) == K && K % GEMM_BK == 0);
  auto C = torch::empty({N, M}, A.options());
  const int n_tiles = (N + GEMM_BM - 1) / GEMM_BM;
  const int m_tiles = (M + GEMM_BN - 1) / GEMM_BN;
  k_gemm_bt<false, false><<<n_tiles * m_tiles, 256, 0, cur_stream()>>>(
      bf_ptr(A), bf_ptr(table), bf_ptr_mut(C), N, M, K, 1.f, 0, nullptr,
      idx_c.data_ptr<long>());
  return C;
}

torch::Tensor gemm_bt_v(torch::Tensor A, torch::Tensor Bt, bool tanh_ep,
                        int64_t variant) {
  return gemm_bt(A, Bt, tanh_ep, (int)variant);
}

// dX GEMM with the dropout keep-mask fused into the epilogue (128-tile path)
torch::Tensor gemm_bt_dropout(torch::Tensor A, torch::Tensor Bt,
                              double keep_prob, int64_t seed,
                              torch::Tensor seed_t) {
  CHECK_DEV(A); CHECK_CONT(A); CHECK_DEV(Bt); CHECK_CONT(Bt);
  const int N = A.size(0), K = A.size(1), M = Bt.size(0);
  TORCH_CHECK(Bt.size(1) == K && K % GEMM_BK == 0);
  const long* seed_ptr = (seed_t.defined() && seed_t.numel() == 1)
                             ? seed_t.data_ptr<long>() : nullptr;
  auto C = torch::empty({N, M}, A.options());
  const int n_tiles = (N + GEMM_BM - 1) / GEMM_BM;
  const int m_tiles = (M + GEMM_BN - 1) / GEMM_BN;
  k_gemm_bt<false, true><<<n_tiles * m_tiles, 256, 0, cur_stream()>>>(
      bf_ptr(A), bf_ptr(Bt), bf_ptr_mut(C), N, M, K, (float)keep_prob,
      (u64)seed, seed_ptr);
  return C;
}

// d_target GEMM: C(V,M) bf16 = A(K,V)^T @ B(K,M), row-major bf16 operands,
// one block per 128-row V-tile (K = batch, contracted; no split-K).
torch::Tensor gemm_tn_bf16(torch::Tensor A, torch::Tensor B) {
  CHECK_DEV(A); CHECK_CONT(A); CHECK_DEV(B); CHECK_CONT(B);
  TORCH_CHECK(A.scalar_type() == torch::kBFloat16 &&
              B.scalar_type() == torch::kBFloat16);
  const int K = A.size(0), V = A.size(1), M = B.size(1);
  TORCH_CHECK(B.size(0) == K, "K mismatch");
  TORCH_CHECK(M <= GNN_BN && M % 8 == 0, "tn GEMM: M must be <=384, mult of 8");
  auto C = torch::empty({V, M}, A.options());
  const size_t lds = 2UL * GNN_BK * (GTN_PKT + GNN_PKB) * 2;  // 78 KiB
  static bool tn_configured = false;
  if (!tn_configured) {
    (void)hipFuncSetAttribute((const void*)k_gemm_tn<false>,
                              hipFuncAttributeMaxDynamicSharedMemorySize,
                              (int)lds);
    (void)hipFuncSetAttribute((const void*)k_gemm_tn<true>,
                              hipFuncAttributeMaxDynamicSharedMemorySize,
                              (int)lds);
    tn_configured = true;
  }
  // measured on the d_target shape (r02_call5): direct 10,022 us vs
  // staged 458 — the k-strided scalar fragment loads swamp the memory
  // pipeline with 2-byte-granule requests; kept for the record, off by
  // default
  static const bool direct = [] {
    const char* e = getenv("C2V_TN_DIRECT");
    return e && e[0] == '1';
  }();
  if (direct && M == 384) {
    k_gemm_tn_direct<false><<<(V + 127) / 128, 512, 0, cur_stream()>>>(
        bf_ptr(A), bf_ptr(B), bf_ptr_mut(C), V, M, K);
    return C;
  }
  k_gemm_tn<false><<<(V + GTN_BV - 1) / GTN_BV, 512, lds, cur_stream()>>>(
      bf_ptr(A), bf_ptr(B), bf_ptr_mut(C), V, M, K);
  return C;
}

// d_target with CE-backward fused into the d_logits staging:
// C(V,M) bf16 = ce_bwd(logits, lse, labels, scale)^T @ code — d_logits is
// computed on the fly, never written to HBM.
torch::Tensor gemm_tn_ce(torch::Tensor logits, torch::Tensor code,
                         torch::Tensor lse, torch::Tensor labels,
                         double scale) {
  CHECK_DEV(logits); CHECK_CONT(logits); CHECK_DEV(code); CHECK_CONT(code);
  const int K = logits.size(0), V = logits.size(1), M = code.size(1);
  TORCH_CHECK(code.size(0) == K && M <= GNN_BN && M % 8 == 0);
  auto labels_c = labels.contiguous();
  auto C = torch::empty({V, M}, logits.options());
  const size_t lds = 2UL * GNN_BK * (GTN_PKT + GNN_PKB) * 2;
  static bool cfg2 = false;
  if (!cfg2) {
    (void)hipFuncSetAttribute((const void*)k_gemm_tn<true>,
                              hipFuncAttributeMaxDynamicSharedMemorySize,
                              (int)lds);
    cfg2 = true;
  }
  // measured on the d_target shape (r02_call5): direct 10,022 us vs
  // staged 458 — the k-strided scalar fragment loads swamp the memory
  // pipeline with 2-byte-granule requests; kept for the record, off by
  // default
  static const bool direct = [] {
    const char* e = getenv("C2V_TN_DIRECT");
    return e && e[0] == '1';
  }();
  if (direct && M == 384) {
    k_gemm_tn_direct<true><<<(V + 127) / 128, 512, 0, cur_stream()>>>(
        bf_ptr(logits), bf_ptr(code), bf_ptr_mut(C), V, M, K,
        lse.data_ptr<float>(), labels_c.data_ptr<long>(), (float)scale);
    return C;
  }
  k_gemm_tn<true><<<(V + GTN_BV - 1) / GTN_BV, 512, lds, cur_stream()>>>(
      bf_ptr(logits), bf_ptr(code), bf_ptr_mut(C), V, M, K,
      lse.data_ptr<float>(), labels_c.data_ptr<long>(), (float)scale);
  return C;
}

// dW GEMM: C(N2,M) fp32 = A(K,N2)^T @ B(K,M) with K huge (batch*contexts)
// and a tiny output — split-K tn (k_gemm_tn<false,true>), partials folded
// by k_splitk_reduce. Shaped for d_w = ctx^T @ d_z (K~205K, out 384x384).
torch::Tensor gemm_tn_splitk(torch::Tensor A, torch::Tensor B) {
  CHECK_DEV(A); CHECK_CONT(A); CHECK_DEV(B); CHECK_CONT(B);
  TORCH_CHECK(A.scalar_type() == torch::kBFloat16 &&
              B.scalar_type() == torch::kBFloat16);
  const int K = A.size(0), N2 = A.size(1), M = B.size(1);
  TORCH_CHECK(B.size(0) == K, "K mismatch");
  TORCH_CHECK(M <= GNN_BN && M % 8 == 0 && N2 % 8 == 0);
  const int row_tiles = (N2 + GTN_BV - 1) / GTN_BV;
  int S = 256 / (row_tiles * 8) * 8;
  if (S < 8) S = 8;
  const int total_ksteps = (K + GNN_BK - 1) / GNN_BK;
  const int kpc = (total_ksteps + S - 1) / S;
  auto P = torch::empty({(long)S, (long)N2, (long)M},
                        A.options().dtype(torch::kFloat32));
  auto C = torch::empty({N2, M}, A.options().dtype(torch::kFloat32));
  const size_t lds = 2UL * GNN_BK * (GTN_PKT + GNN_PKB) * 2;
  static bool cfg3 = false;
  if (!cfg3) {
    (void)hipFuncSetAttribute((const void*)k_gemm_tn<false, true>,
                              hipFuncAttributeMaxDynamicSharedMemorySize,
                              (int)lds);
    cfg3 = true;
  }
  k_gemm_tn<false, true><<<S * row_tiles, 512, lds, cur_stream()>>>(
      bf_ptr(A), bf_ptr(B), nullptr, N2, M, K, nullptr, nullptr, 1.f,
      P.data_ptr<float>(), S, kpc, row_tiles);
  const long total = (long)N2 * M;
  TORCH_CHECK(total % 4 == 0);
  k_splitk_reduce<<<grid_1d(total / 4, 256), 256, 0, cur_stream()>>>(
      P.data_ptr<float>(), C.data_ptr<float>(), S, total);
  return C;
}

// split-K nn GEMM: C(N,M) fp32 = A(N,K) @ B(K,M), row-major bf16 operands.
// Shaped for d_code = d_logits @ target_shadow (N=batch, M=code dim <= 384,
// K=vocab). Partials workspace (S, N, M) fp32 comes from the caching
// allocator; S is a multiple of 8 so the XCD-grouped chunk decode is
// bijective, sized so the grid is ~256 blocks (1 per CU).
// Sampled-softmax d_code: C (N, M) fp32 = A @ gather(table, idx) — the
// candidate-row gather rides the split-K nn GEMM's B staging.
torch::Tensor gemm_nn_splitk_gather(torch::Tensor A, torch::Tensor table,
                                    torch::Tensor idx) {
  CHECK_DEV(A); CHECK_CONT(A); CHECK_DEV(table); CHECK_CONT(table);
  TORCH_CHECK(A.scalar_type() == torch::kBFloat16 &&
              table.scalar_type() == torch::kBFloat16);
  auto idx_c = idx.contiguous();
  TORCH_CHECK(idx_c.scalar_type() == torch::kInt64, "idx must be int64");
  const int N = A.size(0), K = A.size(1), M = table.size(1);
  TORCH_CHECK((int)idx_c.numel() == K, "idx length must equal A cols");
  TORCH_CHECK(M <= GNN_BN && M % 8 == 0);
  const int row_tiles = (N + GNN_BM - 1) / GNN_BM;
  int S = 256 / (row_tiles * 8) * 8;
  if (S < 8) S = 8;
  const int total_ksteps = (K + GNN_BK - 1) / GNN_BK;
  const int kpc = (total_ksteps + S - 1) / S;
  auto P = torch::empty({(long)S, (long)N, (long)M},
                        A.options().dtype(torch::kFloat32));
  auto C = torch::empty({N, M}, A.options().dtype(torch::kFloat32));
  const size_t lds = 2UL * (GNN_BM * GNN_PKA + GNN_BK * GNN_PKB) * 2;
  static bool cfg_g = false;
  if (!cfg_g) {
    (void)hipFuncSetAttribute((const void*)k_gemm_nn_splitk<0>,
                              hipFuncAttributeMaxDynamicSharedMemorySize,
                              (int)lds);
    cfg_g = true;
  }
  k_gemm_nn_splitk<0><<<S * row_tiles, 256, lds, cur_stream()>>>(
      bf_ptr(A), bf_ptr(table), P.data_ptr<float>(), N, M, K, S, kpc,
      row_tiles, nullptr, nullptr, 1.f, nullptr, idx_c.data_ptr<long>());
  const long total = (long)N * M;
  TORCH_CHECK(total % 4 == 0);
  k_splitk_reduce<<<grid_1d(total / 4, 256), 256, 0, cur_stream()>>>(
      P.data_ptr<float>(), C.data_ptr<float>(), S, total);
  return C;
}

torch::Tensor gemm_nn_splitk(torch::Tensor A, torch::Tensor B) {
  CHECK_DEV(A); CHECK_CONT(A); CHECK_DEV(B); CHECK_CONT(B);
  TORCH_CHECK(A.scalar_type() == torch::kBFloat16 &&
              B.scalar_type() == torch::kBFloat16);
  const int N = A.size(0), K = A.size(1), M = B.size(1);
  TORCH_CHECK(B.size(0) == K, "K mismatch");
  TORCH_CHECK(M <= GNN_BN && M % 8 == 0, "nn GEMM: M must be <=384, mult of 8");
  const int row_tiles = (N + GNN_BM - 1) / GNN_BM;
  int S = 256 / (row_tiles * 8) * 8;          // grid ~256, S multiple of 8
  if (S < 8) S = 8;
  const int total_ksteps = (K + GNN_BK - 1) / GNN_BK;
  const int kpc = (total_ksteps + S - 1) / S;
  auto P = torch::empty({(long)S, (long)N, (long)M},
                        A.options().dtype(torch::kFloat32));
  auto C = torch::empty({N, M}, A.options().dtype(torch::kFloat32));
  const size_t lds = 2UL * (GNN_BM * GNN_PKA + GNN_BK * GNN_PKB) * 2;  // 66 KiB
  static bool nn_configured = false;
  if (!nn_configured) {
    (void)hipFuncSetAttribute((const void*)k_gemm_nn_splitk<0>,
                              hipFuncAttributeMaxDynamicSharedMemorySize,
                              (int)lds);
    (void)hipFuncSetAttribute((const void*)k_gemm_nn_splitk<1>,
                              hipFuncAttributeMaxDynamicSharedMemorySize,
                              (int)lds);
    (void)hipFuncSetAttribute((const void*)k_gemm_nn_splitk<2>,
                              hipFuncAttributeMaxDynamicSharedMemorySize,
                              (int)lds);
    nn_configured = true;
  }
  k_gemm_nn_splitk<0><<<S * row_tiles, 256, lds, cur_stream()>>>(
      bf_ptr(A), bf_ptr(B), P.data_ptr<float>(), N, M, K, S, kpc, row_tiles);
  const long total = (long)N * M;
  TORCH_CHECK(total % 4 == 0);
  k_splitk_reduce<<<grid_1d(total / 4, 256), 256, 0, cur_stream()>>>(
      P.data_ptr<float>(), C.data_ptr<float>(), S, total);
  return C;
}

// d_code with CE-backward fused into the d_logits staging:
// C(N,M) fp32 = ce_bwd(logits, lse, labels, scale) @ shadow.
torch::Tensor gemm_nn_splitk_ce(torch::Tensor logits, torch::Tensor shadow,
                                torch::Tensor lse, torch::Tensor labels,
                                double scale) {
  CHECK_DEV(logits); CHECK_CONT(logits);
  CHECK_DEV(shadow); CHECK_CONT(shadow);
  const int N = logits.size(0), K = logits.size(1), M = shadow.size(1);
  TORCH_CHECK(shadow.size(0) == K && M <= GNN_BN && M % 8 == 0);
  auto labels_c = labels.contiguous();
  const int row_tiles = (N + GNN_BM - 1) / GNN_BM;
  int S = 256 / (row_tiles * 8) * 8;
  if (S < 8) S = 8;
  const int total_ksteps = (K + GNN_BK - 1) / GNN_BK;
  const int kpc = (total_ksteps + S - 1) / S;
  auto P = torch::empty({(long)S, (long)N, (long)M},
                        logits.options().dtype(torch::kFloat32));
  auto C = torch::empty({N, M}, logits.options().dtype(torch::kFloat32));
  const size_t lds = 2UL * (GNN_BM * GNN_PKA + GNN_BK * GNN_PKB) * 2;
  static bool cfg2 = false;
  if (!cfg2) {
    (void)hipFuncSetAttribute((const void*)k_gemm_nn_splitk<1>,
                              hipFuncAttributeMaxDynamicSharedMemorySize,
                              (int)lds);
    cfg2 = true;
  }
  k_gemm_nn_splitk<1><<<S * row_tiles, 256, lds, cur_stream()>>>(
      bf_ptr(logits), bf_ptr(shadow), P.data_ptr<float>(), N, M, K, S, kpc,
      row_tiles, lse.data_ptr<float>(), labels_c.data_ptr<long>(),
      (float)scale);
  const long total = (long)N * M;
  TORCH_CHECK(total % 4 == 0);
  k_splitk_reduce<<<grid_1d(total / 4, 256), 256, 0, cur_stream()>>>(
      P.data_ptr<float>(), C.data_ptr<float>(), S, total);
  return C;
}

// CE-backward fused d_code GEMM that ALSO materializes d_logits (CEB=2):
// returns (d_code fp32 (N,M), d_logits bf16 (N,K)) — replaces the separate
// k_ce_bwd pass; d_target consumes the returned d_logits.
std::vector<torch::Tensor> gemm_nn_splitk_ce_write(torch::Tensor logits,
                                                   torch::Tensor shadow,
                                                   torch::Tensor lse,
                                                   torch::Tensor labels,
                                                   double scale) {
  CHECK_DEV(logits); CHECK_CONT(logits);
  CHECK_DEV(shadow); CHECK_CONT(shadow);
  const int N = logits.size(0), K = logits.size(1), M = shadow.size(1);
  TORCH_CHECK(shadow.size(0) == K && M <= GNN_BN && M % 8 == 0);
  auto labels_c = labels.contiguous();
  const int row_tiles = (N + GNN_BM - 1) / GNN_BM;
  int S = 256 / (row_tiles * 8) * 8;
  if (S < 8) S = 8;
  const int total_ksteps = (K + GNN_BK - 1) / GNN_BK;
  const int kpc = (total_ksteps + S - 1) / S;
  auto P = torch::empty({(long)S, (long)N, (long)M},
                        logits.options().dtype(torch::kFloat32));
  auto C = torch::empty({N, M}, logits.options().dtype(torch::kFloat32));
  auto DL = torch::empty_like(logits);
  const size_t lds = 2UL * (GNN_BM * GNN_PKA + GNN_BK * GNN_PKB) * 2;
  static bool cfg4 = false;
  if (!cfg4) {
    (void)hipFuncSetAttribute((const void*)k_gemm_nn_splitk<2>,
                              hipFuncAttributeMaxDynamicSharedMemorySize,
                              (int)lds);
    cfg4 = true;
  }
  k_gemm_nn_splitk<2><<<S * row_tiles, 256, lds, cur_stream()>>>(
      bf_ptr(logits), bf_ptr(shadow), P.data_ptr<float>(), N, M, K, S, kpc,
      row_tiles, lse.data_ptr<float>(), labels_c.data_ptr<long>(),
      (float)scale, bf_ptr_mut(DL));
  const long total = (long)N * M;
  TORCH_CHECK(total % 4 == 0);
  k_splitk_reduce<<<grid_1d(total / 4, 256), 256, 0, cur_stream()>>>(
      P.data_ptr<float>(), C.data_ptr<float>(), S, total);
  return {C, DL};
}

torch::Tensor tanh_bwd_mul(torch::Tensor dy, torch::Tensor y) {
  CHECK_DEV(dy); CHECK_CONT(dy); CHECK_DEV(y); CHECK_CONT(y);
  auto dz = torch::empty_like(dy);
  const long total = dy.numel();
  TORCH_CHECK(total % 8 == 0);
  k_tanh_bwd_mul<<<grid_1d(total / 8, 256), 256, 0, cur_stream()>>>(
      bf_ptr(dy), bf_ptr(y), bf_ptr_mut(dz), total);
  return dz;
}

std::vector<torch::Tensor> attention_fwd(torch::Tensor comb, torch::Tensor a,
                                         torch::Tensor mask) {
  CHECK_DEV(comb); CHECK_CONT(comb); CHECK_DEV(a); CHECK_DEV(mask);
  TORCH_CHECK(comb.dim() == 3);
  const int B = comb.size(0), C = comb.size(1), D = comb.size(2);
  TORCH_CHECK(D % 64 == 0 && D <= 512,
              "code vector size must be a multiple of 64, <= 512");
  auto a32 = a.to(torch::kFloat32).contiguous();
  auto mask32 = mask.to(torch::kFloat32).contiguous();
  auto code = torch::empty({B, D}, comb.options().dtype(torch::kFloat32));
  auto alpha = torch::empty({B, C}, comb.options().dtype(torch::kFloat32));
  const size_t lds = (size_t)(C + D) * 4;  // scores + code accumulator
  k_attn_fwd<<<B, 256, lds, cur_stream()>>>(
      bf_ptr(comb), a32.data_ptr<float>(), mask32.data_ptr<float>(),
      code.data_ptr<float>(), alpha.data_ptr<float>(), B, C, D);
  return {code, alpha};
}

std::vector<torch::Tensor> attention_bwd(torch::Tensor comb, torch::Tensor a,
                                         torch::Tensor alpha,
                                         torch::Tensor d_code,
                                         bool fuse_tanh_bwd) {
  CHECK_DEV(comb); CHECK_CONT(comb);
  const int B = comb.size(0), C = comb.size(1), D = comb.size(2);
  TORCH_CHECK(D % 64 == 0 && D <= 512);
  auto a32 = a.to(torch::kFloat32).contiguous();
  auto alpha32 = alpha.contiguous();
  auto dcode32 = d_code.to(torch::kFloat32).contiguous();
  auto d_comb = torch::empty_like(comb);
  auto d_a_partial = torch::empty({B, D}, comb.options().dtype(torch::kFloat32));
  const size_t lds = (size_t)(C + D) * 4;  // d_e scratch + d_a accumulator
  k_attn_bwd<<<B, 256, lds, cur_stream()>>>(
      bf_ptr(comb), a32.data_ptr<float>(), alpha32.data_ptr<float>(),
      dcode32.data_ptr<float>(), bf_ptr_mut(d_comb),
      d_a_partial.data_ptr<float>(), B, C, D, fuse_tanh_bwd ? 1 : 0);
  auto d_a = d_a_partial.sum(0);
  return {d_comb, d_a};
}

std::vector<torch::Tensor> topk(torch::Tensor logits, int64_t k) {
  CHECK_DEV(logits); CHECK_CONT(logits);
  TORCH_CHECK(logits.scalar_type() == torch::kBFloat16);
  const int B = logits.size(0), V = logits.size(1);
  TORCH_CHECK(k >= 1 && k <= 32 && k <= V);
  auto vals = torch::empty({B, k}, logits.options().dtype(torch::kFloat32));
  auto idx = torch::empty({B, k}, logits.options().dtype(torch::kInt64));
  const size_t lds = 256 * (size_t)k * 8;
  k_topk<<<B, 256, lds, cur_stream()>>>(bf_ptr(logits),
                                        vals.data_ptr<float>(),
                                        idx.data_ptr<long>(), V, (int)k);
  return {vals, idx};
}

std::vector<torch::Tensor> ce_fwd(torch::Tensor logits, torch::Tensor labels) {
  CHECK_DEV(logits); CHECK_CONT(logits);
  TORCH_CHECK(labels.scalar_type() == torch::kInt64);
  const int B = logits.size(0), V = logits.size(1);
  auto labels_c = labels.contiguous();
  auto loss = torch::empty({B}, logits.options().dtype(torch::kFloat32));
  auto lse = torch::empty({B}, logits.options().dtype(torch::kFloat32));
  k_ce_fwd<<<B, 256, 0, cur_stream()>>>(
      bf_ptr(logits), labels_c.data_ptr<long>(), loss.data_ptr<float>(),
      lse.data_ptr<float>(), B, V);
  return {loss, lse};
}

torch::Tensor ce_bwd(torch::Tensor logits, torch::Tensor lse,
                     torch::Tensor labels, double scale) {
  CHECK_DEV(logits); CHECK_CONT(logits);
  const int B = logits.size(0), V = logits.size(1);
  auto labels_c = labels.contiguous();
  auto d = torch::empty_like(logits);
  dim3 grid(grid_1d(V / 16, 256, 64), B);
  k_ce_bwd<<<grid, 256, 0, cur_stream()>>>(
      bf_ptr(logits), lse.data_ptr<float>(), labels_c.data_ptr<long>(),
      bf_ptr_mut(d), (float)scale, B, V);
  return d;
}

void adam_dense_step(torch::Tensor p, torch::Tensor g, torch::Tensor m,
                     torch::Tensor v, int64_t step, double lr, double beta1,
                     double beta2, double eps, torch::Tensor shadow,
                     torch::Tensor lrt_t) {
  const float* lrt_ptr = (lrt_t.defined() && lrt_t.numel() == 1)
                             ? lrt_t.data_ptr<float>() : nullptr;
  CHECK_DEV(p); CHECK_CONT(p);
  auto g_c = g.contiguous();
  const long n = p.numel();
  TORCH_CHECK(g_c.numel() == n && m.numel() == n && v.numel() == n);
  const float lr_t = (float)(lr * std::sqrt(1.0 - std::pow(beta2, (double)step)) /
                             (1.0 - std::pow(beta1, (double)step)));
  ushort* shadow_ptr = nullptr;
  if (shadow.defined() && shadow.numel() == n)
    shadow_ptr = reinterpret_cast<ushort*>(shadow.data_ptr<at::BFloat16>());
  // A/B on MI355X (java14m target-table shape, r02_call4): width-1 NT
  // stores 500 us, width-1 cached 530, width-2 532 — NT default, w2 off
  static const bool use_nt = [] {
    const char* e = getenv("C2V_ADAM_NT");
    return !e || e[0] == '1';
  }();
  static const bool use_w2 = [] {
    const char* e = getenv("C2V_ADAM_W2");
    return e && e[0] == '1';
  }();
  const int grid = grid_1d(std::max<long>(n / 4, 1), 256);
  if (use_w2 && g_c.scalar_type() == torch::kBFloat16) {
    if (use_nt)
      k_adam_dense_w2<ushort, true><<<grid, 256, 0, cur_stream()>>>(
          p.data_ptr<float>(), bf_ptr(g_c), m.data_ptr<float>(),
          v.data_ptr<float>(), shadow_ptr, n, lr_t, (float)beta1,
          (float)beta2, (float)eps, lrt_ptr);
    else
      k_adam_dense_w2<ushort, false><<<grid, 256, 0, cur_stream()>>>(
          p.data_ptr<float>(), bf_ptr(g_c), m.data_ptr<float>(),
          v.data_ptr<float>(), shadow_ptr, n, lr_t, (float)beta1,
          (float)beta2, (float)eps, lrt_ptr);
    return;
  }
  if (use_nt && g_c.scalar_type() == torch::kBFloat16) {
    k_adam_dense<ushort, true><<<grid, 256, 0, cur_stream()>>>(
        p.data_ptr<float>(), bf_ptr(g_c), m.data_ptr<float>(),
        v.data_ptr<float>(), shadow_ptr, n, lr_t, (float)beta1, (float)beta2,
        (float)eps, lrt_ptr);
    return;
  }
  if (g_c.scalar_type() == torch::kBFloat16)
    k_adam_dense<ushort><<<grid, 256, 0, cur_stream()>>>(
        p.data_ptr<float>(), bf_ptr(g_c), m.data_ptr<float>(),
        v.data_ptr<float>(), shadow_ptr, n, lr_t, (float)beta1, (float)beta2,
        (float)eps, lrt_ptr);
  else
    k_adam_dense<float><<<grid, 256, 0, cur_stream()>>>(
        p.data_ptr<float>(), g_c.data_ptr<float>(), m.data_ptr<float>(),
        v.data_ptr<float>(), shadow_ptr, n, lr_t, (float)beta1, (float)beta2,
        (float)eps, lrt_ptr);
}

// ---------------------------------------------------------------------------
// Rank-local sparse-gradient dedup+sum for data-parallel training: the same
// hash claim/compact/lookup/accumulate pipeline the sparse Adam uses, stopped
// before the Adam update so the (unique ids, summed rows) pairs can go on the
// wire instead of every raw contribution. On Zipf-distributed real-data ids
// this cuts the per-rank all-gather volume by 3-4x (SURVEY §2.4 sparse
// strategy; ROADMAP-R2 "Scaling" item b). Returns {uniq_ids int64[n],
// acc fp32[n,d], n_uniq int32[1] device} — callers slice by the count.
// ---------------------------------------------------------------------------

struct DedupState {
  torch::Tensor uniq, inverse, n_uniq;
  torch::Tensor hot2cidx, n_hot;
};

static DedupState hash_dedup_ids(const torch::Tensor& ids_c) {
  const long n = ids_c.numel();
  long want = 2 * n;
  u32 cap = 1;
  while (cap < (u32)want) cap <<= 1;
  auto opts_i32 = torch::TensorOptions().device(ids_c.device())
                      .dtype(torch::kInt32);
  // C2V_HASH_WS=1: single workspace + one init kernel instead of five
  // torch fills ([tbl_id | pad | tbl_cidx | pad | tbl_cnt | n_hot |
  // n_uniq], counters as narrow() views keeping it alive). Measured 300
  // us/step SLOWER on the sampled bench across two same-box A/Bs — and
  // the 4.25 KB inter-section pads did NOT recover it, so the obvious
  // power-of-two channel-aliasing explanation is falsified. The cost is
  // some unidentified sensitivity of the claim kernel to the captured
  // allocation layout. Default OFF: the ~15 fill launches it saves are
  // worth ~60 us, the regression costs 5x that.
  static const bool use_ws = [] {
    const char* e = getenv("C2V_HASH_WS");
    return e && e[0] == '1';
  }();
  torch::Tensor tbl_id, tbl_cidx, tbl_cnt, n_hot, n_uniq;
  if (use_ws) {
    // 4.25 KB pads between the sections break the exact power-of-two
    // offsets (the aliasing suspect); pad bytes land in the -1/0 fill
    // regions and are never read
    const long P = 1088;
    const long ws_len = 3 * (long)cap + 2 * P + 2;
    auto ws = torch::empty({ws_len}, opts_i32);
    tbl_id = ws.narrow(0, 0, cap);
    tbl_cidx = ws.narrow(0, cap + P, cap);
    tbl_cnt = ws.narrow(0, 2 * ((long)cap + P), cap);
    n_hot = ws.narrow(0, 3 * (long)cap + 2 * P, 1);
    n_uniq = ws.narrow(0, 3 * (long)cap + 2 * P + 1, 1);
    k_hash_ws_init<<<grid_1d(ws_len / 4 + 1, 256), 256, 0, cur_stream()>>>(
        ws.data_ptr<int>(), 2 * ((long)cap + P), ws_len);
  } else {
    tbl_id = torch::full({(long)cap}, -1, opts_i32);
    tbl_cidx = torch::full({(long)cap}, -1, opts_i32);
    tbl_cnt = torch::zeros({(long)cap}, opts_i32);
    n_hot = torch::zeros({1}, opts_i32);
    n_uniq = torch::zeros({1}, opts_i32);
  }
  auto tbl_hot = torch::empty({(long)cap}, opts_i32);
  auto hot2cidx = torch::empty({HOT_CAP}, opts_i32);
  auto uniq = torch::empty({n}, opts_i32.dtype(torch::kInt64));
  auto inverse = torch::empty({n}, opts_i32);
  const u32 mask_ = cap - 1;
  if (ids_c.scalar_type() == torch::kInt32) {
    k_hash_claim<int><<<grid_1d(n, 256), 256, 0, cur_stream()>>>(
        ids_c.data_ptr<int>(), n, tbl_id.data_ptr<int>(), mask_,
        tbl_cnt.data_ptr<int>());
    k_hash_compact<<<grid_1d(cap, 256), 256, 0, cur_stream()>>>(
        tbl_id.data_ptr<int>(), tbl_cidx.data_ptr<int>(),
        uniq.data_ptr<long>(), n_uniq.data_ptr<int>(), cap,
        tbl_cnt.data_ptr<int>(), tbl_hot.data_ptr<int>(),
        hot2cidx.data_ptr<int>(), n_hot.data_ptr<int>());
    k_hash_lookup<int><<<grid_1d(n, 256), 256, 0, cur_stream()>>>(
        ids_c.data_ptr<int>(), n, tbl_id.data_ptr<int>(),
        tbl_cidx.data_ptr<int>(), inverse.data_ptr<int>(), mask_,
        tbl_cnt.data_ptr<int>(), tbl_hot.data_ptr<int>());
  } else {
    k_hash_claim<long><<<grid_1d(n, 256), 256, 0, cur_stream()>>>(
        ids_c.data_ptr<long>(), n, tbl_id.data_ptr<int>(), mask_,
        tbl_cnt.data_ptr<int>());
    k_hash_compact<<<grid_1d(cap, 256), 256, 0, cur_stream()>>>(
        tbl_id.data_ptr<int>(), tbl_cidx.data_ptr<int>(),
        uniq.data_ptr<long>(), n_uniq.data_ptr<int>(), cap,
        tbl_cnt.data_ptr<int>(), tbl_hot.data_ptr<int>(),
        hot2cidx.data_ptr<int>(), n_hot.data_ptr<int>());
    k_hash_lookup<long><<<grid_1d(n, 256), 256, 0, cur_stream()>>>(
        ids_c.data_ptr<long>(), n, tbl_id.data_ptr<int>(),
        tbl_cidx.data_ptr<int>(), inverse.data_ptr<int>(), mask_,
        tbl_cnt.data_ptr<int>(), tbl_hot.data_ptr<int>());
  }
  return {uniq, inverse, n_uniq, hot2cidx, n_hot};
}

// zero acc prefix, accumulate rows (with hot-id replica spreading), fold
static torch::Tensor accum_rows_common(const DedupState& st,
                                       const torch::Tensor& rows_c, long n,
                                       int d) {
  auto acc = torch::empty({n, (long)d},
                          rows_c.options().dtype(torch::kFloat32));
  auto hot_acc = torch::empty({(long)HOT_CAP * HOT_R, (long)d},
                              rows_c.options().dtype(torch::kFloat32));
  k_zero_rows_dyn<<<grid_1d((long)HOT_CAP * HOT_R * d / 4, 256), 256, 0,
                    cur_stream()>>>(
      hot_acc.data_ptr<float>(), st.n_hot.data_ptr<int>(), HOT_R * d,
      HOT_CAP);
  k_zero_rows_dyn<<<grid_1d(n * d / 4, 256), 256, 0, cur_stream()>>>(
      acc.data_ptr<float>(), st.n_uniq.data_ptr<int>(), d);
  if (rows_c.scalar_type() == torch::kBFloat16)
    k_rows_accum<ushort><<<grid_1d(n * d, 256), 256, 0, cur_stream()>>>(
        bf_ptr(rows_c), st.inverse.data_ptr<int>(), acc.data_ptr<float>(),
        n, d, hot_acc.data_ptr<float>());
  else
    k_rows_accum<float><<<grid_1d(n * d, 256), 256, 0, cur_stream()>>>(
        rows_c.data_ptr<float>(), st.inverse.data_ptr<int>(),
        acc.data_ptr<float>(), n, d, hot_acc.data_ptr<float>());
  k_hot_fold<<<grid_1d((long)HOT_CAP * d, 256), 256, 0, cur_stream()>>>(
      hot_acc.data_ptr<float>(), st.hot2cidx.data_ptr<int>(),
      st.n_hot.data_ptr<int>(), acc.data_ptr<float>(), d);
  return acc;
}

static torch::Tensor accum_ctx_common(const DedupState& st,
                                      const torch::Tensor& d_ctx, int off0,
                                      int off1, long n_per_seg, int n_seg,
                                      int d) {
  const long n = n_per_seg * n_seg;
  const int ld = (int)d_ctx.size(1);
  auto acc = torch::empty({n, (long)d},
                          d_ctx.options().dtype(torch::kFloat32));
  auto hot_acc = torch::empty({(long)HOT_CAP * HOT_R, (long)d},
                              d_ctx.options().dtype(torch::kFloat32));
  k_zero_rows_dyn<<<grid_1d((long)HOT_CAP * HOT_R * d / 4, 256), 256, 0,
                    cur_stream()>>>(
      hot_acc.data_ptr<float>(), st.n_hot.data_ptr<int>(), HOT_R * d,
      HOT_CAP);
  k_zero_rows_dyn<<<grid_1d(n * d / 4, 256), 256, 0, cur_stream()>>>(
      acc.data_ptr<float>(), st.n_uniq.data_ptr<int>(), d);
  k_rows_accum_ctx<<<grid_1d(n * d, 256), 256, 0, cur_stream()>>>(
      bf_ptr(d_ctx), ld, off0, off1, n_per_seg, n_seg,
      st.inverse.data_ptr<int>(), acc.data_ptr<float>(), d,
      hot_acc.data_ptr<float>());
  k_hot_fold<<<grid_1d((long)HOT_CAP * d, 256), 256, 0, cur_stream()>>>(
      hot_acc.data_ptr<float>(), st.hot2cidx.data_ptr<int>(),
      st.n_hot.data_ptr<int>(), acc.data_ptr<float>(), d);
  return acc;
}

void adam_sparse_rows_step(torch::Tensor p, torch::Tensor uniq_ids,
                           torch::Tensor inverse, torch::Tensor grad_rows,
                           torch::Tensor m, torch::Tensor v, int64_t step,
                           double lr, double beta1, double beta2, double eps,
                           torch::Tensor shadow) {
  CHECK_DEV(p); CHECK_CONT(p);
  auto rows_c = grad_rows.contiguous();
  auto inv_c = inverse.contiguous();
  auto ids_c = uniq_ids.contiguous();
  const long n_rows = rows_c.size(0);
  const int d = rows_c.size(1);
  const long n_uniq = ids_c.numel();
  auto acc = torch::zeros({n_uniq, (long)d},
                          p.options().dtype(torch::kFloat32));
  const float lr_t = (float)(lr * std::sqrt(1.0 - std::pow(beta2, (double)step)) /
                             (1.0 - std::pow(beta1, (double)step)));
  if (rows_c.scalar_type() == torch::kBFloat16)
    k_rows_accum<ushort><<<grid_1d(n_rows * d, 256), 256, 0, cur_stream()>>>(
        bf_ptr(rows_c), inv_c.data_ptr<int>(), acc.data_ptr<float>(), n_rows, d);
  else
    k_rows_accum<float><<<grid_1d(n_rows * d, 256), 256, 0, cur_stream()>>>(
        rows_c.data_ptr<float>(), inv_c.data_ptr<int>(), acc.data_ptr<float>(),
        n_rows, d);
  ushort* shadow_ptr = nullptr;
  if (shadow.defined() && shadow.numel() == p.numel())
    shadow_ptr = reinterpret_cast<ushort*>(shadow.data_ptr<at::BFloat16>());
  k_adam_rows<<<grid_1d(n_uniq * d, 256), 256, 0, cur_stream()>>>(
      p.data_ptr<float>(), ids_c.data_ptr<long>(), acc.data_ptr<float>(),
      m.data_ptr<float>(), v.data_ptr<float>(), shadow_ptr, n_uniq, d, lr_t,
      (float)beta1, (float)beta2, (float)eps);
}

void adam_sparse_rows_hash(torch::Tensor p, torch::Tensor ids,
                           torch::Tensor grad_rows, torch::Tensor m,
                           torch::Tensor v, int64_t step, double lr,
                           double beta1, double beta2, double eps,
                           torch::Tensor shadow, torch::Tensor lrt_t) {
  const float* lrt_ptr = (lrt_t.defined() && lrt_t.numel() == 1)
                             ? lrt_t.data_ptr<float>() : nullptr;
  CHECK_DEV(p); CHECK_CONT(p);
  auto ids_c = ids.contiguous();
  auto rows_c = grad_rows.contiguous();
  const long n = ids_c.numel();
  const int d = rows_c.size(1);
  auto st = hash_dedup_ids(ids_c);
  auto acc = accum_rows_common(st, rows_c, n, d);
  const float lr_t = (float)(lr * std::sqrt(1.0 - std::pow(beta2, (double)step)) /
                             (1.0 - std::pow(beta1, (double)step)));
  ushort* shadow_ptr = nullptr;
  if (shadow.defined() && shadow.numel() == p.numel())
    shadow_ptr = reinterpret_cast<ushort*>(shadow.data_ptr<at::BFloat16>());
  k_adam_rows_dyn<<<grid_1d(n * d, 256), 256, 0, cur_stream()>>>(
      p.data_ptr<float>(), st.uniq.data_ptr<long>(), acc.data_ptr<float>(),
      m.data_ptr<float>(), v.data_ptr<float>(), shadow_ptr,
      st.n_uniq.data_ptr<int>(), d, lr_t, (float)beta1, (float)beta2,
      (float)eps, lrt_ptr);
}

void adam_sparse_rows_hash_ctx(torch::Tensor p, torch::Tensor ids,
                               torch::Tensor d_ctx, int64_t off0, int64_t off1,
                               int64_t n_seg, int64_t d, torch::Tensor m,
                               torch::Tensor v, int64_t step, double lr,
                               double beta1, double beta2, double eps,
                               torch::Tensor lrt_t) {
  CHECK_DEV(p); CHECK_CONT(p); CHECK_DEV(d_ctx); CHECK_CONT(d_ctx);
  const float* lrt_ptr = (lrt_t.defined() && lrt_t.numel() == 1)
                             ? lrt_t.data_ptr<float>() : nullptr;
  auto ids_c = ids.contiguous();
  const long n = ids_c.numel();
  const long n_per_seg = d_ctx.size(0);
  TORCH_CHECK(n == n_per_seg * n_seg, "ids length mismatch");
  TORCH_CHECK(ids_c.scalar_type() == torch::kInt32, "ctx path expects int32 ids");
  auto st = hash_dedup_ids(ids_c);
  auto acc = accum_ctx_common(st, d_ctx, (int)off0, (int)off1, n_per_seg,
                              (int)n_seg, (int)d);
  const float lr_t = (float)(lr * std::sqrt(1.0 - std::pow(beta2, (double)step)) /
                             (1.0 - std::pow(beta1, (double)step)));
  k_adam_rows_dyn<<<grid_1d(n * d, 256), 256, 0, cur_stream()>>>(
      p.data_ptr<float>(), st.uniq.data_ptr<long>(), acc.data_ptr<float>(),
      m.data_ptr<float>(), v.data_ptr<float>(), nullptr,
      st.n_uniq.data_ptr<int>(), (int)d, lr_t, (float)beta1, (float)beta2,
      (float)eps, lrt_ptr);
}

// Phase split for forward-overlap: the hash build (claim/compact/lookup)
// depends only on the ids — launch it on a side stream at step START so it
// hides under the forward GEMMs; the accumulate/Adam phases consume the
// prebuilt state after d_ctx exists (~450 us off the backward tail).
std::vector<torch::Tensor> sparse_hash_build(torch::Tensor ids) {
  auto ids_c = ids.contiguous();
  auto st = hash_dedup_ids(ids_c);
  return {st.uniq, st.inverse, st.n_uniq, st.hot2cidx, st.n_hot};
}

static DedupState state_from(torch::Tensor uniq, torch::Tensor inverse,
                             torch::Tensor n_uniq, torch::Tensor hot2cidx,
                             torch::Tensor n_hot) {
  return {uniq, inverse, n_uniq, hot2cidx, n_hot};
}

void adam_sparse_rows_hash_ctx_pre(
    torch::Tensor p, torch::Tensor uniq, torch::Tensor inverse,
    torch::Tensor n_uniq, torch::Tensor hot2cidx, torch::Tensor n_hot,
    torch::Tensor d_ctx, int64_t off0, int64_t off1, int64_t n_seg,
    int64_t d, torch::Tensor m, torch::Tensor v, int64_t step, double lr,
    double beta1, double beta2, double eps, torch::Tensor lrt_t) {
  CHECK_DEV(p); CHECK_CONT(p); CHECK_DEV(d_ctx); CHECK_CONT(d_ctx);
  const float* lrt_ptr = (lrt_t.defined() && lrt_t.numel() == 1)
                             ? lrt_t.data_ptr<float>() : nullptr;
  const long n = inverse.numel();
  const long n_per_seg = d_ctx.size(0);
  TORCH_CHECK(n == n_per_seg * n_seg, "ids length mismatch");
  auto st = state_from(uniq, inverse, n_uniq, hot2cidx, n_hot);
  auto acc = accum_ctx_common(st, d_ctx, (int)off0, (int)off1, n_per_seg,
                              (int)n_seg, (int)d);
  const float lr_t = (float)(lr * std::sqrt(1.0 - std::pow(beta2, (double)step)) /
                             (1.0 - std::pow(beta1, (double)step)));
  k_adam_rows_dyn<<<grid_1d(n * d, 256), 256, 0, cur_stream()>>>(
      p.data_ptr<float>(), st.uniq.data_ptr<long>(), acc.data_ptr<float>(),
      m.data_ptr<float>(), v.data_ptr<float>(), nullptr,
      st.n_uniq.data_ptr<int>(), (int)d, lr_t, (float)beta1, (float)beta2,
      (float)eps, lrt_ptr);
}

std::vector<torch::Tensor> sparse_dedup_sum_ctx_pre(
    torch::Tensor uniq, torch::Tensor inverse, torch::Tensor n_uniq,
    torch::Tensor hot2cidx, torch::Tensor n_hot, torch::Tensor d_ctx,
    int64_t off0, int64_t off1, int64_t n_seg, int64_t d) {
  CHECK_DEV(d_ctx); CHECK_CONT(d_ctx);
  const long n = inverse.numel();
  const long n_per_seg = d_ctx.size(0);
  TORCH_CHECK(n == n_per_seg * n_seg, "ids length mismatch");
  auto st = state_from(uniq, inverse, n_uniq, hot2cidx, n_hot);
  auto acc = accum_ctx_common(st, d_ctx, (int)off0, (int)off1, n_per_seg,
                              (int)n_seg, (int)d);
  return {st.uniq, acc, st.n_uniq};
}

std::vector<torch::Tensor> sparse_dedup_sum_ctx(torch::Tensor ids,
                                                torch::Tensor d_ctx,
                                                int64_t off0, int64_t off1,
                                                int64_t n_seg, int64_t d) {
  CHECK_DEV(d_ctx); CHECK_CONT(d_ctx);
  auto ids_c = ids.contiguous();
  const long n = ids_c.numel();
  const long n_per_seg = d_ctx.size(0);
  TORCH_CHECK(n == n_per_seg * n_seg, "ids length mismatch");
  auto st = hash_dedup_ids(ids_c);
  auto acc = accum_ctx_common(st, d_ctx, (int)off0, (int)off1, n_per_seg,
                              (int)n_seg, (int)d);
  return {st.uniq, acc, st.n_uniq};
}

std::vector<torch::Tensor> sparse_dedup_sum_rows(torch::Tensor ids,
                                                 torch::Tensor rows) {
  CHECK_DEV(rows);
  auto ids_c = ids.contiguous();
  auto rows_c = rows.contiguous();
  const long n = ids_c.numel();
  const int d = rows_c.size(1);
  TORCH_CHECK(rows_c.size(0) == n, "row/id count mismatch");
  auto st = hash_dedup_ids(ids_c);
  auto acc = accum_rows_common(st, rows_c, n, d);
  return {st.uniq, acc, st.n_uniq};
}

torch::Tensor adam_lrt(torch::Tensor step_t, double lr, double beta1,
                       double beta2) {
  CHECK_DEV(step_t);
  auto out = torch::empty({1}, step_t.options().dtype(torch::kFloat32));
  if (step_t.scalar_type() == torch::kInt64)
    k_adam_lrt<long><<<1, 1, 0, cur_stream()>>>(
        step_t.data_ptr<long>(), out.data_ptr<float>(), (float)lr,
        (float)std::log(beta1), (float)std::log(beta2));
  else
    k_adam_lrt<int><<<1, 1, 0, cur_stream()>>>(
        step_t.data_ptr<int>(), out.data_ptr<float>(), (float)lr,
        (float)std::log(beta1), (float)std::log(beta2));
  return out;
}

std::vector<torch::Tensor> sampled_ce_fwd(torch::Tensor logits_cand,
                                          torch::Tensor labels,
                                          torch::Tensor sampled,
                                          int64_t vocab) {
  CHECK_DEV(logits_cand); CHECK_CONT(logits_cand);
  const int B = logits_cand.size(0);
  const int S = (int)sampled.numel();
  TORCH_CHECK(logits_cand.size(1) == B + S, "candidate layout mismatch");
  auto labels_c = labels.contiguous();
  auto sampled_c = sampled.contiguous();
  const float sol = (float)((double)S / std::log((double)vocab + 1.0));
  auto loss = torch::empty({B}, logits_cand.options().dtype(torch::kFloat32));
  auto lse = torch::empty({B}, logits_cand.options().dtype(torch::kFloat32));
  k_sampled_ce_fwd<<<B, 256, 0, cur_stream()>>>(
      bf_ptr(logits_cand), labels_c.data_ptr<long>(),
      sampled_c.data_ptr<long>(), sol,
      loss.data_ptr<float>(), lse.data_ptr<float>(), B, S);
  return {loss, lse};
}

torch::Tensor sampled_ce_bwd(torch::Tensor logits_cand, torch::Tensor labels,
                             torch::Tensor sampled, int64_t vocab,
                             torch::Tensor lse, double scale) {
  CHECK_DEV(logits_cand); CHECK_CONT(logits_cand);
  const int B = logits_cand.size(0);
  const int S = (int)sampled.numel();
  auto labels_c = labels.contiguous();
  auto sampled_c = sampled.contiguous();
  const float sol = (float)((double)S / std::log((double)vocab + 1.0));
  // torch::empty, not zeros: the kernel writes every column (blockIdx.x==0
  // zeroes the B true-label columns), saving the 10 MB fill launch
  auto d = torch::empty_like(logits_cand);
  dim3 grid(grid_1d(S, 256, 32), B);
  k_sampled_ce_bwd<<<grid, 256, 0, cur_stream()>>>(
      bf_ptr(logits_cand), labels_c.data_ptr<long>(),
      sampled_c.data_ptr<long>(), sol,
      lse.data_ptr<float>(), bf_ptr_mut(d), (float)scale, B, S);
  return d;
}

}  // namespace

// defined with their kernels, in files of their own
void bind_gated(pybind11::module_& mod);
void bind_mxfp4(pybind11::module_& mod);

PYBIND11_MODULE(TORCH_EXTENSION_NAME, mod) {
  bind_gated(mod);
  bind_mxfp4(mod);
  mod.def("gather_concat_fwd", &gather_concat_fwd);
  mod.def("gather_concat_bwd", &gather_concat_bwd);
  mod.def("transform_tanh_fwd", &transform_tanh_fwd);
  mod.def("gemm_bt_bf16", &gemm_bt_bf16);
  mod.def("gemm_bt_v", &gemm_bt_v);
  mod.def("gemm_bt_dropout", &gemm_bt_dropout);
  mod.def("logits_ce_fused", &logits_ce_fused);
  mod.def("gemm_nn_splitk", &gemm_nn_splitk);
  mod.def("gemm_bt_gather", &gemm_bt_gather);
  mod.def("gemm_nn_splitk_gather", &gemm_nn_splitk_gather);
  mod.def("gemm_tn_bf16", &gemm_tn_bf16);
  mod.def("gemm_tn_ce", &gemm_tn_ce);
  mod.def("gemm_tn_splitk", &gemm_tn_splitk);
  mod.def("gemm_nn_splitk_ce", &gemm_nn_splitk_ce);
  mod.def("gemm_nn_splitk_ce_write", &gemm_nn_splitk_ce_write);
  mod.def("tanh_bwd_mul", &tanh_bwd_mul);
  mod.def("attention_fwd", &attention_fwd);
  mod.def("attention_bwd", &attention_bwd);
  mod.def("ce_fwd", &ce_fwd);
  mod.def("ce_bwd", &ce_bwd);
  mod.def("adam_dense_step", &adam_dense_step);
  mod.def("adam_lrt", &adam_lrt);
  mod.def("adam_sparse_rows_step", &adam_sparse_rows_step);
  mod.def("adam_sparse_rows_hash", &adam_sparse_rows_hash);
  mod.def("adam_sparse_rows_hash_ctx", &adam_sparse_rows_hash_ctx);
  mod.def("sparse_dedup_sum_ctx", &sparse_dedup_sum_ctx);
  mod.def("sparse_hash_build", &sparse_hash_build);
  mod.def("adam_sparse_rows_hash_ctx_pre", &adam_sparse_rows_hash_ctx_pre);
  mod.def("sparse_dedup_sum_ctx_pre", &sparse_dedup_sum_ctx_pre);
  mod.def("sparse_dedup_sum_rows", &sparse_dedup_sum_rows);
  mod.def("sampled_ce_fwd", &sampled_ce_fwd);
  mod.def("sampled_ce_bwd", &sampled_ce_bwd);
  mod.def("topk", &topk);
}
