// Microscaled 4-bit floating point (MXFP4) on gfx950: quantisation and
// products.
//
// A row is cut into blocks of 32 values. A block is held as one power of two
// (an exponent byte, 2^(byte - 127)) and 32 codes of 4 bits, each a sign and
// one of 0, .5, 1, 1.5, 2, 3, 4, 6. Two codes share a byte, the even one in
// the low half. Rows whose length is no multiple of 32 end in a block filled
// up with zeros. Byte 255 stands for a block that held a NaN or an infinity:
// all its values are NaN.

#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>

#include "c2v_device.h"

namespace {

// vectors at any address of their element's type
using u16x8_any = u16x8 __attribute__((aligned(2)));
using f32x4_any = f32x4 __attribute__((aligned(4)));

DEVI float scale_of(u32 byte) {
  // what the conversion instructions read of a scale is its exponent field,
  // so byte 0 does mean 2^-127 to them
  return __builtin_bit_cast(float, byte << 23);
}

// eight codes of one block as bf16: exact, a code has two significant bits
DEVI bf16x8 decode8(u32 codes, float scale) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3);
  const bf16x4 lo = __builtin_shufflevector(a, b, 0, 1, 2, 3);
  const bf16x4 hi = __builtin_shufflevector(c, d, 0, 1, 2, 3);
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// ---------------------------------------------------------------------------
// Quantisation. Four lanes share a block, eight values each. The exponent is
// that of the block's largest magnitude less two (so that it lands in 4..8
// and saturates to 6); it is taken from the bits, whose order as integers is
// that of the magnitudes, with infinities and NaN on top. The conversion
// instruction rounds to nearest, ties to the even code.
// ---------------------------------------------------------------------------

template <bool F32>
__launch_bounds__(256)
__global__ void k_mxfp4_quantize(const void* __restrict__ x, long ldx,
                                 u32* __restrict__ codes,
                                 uint8_t* __restrict__ scales, long R, int K,
                                 int nb, int vec) {
  const long per_row = (long)nb * 4, total = R * per_row;
  // whole wavefronts stay in the loop together: the shuffles need all lanes
  for (long base = (long)blockIdx.x * 256; base < total;
       base += (long)gridDim.x * 256) {
    const long t = base + threadIdx.x;
    const long r = t / per_row;
    const int k = (int)(t - r * per_row) * 8;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (t < total) {
      if constexpr (F32) {
        const float* p = reinterpret_cast<const float*>(x) + r * ldx + k;
        if (vec && k + 8 <= K) {
          const f32x4 a = *reinterpret_cast<const f32x4*>(p);
          const f32x4 b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
          for (int j = 0; j < 4; ++j) { v[j] = a[j]; v[4 + j] = b[j]; }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) if (k + j < K) v[j] = p[j];
        }
      } else {
        const ushort* p = reinterpret_cast<const ushort*>(x) + r * ldx + k;
        if (vec && k + 8 <= K) {
          const u16x8 a = *reinterpret_cast<const u16x8*>(p);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = bf2f(a[j]);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) if (k + j < K) v[j] = bf2f(p[j]);
        }
      }
    }
    u32 top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      top = max(top, __builtin_bit_cast(u32, v[j]) & 0x7FFFFFFFu);
    top = max(top, (u32)__shfl_xor((int)top, 1, 64));
    top = max(top, (u32)__shfl_xor((int)top, 2, 64));
    const int field = (int)(top >> 23);
    const bool bad = field == 255;
    const u32 byte = bad ? 255u : (u32)max(field - 2, 0);
    const float s = scale_of(byte);
    u32 c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], s, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], s, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], s, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], s, 3);
    if (t < total) {
      codes[t] = bad ? 0u : c;
      if ((t & 3) == 0) scales[t >> 2] = (uint8_t)byte;
    }
  }
}

template <bool F32>
__launch_bounds__(256)
__global__ void k_mxfp4_dequantize(const u32* __restrict__ codes,
                                   const uint8_t* __restrict__ scales,
                                   void* __restrict__ out, long R, int K,
                                   int nb) {
  const int per_row = (K + 7) / 8;
  const long total = R * per_row;
  for (long t = (long)blockIdx.x * 256 + threadIdx.x; t < total;
       t += (long)gridDim.x * 256) {
    const long r = t / per_row;
    const int c8 = (int)(t - r * per_row), k = c8 * 8;
    const bf16x8 v = decode8(codes[r * nb * 4 + c8],
                             scale_of(scales[r * nb + (c8 >> 2)]));
    if constexpr (F32) {
      float* o = reinterpret_cast<float*>(out) + r * K + k;
      f32x4 a, b;
#pragma unroll
      for (int j = 0; j < 4; ++j) { a[j] = (float)v[j]; b[j] = (float)v[4 + j]; }
      if (k + 8 <= K) {
        *reinterpret_cast<f32x4_any*>(o) = a;
        *reinterpret_cast<f32x4_any*>(o + 4) = b;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) if (k + j < K) o[j] = (float)v[j];
      }
    } else {
      ushort* o = reinterpret_cast<ushort*>(out) + r * K + k;
      const u16x8 a = __builtin_bit_cast(u16x8, v);
      if (k + 8 <= K) {
        *reinterpret_cast<u16x8_any*>(o) = a;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) if (k + j < K) o[j] = a[j];
      }
    }
  }
}

// ---------------------------------------------------------------------------
// y[n][m] = sum_k x[n][k] w[m][k], w in MXFP4, x in bf16 or in MXFP4.
//
// A block keeps a tile of x in LDS and walks over rows of w, which go from
// memory into registers in their packed form and are decoded there (x in
// bf16) or fed to the scaled matrix instruction as they are (x in MXFP4).
// Nothing but the tile of x is shared by the waves, so the walk has no
// barrier. Rows of w are the matrix instruction's A operand, in such an order
// that a lane ends up with 4*MT consecutive columns of one row of y.
//
// Lane (i, q) holds block 4s + q of its row in step s of 128 values: for x in
// bf16 sub-step j multiplies values 8j..8j+7 of that block.
//
// Large products are bound by writing y, and y's rows need not start on a
// cache line. Lines that are written in two halves halve the rate, so a tile
// takes rows that all lie the same way: every `period`-th one. The columns of
// its passes then begin on lines, `shift` columns before those of row 0 of
// the table (the first pass has columns below zero, which are not stored).
// ---------------------------------------------------------------------------

struct MxArgs {
  const ushort* x;            // bf16 (N, K), rows ldx apart; or null
  long ldx;
  const uint8_t* xc;          // codes (N, 16 nb) and scales (N, nb) of x; or null
  const uint8_t* xs;
  const uint8_t* wc;          // (M, 16 nb)
  const uint8_t* ws;          // (M, nb)
  void* y;                    // (N, M)
  int N, M, K, nb;
  int kc;                     // values of a row of x in LDS, a multiple of 128
  int period, n_tiles;        // tiles of x: n_tiles, a multiple of period
  int chunks_each;            // passes over rows of w a block
  int vec;                    // x can be read 16 bytes at a time
};

constexpr int MX_WAVES = 4;

template <bool X4, bool OUT32, int XT, int MT>
__launch_bounds__(MX_WAVES * 64, XT == 1 ? 4 : 3)
__global__ void k_mxfp4_rows(MxArgs p) {
  constexpr int T = MX_WAVES * 64;
  constexpr int ROWS = XT * 16;                // rows of x a block
  constexpr int CHUNK = MX_WAVES * MT * 16;    // rows of w a pass
  constexpr int ES = OUT32 ? 4 : 2;
  extern __shared__ uint8_t sm[];
  // an odd number of 16-byte units a row, so that 8 rows lie on all banks
  const int stride = (X4 ? p.kc / 2 : p.kc * 2) + 16;
  const int kb = p.kc / 32;
  uint8_t* sm_scales = sm + ROWS * stride;     // X4: (ROWS, kb)

  const int b = xcd_chunked(blockIdx.x, gridDim.x);
  const int tile = b % p.n_tiles;
  const int n0 = tile % p.period + tile / p.period * ROWS * p.period;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, q = lane >> 4;

  const int shift = p.period == 1 ? 0 :
      (int)(((u64)p.y + (u64)n0 * p.M * ES) & 127) / ES;
  const int chunks = (p.M + shift + CHUNK - 1) / CHUNK;
  const int chunk0 = b / p.n_tiles * p.chunks_each;
  const int chunk1 = min(chunk0 + p.chunks_each, chunks);
  const int k_chunks = (p.nb + kb - 1) / kb;

  auto stage = [&](int b0) {    // blocks b0 .. b0 + kb of the rows into LDS
    if constexpr (X4) {
      for (int c = tid; c < ROWS * kb; c += T) {
        const int r = c / kb, blk = c % kb;
        const long n = n0 + (long)r * p.period;
        u32x4 v = {0u, 0u, 0u, 0u};
        uint8_t s = 127;
        if (n < p.N && b0 + blk < p.nb) {
          const long at = n * p.nb + b0 + blk;
          v = *reinterpret_cast<const u32x4*>(p.xc + at * 16);
          s = p.xs[at];
        }
        *reinterpret_cast<u32x4*>(sm + r * stride + blk * 16) = v;
        sm_scales[r * kb + blk] = s;
      }
    } else {
      const int c8 = p.kc / 8;
      for (int c = tid; c < ROWS * c8; c += T) {
        const int r = c / c8, k = b0 * 32 + c % c8 * 8;
        const long n = n0 + (long)r * p.period;
        u16x8 v = {};
        if (n < p.N) {
          const ushort* s = p.x + n * p.ldx + k;
          if (p.vec && k + 8 <= p.K) {
            v = *reinterpret_cast<const u16x8*>(s);
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) if (k + j < p.K) v[j] = s[j];
          }
        }
        *reinterpret_cast<u16x8*>(sm + r * stride + c % c8 * 16) = v;
      }
    }
  };

  // Rows of w of this lane in a pass, and what it holds of them in a step.
  // A step behind a row's last block repeats that block's codes: x has zeros
  // there, and the scale is made harmless.
  const int row_in = wid * MT * 16 + (l16 >> 2) * (4 * MT) + (l16 & 3);
  struct Held { u32x4 c[MT]; u32 s[MT]; };
  auto load = [&](int ch, int blk, Held& h) {
    const int m0 = ch * CHUNK - shift + row_in;
    const int at = min(blk, p.nb - 1);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const u64 i = (u64)max(0, min(m0 + t * 4, p.M - 1)) * p.nb + at;
      h.c[t] = *reinterpret_cast<const u32x4*>(p.wc + i * 16);
      const u32 s = p.ws[i];
      h.s[t] = blk < p.nb ? s : 127;
    }
  };

  f32x4 acc[XT][MT];
  auto clear = [&] {
#pragma unroll
    for (int i = 0; i < XT; ++i)
#pragma unroll
      for (int t = 0; t < MT; ++t) acc[i][t] = {0.f, 0.f, 0.f, 0.f};
  };
  auto step = [&](int s, const Held& h) {
    if constexpr (X4) {
      i32x8 xf[XT];
      int xsc[XT];
#pragma unroll
      for (int i = 0; i < XT; ++i) {
        const int r = i * 16 + l16;
        const u32x4 v = *reinterpret_cast<const u32x4*>(
            sm + r * stride + (s * 4 + q) * 16);
        xf[i] = i32x8{(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0};
        xsc[i] = sm_scales[r * kb + s * 4 + q];
      }
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const i32x8 wf = {(int)h.c[t][0], (int)h.c[t][1], (int)h.c[t][2],
                          (int)h.c[t][3], 0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < XT; ++i)
          acc[i][t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
              wf, xf[i], acc[i][t], 4, 4, 0, (int)h.s[t], 0, xsc[i]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        bf16x8 xf[XT];
#pragma unroll
        for (int i = 0; i < XT; ++i)
          xf[i] = *reinterpret_cast<const bf16x8*>(
              sm + (i * 16 + l16) * stride + (s * 128 + q * 32 + j * 8) * 2);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          const bf16x8 wf = decode8(h.c[t][j], scale_of(h.s[t]));
#pragma unroll
          for (int i = 0; i < XT; ++i)
            acc[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                wf, xf[i], acc[i][t], 0, 0, 0);
        }
      }
    }
  };
  auto store = [&](int ch) {
    const int m = ch * CHUNK - shift + wid * MT * 16 + q * 4 * MT;
#pragma unroll
    for (int i = 0; i < XT; ++i) {
      const long n = n0 + (long)(i * 16 + l16) * p.period;
      if (n >= p.N) continue;
      if constexpr (OUT32) {
        float* o = reinterpret_cast<float*>(p.y) + n * p.M + m;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          if (m + t * 4 >= 0 && m + t * 4 + 4 <= p.M) {
            *reinterpret_cast<f32x4_any*>(o + t * 4) = acc[i][t];
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if ((u32)(m + t * 4 + r) < (u32)p.M) o[t * 4 + r] = acc[i][t][r];
          }
        }
      } else {
        ushort* o = reinterpret_cast<ushort*>(p.y) + n * p.M + m;
#pragma unroll
        for (int t = 0; t < MT; t += 2) {
          bf16x8 v8;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            v8[r] = (__bf16)acc[i][t][r];
            v8[4 + r] = (__bf16)acc[i][t + 1][r];
          }
          const u16x8 v = __builtin_bit_cast(u16x8, v8);
          if (m + t * 4 >= 0 && m + t * 4 + 8 <= p.M) {
            *reinterpret_cast<u16x8_any*>(o + t * 4) = v;
          } else {
#pragma unroll
            for (int r = 0; r < 8; ++r)
              if ((u32)(m + t * 4 + r) < (u32)p.M) o[t * 4 + r] = v[r];
          }
        }
      }
    }
  };

  if (chunk0 >= chunk1) return;
  // one step ahead of the matrix instructions, over the ends of passes
  Held now, next;
  load(chunk0, q, now);
  if (k_chunks == 1) {
    const int steps = (p.nb + 3) / 4;
    stage(0);
    __syncthreads();
    for (int ch = chunk0; ch < chunk1; ++ch) {
      clear();
#pragma unroll 1
      for (int s = 0; s < steps; ++s) {
        const bool end = s + 1 == steps;
        // behind the last pass: its rows once more
        load(end ? min(ch + 1, chunk1 - 1) : ch, (end ? 0 : s + 1) * 4 + q, next);
        step(s, now);
        now = next;
      }
      store(ch);
    }
  } else {
    for (int ch = chunk0; ch < chunk1; ++ch) {
      clear();
      for (int b0 = 0; b0 < p.nb; b0 += kb) {
        __syncthreads();
        stage(b0);
        __syncthreads();
        const int steps = (min(kb, p.nb - b0) + 3) / 4;
#pragma unroll 1
        for (int s = 0; s < steps; ++s) {
          const int blk = b0 + (s + 1) * 4;
          const bool end = blk >= p.nb;
          load(end ? min(ch + 1, chunk1 - 1) : ch, (end ? 0 : blk) + q, next);
          step(s, now);
          now = next;
        }
      }
      store(ch);
    }
  }
}

// ===========================================================================
// host wrappers
// ===========================================================================

inline hipStream_t cur_stream() {
  return at::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream();
}

inline int grid_of(long items, int block, long cap) {
  return (int)std::max(1L, std::min((items + block - 1) / block, cap));
}

using Guard = c10::hip::OptionalHIPGuardMasqueradingAsCUDA;

std::vector<torch::Tensor> mxfp4_quantize(torch::Tensor x) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2, "x must be (rows, K) on a GPU");
  const bool f32 = x.scalar_type() == torch::kFloat32;
  TORCH_CHECK(f32 || x.scalar_type() == torch::kBFloat16,
              "x must be float32 or bfloat16");
  TORCH_CHECK(x.size(1) < (1L << 30), "rows of x are too long");
  const Guard guard(x.device());
  const long R = x.size(0);
  const int K = x.size(1), nb = (K + 31) / 32;
  auto codes = torch::empty({R, nb * 16L}, x.options().dtype(torch::kUInt8));
  auto scales = torch::empty({R, (long)nb}, x.options().dtype(torch::kUInt8));
  if (R == 0 || K == 0) return {codes, scales};
  auto src = K == 1 || x.stride(1) == 1 ? x : x.contiguous();
  const long ld = R == 1 ? K : src.stride(0);
  const int vec = (ld % (f32 ? 4 : 8)) == 0 &&
                  (reinterpret_cast<uintptr_t>(src.data_ptr()) & 15) == 0;
  const int grid = grid_of(R * nb * 4, 256, 16384);
  auto* fn = f32 ? &k_mxfp4_quantize<true> : &k_mxfp4_quantize<false>;
  fn<<<grid, 256, 0, cur_stream()>>>(
      src.data_ptr(), ld, reinterpret_cast<u32*>(codes.data_ptr()),
      scales.data_ptr<uint8_t>(), R, K, nb, vec);
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return {codes, scales};
}

// codes (rows, 16 nb) and scales (rows, nb) of rows of K values
void check_mx(const torch::Tensor& codes, const torch::Tensor& scales, long K,
              const char* name) {
  const long nb = (K + 31) / 32;
  TORCH_CHECK(codes.is_cuda() && scales.device() == codes.device(), name,
              " must be on one GPU");
  TORCH_CHECK(codes.scalar_type() == torch::kUInt8 &&
              scales.scalar_type() == torch::kUInt8, name, " must be uint8");
  TORCH_CHECK(codes.dim() == 2 && scales.dim() == 2 &&
              codes.size(0) == scales.size(0) && scales.size(1) == nb &&
              codes.size(1) == 16 * nb, name, " does not hold rows of ", K);
  TORCH_CHECK(codes.is_contiguous() && scales.is_contiguous() &&
              (reinterpret_cast<uintptr_t>(codes.data_ptr()) & 15) == 0,
              name, " must be contiguous and start on 16 bytes");
  TORCH_CHECK(codes.size(0) < (1L << 30) && K < (1L << 30), name, " is too large");
}

torch::Tensor mxfp4_dequantize(torch::Tensor codes, torch::Tensor scales,
                               int64_t K, bool f32) {
  check_mx(codes, scales, K, "q");
  const Guard guard(codes.device());
  const long R = codes.size(0);
  auto out = torch::empty({R, K}, codes.options().dtype(
      f32 ? torch::kFloat32 : torch::kBFloat16));
  if (R == 0 || K == 0) return out;
  const int grid = grid_of(R * ((K + 7) / 8), 256, 16384);
  auto* fn = f32 ? &k_mxfp4_dequantize<true> : &k_mxfp4_dequantize<false>;
  fn<<<grid, 256, 0, cur_stream()>>>(
      reinterpret_cast<const u32*>(codes.data_ptr()), scales.data_ptr<uint8_t>(),
      out.data_ptr(), R, (int)K, (int)scales.size(1));
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return out;
}

template <bool X4, bool OUT32, int XT, int MT>
void launch_mx(MxArgs a) {
  constexpr int ROWS = XT * 16, CHUNK = MX_WAVES * MT * 16;
  // what of a row of x fits LDS: all of it, or a part
  const int most = X4 ? 2048 : (XT == 4 ? 512 : 1024);
  a.kc = std::min((a.nb * 32 + 127) / 128 * 128, most);
  const size_t bytes = (size_t)ROWS * ((X4 ? a.kc / 2 : a.kc * 2) + 16) +
                       (X4 ? (size_t)ROWS * (a.kc / 32) : 0);
  const int per = (a.N + a.period - 1) / a.period;
  a.n_tiles = a.period * ((per + ROWS - 1) / ROWS);
  const int chunks = (int)(((long)a.M + (a.period > 1 ? 63 : 0) + CHUNK - 1) / CHUNK);
  const int want = std::max(1, (768 + a.n_tiles - 1) / a.n_tiles);
  a.chunks_each = (chunks + want - 1) / want;
  const long blocks = (long)a.n_tiles * ((chunks + a.chunks_each - 1) / a.chunks_each);
  auto* fn = &k_mxfp4_rows<X4, OUT32, XT, MT>;
  if (bytes > 64 * 1024)
    C10_HIP_CHECK(hipFuncSetAttribute((const void*)fn,
                                      hipFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)bytes));
  TORCH_CHECK(blocks < (1L << 31), "too many tiles");
  fn<<<(int)blocks, MX_WAVES * 64, bytes, cur_stream()>>>(a);
  C10_HIP_KERNEL_LAUNCH_CHECK();
}

template <bool X4, bool OUT32>
void pick_mx(MxArgs a) {
  // rows this many apart start on the same place of a 128-byte line
  const int over = (int)((long)a.M * (OUT32 ? 4 : 2) % 128);
  a.period = 1;
  for (int v = 128; over && v > 1 && over % v; v /= 2) a.period *= 2;
  if (a.N < 16 * a.period) a.period = 1;     // too few of them for a tile
  // a tile costs its rows, and about as much as 16 for the rows of w
  const int per = (a.N + a.period - 1) / a.period;
  auto cost = [&](int xt) { return (per + 16 * xt - 1) / (16 * xt) * (16 * xt + 16); };
  if (cost(1) <= cost(2) && cost(1) <= cost(4)) launch_mx<X4, OUT32, 1, 4>(a);
  else if (cost(2) <= cost(4)) launch_mx<X4, OUT32, 2, 4>(a);
  else launch_mx<X4, OUT32, 4, 4>(a);
}

// x: bf16 (N, K) with x_scales empty, or the codes of x and their scales
torch::Tensor mxfp4_matmul(torch::Tensor x, torch::Tensor x_scales,
                           torch::Tensor w_codes, torch::Tensor w_scales,
                           int64_t K, bool f32) {
  check_mx(w_codes, w_scales, K, "w");
  const bool x4 = x.scalar_type() == torch::kUInt8;
  TORCH_CHECK(x.device() == w_codes.device(), "x and w must be on one GPU");
  const Guard guard(x.device());
  torch::Tensor src = x;
  MxArgs a{};
  if (x4) {
    check_mx(x, x_scales, K, "x");
    a.xc = x.data_ptr<uint8_t>();
    a.xs = x_scales.data_ptr<uint8_t>();
  } else {
    TORCH_CHECK(x.scalar_type() == torch::kBFloat16 && x.dim() == 2 &&
                x.size(1) == K, "x must be a bfloat16 (N, K)");
    TORCH_CHECK(x.size(0) < (1L << 30), "x is too large");
    if (K > 1 && x.stride(1) != 1) src = x.contiguous();
    a.x = reinterpret_cast<const ushort*>(src.data_ptr<at::BFloat16>());
    a.ldx = x.size(0) == 1 ? K : src.stride(0);
    a.vec = a.ldx % 8 == 0 && (reinterpret_cast<uintptr_t>(a.x) & 15) == 0;
  }
  a.N = x.size(0);
  a.M = w_codes.size(0);
  a.K = K;
  a.nb = w_scales.size(1);
  a.wc = w_codes.data_ptr<uint8_t>();
  a.ws = w_scales.data_ptr<uint8_t>();
  auto y = torch::empty({a.N, a.M}, w_codes.options().dtype(
      f32 ? torch::kFloat32 : torch::kBFloat16));
  a.y = y.data_ptr();
  if (a.N == 0 || a.M == 0) return y;
  if (K == 0) return y.zero_();
  if (x4) { if (f32) pick_mx<true, true>(a); else pick_mx<true, false>(a); }
  else { if (f32) pick_mx<false, true>(a); else pick_mx<false, false>(a); }
  return y;
}

}  // namespace

void bind_mxfp4(pybind11::module_& mod) {
  mod.def("mxfp4_quantize", &mxfp4_quantize);
  mod.def("mxfp4_dequantize", &mxfp4_dequantize);
  mod.def("mxfp4_matmul", &mxfp4_matmul);
}
