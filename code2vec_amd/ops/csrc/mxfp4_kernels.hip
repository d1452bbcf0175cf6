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

#include <type_traits>

#include "c2v_device.h"

namespace {

// vectors at any address of their element's type
using u16x8_any = u16x8 __attribute__((aligned(2)));
using f32x4_any = f32x4 __attribute__((aligned(4)));
using u32x4_any = u32x4 __attribute__((aligned(2)));

DEVI float scale_of(u32 byte) {
  // what the conversion instructions read of a scale is its exponent field,
  // so byte 0 does mean 2^-127 to them
  return __builtin_bit_cast(float, byte << 23);
}

// keeps a pointer in scalar registers, so that lanes add 32-bit offsets to it
template <typename P>
DEVI P* in_scalar(P* p) {
  const u64 v = (u64)p;
  u32 lo = __builtin_amdgcn_readfirstlane((u32)v);
  u32 hi = __builtin_amdgcn_readfirstlane((u32)(v >> 32));
  u64 w = (u64)hi << 32 | lo;
  asm("" : "+s"(w));
  return (P*)w;
}

DEVI u16x8 pack8(f32x4 a, f32x4 b) {
  bf16x8 v;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    v[r] = (__bf16)a[r];
    v[4 + r] = (__bf16)b[r];
  }
  return __builtin_bit_cast(u16x8, v);
}

// each lane's 16 (or 4) bytes to LDS, one lane's behind the other's
template <int BYTES>
DEVI void to_lds(const uint8_t* src, uint8_t* dst) {
  const auto* s = (const __attribute__((address_space(1))) u32*)src;
  auto* d = (__attribute__((address_space(3))) u32*)dst;
  if constexpr (BYTES == 16) __builtin_amdgcn_global_load_lds(s, d, 16, 0, 0);
  else __builtin_amdgcn_global_load_lds(s, d, 4, 0, 0);
}

// A barrier after which no more than A (or, where `more`, B) of this wave's
// loads and stores are outstanding, and nothing that it reads from LDS.
template <int A, int B>
DEVI void wait_queue(bool more) {
  static_assert(A < 64 && B < 64, "vmcnt has 6 bits");
  // vmcnt in bits 3:0 and 15:14, expcnt 6:4 (no wait), lgkmcnt 11:8 (zero)
  constexpr int a = 0x70 | (A & 15) | (A >> 4 << 14), b = 0x70 | (B & 15) | (B >> 4 << 14);
  asm volatile("" ::: "memory");
  if (more) __builtin_amdgcn_s_waitcnt(b);
  else __builtin_amdgcn_s_waitcnt(a);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
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
// Rows of w are the matrix instruction's A operand, in such an order that a
// lane ends up with 16 consecutive columns of one row of y for every 16 rows
// of x.
//
// Lane (i, q) holds block 4s + q of its row in step s of 128 values: for x in
// bf16 sub-step j multiplies values 8j..8j+7 of that block.
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
  int n_tiles;                // tiles of rows of x
  int passes_each;            // passes over rows of w a block
  int vec;                    // x can be read 16 bytes at a time
};

constexpr int MT = 4;         // 16-row tiles of w a wave

// the 16 bytes of unit u (a block in MXFP4, eight values in bf16) of row n of
// x, and a block's scale; zeros and one behind the row's end
template <bool X4>
DEVI u32x4 x_unit(const MxArgs& p, long n, int u, u32& scale) {
  u32x4 v = {0u, 0u, 0u, 0u};
  scale = 127;
  if constexpr (X4) {
    if (u < p.nb) {
      v = *reinterpret_cast<const u32x4*>(p.xc + (n * p.nb + u) * 16);
      scale = p.xs[n * p.nb + u];
    }
  } else {
    const ushort* s = p.x + n * p.ldx + u * 8;
    if (p.vec && u * 8 + 8 <= p.K) {
      v = *reinterpret_cast<const u32x4*>(s);
    } else {
      u16x8 e = {};
#pragma unroll
      for (int j = 0; j < 8; ++j) if (u * 8 + j < p.K) e[j] = s[j];
      v = __builtin_bit_cast(u32x4, e);
    }
  }
  return v;
}

// what a lane holds of its MT rows of w in a step: codes, and scales as bytes
struct Held { u32x4 c[MT]; u32 s[MT]; };

// One step of 128 values. `x` and `xsc` point at this lane's unit of row 0 of
// the tile in LDS; rows are `stride` and `kb` bytes apart.
template <bool X4, int XT>
DEVI void mx_step(const Held& h, const uint8_t* x, const uint8_t* xsc,
                  int stride, int kb, f32x4 (&acc)[XT][MT]) {
  if constexpr (X4) {
#pragma unroll
    for (int i = 0; i < XT; ++i) {
      const u32x4 v = *reinterpret_cast<const u32x4*>(x + i * 16 * stride);
      const int sc = xsc[i * 16 * kb];
      const i32x8 xf = {(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0};
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const i32x8 wf = {(int)h.c[t][0], (int)h.c[t][1], (int)h.c[t][2],
                          (int)h.c[t][3], 0, 0, 0, 0};
        acc[i][t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
            wf, xf, acc[i][t], 4, 4, 0, (int)h.s[t], 0, sc);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      bf16x8 wf[MT];
#pragma unroll
      for (int t = 0; t < MT; ++t) wf[t] = decode8(h.c[t][j], scale_of(h.s[t]));
#pragma unroll
      for (int i = 0; i < XT; ++i) {
        const bf16x8 xf = *reinterpret_cast<const bf16x8*>(x + i * 16 * stride + j * 16);
#pragma unroll
        for (int t = 0; t < MT; ++t)
          acc[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf[t], xf, acc[i][t],
                                                              0, 0, 0);
      }
      // the next sub-step's operands would only take registers
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}

template <int XT>
DEVI void mx_clear(f32x4 (&acc)[XT][MT]) {
#pragma unroll
  for (int i = 0; i < XT; ++i)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[i][t] = {0.f, 0.f, 0.f, 0.f};
}

// The sums are made here and not where they are used: the compiler would
// otherwise move the products behind the loads that overwrite their operands,
// and keep both. No instruction stands in the asm.
template <int XT>
DEVI void mx_pin(f32x4 (&acc)[XT][MT]) {
#pragma unroll
  for (int i = 0; i < XT; ++i)
#pragma unroll
    for (int t = 0; t < MT; ++t) asm volatile("" : "+v"(acc[i][t]));
}

// Few rows of x, and any K and M. Bound by reading w: four waves of a block
// each go over their own 64 rows, one step ahead of the matrix instructions;
// nothing but the tile of x is shared, so there is no barrier unless rows of
// x do not fit LDS and are brought in parts.
template <bool X4, bool OUT32, int XT>
__launch_bounds__(256, XT == 1 ? 4 : 3)
__global__ void k_mxfp4_rows(MxArgs p) {
  constexpr int T = 256, ROWS = XT * 16, PASS = 4 * MT * 16;
  extern __shared__ uint8_t sm[];
  // an odd number of 16-byte units a row, so that 8 rows lie on all banks
  const int stride = (X4 ? p.kc / 2 : p.kc * 2) + 16;
  const int kb = p.kc / 32;
  uint8_t* sm_scales = sm + ROWS * stride;     // X4: (ROWS, kb)

  const int b = xcd_chunked(blockIdx.x, gridDim.x);
  const int n0 = b % p.n_tiles * ROWS;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, q = lane >> 4;
  const int pass0 = b / p.n_tiles * p.passes_each;
  const int pass1 = min(pass0 + p.passes_each, (p.M + PASS - 1) / PASS);
  if (pass0 >= pass1) return;
  const int k_parts = (p.nb + kb - 1) / kb;

  // A step behind a row's last block repeats that block's codes: x has zeros
  // there, and the scale is made harmless.
  const int row_in = wid * MT * 16 + (l16 >> 2) * (4 * MT) + (l16 & 3);
  auto load = [&](int pass, int blk, Held& h) {
    const int m0 = pass * PASS + row_in;
    const int at = min(blk, p.nb - 1);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const u64 i = (u64)min(m0 + t * 4, p.M - 1) * p.nb + at;
      h.c[t] = *reinterpret_cast<const u32x4*>(p.wc + i * 16);
      const u32 s = p.ws[i];
      h.s[t] = blk < p.nb ? s : 127;
    }
  };

  f32x4 acc[XT][MT];
  Held now, next;
  load(pass0, q, now);
  for (int pass = pass0; pass < pass1; ++pass) {
    mx_clear(acc);
    for (int b0 = 0; b0 < p.nb; b0 += kb) {
      if (k_parts > 1 || pass == pass0) {
        __syncthreads();
        const int units = X4 ? kb : kb * 4;
        for (int c = tid; c < ROWS * units; c += T) {
          const int r = c / units, u = c % units;
          u32 scale = 127;
          u32x4 v = {0u, 0u, 0u, 0u};
          if (n0 + r < p.N) v = x_unit<X4>(p, n0 + r, (X4 ? b0 : b0 * 4) + u, scale);
          *reinterpret_cast<u32x4*>(sm + r * stride + u * 16) = v;
          if (X4) sm_scales[r * kb + u] = (uint8_t)scale;
        }
        __syncthreads();
      }
      const int steps = (min(kb, p.nb - b0) + 3) / 4;
#pragma unroll 1
      for (int s = 0; s < steps; ++s) {
        const int blk = b0 + (s + 1) * 4;
        const bool end = blk >= p.nb;
        // behind the last pass: its rows once more
        load(end ? min(pass + 1, pass1 - 1) : pass, (end ? 0 : blk) + q, next);
        mx_step<X4, XT>(now, sm + l16 * stride + (s * 4 + q) * (X4 ? 16 : 64),
                        sm_scales + l16 * kb + s * 4 + q, stride, kb, acc);
        now = next;
      }
    }
    const int m = pass * PASS + wid * MT * 16 + q * 4 * MT;
#pragma unroll
    for (int i = 0; i < XT; ++i) {
      const long n = n0 + i * 16 + l16;
      if (n >= p.N) continue;
#pragma unroll
      for (int t = 0; t < MT; t += 2) {
        if constexpr (OUT32) {
          float* o = reinterpret_cast<float*>(p.y) + n * p.M + m + t * 4;
          if (m + t * 4 + 8 <= p.M) {
            *reinterpret_cast<f32x4_any*>(o) = acc[i][t];
            *reinterpret_cast<f32x4_any*>(o + 4) = acc[i][t + 1];
          } else {
#pragma unroll
            for (int r = 0; r < 8; ++r)
              if (m + t * 4 + r < p.M) o[r] = acc[i][t + r / 4][r & 3];
          }
        } else {
          ushort* o = reinterpret_cast<ushort*>(p.y) + n * p.M + m + t * 4;
          const u16x8 v = pack8(acc[i][t], acc[i][t + 1]);
          if (m + t * 4 + 8 <= p.M) {
            *reinterpret_cast<u16x8_any*>(o) = v;
          } else {
#pragma unroll
            for (int r = 0; r < 8; ++r)
              if (m + t * 4 + r < p.M) o[r] = v[r];
          }
        }
      }
    }
  }
}

// Many rows of x, of up to 128*R values. What bounds these is the writing of
// y, whose rows need not start on a cache line, and that reads wait behind
// the writes. So:
//
// A wave holds its 16*XT rows of x in registers for good, and rows of w are
// what moves: 64 at a time, through a ring of LDS buffers that the block's
// eight waves share, so that w is read once for 128*XT rows of x.
//
// Lines of y that are written in two halves cost twice (measured on 2.1 GB:
// 950 us as the lanes hold them, 500 us as whole rows of 512, 405 us as whole
// lines). So a wave's 64 columns go through LDS, 16 rows at a time, and whole
// lines go out; what is left behind a row's last line is carried to the next
// pass. Only the ends of a block's columns are written in parts.
//
// A wave's loads and stores are counted in one queue. The wait for a tile of
// w therefore counts the stores after it, which are the same number in every
// pass but a block's first and last: rows behind the last one repeat it.
template <bool X4, bool OUT32, int R>
struct Stream {
  static constexpr int XT = X4 ? 4 : 2;            // 16-row tiles of x a wave
  static constexpr int ES = OUT32 ? 4 : 2;
  static constexpr int ROWS = 8 * XT * 16;         // rows of x a block
  static constexpr int LINE = 128 / ES;
  static constexpr int CROW = (LINE + 64) * ES + 16;   // carried columns, then new
  static constexpr int RING = 64 * 4 * R * 17;     // codes, then scales
  static constexpr int OWN = XT * 16 * 128 + 16 * CROW;
  // tiles of w in LDS: as many as fit, four at most
  static constexpr int DEPTH = (160 * 1024 - 8 * OWN) / RING >= 4   ? 4
                               : (160 * 1024 - 8 * OWN) / RING >= 3 ? 3 : 2;
  static constexpr int BYTES = DEPTH * RING + 8 * OWN;
  static constexpr int STORES = XT * 16 * 64 * ES / 1024;   // a wave and pass
  static constexpr int LOADS = 3;                           // a wave and tile
};

template <bool X4, bool OUT32, int R>
__launch_bounds__(512, 2)
__global__ void k_mxfp4_stream(MxArgs p) {
  using S = Stream<X4, OUT32, R>;
  constexpr int XT = S::XT, ES = S::ES, LINE = S::LINE, CROW = S::CROW, D = S::DEPTH;
  extern __shared__ uint8_t sm[];

  const int b = xcd_chunked(blockIdx.x, gridDim.x);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, q = lane >> 4;
  const int pass0 = b / p.n_tiles * p.passes_each;
  const int pass1 = min(pass0 + p.passes_each, (p.M + 63) / 64);
  if (pass0 >= pass1) return;
  const int n0 = b % p.n_tiles * S::ROWS + wid * XT * 16;    // this wave's
  uint8_t* carry = sm + D * S::RING + wid * S::OWN;          // (16 XT, LINE)
  uint8_t* cbuf = carry + XT * 16 * 128;                     // (16, CROW)

  // Rows of w lie in LDS in the order in which lanes take them: row 16t + i
  // is row 16(i/4) + 4t + i%4 of the 64. A row's 16-byte blocks change places
  // within groups of `group`, the power of two in their number, so that the
  // 16 rows of a read lie on all banks.
  const int nb = p.nb;
  const int group = min(nb & -nb, 16);
  const int fold = __builtin_ctz(16 / group);
  auto key = [&](int row) { return ((row & 15) >> fold) & (group - 1); };
  auto fetch = [&](int pass) {
    const int m0 = min(pass, pass1 - 1) * 64;
    uint8_t* ring = sm + (pass % D) * S::RING;
    const uint8_t* wc = in_scalar(p.wc + (u64)m0 * nb * 16);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      // 64 blocks an instruction, nb instructions a tile; a wave without one
      // repeats another
      const int e = wid + 8 * k < nb ? wid + 8 * k : wid % nb;
      const int u = e * 64 + lane, j = u / nb, at = u % nb;
      const int i = j & 15, row = (i >> 2) * 16 + (j >> 4) * 4 + (i & 3);
      const u32 off = (u32)(min(row, p.M - 1 - m0) * nb + (at ^ key(j))) * 16;
      to_lds<16>(wc + off, ring + e * 1024);
    }
    const int e = wid * 4 < nb ? wid : 0;
    const int whole = (min(64, p.M - m0) * nb) >> 2;       // words of scales
    // (a tile without a whole word: it is filled in below)
    const uint8_t* ws = in_scalar(p.ws + (whole ? (u64)m0 * nb : 0));
    to_lds<4>(ws + (u32)max(0, min(e * 64 + lane, whole - 1)) * 4,
              ring + 64 * 4 * R * 16 + e * 256);
  };

  // x into registers; blocks behind a row's end are zeros
  u32x4 xf[XT][X4 ? R : R * 4];
  u32 xs[XT][R];
#pragma unroll
  for (int i = 0; i < XT; ++i) {
    const int n = min(n0 + i * 16 + l16, p.N - 1);
#pragma unroll
    for (int s = 0; s < R; ++s) {
      if constexpr (X4) {
        xf[i][s] = x_unit<true>(p, n, s * 4 + q, xs[i][s]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          xf[i][s * 4 + j] = x_unit<false>(p, n, (s * 4 + q) * 4 + j, xs[i][s]);
      }
    }
  }
  for (int k = 0; k < D - 1; ++k) fetch(pass0 + k);

  // where this lane finds its block of step s in row l16 of a tile, and its
  // scale; a step may have fewer than four blocks: the others repeat the last
  u32 c_at[R], s_at[R];
#pragma unroll
  for (int s = 0; s < R; ++s) {
    const int blk = min(s * 4 + q, nb - 1);
    c_at[s] = (l16 * nb + (blk ^ key(l16))) * 16;
    s_at[s] = 64 * 4 * R * 16 + ((l16 >> 2) * 16 + (l16 & 3)) * nb + blk;
  }

  f32x4 acc[XT][MT];
  for (int pass = pass0; pass < pass1; ++pass) {
    const int m0 = pass * 64;
    wait_queue<(D - 2) * S::LOADS, (D - 2) * S::LOADS + (D - 1) * S::STORES>(
        pass - pass0 >= D);
    const int odd = pass == (p.M - 1) / 64 ? (p.M - m0) * nb & 3 : 0;
    if (odd) {
      // the table's last scales, where they fill no word
      const int at = ((p.M - m0) * nb & ~3) + tid;
      if (tid < odd)
        sm[(pass % D) * S::RING + 64 * 4 * R * 16 + at] = p.ws[(u64)m0 * nb + at];
      __syncthreads();
    }
    fetch(pass + D - 1);
    asm volatile("" ::: "memory");
    const uint8_t* ring = sm + (pass % D) * S::RING;

    mx_clear(acc);
#pragma unroll
    for (int s = 0; s < R; ++s) {
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const u32x4 c = *reinterpret_cast<const u32x4*>(ring + c_at[s] + t * 256 * nb);
        u32 sc = ring[s_at[s] + t * 4 * nb];
        sc = s * 4 + q < nb ? sc : 127;
        if constexpr (X4) {
          const i32x8 wf = {(int)c[0], (int)c[1], (int)c[2], (int)c[3], 0, 0, 0, 0};
#pragma unroll
          for (int i = 0; i < XT; ++i) {
            const i32x8 xv = {(int)xf[i][s][0], (int)xf[i][s][1], (int)xf[i][s][2],
                              (int)xf[i][s][3], 0, 0, 0, 0};
            acc[i][t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                wf, xv, acc[i][t], 4, 4, 0, (int)sc, 0, (int)xs[i][s]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const bf16x8 wf = decode8(c[j], scale_of(sc));
#pragma unroll
            for (int i = 0; i < XT; ++i)
              acc[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                  wf, __builtin_bit_cast(bf16x8, xf[i][s * 4 + j]), acc[i][t], 0, 0, 0);
          }
        }
      }
    }
    mx_pin(acc);

    // one 16-byte piece of a row a lane, RPI rows an instruction
    constexpr int PER = 16 / ES, LPR = 64 / PER, RPI = 64 / LPR;
    const bool first = pass == pass0, last = pass == pass1 - 1;
    const int end = min(p.M - m0, 64);
    int rl = lane / LPR;
    // addresses are made here, not once for all passes: they would spill
    asm volatile("" : "+v"(rl));
#pragma unroll
    for (int i = 0; i < XT; ++i) {
      uint8_t* mine = cbuf + l16 * CROW + (LINE + q * 16) * ES;
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        if constexpr (OUT32) {
          *reinterpret_cast<f32x4*>(mine + t * 16) = acc[i][t];
        } else if (t % 2 == 0) {
          *reinterpret_cast<u16x8*>(mine + t * 8) = pack8(acc[i][t], acc[i][t + 1]);
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<u32x4*>(cbuf + (h * 8 + (lane >> 3)) * CROW + (lane & 7) * 16) =
            *reinterpret_cast<const u32x4*>(carry + i * 2048 + h * 1024 + lane * 16);
#pragma unroll
      for (int h = 0; h < 16; h += RPI) {
        // column c of the pass is at row + (LINE + c) * ES; those below zero
        // are carried from the pass before
        const uint8_t* row = cbuf + (h + rl) * CROW;
        const int n = min(n0 + i * 16 + h + rl, p.N - 1);
        uint8_t* o = reinterpret_cast<uint8_t*>(p.y) + ((u64)n * p.M + m0) * ES;
        const int tail = (int)((u64)o & 127) / ES;     // the same in all passes
        const int c = lane % LPR * PER - tail;
        if (!first && !last) {
          *reinterpret_cast<u32x4*>(o + (long)c * ES) =
              *reinterpret_cast<const u32x4_any*>(row + (LINE + c) * ES);
        } else {
          if ((c >= 0 || !first) && c + PER <= end)
            *reinterpret_cast<u32x4*>(o + (long)c * ES) =
                *reinterpret_cast<const u32x4_any*>(row + (LINE + c) * ES);
          // the ends of the block's columns, a lane a value
          const int e = lane % LPR;
          auto one = [&](int at) {
            if constexpr (OUT32)
              *reinterpret_cast<float*>(o + (long)at * 4) =
                  *reinterpret_cast<const float*>(row + (LINE + at) * 4);
            else
              *reinterpret_cast<ushort*>(o + (long)at * 2) =
                  *reinterpret_cast<const ushort*>(row + (LINE + at) * 2);
          };
          if (first && e < min((PER - tail % PER) % PER, end)) one(e);
          if (last) {
            // whole pieces of the last line, then what is left of it
            const int c2 = 64 - tail + e * PER;
            if (c2 + PER <= end)
              *reinterpret_cast<u32x4*>(o + (long)c2 * ES) =
                  *reinterpret_cast<const u32x4_any*>(row + (LINE + c2) * ES);
            const int at = (end + tail) / PER * PER - tail + e;
            if (e < PER && (at >= 0 || !first) && at < end) one(at);
          }
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<u32x4*>(carry + i * 2048 + h * 1024 + lane * 16) =
            *reinterpret_cast<const u32x4*>(cbuf + (h * 8 + (lane >> 3)) * CROW +
                                            64 * ES + (lane & 7) * 16);
    }
  }
  // tiles of w that nobody needs may still be on their way into LDS
  __builtin_amdgcn_s_waitcnt(0x0F70);
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
  TORCH_CHECK(x.size(1) < (1L << 20), "rows of x are too long");
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
              (reinterpret_cast<uintptr_t>(codes.data_ptr()) & 15) == 0 &&
              (reinterpret_cast<uintptr_t>(scales.data_ptr()) & 3) == 0, name,
              " must be contiguous and start on 16 bytes, its scales on 4");
  TORCH_CHECK(codes.size(0) < (1L << 26) && K < (1L << 20), name, " is too large");
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

// How a launch's blocks share the work, `wanted` of them at a time.
long share(MxArgs& a, int rows, int pass, int wanted) {
  a.n_tiles = (a.N + rows - 1) / rows;
  const int passes = (a.M + pass - 1) / pass;
  const int want = std::max(1, (wanted + a.n_tiles - 1) / a.n_tiles);
  a.passes_each = (passes + want - 1) / want;
  const long blocks = (long)a.n_tiles * ((passes + a.passes_each - 1) / a.passes_each);
  TORCH_CHECK(blocks < (1L << 31), "too many tiles");
  return blocks;
}

template <typename Fn>
void launch_mx(Fn* fn, const MxArgs& a, long blocks, int threads, size_t bytes) {
  if (bytes > 64 * 1024)
    C10_HIP_CHECK(hipFuncSetAttribute((const void*)fn,
                                      hipFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)bytes));
  fn<<<(int)blocks, threads, bytes, cur_stream()>>>(a);
  C10_HIP_KERNEL_LAUNCH_CHECK();
}

template <bool X4, bool OUT32, int XT>
void launch_rows(MxArgs a) {
  constexpr int ROWS = XT * 16;
  const long blocks = share(a, ROWS, 256, 768);
  // what of a row of x fits LDS: all of it, or a part
  const int most = X4 ? 2048 : (XT == 4 ? 512 : 1024);
  a.kc = std::min((a.nb * 32 + 127) / 128 * 128, most);
  const size_t bytes = (size_t)ROWS * ((X4 ? a.kc / 2 : a.kc * 2) + 16) +
                       (X4 ? (size_t)ROWS * (a.kc / 32) : 0);
  launch_mx(&k_mxfp4_rows<X4, OUT32, XT>, a, blocks, 256, bytes);
}

template <bool X4, bool OUT32, int R>
void launch_stream(const MxArgs& args) {
  using S = Stream<X4, OUT32, R>;
  static_assert(S::BYTES <= 160 * 1024, "LDS");
  MxArgs a = args;
  // one block a CU, 256 of them at a time
  a.n_tiles = (a.N + S::ROWS - 1) / S::ROWS;
  const int passes = (a.M + 63) / 64, slices = std::max(1, 256 / a.n_tiles);
  a.passes_each = (passes + slices - 1) / slices;
  const long blocks = (long)a.n_tiles * ((passes + a.passes_each - 1) / a.passes_each);
  TORCH_CHECK(blocks < (1L << 31), "too many tiles");
  launch_mx(&k_mxfp4_stream<X4, OUT32, R>, a, blocks, 512, S::BYTES);
}

template <bool X4, bool OUT32>
void pick_mx(const MxArgs& a) {
  const int steps = (a.nb + 3) / 4;
  if (a.N <= 16) launch_rows<X4, OUT32, 1>(a);
  else if (a.N <= 128 || a.M < 64 || steps > 4) launch_rows<X4, OUT32, 4>(a);
  else if (steps <= 2) launch_stream<X4, OUT32, 2>(a);
  else if (steps == 3) launch_stream<X4, OUT32, 3>(a);
  else launch_stream<X4, OUT32, 4>(a);
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
    TORCH_CHECK(x.size(0) < (1L << 26), "x is too large");
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
