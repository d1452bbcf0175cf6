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

#include <type_traits>

#include "c2v_device.h"
#include "c2v_launch.h"

namespace {

// vectors at any address of their element's type
using u16x8_any = u16x8 __attribute__((aligned(2)));
using f32x4_any = f32x4 __attribute__((aligned(4)));

DEVI float scale_of(u32 byte) {
  // what the conversion instructions read of a scale is its exponent field,
  // so byte 0 does mean 2^-127 to them
  return __builtin_bit_cast(float, byte << 23);
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
// instruction rounds to nearest, ties to the even code. One pass, bound by
// memory: 261246 rows of 384 float32 (401 MB read, 53 written) in 99 us, 4.6
// TB/s; back to bf16 (53 read, 201 written) in 46 us, 5.6 TB/s.
// ---------------------------------------------------------------------------

template <bool F32>
__launch_bounds__(256)
__global__ void k_mxfp4_quantize(const void* __restrict__ x, long ldx,
                                 u32* __restrict__ codes,
                                 uint8_t* __restrict__ scales, long R, int K,
                                 int nb, int flat) {
  const long per_row = (long)nb * 4, total = R * per_row;
  // whole wavefronts stay in the loop together: the shuffles need all lanes
  for (long base = (long)blockIdx.x * 256; base < total;
       base += (long)gridDim.x * 256) {
    const long t = base + threadIdx.x;
    // (a division of 32 bits is a third of one of 64)
    const long r = flat ? 0 : total <= 0xFFFFFFFFl ? (long)((u32)t / (u32)per_row)
                                                   : t / per_row;
    const long k = (t - r * per_row) * 8;
    const long K_ = flat ? R * K : K;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (t < total) {
      if constexpr (F32) {
        const float* p = reinterpret_cast<const float*>(x) + r * ldx + k;
        if (k + 8 <= K_) {
          const f32x4 a = *reinterpret_cast<const f32x4_any*>(p);
          const f32x4 b = *reinterpret_cast<const f32x4_any*>(p + 4);
#pragma unroll
          for (int j = 0; j < 4; ++j) { v[j] = a[j]; v[4 + j] = b[j]; }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) if (k + j < K_) v[j] = p[j];
        }
      } else {
        const ushort* p = reinterpret_cast<const ushort*>(x) + r * ldx + k;
        if (k + 8 <= K_) {
          const u16x8 a = *reinterpret_cast<const u16x8_any*>(p);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = bf2f(a[j]);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) if (k + j < K_) v[j] = bf2f(p[j]);
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
  const bool flat = K % 32 == 0;
  for (long t = (long)blockIdx.x * 256 + threadIdx.x; t < total;
       t += (long)gridDim.x * 256) {
    const long r = flat ? 0 : total <= 0xFFFFFFFFl ? (long)((u32)t / (u32)per_row)
                                                   : t / per_row;
    const long c8 = t - r * per_row, k = c8 * 8;
    const long K_ = flat ? R * K : K;
    const bf16x8 v = decode8(codes[r * nb * 4 + c8],
                             scale_of(scales[r * nb + (c8 >> 2)]));
    if constexpr (F32) {
      float* o = reinterpret_cast<float*>(out) + r * K + k;
      f32x4 a, b;
#pragma unroll
      for (int j = 0; j < 4; ++j) { a[j] = (float)v[j]; b[j] = (float)v[4 + j]; }
      if (k + 8 <= K_) {
        *reinterpret_cast<f32x4_any*>(o) = a;
        *reinterpret_cast<f32x4_any*>(o + 4) = b;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) if (k + j < K_) o[j] = (float)v[j];
      }
    } else {
      ushort* o = reinterpret_cast<ushort*>(out) + r * K + k;
      const u16x8 a = __builtin_bit_cast(u16x8, v);
      if (k + 8 <= K_) {
        *reinterpret_cast<u16x8_any*>(o) = a;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) if (k + j < K_) o[j] = a[j];
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
//
// One row by 261246 of 384: 13.3 us, bound by the reading of w (53 MB, 4.0 TB/s,
// where bf16 weights would be 201 MB). 37 rows by 50001 of 201, y in float32:
// 9.7 us, bound by latency, in blocks that live for one pass, and by y's broken lines
// (7.4 MB).
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
  int passes, passes_each;    // passes over rows of w, in all and a block
  int period;                 // rows of y this many apart lie alike on lines
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
    if (u * 8 + 8 <= p.K) {
      v = __builtin_bit_cast(u32x4, *reinterpret_cast<const u16x8_any*>(s));
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
// what moves: 64 at a time, through a ring of four LDS buffers that the
// block's eight waves share, so that w is read once for 128*XT rows of x.
//
// Lines of y that are written in two halves cost twice (2.1 GB of bf16 with
// an odd number of words a row: 950 us, against 430 us for whole lines). So a
// wave takes rows of x that lie the same way on lines, every `period`-th one,
// and its columns begin on a line: `shift` columns before those of the tile
// of w, out of this tile and the one before it. The block next to it ends
// where this one begins.
//
// A wave's loads and stores are counted in one queue. The wait for a tile of
// w therefore counts the stores behind it: they are the same number in every
// pass but at the table's ends, because rows of x behind the last one repeat
// it, and store the same again.
//
// 261246 columns, K = 384, y in bf16: 1024 rows of bf16 206 us (535 MB written,
// 1000 TFLOP/s; bound by the decoding of w, which every wave does for its 32 rows,
// next to the products: matrix units work in 45% of the cycles, and 3.4 other vector
// instructions go with each of theirs), 4096 rows in 4 bits 516 us (2.1 GB, 4.1
// TB/s: writing).
template <bool X4, bool OUT32, int R>
struct Stream {
  static constexpr int XT = X4 ? 4 : R > 4 ? 1 : 2;   // 16-row tiles of x a wave
  static constexpr int ES = OUT32 ? 4 : 2;
  static constexpr int STORES = XT * 64 * ES / 64;          // a wave and pass
  static constexpr int FETCH = (4 * R + 7) / 8;             // of them codes
  static constexpr int LOADS = FETCH + 1;                   // a wave and tile
  static constexpr int RING = 4 * 64 * 4 * R * 17;
};

template <bool X4, bool OUT32, int R>
__launch_bounds__(512, 2)
__global__ void k_mxfp4_stream(MxArgs p) {
  using S = Stream<X4, OUT32, R>;
  constexpr int XT = S::XT, ES = S::ES;
  extern __shared__ uint8_t sm[];              // 4 x 64 rows of codes, of scales
  uint8_t* const sm_scales = sm + 4 * 64 * 4 * R * 16;

  const int b = xcd_chunked(blockIdx.x, gridDim.x);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, q = lane >> 4;
  const int nb = p.nb;
  const int pass0 = b / p.n_tiles * p.passes_each;
  const int pass1 = min(pass0 + p.passes_each, p.passes);
  if (pass0 >= pass1) return;

  // this wave's rows: n0, n0 + period, ..; some waves have none
  const int wave = b % p.n_tiles * 8 + wid;
  const int first_n = wave % p.period + wave / p.period * (XT * 16) * p.period;
  const bool idle = first_n >= p.N;
  const int n0 = min(first_n, p.N - 1);
  const int last = (p.N - 1 - n0) / p.period;
  const int shift = p.period == 1 ? 0 :
      (int)(((u64)p.y + (u64)n0 * p.M * ES) & 127) / ES;

  // Four 16-byte blocks of a row change places by the row's number, where the
  // number of blocks has the powers of two for it: a read's 16 rows then lie
  // on more banks.
  const int group = min(nb & -nb, 4);
  auto key = [&](int row) { return (row >> 4) & (group - 1); };
  auto fetch = [&](int tile) {        // rows 64 * tile ..
    const int m0 = max(0, min(tile * 64, (p.M - 1) / 64 * 64));
    const uint8_t* wc = in_scalar(p.wc + (u64)m0 * nb * 16);
    uint8_t* codes = sm + (tile & 3) * 64 * nb * 16;
#pragma unroll
    for (int k = 0; k < S::FETCH; ++k) {
      // 64 blocks an instruction, nb instructions a tile; a wave without one
      // repeats another
      const int e = wid + 8 * k < nb ? wid + 8 * k : wid % nb;
      const int u = e * 64 + lane, row = u / nb, at = u % nb;
      const u32 off = (u32)(min(row, p.M - 1 - m0) * nb + (at ^ key(row))) * 16;
      to_lds<16>(wc + off, codes + e * 1024);
    }
    const int e = wid * 4 < nb ? wid : 0;
    const int whole = (min(64, p.M - m0) * nb) >> 2;       // words of scales
    // (a tile without a whole word: it is filled in below)
    const uint8_t* ws = in_scalar(p.ws + (whole ? (u64)m0 * nb : 0));
    to_lds<4>(ws + (u32)max(0, min(e * 64 + lane, whole - 1)) * 4,
              sm_scales + (tile & 3) * 256 * R + e * 256);
  };

  // x into registers; blocks behind a row's end are zeros
  u32x4 xf[XT][X4 ? R : R * 4];
  u32 xs[XT][R];
  u32 y_off[XT];
#pragma unroll
  for (int i = 0; i < XT; ++i) {
    const int j = min(i * 16 + l16, last);
    const long n = n0 + (long)j * p.period;
    y_off[i] = (u32)j * (u32)p.period * (u32)p.M * ES + q * 16 * ES;
#pragma unroll
    for (int s = 0; s < R; ++s) {
      if constexpr (X4) {
        xf[i][s] = x_unit<true>(p, n, s * 4 + q, xs[i][s]);
      } else {
#pragma unroll
        for (int j4 = 0; j4 < 4; ++j4)
          xf[i][s * 4 + j4] = x_unit<false>(p, n, (s * 4 + q) * 4 + j4, xs[i][s]);
      }
    }
  }
  for (int k = -1; k < 2; ++k) fetch(pass0 + k);

  // Row t*4 of this lane in a pass: behind the tile's first row, or in the
  // tile before it. A row's last step may have fewer than four blocks: the
  // others repeat the last, under a scale of one, because what lies behind a row
  // is another row, whose NaN would outlive the zeros that x has there.
  const int row_in = (l16 >> 2) * (4 * MT) + (l16 & 3) - shift;
  const int s_end = R == 2 && nb <= 4 ? 0 : R - 1;   // (other R: nb > 4 * (R - 1))
  const int left = nb - s_end * 4;
  const int q_end = min(q, left - 1);

  const int end = (p.M - 1) / 64;                  // the table's last tile
  const int odd = (int)(((long)p.M * nb) & 3);
  f32x4 acc[XT][MT];
  for (int pass = pass0; pass < pass1; ++pass) {
    // behind this pass's tile: the next one, and the stores of two passes
    const int m0 = pass * 64 - shift;
    wait_queue<S::LOADS, S::LOADS + 2 * S::STORES>(
        !idle && pass - pass0 >= 3 && m0 <= p.M);
    if (odd && (pass == end || (pass == pass0 && pass == end + 1))) {
      // the table's last scales, where they fill no word
      const int at = ((p.M - end * 64) * nb & ~3) + tid;
      if (tid < odd) sm_scales[(end & 3) * 256 * R + at] = p.ws[(u64)end * 64 * nb + at];
      __syncthreads();
    }
    fetch(pass + 2);
    asm volatile("" ::: "memory");
    if (idle) continue;

    mx_clear(acc);
    const u32 now = (pass & 3) * 64, before = ((pass - 1) & 3) * 64;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const int row = row_in + t * 4;
      const int in = row & 63;
      const u32 at = row < 0 ? before : now;
      const uint8_t* c_row = sm + (at + in) * nb * 16;
      const uint8_t* s_row = sm_scales + at * 4 * R + in * nb;
#pragma unroll
      for (int s = 0; s < R; ++s) {
        if (R == 2 && s > s_end) break;
        const int at_q = s == s_end ? q_end : q;
        const u32x4 c = *reinterpret_cast<const u32x4*>(
            c_row + s * 64 + (at_q ^ key(in)) * 16);
        u32 sc = s_row[s * 4 + at_q];
        if (s == s_end && q >= left) sc = 127;
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

    if (m0 >= 0 && m0 + 64 <= p.M) {
      uint8_t* o = in_scalar(reinterpret_cast<uint8_t*>(p.y) +
                             ((u64)n0 * p.M + m0) * ES);
#pragma unroll
      for (int i = 0; i < XT; ++i) {
        if constexpr (OUT32) {
#pragma unroll
          for (int t = 0; t < MT; ++t)
            *reinterpret_cast<f32x4_any*>(o + y_off[i] + t * 16) = acc[i][t];
        } else {
#pragma unroll
          for (int t = 0; t < MT; t += 2)
            *reinterpret_cast<u16x8_any*>(o + y_off[i] + t * 8) =
                pack8(acc[i][t], acc[i][t + 1]);
        }
      }
    } else {
      // an end of the table
#pragma unroll
      for (int i = 0; i < XT; ++i) {
        const long n = n0 + (long)min(i * 16 + l16, last) * p.period;
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int m = m0 + q * 16 + t * 4 + r;
            if (m < 0 || m >= p.M) continue;
            if constexpr (OUT32)
              reinterpret_cast<float*>(p.y)[n * p.M + m] = acc[i][t][r];
            else
              reinterpret_cast<__bf16*>(p.y)[n * p.M + m] = (__bf16)acc[i][t][r];
          }
      }
    }
  }
  // tiles of w that nobody needs may still be on their way into LDS
  __builtin_amdgcn_s_waitcnt(0x0F70);
}

// ===========================================================================
// host wrappers
// ===========================================================================

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
  // dense rows of whole blocks are one long row: no division is needed
  const int flat = K % 32 == 0 && (ld == K || R == 1);
  const int grid = grid_of(R * nb * 4, 256, 16384);
  auto* fn = f32 ? &k_mxfp4_quantize<true> : &k_mxfp4_quantize<false>;
  fn<<<grid, 256, 0, cur_stream()>>>(
      src.data_ptr(), ld, reinterpret_cast<u32*>(codes.data_ptr()),
      scales.data_ptr<uint8_t>(), R, K, nb, flat);
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return {codes, scales};
}

// codes (rows, 16 nb) and scales (rows, nb) of rows of K values
void check_mx(const torch::Tensor& codes, const torch::Tensor& scales, long K,
              const char* name) {
  const long nb = (K + 31) / 32;
  TORCH_CHECK_VALUE(codes.is_cuda() && scales.device() == codes.device(), name,
                    " must be on one GPU");
  TORCH_CHECK_VALUE(codes.scalar_type() == torch::kUInt8 &&
                    scales.scalar_type() == torch::kUInt8, name, " must be uint8");
  // (a K from -62 on would make no blocks, like none)
  TORCH_CHECK_VALUE(K >= 0 && codes.dim() == 2 && scales.dim() == 2 &&
                    codes.size(0) == scales.size(0) && scales.size(1) == nb &&
                    codes.size(1) == 16 * nb, name, " does not hold rows of ", K);
  TORCH_CHECK_VALUE(codes.is_contiguous() && scales.is_contiguous(), name,
                    " must be contiguous");
  TORCH_CHECK((reinterpret_cast<uintptr_t>(codes.data_ptr()) & 15) == 0, name,
              " must start on 16 bytes");
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
  a.passes = (a.M + pass - 1) / pass;
  const int want = std::max(1, (wanted + a.n_tiles - 1) / a.n_tiles);
  a.passes_each = (a.passes + want - 1) / want;
  const long blocks = (long)a.n_tiles * ((a.passes + a.passes_each - 1) / a.passes_each);
  TORCH_CHECK(blocks < (1L << 31), "too many tiles");
  return blocks;
}

template <void (*KERNEL)(MxArgs)>
void launch_mx(const MxArgs& a, long blocks, int threads, size_t bytes) {
  static std::atomic<u64> ready{0};
  auto* fn = KERNEL;
  allow_lds(fn, 160 * 1024, ready);
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
  launch_mx<&k_mxfp4_rows<X4, OUT32, XT>>(a, blocks, 256, bytes);
}

template <bool X4, bool OUT32, int R>
void launch_stream(const MxArgs& args) {
  using S = Stream<X4, OUT32, R>;
  constexpr int rows = S::XT * 16;              // a wave
  MxArgs a = args;
  const int over = (int)((long)a.M * S::ES % 128);
  a.period = 1;
  for (int v = 128; over && v > 1 && over % v; v /= 2) a.period *= 2;
  // In order a wave writes broken lines. The cache behind L2 mends them as long
  // as y is not much larger than it, and rows that lie alike have to fill their
  // waves. (M = 261246, K = 384, bf16 y; rows alike against in order: bf16 x, 512
  // rows in half-filled waves 208 us to 118, 1024 in full ones 217 to 249; 4-bit
  // x 512 rows in a quarter 150 to 92, 768 in 3/8 172 to 215, 4096 518 to 1142.
  // M = 50001, 4-bit x: 1024 rows, 102 MB, 60 to 46; 4096, 410 MB, 117 to 228.)
  const long alike = (a.N + a.period - 1) / a.period;
  const long held = (alike + rows - 1) / rows * rows;
  if ((long)a.N * a.M * S::ES < (192L << 20) ||
      (X4 ? 8 * alike < 3 * held : 4 * alike <= 3 * held) ||
      (long)rows * a.period * a.M * S::ES >= (1L << 32))
    a.period = 1;
  const int per = (a.N + a.period - 1) / a.period;
  const long waves = (long)a.period * ((per + rows - 1) / rows);
  // one block a CU, 256 of them at a time
  a.n_tiles = (int)((waves + 7) / 8);
  a.passes = (a.M + (a.period > 1 ? 63 : 0) + 63) / 64;
  const int slices = std::max(1, 256 / a.n_tiles);
  a.passes_each = (a.passes + slices - 1) / slices;
  const long blocks = (long)a.n_tiles * ((a.passes + a.passes_each - 1) / a.passes_each);
  TORCH_CHECK(blocks < (1L << 31), "too many tiles");
  launch_mx<&k_mxfp4_stream<X4, OUT32, R>>(a, blocks, 512, S::RING);
}

constexpr int FEW = 128;

// Up to 128 rows of x go by tiles of 16 or of 64: 16 fill the chip with blocks
// where w is short, 64 read w once. (64 and 16, y in bf16: x in bf16, K = 384, 37
// rows by 25000 10.0 and 7.1 us, 64 by 50001 12.6 and 12.4, 128 by 50001 18.5 and
// 23.3, 37 by 261246 26.9 and 26.2; rows of 700, which 64 at a time do not fit
// LDS, 128 by 261246 173 and 126; x in 4 bits, 64 by 25000 7.4 and 6.4, 64 by
// 50001 8.7 and 11.2.) More go through k_mxfp4_stream.
template <bool X4, bool OUT32>
void pick_mx(const MxArgs& a) {
  const int steps = (a.nb + 3) / 4;
  const long blocks = (long)((a.N + 15) / 16) * ((a.M + 255) / 256);
  if (a.N <= 16 || (a.N <= FEW && (blocks <= (X4 ? 512 : 1024) ||
                                   (!X4 && (a.N <= 48 || steps > 4)))))
    launch_rows<X4, OUT32, 1>(a);
  else if (a.N <= FEW || a.M < 64 || steps > 6 || 64l * a.M * (OUT32 ? 4 : 2) >= (1L << 32))
    launch_rows<X4, OUT32, 4>(a);
  else if (steps <= 2) launch_stream<X4, OUT32, 2>(a);
  else if (steps == 3) launch_stream<X4, OUT32, 3>(a);
  else if (steps == 4) launch_stream<X4, OUT32, 4>(a);
  else if (steps == 5) launch_stream<X4, OUT32, 5>(a);
  else launch_stream<X4, OUT32, 6>(a);
}

// x: bf16 (N, K), or the codes of x with their scales
torch::Tensor mxfp4_matmul(torch::Tensor x,
                           c10::optional<torch::Tensor> x_scales,
                           torch::Tensor w_codes, torch::Tensor w_scales,
                           int64_t K, bool f32) {
  check_mx(w_codes, w_scales, K, "w");
  const bool x4 = x_scales.has_value();
  TORCH_CHECK_VALUE(x.device() == w_codes.device(), "x and w must be on one GPU");
  const Guard guard(x.device());
  torch::Tensor src = x;
  MxArgs a{};
  if (x4) {
    check_mx(x, *x_scales, K, "x");
    a.xc = x.data_ptr<uint8_t>();
    a.xs = x_scales->data_ptr<uint8_t>();
  } else {
    TORCH_CHECK(x.scalar_type() == torch::kBFloat16, "x must be bfloat16");
    TORCH_CHECK_VALUE(x.dim() == 2 && x.size(1) == K, "x must be (N, ", K, ")");
    TORCH_CHECK(x.size(0) < (1L << 26), "x is too large");
    if (K > 1 && x.stride(1) != 1) src = x.contiguous();
    a.x = reinterpret_cast<const ushort*>(src.data_ptr<at::BFloat16>());
    a.ldx = x.size(0) == 1 ? K : src.stride(0);
  }
  a.N = x.size(0);
  a.M = w_codes.size(0);
  a.K = K;
  a.nb = w_scales.size(1);
  a.wc = w_codes.data_ptr<uint8_t>();
  // k_mxfp4_stream reads scales as words: those of some rows of a table may start
  // on any byte, and are copied (a 17th of the table)
  if (a.N > FEW && (reinterpret_cast<uintptr_t>(w_scales.data_ptr()) & 3))
    w_scales = w_scales.clone();
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
