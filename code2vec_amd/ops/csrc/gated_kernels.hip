// The gated context transform (gfx950), forward and backward.
//
//   g = x Wg^T,  u = x Wu^T,  y = act(g) * u                     x (N,K)
//   du = dy * act(g),  dg = dy * u * act'(g)
//   dx = dg Wg + du Wu,  dW = x^T [dg | du]
//
// The backward forms g and u again from x: to write and read them costs as
// much, or loses precision. (204800 rows, K = H = 384, forward and backward: in
// fp32 835 us, again 700; 14351 rows, 1440: 565 and 579; in bf16 670 and 476,
// but with gradients off by 0.0030 of their norm where once rounded ones are by
// 0.0017 and these by 0.0024.) bf16 operands, fp32 accumulation and activations.
// What is rounded to bf16 on the way are dg and du, as operands of the two products
// that consume them: each by at most 2^-8 of itself, so that a sum of 2H or N such
// terms is off by at most 2^-8 of the sum of its terms' magnitudes, whatever of them
// cancels. Their errors have either sign, and the 0.0024 is what they come to next to
// the result's own rounding. dW may leave as it was summed, in fp32.

#include <torch/extension.h>

#include "c2v_device.h"
#include "c2v_launch.h"

namespace {

enum Activation : int { SILU = 0, GELU = 1, SIGMOID = 2, TANH = 3, RELU = 4 };

// The hardware's reciprocal is off by about one step of fp32. Its exponential
// takes g log2(e), whose rounding alone moves the result by about |g| steps: far
// below bf16's 2^-8 wherever it counts. Their limits are right: 1 / (1 + exp(200))
// is zero.
DEVI float sigmoid(float g) {
  return __builtin_amdgcn_rcpf(1.f + __expf(-g));
}

// 1 - 2 / (exp(2g) + 1) loses what is small next to one, so that near zero
// the series takes over: its next term is below 2e-9 of the result
DEVI float tanh_of(float g) {
  const float far = 1.f - 2.f * __builtin_amdgcn_rcpf(1.f + __expf(2.f * g));
  const float s = g * g;
  const float near = g + g * s * (-0.33333333f + s * (0.13333333f - s * 0.05396825f));
  return fabsf(g) < 0.125f ? near : far;
}

// act(g) and act'(g); the derivative costs nothing where it is not used
template <int ACT>
DEVI void act_both(float g, float& a, float& da) {
  if constexpr (ACT == SILU) {
    const float s = sigmoid(g);
    a = g * s;
    da = s + a * (1.f - s);
  } else if constexpr (ACT == GELU) {
    // erfc and not 1 + erf: far left the sum would leave no digits
    const float cdf = 0.5f * erfcf(g * -0.70710678f);
    a = g * cdf;
    da = cdf + g * __expf(-0.5f * g * g) * 0.39894228f;
  } else if constexpr (ACT == SIGMOID) {
    a = sigmoid(g);
    da = a * (1.f - a);
  } else if constexpr (ACT == TANH) {
    a = tanh_of(g);
    da = 1.f - a * a;
  } else {
    a = g > 0.f ? g : (g != g ? g : 0.f);
    da = g > 0.f ? 1.f : 0.f;
  }
}

DEVI void to_lds16(const void* src, ushort* dst) {
  __builtin_amdgcn_global_load_lds(
      (const __attribute__((address_space(1))) u32*)src,
      (__attribute__((address_space(3))) u32*)dst, 16, 0, 0);
}

// what a chunk beyond the reduction's end reads
__device__ __attribute__((aligned(16))) const ushort k_zero_chunk[8] = {};

DEVI u16x8 pack8(const float* v) {
  bf16x8 b;
#pragma unroll
  for (int j = 0; j < 8; ++j) b[j] = (__bf16)v[j];
  return __builtin_bit_cast(u16x8, b);
}

// ---------------------------------------------------------------------------
// Products whose reduction runs along the rows of both operands.
//
// The weights take the place of the matrix instruction's A operand and the
// rows of x that of its B operand: a lane then holds consecutive output
// columns of ONE row. Weight rows are put into LDS in such an order that the
// 4 x GT values of a lane in one group of GT tiles are 4*GT consecutive
// columns, which go out as 16-byte stores. A wave has two groups: the gate
// and the up columns of the same outputs, or two neighbours for a plain
// product.
// ---------------------------------------------------------------------------

// Tiles go from memory into a ring of LDS buffers ahead of the matrix
// instructions. A step begins when its own tile has arrived, which is when no
// more than N of the loads and stores that this wave issued after it are
// outstanding, and when every wave has read the tile that the step's new loads
// overwrite.
template <int N>
DEVI void wait_queue() {
  static_assert(N < 64, "vmcnt has 6 bits");
  // vmcnt in bits 3:0 and 15:14, expcnt 6:4 (no wait), lgkmcnt 11:8 (zero)
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x70 | (N & 15) | (N >> 4 << 14));
}

DEVI void block_barrier() {
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// GATED: y; DGATED: dg and du
enum Epilogue : int { GATED = 0, PLAIN = 1, DGATED = 2 };

struct BtArgs {
  const ushort* x;    // (N, K), rows ldx apart
  const ushort* w;    // (2, H, K); PLAIN: (H, K)
  ushort* y;          // (N, H); DGATED: dgu (N, 2, Hp)
  const ushort* dy;   // DGATED: (N, Hp), rows lddy apart, zeros behind H
  long ldx, lddy;
  int N, H, Hp, K;
  float keep_prob;    // PLAIN with dropout: below one
  u64 seed;
  const long* seed_ptr;
};

// GT f32x4 of a lane, consecutive columns from h of a row of H: 16-byte stores
// (8 for GT = 1) where rows lie on them
template <int GT>
DEVI void put(ushort* base, const float* v, int h, int H) {
  constexpr int W = GT == 1 ? 4 : 8;
  if (H % W == 0) {
#pragma unroll
    for (int c = 0; c < 4 * GT; c += W)
      if (h + c < H) {
        if constexpr (GT == 1) {
          bf16x4 b;
#pragma unroll
          for (int j = 0; j < 4; ++j) b[j] = (__bf16)v[j];
          *reinterpret_cast<bf16x4*>(base) = b;
        } else {
          *reinterpret_cast<u16x8*>(base + c) = pack8(v + c);
        }
      }
  } else {
#pragma unroll
    for (int c = 0; c < 4 * GT; ++c)
      if (h + c < H) base[c] = __builtin_bit_cast(ushort, (__bf16)v[c]);
  }
}

// A lane's columns from h of one row; `to` is where they go.
template <int ACT, int GT>
DEVI void put_gated(const BtArgs& p, ushort* to, int h, const f32x4* g, const f32x4* u) {
  float yv[4 * GT];
#pragma unroll
  for (int j = 0; j < 4 * GT; ++j) {
    float a, da;
    act_both<ACT>(g[j / 4][j & 3], a, da);
    yv[j] = a * u[j / 4][j & 3];
  }
  put<GT>(to, yv, h, p.H);
}

// the same columns of dy, two a register
template <int GT>
struct DyPart {
  u32 v[2 * GT];
};

template <int GT>
DEVI DyPart<GT> read_dy(const BtArgs& p, const ushort* from, int h) {
  constexpr int W = GT == 1 ? 4 : 8;
  DyPart<GT> d = {};
#pragma unroll
  for (int c = 0; c < 4 * GT; c += W)
    if (h + c < p.Hp)
      __builtin_memcpy(d.v + c / 2, __builtin_assume_aligned(from + c, 2 * W), 2 * W);
  return d;
}

// what is behind H comes out as zeros, up to Hp
template <int ACT, int GT>
DEVI void put_dgated(const BtArgs& p, ushort* to, int h, const f32x4* g, const f32x4* u,
                     const DyPart<GT>& d) {
  float dg[4 * GT], du[4 * GT];
#pragma unroll
  for (int j = 0; j < 4 * GT; ++j) {
    float a, da;
    act_both<ACT>(g[j / 4][j & 3], a, da);
    const float dy = __builtin_bit_cast(
        float, j & 1 ? d.v[j / 2] & 0xFFFF0000u : d.v[j / 2] << 16);
    dg[j] = dy * u[j / 4][j & 3] * da;
    du[j] = dy * a;
  }
  if (p.Hp != p.H)
#pragma unroll
    for (int j = 0; j < 4 * GT; ++j)
      if (h + j >= p.H) dg[j] = du[j] = 0.f;
  put<GT>(to, dg, h, p.Hp);
  put<GT>(to + p.Hp, du, h, p.Hp);
}

template <int GT>
DEVI void put_plain(const BtArgs& p, ushort* to, long n, int h, const f32x4* a) {
  float v[4 * GT];
#pragma unroll
  for (int j = 0; j < 4 * GT; ++j) v[j] = a[j / 4][j & 3];
  if (p.keep_prob < 1.f) {
    const u64 seed = p.seed_ptr ? (u64)*p.seed_ptr : p.seed;
    const float inv_keep = 1.f / p.keep_prob;
#pragma unroll
    for (int j = 0; j < 4 * GT; ++j)
      v[j] = hash_uniform(seed, (u64)n * p.H + h + j) < p.keep_prob ? v[j] * inv_keep
                                                                   : 0.f;
  }
  put<GT>(to, v, h, p.H);
}

// 204800 rows, K = H = 384: y 141 us (860 TFLOP/s), dg and du 200 us, dx 158 us and
// with the dropout mask 206; 14351 rows of 1440: 124, 131 and 116 us (960, 905 and
// 1030 TFLOP/s). Counted at 204800 rows (profiles/gated_mxfp4_counters.csv), of the
// cycles in which a CU has waves: the matrix units work in 38% for y, 26% for dg
// and du and 32% for dx, LDS reads in 14, 10 and 16%, without bank conflicts. None of
// them is full: what is left are waits, because rounds of all blocks load, multiply
// and store in step, so that what moves (314 MB for y, 630 for dg and du, at 5
// TB/s) adds to the products in part. The epilogue of dg and du takes 18 vector
// instructions an element; the mask is a hash of 64 bits for each element of dx.
template <int EPI, int ACT, int WR, int WC, int XT, int GT, int BK,
          int STAGES>
__launch_bounds__(WR * WC * 64, 2)
__global__ void k_rows_gemm(BtArgs p) {
  constexpr int T = WR * WC * 64;
  constexpr int BM = WR * XT * 16;         // rows of x a block
  constexpr int BG = WC * GT * 16;         // columns of one group
  constexpr int BN = 2 * BG;               // rows of w a block
  constexpr int HT = EPI == PLAIN ? BN : BG;   // output columns a block
  constexpr int CH = BK / 8;               // 16-byte chunks a row
  constexpr int IT = (BM + BN) * CH / T;
  // Operands of one half of a step are read while the other half is multiplied,
  // those of a step's first half behind a barrier in the middle of the step
  // before. For the largest tile there are not registers enough, and with dy the
  // compiler finds no good order; their steps begin with their barrier. (Gated,
  // 50000 rows, K = H = 640, tiles of 128 by 64: 89 us, with the barriers between
  // the steps 98; the largest tile, 204800 rows of 384: 240 with spills, and 163;
  // with dy, tiles of 128 by 64: 257, and 241.)
  constexpr bool PIPE = GT == 1 || (GT == 2 && EPI != DGATED);
  static_assert(BK == 64 && (PIPE || STAGES == 2), "two halves a step");
  // where a row's 16-byte chunks lie: 8 rows read at once cover all banks
  auto place = [](int row) { return row & 7; };
  constexpr int ITX = BM * CH / T;         // of them from x
  static_assert(BM * CH % T == 0 && BN * CH % T == 0, "staging");
  extern __shared__ ushort lds[];          // STAGES x (BM + BN) x BK

  // An XCD's blocks go over a run of tiles together, those of one tile of x
  // next to each other: its rows come from one L2.
  const int nC = (p.H + HT - 1) / HT;
  const int tiles = (int)((p.N + (long)BM - 1) / BM * nC);
  const int xcd = blockIdx.x & 7, each = (gridDim.x + 7 - xcd) >> 3;
  const int tile0 = xcd * (tiles >> 3) + min(xcd, tiles & 7);
  const int tile1 = tile0 + (tiles >> 3) + (xcd < (tiles & 7));
  int tile = tile0 + (blockIdx.x >> 3);
  if (tile >= tile1) return;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wid / WC, wc = wid % WC;
  const int l16 = lane & 15, q = lane >> 4;

  // Where each of this thread's chunks comes from: bytes behind the tile's
  // first row of x, or behind w. A step adds to the bases alone.
  long row0;
  int h0;
  u32 off[IT];
  const char* xb;
  const char* wb = reinterpret_cast<const char*>(p.w);
  auto begin = [&](int t) {
    row0 = (long)(t / nC) * BM;
    h0 = t % nC * HT;
    xb = reinterpret_cast<const char*>(p.x + row0 * p.ldx);
    // made here for each tile: kept over the tiles its parts would spill
    int me = tid;
    asm volatile("" : "+v"(me));
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      const int c = it * T + me;
      const int r = c / CH, pos = c % CH;
      const u32 col = (pos ^ place(r)) * 16;
      if (it < ITX) {
        const long n = min((long)r, (long)p.N - 1 - row0);
        off[it] = (u32)(n * p.ldx * 2) + col;
      } else {
        const int j = r - BM;                       // row of w in LDS
        const int i = j & 15, mi = (j >> 4) % GT;
        const int grp = (j >> 4) / GT % 2, cw = (j >> 4) / (2 * GT);
        const int in_group = (i >> 2) * (4 * GT) + mi * 4 + (i & 3);
        long wrow;
        if constexpr (EPI == PLAIN)
          wrow = min(h0 + (cw * 2 + grp) * GT * 16 + in_group, p.H - 1);
        else
          wrow = (long)grp * p.H + min(h0 + cw * GT * 16 + in_group, p.H - 1);
        off[it] = (u32)(wrow * p.K * 2) + col;
      }
    }
  };
  auto stage = [&](int k0, int buf) {
    ushort* dst = lds + buf * (BM + BN) * BK + wid * 512;
    if (k0 + BK <= p.K) {
      const char* xk = in_scalar(xb + k0 * 2l);
      const char* wk = in_scalar(wb + k0 * 2l);
#pragma unroll
      for (int it = 0; it < IT; ++it)
        to_lds16((it < ITX ? xk : wk) + off[it], dst + it * T * 8);
    } else {
#pragma unroll
      for (int it = 0; it < IT; ++it) {
        const int r = (it * T + tid) / CH, pos = (it * T + tid) % CH;
        const char* s = (it < ITX ? xb : wb) + k0 * 2l + off[it];
        to_lds16(k0 + (pos ^ place(r)) * 8 < p.K ? (const void*)s : k_zero_chunk,
                 dst + it * T * 8);
      }
    }
  };

  // stores of a wave in a tile's end, where all of it is there
  constexpr int PUT = XT * (GT >= 2 ? GT / 2 : 1) * (EPI == GATED ? 1 : 2);
  const int steps = (p.K + BK - 1) / BK;

  // What is asked for runs ahead of what is multiplied, from one tile into the
  // next: of `ltile` the step `lstep` is next, and `ahead` steps that were
  // asked for have not been waited for.
  int ltile = tile, lstep = 0, lbuf = 0, ahead = 0;
  auto ask = [&](bool always) {
    if (lstep == steps && ltile < tile1) {
      ltile += each;
      lstep = 0;
      if (ltile < tile1) begin(ltile);
    }
    const bool any = ltile < tile1;
    if (!any && !always) return;
    stage((any ? lstep : 0) * BK, lbuf);
    lbuf = lbuf == STAGES - 1 ? 0 : lbuf + 1;
    lstep += any;
    ahead += any;
  };
  // The next step is there: behind it in the queue are the steps that were asked
  // for after it and perhaps the stores of the tile before. Every wave has read
  // the step before it, whose buffer is the next to fill.
  auto arrive = [&](bool stores) {
    if (STAGES == 3 && ahead == 3) {
      wait_queue<2 * IT>();
    } else if (ahead >= 2) {
      if (stores) wait_queue<IT + PUT>();
      else wait_queue<IT>();
    } else {
      if (stores) wait_queue<PUT>();
      else wait_queue<0>();
    }
    block_barrier();
    --ahead;
  };
  int buf = 0;
  struct Half { bf16x8 x[XT], w[2 * GT]; };
  auto read = [&](Half& f, int kk) {
    const ushort* xs = lds + buf * (BM + BN) * BK + wr * XT * 16 * BK;
    const ushort* ws = lds + buf * (BM + BN) * BK + (BM + wc * 2 * GT * 16) * BK;
    const int off = l16 * BK + (((kk * 4 + q) ^ place(l16)) * 8);
#pragma unroll
    for (int i = 0; i < XT; ++i)
      f.x[i] = *reinterpret_cast<const bf16x8*>(xs + i * 16 * BK + off);
#pragma unroll
    for (int j = 0; j < 2 * GT; ++j)
      f.w[j] = *reinterpret_cast<const bf16x8*>(ws + j * 16 * BK + off);
  };
  bool whole = false;                      // the tile before was
  begin(tile);
#pragma unroll 1
  for (int s = 0; s < STAGES; ++s) ask(false);
  Half f, g;
  if (PIPE) {
    arrive(false);
    read(f, 0);
  }
  for (; tile < tile1; tile += each) {
    f32x4 acc[XT][2 * GT];
#pragma unroll
    for (int i = 0; i < XT; ++i)
#pragma unroll
      for (int j = 0; j < 2 * GT; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};
    const long row = row0;
    const int h = h0;
    auto multiply = [&](const Half& f) {
#pragma unroll
      for (int i = 0; i < XT; ++i)
#pragma unroll
        for (int j = 0; j < 2 * GT; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f.w[j], f.x[i], acc[i][j],
                                                              0, 0, 0);
    };
    auto flip = [&] { buf = buf == STAGES - 1 ? 0 : buf + 1; };
    for (int s = 0; s < steps - 1; ++s) {
      if (PIPE) {
        read(g, 1);
        multiply(f);
        arrive(whole && s < STAGES - 1);
        flip();
        ask(false);
        read(f, 0);
        multiply(g);
      } else {
        arrive(whole && s < STAGES);
        // (the other buffer holds step 1 when step 0 begins)
        if (s > 0) ask(false);
        read(f, 0);
        read(g, 1);
        multiply(f);
        multiply(g);
        flip();
      }
    }
    // A lane's columns in its rows of the tile, and their places behind the
    // tile's first row.
    const int hl = h + (EPI == PLAIN ? 2 : 1) * wc * GT * 16 + q * 4 * GT;
    const int r = wr * XT * 16 + l16;
    const int ldy = EPI == DGATED ? 2 * p.Hp : p.H;
    const u32 at = ((u32)r * ldy + hl) * 2;
    // The last step. What is asked for behind the stores arrives after them: the
    // next tile's first steps go ahead, and dy ahead of those. (With dy, a
    // block's last tile asks for a step in vain: a number of loads that is always
    // the same is one that can be waited for.)
    DyPart<GT> dy[EPI == DGATED ? XT : 1];
    auto ask_dy = [&] {
      if constexpr (EPI == DGATED) {
        const char* dyb = reinterpret_cast<const char*>(p.dy + row * p.lddy);
#pragma unroll
        for (int i = 0; i < XT; ++i)
          dy[i] = read_dy<GT>(p, reinterpret_cast<const ushort*>(dyb + (u32)(
              min((long)r + i * 16, p.N - 1 - row) * p.lddy + hl) * 2), hl);
        asm volatile("" ::: "memory");
      }
    };
    if (PIPE) {
      read(g, 1);
      multiply(f);
      const bool next = tile + each < tile1;
      if (next) {
        arrive(whole && steps - 1 < STAGES - 1);
        flip();
      }
      ask_dy();
      ask(EPI == DGATED);
      if (next) read(f, 0);
      multiply(g);
    } else {
      arrive(whole && steps - 1 < STAGES);
      ask_dy();
      ask(EPI == DGATED);
      read(f, 0);
      read(g, 1);
      multiply(f);
      multiply(g);
      flip();
      // every wave has what it read of the buffer that is filled next
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_waitcnt(0xC07F);        // lgkmcnt alone
      block_barrier();
      ask(EPI == DGATED);
    }
#pragma unroll
    for (int i = 0; i < XT; ++i) {
      // (of the largest tile one row after the other, for want of registers)
      if (EPI == DGATED && GT == 4) {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
      }
      const long n = row + r + i * 16;
      if (n >= p.N) continue;
      ushort* to = reinterpret_cast<ushort*>(
          reinterpret_cast<char*>(p.y + (row + i * 16) * ldy) + at);
      if constexpr (EPI == GATED) {
        put_gated<ACT, GT>(p, to, hl, acc[i], acc[i] + GT);
      } else if constexpr (EPI == DGATED) {
        put_dgated<ACT, GT>(p, to, hl, acc[i], acc[i] + GT, dy[i]);
      } else {
        put_plain<GT>(p, to, n, hl, acc[i]);
        put_plain<GT>(p, to + GT * 16, n, hl + GT * 16, acc[i] + GT);
      }
    }
    whole = row + BM <= p.N && h + HT <= p.H && p.H % (GT == 1 ? 4 : 8) == 0;
  }
  if (EPI == DGATED) wait_queue<0>();
}

// The same for few rows of x. Bound by reading w, and by how long that takes
// one after the other: a block's four waves share 16 columns (of gate and up;
// 32 of a plain product) and cut the reduction, step by step in turn; their
// sums are added in order in LDS. Operands go from memory to registers, two
// steps ahead. (200 rows, K = H = 384: 4.2 us; side by side 4.6, where the
// tiles of 64 by 32 took 4.7 and an empty launch 2.)
template <int EPI, int ACT, int XT>
__launch_bounds__(256)
__global__ void k_rows_skinny(BtArgs p) {
  constexpr int HT = EPI == PLAIN ? 32 : 16;
  __shared__ f32x4 sums[4][XT][2][64];
  const int nC = (p.H + HT - 1) / HT;
  const int wg = xcd_chunked(blockIdx.x, gridDim.x);
  const long row0 = (long)(wg / nC) * XT * 16;
  const int h0 = (wg % nC) * HT;
  const int lane = threadIdx.x & 63;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, q = lane >> 4;

  const ushort *x[XT], *w[2];
#pragma unroll
  for (int i = 0; i < XT; ++i)
    x[i] = p.x + min(row0 + i * 16 + l16, (long)p.N - 1) * p.ldx;
#pragma unroll
  for (int g = 0; g < 2; ++g)
    w[g] = p.w + (EPI == PLAIN ? (long)min(h0 + g * 16 + l16, p.H - 1)
                               : (long)g * p.H + min(h0 + l16, p.H - 1)) * p.K;
  struct Step { bf16x8 x[XT], w[2]; };
  auto load = [&](int s) {
    const int k = s * 32 + q * 8;
    Step v;
#pragma unroll
    for (int i = 0; i < XT; ++i)
      v.x[i] = *reinterpret_cast<const bf16x8*>(k < p.K ? x[i] + k : k_zero_chunk);
#pragma unroll
    for (int g = 0; g < 2; ++g)
      v.w[g] = *reinterpret_cast<const bf16x8*>(k < p.K ? w[g] + k : k_zero_chunk);
    return v;
  };
  f32x4 acc[XT][2];
#pragma unroll
  for (int i = 0; i < XT; ++i)
#pragma unroll
    for (int g = 0; g < 2; ++g) acc[i][g] = {0.f, 0.f, 0.f, 0.f};
  auto step = [&](const Step& v) {
#pragma unroll
    for (int i = 0; i < XT; ++i)
#pragma unroll
      for (int g = 0; g < 2; ++g)
        acc[i][g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v.w[g], v.x[i], acc[i][g],
                                                            0, 0, 0);
  };
  // beyond the end the chunks are zeros, and add nothing
  Step a = load(wid), b = load(wid + 4);
  const int steps = (p.K + 31) / 32;
  for (int s = wid; s < steps; s += 8) {
    const Step c = load(s + 8), d = load(s + 12);
    step(a);
    step(b);
    a = c;
    b = d;
  }
#pragma unroll
  for (int i = 0; i < XT; ++i)
#pragma unroll
    for (int g = 0; g < 2; ++g) sums[wid][i][g][lane] = acc[i][g];
  __syncthreads();
  if (wid >= XT) return;
  const long n = row0 + wid * 16 + l16;
  if (n >= p.N) return;
  f32x4 v[2];
#pragma unroll
  for (int g = 0; g < 2; ++g)
    v[g] = sums[0][wid][g][lane] + sums[1][wid][g][lane] + sums[2][wid][g][lane] +
           sums[3][wid][g][lane];
  const int h = h0 + q * 4;
  ushort* to = p.y + n * (EPI == DGATED ? 2 * p.Hp : p.H) + h;
  if constexpr (EPI == GATED) {
    put_gated<ACT, 1>(p, to, h, v, v + 1);
  } else if constexpr (EPI == DGATED) {
    put_dgated<ACT, 1>(p, to, h, v, v + 1, read_dy<1>(p, p.dy + n * p.lddy + h, h));
  } else {
    put_plain<1>(p, to, n, h, v);
    put_plain<1>(p, to + 16, n, h + 16, v + 1);
  }
}

// ---------------------------------------------------------------------------
// dW: the reduction runs down the columns of both operands, over N rows. The
// tiles lie in LDS as they lie in memory, and the transposing LDS read hands
// each lane four rows of its column. The order of the rows within a step of
// 32 is the same for both operands and does not matter to the sum: lane
// group q takes rows 4q..4q+3 and 16+4q..16+4q+3, so that one read covers 16
// neighbouring rows, whose 32-byte units the exclusive-or below spreads over
// all banks. N is split over blocks; the parts are added in order by
// k_dw_reduce, so that a result never depends on timing.
// 204800 rows, K = H = 384: 155 us (780 TFLOP/s, 472 MB read and 66 written),
// the parts' sum 12 us; 14351 rows of 1440: 144 us (830 TFLOP/s) and 11. Bound as
// the products above: matrix units 33% of the cycles, LDS reads 13%. Reading the next step's operands ahead needs registers that
// the sums take (272 us with spills; with sums of 192 by 128, 211).
// ---------------------------------------------------------------------------

constexpr int TN_ROWS = 32;

// where the 16-column unit `unit` of row r lies, in rows of `cols` columns
DEVI int dw_place(int unit, int r, int cols) {
  return unit ^ (r & 7 & (cols / 16 - 1));
}

DEVI bf16x8 tr_read(const ushort* tile, int stride, int c0, int l16, int q) {
  s16x4 v[2];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int r = half * 16 + q * 4 + (l16 >> 2);
    const int unit = dw_place(c0 >> 4, r, stride);
    const ushort* a = tile + r * stride + unit * 16 + (l16 & 3) * 4;
    v[half] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s16x4*)a);
  }
  bf16x4 lo = __builtin_bit_cast(bf16x4, v[0]);
  bf16x4 hi = __builtin_bit_cast(bf16x4, v[1]);
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// d_w is float32 or bf16: one of d_w32 and d_w is null
DEVI void put_sums(float* to, const float* v, int h, int H) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (h + j < H) to[j] = v[j];
}

template <int WA, int WB, int AT, int BT>
__launch_bounds__(WA * WB * 64, 2)
__global__ void k_dw_part(const ushort* __restrict__ dgu,
                          const ushort* __restrict__ x, long ldx,
                          float* __restrict__ part, ushort* __restrict__ d_w,
                          float* __restrict__ d_w32, int N, int C2, int K, int K8,
                          int H, int rows_each, int tiles) {
  constexpr int T = WA * WB * 64;
  constexpr int CA = WA * AT * 16;     // columns of dgu a block
  constexpr int CB = WB * BT * 16;     // columns of x a block
  constexpr int ITA = TN_ROWS * CA / 8 / T, ITB = TN_ROWS * CB / 8 / T;
  static_assert(TN_ROWS * CA / 8 % T == 0 && TN_ROWS * CB / 8 % T == 0, "staging");
  extern __shared__ ushort lds[];
  constexpr int BUF = TN_ROWS * (CA + CB);

  const int nB = (K + CB - 1) / CB;
  // the tiles of one part of the rows share an L2
  const int wg = xcd_chunked(blockIdx.x, gridDim.x);
  const int tile = wg % tiles, slice = wg / tiles;
  const int a0 = tile / nB * CA, b0 = tile % nB * CB;
  const long n0 = (long)slice * rows_each;
  const long n1 = min(n0 + rows_each, (long)N);

  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wa = wid / WB, wb = wid % WB;
  const int l16 = lane & 15, q = lane >> 4;

  // bytes behind the step's first row of dgu or of x; columns that are not
  // there read others, and what becomes of them is not stored
  u32 off[ITA + ITB];
#pragma unroll
  for (int it = 0; it < ITA + ITB; ++it) {
    const bool ina = it < ITA;
    const int c = (ina ? it : it - ITA) * T + tid;
    const int per = (ina ? CA : CB) / 8;
    const int r = c / per, pos = c % per;
    const int cc = (dw_place(pos >> 1, r, ina ? CA : CB) * 2 + (pos & 1)) * 8;
    off[it] = ina ? (u32)((long)r * C2 + (a0 + cc < C2 ? a0 + cc : 0)) * 2
                  : (u32)((long)r * ldx + (b0 + cc < K8 ? b0 + cc : 0)) * 2;
  }
  auto stage = [&](long n, int buf) {
    ushort* dst = lds + buf * BUF + wid * 512;
    const char* ap = reinterpret_cast<const char*>(dgu + n * C2);
    const char* bp = reinterpret_cast<const char*>(x + n * ldx);
    if (n + TN_ROWS <= n1) {
      ap = in_scalar(ap);
      bp = in_scalar(bp);
#pragma unroll
      for (int it = 0; it < ITA + ITB; ++it)
        to_lds16((it < ITA ? ap : bp) + off[it],
                 dst + (it < ITA ? it * T * 8 : TN_ROWS * CA + (it - ITA) * T * 8));
    } else {
#pragma unroll
      for (int it = 0; it < ITA + ITB; ++it) {
        const bool ina = it < ITA;
        const int r = ((ina ? it : it - ITA) * T + tid) / ((ina ? CA : CB) / 8);
        const char* s = (ina ? ap : bp) + off[it];
        to_lds16(n + r < n1 ? (const void*)s : k_zero_chunk,
                 dst + (ina ? it * T * 8 : TN_ROWS * CA + (it - ITA) * T * 8));
      }
    }
  };

  f32x4 acc[AT][BT];
#pragma unroll
  for (int i = 0; i < AT; ++i)
#pragma unroll
    for (int j = 0; j < BT; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};

  const int steps = (int)((n1 - n0 + TN_ROWS - 1) / TN_ROWS);
  if (steps > 0) stage(n0, 0);
  if (steps > 1) stage(n0 + TN_ROWS, 1);
  int buf = 0;
  for (int s = 0; s < steps; ++s) {
    if (s + 1 < steps) wait_queue<ITA + ITB>();
    else wait_queue<0>();
    block_barrier();
    if (s + 2 < steps)
      stage(n0 + (long)(s + 2) * TN_ROWS, buf == 0 ? 2 : buf - 1);
    const ushort* la = lds + buf * BUF;
    const ushort* lb = la + TN_ROWS * CA;
    buf = buf == 2 ? 0 : buf + 1;
    bf16x8 af[AT], bf[BT];
#pragma unroll
    for (int i = 0; i < AT; ++i)
      af[i] = tr_read(la, CA, (wa * AT + i) * 16, l16, q);
#pragma unroll
    for (int j = 0; j < BT; ++j)
      bf[j] = tr_read(lb, CB, (wb * BT + j) * 16, l16, q);
#pragma unroll
    for (int i = 0; i < AT; ++i)
#pragma unroll
      for (int j = 0; j < BT; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af[i], bf[j],
                                                            acc[i][j], 0, 0, 0);
  }
  // part (S, K, C2), or d_w itself if the rows are one part: a lane holds four
  // consecutive columns of C2
#pragma unroll
  for (int j = 0; j < BT; ++j) {
    const int k = b0 + (wb * BT + j) * 16 + l16;
    if (k >= K) continue;
#pragma unroll
    for (int i = 0; i < AT; ++i) {
      const int c = a0 + (wa * AT + i) * 16 + q * 4;
      if (c >= C2) continue;
      if (part) {
        *reinterpret_cast<f32x4*>(part + ((long)slice * K + k) * C2 + c) = acc[i][j];
      } else {
        const int g = c >= C2 / 2, h = c - g * (C2 / 2);
        const float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
        const long at = ((long)g * K + k) * H + h;
        if (d_w32) put_sums(d_w32 + at, v, h, H);
        else put<1>(d_w + at, v, h, H);
      }
    }
  }
}

// d_w (2, K, H) from the parts (S, K, 2, Hp). 56 parts of 384 by 768 (66 MB):
// 11.9 us, and 17.7 with fewer loads on their way at a time.
__launch_bounds__(256)
__global__ void k_dw_reduce(const float* __restrict__ part,
                            ushort* __restrict__ d_w, float* __restrict__ d_w32,
                            int S, int K, int H, int Hp) {
  const long quads = (long)K * 2 * Hp / 4;
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= quads) return;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int s = 0; s < S; ++s)
    sum += *reinterpret_cast<const f32x4*>(part + (s * quads + i) * 4);
  const long k = i * 4 / (2 * Hp);
  const int c = (int)(i * 4 % (2 * Hp));
  const int g = c / Hp, h = c % Hp;
  const float v[4] = {sum[0], sum[1], sum[2], sum[3]};
  const long at = ((long)g * K + k) * H + h;
  if (d_w32) put_sums(d_w32 + at, v, h, H);
  else put<1>(d_w + at, v, h, H);
}

// (R, C) with rows ld apart -> (R, Cp), the columns behind C zero
__launch_bounds__(256)
__global__ void k_pad_cols(const ushort* __restrict__ in, long ld,
                           ushort* __restrict__ out, long R, int C, int Cp) {
  const long total = R * (Cp / 8);
  for (long c = (long)blockIdx.x * 256 + threadIdx.x; c < total;
       c += (long)gridDim.x * 256) {
    const long r = c / (Cp / 8);
    const int k = (int)(c % (Cp / 8)) * 8;
    u16x8 v = {};
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (k + j < C) v[j] = in[r * ld + k + j];
    *reinterpret_cast<u16x8*>(out + r * Cp + k) = v;
  }
}

// ===========================================================================
// host wrappers
// ===========================================================================

inline int pad8(int v) { return (v + 7) / 8 * 8; }

const ushort* bf_ptr(const torch::Tensor& t) {
  return reinterpret_cast<const ushort*>(t.data_ptr<at::BFloat16>());
}
ushort* bf_mut(const torch::Tensor& t) {
  return reinterpret_cast<ushort*>(t.data_ptr<at::BFloat16>());
}

void check_bf16(const torch::Tensor& t, const char* name, int dims,
                const torch::Tensor& like) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), name,
              " must be on the GPU that ctx is on");
  TORCH_CHECK(t.scalar_type() == torch::kBFloat16, name, " must be bfloat16");
  TORCH_CHECK(t.dim() == dims, name, " must have ", dims, " dimensions");
}

void check_size(long N, long K, long H) {
  TORCH_CHECK(N < (1L << 31) && K < (1L << 22) && H < (1L << 21) &&
              (K + 8) * (H + 8) < (1L << 30),
              "ctx (", N, ", ", K, ") or the weights to ", H, " are too large");
}

// Rows whose values follow each other, start on 16 bytes and are a multiple
// of eight long: `t` itself, or a padded copy of it.
struct Rows {
  torch::Tensor held;
  const ushort* p;
  long ld;
};

Rows chunked_rows(const torch::Tensor& t, int cols) {
  const bool dense = t.size(1) <= 1 || t.stride(1) == 1;
  const long ld = t.size(0) <= 1 ? pad8(cols) : t.stride(0);
  // (offsets within a tile have 32 bits)
  if (dense && cols % 8 == 0 && ld % 8 == 0 && ld >= 0 && ld < (1l << 23) &&
      (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0)
    return {t, bf_ptr(t), ld};
  auto src = dense ? t : t.contiguous();
  auto out = torch::empty({t.size(0), (long)pad8(cols)}, t.options());
  const long items = t.size(0) * (pad8(cols) / 8);
  k_pad_cols<<<grid_of(items, 256, 8192), 256, 0, cur_stream()>>>(
      bf_ptr(src), src.size(0) <= 1 ? cols : src.stride(0), bf_mut(out),
      t.size(0), cols, pad8(cols));
  return {out, bf_ptr(out), (long)pad8(cols)};
}

// `slots` blocks at a time, each over several tiles
template <int EPI, int ACT, int WR, int WC, int XT, int GT, int BK, int STAGES>
void launch_rows(const BtArgs& a, long slots) {
  constexpr int BM = WR * XT * 16, BG = WC * GT * 16;
  constexpr int HT = EPI == PLAIN ? 2 * BG : BG;
  constexpr size_t bytes = (size_t)STAGES * (BM + 2 * BG) * BK * sizeof(ushort);
  auto* fn = &k_rows_gemm<EPI, ACT, WR, WC, XT, GT, BK, STAGES>;
  static std::atomic<u64> ready{0};
  allow_lds(fn, bytes, ready);
  const long tiles = ((long)a.N + BM - 1) / BM * ((a.H + HT - 1) / HT);
  TORCH_CHECK(tiles < (1L << 31), "too many tiles for one launch");
  // (asking ahead goes into the next tile, not into the one after that)
  const bool stay = (a.K + BK - 1) / BK >= STAGES;
  fn<<<(int)(stay ? std::min(tiles, slots) : tiles), WR * WC * 64, bytes,
       cur_stream()>>>(a);
  C10_HIP_KERNEL_LAUNCH_CHECK();
}

template <int EPI, int ACT, int XT>
void launch_skinny(const BtArgs& a) {
  constexpr int HT = EPI == PLAIN ? 32 : 16;
  const long tiles = ((long)a.N + XT * 16 - 1) / (XT * 16) * ((a.H + HT - 1) / HT);
  TORCH_CHECK(tiles < (1L << 31), "too many tiles for one launch");
  auto* fn = &k_rows_skinny<EPI, ACT, XT>;
  fn<<<(int)tiles, 256, 0, cur_stream()>>>(a);
  C10_HIP_KERNEL_LAUNCH_CHECK();
}

// What a launch takes, in us: `slots` blocks run at a time; a step takes one
// of them `alone` in an idle chip and `full` in a full one.
double launch_us(double blocks, double slots, double steps, double alone,
                 double full, double fixed) {
  const double load = std::min(1.0, blocks / slots);
  return std::ceil(blocks / slots) * (fixed + steps * (alone + (full - alone) * load));
}

// Tiles from 256 rows by 128 columns of gate and up down to 16 by 16: large
// ones read least, small ones fill the chip. The rates are fitted to both
// products at 1..204800 rows and widths of 96..1440; what they choose is the
// best or within a tenth of it at six sizes of seven. The gated product, in us (20
// calls of each; in a longer run the last row's first is 141, the one above it 124):
//   rows  width   256x128   128x64   64x32   32x16
//    200    384      13.1      6.7     4.7     4.6
//   1024    768      22.9     11.3     8.7    19.5
//   4096   1440      47.8     48.5    83.8   182
//  14351   1440       135      144     257    624
// 204800    384       154      168     279    906
// A plain product of the largest tile needs more registers than there are
// (K = 768 to H = 384, 204800 rows: 207 us, in tiles of 128 by 128 162).
template <int EPI, int ACT>
void rows_gemm(const BtArgs& a) {
  constexpr double plain = EPI == PLAIN ? 2 : 1;    // groups of columns a tile
  auto blocks = [&](double rows, double cols) {
    return std::ceil(a.N / rows) * std::ceil(a.H / (cols * plain));
  };
  const double k64 = (a.K + 63) / 64, k32 = (a.K + 31) / 32;
  const double us[] = {
      launch_us(blocks(256, 128), 256, k64, 1.25, 2.2, 5.0),
      launch_us(blocks(128, 64), 512, k64, 0.60, 1.25, 3.0),
      launch_us(blocks(64, 32), 768, k64, 0.30, 0.85, 2.0),
      launch_us(blocks(a.N <= 16 ? 16 : 32, 16), 1024, k32, 0.045, 0.36, 2.6)};
  const int first = EPI == PLAIN ? 1 : 0;
  switch (std::min_element(us + first, us + 4) - us) {
    case 0:
      if constexpr (EPI != PLAIN) return launch_rows<EPI, ACT, 4, 2, 4, 4, 64, 2>(a, 256);
    case 1: return launch_rows<EPI, ACT, 2, 2, 4, 2, 64, 2>(a, 512);
    case 2: return launch_rows<EPI, ACT, 2, 2, 2, 1, 64, 3>(a, 768);
    default:
      if (a.N <= 16) launch_skinny<EPI, ACT, 1>(a);
      else launch_skinny<EPI, ACT, 2>(a);
  }
}

// dW by tiles of CA columns of dgu by CB of x, the rows in S parts. A part
// more than fills the chip costs a whole round, and every part costs the
// writing and reading of its sums. Fitted like the rates of rows_gemm; what is
// chosen is the best of these, or within 13% of it, at ten sizes. In us, each
// tile with its best number of parts, their sum included (20 calls of each, as above):
//   rows  K to H       256x128   128x128   64x64
//    512  192 to 192      11.8       9.7     8.3
//   2000 1000 to 1000     30.0      27.0    29.5
//   7000 1250 to 720      52.1      50.8    67.6
//  14351 1440 to 1440      169       171     226
// 100000  200 to 200       181        61      68
// 204800  384 to 384       187       192     272
struct DwPlan { double us; int S; };

DwPlan plan_dw(long N, long C2, long K, int CA, int CB, double slots, double fixed,
               double alone, double full) {
  const double tiles = std::ceil(C2 / (double)CA) * std::ceil(K / (double)CB);
  DwPlan best{1e30, 1};
  for (int S = 1; S <= 64 && (S == 1 || N / S >= 64); ++S) {
    const double us = launch_us(tiles * S, slots, std::ceil(N / (double)S / TN_ROWS),
                                alone, full, fixed) +
                      (S > 1 ? 4.5 + S * (double)(C2 * K) * 8 / 5e6 : 0);
    if (us < best.us) best = {us, S};
  }
  return best;
}

template <int WA, int WB, int AT, int BT>
void launch_dw(const torch::Tensor& d_w, const ushort* dgu, const Rows& x, long N,
               int K, int H, int Hp, int S) {
  constexpr int CA = WA * AT * 16, CB = WB * BT * 16;
  constexpr size_t bytes = 3ul * TN_ROWS * (CA + CB) * sizeof(ushort);
  const int tiles = (2 * Hp + CA - 1) / CA * ((K + CB - 1) / CB);
  const int rows_each = (int)(((N + S - 1) / S + TN_ROWS - 1) / TN_ROWS * TN_ROWS);
  const bool f32 = d_w.scalar_type() == torch::kFloat32;
  ushort* dw16 = f32 ? nullptr : bf_mut(d_w);
  float* dw32 = f32 ? d_w.data_ptr<float>() : nullptr;
  torch::Tensor part;
  if (S > 1)
    part = torch::empty({S, K, 2L * Hp}, d_w.options().dtype(torch::kFloat32));
  auto* fn = &k_dw_part<WA, WB, AT, BT>;
  static std::atomic<u64> ready{0};
  allow_lds(fn, bytes, ready);
  fn<<<tiles * S, WA * WB * 64, bytes, cur_stream()>>>(
      dgu, x.p, x.ld, S > 1 ? part.data_ptr<float>() : nullptr, dw16, dw32, (int)N,
      2 * Hp, K, pad8(K), H, rows_each, tiles);
  C10_HIP_KERNEL_LAUNCH_CHECK();
  if (S == 1) return;
  const long quads = (long)K * 2 * Hp / 4;
  k_dw_reduce<<<(int)((quads + 255) / 256), 256, 0, cur_stream()>>>(
      part.data_ptr<float>(), dw16, dw32, S, K, H, Hp);
  C10_HIP_KERNEL_LAUNCH_CHECK();
}

#define WITH_ACT(act, ...)                                              \
  switch (act) {                                                        \
    case SILU: { constexpr int A = SILU; __VA_ARGS__; break; }          \
    case GELU: { constexpr int A = GELU; __VA_ARGS__; break; }          \
    case SIGMOID: { constexpr int A = SIGMOID; __VA_ARGS__; break; }    \
    case TANH: { constexpr int A = TANH; __VA_ARGS__; break; }          \
    case RELU: { constexpr int A = RELU; __VA_ARGS__; break; }          \
    default: TORCH_CHECK(false, "unknown activation ", act);            \
  }

// y (N,H)
torch::Tensor transform_gated_fwd(torch::Tensor ctx, torch::Tensor w_oi, int64_t act) {
  check_bf16(ctx, "ctx", 2, ctx);
  check_bf16(w_oi, "w_oi", 3, ctx);
  TORCH_CHECK(w_oi.size(0) == 2 && w_oi.size(2) == ctx.size(1) &&
              w_oi.is_contiguous(), "w_oi must be a contiguous (2, H, K)");
  check_size(ctx.size(0), ctx.size(1), w_oi.size(1));
  const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(ctx.device());
  const int N = ctx.size(0), K = ctx.size(1), H = w_oi.size(1);
  auto y = torch::empty({N, H}, ctx.options());
  if (N == 0 || H == 0) return y;
  if (K == 0) return y.zero_();          // act(0) * 0
  const Rows x = chunked_rows(ctx, K), w = chunked_rows(w_oi.view({2L * H, K}), K);
  BtArgs a{x.p, w.p, bf_mut(y), nullptr, x.ld, 0, N, H, pad8(H), pad8(K), 1.f, 0,
           nullptr};
  WITH_ACT(act, (rows_gemm<GATED, A>(a)));
  return y;
}

// d_ctx (N,K) and d_w (2,K,H), bf16 or, as it was summed, float32
std::vector<torch::Tensor> transform_gated_bwd(torch::Tensor ctx,
                                               torch::Tensor w_io,
                                               torch::Tensor w_oi,
                                               torch::Tensor d_y, int64_t act,
                                               double keep_prob, int64_t seed,
                                               c10::optional<torch::Tensor> seed_t,
                                               bool dw_f32) {
  check_bf16(ctx, "ctx", 2, ctx);
  check_bf16(w_io, "w_io", 2, ctx);
  check_bf16(d_y, "d_y", 2, ctx);
  const int N = ctx.size(0), K = ctx.size(1), H = d_y.size(1), Hp = pad8(H);
  check_size(ctx.size(0), ctx.size(1), d_y.size(1));
  TORCH_CHECK(d_y.size(0) == N, "d_y must have as many rows as ctx");
  TORCH_CHECK(w_io.size(0) == K && w_io.size(1) == 2L * H && w_io.is_contiguous(),
              "w_io must be a contiguous (K, 2H)");
  check_bf16(w_oi, "w_oi", 3, ctx);
  TORCH_CHECK(w_oi.size(0) == 2 && w_oi.size(1) == H && w_oi.size(2) == K &&
              w_oi.is_contiguous(), "w_oi must be a contiguous (2, H, K)");
  TORCH_CHECK(keep_prob > 0.0 && keep_prob <= 1.0, "keep_prob must be in (0, 1]");
  const long* seed_ptr = nullptr;
  if (seed_t) {
    TORCH_CHECK(seed_t->numel() == 1 && seed_t->device() == ctx.device() &&
                seed_t->scalar_type() == torch::kInt64,
                "seed_t must be one int64 on the GPU that ctx is on");
    seed_ptr = seed_t->data_ptr<long>();
  }
  const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(ctx.device());
  auto d_ctx = torch::empty({N, K}, ctx.options());
  auto d_w = torch::empty({2, K, H}, ctx.options().dtype(
      dw_f32 ? torch::kFloat32 : torch::kBFloat16));
  if (N == 0 || H == 0 || K == 0) return {d_ctx.zero_(), d_w.zero_()};

  const Rows x = chunked_rows(ctx, K);
  auto dgu = torch::empty({N, 2, Hp}, ctx.options());
  {
    const Rows dy = chunked_rows(d_y, H);
    const Rows w = chunked_rows(w_oi.view({2L * H, K}), K);
    BtArgs a{x.p, w.p, bf_mut(dgu), dy.p, x.ld, dy.ld, N, H, Hp, pad8(K), 1.f, 0,
             nullptr};
    WITH_ACT(act, (rows_gemm<DGATED, A>(a)));
  }

  Rows w;
  if (H == Hp) {
    w = chunked_rows(w_io, 2 * H);
  } else {
    w = chunked_rows(w_io.view({2L * K, H}), H);   // (K, 2, Hp)
  }
  BtArgs a{bf_ptr(dgu), w.p, bf_mut(d_ctx), nullptr, 2L * Hp, 0, N, K,
           pad8(K), 2 * Hp, (float)keep_prob, (u64)seed, seed_ptr};
  rows_gemm<PLAIN, SILU>(a);

  const DwPlan large = plan_dw(N, 2L * Hp, K, 256, 128, 512, 4.25, 0.86, 0.9);
  const DwPlan middle = plan_dw(N, 2L * Hp, K, 128, 128, 768, 1.8, 0.7, 0.76);
  const DwPlan small = plan_dw(N, 2L * Hp, K, 64, 64, 1536, 1.0, 0.5, 0.75);
  if (large.us <= std::min(middle.us, small.us))
    launch_dw<2, 2, 8, 4>(d_w, bf_ptr(dgu), x, N, K, H, Hp, large.S);
  else if (middle.us <= small.us)
    launch_dw<2, 2, 4, 4>(d_w, bf_ptr(dgu), x, N, K, H, Hp, middle.S);
  else
    launch_dw<2, 2, 2, 2>(d_w, bf_ptr(dgu), x, N, K, H, Hp, small.S);
  return {d_ctx, d_w};
}

}  // namespace

void bind_gated(pybind11::module_& mod) {
  mod.def("transform_gated_fwd", &transform_gated_fwd);
  mod.def("transform_gated_bwd", &transform_gated_bwd);
}
