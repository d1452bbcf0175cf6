// Device helpers shared by the kernels of this extension (gfx950).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#define DEVI __device__ __forceinline__

using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using bf16x4 = __attribute__((ext_vector_type(4))) __bf16;
using bf16x2 = __attribute__((ext_vector_type(2))) __bf16;
using u16x8 = __attribute__((ext_vector_type(8))) unsigned short;
using u16x4 = __attribute__((ext_vector_type(4))) unsigned short;
using s16x4 = __attribute__((ext_vector_type(4))) short;
using f32x4 = __attribute__((ext_vector_type(4))) float;
using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;
using i32x8 = __attribute__((ext_vector_type(8))) int;
using u32 = uint32_t;
using u64 = uint64_t;

DEVI float bf2f(ushort u) {
  union { u32 u; float f; } cvt;
  cvt.u = ((u32)u) << 16;
  return cvt.f;
}

// splitmix64 — must match code2vec_amd/ops/reference.py::_splitmix64 bit-for-bit
DEVI u64 splitmix64(u64 x) {
  u64 z = x * 0x9E3779B97F4A7C15ull;
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
  return z ^ (z >> 31);
}

DEVI float hash_uniform(u64 seed, u64 idx) {
  u64 h = splitmix64(seed + idx);
  return (float)((h >> 40) & 0xFFFFFFull) * (1.0f / 16777216.0f);
}

// Workgroups go round-robin over the 8 XCDs, each with an L2 of its own.
// This bijection gives each XCD a contiguous run of tile numbers instead, so
// that tiles that share a panel share an L2.
DEVI int xcd_chunked(int wg, int nwg) {
  const int nxcd = 8;
  const int q = nwg / nxcd, r = nwg % nxcd;
  const int xcd = wg % nxcd, orig = wg / nxcd;
  return (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + orig;
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
