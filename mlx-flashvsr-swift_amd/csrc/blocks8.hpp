// The 8-bit form of a matrix of tokens or weights, shared by the kernels that write and read it (rows8.hip,
// linear8.hip).
//
// A row of C channels is cut into runs of 128 (the last padded with zeros). A run has a scale 2^e, the smallest with e
// >= -127 and max |x| <= 448 * 2^e over its finite values, and each channel a code: the e4m3 number nearest to x / 2^e,
// ties to even, but at most 240 under the largest scale, 2^120, where the next number, 256, would stand for 2^128 (so
// what is finite comes back finite, and within 2^-4 of what it was: 240 * 2^120 is 15 / 16 of 2^128); an infinity or
// NaN becomes NaN. Codes are stored (rows, 128 * runs), scales as the byte e + 127 (E8M0), (rows, runs rounded up to
// 4), the bytes past the last run 0.
//
// Why a power of two: x / 2^e is exact, so the codes do not depend on how the quotient is formed; an element's value
// code * 2^e has 4 significant bits and is exact in bf16 and fp32; and the matrix cores' scaled products take the byte
// as it is, so no vector instruction ever multiplies by a scale. e4m3 being a floating format, a scale up to twice the
// tightest one costs no relative precision above its subnormals.
#pragma once
#include "common.hpp"

namespace fvsr {

constexpr int kRun = 128;
constexpr int kMaxFeatures = 1 << 20;   // channels of a row: a tile's 256 rows of codes stay below 2^31 bytes

// vectors of whole elements at any address: the hardware reads and writes global memory unaligned, in one instruction
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef u32x4 any16 __attribute__((aligned(2)));
typedef u32x2 any8 __attribute__((aligned(2)));
typedef f32x4 any_f32x4 __attribute__((aligned(4)));

struct In8 {
  const uint8_t* codes;
  const uint8_t* scales;
};
struct Out8 {
  uint8_t* codes;
  uint8_t* scales;
};

__host__ __device__ __forceinline__ int runs_of(int channels) { return (channels + kRun - 1) / kRun; }
__host__ __device__ __forceinline__ int scale_stride(int channels) { return (runs_of(channels) + 3) & ~3; }

// max over each 16 lanes of a wave (every lane active, x >= 0), in every one of them: DPP rotations within the rows of
// 16
__device__ __forceinline__ float max16(float x) {
  auto rot = [](float v, auto ctrl) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, 0xf, 0xf, false));
  };
  x = fmaxf(x, rot(x, std::integral_constant<int, 0x128>{}));   // row_ror:8
  x = fmaxf(x, rot(x, std::integral_constant<int, 0x124>{}));
  x = fmaxf(x, rot(x, std::integral_constant<int, 0x122>{}));
  x = fmaxf(x, rot(x, std::integral_constant<int, 0x121>{}));
  return x;
}

// Encodes a run held by 16 lanes, 8 values each: the codes of this lane's values in order, and the run's scale byte.
// With top = 1.f * 2^(E - 127), the smallest e is E - 127 - 8, one more where 1.f > 1.75 (448 = 1.75 * 2^8). Magnitudes
// above 240 * 2^120 exist under the scale 2^120 only, and are cut to that: it changes no other value's code.
__device__ __forceinline__ uint2 encode8(const float (&v)[8], uint32_t& scale) {
  float top = 0.f;
  float f[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const bool finite = fabsf(v[e]) <= 3.402823466e38f;   // false for NaN
    f[e] = finite ? __builtin_amdgcn_fmed3f(v[e], -0x1.ep127f, 0x1.ep127f) : __uint_as_float(0x7fc00000u);
    top = fmaxf(top, fabsf(f[e]));                        // the other one where f is NaN
  }
  const uint32_t bits = __float_as_uint(max16(top));
  const int s = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  scale = (uint32_t)max(s, 0);                                       // <= 247
  const float inv = __uint_as_float((254u - scale) << 23);           // 2^-e, a normal number
  uint2 c;
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(f[0] * inv, f[1] * inv, 0, false);
  c.x = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[2] * inv, f[3] * inv, w, true);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(f[4] * inv, f[5] * inv, 0, false);
  c.y = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[6] * inv, f[7] * inv, w, true);
  return c;
}

// the values of 8 codes under a scale byte (exact)
__device__ __forceinline__ void decode8(uint2 c, uint32_t scale, float (&v)[8]) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const float by = __uint_as_float(scale << 23);   // the instruction reads the exponent bits: 2^(scale - 127)
  f32x2 p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c.x, by, false);
  v[0] = p[0]; v[1] = p[1];
  p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c.x, by, true);
  v[2] = p[0]; v[3] = p[1];
  p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c.y, by, false);
  v[4] = p[0]; v[5] = p[1];
  p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c.y, by, true);
  v[6] = p[0]; v[7] = p[1];
}

// A lane (l16 = lane % 16) holds 8 adjacent channels of a run, 8 l16 .. 8 l16 + 7. As they lie in memory, zeros past
// the row's end: loaded now, widened when they are needed. Rows of any length and alignment are read and written by
// whole vectors, but for a last part of 8; EIGHTS: rows have none (C is a multiple of 8), and no registers are spent on
// it.
template <typename T>
struct Raw8 {
  T v[8];
};
template <typename T, bool EIGHTS>
__device__ __forceinline__ Raw8<T> load_raw8(const T* row, int c0, int l16, int C) {
  Raw8<T> r;
  const int c = c0 + l16 * 8;
  u32x4* const to = (u32x4*)r.v;
  to[0] = u32x4{0, 0, 0, 0};
  if constexpr (sizeof(T) == 4) to[1] = u32x4{0, 0, 0, 0};
  if (c + 8 <= C) {
    to[0] = *(const any16*)(row + c);
    if constexpr (sizeof(T) == 4) to[1] = *(const any16*)(row + c + 4);
  } else if (!EIGHTS && c < C) {
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (c + e < C) r.v[e] = row[c + e];
  }
  return r;
}
template <typename T, bool EIGHTS>
__device__ __forceinline__ void load8(const T* row, int c0, int l16, int C, float (&v)[8]) {
  const Raw8<T> r = load_raw8<T, EIGHTS>(row, c0, l16, C);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (float)r.v[e];
}

// the other way: channels c .. c + 7, but for the first `skip` and those past the row's end
template <typename T, bool EIGHTS>
__device__ __forceinline__ void store8(T* row, int c, int skip, int C, const float (&v)[8]) {
  T t[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) t[e] = (T)v[e];
  if (c + 8 <= C && (EIGHTS || skip == 0)) {
    *(any16*)(row + c) = *(u32x4*)t;
    if constexpr (sizeof(T) == 4) *(any16*)(row + c + 4) = ((u32x4*)t)[1];
  } else if (!EIGHTS) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e >= skip && c + e < C) row[c + e] = t[e];
  }
}

// the 8 codes of a lane of a run that starts at `run` (whole runs are stored: what lies past the last channel is 0)
__device__ __forceinline__ void store_codes(uint8_t* run, int l16, uint2 c) { *(uint2*)(run + l16 * 8) = c; }
__device__ __forceinline__ uint2 load_codes(const uint8_t* run, int l16) { return *(const uint2*)(run + l16 * 8); }

}  // namespace fvsr
