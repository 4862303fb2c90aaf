// Pieces the matrix-core attention kernels share: operand types, the
// transposing LDS read, conversions to halves.
//
// Operands of v_mfma_f32_32x32x16_f16, lane l, h = l / 32: A (m = l % 32) and
// B (n = l % 32) hold k = 8h .. 8h+7; C holds n = l % 32 and, in register i,
// m = 8 (i / 4) + 4h + i % 4. Of v_mfma_f32_16x16x32_f16, g = l / 16: A and B
// hold k = 8g .. 8g+7 of row or column l % 16; C holds n = l % 16 and, in
// register i, m = 4g + i. Both take f16 subnormals as they are.
#pragma once

#include "common.h"

namespace prana {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// A value in device memory, at a byte offset from a base. Said outright: a
// pointer that came through a register exchange or an opaque assembly statement
// may point anywhere for all the compiler knows, and its generic loads count
// as LDS accesses too, so that each wait for LDS would wait for the loads of the
// next tile with it (4 prompts up to 1025, 8/1 x 256: 39.1 us with them, 37.3
// without; 2 prompts up to 8191, 32/8 x 128: 828, 816).
template <class T>
using device_t = __attribute__((address_space(1))) T;
template <class T>
__device__ __forceinline__ T load_at(const void* base, uint32_t off = 0) {
  return *(const device_t<T>*)((const device_t<unsigned char>*)(base) + off);
}

// Transposing LDS read of halves: the 16 lanes of a group read 4 rows of 16
// (lane l the four at row l / 4, column 4 (l % 4)), and lane l gets column l,
// rows 0..3.
__device__ __forceinline__ half4 lds_read_tr(const uint16_t* p) {
  typedef __attribute__((address_space(3))) short4v* lds_ptr;
  const short4v v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p));
  return __builtin_bit_cast(half4, v);
}

__device__ __forceinline__ half8 join(half4 a, half4 b) {
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// For a stretch of N LDS reads that feed M products each: two reads first, then
// one after each read's products, so that a read's wait is behind those of the
// one before. (On its own the compiler waits for pairs where registers are few.)
template <int N, int M>
__device__ __forceinline__ void reads_ahead() {
  constexpr int kProduct = 0x008, kRead = 0x100;
  __builtin_amdgcn_sched_group_barrier(kRead, 2, 0);
#pragma unroll
  for (int i = 0; i < N - 2; i++) {
    __builtin_amdgcn_sched_group_barrier(kProduct, M, 0);
    __builtin_amdgcn_sched_group_barrier(kRead, 1, 0);
  }
  __builtin_amdgcn_sched_group_barrier(kProduct, 2 * M, 0);
}

// 2^x as the hardware computes it (1 ulp; results under 2^-126 are 0).
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// Scores of 2^22 and more (log2 units) lie half a unit and more apart: a
// difference of them is taken before it is multiplied or shifted, or rounding
// could carry a probability past a half's end.
__device__ __forceinline__ bool coarse(float x) { return fabsf(x) >= 0x1p22f; }

// Bit 15 of each half of the result: that half of w is an infinity or NaN
// (its exponent, all ones, carries into the sign's place).
__device__ __forceinline__ uint32_t odd_halves(uint32_t w) { return (w & 0x7c007c00u) + 0x04000400u; }
__device__ __forceinline__ uint32_t odd_halves(u32x4 v) {
  return odd_halves(v.x) | odd_halves(v.y) | odd_halves(v.z) | odd_halves(v.w);
}
constexpr uint32_t kOddBits = 0x80008000u;
// w with its halves that are not finite replaced by 0.
__device__ __forceinline__ uint32_t only_finite(uint32_t w) {
  return w & ~(((odd_halves(w) & kOddBits) >> 15) * 0xffffu);
}
__device__ __forceinline__ u32x4 only_finite(u32x4 v) {
  return u32x4{only_finite(v.x), only_finite(v.y), only_finite(v.z), only_finite(v.w)};
}

// Two f32 as two halves each, x = hi + lo to 22 bits (|x| under 65504; lo has
// steps of at least 2^-24): one conversion for the pair of hi, and one
// instruction for each lo, x - hi rounded to a half. The values are opaque: a
// product that feeds one would be fused with its rounding to hi, but not with
// the one to lo, and the two would not belong together where the product lies
// near a tie. The factor is, or the product with it would become a subtraction
// and a rounding of its own.
__device__ __forceinline__ void split_pair(float x0, float x1, half2v& hi, half2v& lo) {
  float minus = -1.0f;
  asm("" : "+v"(x0), "+v"(x1));
  asm("" : "+s"(minus));
  const f32x2 x = {x0, x1};
  hi = __builtin_convertvector(x, half2v);
  lo = half2v{static_cast<_Float16>(fmaf(static_cast<float>(hi.x), minus, x0)),
              static_cast<_Float16>(fmaf(static_cast<float>(hi.y), minus, x1))};
}
// The power of two that brings amax into [2^9, 2^10), where both halves of a
// split are far from their limits; 1 where amax is 0 or not finite.
__device__ __forceinline__ float row_factor(float amax) {
  const uint32_t e = __float_as_uint(amax) >> 23;
  if (e == 0u || e == 255u) return amax > 0.0f && e == 0u ? 0x1p126f : 1.0f;
  const int k = 9 + 127 - static_cast<int>(e);
  return __builtin_ldexpf(1.0f, k < -126 ? -126 : k > 126 ? 126 : k);
}

// A row's q as the score product's operand, PIECES pieces of 8 dims, piece s at
// dim s * STEP + d0: loaded raw first (so that the first tile's loads can
// follow at once; loads return in order), then as halves, the f32 form as two
// each, normalised. LANES: lanes (a power of two apart) that hold one row.
template <int PIECES, int STEP, int LANES, bool HALF>
struct QRow {
  static constexpr int kWords = HALF ? 4 : 8;  // registers of 8 values
  uint32_t raw[PIECES][kWords];
  __device__ __forceinline__ void load(const void* q, size_t at, uint32_t d0, uint32_t hd) {
#pragma unroll
    for (int s = 0; s < PIECES; s++) {
      const unsigned char* p =
          static_cast<const unsigned char*>(q) + (at + min(s * STEP + d0, hd - 8)) * (HALF ? 2 : 4);
#pragma unroll
      for (int j = 0; j < kWords; j += 4) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(p + j * 4);
        raw[s][j] = w.x;
        raw[s][j + 1] = w.y;
        raw[s][j + 2] = w.z;
        raw[s][j + 3] = w.w;
      }
    }
  }
  // Returns what a score is multiplied with to be in log2 units.
  __device__ __forceinline__ float halves(float scale, uint32_t d0, uint32_t hd, half8* qh, half8* ql) {
#pragma unroll
    for (int s = 0; s < PIECES; s++)
      if (s * STEP + d0 >= hd)
#pragma unroll
        for (int j = 0; j < kWords; j++) raw[s][j] = 0;  // past the head's width
    if constexpr (HALF) {
#pragma unroll
      for (int s = 0; s < PIECES; s++)
        qh[s] = __builtin_bit_cast(half8, u32x4{raw[s][0], raw[s][1], raw[s][2], raw[s][3]});
      return scale;
    } else {
      float amax = 0.0f;
#pragma unroll
      for (int s = 0; s < PIECES; s++)
#pragma unroll
        for (int j = 0; j < 8; j++) amax = fmaxf(amax, fabsf(__uint_as_float(raw[s][j])));
#pragma unroll
      for (int o = 64 / LANES; o < 64; o <<= 1) amax = fmaxf(amax, __shfl_xor(amax, o, 64));
      const float f = row_factor(amax);
#pragma unroll
      for (int s = 0; s < PIECES; s++)
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          half2v xh, xl;
          split_pair(__uint_as_float(raw[s][j]) * f * scale, __uint_as_float(raw[s][j + 1]) * f * scale, xh, xl);
          qh[s][j] = xh.x;
          qh[s][j + 1] = xh.y;
          ql[s][j] = xl.x;
          ql[s][j + 1] = xl.y;
        }
      return 1.0f / f;  // a power of two: exact
    }
  }
};

}  // namespace prana
