// Blocks of 128 values in 8 bits with a power-of-two scale, and element types
// (gfx950): shared by the 8-bit optimizer states (tt_adamw.hip) and the
// embedding catalogue (tt_catalogue.hip).
//
// A power of two as scale makes every step but the rounding itself exact:
// scaling moves the exponent only, a decoded e4m3 value times its scale is
// exact in bfloat16 (4 significant bits).  It costs up to one of e4m3's 17
// binades of range, no precision.
#pragma once
#include "tt_common.h"

namespace tt {
namespace b8 {

constexpr int BLK = TT_BLOCK;    // values that share a scale
constexpr int LANES = 16;        // lanes that hold one block: 8 values each, one DPP row
constexpr int MIN_EXP = -100;    // smallest scale exponent: 2^-e stays a normal float
// Added to the bits of the largest magnitude, these carry into the exponent
// exactly when its significand exceeds that of the largest code: 448 = 1.75 * 2^8
// (e4m3), 480 = 1.875 * 2^8 (unsigned e4m4, whose code 255 stands for NaN).
constexpr uint32_t CARRY_M = 0x1FFFFFu, CARRY_R = 0x0FFFFFu;
constexpr int MANT_M = 3, MANT_R = 4;
constexpr uint32_t NAN_M = 0x7Fu, NAN_R = 0xFFu;

// scale byte (exponent + 127) of a block whose largest finite magnitude has these bits
__device__ __forceinline__ int scale_byte(uint32_t amax_bits, uint32_t carry) {
  return max((int)((amax_bits + carry) >> 23) - 135, MIN_EXP) + 127;
}
// 2^(byte - 127), for any stored byte (0 is 2^-127, a subnormal; 255 is NaN),
// and the inverse for a byte in [27, 247], as scale_byte gives it
__device__ __forceinline__ float scale_of(uint32_t byte) {
  return __uint_as_float(byte == 0 ? 0x400000u : byte == 255 ? 0x7FC00000u : byte << 23);
}
__device__ __forceinline__ float inv_scale(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

__device__ __forceinline__ bool finite_bits(uint32_t a) { return a < 0x7F800000u; }  // a: magnitude bits

// largest of the 16 lanes of a DPP row (magnitude bits order as integers)
__device__ __forceinline__ uint32_t row_max16(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, false));   // quad_perm [1,0,3,2]
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, false));   // quad_perm [2,3,0,1]
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xF, 0xF, false));  // row_half_mirror
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x140, 0xF, 0xF, false));  // row_mirror
  return v;
}

// ---- element types -------------------------------------------------------
__device__ __forceinline__ float half_bits_to_float(uint16_t h) { return (float)__builtin_bit_cast(_Float16, h); }
__device__ __forceinline__ uint16_t float_to_half_bits(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }

template <int DT> struct Elem;
template <> struct Elem<TT_F32> {
  static constexpr int SIZE = 4;
};
template <> struct Elem<TT_BF16> {
  static constexpr int SIZE = 2;
};
template <> struct Elem<TT_F16> {
  static constexpr int SIZE = 2;
};

// one value / N consecutive values.  Any address that the type's own
// alignment allows: gfx950 does unaligned vector accesses in hardware.
template <int DT>
__device__ __forceinline__ float ld1(const void* p, int64_t i) {
  if constexpr (DT == TT_F32) return reinterpret_cast<const float*>(p)[i];
  const uint16_t h = reinterpret_cast<const uint16_t*>(p)[i];
  return DT == TT_BF16 ? bf16_val(h) : half_bits_to_float(h);
}
template <int DT>
__device__ __forceinline__ void st1(void* p, int64_t i, float v) {
  if constexpr (DT == TT_F32)
    reinterpret_cast<float*>(p)[i] = v;
  else
    reinterpret_cast<uint16_t*>(p)[i] = DT == TT_BF16 ? bf16_bits(v) : float_to_half_bits(v);
}
template <int DT, int N>
__device__ __forceinline__ void ldv(const void* p, int64_t i, float (&x)[N]) {
  if constexpr (DT == TT_F32) {
    __builtin_memcpy(x, reinterpret_cast<const float*>(p) + i, 4 * N);
  } else {
    uint16_t h[N];
    __builtin_memcpy(h, reinterpret_cast<const uint16_t*>(p) + i, 2 * N);
#pragma unroll
    for (int k = 0; k < N; ++k) x[k] = DT == TT_BF16 ? bf16_val(h[k]) : half_bits_to_float(h[k]);
  }
}
template <int DT, int N>
__device__ __forceinline__ void stv(void* p, int64_t i, const float (&x)[N]) {
  if constexpr (DT == TT_F32) {
    __builtin_memcpy(reinterpret_cast<float*>(p) + i, x, 4 * N);
  } else {
    uint32_t h[N / 2];
#pragma unroll
    for (int k = 0; k < N / 2; ++k)
      h[k] = DT == TT_BF16 ? pk_bf16(x[2 * k], x[2 * k + 1])
                           : float_to_half_bits(x[2 * k]) | (uint32_t)float_to_half_bits(x[2 * k + 1]) << 16;
    __builtin_memcpy(reinterpret_cast<uint16_t*>(p) + i, h, 2 * N);
  }
}
// the first k (0..N) of N values; the rest read as zero, are not written
template <int DT, int N>
__device__ __forceinline__ void ldn(const void* p, int64_t i, int k, float (&x)[N]) {
  if (k >= N) {
    ldv<DT, N>(p, i, x);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = j < k ? ld1<DT>(p, i + j) : 0.f;
  }
}
template <int DT, int N>
__device__ __forceinline__ void stn(void* p, int64_t i, int k, const float (&x)[N]) {
  if (k >= N) {
    stv<DT, N>(p, i, x);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < k) st1<DT>(p, i + j, x[j]);
  }
}
template <int DT>
__device__ __forceinline__ void ld8n(const void* p, int64_t i, int k, float (&x)[8]) { ldn<DT, 8>(p, i, k, x); }
template <int DT>
__device__ __forceinline__ void st8n(void* p, int64_t i, int k, const float (&x)[8]) { stn<DT, 8>(p, i, k, x); }
template <int DT>
__device__ __forceinline__ void st8(void* p, int64_t i, const float (&x)[8]) { stv<DT, 8>(p, i, x); }

// ---- e4m3, rounded to nearest even (the catalogue) -------------------------
// 8 values under a scale byte -> 8 code bytes; infinities become NaN: e4m3 has none.
// Under the largest scale the code after 240 stands for 2^128, which no float
// holds: what would round to it stays at 240 (off by 2^-4 of the value at most).
constexpr uint32_t TOP_BYTE = 247u;
__device__ __forceinline__ u32x2 encode8_scaled(const float (&x)[8], uint32_t byte) {
  const float inv = inv_scale(byte), most = byte == TOP_BYTE ? 240.f : 448.f;
  float y[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const uint32_t a = __float_as_uint(x[k]) & 0x7FFFFFFFu;
    y[k] = finite_bits(a) ? __builtin_amdgcn_fmed3f(x[k] * inv, -most, most) : __uint_as_float(0x7FC00000u);
  }
  int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true);
  int hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], 0, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], hi, true);
  return (u32x2){(uint32_t)lo, (uint32_t)hi};
}
// 8 values of a block spread over 16 lanes -> 8 code bytes; every lane of the
// row gets the block's scale byte
__device__ __forceinline__ u32x2 encode8(const float (&x)[8], uint32_t& byte) {
  uint32_t amax = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const uint32_t a = __float_as_uint(x[k]) & 0x7FFFFFFFu;
    amax = max(amax, finite_bits(a) ? a : 0u);
  }
  byte = (uint32_t)scale_byte(row_max16(amax), CARRY_M);
  return encode8_scaled(x, byte);
}
__device__ __forceinline__ void decode4(uint32_t w, float s, float* x) {
  const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  const auto b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  x[0] = a[0] * s;
  x[1] = a[1] * s;
  x[2] = b[0] * s;
  x[3] = b[1] * s;
}
__device__ __forceinline__ void decode8(u32x2 c, float s, float (&x)[8]) {
  decode4(c[0], s, x);
  decode4(c[1], s, x + 4);
}

// ---- magnitudes rounded up or down by 16 random bits (the states) ----------
// The code of x >= 0 under a scale 2^(byte - 127) is x's own float bits after
// x * 2^(127 - byte - 120) has moved the code's exponent bias (7) to the
// float's: normal and subnormal codes alike are then the top bits, what is cut
// off is the rest, and adding random bits below the cut rounds up with the
// probability of what is cut.
template <int MANT>
__device__ __forceinline__ uint32_t round_code(float x, uint32_t byte, uint32_t rnd16) {
  constexpr int SH = 23 - MANT;
  return (__float_as_uint(__builtin_amdgcn_ldexpf(x, 7 - (int)byte)) + (rnd16 << (SH - 16))) >> SH;
}
template <int MANT>
__device__ __forceinline__ float code_value(uint32_t mag, uint32_t byte) {
  return __builtin_amdgcn_ldexpf(__uint_as_float(mag << (23 - MANT)), (int)byte - 7);
}

}  // namespace b8
}  // namespace tt
