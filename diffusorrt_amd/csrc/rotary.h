// Rotary positions: the angle of a pair at a position, its cosine and sine.
//
// A pair's frequency is kept in turns a position as a 64-bit fraction F = 2^64 f / 2 pi, so position
// p's angle is the upper half of the low 64 bits of p F: whole turns fall off in the multiplication, and
// the angle is right to 2^-32 of a turn and p 2^-64 of one at any 32-bit position (a product of p and f
// in fp32 is off by whole radians from p = 2^24 on). Three integer instructions; no table is read.
#pragma once
#include "common.h"

// The fraction of a turn, in 2^-32.
DRT_DEV uint32_t rotary_turn(uint64_t freq, int32_t p) {
  const uint32_t lo = (uint32_t)freq, hi = (uint32_t)(freq >> 32), u = (uint32_t)p;
  // (a negative p is u - 2^32: 2^32 F takes lo from the upper half)
  return hi * u + __umulhi(lo, u) - (p < 0 ? lo : 0u);
}

// Cosine and sine of a fraction of a turn: the nearest quarter taken off, the rest (within pi / 4) by the
// Taylor series to x^9 and x^10, whose next terms are below 2^-29. Off by 2^-23 at most.
DRT_DEV float2 rotary_cos_sin(uint32_t turn) {
  const uint32_t quarter = (turn + 0x20000000u) >> 30;
  const float x = (float)(int32_t)(turn - (quarter << 30)) * 1.4629180792671596e-9f;  // 2 pi / 2^32
  const float y = x * x;
  float s = fmaf(y, 1.f / 362880.f, -1.f / 5040.f);
  s = fmaf(y, s, 1.f / 120.f);
  s = fmaf(y, s, -1.f / 6.f);
  s = fmaf(x * y, s, x);
  float c = fmaf(y, -1.f / 3628800.f, 1.f / 40320.f);
  c = fmaf(y, c, -1.f / 720.f);
  c = fmaf(y, c, 1.f / 24.f);
  c = fmaf(y, c, -0.5f);
  c = fmaf(y, c, 1.f);
  const float a = quarter & 1 ? s : c, b = quarter & 1 ? c : s;
  return make_float2((quarter + 1) & 2 ? -a : a, quarter & 2 ? -b : b);
}

// Eight elements in a row of type DT (0 fp32, 1 fp16, 2 bf16), as fp32; aligned to their type only.
template <int DT> DRT_DEV void rotary_load8(const void* p, float (&x)[8]) {
  if constexpr (DT == 0) {
    const f32x4 a = *(const f32x4_e*)p, b = *(const f32x4_e*)((const float*)p + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = a[e];
      x[4 + e] = b[e];
    }
  } else {
    const u32x4 w = *(const u32x4_e*)p;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t y = w[e];
      if constexpr (DT == 1) {
        const f16x2 h = __builtin_bit_cast(f16x2, y);
        x[2 * e] = (float)h[0];
        x[2 * e + 1] = (float)h[1];
      } else {
        x[2 * e] = bf16_bits_to_float(y & 0xffffu);
        x[2 * e + 1] = __uint_as_float(y & 0xffff0000u);
      }
    }
  }
}
// Eight values as 16-bit elements.
template <int DT> DRT_DEV u32x4 rotary_pack8(const float (&x)[8]) {
  u32x4 w;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (DT == 1)
      w[e] = pack_half2((_Float16)x[2 * e], (_Float16)x[2 * e + 1]);
    else
      w[e] = (uint32_t)float_to_bf16_bits(x[2 * e]) | ((uint32_t)float_to_bf16_bits(x[2 * e + 1]) << 16);
  }
  return w;
}
template <int DT> DRT_DEV void rotary_store8(void* p, const float (&x)[8]) {
  if constexpr (DT == 0) {
    *(f32x4_e*)p = f32x4{x[0], x[1], x[2], x[3]};
    *(f32x4_e*)((float*)p + 4) = f32x4{x[4], x[5], x[6], x[7]};
  } else {
    *(u32x4_e*)p = rotary_pack8<DT>(x);
  }
}
// Two neighbours, aligned to their type only.
template <int DT> DRT_DEV void rotary_load2(const void* p, int64_t i, float& a, float& b) {
  typedef float f32x2_e __attribute__((ext_vector_type(2), aligned(4)));
  typedef uint16_t u16x2_e __attribute__((ext_vector_type(2), aligned(2)));
  if constexpr (DT == 0) {
    const f32x2_e w = *(const f32x2_e*)((const float*)p + i);
    a = w[0];
    b = w[1];
  } else {
    const u16x2_e w = *(const u16x2_e*)((const uint16_t*)p + i);
    if constexpr (DT == 1) {
      a = (float)__builtin_bit_cast(_Float16, (uint16_t)w[0]);
      b = (float)__builtin_bit_cast(_Float16, (uint16_t)w[1]);
    } else {
      a = bf16_bits_to_float(w[0]);
      b = bf16_bits_to_float(w[1]);
    }
  }
}
template <int DT> DRT_DEV float rotary_load1(const void* p, int64_t i) {
  if constexpr (DT == 0) return ((const float*)p)[i];
  else if constexpr (DT == 1) return (float)((const _Float16*)p)[i];
  else return bf16_bits_to_float(((const uint16_t*)p)[i]);
}
template <int DT> DRT_DEV void rotary_store1(void* p, int64_t i, float x) {
  if constexpr (DT == 0) ((float*)p)[i] = x;
  else if constexpr (DT == 1) ((_Float16*)p)[i] = (_Float16)x;
  else ((uint16_t*)p)[i] = float_to_bf16_bits(x);
}

// a + i b turned: c, s with the magnitude in them. (A turn of zero by magnitude one gives a and b back.)
DRT_DEV void rotary_turn_pair(float& a, float& b, float c, float s) {
  const float y = a * c - b * s;
  b = b * c + a * s;
  a = y;
}
