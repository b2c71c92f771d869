// What the attentions over a cache's tiles share (cache_attention.hip, paged_attention.hip): element
// types, the softmax base's bounds, values that are not finite beside rows that do not see them.
#pragma once
#include "kv8.h"

#include <cmath>

constexpr float CA_RESCALE_LOG2 = 8.f;
// A base beyond this is rounded by more than 2^-4: p' = 2^(fma(s, a, off - base)) would then be off by
// that, without bound; with the exponent rounded before the base is taken off it never passes 2^8.
constexpr float CA_LARGE = 1048576.f;

DRT_DEV float ca_max_xor32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// A barrier for LDS: __syncthreads() would wait for the loads on their way too.
DRT_DEV void ca_lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// What a cache's element type means to the kernel: 0 = 8-bit, 1 = fp16, 2 = bf16.
template <int DT> struct CacheT {
  static constexpr int TILE = DT == 0 ? KV8_TILE : 2 * KV8_TILE, LOADS = DT == 0 ? 4 : 8;
  typedef f16x8 vec;
  static DRT_DEV f32x16 mma(vec a, vec b, f32x16 c) { return mfma_f16(a, b, c); }
  static DRT_DEV _Float16 weight(float p) { return (_Float16)p; }
};
template <> struct CacheT<2> {
  static constexpr int TILE = 2 * KV8_TILE, LOADS = 8;
  typedef bf16x8 vec;
  static DRT_DEV f32x16 mma(vec a, vec b, f32x16 c) { return mfma_bf16(a, b, c); }
  // (bf16 as the values are, and as the attention over all of a bf16 cache has them: the product has one
  // type. Results are off by 1.9 to 2.2 * 10^-3 in all where fp16 weights leave 1.7, a bf16 result's own.)
  static DRT_DEV __bf16 weight(float p) { return (__bf16)p; }
};
// Operand i of the eight of a tile's K or V from its registers.
template <int DT, int N> DRT_DEV typename CacheT<DT>::vec ca_operand(const u32x4 (&r)[N], int i) {
  if constexpr (DT == 0)
    return kv8_to_f16(r[i >> 1][2 * (i & 1)], r[i >> 1][2 * (i & 1) + 1]);
  else
    return __builtin_bit_cast(typename CacheT<DT>::vec, r[i]);
}

// The values (16 bits) of a tile's 32 head dims in a lane's two operands that are not finite, taken out of
// them: in their place every query column that sees one's key gets infinity or NaN in that head dim, as
// p * V would be, and the others nothing, where 0 * V would be NaN. An indicator product for each of the
// three. QT query tiles; o[j] is their O of these head dims, end[j] the keys their columns see.
template <int DT, int QT>
DRT_DEV void ca_values_apart(u32x4 (&vr)[2], int key0, const int (&end)[QT], int lane,
                             f32x16* const (&o)[QT]) {
  typedef CacheT<DT> T;
  typedef typename T::vec vec;
  constexpr uint32_t EXP = DT == 1 ? 0x7c00u : 0x7f80u, ONE = DT == 1 ? 0x3c00u : 0x3f80u;
#pragma unroll 1
  for (int kind = 0; kind < 3; ++kind) {  // NaN, +infinity, -infinity
    const float put = kind == 0 ? NAN : kind == 1 ? INFINITY : -INFINITY;
    vec marks[2];
#pragma unroll
    for (int kh = 0; kh < 2; ++kh) {
      u32x4 w = vr[kh];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t y = w[e];
        uint32_t mark = 0u;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t z = (y >> (16 * h)) & 0xffffu;
          const bool hit = kind == 0   ? (z & 0x7fffu) > EXP
                           : kind == 1 ? z == EXP
                                       : z == (EXP | 0x8000u);
          mark |= hit ? ONE << (16 * h) : 0u;
        }
        w[e] = mark;
      }
      marks[kh] = __builtin_bit_cast(vec, w);
    }
#pragma unroll
    for (int j = 0; j < QT; ++j) {
      f32x16 n = f32x16{};
#pragma unroll
      for (int kh = 0; kh < 2; ++kh) {
        vec sees;  // 1 for the keys of this lane's that its column sees
#pragma unroll
        for (int e = 0; e < 8; ++e)
          sees[e] = T::weight(key0 + mfma_row(kh * 8 + e, lane) < end[j] ? 1.f : 0.f);
        n = T::mma(marks[kh], sees, n);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) (*o[j])[r] = n[r] > 0.f ? (*o[j])[r] + put : (*o[j])[r];
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t y = vr[i][e];
      const uint32_t keep = ((y & EXP) == EXP ? 0u : 0xffffu) |
                            ((y & (EXP << 16)) == EXP << 16 ? 0u : 0xffff0000u);
      vr[i][e] = y & keep;
    }
}
