// The 8-bit K/V cache: its tile layout and how its codes become MFMA operands.
//
// A tile is 32 keys of one K/V head, 8 KiB: K (4096 bytes), then V. A byte is a code + 128,
// code in [-127, 127]; a value is code * scale, one power of two for the tile's K and one
// for its V (scales[head][tile] = {K, V}). A tile whose K or V does not all fit is NaN as a whole: its
// scale is NaN, its codes are 0.
//
// Bytes (key kk, head dim hd):
//   K: ((p*2 + h)*32 + kk)*16 + s*8 + e    p = hd/32, s = (hd/16)&1, h = (hd/8)&1, e = hd&7
//   V: 4096 + ((hb*2 + h)*32 + hl)*16 + kh*8 + j
//        hb = hd/32, hl = hd&31, kh = kk/16, h = (kk>>2)&1, j = (kk&3) + 4*((kk>>3)&1)
// so 16 bytes are two of the eight-element operands of a 32x32x16 product (head dim steps
// 2p and 2p + 1 of K, key steps 0 and 1 of V), and every load of a wave is 1 KiB in a row.
#pragma once
#include "common.h"
#include "launch.h"

constexpr int KV8_TILE = 8192;
constexpr int KV8_MIN_EXP = -40, KV8_MAX_EXP = 40;

DRT_DEV int kv8_k_at(int kk, int hd) {
  return (((hd >> 5) * 2 + ((hd >> 3) & 1)) * 32 + kk) * 16 + ((hd >> 4) & 1) * 8 + (hd & 7);
}
DRT_DEV int kv8_v_at(int kk, int hd) {
  return 4096 + (((hd >> 5) * 2 + ((kk >> 2) & 1)) * 32 + (hd & 31)) * 16 + (kk >> 4) * 8 +
         (kk & 3) + 4 * ((kk >> 3) & 1);
}

// Eight bytes as fp16 operands in one instruction a pair: a byte b alone is the subnormal fp16
// b * 2^-24, which the matrix instructions (and v_dot2_f32_f16) multiply exactly. With a code
// c = b - 128, a product with x is 2^-24 (sum x c + 128 sum x): the 2^24 goes where a scale is applied
// anyway, and 128 times the sum of x is taken off in fp32 (x the query: once per query vector; x the
// weights: one running sum). The exact fp16 c (1024 + b, less 1152) takes twice the instructions.
DRT_DEV f16x8 kv8_to_f16(uint32_t lo, uint32_t hi) {
  const u32x4 r = {
      __builtin_amdgcn_perm(lo, lo, 0x0c050c04u), __builtin_amdgcn_perm(lo, lo, 0x0c070c06u),
      __builtin_amdgcn_perm(hi, hi, 0x0c050c04u), __builtin_amdgcn_perm(hi, hi, 0x0c070c06u)};
  return __builtin_bit_cast(f16x8, r);
}
constexpr float KV8_POW = 16777216.f;  // 2^24
constexpr float KV8_BIAS = 128.f;
// c + the sum of eight fp16 values, in fp32.
DRT_DEV float kv8_add8(const f16x8 p, float c) {
  const f16x2 one = {(_Float16)1.f, (_Float16)1.f};
  const u32x4 w = __builtin_bit_cast(u32x4, p);
  const uint32_t w0 = w[0], w1 = w[1], w2 = w[2], w3 = w[3];
  c = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w0), one, c, false);
  c = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w1), one, c, false);
  c = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w2), one, c, false);
  return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w3), one, c, false);
}

// The number of keys a row sees, always the first ones (no more than n_keys).
DRT_DEV int key_end_of(int row, const drt::AttnWhere& w) {
  if (!w.masked) return w.n_keys;
  const int p = w.row_pos0 + row;
  if (p < w.prompt_len) return min(w.n_keys, w.prompt_len);
  const uint32_t mine = (uint32_t)(p - w.prompt_len) / (uint32_t)w.block;
  const int64_t end = w.prompt_len + ((int64_t)mine + 1) * w.block;
  return (int)min((int64_t)w.n_keys, end);
}
