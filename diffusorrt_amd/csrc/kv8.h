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

// Eight codes as exact fp16 values: a byte b under the exponent of 1024 is the fp16 1024 + b,
// and one packed subtraction of 1152 leaves b - 128.
DRT_DEV uint32_t kv8_pair_to_f16(uint32_t codes, uint32_t which) {
  const f16x2 bias = {(_Float16)-1152.f, (_Float16)-1152.f};
  const uint32_t w = __builtin_amdgcn_perm(codes, 0x64646464u, which);
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, w) + bias);
}
DRT_DEV f16x8 kv8_to_f16(uint32_t lo, uint32_t hi) {
  const u32x4 r = {kv8_pair_to_f16(lo, 0x00050004u), kv8_pair_to_f16(lo, 0x00070006u),
                   kv8_pair_to_f16(hi, 0x00050004u), kv8_pair_to_f16(hi, 0x00070006u)};
  return __builtin_bit_cast(f16x8, r);
}

// The number of keys a row sees, always the first ones (no more than n_keys).
DRT_DEV int key_end_of(int row, const drt::AttnWhere& w) {
  if (!w.masked) return w.n_keys;
  const int p = w.row_pos0 + row;
  if (p < w.prompt_len) return min(w.n_keys, w.prompt_len);
  const int64_t end = w.prompt_len + ((int64_t)(p - w.prompt_len) / w.block + 1) * w.block;
  return (int)min((int64_t)w.n_keys, end);
}
