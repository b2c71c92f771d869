// Rows into and out of the prefix cache where the cache is more than a copy of them: the
// 8-bit store, the reading back of rows, and the sums of a tile's keys.
#include "kv8.h"
#include "launch.h"

namespace {

// One 256-thread work-group per (tile, K/V head); thread t holds 16 head dims of key t / 8, of K
// and of V: the new rows from their source, the tile's other rows as they read. The largest
// magnitudes choose the powers of two (a comparison of bits, in which NaN and infinities are
// the largest), every value is rounded once (x / scale is exact), and the codes meet in LDS, from
// where the tile leaves in 16-byte pieces.
//   e = the least integer >= -40 with max <= 127 * 2^e;  code = rint(x * 2^-e)
// A power of two, not max / 127: a tile that is stored to again is quantized anew from
// what it reads as, which with these scales is one more rounding only when e rises, each time to
// half the resolution or less, so any number of stores stays within one step of what they wrote
// (1/2 + 1/4 + ...); and x / scale never falls on the wrong side of a rounding.
// Bound: the rows read and the codes written (131072 bf16 rows x 8 heads: 805 MB in 154 us, 5.2 TB/s,
// 168 with sums; 2000 fp32 rows x 4 heads 5.8 us); of a block of 32 rows, 4.2 us, the chain of a
// launch, the loads, two barriers and the stores. A work-group has a tile alone: its scale
// needs every row of it, and no other work-group's. Codes cross LDS as words: byte by byte, and
// with every head dim's sum exchanged by itself, 222 us with sums, and 5.7 for the block.
// Where byte `at` of the tile is in LDS: 16-byte pieces change places within 256 bytes, so that
// the threads' words, 256 and 1024 bytes apart, meet more banks.
DRT_DEV int kv8_lds(int at) { return at ^ (((at >> 8) & 3) << 4) ^ (((at >> 10) & 3) << 6); }

template <bool SRC_BF16>
__global__ __launch_bounds__(256) void kv8_store_kernel(
    const void* __restrict__ k_src, const void* __restrict__ v_src, int n, int Hkv, int pos0,
    uint8_t* __restrict__ kv, int64_t kv_head_stride, float* __restrict__ scales,
    float* __restrict__ sums) {
  const int t = (pos0 >> 5) + blockIdx.x, h = blockIdx.y;
  const int64_t tiles = kv_head_stride / KV8_TILE;
  const int64_t row_t = (int64_t)32 * t - pos0;  // source row of the tile's key 0 (may be negative)
  uint8_t* tile = kv + h * kv_head_stride + (int64_t)t * KV8_TILE;
  float* sc = scales + (h * tiles + t) * 2;
  __shared__ __align__(16) uint8_t codes[KV8_TILE];
  __shared__ uint32_t most[2][4];
  __shared__ int part[4][128];
  const int tid = threadIdx.x, kk = tid >> 3, d0 = (tid & 7) * 16;
  const int64_t src_row = row_t + kk;
  const bool fresh = src_row >= 0 && src_row < n;
  float x[2][16];
  if (fresh) {
    const int64_t at = (src_row * Hkv + h) * 128 + d0;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const void* s = w ? v_src : k_src;
      if (SRC_BF16) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const u32x4 r = *(const u32x4_e*)((const uint16_t*)s + at + 8 * c);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[w][8 * c + 2 * e] = bf16_bits_to_float(r[e] & 0xffffu);
            x[w][8 * c + 2 * e + 1] = bf16_bits_to_float(r[e] >> 16);
          }
        }
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const f32x4 r = *(const f32x4_e*)((const float*)s + at + 4 * c);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[w][4 * c + e] = r[e];
        }
      }
    }
  } else {  // a row that stays
    const float sk = sc[0], sv = sc[1];
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // eight head dims of K are eight bytes in a row
      const uint2 w = *(const uint2*)(tile + kv8_k_at(kk, d0 + 8 * h));
#pragma unroll
      for (int e = 0; e < 8; ++e)
        x[0][8 * h + e] = sk * (float)((int)(((e < 4 ? w.x : w.y) >> (8 * (e & 3))) & 0xffu) - 128);
    }
#pragma unroll
    for (int e = 0; e < 16; ++e)
      x[1][e] = sv * (float)((int)tile[kv8_v_at(kk, d0 + e)] - 128);
  }
  uint32_t m[2] = {0u, 0u};
#pragma unroll
  for (int w = 0; w < 2; ++w) {
#pragma unroll
    for (int e = 0; e < 16; ++e) m[w] = max(m[w], __float_as_uint(x[w][e]) & 0x7fffffffu);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m[w] = max(m[w], (uint32_t)__shfl_xor((int)m[w], o, 64));
    if ((tid & 63) == 0) most[w][tid >> 6] = m[w];
  }
  __syncthreads();  // (also: every row that stays has been read)
  float scale[2];
  uint32_t y[2][4];  // the thread's codes + 128, as bytes
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const uint32_t b = max(max(most[w][0], most[w][1]), max(most[w][2], most[w][3]));
    // 127 = 1.984375 * 2^6
    const int e = max(KV8_MIN_EXP, (int)(b >> 23) - 133 + ((b & 0x7fffffu) > 0x7e0000u ? 1 : 0));
    const bool fits = e <= KV8_MAX_EXP;
    const float inv = __uint_as_float((uint32_t)(127 - min(e, KV8_MAX_EXP)) << 23);
    scale[w] = fits ? __uint_as_float((uint32_t)(127 + e) << 23) : __uint_as_float(0x7fc00000u);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint32_t z = 0u;
#pragma unroll
      for (int i = 0; i < 4; ++i)  // (a whole number before its conversion)
        z = __builtin_amdgcn_cvt_pk_u8_f32(rintf(x[w][4 * q + i] * inv) + 128.f, i, z);
      y[w][q] = fits ? z : 0x80808080u;
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h)
    *(uint2*)(codes + kv8_lds(kv8_k_at(kk, d0 + 8 * h))) = make_uint2(y[0][2 * h], y[0][2 * h + 1]);
  // V has four keys in a row: the threads of four neighbouring ones (lanes 8 and 16 apart) exchange
  // their words, until thread kk & 3 = r has head dims 4 r .. + 4 of all four, and turn the bytes.
  const int b0 = tid & 8, b1 = tid & 16, r = (tid >> 3) & 3;
  {
    const uint32_t s0 = (uint32_t)__shfl_xor((int)(b0 ? y[1][0] : y[1][1]), 8, 64);
    const uint32_t s1 = (uint32_t)__shfl_xor((int)(b0 ? y[1][2] : y[1][3]), 8, 64);
    const uint32_t u0 = b0 ? s0 : y[1][0], u1 = b0 ? y[1][1] : s0;  // dims 4 (r & 1) of keys 0, 1
    const uint32_t v0 = b0 ? s1 : y[1][2], v1 = b0 ? y[1][3] : s1;  // dims 8 + 4 (r & 1)
    const uint32_t t0 = (uint32_t)__shfl_xor((int)(b1 ? u0 : v0), 16, 64);
    const uint32_t t1 = (uint32_t)__shfl_xor((int)(b1 ? u1 : v1), 16, 64);
    const uint32_t k0 = b1 ? t0 : u0, k1 = b1 ? t1 : u1, k2 = b1 ? v0 : t0, k3 = b1 ? v1 : t1;
    const uint32_t lo01 = __builtin_amdgcn_perm(k1, k0, 0x05010400u);  // dims 0, 1 of keys 0, 1
    const uint32_t hi01 = __builtin_amdgcn_perm(k1, k0, 0x07030602u);  // dims 2, 3
    const uint32_t lo23 = __builtin_amdgcn_perm(k3, k2, 0x05010400u);
    const uint32_t hi23 = __builtin_amdgcn_perm(k3, k2, 0x07030602u);
    const uint32_t z[4] = {__builtin_amdgcn_perm(lo23, lo01, 0x05040100u),
                           __builtin_amdgcn_perm(lo23, lo01, 0x07060302u),
                           __builtin_amdgcn_perm(hi23, hi01, 0x05040100u),
                           __builtin_amdgcn_perm(hi23, hi01, 0x07060302u)};
#pragma unroll
    for (int c = 0; c < 4; ++c)
      *(uint32_t*)(codes + kv8_lds(kv8_v_at(kk & ~3, d0 + 4 * r + c))) = z[c];
  }
  if (sums) {  // whole numbers: exact in any order
    // two head dims a word (4 q + o and 4 q + o + 2 in word 2 q + o), the eight keys of the wave added
    // up; each exchange leaves a lane half of the words
    uint32_t a[8];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      a[2 * q] = y[0][q] & 0x00ff00ffu;
      a[2 * q + 1] = (y[0][q] >> 8) & 0x00ff00ffu;
    }
#pragma unroll
    for (int n = 4; n > 0; n >>= 1) {
      const int bit = 32 / n;  // lanes 8, 16, 32 apart
      const bool up = tid & bit;
#pragma unroll
      for (int i = 0; i < n; ++i) {
        const uint32_t give = up ? a[i] : a[i + n], keep = up ? a[i + n] : a[i];
        a[i] = keep + (uint32_t)__shfl_xor((int)give, bit, 64);
      }
    }
    const int i = (tid & 8 ? 4 : 0) + (tid & 16 ? 2 : 0) + (tid & 32 ? 1 : 0);
    int* to = part[tid >> 6] + d0 + 4 * (i >> 1) + (i & 1);
    to[0] = (int)(a[0] & 0xffffu) - 8 * 128;
    to[2] = (int)(a[0] >> 16) - 8 * 128;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i)
    *(u32x4*)(tile + (tid + 256 * i) * 16) = *(const u32x4*)(codes + kv8_lds((tid + 256 * i) * 16));
  if (tid < 2) sc[tid] = tid ? scale[1] : scale[0];
  if (sums && tid < 128)
    sums[(h * tiles + t) * 128 + tid] =
        scale[0] * (float)(part[0][tid] + part[1][tid] + part[2][tid] + part[3][tid]);
}

// Rows [pos0, pos0 + n) of a cache back as [n][Hkv][128] values. One 256-thread work-group
// per (tile, head), which reads the tile whole: 16-byte pieces by way of LDS, whose few rows of a
// ragged end cost no launch of their own. Bound as the store is: 32 rows x 8 heads 3.1 us, a launch;
// 2000 x 4 heads to fp32 4.3 us, 10.2 MB.
// DT: 0 = 8-bit, 1 = fp16, 2 = bf16.
DRT_DEV int kv16_k_at(int kk, int hd) { return ((hd >> 3) * 32 + kk) * 8 + (hd & 7); }
DRT_DEV int kv16_v_at(int kk, int hd) {
  return 4096 + ((((hd >> 5) * 2 + (kk >> 4)) * 2 + ((kk >> 2) & 1)) * 32 + (hd & 31)) * 8 +
         (kk & 3) + 4 * ((kk >> 3) & 1);
}
template <int DT> DRT_DEV float kv_value(const void* tile, int at, float scale) {
  if (DT == 0) return scale * (float)((int)((const uint8_t*)tile)[at] - 128);
  if (DT == 1) return (float)((const _Float16*)tile)[at];
  return bf16_bits_to_float(((const uint16_t*)tile)[at]);
}

template <int DT, bool OUT_BF16>
__global__ __launch_bounds__(256) void kv_load_kernel(const uint8_t* __restrict__ kv,
                                                      int64_t head_stride_bytes,
                                                      const float* __restrict__ scales, int n,
                                                      int Hkv, int pos0, void* __restrict__ k_out,
                                                      void* __restrict__ v_out) {
  constexpr int TILE = DT == 0 ? KV8_TILE : 2 * KV8_TILE;
  const int t = (pos0 >> 5) + blockIdx.x, h = blockIdx.y;
  const int64_t tiles = head_stride_bytes / TILE;
  __shared__ __align__(16) uint8_t tile[TILE];
  const int tid = threadIdx.x;
  const uint8_t* src = kv + h * head_stride_bytes + (int64_t)t * TILE;
#pragma unroll
  for (int i = 0; i < TILE / 4096; ++i)
    *(u32x4*)(tile + (tid + 256 * i) * 16) = *(const u32x4*)(src + (tid + 256 * i) * 16);
  const float sk = DT == 0 ? scales[(h * tiles + t) * 2] : 1.f;
  const float sv = DT == 0 ? scales[(h * tiles + t) * 2 + 1] : 1.f;
  __syncthreads();
  for (int it = tid; it < 32 * 32; it += 256) {  // four head dims of a key
    const int kk = it >> 5, d = (it & 31) * 4;
    const int64_t row = (int64_t)32 * t - pos0 + kk;
    if (row < 0 || row >= n) continue;
    const int64_t at = (row * Hkv + h) * 128 + d;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        x[e] = kv_value<DT>(tile,
                            DT == 0 ? (w ? kv8_v_at(kk, d + e) : kv8_k_at(kk, d + e))
                                    : (w ? kv16_v_at(kk, d + e) : kv16_k_at(kk, d + e)),
                            w ? sv : sk);
      void* out = w ? v_out : k_out;
      if (OUT_BF16) {
        uint32_t p[2];
#pragma unroll
        for (int e = 0; e < 2; ++e)
          p[e] = (uint32_t)float_to_bf16_bits(x[2 * e]) |
                 ((uint32_t)float_to_bf16_bits(x[2 * e + 1]) << 16);
        *(uint2*)((uint16_t*)out + at) = make_uint2(p[0], p[1]);
      } else {
        *(f32x4*)((float*)out + at) = f32x4{x[0], x[1], x[2], x[3]};
      }
    }
  }
}

// Rows into a 16-bit cache, as kv_pack_kernel (attention.hip) writes them, and the touched tiles'
// keys added up, the rows that stay among them, in 64 bits and rounded once. One 256-thread
// work-group per (tile, head): thread (kk, c) has head dims 8 c .. + 8 of keys kk and kk + 16; of V
// the eight keys that share 16 bytes. One launch for both: 9 rows x 4 heads 4.3 us, all latency (a
// sum kernel behind the store 3.4 + 1.7, and the gap between them).
template <typename T> DRT_DEV T kv16_of(float f);
template <> DRT_DEV _Float16 kv16_of<_Float16>(float f) { return (_Float16)f; }
template <> DRT_DEV __bf16 kv16_of<__bf16>(float f) { return (__bf16)f; }

template <typename T, bool SRC_BF16>
__global__ __launch_bounds__(256) void kv16_store_kernel(const void* __restrict__ k_src,
                                                         const void* __restrict__ v_src, int n,
                                                         int Hkv, int pos0, T* __restrict__ kv,
                                                         int64_t kv_head_stride,
                                                         float* __restrict__ sums) {
  const int t = (pos0 >> 5) + blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
  const int64_t row_t = (int64_t)32 * t - pos0;  // source row of the tile's key 0 (may be negative)
  T* tile = kv + h * kv_head_stride + (int64_t)t * KV8_TILE;
  const int64_t stride = (int64_t)Hkv * 128;
  __shared__ double part[4][128];
  auto valid = [&](int kk) { return row_t + kk >= 0 && row_t + kk < n; };
  auto at = [&](int kk) { return (row_t + kk) * stride + h * 128; };
  double sum[8] = {};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int kk = (tid >> 4) + 16 * i, c = tid & 15;
    T o[8];
    if (valid(kk)) {
      if (SRC_BF16) {
        const u32x4 w = *(const u32x4_e*)((const uint16_t*)k_src + at(kk) + 8 * c);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          o[2 * e] = kv16_of<T>(bf16_bits_to_float(w[e] & 0xffffu));
          o[2 * e + 1] = kv16_of<T>(bf16_bits_to_float(w[e] >> 16));
        }
      } else {
        const float* p = (const float*)k_src + at(kk) + 8 * c;
        const f32x4 a = *(const f32x4_e*)p, b = *(const f32x4_e*)(p + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          o[e] = kv16_of<T>(a[e]);
          o[4 + e] = kv16_of<T>(b[e]);
        }
      }
      *(u32x4*)(tile + (c * 32 + kk) * 8) = __builtin_bit_cast(u32x4, o);
    } else {
      __builtin_memcpy(o, tile + (c * 32 + kk) * 8, 16);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[e] += (double)(float)o[e];
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {  // the four keys of this wave's lanes
    sum[e] += __shfl_xor(sum[e], 16, 64);
    sum[e] += __shfl_xor(sum[e], 32, 64);
    if ((tid & 63) < 16) part[tid >> 6][8 * (tid & 15) + e] = sum[e];
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int it = tid + 256 * i, hd = it & 127, kh = it >> 8, hh = (it >> 7) & 1;
    T o[8];
    bool all = true;
#pragma unroll
    for (int j = 0; j < 8; ++j) {  // slot j holds key 16 kh + 4 hh + (j & 3) + 8 (j >> 2)
      const int kk = 16 * kh + 4 * hh + (j & 3) + 8 * (j >> 2);
      all = all && valid(kk);
      const int64_t s = at(valid(kk) ? kk : (int)-row_t) + hd;  // (source row 0: never stored)
      o[j] = kv16_of<T>(SRC_BF16 ? bf16_bits_to_float(((const uint16_t*)v_src)[s])
                                 : ((const float*)v_src)[s]);
    }
    T* dst = tile + 4096 + ((((hd >> 5) * 2 + kh) * 2 + hh) * 32 + (hd & 31)) * 8;
    if (all) {
      *(u32x4*)dst = __builtin_bit_cast(u32x4, o);
    } else {  // the tile's other keys stay as they are
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (valid(16 * kh + 4 * hh + (j & 3) + 8 * (j >> 2))) dst[j] = o[j];
    }
  }
  __syncthreads();
  if (tid < 128)
    sums[(h * (kv_head_stride / KV8_TILE) + t) * 128 + tid] =
        (float)((part[0][tid] + part[1][tid]) + (part[2][tid] + part[3][tid]));
}

unsigned tiles_of(int pos0, int n) { return (unsigned)(((int64_t)pos0 + n - 1) / 32 - pos0 / 32 + 1); }

}  // namespace

namespace drt {

void kv8_store(const void* k, const void* v, bool src_bf16, int n, int Hkv, int pos0, void* kv,
               int64_t head_stride, float* scales, float* sums, hipStream_t s) {
  const dim3 grid(tiles_of(pos0, n), (unsigned)Hkv);
  if (src_bf16)
    hipLaunchKernelGGL(kv8_store_kernel<true>, grid, dim3(256), 0, s, k, v, n, Hkv, pos0,
                       (uint8_t*)kv, head_stride, scales, sums);
  else
    hipLaunchKernelGGL(kv8_store_kernel<false>, grid, dim3(256), 0, s, k, v, n, Hkv, pos0,
                       (uint8_t*)kv, head_stride, scales, sums);
  DRT_HIP(hipGetLastError());
}

void kv_load(KvType type, const void* kv, int64_t head_stride, const float* scales, int n, int Hkv,
             int pos0, void* k, void* v, bool out_bf16, hipStream_t s) {
  const dim3 grid(tiles_of(pos0, n), (unsigned)Hkv);
  const int64_t bytes = type == KvType::I8 ? head_stride : 2 * head_stride;
#define DRT_KVL(DT, B)                                                                       \
  hipLaunchKernelGGL((kv_load_kernel<DT, B>), grid, dim3(256), 0, s, (const uint8_t*)kv,     \
                     bytes, scales, n, Hkv, pos0, k, v)
#define DRT_KVL2(DT) do { if (out_bf16) DRT_KVL(DT, true); else DRT_KVL(DT, false); } while (0)
  if (type == KvType::I8) DRT_KVL2(0);
  else if (type == KvType::F16) DRT_KVL2(1);
  else DRT_KVL2(2);
#undef DRT_KVL2
#undef DRT_KVL
  DRT_HIP(hipGetLastError());
}

void kv16_store(bool kv_bf16, const void* k, const void* v, bool src_bf16, int n, int Hkv, int pos0,
                void* kv, int64_t head_stride, float* sums, hipStream_t s) {
  const dim3 grid(tiles_of(pos0, n), (unsigned)Hkv);
#define DRT_KV16(T, B)                                                                        \
  hipLaunchKernelGGL((kv16_store_kernel<T, B>), grid, dim3(256), 0, s, k, v, n, Hkv, pos0,    \
                     (T*)kv, head_stride, sums)
  if (kv_bf16) {
    if (src_bf16) DRT_KV16(__bf16, true); else DRT_KV16(__bf16, false);
  } else {
    if (src_bf16) DRT_KV16(_Float16, true); else DRT_KV16(_Float16, false);
  }
#undef DRT_KV16
  DRT_HIP(hipGetLastError());
}

}  // namespace drt
