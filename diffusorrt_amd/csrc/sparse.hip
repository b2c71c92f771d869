// Block-sparse GQA attention for gfx950: which blocks of keys each query row reads, and the
// attention over them.
//
// Blocks are `block` keys (whole tiles of 32) of a K/V head. A row's blocks for a K/V head are
// its first `sinks`, its last `local` (the last one it sees among them) and, of those between, the ones with
// the largest
//   score(row, b) = (sum of the head group's queries of the row) . (sum of the block's keys)
// - up to a factor, the mean product of the group's queries with the block's keys. Every scored block
// is seen whole: the last block, which the mask may cut, is taken without a score, so that
// no key behind the mask has a say. Equal scores: the lower block. The score is
// a 64-bit sum: of 11-bit queries and 24-bit sums of keys it is all but exact, and the
// choice does not depend on the order of addition.
#include "kv8.h"
#include "launch.h"

#include <cmath>

using drt::AttnWhere;
using drt::SparseSel;

namespace {

DRT_DEV float q_value(uint16_t bits, int bf16) {
  return bf16 ? bf16_bits_to_float(bits) : (float)__builtin_bit_cast(_Float16, bits);
}

// The scores as whole numbers of the same order (a NaN the largest, either zero the same).
DRT_DEV uint64_t score_key(double x) {
  x += 0.0;
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  if (x != x) return ~0ull;
  return b >> 63 ? ~b : b | (1ull << 63);
}

// Scores of 16 rows against 64 blocks of one K/V head: thread (b, r) holds block b of rows 4r ..
// 4r + 3, the queries' and the blocks' sums meet in LDS in 64 bits, 32 head dims at a time.
// Grid: (row group * chunks + chunk) * Hkv + head.
constexpr int SEL_ROWS = 16, SEL_BLOCKS = 64, SEL_DIMS = 32;
__global__ __launch_bounds__(256) void block_scores_kernel(
    const uint16_t* __restrict__ q, int q_bf16, const float* __restrict__ sums,
    int64_t sums_head_stride, int row0, int n_rows, int Hq, int Hkv, const AttnWhere where,
    const SparseSel sel, int n_blocks, uint64_t* __restrict__ keys) {
  const int kvh = blockIdx.x % Hkv, rest = blockIdx.x / Hkv;
  const int chunks = (n_blocks + SEL_BLOCKS - 1) / SEL_BLOCKS;
  const int chunk = rest % chunks, r0 = (rest / chunks) * SEL_ROWS;
  const int G = Hq / Hkv, tid = threadIdx.x, m = sel.block >> 5;
  // the last row of the group sees the most: blocks at or beyond its last `local` are never scored
  const int rows = min(SEL_ROWS, n_rows - r0);
  const int scored = (key_end_of(row0 + r0 + rows - 1, where) + sel.block - 1) / sel.block - sel.local;
  const int b0 = chunk * SEL_BLOCKS;
  if (b0 >= scored) return;
  __shared__ double qs[SEL_ROWS][SEL_DIMS];
  __shared__ double bs[SEL_DIMS][SEL_BLOCKS + 1];
  const int lb = tid & 63, lr = (tid >> 6) * 4;
  double acc[4] = {0.0, 0.0, 0.0, 0.0};
  for (int d0 = 0; d0 < 128; d0 += SEL_DIMS) {
    __syncthreads();
    for (int i = tid; i < SEL_ROWS * SEL_DIMS; i += 256) {
      const int r = i / SEL_DIMS, d = i % SEL_DIMS;
      double s = 0.0;
      if (r < rows) {
        const uint16_t* p = q + ((int64_t)(row0 + r0 + r) * Hq + kvh * G) * 128 + d0 + d;
        for (int g = 0; g < G; ++g) s += (double)q_value(p[g * 128], q_bf16);
      }
      qs[r][d] = s;
    }
    for (int i = tid; i < SEL_BLOCKS * SEL_DIMS; i += 256) {
      const int b = i / SEL_DIMS, d = i % SEL_DIMS;
      double s = 0.0;
      if (b0 + b < scored) {
        const float* p = sums + kvh * sums_head_stride + (int64_t)(b0 + b) * m * 128 + d0 + d;
        for (int t = 0; t < m; ++t) s += (double)p[t * 128];
      }
      bs[d][b] = s;
    }
    __syncthreads();
#pragma unroll 4
    for (int d = 0; d < SEL_DIMS; ++d) {
      const double x = bs[d][lb];
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = fma(qs[lr + e][d], x, acc[e]);
    }
  }
  if (b0 + lb >= scored) return;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (lr + e < rows)
      keys[((int64_t)(r0 + lr + e) * Hkv + kvh) * n_blocks + b0 + lb] = score_key(acc[e]);
}

// A row's choice for one K/V head, one wave: the need-th largest key by its bits from the
// top (a candidate prefix stands when at least `need` keys reach it; when exactly `need` do, they are the choice),
// then the blocks in ascending order. R: keys a lane holds, block 64 i + lane (0: read anew each time).
template <int R>
__global__ __launch_bounds__(256) void choose_blocks_kernel(const uint64_t* __restrict__ keys,
                                                            int row0, int n_rows, int Hkv,
                                                            const AttnWhere where,
                                                            const SparseSel sel, int n_blocks,
                                                            int32_t* __restrict__ blocks) {
  const int lane = threadIdx.x & 63;
  const int64_t id = blockIdx.x * (int64_t)4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (id >= (int64_t)n_rows * Hkv) return;
  const int row = row0 + (int)(id / Hkv);
  const uint64_t* mine = keys + id * n_blocks;
  int32_t* out = blocks + ((int64_t)row0 * Hkv + id) * sel.count;
  const int nb = (key_end_of(row, where) + sel.block - 1) / sel.block;  // blocks the row sees
  if (nb <= sel.count) {
    for (int i = lane; i < sel.count; i += 64) out[i] = i < nb ? i : -1;
    return;
  }
  const int lo = sel.sinks, hi = nb - sel.local;  // scored blocks
  const int need = sel.count - sel.sinks - sel.local;
  uint64_t held[R ? R : 1];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int b = 64 * i + lane;
    held[i] = b >= lo && b < hi ? mine[b] : 0ull;
  }
  // f(i, key of block 64 i + lane) for every i; 0, below every score's, where none is scored
  auto each = [&](auto&& f) {
    if constexpr (R > 0) {
#pragma unroll
      for (int i = 0; i < R; ++i) f(i, held[i]);
    } else {
      for (int i = 0; i < (nb + 63) / 64; ++i) {
        const int b = 64 * i + lane;
        f(i, b >= lo && b < hi ? mine[b] : 0ull);
      }
    }
  };
  uint64_t cut = 0ull;  // the largest prefix that at least `need` keys reach
  bool exact = need == 0;
  for (int bit = 63; bit >= 0 && !exact; --bit) {
    const uint64_t want = cut | (1ull << bit);
    int n = 0;
    each([&](int, uint64_t k) { n += __popcll(__ballot(k >= want)); });
    if (n >= need) {
      cut = want;
      exact = n == need;
    }
  }
  if (need == 0) cut = ~0ull;
  // keys above the cut all count, of those at it the first
  int ties = need;
  each([&](int, uint64_t k) { ties -= __popcll(__ballot(k > cut)); });
  int at = 0;
  const uint64_t below = (1ull << lane) - 1;
  each([&](int i, uint64_t k) {
    const int b = 64 * i + lane;
    const bool scored = b >= lo && b < hi;
    const uint64_t tied = __ballot(scored && k == cut);
    bool take = scored ? k > cut : b < nb;
    if (scored && k == cut) take = (int)__popcll(tied & below) < ties;
    ties -= min(ties, (int)__popcll(tied));
    const uint64_t mask = __ballot(take);
    if (take) out[at + __popcll(mask & below)] = b;
    at += __popcll(mask);
  });
}

// ---- attention over the listed blocks

template <int DT> struct SparseT;  // 0 = 8-bit (fp16 products), 1 = fp16, 2 = bf16
template <> struct SparseT<0> { typedef f16x8 vec; };
template <> struct SparseT<1> { typedef f16x8 vec; };
template <> struct SparseT<2> { typedef bf16x8 vec; };
DRT_DEV f32x4 mma16(const f16x8 a, const f16x8 b, const f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
DRT_DEV f32x4 mma16(const bf16x8 a, const bf16x8 b, const f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

constexpr int SP_LIST = 1024;  // the longest list of blocks

struct SpOut {
  void* out;       // [rows][Hq * 128], bf16 or fp32
  float* o_part;   // [splits][rows][Hq][128] (splits > 1)
  float* ml_part;  // [splits][rows][Hq][2]
  int bf16;
};

// One wave per (row, K/V head, key range), up to 16 query heads of the group as the columns of
// 16x16x32 products, two tiles (64 keys) at a time straight from the cache:
//   S^T: row i = 4g + r of product n is key 4(g&1) + r + 8n of tile g/2, so lane (g, column)
//        ends up with the keys that the second product wants from it;
//   O^T: k group g is tile g/2, keys 16kh + 4(g&1) + {0..3, 8..11} for kh = 0, 1.
// Both are 16 bytes a lane of the cache as it is, either element size. The four waves of a
// work-group take neighbouring rows, whose blocks are likely the same.
// Lists: ascending, -1 behind; an entry no larger than one before it, or beyond the row's
// keys, is passed over. Statistics as in the dense kernels (8-bit tiles: attention8.hip).
template <int DT>
__global__ __launch_bounds__(256) void sparse_attn_kernel(
    const uint16_t* __restrict__ q, int q_bf16, const uint8_t* __restrict__ kv,
    int64_t head_stride_bytes, const float* __restrict__ scales, int n_rows, int Hq, int Hkv,
    const AttnWhere where, const int32_t* __restrict__ blocks, int count, int block, int splits,
    int cgroups, float c, const SpOut ao) {
  typedef typename SparseT<DT>::vec vec;
  constexpr int TILE = DT == 0 ? KV8_TILE : 2 * KV8_TILE;
  __shared__ int lists[4][SP_LIST];
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int id = blockIdx.x;
  const int kvh = id % Hkv;
  id /= Hkv;
  const int cg = id % cgroups;
  id /= cgroups;
  const int split = id % splits, row = (id / splits) * 4 + wave;
  const int G = Hq / Hkv;
  if (row >= n_rows) return;  // (no barrier in this kernel)
  int* list = lists[wave];
  const int key_end = key_end_of(row, where);

  // the list's entries that count
  int n_list = 0, top = -1;
  {
    const int32_t* src = blocks + ((int64_t)row * Hkv + kvh) * count;
    for (int i = 0; i < count; i += 64) {
      const int b = i + lane < count ? src[i + lane] : -1;
      int run = max(b, top);  // largest up to here
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(run, o, 64);
        if (lane >= o) run = max(run, y);
      }
      int before = __shfl_up(run, 1, 64);
      if (lane == 0) before = top;
      const bool ok = b > before && (int64_t)b * block < key_end;
      const uint64_t mask = __ballot(ok);
      if (ok) list[n_list + __popcll(mask & ((1ull << lane) - 1))] = b;
      n_list += __popcll(mask);
      top = __shfl(run, 63, 64);
    }
  }
  const int m = block >> 5;
  // (of the last block only the tiles that the row sees)
  const int64_t n_tiles =
      n_list == 0 ? 0 : (int64_t)(n_list - 1) * m + min(m, ((key_end + 31) >> 5) - list[n_list - 1] * m);
  const int j0 = (int)(n_tiles * split / splits), j1 = (int)(n_tiles * (split + 1) / splits);

  // queries: column = head kvh * G + cg * 16 + col
  const int gi = cg * 16 + col, head = kvh * G + min(gi, G - 1);
  vec qf[4];
  float cq = c, nq = 0.f;  // (8-bit: kv8.h's 2^24 in c, -128 * 2^-24 the queries' sum)
  {
    const uint16_t* p = q + ((int64_t)row * Hq + head) * 128;
    u32x4 raw[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)  // head dims of k group g in step i, as the cache has them
      raw[i] = *(const u32x4*)(p + (DT == 0 ? 32 * (2 * (i >> 1) + (g >> 1)) + 16 * (i & 1) + 8 * (g & 1)
                                            : 32 * i + 8 * g));
    if (DT == 0 && q_bf16) {
      uint32_t most = 0u;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          most = max(most, max((raw[i][e] << 16) & 0x7fffffffu, raw[i][e] & 0x7fff0000u));
      most = max(most, (uint32_t)__shfl_xor((int)most, 16, 64));
      most = max(most, (uint32_t)__shfl_xor((int)most, 32, 64));
      const int x = most ? min(max((int)(most >> 23) - 127, -126), 126) : 0;
      cq = c * __uint_as_float((uint32_t)(127 + x) << 23);
      const float inv = __uint_as_float((uint32_t)(127 - x) << 23);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          raw[i][e] = pack_half2((_Float16)(__uint_as_float(raw[i][e] << 16) * inv),
                                 (_Float16)(__uint_as_float(raw[i][e] & 0xffff0000u) * inv));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) qf[i] = __builtin_bit_cast(vec, raw[i]);
    if constexpr (DT == 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) nq = kv8_add8(qf[i], nq);
      nq += __shfl_xor(nq, 16, 64);
      nq += __shfl_xor(nq, 32, 64);
      nq *= -KV8_BIAS / KV8_POW;
    }
  }
  float m_run = -INFINITY, l_run = 0.f, p_run = 0.f;
  int fold = 16;
  f32x4 o[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = f32x4{};
  const uint8_t* base = kv + kvh * head_stride_bytes;
  const float2* sc = (const float2*)scales + kvh * (head_stride_bytes / TILE);
  auto tile_at = [&](int j) {
    const int e = j / m;
    return __builtin_amdgcn_readfirstlane(list[e]) * m + (j - e * m);
  };
  for (int j = j0; j < j1; j += 2) {
    const int t0 = tile_at(j);
    const bool two = j + 1 < j1;
    const int t1 = two ? tile_at(j + 1) : t0;
    const int krow = col >> 3;  // the tile of this lane's row of S^T's first operand
    const uint8_t* kp = base + (int64_t)(krow ? t1 : t0) * TILE;
    const int tv = g >> 1 ? t1 : t0;
    const uint8_t* vp = base + (int64_t)tv * TILE + TILE / 2;
    const int kk = 4 * ((col >> 2) & 1) + (col & 3);  // + 8 n
    f32x4 s[4];
    u32x4 kr[4][DT == 0 ? 2 : 4];
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int i = 0; i < (DT == 0 ? 2 : 4); ++i)
        kr[n][i] = *(const u32x4*)(kp + (DT == 0 ? (((2 * i + (g >> 1)) * 2 + (g & 1)) * 32 + kk + 8 * n)
                                                 : ((4 * i + g) * 32 + kk + 8 * n)) * 16);
    u32x4 vr[8][DT == 0 ? 1 : 2];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int kh = 0; kh < (DT == 0 ? 1 : 2); ++kh)
        vr[i][kh] = *(const u32x4*)(vp + (DT == 0 ? ((i >> 1) * 2 + (g & 1)) * 32 + (i & 1) * 16 + col
                                                  : (((i >> 1) * 2 + kh) * 2 + (g & 1)) * 32 +
                                                        (i & 1) * 16 + col) * 16);
    float sk = 1.f, sv = 1.f;
    if (DT == 0) {
      const float2 x = sc[tv];
      sk = x.x;
      sv = x.y;
    }
    const int key0 = tv * 32 + 4 * (g & 1);  // + r + 8 n: this lane's keys
    const int end = (g >> 1) && !two ? 0 : key_end;
    if (DT == 0) {
      const bool bad = !(sk + sv < INFINITY);
      // a tile that is NaN: so is every row that sees it (tv * 32 < end: all of its lanes' columns)
      if (__ballot(bad && tv * 32 < end)) {
        l_run = NAN;
        if (m_run == -INFINITY) m_run = 0.f;
      }
      if (bad) sk = sv = 1.f;
    }
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      s[n] = f32x4{};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        vec kf;
        if constexpr (DT == 0)
          kf = kv8_to_f16(kr[n][i >> 1][2 * (i & 1)], kr[n][i >> 1][2 * (i & 1) + 1]);
        else
          kf = __builtin_bit_cast(vec, kr[n][DT == 0 ? 0 : i]);
        s[n] = mma16(kf, qf[i], s[n]);
      }
    }
    if (!two || max(t0, t1) * 32 + 32 > key_end) {
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[n][r] = key0 + r + 8 * n < end ? s[n][r] : -INFINITY;
      if (DT != 0) {  // what lies behind the row's keys is not even multiplied by zero
#pragma unroll
        for (int kh = 0; kh < (DT == 0 ? 1 : 2); ++kh)
#pragma unroll
          for (int e = 0; e < 4; ++e) {  // elements 2 e and 2 e + 1
            const int k0 = key0 + 16 * kh + 2 * (e & 1) + 8 * (e >> 1);
            const uint32_t keep = (k0 < end ? 0xffffu : 0u) | (k0 + 1 < end ? 0xffff0000u : 0u);
#pragma unroll
            for (int i = 0; i < 8; ++i) vr[i][kh][e] &= keep;
          }
      }
    }
    float a = DT == 0 ? __builtin_amdgcn_fmed3f(sk * cq, 1e-37f, 3e38f) : cq;
    const float lb = DT == 0 ? (float)((int)(__float_as_uint(sv) >> 23) - 127) : 0.f;
    const float inv_sv = DT == 0 ? __uint_as_float((254u << 23) - __float_as_uint(sv)) : 1.f;
    float tmax = s[0][0];
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) tmax = fmaxf(tmax, s[n][r]);
    const float off0 = DT == 0 ? fmaf(nq, a, lb) : 0.f;
    float u = fmaf(tmax, a, off0);
    u = fmaxf(u, __shfl_xor(u, 16, 64));
    u = fmaxf(u, __shfl_xor(u, 32, 64));
    const bool up = u > m_run + 8.f;
    if (__ballot(up) || (DT == 0 && --fold == 0)) {
      const float alpha = up ? __builtin_amdgcn_exp2f(m_run - u) : 1.f;
      float less = 0.f;
      if (DT == 0) {  // (kv8.h: the bytes' 128)
        less = p_run + __shfl_xor(p_run, 16, 64);
        less = alpha * (-KV8_BIAS / KV8_POW) * (less + __shfl_xor(less, 32, 64));
        p_run = 0.f;
        fold = 16;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] = fmaf(o[i][e], alpha, less);
      l_run *= alpha;
      m_run = up ? u : m_run;
    }
    const float mb = m_run == -INFINITY ? 0.f : m_run;
    float off = off0 - mb;
    if (__ballot(fabsf(mb) > 1048576.f)) {  // (attention8.hip: A8_LARGE)
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[n][r] = fmaf(s[n][r], a, off0);
      a = 1.f;
      off = -mb;
    }
    float psum = 0.f;
    vec pf[2];
#pragma unroll
    for (int kh = 0; kh < 2; ++kh)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float p = __builtin_amdgcn_exp2f(fmaf(s[2 * kh + (e >> 2)][e & 3], a, off));
        psum += p;
        if constexpr (DT == 2) pf[kh][e] = (__bf16)p;
        else pf[kh][e] = (_Float16)p;
      }
    if constexpr (DT == 0) p_run = kv8_add8(pf[1], kv8_add8(pf[0], p_run));
    l_run = fmaf(psum, inv_sv, l_run);
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int kh = 0; kh < 2; ++kh) {
        vec vf;
        if constexpr (DT == 0) vf = kv8_to_f16(vr[i][0][2 * kh], vr[i][0][2 * kh + 1]);
        else vf = __builtin_bit_cast(vec, vr[i][DT == 0 ? 0 : kh]);
        o[i] = mma16(vf, pf[kh], o[i]);
      }
  }
  l_run += __shfl_xor(l_run, 16, 64);
  l_run += __shfl_xor(l_run, 32, 64);
  if (DT == 0) {
    p_run += __shfl_xor(p_run, 16, 64);
    p_run += __shfl_xor(p_run, 32, 64);
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = fmaf(o[i][e], KV8_POW, -KV8_BIAS * p_run);
  }
  if (gi >= G) return;
  if (splits > 1) {
    const int64_t at = ((int64_t)split * n_rows + row) * Hq + head;
    float* p = ao.o_part + at * 128 + 4 * g;
#pragma unroll
    for (int i = 0; i < 8; ++i) *(f32x4*)(p + 16 * i) = o[i];
    if (g == 0) *(float2*)(ao.ml_part + at * 2) = make_float2(m_run, l_run);
    return;
  }
  const float inv = l_run == 0.f ? 0.f : 1.f / l_run;  // no key: zeros
  const int64_t at = ((int64_t)row * Hq + head) * 128 + 4 * g;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const f32x4 y = o[i] * inv;
    if (ao.bf16)
      *(uint2*)((uint16_t*)ao.out + at + 16 * i) =
          make_uint2((uint32_t)float_to_bf16_bits(y[0]) | ((uint32_t)float_to_bf16_bits(y[1]) << 16),
                     (uint32_t)float_to_bf16_bits(y[2]) | ((uint32_t)float_to_bf16_bits(y[3]) << 16));
    else
      *(f32x4*)((float*)ao.out + at + 16 * i) = y;
  }
}

// Rows whose scores one pass holds: 256 MiB of them at most.
int select_rows(int n_rows, int Hkv, int n_blocks) {
  const int64_t most = ((int64_t)1 << 28) / ((int64_t)Hkv * n_blocks * 8);
  return (int)std::min<int64_t>(n_rows, std::max<int64_t>(SEL_ROWS, most / SEL_ROWS * SEL_ROWS));
}

}  // namespace

namespace drt {

size_t select_blocks_bytes(int n_rows, int Hkv, int n_keys, int block) {
  const int nb = (int)(((int64_t)n_keys + block - 1) / block);
  return (size_t)select_rows(n_rows, Hkv, nb) * Hkv * nb * 8;
}

void select_blocks(const void* q, bool q_bf16, const float* sums, int64_t sums_head_stride,
                   int n_rows, int Hq, int Hkv, const AttnWhere& where, const SparseSel& sel,
                   void* workspace, int32_t* blocks, hipStream_t s) {
  const int nb = (int)(((int64_t)where.n_keys + sel.block - 1) / sel.block);
  const int step = select_rows(n_rows, Hkv, nb);
  const int64_t chunks = (nb + SEL_BLOCKS - 1) / SEL_BLOCKS;
  for (int r = 0; r < n_rows; r += step) {
    const int rows = std::min(step, n_rows - r);
    const int64_t grid = (rows + SEL_ROWS - 1) / SEL_ROWS * chunks * Hkv;
    require(grid < ((int64_t)1 << 31), "select_blocks: too many blocks for one call");
    if (nb > sel.count)
      hipLaunchKernelGGL(block_scores_kernel, dim3((unsigned)grid), dim3(256), 0, s,
                         (const uint16_t*)q, (int)q_bf16, sums, sums_head_stride, r, rows, Hq, Hkv,
                         where, sel, nb, (uint64_t*)workspace);
    const dim3 cgrid((unsigned)(((int64_t)rows * Hkv + 3) / 4));
#define DRT_CHOOSE(R)                                                                            \
  hipLaunchKernelGGL(choose_blocks_kernel<R>, cgrid, dim3(256), 0, s, (const uint64_t*)workspace, r, \
                     rows, Hkv, where, sel, nb, blocks)
    if (nb <= 256) DRT_CHOOSE(4);
    else if (nb <= 1024) DRT_CHOOSE(16);
    else if (nb <= 2048) DRT_CHOOSE(32);
    else DRT_CHOOSE(0);
#undef DRT_CHOOSE
    DRT_HIP(hipGetLastError());
  }
}

int sparse_splits(int n_rows, int Hq, int Hkv, int count, int block) {
  const int cgroups = (Hq / Hkv + 15) / 16;
  const int64_t waves = (int64_t)n_rows * Hkv * cgroups, pairs = ((int64_t)count * (block / 32) + 1) / 2;
  return (int)std::max<int64_t>(1, std::min<int64_t>({2048 / waves, pairs, 32}));
}

size_t sparse_part_bytes(int n_rows, int Hq, int splits) {
  return splits == 1 ? 0 : (size_t)splits * n_rows * Hq * 130 * 4;
}

void sparse_attention(KvType type, const void* q, bool q_bf16, const void* kv_layer,
                      int64_t kv_head_stride, const float* scales, int n_rows, int Hq, int Hkv,
                      const AttnWhere& where, const int32_t* blocks, int count, int block,
                      int splits, float* part, void* out, bool out_bf16, hipStream_t s) {
  const float c = 1.44269504088896340736f / sqrtf(128.0f) * (type == KvType::I8 ? KV8_POW : 1.f);
  const int cgroups = (Hq / Hkv + 15) / 16;
  const int64_t grid = ((int64_t)n_rows + 3) / 4 * splits * cgroups * Hkv;
  require(grid < ((int64_t)1 << 31), "sparse_attention: too many rows for one call");
  const int64_t n = (int64_t)n_rows * Hq;
  float* ml = part ? part + (size_t)splits * n * 128 : nullptr;
  const SpOut ao{out, part, ml, out_bf16};
  const int64_t bytes = type == KvType::I8 ? kv_head_stride : 2 * kv_head_stride;
#define DRT_SPARSE(DT)                                                                          \
  hipLaunchKernelGGL(sparse_attn_kernel<DT>, dim3((unsigned)grid), dim3(256), 0, s,             \
                     (const uint16_t*)q, (int)q_bf16, (const uint8_t*)kv_layer, bytes, scales,  \
                     n_rows, Hq, Hkv, where, blocks, count, block, splits, cgroups, c, ao)
  if (type == KvType::I8) DRT_SPARSE(0);
  else if (type == KvType::F16) DRT_SPARSE(1);
  else DRT_SPARSE(2);
#undef DRT_SPARSE
  DRT_HIP(hipGetLastError());
  if (splits > 1) part_combine(part, ml, splits, n, out, out_bf16, s);
}

}  // namespace drt
