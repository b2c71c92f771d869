// Which blocks of keys each query row reads in a block-sparse attention (cache_attention.hip).
//
// Blocks are `block` keys (whole tiles of 32) of a K/V head. A row's blocks for a K/V head are
// its first `sinks`, its last `local` (the last one it sees among them) and, of those between, the
// ones with the largest
//   score(row, b) = (sum of the head group's queries of the row) . (sum of the block's keys)
// - up to a factor, the mean product of the group's queries with the block's keys. Every scored block
// is seen whole: the last block, which the mask may cut, is taken without a score, so that
// no key behind the mask has a say. Equal scores: the lower block. The score is
// a 64-bit sum in a fixed order, from 24-bit sums of a tile's keys (exact over 8 bits, rounded once
// over 16): blocks whose scores are apart by more than some 2^-46 of the magnitudes added up
// are told apart, whatever the order.
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

// Blocks a row sees (one at least).
DRT_DEV int blocks_of(int row, const AttnWhere& where, int block) {
  return (int)((uint32_t)(key_end_of(row, where) - 1) / (uint32_t)block) + 1;
}

// The largest of the wave's values, by lane moves within 16 lanes, then from row to row.
DRT_DEV uint32_t wave_most(uint32_t x) {
#define DRT_STEP(CTRL) \
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, false))
  DRT_STEP(0x111);  // from 1, 2, 4, 8 lanes below
  DRT_STEP(0x112);
  DRT_STEP(0x114);
  DRT_STEP(0x118);
  DRT_STEP(0x142);  // lane 15 of a row to the next row, lane 31 to the upper half
  DRT_STEP(0x143);
#undef DRT_STEP
  return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}

// Set bits of a mask below this lane.
DRT_DEV int bits_below(uint64_t mask) {
  return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32),
                                        __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u));
}

// Scores of 16 rows against 16 blocks at a time, as 16x16x4 products in 64 bits. The rows' queries,
// the group's heads added up, meet in LDS; lane (i, g) then holds head dims 16 c + 4 g .. + 4
// (c = 0..7) of row i, and of block i as they are in memory (64 bytes in a row of 16 blocks a load),
// its tiles added up: a product takes one of them of each lane group, and leaves rows g, g + 4,
// g + 8, g + 12 of block i. The 32 products of 16 x 16 scores take a SIMD 2048 cycles.
typedef double f64x4 __attribute__((ext_vector_type(4)));
constexpr int SEL_QROW = 130;  // doubles of a row in LDS

template <int THREADS>
DRT_DEV void add_queries(const uint16_t* __restrict__ q, int q_bf16, int64_t row, int rows, int Hq,
                         int G, int kvh, double* qs) {
  constexpr int N = 2048 / THREADS;  // head dims a thread (8 or 2)
  const int r = threadIdx.x * N / 128, d = threadIdx.x * N % 128;
  const uint16_t* p = q + ((row + min(r, rows - 1)) * Hq + kvh * G) * 128 + d;
  double a[N] = {};
#pragma unroll 4
  for (int h = 0; h < G; ++h) {
    uint32_t w[N / 2];
    if constexpr (N == 8) {
      const u32x4 y = *(const u32x4*)(p + h * 128);
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = y[e];
    } else {
      w[0] = *(const uint32_t*)(p + h * 128);
    }
#pragma unroll
    for (int e = 0; e < N / 2; ++e) {
      a[2 * e] += (double)q_value((uint16_t)(w[e] & 0xffffu), q_bf16);
      a[2 * e + 1] += (double)q_value((uint16_t)(w[e] >> 16), q_bf16);
    }
  }
#pragma unroll
  for (int e = 0; e < N; ++e) qs[r * SEL_QROW + d + e] = a[e];
}

// Blocks b0 .. + 16, b0 + step .. + 16, ... below b_end: put(block, row of the 16, key). ready()
// is called once the first blocks are on their way, and returns with the queries in qs.
template <typename Ready, typename Put>
DRT_DEV void score_blocks(const float* __restrict__ sums, int b0, int step, int b_end, int m,
                          const double* qs, Ready&& ready, Put&& put) {
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const float* base = sums + 4 * g;
  f32x4 x[8];  // a block's first tile, loaded a step ahead
  auto load = [&](int b) {
    const float* p = base + (int64_t)min(b + i, b_end - 1) * m * 128;
#pragma unroll
    for (int c = 0; c < 8; ++c) x[c] = *(const f32x4_e*)(p + 16 * c);
  };
  if (b0 < b_end) load(b0);
  ready();
  if (b0 >= b_end) return;
  const double* a = qs + i * SEL_QROW + 4 * g;
  for (; b0 < b_end; b0 += step) {
    double y[32];
#pragma unroll
    for (int d = 0; d < 32; ++d) y[d] = (double)x[d >> 2][d & 3];
    const float* p = base + (int64_t)min(b0 + i, b_end - 1) * m * 128;
    for (int t = 1; t < m; ++t) {
#pragma unroll
      for (int c = 0; c < 8; ++c) x[c] = *(const f32x4_e*)(p + (int64_t)t * 128 + 16 * c);
#pragma unroll
      for (int d = 0; d < 32; ++d) y[d] += (double)x[d >> 2][d & 3];
    }
    load(b0 + step);  // (behind the last: loaded, not used)
    asm volatile("" ::: "memory");  // (queries read block by block: no registers for them all)
    f64x4 acc = f64x4{}, acc1 = f64x4{};  // (two chains: a product waits for the one before it)
#pragma unroll
    for (int d = 0; d < 32; d += 2) {
      const double* e = a + 16 * (d >> 2) + (d & 3);
      acc = __builtin_amdgcn_mfma_f64_16x16x4f64(e[0], y[d], acc, 0, 0, 0);
      acc1 = __builtin_amdgcn_mfma_f64_16x16x4f64(e[1], y[d + 1], acc1, 0, 0, 0);
    }
    acc += acc1;
    if (b0 + i < b_end) {
#pragma unroll
      for (int e = 0; e < 4; ++e) put(b0 + i, g + 4 * e, score_key(acc[e]));
    }
  }
}

// A row's choice for one K/V head, one wave: a cut that exactly `need` keys reach, then the blocks in
// ascending order. The cut lies between one that enough keys reach (first an exponent below the
// largest key, where that of scores mostly is, then two, four, ...) and one that too few do, and is
// found by halving; the upper halves of the keys alone mostly decide it, in about ten steps. Where
// equal keys leave none, the least key of the choice, found bit by bit.
// key_at(b): the key of scored block b. R: keys a lane holds, block 64 i + lane (0: asked for anew
// each time). A step costs each of the wave's rounds a comparison and a count.
template <int R, typename KeyAt>
DRT_DEV void choose_row(KeyAt&& key_at, int nb, const SparseSel& sel, int32_t* out) {
  const int lane = threadIdx.x & 63;
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
    held[i] = b >= lo && b < hi ? key_at(b) : 0ull;
  }
  // f(i, key of block 64 i + lane) for every i; 0, below every score's, where none is scored
  auto each = [&](auto&& f) {
    if constexpr (R > 0) {
#pragma unroll
      for (int i = 0; i < R; ++i) f(i, held[i]);
    } else {
      for (int i = 0; i < (nb + 63) / 64; ++i) {
        const int b = 64 * i + lane;
        f(i, b >= lo && b < hi ? key_at(b) : 0ull);
      }
    }
  };
  auto reach = [&](uint32_t want) {
    int n = 0;
    each([&](int, uint64_t k) { n += (int)__popcll(__ballot((uint32_t)(k >> 32) >= want)); });
    return n;
  };
  uint32_t upper = 0u;  // the largest that at least `need` keys' upper halves reach
  bool exact = need == 0;
  if (!exact) {
    uint32_t most = 0u;
    each([&](int, uint64_t k) { most = max(most, (uint32_t)(k >> 32)); });
    most = wave_most(most);
    // (no key's upper half is past `most`: that one may be ~0u, a NaN's, and is tried as it is)
    uint32_t high = most, down = 1u << 20;
    int n = reach(most);
    if (n >= need) {
      upper = most;
    } else {
      for (;;) {
        upper = most > down ? most - down : 0u;
        n = upper ? reach(upper) : need + 1;  // (0: reached by all, those without a score too)
        if (n >= need) break;
        high = upper;
        down = down < 1u << 31 ? down << 1 : ~0u;
      }
      while (n != need && high - upper > 1u) {
        const uint32_t mid = upper + (high - upper) / 2;
        const int k = reach(mid);
        if (k >= need) {
          upper = mid;
          n = k;
        } else {
          high = mid;
        }
      }
    }
    exact = n == need;
  }
  uint64_t cut = (uint64_t)upper << 32;
  for (int bit = 31; bit >= 0 && !exact; --bit) {
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
  each([&](int i, uint64_t k) {
    const int b = 64 * i + lane;
    const bool scored = b >= lo && b < hi;
    const uint64_t tied = __ballot(scored && k == cut);
    bool take = scored ? k > cut : b < nb;
    if (scored && k == cut) take = bits_below(tied) < ties;
    ties -= min(ties, (int)__popcll(tied));
    const uint64_t mask = __ballot(take);
    if (take) out[at + bits_below(mask)] = b;
    at += __popcll(mask);
  });
}

struct SelArgs {
  const uint16_t* q;   // [rows][Hq][128]
  const float* sums;   // [Hkv][tiles][128]
  int64_t sums_head_stride;
  int q_bf16, row0, n_rows, Hq, Hkv, n_blocks, per;
  AttnWhere where;
  SparseSel sel;
  uint64_t* keys;      // [n_rows][Hkv][n_blocks]
  int32_t* blocks;     // [rows][Hkv][count]
};

// Both steps for 16 rows of one K/V head in a work-group of 16 waves, the keys in LDS (RB rounds of
// 64 blocks). 1000 rows x 4 heads, 500 blocks: 22.1 us (23.8 with the choice's bits one after the other
// and divisions of 64 bits); in two launches, with the keys in memory, 22 + 14. Bound: a
// work-group's chain (queries, scores, barrier, the choice), of 252 work-groups on as many CUs at
// once; the 1 MB of sums is read from L2 and the products would take 7 us. Many more rows: L2, which
// every 16 rows read all sums from (2048 rows x 8 heads, 512 blocks of two tiles: 96 us, products 29).
template <int RB>
__global__ __launch_bounds__(1024, 4) void select_kernel(const SelArgs x) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kvh = blockIdx.x % x.Hkv, r0 = blockIdx.x / x.Hkv * 16;
  const int rows = min(16, x.n_rows - r0), G = x.Hq / x.Hkv;
  __shared__ double qs[16 * SEL_QROW];
  __shared__ uint64_t keys[16][RB * 64];
  // the last row sees the most: blocks at or beyond its last `local` are never scored
  const int nb_last = blocks_of(x.row0 + r0 + rows - 1, x.where, x.sel.block);
  const int b_end = nb_last <= x.sel.count ? 0 : nb_last - x.sel.local;
  score_blocks(x.sums + kvh * x.sums_head_stride, wave * 16, 256, b_end, x.sel.block >> 5, qs,
               [&] {
                 add_queries<1024>(x.q, x.q_bf16, x.row0 + r0, rows, x.Hq, G, kvh, qs);
                 __syncthreads();
               },
               [&](int b, int r, uint64_t k) { keys[r][b] = k; });
  __syncthreads();
  if (wave < rows) {
    const int64_t row = x.row0 + r0 + wave;
    choose_row<RB>([&](int b) { return keys[wave][b]; },
                   blocks_of((int)row, x.where, x.sel.block), x.sel,
                   x.blocks + (row * x.Hkv + kvh) * x.sel.count);
  }
}

// The scores alone: 16 rows against 64 * per blocks of one K/V head, four waves. For few rows: those
// of a block find 128 work-groups here, 16 above (32 rows x 8 heads over 512 blocks 6.7 us, and
// 5.7 for the choice, 12.4 a call; at once 24).
__global__ __launch_bounds__(256, 2) void block_scores_kernel(const SelArgs x) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // work-group: (row tile * chunks + chunk) * Hkv + head
  const int chunks = (x.n_blocks + 64 * x.per - 1) / (64 * x.per);
  const int kvh = blockIdx.x % x.Hkv, rest = blockIdx.x / x.Hkv, chunk = rest % chunks;
  const int r0 = rest / chunks * 16, rows = min(16, x.n_rows - r0), G = x.Hq / x.Hkv;
  const int scored = blocks_of(x.row0 + r0 + rows - 1, x.where, x.sel.block) - x.sel.local;
  if (chunk * x.per * 64 >= scored) return;
  __shared__ double qs[16 * SEL_QROW];
  const int b0 = (chunk * 4 + wave) * x.per * 16;
  score_blocks(x.sums + kvh * x.sums_head_stride, b0, 16, min(scored, b0 + x.per * 16),
               x.sel.block >> 5, qs,
               [&] {
                 add_queries<256>(x.q, x.q_bf16, x.row0 + r0, rows, x.Hq, G, kvh, qs);
                 __syncthreads();
               },
               [&](int b, int r, uint64_t k) {
                 if (r < rows) x.keys[((int64_t)(r0 + r) * x.Hkv + kvh) * x.n_blocks + b] = k;
               });
}

template <int R> __global__ __launch_bounds__(256) void choose_blocks_kernel(const SelArgs x) {
  const int64_t id = blockIdx.x * (int64_t)4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (id >= (int64_t)x.n_rows * x.Hkv) return;
  const uint64_t* mine = x.keys + id * x.n_blocks;
  choose_row<R>([&](int b) { return mine[b]; },
                blocks_of(x.row0 + (int)(id / x.Hkv), x.where, x.sel.block), x.sel,
                x.blocks + ((int64_t)x.row0 * x.Hkv + id) * x.sel.count);
}

// Rows whose scores one pass holds: 256 MiB of keys, or those of 16 rows where these are more (which
// share what a pass reads of the sums; a quarter of the sums' bytes at most).
int select_rows(int n_rows, int Hkv, int n_blocks) {
  const int64_t most = ((int64_t)1 << 28) / ((int64_t)Hkv * n_blocks * 8);
  return (int)std::min<int64_t>(n_rows, std::max<int64_t>(16, most / 16 * 16));
}

}  // namespace

namespace drt {

// Both steps in one launch: work-groups of 16 rows and a K/V head that find half the CUs at
// least something to do, and keys that fit LDS; or so few blocks that one work-group's time for them
// is less than a second launch's (a call of 32 rows x 8 heads, blocks of 64: 128 of them 9.8 us, in
// two launches 12.2; 256 of them 14.7 and 12.3).
static bool select_at_once(int n_rows, int Hkv, int n_blocks) {
  return n_blocks <= 128 || (n_blocks <= 1024 && (int64_t)((n_rows + 15) / 16) * Hkv >= 128);
}

size_t select_blocks_bytes(int n_rows, int Hkv, int n_keys, int block) {
  const int nb = (int)(((int64_t)n_keys + block - 1) / block);
  return select_at_once(n_rows, Hkv, nb) ? 0 : (size_t)select_rows(n_rows, Hkv, nb) * Hkv * nb * 8;
}

void select_blocks(const void* q, bool q_bf16, const float* sums, int64_t sums_head_stride,
                   int n_rows, int Hq, int Hkv, const AttnWhere& where, const SparseSel& sel,
                   void* workspace, int32_t* blocks, hipStream_t s) {
  const int nb = (int)(((int64_t)where.n_keys + sel.block - 1) / sel.block);
  SelArgs a{(const uint16_t*)q, sums, sums_head_stride, (int)q_bf16, 0, n_rows, Hq, Hkv, nb, 1, where,
            sel, (uint64_t*)workspace, blocks};
  if (select_at_once(n_rows, Hkv, nb)) {
    const int64_t wgs = (int64_t)((n_rows + 15) / 16) * Hkv;
    require(wgs < ((int64_t)1 << 31), "select_blocks: too many rows for one call");
    const dim3 grid((unsigned)wgs);
    if (nb <= 128) hipLaunchKernelGGL(select_kernel<2>, grid, dim3(1024), 0, s, a);
    else if (nb <= 256) hipLaunchKernelGGL(select_kernel<4>, grid, dim3(1024), 0, s, a);
    else if (nb <= 512) hipLaunchKernelGGL(select_kernel<8>, grid, dim3(1024), 0, s, a);
    else hipLaunchKernelGGL(select_kernel<16>, grid, dim3(1024), 0, s, a);
    DRT_HIP(hipGetLastError());
    return;
  }
  const int step = select_rows(n_rows, Hkv, nb);
  for (int r = 0; r < n_rows; r += step) {
    a.row0 = r;
    a.n_rows = std::min(step, n_rows - r);
    const int64_t tiles = (a.n_rows + 15) / 16;
    if (nb > sel.count) {
      // 16 x 16 scores a wave: as few as leave no SIMD without a wave, four at most
      a.per = (int)std::max<int64_t>(1, std::min<int64_t>(4, tiles * ((nb + 15) / 16) * Hkv / 1024));
      const int64_t wgs = tiles * ((nb + 64 * a.per - 1) / (64 * a.per)) * Hkv;
      require(wgs < ((int64_t)1 << 31), "select_blocks: too many blocks for one call");
      hipLaunchKernelGGL(block_scores_kernel, dim3((unsigned)wgs), dim3(256), 0, s, a);
    }
    const dim3 grid((unsigned)(((int64_t)a.n_rows * Hkv + 3) / 4));
    if (nb <= 256) hipLaunchKernelGGL(choose_blocks_kernel<4>, grid, dim3(256), 0, s, a);
    else if (nb <= 512) hipLaunchKernelGGL(choose_blocks_kernel<8>, grid, dim3(256), 0, s, a);
    else if (nb <= 1024) hipLaunchKernelGGL(choose_blocks_kernel<16>, grid, dim3(256), 0, s, a);
    else if (nb <= 2048) hipLaunchKernelGGL(choose_blocks_kernel<32>, grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL(choose_blocks_kernel<0>, grid, dim3(256), 0, s, a);
    DRT_HIP(hipGetLastError());
  }
}

}  // namespace drt
