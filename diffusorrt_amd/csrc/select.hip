// Which blocks of keys each query row reads in a block-sparse attention (cache_attention.hip).
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

}  // namespace drt
