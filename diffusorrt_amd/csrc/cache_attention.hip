// GQA attention over the prefix cache for gfx950: over all of an 8-bit cache's keys (kv8.h), decode
// blocks and prompts alike, and over listed blocks of either cache's.
//
// Queries of one K/V head are flattened to query vectors (row, head of the group) in tiles of 32, keys
// come in tiles of 32, and a wave computes S^T = K Q^T and O^T += V^T P^T as 32x32x16 products, as
// the attention over a whole 16-bit cache (attention.hip) does.
// A wave loads a tile (8 KiB of codes, 16 KiB of 16-bit values) straight into registers, 16 bytes a
// lane and load, and makes fp16 operands of codes there: no staging, no barrier in the loop. A tile's K
// registers are loaded anew as soon as its scores are done, its V registers after its products.
//
// Scales. With K = 2^a k and V = 2^b v for a tile (k, v the codes), the base-2 exponent of a
// weighted value is u = (k . q) * 2^a * c, c = log2(e) / sqrt(128), and
//   o = sum p v 2^b / sum p,  p = 2^u.
// The wave keeps p' = 2^(u + b - base): its sum against v needs no factor, and the normaliser
// adds 2^-b of a tile's sum of p'. So a tile's scales cost a few operations a lane, not one a
// score, and p' is largest where a tile's part of the result is: fp16 holds it to 2^-11 of its value
// wherever it counts. The running base is raised when a tile's largest u + b exceeds it by more than
// 8 (p' <= 2^8); any base gives the same quotient. p' is the one rounding ahead of the sums
// (to the product's operand type); scores, base, normaliser and O are fp32. The normaliser adds p'
// before that rounding: weights on a tile of tiny values may vanish in fp16 beside others, not in it.
// Queries over 8 bits: fp16 as they are; bf16 ones are scaled by a power of two per query vector to a
// largest magnitude in [1, 2) (exact: fp16 has three bits more; elements below 2^-14 of the
// vector's largest lose some, at most 2^-25 of that largest).
//
// Listed blocks. A query tile is the 32 / G rows (G heads a group; 32 heads at a time above that) of
// neighbours, and the tile's blocks are the union of its rows' lists, each with a bit per row: an
// LDS bitmap, CA_WIN blocks at a time, so a list is a set, whatever its order and repetitions.
// Neighbouring queries mostly choose the same blocks: a block is then loaded and made operands once
// for all of them, and every column of the products is in use (one wave per row, 16 columns of
// which G are used: 2048 rows x 16 heads, 16 blocks of 64 of 32768 keys, 226 us; 52 here).
//
// Bound. A long cache's codes (32 rows x 16 heads over 131072 keys x 8 heads, 268 MB: 57 us, 4.7
// TB/s, what a large copy reaches). Many rows: the instructions of the softmax and of making
// operands, by the counters 52 % of all cycles on the VALU and 33 % on the matrix units, which two
// waves a SIMD overlap little (2048 rows x 16 heads over 4096 keys under the mask: 62 us, 0.83 PFLOP/s;
// over 32768 506 us, 1.05). Many rows over lists: 46 and 21 %, and between them the wait for tiles, one
// a wave under way (2048 rows x 16 heads, 16 blocks of 64: 463 MB asked of L2, of which 168 miss). A
// block of 32 rows x 16 heads over 8224 keys: 11.5 us with its combine, in a graph, of which about 7
// are there without any tile (launches, queries, the ways' meeting, parts out and in). Three waves a
// SIMD spill; a larger window of blocks in LDS for two (60 us for 57), weights' sums by other chains or
// by dot products did not pay.
#include "cache_dev.h"
#include "launch.h"

#include <cmath>

using drt::AttnWhere;

namespace {

// The bytes' 128 leaves O with the running sum of weights, at the latest after so many tiles: its
// share of the sum in fp32, which costs O precision, stays that of 1024 keys.
constexpr int CA_FOLD = 32;
constexpr int CA_QROW = 136;  // 16-bit elements per query vector in LDS (+ 16 bytes)
constexpr int CA_WIN = 2048;  // blocks of one bitmap

// The value of another lane: one away, two away, the mirror image in eight, in sixteen. The four steps
// join 16 lanes.
template <int STEP> DRT_DEV uint32_t ca_of_16(uint32_t x) {
  constexpr int CTRL = STEP == 0 ? 0xb1 : STEP == 1 ? 0x4e : STEP == 2 ? 0x141 : 0x140;
  return (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, CTRL, 0xf, 0xf, true);
}
DRT_DEV uint32_t ca_max16(uint32_t x) {
  x = max(x, ca_of_16<0>(x));
  x = max(x, ca_of_16<1>(x));
  x = max(x, ca_of_16<2>(x));
  return max(x, ca_of_16<3>(x));
}
DRT_DEV float ca_sum16(float x) {
  x += __uint_as_float(ca_of_16<0>(__float_as_uint(x)));
  x += __uint_as_float(ca_of_16<1>(__float_as_uint(x)));
  x += __uint_as_float(ca_of_16<2>(__float_as_uint(x)));
  return x + __uint_as_float(ca_of_16<3>(__float_as_uint(x)));
}

struct CaArgs {
  const uint16_t* q;       // [rows][Hq][128]
  const uint8_t* kv;       // this layer
  int64_t head_stride;     // bytes
  const float* scales;     // 8-bit
  const int32_t* blocks;   // [rows][Hkv][count] (listed blocks)
  int q_bf16, n_rows, Hq, Hkv, splits, count, block;
  float c;                 // log2(e) / sqrt(128), times 2^24 over 8 bits
  AttnWhere where;
  void* out;               // [rows][Hq * 128], bf16 or fp32
  float* o_part;           // [splits][rows][Hq][128] (not OUT)
  float* ml_part;          // [splits][rows][Hq][2]
  int out_bf16;
};

// QT query tiles, KW waves over keys (wave kw takes key tiles kw, kw + KW, ...; their parts meet in LDS
// at the end). OUT: one key range, the result itself; otherwise a part for the combine.
// SPARSE: the listed blocks' keys.
template <int DT, int QT, int KW, bool OUT, bool SPARSE>
__global__ __launch_bounds__(64 * KW, 2) void cache_attn_kernel(const CaArgs x) {
  typedef CacheT<DT> T;
  typedef typename T::vec vec;
  constexpr int THREADS = 64 * KW, NQ = 32 * QT, TILE = T::TILE, LD = T::LOADS;
  static_assert(!SPARSE || QT == 1, "a work-group has one union of lists");
  // LDS: the queries, then halves (64 head dims) of every wave's O, one after the other: the first is
  // on its way to memory under the second (32 rows over 8224 keys 12.3 us; all at once 12.7). One
  // query tile has little to write: all at once (one row over 8192 keys 6.4 us; halves 6.9).
  constexpr int PASSES = KW == 8 && !SPARSE ? 1 : 2, PIECES = 32 / PASSES, WAVE_O = 32 * PIECES * 16;
  constexpr int Q_BYTES = NQ * CA_QROW * 2, O_BYTES = KW * QT * WAVE_O;
  __shared__ __align__(16) char smem[Q_BYTES > O_BYTES ? Q_BYTES : O_BYTES];
  __shared__ float2 ml[KW][NQ];  // base and sum of every way
  __shared__ float2 qinfo[NQ];  // c times a query vector's power of two; -128 * 2^-24 its sum
  __shared__ uint32_t bits[SPARSE ? CA_WIN : 1];  // rows that list a block of the window
  __shared__ int2 list[SPARSE ? CA_WIN : 1];      // its blocks and their rows
  __shared__ int tally[SPARSE ? KW : 1];
  const int lane = threadIdx.x & 63, tid = threadIdx.x;
  const int kw = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const AttnWhere& where = x.where;
  const int G = x.Hq / x.Hkv, kvh = blockIdx.x % x.Hkv, split = blockIdx.x / x.Hkv;
  // the last rows, which see the most keys, start first
  const int group = (int)gridDim.y - 1 - (int)blockIdx.y;

  // The (row, head) of query vector v of the work-group.
  const int GC = SPARSE ? min(G, 32) : G, RPT = 32 / GC;  // (listed blocks) heads and rows of a tile
  const int head0 = SPARSE ? (int)blockIdx.z * 32 : 0, row0 = SPARSE ? group * RPT : 0;
  const int qt0 = SPARSE ? 0 : group * QT, n_qv = x.n_rows * G;
  auto row_of = [&](int v) { return SPARSE ? row0 + v / GC : (qt0 * 32 + v) / G; };
  auto head_of = [&](int v) {
    return kvh * G + (SPARSE ? head0 + v % GC : (qt0 * 32 + v) % G);
  };
  auto exists = [&](int v) {
    return SPARSE ? v < RPT * GC && row0 + v / GC < x.n_rows && head0 + v % GC < G
                  : qt0 * 32 + v < n_qv;
  };

  // the tile's lists, their first entries on their way
  const int end_row = min(SPARSE ? row0 + RPT - 1 : 0, x.n_rows - 1);
  const int n_entries = SPARSE ? (end_row - row0 + 1) * x.count : 0;
  auto entry = [&](int i, int& r) {
    r = (int)((uint32_t)i / (uint32_t)x.count);
    return x.blocks[((int64_t)(row0 + r) * x.Hkv + kvh) * x.count + (i - r * x.count)];
  };
  int entry0 = -1, entry0_row = 0;
  if (SPARSE && tid < n_entries) entry0 = entry(tid, entry0_row);

  // the queries, 16 threads (eight elements each) a query vector, on their way
  constexpr int QL = NQ * 16 / THREADS;
  static_assert(QL * THREADS == NQ * 16, "whole rounds of the queries");
  u32x4 qraw[QL];
#pragma unroll
  for (int it = 0; it < QL; ++it) {
    const int v = (it * THREADS + tid) >> 4;
    qraw[it] = u32x4{0u, 0u, 0u, 0u};
    if (exists(v))
      qraw[it] = *(const u32x4*)(x.q + ((int64_t)row_of(v) * x.Hq + head_of(v)) * 128 + (tid & 15) * 8);
  }

  const uint16_t* ql = (const uint16_t*)smem + (lane & 31) * CA_QROW + 8 * (lane >> 5);
  constexpr bool HOLD = QT == 1 && DT == 0;  // the queries' operands in registers (16 bits: too many)
  vec qr[HOLD ? 8 : 1];
  int q_end[QT];
  float cq[QT], nq[QT], m_run[QT], l_run[QT], p_run[QT];
  f32x16 o[QT][4];
  const int last_row = x.n_rows - 1;
#pragma unroll
  for (int j = 0; j < QT; ++j)
    q_end[j] = key_end_of(min(row_of(j * 32 + (lane & 31)), last_row), where);
  // Queries into LDS and from there to the waves. Called by every thread, once, with the
  // first tile's loads under way.
  auto stage = [&] {
#pragma unroll
    for (int it = 0; it < QL; ++it) {
      const int v = (it * THREADS + tid) >> 4, ch = tid & 15;
      u32x4 raw = qraw[it];
      float pw = 1.f, sum = 0.f;
      if constexpr (DT == 0) {
        if (x.q_bf16) {
          uint32_t most = 0u;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            most = max(most, max((raw[e] << 16) & 0x7fffffffu, raw[e] & 0x7fff0000u));
          most = ca_max16(most);
          const int ex = most ? min(max((int)(most >> 23) - 127, -126), 126) : 0;
          // (beyond 2^80 the scores are further apart than fp32 tells, and would overflow)
          pw = __uint_as_float((uint32_t)(127 + min(ex, 80)) << 23);
          const float inv = __uint_as_float((uint32_t)(127 - ex) << 23);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            raw[e] = pack_half2((_Float16)(__uint_as_float(raw[e] << 16) * inv),
                                (_Float16)(__uint_as_float(raw[e] & 0xffff0000u) * inv));
        }
        sum = ca_sum16(kv8_add8(__builtin_bit_cast(f16x8, raw), 0.f));
      }
      *(u32x4*)(smem + (v * CA_QROW + ch * 8) * 2) = raw;
      if (ch == 0) qinfo[v] = make_float2(x.c * pw, -KV8_BIAS / KV8_POW * sum);
    }
    ca_lds_barrier();
    if (HOLD) {
#pragma unroll
      for (int i = 0; i < 8; ++i) qr[HOLD ? i : 0] = *(const vec*)(ql + 16 * i);
    }
#pragma unroll
    for (int j = 0; j < QT; ++j) {
      const float2 y = qinfo[j * 32 + (lane & 31)];
      cq[j] = y.x;
      nq[j] = y.y;
    }
  };
  auto reset = [&] {
#pragma unroll
    for (int j = 0; j < QT; ++j) {
      m_run[j] = -INFINITY;
      l_run[j] = p_run[j] = 0.f;
#pragma unroll
      for (int hb = 0; hb < 4; ++hb) o[j][hb] = f32x16{};
    }
  };
  reset();
  // (ends never fall from row to row) keys that every row of the work-group sees, and any of them
  const int full_end = key_end_of(min(row_of(0), last_row), where);
  const int any_end = key_end_of(SPARSE ? end_row : min(row_of(QT * 32 - 1), last_row), where);
  const uint32_t my_row = SPARSE ? 1u << ((lane & 31) / GC & 31) : 0u;
  const uint32_t all_rows = SPARSE ? (uint32_t)((1ull << (end_row - row0 + 1)) - 1) : 0u;

  const uint8_t* base = x.kv + kvh * x.head_stride + lane * 16;
  // (scalar loads: a vector load's value would be waited for with the tile in flight)
  const auto* sc = (const __attribute__((address_space(4))) float*)(uintptr_t)(
      DT == 0 ? x.scales + kvh * (x.head_stride / TILE) * 2 : nullptr);
  auto scales_of = [&](int t) { return make_float2(sc[2 * (int64_t)t], sc[2 * (int64_t)t + 1]); };
  u32x4 kr[LD], vr[LD];
  float2 st = make_float2(1.f, 1.f);
  int fold = CA_FOLD;
  uint32_t heard = 0u;  // whether this lane's row sees any of the wave's tiles

  auto first = [&](int n, int t) {
    if (n <= 0) return;
    const uint8_t* p = base + (int64_t)t * TILE;
#pragma unroll
    for (int i = 0; i < LD; ++i) kr[i] = *(const u32x4*)(p + i * 1024);
#pragma unroll
    for (int i = 0; i < LD; ++i) vr[i] = *(const u32x4*)(p + TILE / 2 + i * 1024);
    if (DT == 0) st = scales_of(t);
  };
  // n tiles, the first (on its way) at t with its rows; next(t, rows) steps to the wave's following
  // tile. careful (16 bits): see below.
  auto run = [&](int n, int t, uint32_t rows, bool careful, auto&& next) {
    for (int it = 0; it < n; ++it) {
      const int key0 = t * 32;
      const uint32_t seen = rows;
      const float sk = st.x, sv = st.y;
      if (it + 1 < n) next(t, rows);  // (the last tile's own again: loaded, not used)
      const uint8_t* p = base + (int64_t)t * TILE;
      f32x16 s[QT];
#pragma unroll
      for (int j = 0; j < QT; ++j) s[j] = f32x16{};
      if (!HOLD) asm volatile("" ::: "memory");  // (read the queries here, tile by tile)
      // products ahead of another wave's softmax: 75 -> 72 us for 2048 rows over 4096 keys
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const vec kf = ca_operand<DT>(kr, i);
#pragma unroll
        for (int j = 0; j < QT; ++j)
          s[j] = T::mma(
              kf, HOLD ? qr[HOLD ? i : 0] : *(const vec*)(ql + j * 32 * CA_QROW + 16 * i), s[j]);
      }
#pragma unroll
      for (int i = 0; i < LD; ++i) kr[i] = *(const u32x4*)(p + i * 1024);
      __builtin_amdgcn_s_setprio(0);
      // (a scalar load among the reads of LDS would be waited for with them)
      asm volatile("" ::: "memory");
      if (DT == 0) st = scales_of(t);
      const bool bad = DT == 0 && !(sk + sv < INFINITY);  // a NaN tile: so is every row that sees it
      // A row that does not list the tile's block weighs it nothing: by its exponent's offset where
      // its end is not in the tile either. (A NaN score then still is one: see careful, heard.)
      const bool hit = !SPARSE || (seen & my_row) != 0u;
      if (SPARSE) heard |= key0 < q_end[0] ? seen & my_row : 0u;
      const bool part = key0 + 32 > full_end || (SPARSE && seen != all_rows);
      if (key0 + 32 > full_end || bad || (careful && part)) {
#pragma unroll
        for (int j = 0; j < QT; ++j) {
          const int mine = hit ? q_end[j] : 0;
          if (bad && key0 < mine) {
            l_run[j] = NAN;
            m_run[j] = m_run[j] == -INFINITY ? 0.f : m_run[j];
          }
          const int end = bad ? 0 : mine;
#pragma unroll
          for (int r = 0; r < 16; ++r) s[j][r] = key0 + mfma_row(r, lane) < end ? s[j][r] : -INFINITY;
        }
      }
      const uint32_t vb = __float_as_uint(sv);  // sv = 2^lb
      const float lb = DT != 0 || bad ? 0.f : (float)((int)(vb >> 23) - 127);
      const float inv_sv = DT != 0 ? 1.f : bad ? 0.f : __uint_as_float((254u << 23) - vb);
      vec pf[QT][2];
#pragma unroll
      for (int j = 0; j < QT; ++j) {
        // (within the finite numbers above zero whatever the powers of two: no 0 * inf)
        float a = DT != 0 ? cq[j] : bad ? 1.f : __builtin_amdgcn_fmed3f(sk * cq[j], 1e-37f, 3e38f);
        float tmax = s[j][0];
#pragma unroll
        for (int r = 1; r < 16; ++r) tmax = fmaxf(tmax, s[j][r]);
        const float off0 = DT != 0 ? 0.f : fmaf(nq[j], a, lb);
        const float u = hit ? fmaf(ca_max_xor32(tmax), a, off0) : -INFINITY;  // -inf: no visible key
        const bool up = u > m_run[j] + CA_RESCALE_LOG2;
        if (__ballot(up) || (DT == 0 && fold == 1)) {
          const float alpha = up ? __builtin_amdgcn_exp2f(m_run[j] - u) : 1.f;  // 0 from -inf
          const float less = DT != 0 ? 0.f
                                     : alpha * (-KV8_BIAS / KV8_POW) *
                                           (p_run[j] + __shfl_xor(p_run[j], 32, 64));
#pragma unroll
          for (int hb = 0; hb < 4; ++hb)
#pragma unroll
            for (int r = 0; r < 16; ++r)
              o[j][hb][r] = DT == 0 ? fmaf(o[j][hb][r], alpha, less) : o[j][hb][r] * alpha;
          l_run[j] *= alpha;
          p_run[j] = 0.f;
          m_run[j] = up ? u : m_run[j];
        }
        const float mb = m_run[j] == -INFINITY ? 0.f : m_run[j];
        float off = off0 - mb;
        if (__ballot(fabsf(mb) > CA_LARGE)) {  // exponents rounded as the base was
#pragma unroll
          for (int r = 0; r < 16; ++r) s[j][r] = fmaf(s[j][r], a, off0);
          a = 1.f;
          off = -mb;
        }
        if (SPARSE) off = hit ? off : -INFINITY;
        float psum = 0.f;
#pragma unroll
        for (int kh = 0; kh < 2; ++kh)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float w = __builtin_amdgcn_exp2f(fmaf(s[j][kh * 8 + e], a, off));
            psum += w;
            pf[j][kh][e] = T::weight(w);
          }
        if constexpr (DT == 0) p_run[j] = kv8_add8(pf[j][1], kv8_add8(pf[j][0], p_run[j]));
        l_run[j] = fmaf(psum, inv_sv, l_run[j]);
      }
      fold = fold == 1 ? CA_FOLD : fold - 1;
      if constexpr (DT != 0) {
        if (careful && part) {
          int mine[QT];
#pragma unroll
          for (int j = 0; j < QT; ++j) mine[j] = hit ? q_end[j] : 0;
#pragma unroll
          for (int hb = 0; hb < 4; ++hb) {
            f32x16* at[QT];
#pragma unroll
            for (int j = 0; j < QT; ++j) at[j] = &o[j][hb];
            u32x4 two[2] = {vr[2 * hb], vr[2 * hb + 1]};
            ca_values_apart<DT, QT>(two, key0, mine, lane, at);
            vr[2 * hb] = two[0];
            vr[2 * hb + 1] = two[1];
          }
        }
      }
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int hb = 0; hb < 4; ++hb)
#pragma unroll
        for (int kh = 0; kh < 2; ++kh) {
          const vec vf = ca_operand<DT>(vr, hb * 2 + kh);
#pragma unroll
          for (int j = 0; j < QT; ++j) o[j][hb] = T::mma(vf, pf[j][kh], o[j][hb]);
        }
#pragma unroll
      for (int i = 0; i < LD; ++i) vr[i] = *(const u32x4*)(p + TILE / 2 + i * 1024);
    }
    __builtin_amdgcn_s_setprio(0);
  };

  // Where range k of n tiles begins. (Below 2^26 tiles, up to 64 ranges: 32 bits hold the product, and
  // a division of 64 would take as long as a tile.)
  auto share = [&](int n, int k) { return (int)((uint32_t)n * (uint32_t)k / (uint32_t)x.splits); };
  if constexpr (!SPARSE) {
    const int n_tiles = (where.n_keys + 31) >> 5;
    const int t0 = share(n_tiles, split) + kw;
    const int t_end = min(share(n_tiles, split + 1), (any_end + 31) >> 5);
    const int n = (t_end - t0 + KW - 1) / KW;
    first(n, t0);
    stage();
    run(n, t0, 0u, false, [&](int& t, uint32_t&) { t += KW; });
  } else {
    const int m = x.block >> 5;
    const int n_blocks = (int)((uint32_t)(any_end - 1) / (uint32_t)x.block) + 1;
    const int step_e = KW / m, step_r = KW % m;
    // 16 bits: a V that is not finite makes 0 * V of a row that does not see it NaN too, and a K the
    // score of one that does not list it. Rows are looked at afterwards, and only if some are not
    // finite is it all done again with care.
    bool careful = false, staged = false;
    for (;;) {
      for (int w0 = 0; w0 < n_blocks; w0 += CA_WIN) {
        const int n_win = min(CA_WIN, n_blocks - w0);
        if (w0 || careful) ca_lds_barrier();  // the window before has been read
        for (int i = tid; i < n_win; i += THREADS) bits[i] = 0u;
        ca_lds_barrier();
        for (int i = tid; i < n_entries; i += THREADS) {
          int r = entry0_row;
          const int b = i == tid ? entry0 : entry(i, r);
          // (one beyond its row's keys only: its tiles are masked key by key)
          if (b >= w0 && b < w0 + n_win) atomicOr(&bits[b - w0], 1u << r);
        }
        ca_lds_barrier();
        // the window's blocks in order: wave w finds those of its share, then all take their places
        const int part_of = (n_win + 64 * KW - 1) / (64 * KW) * 64, i0 = kw * part_of;
        auto rows_of = [&](int i) { return i + lane < n_win ? bits[min(i + lane, CA_WIN - 1)] : 0u; };
        const uint32_t rows0 = rows_of(i0);
        int found = (int)__popcll(__ballot(rows0 != 0u));
        for (int i = i0 + 64; i < min(n_win, i0 + part_of); i += 64)
          found += (int)__popcll(__ballot(rows_of(i) != 0u));
        if (lane == 0) tally[kw] = found;
        ca_lds_barrier();
        int at = 0, n_list = 0;
#pragma unroll
        for (int w = 0; w < KW; ++w) {
          at += w < kw ? tally[w] : 0;
          n_list += tally[w];
        }
        for (int i = i0; i < min(n_win, i0 + part_of); i += 64) {
          const uint32_t b = i == i0 ? rows0 : rows_of(i);
          const uint64_t hit = __ballot(b != 0u);
          if (b) list[at + __popcll(hit & ((1ull << lane) - 1))] = make_int2(w0 + i + lane, (int)b);
          at += __popcll(hit);
        }
        ca_lds_barrier();
        n_list = __builtin_amdgcn_readfirstlane(n_list);
        // tiles in all (of the last block those that the rows see), and this wave's of this range
        const int last = __builtin_amdgcn_readfirstlane(list[max(n_list - 1, 0)].x);
        const int n = n_list == 0 ? 0 : (n_list - 1) * m + min(m, ((any_end + 31) >> 5) - last * m);
        const int j0 = share(n, split) + kw, j1 = share(n, split + 1);
        int e = j0 / m, r = j0 - e * m;
        auto here = [&](int& t, uint32_t& rows) {
          const int2 b = list[min(e, n_list - 1)];
          t = __builtin_amdgcn_readfirstlane(b.x) * m + r;
          rows = (uint32_t)__builtin_amdgcn_readfirstlane(b.y);
        };
        int t = 0;
        uint32_t rows = 0u;
        if (j0 < j1) here(t, rows);
        first(j1 - j0, t);
        if (!staged) stage();
        staged = true;
        run((j1 - j0 + KW - 1) / KW, t, rows, careful, [&](int& t2, uint32_t& rows2) {
          e += step_e;
          r += step_r;
          if (r >= m) {
            r -= m;
            ++e;
          }
          here(t2, rows2);
        });
      }
      if (DT == 0 || careful) break;
      bool odd = false;
#pragma unroll
      for (int hb = 0; hb < 4; ++hb)
#pragma unroll
        for (int r = 0; r < 16; ++r) odd = odd || !(fabsf(o[0][hb][r]) < INFINITY);
      if (!__syncthreads_or(odd)) break;
      careful = true;
      reset();
    }
  }
#pragma unroll
  for (int j = 0; j < QT; ++j) {
    l_run[j] += __shfl_xor(l_run[j], 32, 64);
    if (DT == 0) {
      if (SPARSE && !heard) {  // (a NaN query's scores of tiles that its row does not see)
        l_run[j] = p_run[j] = 0.f;
#pragma unroll
        for (int hb = 0; hb < 4; ++hb) o[j][hb] = f32x16{};
      }
      p_run[j] += __shfl_xor(p_run[j], 32, 64);
#pragma unroll
      for (int hb = 0; hb < 4; ++hb)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[j][hb][r] = fmaf(o[j][hb][r], KV8_POW, -KV8_BIAS * p_run[j]);
    }
  }

  // The key ways joined and rows out: every wave leaves its O, or half of it, in LDS as 16-byte
  // pieces (query v, piece p at p ^ v: every bank in turn both ways), then threads with eight head
  // dims of a query vector add the ways' and write theirs, all waves taking part.
  constexpr int CH = PIECES / 2;
#pragma unroll
  for (int hf = 0; hf < PASSES; ++hf) {
    __syncthreads();  // the queries, or the first half, have been read
#pragma unroll
    for (int j = 0; j < QT; ++j) {
      f32x4* d = (f32x4*)(smem + (kw * QT + j) * WAVE_O);
#pragma unroll
      for (int b = 0; b < 4 / PASSES; ++b) {
        const f32x16& y = o[j][hf * (4 / PASSES) + b];
#pragma unroll
        for (int r = 0; r < 4; ++r)
          d[(lane & 31) * PIECES + ((b * 8 + 2 * r + (lane >> 5)) ^ (lane & 15))] =
              f32x4{y[4 * r], y[4 * r + 1], y[4 * r + 2], y[4 * r + 3]};
      }
      if (hf == 0 && lane < 32) ml[kw][j * 32 + lane] = make_float2(m_run[j], l_run[j]);
    }
    __syncthreads();
#pragma unroll
    for (int it = 0; it < (NQ * CH + THREADS - 1) / THREADS; ++it) {
      const int v = (it * THREADS + tid) / CH, ch = tid % CH;
      if (v >= NQ || !exists(v)) continue;
      float2 w[KW];
      float m = -INFINITY, l = 0.f;
#pragma unroll
      for (int k = 0; k < KW; ++k) {
        w[k] = ml[k][v];
        m = fmaxf(m, w[k].x);
      }
      f32x4 y0 = f32x4{}, y1 = f32x4{};
#pragma unroll
      for (int k = 0; k < KW; ++k) {
        const f32x4* d =
            (const f32x4*)(smem + (k * QT + (v >> 5)) * WAVE_O) + (v & 31) * PIECES;
        const float f = w[k].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(w[k].x - m);
        y0 += f * d[(2 * ch) ^ (v & 15)];
        y1 += f * d[(2 * ch + 1) ^ (v & 15)];
        l = fmaf(f, w[k].y, l);
      }
      const int64_t rh = (int64_t)row_of(v) * x.Hq + head_of(v);
      const int64_t at = rh * 128 + hf * 64 + ch * 8;
      if (OUT) {
        const float inv = SPARSE && l == 0.f ? 0.f : 1.f / l;  // no key: zeros
        y0 *= inv;
        y1 *= inv;
        if (x.out_bf16) {
          u32x4 z;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            z[e] = (uint32_t)float_to_bf16_bits(y0[2 * e]) |
                   ((uint32_t)float_to_bf16_bits(y0[2 * e + 1]) << 16);
            z[2 + e] = (uint32_t)float_to_bf16_bits(y1[2 * e]) |
                       ((uint32_t)float_to_bf16_bits(y1[2 * e + 1]) << 16);
          }
          *(u32x4*)((uint16_t*)x.out + at) = z;
        } else {
          *(f32x4*)((float*)x.out + at) = y0;
          *(f32x4*)((float*)x.out + at + 4) = y1;
        }
      } else {
        const int64_t n = (int64_t)x.n_rows * x.Hq;
        *(f32x4*)(x.o_part + split * n * 128 + at) = y0;
        *(f32x4*)(x.o_part + split * n * 128 + at + 4) = y1;
        if (hf == 0 && ch == 0) *(float2*)(x.ml_part + (split * n + rh) * 2) = make_float2(m, l);
      }
    }
  }
}

// The key ranges of a (row, head) joined, one wave each: lane (sg, ch) adds head dims 8 ch .. + 8 of
// ranges sg, sg + 4, ..., all of a batch's loads before their use, and the four groups meet by lane
// exchanges. A row without a key gives zeros. Bound by its launch and one round of loads: 32 rows x 16
// heads, 32 ranges (8.5 MB, of L2) 4.0 us, nine rows x 28 heads 2.5; batches of eight no faster.
__global__ __launch_bounds__(128) void part_combine_kernel(const float* __restrict__ o_part,
                                                           const float* __restrict__ ml_part,
                                                           int splits, int64_t n,
                                                           void* __restrict__ out, int bf16) {
  const int64_t id = blockIdx.x * (int64_t)2 + (threadIdx.x >> 6);
  if (id >= n) return;
  const int lane = threadIdx.x & 63, ch = lane & 15, sg = lane >> 4;
  constexpr int SB = 4;
  float m = -INFINITY, l = 0.f;
  f32x4 a0 = f32x4{}, a1 = f32x4{};
  for (int s0 = sg; s0 < splits; s0 += 4 * SB) {
    float2 ml[SB];
    f32x4 p0[SB], p1[SB];
#pragma unroll
    for (int j = 0; j < SB; ++j) {
      const int64_t at = (int64_t)min(s0 + 4 * j, splits - 1) * n + id;
      ml[j] = *(const float2*)(ml_part + at * 2);
      p0[j] = *(const f32x4*)(o_part + at * 128 + 8 * ch);
      p1[j] = *(const f32x4*)(o_part + at * 128 + 8 * ch + 4);
    }
    float mb = m;
#pragma unroll
    for (int j = 0; j < SB; ++j) {
      if (s0 + 4 * j >= splits) {  // (the last range's again: 0 * infinity would be NaN)
        ml[j] = make_float2(-INFINITY, 0.f);
        p0[j] = p1[j] = f32x4{};
      }
      mb = fmaxf(mb, ml[j].x);
    }
    const float sc = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mb);
    a0 *= sc;
    a1 *= sc;
    l *= sc;
#pragma unroll
    for (int j = 0; j < SB; ++j) {
      const float w = ml[j].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[j].x - mb);
      a0 += w * p0[j];
      a1 += w * p1[j];
      l = fmaf(w, ml[j].y, l);
    }
    m = mb;
  }
  const float mm = fmaxf(fmaxf(m, __shfl_xor(m, 16, 64)),
                         fmaxf(__shfl_xor(m, 32, 64), __shfl_xor(m, 48, 64)));
  const float w = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mm);
  a0 *= w;
  a1 *= w;
  l *= w;
#pragma unroll
  for (int o = 16; o < 64; o <<= 1) {
    l += __shfl_xor(l, o, 64);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      a0[e] += __shfl_xor(a0[e], o, 64);
      a1[e] += __shfl_xor(a1[e], o, 64);
    }
  }
  if (sg) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  a0 *= inv;
  a1 *= inv;
  const int64_t at = id * 128 + 8 * ch;
  if (bf16) {
    u32x4 y;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      y[e] = (uint32_t)float_to_bf16_bits(a0[2 * e]) |
             ((uint32_t)float_to_bf16_bits(a0[2 * e + 1]) << 16);
      y[2 + e] = (uint32_t)float_to_bf16_bits(a1[2 * e]) |
                 ((uint32_t)float_to_bf16_bits(a1[2 * e + 1]) << 16);
    }
    *(u32x4*)((uint16_t*)out + at) = y;
  } else {
    *(f32x4*)((float*)out + at) = a0;
    *(f32x4*)((float*)out + at + 4) = a1;
  }
}

}  // namespace

namespace drt {

void part_combine(const float* o_part, const float* ml_part, int splits, int64_t n, void* out,
                  bool bf16, hipStream_t s) {
  hipLaunchKernelGGL(part_combine_kernel, dim3((unsigned)((n + 1) / 2)), dim3(128), 0, s, o_part,
                     ml_part, splits, n, out, (int)bf16);
  DRT_HIP(hipGetLastError());
}

CachePlan plan_attention8(int n_rows, int Hq, int Hkv, int n_keys) {
  CachePlan p;
  const int64_t qtiles = ((int64_t)n_rows * (Hq / Hkv) + 31) / 32;
  const int n_tiles = (int)(((int64_t)n_keys + 31) / 32);
  // Many queries: two query tiles a wave (a tile's codes made operands once for both), four key ways,
  // where that makes work-groups for three in four of the 512 places (2048 rows x 16 heads over 4096
  // keys 79 us, one query tile and eight ways 88; 1000 rows 52 and 44). Otherwise one query tile and
  // eight ways: the least time a work-group (64 rows over 8224 keys: 14 us; four query tiles a
  // work-group and two ways, which read a tile once for all four, 19; over 131072 keys 91 and 95).
  p.groups = (qtiles + 1) / 2;
  p.wide = Hkv * p.groups >= 384;
  if (p.wide) return p;
  p.groups = qtiles;
  // Key ranges by what a call takes, in us: its rounds of 256 work-groups, 2.5 and 0.6 a tile of a
  // wave each; a second launch 4 (one row x 28 heads over 1337 keys: 9.3 a call in one launch, 13.8 in
  // two, in a graph 9.0 and 7.8; over 2048 11.2 and 13.6, 10.8 and 7.9), and the parts, written and
  // read.
  const int64_t wgs = Hkv * qtiles;
  const float part_us = (float)n_rows * (float)Hq * (2 * 130 * 4 / 4.5e6f);
  float best = INFINITY;
  const int most = std::min(64, (n_tiles + 7) / 8);
  for (int s = 1; s <= most; ++s) {
    const float rounds = (float)((wgs * s + 255) / 256);
    const float tiles = (float)((n_tiles + 8 * s - 1) / (8 * s));
    const float us = rounds * (2.5f + 0.6f * tiles) + (s > 1 ? 4.f + part_us * (float)s : 0.f);
    if (us < best) {
      best = us;
      p.splits = s;
    }
  }
  return p;
}

CachePlan plan_sparse(int n_rows, int Hq, int Hkv, int count, int block) {
  CachePlan p;
  const int G = Hq / Hkv, rows = 32 / std::min(G, 32), heads = (G + 31) / 32;
  p.groups = ((int64_t)n_rows + rows - 1) / rows;
  // Few work-groups: as many key ranges as give every CU one, of four of a list's tiles at least (9
  // rows x 28 heads, 16 blocks of 64: 12.4 us; of eight 13.3, of 16 16.2)
  const int64_t wgs = p.groups * Hkv * heads, tiles = (int64_t)count * (block / 32);
  // More than the CUs: four waves a work-group, two of which share a CU (1000 rows x 16 heads, 16
  // blocks of 64 of 32768 keys: 28.7 us; eight waves, in two rounds, 36.5).
  p.wide = wgs > 256;
  // (32 tiles of a tile's rows at most cost less than the second launch: one row x 28 heads, 16 blocks
  // of 64 10.5 us a call, with key ranges 14.1; in a graph 10.1 and 9.2.)
  p.splits = p.wide || tiles * std::min(n_rows, rows) <= 32
                 ? 1
                 : (int)std::max<int64_t>(1, std::min<int64_t>({256 / wgs, (tiles + 3) / 4, 64}));
  return p;
}

size_t cache_part_bytes(const CachePlan& p, int n_rows, int Hq) {
  return p.splits == 1 ? 0 : (size_t)p.splits * n_rows * Hq * 130 * 4;
}

static CaArgs args_of(KvType type, const void* q, bool q_bf16, const void* kv_layer,
                      int64_t kv_head_stride, const float* scales, int n_rows, int Hq, int Hkv,
                      const AttnWhere& where, const CachePlan& p, float* part, void* out,
                      bool out_bf16) {
  CaArgs a{};
  a.q = (const uint16_t*)q;
  a.kv = (const uint8_t*)kv_layer;
  a.head_stride = type == KvType::I8 ? kv_head_stride : 2 * kv_head_stride;
  a.scales = scales;
  a.q_bf16 = q_bf16;
  a.n_rows = n_rows;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.splits = p.splits;
  a.block = 32;
  a.c = 1.44269504088896340736f / sqrtf(128.0f) * (type == KvType::I8 ? KV8_POW : 1.f);
  a.where = where;
  a.out = out;
  a.o_part = part;
  a.ml_part = part ? part + (size_t)p.splits * n_rows * Hq * 128 : nullptr;
  a.out_bf16 = out_bf16;
  return a;
}

#define DRT_CA1(DT, QT, KW, OUT, SPARSE) \
  hipLaunchKernelGGL((cache_attn_kernel<DT, QT, KW, OUT, SPARSE>), grid, dim3(64 * KW), 0, s, a)
#define DRT_CA(DT, QT, KW, SPARSE)                                                                \
  do {                                                                                            \
    if (p.splits == 1) DRT_CA1(DT, QT, KW, true, SPARSE);                                         \
    else DRT_CA1(DT, QT, KW, false, SPARSE);                                                      \
  } while (0)

void attention8(const void* q, bool q_bf16, const void* kv_layer, int64_t kv_head_stride,
                const float* scales, int n_rows, int Hq, int Hkv, const AttnWhere& where,
                const CachePlan& p, float* part, void* out, bool out_bf16, hipStream_t s) {
  const CaArgs a = args_of(KvType::I8, q, q_bf16, kv_layer, kv_head_stride, scales, n_rows, Hq, Hkv,
                           where, p, part, out, out_bf16);
  const dim3 grid((unsigned)(p.splits * Hkv), (unsigned)p.groups);
  if (p.wide) DRT_CA1(0, 2, 4, true, false);
  else DRT_CA(0, 1, 8, false);
  DRT_HIP(hipGetLastError());
  if (p.splits > 1) part_combine(part, a.ml_part, p.splits, (int64_t)n_rows * Hq, out, out_bf16, s);
}

void sparse_attention(KvType type, const void* q, bool q_bf16, const void* kv_layer,
                      int64_t kv_head_stride, const float* scales, int n_rows, int Hq, int Hkv,
                      const AttnWhere& where, const int32_t* blocks, int count, int block,
                      const CachePlan& p, float* part, void* out, bool out_bf16, hipStream_t s) {
  CaArgs a = args_of(type, q, q_bf16, kv_layer, kv_head_stride, scales, n_rows, Hq, Hkv, where, p,
                     part, out, out_bf16);
  a.blocks = blocks;
  a.count = count;
  a.block = block;
  const dim3 grid((unsigned)(p.splits * Hkv), (unsigned)p.groups, (unsigned)((Hq / Hkv + 31) / 32));
#define DRT_SP(DT)                                                                                \
  do { if (p.wide) DRT_CA1(DT, 1, 4, true, true); else DRT_CA(DT, 1, 8, true); } while (0)
  if (type == KvType::I8) DRT_SP(0);
  else if (type == KvType::F16) DRT_SP(1);
  else DRT_SP(2);
#undef DRT_SP
  DRT_HIP(hipGetLastError());
  if (p.splits > 1) part_combine(part, a.ml_part, p.splits, (int64_t)n_rows * Hq, out, out_bf16, s);
}
#undef DRT_CA
#undef DRT_CA1

}  // namespace drt
