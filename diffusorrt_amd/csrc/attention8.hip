// GQA attention over the 8-bit cache (kv8.h) for gfx950, decode blocks and prompts alike.
//
// Queries of one K/V head are flattened to query vectors qv = row * G + gi (G = Hq / Hkv, head
// = kvh * G + gi) in tiles of 32, keys come in tiles of 32, and a wave computes S^T = K Q^T and
// O^T += V^T P^T as 32x32x16 fp16 products, as the attention over a 16-bit cache does.
// A wave loads a tile's codes (8 KiB, 16 bytes a lane and load) straight into registers and makes
// fp16 operands of them there: no staging, no barrier in the loop. A tile's K registers are loaded
// anew as soon as its scores are done, its V registers after its products.
//
// Scales. With K = 2^a k and V = 2^b v for a tile (k, v the codes), the base-2 exponent of a
// weighted value is u = (k . q) * 2^a * c, c = log2(e) / sqrt(128), and
//   o = sum p v 2^b / sum p,  p = 2^u.
// The wave keeps p' = 2^(u + b - base): its sum against v needs no factor, and the normaliser
// adds 2^-b of a tile's sum of p'. So a tile's scales cost a few operations a lane, not one a
// score, and p' is largest where a tile's part of the result is: fp16 holds it to 2^-11 of its value
// wherever it counts. The running base is raised when a tile's largest u + b exceeds it by more than
// 8 (p' <= 2^8); any base gives the same quotient. p' is the one rounding ahead of the sums
// (fp16, the product's operand type); scores, base, normaliser and O are fp32. The normaliser adds p'
// before that rounding: weights on a tile of tiny values may vanish in fp16 beside others, not in it.
// Queries: fp16 as they are; bf16 ones are scaled by a power of two per query vector to a
// largest magnitude in [1, 2) (exact: fp16 has three bits more; elements below 2^-14 of the
// vector's largest lose some, at most 2^-25 of that largest).
#include "kv8.h"
#include "launch.h"

#include <cmath>

using drt::AttnWhere;

namespace {

constexpr float A8_RESCALE_LOG2 = 8.f;
// A base beyond this is rounded by more than 2^-4: p' = 2^(fma(s, a, off - base)) would then be off by
// that, without bound; with the exponent rounded before the base is taken off it never passes 2^8.
constexpr float A8_LARGE = 1048576.f;
// The bytes' 128 leaves O with the running sum of weights, at the latest after so many tiles: its
// share of the sum in fp32, which costs O precision, stays that of 1024 keys.
constexpr int A8_FOLD = 32;
constexpr int A8_QROW = 136;  // fp16 elements per query vector in LDS (+ 16 bytes)

DRT_DEV float a8_max_xor32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

struct A8Out {
  void* out;       // [rows][Hq * 128], bf16 or fp32
  float* o_part;   // [splits][rows][Hq][128] (not OUT)
  float* ml_part;  // [splits][rows][Hq][2]
  int bf16;
};

// QW waves over query tiles, KW waves over keys (wave kw of a query tile takes key
// tiles kw, kw + KW, ...; their parts meet in LDS at the end). OUT: one key range, the
// result itself; otherwise a part for the combine.
template <int QT, int QW, int KW, bool OUT>
__global__ __launch_bounds__(64 * QW * KW, 2) void attn8_kernel(
    const uint16_t* __restrict__ q, const uint8_t* __restrict__ kv, int64_t kv_head_stride,
    const float* __restrict__ scales, int q_bf16, int n_rows, int Hq, int Hkv,
    int tiles_per_split, float c, const AttnWhere where, const A8Out ao) {
  constexpr int NW = QW * KW, THREADS = 64 * NW, NQ = 32 * QT * QW;
  constexpr int O_BYTES = QT * 16384;  // a wave's O
  constexpr int Q_BYTES = NQ * A8_QROW * 2, OUT_BYTES = QW * 8192;
  constexpr int ML_BYTES = QT * 512, MRG = KW > 1 ? (NW / 2) * (O_BYTES + ML_BYTES) : 0;
  constexpr int LDS = Q_BYTES > MRG ? (Q_BYTES > OUT_BYTES ? Q_BYTES : OUT_BYTES)
                                    : (MRG > OUT_BYTES ? MRG : OUT_BYTES);
  __shared__ __align__(16) char smem[LDS];
  __shared__ float2 qinfo[NQ];  // c * 2^24 times a query vector's power of two; -128 * 2^-24 its sum
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int qw = wave % QW, kw = wave / QW;
  const int G = Hq / Hkv, n_qv = n_rows * G;
  const int kvh = blockIdx.x % Hkv, split = blockIdx.x / Hkv;
  // the work-group's first query tile: the last rows, which see the most keys, start first
  const int qt0 = ((int)gridDim.y - 1 - (int)blockIdx.y) * (QW * QT);
  const int n_tiles = (where.n_keys + 31) >> 5;

  // queries into LDS, 16 threads (eight elements each) a query vector
#pragma unroll
  for (int it0 = 0; it0 < NQ * 16; it0 += THREADS) {
    const int it = it0 + threadIdx.x;
    const int v = it >> 4, ch = it & 15, qv = qt0 * 32 + v;
    u32x4 raw = u32x4{0u, 0u, 0u, 0u};
    if (qv < n_qv) {
      const int row = qv / G, head = kvh * G + (qv - row * G);
      raw = *(const u32x4*)(q + ((int64_t)row * Hq + head) * 128 + ch * 8);
    }
    float pw = 1.f;
    if (q_bf16) {
      uint32_t most = 0u;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        most = max(most, max((raw[e] << 16) & 0x7fffffffu, raw[e] & 0x7fff0000u));
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, o, 64));
      const int x = most ? min(max((int)(most >> 23) - 127, -126), 126) : 0;
      pw = __uint_as_float((uint32_t)(127 + x) << 23);
      const float inv = __uint_as_float((uint32_t)(127 - x) << 23);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        raw[e] = pack_half2((_Float16)(__uint_as_float(raw[e] << 16) * inv),
                            (_Float16)(__uint_as_float(raw[e] & 0xffff0000u) * inv));
    }
    *(u32x4*)(smem + (v * A8_QROW + ch * 8) * 2) = raw;
    float sum = kv8_add8(__builtin_bit_cast(f16x8, raw), 0.f);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if (ch == 0) qinfo[v] = make_float2(c * pw, -KV8_BIAS / KV8_POW * sum);
  }
  __syncthreads();

  const _Float16* ql = (const _Float16*)smem + (qw * QT * 32 + (lane & 31)) * A8_QROW + 8 * (lane >> 5);
  constexpr bool HOLD = QT == 1;  // the queries' operands in registers
  f16x8 qr[HOLD ? 8 : 1];
  if (HOLD) {
#pragma unroll
    for (int i = 0; i < 8; ++i) qr[HOLD ? i : 0] = *(const f16x8*)(ql + 16 * i);
  }
  const int wt0 = qt0 + qw * QT;  // the wave's first query tile
  int q_end[QT];
  float cq[QT], nq[QT], m_run[QT], l_run[QT], p_run[QT];
  f32x16 o[QT][4];
#pragma unroll
  for (int j = 0; j < QT; ++j) {
    q_end[j] = key_end_of(min((wt0 + j) * 32 + (lane & 31), n_qv - 1) / G, where);
    const float2 x = qinfo[(qw * QT + j) * 32 + (lane & 31)];
    cq[j] = x.x;
    nq[j] = x.y;
    m_run[j] = -INFINITY;
    l_run[j] = p_run[j] = 0.f;
#pragma unroll
    for (int hb = 0; hb < 4; ++hb) o[j][hb] = f32x16{};
  }
  // (ends never fall from row to row) keys every row of the wave sees, and any of them
  const int wave_full = key_end_of(min(wt0 * 32, n_qv - 1) / G, where);
  const int wave_end = key_end_of(min((wt0 + QT) * 32 - 1, n_qv - 1) / G, where);
  const bool idle = wt0 * 32 >= n_qv;
  const int t_begin = split * tiles_per_split;
  const int t_end = idle ? 0 : min(min(n_tiles, t_begin + tiles_per_split), (wave_end + 31) >> 5);

  const uint8_t* base = kv + kvh * kv_head_stride + lane * 16;
  const float2* sc = (const float2*)(scales + kvh * (kv_head_stride / KV8_TILE) * 2);
  u32x4 kr[4], vr[4];
  float2 st = make_float2(1.f, 1.f);
  int t = t_begin + kw, fold = A8_FOLD;
  if (t < t_end) {
    const uint8_t* p = base + (int64_t)t * KV8_TILE;
#pragma unroll
    for (int i = 0; i < 4; ++i) kr[i] = *(const u32x4*)(p + i * 1024);
#pragma unroll
    for (int i = 0; i < 4; ++i) vr[i] = *(const u32x4*)(p + 4096 + i * 1024);
    st = sc[t];
  }
  for (; t < t_end; t += KW) {
    const int key0 = t * 32;
    const float sk = st.x, sv = st.y;
    const int tn = min(t + KW, t_end - 1);  // (the last tile's own again: loaded, not used)
    const uint8_t* p = base + (int64_t)tn * KV8_TILE;
    f32x16 s[QT];
#pragma unroll
    for (int j = 0; j < QT; ++j) s[j] = f32x16{};
    if (!HOLD) asm volatile("" ::: "memory");  // (read the queries here, tile by tile)
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const f16x8 kf = kv8_to_f16(kr[i >> 1][2 * (i & 1)], kr[i >> 1][2 * (i & 1) + 1]);
#pragma unroll
      for (int j = 0; j < QT; ++j)
        s[j] = mfma_f16(kf, HOLD ? qr[HOLD ? i : 0] : *(const f16x8*)(ql + j * 32 * A8_QROW + 16 * i),
                        s[j]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) kr[i] = *(const u32x4*)(p + i * 1024);
    __builtin_amdgcn_s_setprio(0);
    asm volatile("" ::: "memory");  // (a scalar load among the reads of LDS would be waited for with them)
    st = sc[tn];
    const bool bad = !(sk + sv < INFINITY);  // a tile that is NaN: so is every row that sees it
    if (key0 + 32 > wave_full || bad) {
#pragma unroll
      for (int j = 0; j < QT; ++j) {
        if (bad && key0 < q_end[j]) {
          l_run[j] = NAN;
          m_run[j] = m_run[j] == -INFINITY ? 0.f : m_run[j];
        }
        const int end = bad ? 0 : q_end[j];
#pragma unroll
        for (int r = 0; r < 16; ++r) s[j][r] = key0 + mfma_row(r, lane) < end ? s[j][r] : -INFINITY;
      }
    }
    const float lb = bad ? 0.f : (float)((int)(__float_as_uint(sv) >> 23) - 127);  // sv = 2^lb
    const float inv_sv = bad ? 0.f : __uint_as_float((254u << 23) - __float_as_uint(sv));
    f16x8 pf[QT][2];
#pragma unroll
    for (int j = 0; j < QT; ++j) {
      // (within the finite numbers above zero whatever the powers of two: no 0 * inf)
      float a = bad ? 1.f : __builtin_amdgcn_fmed3f(sk * cq[j], 1e-37f, 3e38f);
      float tmax = s[j][0];
#pragma unroll
      for (int r = 1; r < 16; ++r) tmax = fmaxf(tmax, s[j][r]);
      const float off0 = fmaf(nq[j], a, lb);
      const float u = fmaf(a8_max_xor32(tmax), a, off0);  // -inf: no visible key in the tile
      const bool up = u > m_run[j] + A8_RESCALE_LOG2;
      if (__ballot(up) || fold == 1) {
        const float alpha = up ? __builtin_amdgcn_exp2f(m_run[j] - u) : 1.f;  // 0 from -inf
        const float less = alpha * (-KV8_BIAS / KV8_POW) * (p_run[j] + __shfl_xor(p_run[j], 32, 64));
#pragma unroll
        for (int hb = 0; hb < 4; ++hb)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[j][hb][r] = fmaf(o[j][hb][r], alpha, less);
        l_run[j] *= alpha;
        p_run[j] = 0.f;
        m_run[j] = up ? u : m_run[j];
      }
      const float mb = m_run[j] == -INFINITY ? 0.f : m_run[j];
      float off = off0 - mb;
      if (__ballot(fabsf(mb) > A8_LARGE)) {  // exponents rounded as the base was
#pragma unroll
        for (int r = 0; r < 16; ++r) s[j][r] = fmaf(s[j][r], a, off0);
        a = 1.f;
        off = -mb;
      }
      float psum = 0.f;
#pragma unroll
      for (int kh = 0; kh < 2; ++kh)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = __builtin_amdgcn_exp2f(fmaf(s[j][kh * 8 + e], a, off));
          psum += x;
          pf[j][kh][e] = (_Float16)x;
        }
      p_run[j] = kv8_add8(pf[j][1], kv8_add8(pf[j][0], p_run[j]));
      l_run[j] = fmaf(psum, inv_sv, l_run[j]);
    }
    fold = fold == 1 ? A8_FOLD : fold - 1;
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int hb = 0; hb < 4; ++hb)
#pragma unroll
      for (int kh = 0; kh < 2; ++kh) {
        const f16x8 vf = kv8_to_f16(vr[hb][2 * kh], vr[hb][2 * kh + 1]);
#pragma unroll
        for (int j = 0; j < QT; ++j) o[j][hb] = mfma_f16(vf, pf[j][kh], o[j][hb]);
      }
#pragma unroll
    for (int i = 0; i < 4; ++i) vr[i] = *(const u32x4*)(p + 4096 + i * 1024);
  }
#pragma unroll
  for (int j = 0; j < QT; ++j) {
    l_run[j] += __shfl_xor(l_run[j], 32, 64);
    p_run[j] += __shfl_xor(p_run[j], 32, 64);
#pragma unroll
    for (int hb = 0; hb < 4; ++hb)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[j][hb][r] = fmaf(o[j][hb][r], KV8_POW, -KV8_BIAS * p_run[j]);
  }

  // the key ways of a wave's queries in pairs
  if (KW > 1) {
#pragma unroll
    for (int half = KW / 2; half > 0; half >>= 1) {
      __syncthreads();  // the queries, or the round before, have been read
      if (kw >= half && kw < 2 * half) {
        char* d = smem + ((kw - half) * QW + qw) * (O_BYTES + ML_BYTES);
#pragma unroll
        for (int j = 0; j < QT; ++j) {
#pragma unroll
          for (int hb = 0; hb < 4; ++hb)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              ((f32x4*)d)[(j * 16 + hb * 4 + r) * 64 + lane] =
                  f32x4{o[j][hb][4 * r], o[j][hb][4 * r + 1], o[j][hb][4 * r + 2], o[j][hb][4 * r + 3]};
          ((float2*)(d + O_BYTES))[j * 64 + lane] = make_float2(m_run[j], l_run[j]);
        }
      }
      __syncthreads();
      if (kw < half) {
        const char* d = smem + (kw * QW + qw) * (O_BYTES + ML_BYTES);
#pragma unroll
        for (int j = 0; j < QT; ++j) {
          const float2 ml = ((const float2*)(d + O_BYTES))[j * 64 + lane];
          const float mm = fmaxf(m_run[j], ml.x);
          const float w0 = m_run[j] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run[j] - mm);
          const float w1 = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - mm);
#pragma unroll
          for (int hb = 0; hb < 4; ++hb)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const f32x4 y = ((const f32x4*)d)[(j * 16 + hb * 4 + r) * 64 + lane];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                o[j][hb][4 * r + e] = fmaf(w1, y[e], w0 * o[j][hb][4 * r + e]);
            }
          l_run[j] = fmaf(w1, ml.y, w0 * l_run[j]);
          m_run[j] = mm;
        }
      }
    }
  }
  __syncthreads();
  if (kw > 0) return;  // (no barrier follows)
  // Rows out: half a query tile's O^T (64 head dims) at a time through 8 KiB of the wave's own, as 16-byte
  // pieces (query v, piece p at p ^ v: every bank in turn both ways), eight lanes a query vector.
  f32x4* ot = (f32x4*)(smem + qw * 8192);
#pragma unroll
  for (int jh = 0; jh < 2 * QT; ++jh) {
    const int j = jh >> 1, hf = jh & 1;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        ot[(lane & 31) * 16 + ((b * 8 + 2 * r + (lane >> 5)) ^ (lane & 15))] =
            f32x4{o[j][2 * hf + b][4 * r], o[j][2 * hf + b][4 * r + 1], o[j][2 * hf + b][4 * r + 2],
                  o[j][2 * hf + b][4 * r + 3]};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int v = (lane >> 3) + 8 * i, ch = lane & 7, qv = (wt0 + j) * 32 + v;
      const float m = __shfl(m_run[j], v, 64), l = __shfl(l_run[j], v, 64);
      f32x4 y0 = ot[v * 16 + ((2 * ch) ^ (v & 15))], y1 = ot[v * 16 + ((2 * ch + 1) ^ (v & 15))];
      if (qv >= n_qv) continue;
      const int row = qv / G;
      const int64_t rh = (int64_t)row * Hq + kvh * G + (qv - row * G);
      const int64_t at = rh * 128 + hf * 64 + ch * 8;
      if (OUT) {
        const float inv = 1.f / l;
        y0 *= inv;
        y1 *= inv;
        if (ao.bf16) {
          u32x4 w;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            w[e] = (uint32_t)float_to_bf16_bits(y0[2 * e]) |
                   ((uint32_t)float_to_bf16_bits(y0[2 * e + 1]) << 16);
            w[2 + e] = (uint32_t)float_to_bf16_bits(y1[2 * e]) |
                       ((uint32_t)float_to_bf16_bits(y1[2 * e + 1]) << 16);
          }
          *(u32x4*)((uint16_t*)ao.out + at) = w;
        } else {
          *(f32x4*)((float*)ao.out + at) = y0;
          *(f32x4*)((float*)ao.out + at + 4) = y1;
        }
      } else {
        const int64_t n = (int64_t)n_rows * Hq;
        *(f32x4*)(ao.o_part + split * n * 128 + at) = y0;
        *(f32x4*)(ao.o_part + split * n * 128 + at + 4) = y1;
        if (hf == 0 && ch == 0) *(float2*)(ao.ml_part + (split * n + rh) * 2) = make_float2(m, l);
      }
    }
  }
}

// The key ranges of a (row, head) joined, one wave each: lane (sg, ch) adds head dims 8 ch .. + 8 of ranges sg,
// sg + 4, ..., all of a batch's loads before their use, and the four groups meet by lane exchanges.
// A row without a key gives zeros.
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
      if (s0 + 4 * j >= splits) ml[j] = make_float2(-INFINITY, 0.f);
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
  const float mm = fmaxf(fmaxf(m, __shfl_xor(m, 16, 64)), fmaxf(__shfl_xor(m, 32, 64), __shfl_xor(m, 48, 64)));
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
      y[e] = (uint32_t)float_to_bf16_bits(a0[2 * e]) | ((uint32_t)float_to_bf16_bits(a0[2 * e + 1]) << 16);
      y[2 + e] =
          (uint32_t)float_to_bf16_bits(a1[2 * e]) | ((uint32_t)float_to_bf16_bits(a1[2 * e + 1]) << 16);
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

Attn8Plan plan_attention8(int n_rows, int Hq, int Hkv, int n_keys) {
  Attn8Plan p;
  const int qtiles = (int)(((int64_t)n_rows * (Hq / Hkv) + 31) / 32);
  // Many queries: two query tiles a wave (a tile's codes made operands once for both), four key
  // ways in a work-group of their own, so that work-groups are as many as can be (2048 rows x 16
  // heads over 4096 keys: 72 us; two and one key ways, which need key ranges to fill the chip:
  // 101, 110). Few: eight waves over the one, two or four query tiles.
  p.wide = qtiles > 4;
  p.qw = p.wide || qtiles == 1 ? 1 : qtiles == 2 ? 2 : 4;
  p.kw = p.wide ? 4 : 8 / p.qw;
  const int per = p.wide ? 2 : p.qw;  // query tiles of a work-group
  p.qgroups = (qtiles + per - 1) / per;
  const int n_tiles = (n_keys + 31) / 32;
  const int64_t wgs = (int64_t)Hkv * p.qgroups;
  const int target = p.wide ? 512 : 256;
  int64_t splits = std::max<int64_t>(1, target / wgs);
  splits = std::min<int64_t>({splits, (n_tiles + p.kw - 1) / p.kw, 64});
  p.tiles_per_split = (int)((n_tiles + splits - 1) / splits);
  p.splits = (n_tiles + p.tiles_per_split - 1) / p.tiles_per_split;
  return p;
}

size_t attention8_part_bytes(const Attn8Plan& p, int n_rows, int Hq) {
  return p.splits == 1 ? 0 : (size_t)p.splits * n_rows * Hq * 130 * 4;
}

void attention8(const void* q, bool q_bf16, const void* kv_layer, int64_t kv_head_stride,
                const float* scales, int n_rows, int Hq, int Hkv, const AttnWhere& where,
                const Attn8Plan& p, float* part, void* out, bool out_bf16, hipStream_t s) {
  const float c = 1.44269504088896340736f / sqrtf(128.0f) * KV8_POW;
  float* ml = part ? part + (size_t)p.splits * n_rows * Hq * 128 : nullptr;
  const A8Out ao{out, part, ml, out_bf16};
  const dim3 grid((unsigned)(p.splits * Hkv), (unsigned)p.qgroups);
#define DRT_A8(QT, QW, KW, OUT)                                                                   \
  hipLaunchKernelGGL((attn8_kernel<QT, QW, KW, OUT>), grid, dim3(64 * QW * KW), 0, s,             \
                     (const uint16_t*)q, (const uint8_t*)kv_layer, kv_head_stride, scales,    \
                     (int)q_bf16, n_rows, Hq, Hkv, p.tiles_per_split, c, where, ao)
#define DRT_A8O(QT, QW, KW)                                                                       \
  do { if (p.splits == 1) DRT_A8(QT, QW, KW, true); else DRT_A8(QT, QW, KW, false); } while (0)
  if (p.wide) DRT_A8O(2, 1, 4);
  else if (p.qw == 1) DRT_A8O(1, 1, 8);
  else if (p.qw == 2) DRT_A8O(1, 2, 4);
  else DRT_A8O(1, 4, 2);
#undef DRT_A8O
#undef DRT_A8
  DRT_HIP(hipGetLastError());
  if (p.splits > 1) part_combine(part, ml, p.splits, (int64_t)n_rows * Hq, out, out_bf16, s);
}

}  // namespace drt
