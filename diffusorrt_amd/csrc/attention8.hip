// GQA attention over the 8-bit cache (kv8.h) for gfx950, decode blocks and prompts alike.
//
// Queries of one K/V head are flattened to query vectors qv = row * G + gi (G = Hq / Hkv, head
// = kvh * G + gi) in tiles of 32, keys come in tiles of 32, and a wave computes S^T = K Q^T and
// O^T += V^T P^T as 32x32x16 fp16 products, as the attention over a 16-bit cache does.
// A wave loads a tile's codes (8 KiB, 16 bytes a lane and load) straight into registers, a tile ahead,
// and turns them into exact fp16 whole numbers there: no staging, no barrier in the loop.
//
// Scales. With K = 2^a k and V = 2^b v for a tile (k, v the codes), the base-2 exponent of a
// weighted value is u = (k . q) * 2^a * c, c = log2(e) / sqrt(128), and
//   o = sum p v 2^b / sum p,  p = 2^u.
// The wave keeps p' = 2^(u + b - base): its sum against v needs no factor, and the normaliser
// adds 2^-b of a tile's sum of p'. So a tile's scales cost one product and one add a tile and lane,
// and p' is largest where a tile's part of the result is: fp16 holds it to 2^-12 of its value wherever it
// counts. The running base is raised when a tile's largest u + b exceeds it by more than
// 8 (p' <= 2^8); any base gives the same quotient. p' is the one rounding ahead of the sums
// (fp16, the product's operand type); scores, base, normaliser and O are fp32.
// Queries: fp16 as they are; bf16 ones are scaled by a power of two per query vector to a
// largest magnitude in [1, 2) (exact: fp16 has three bits more; elements below 2^-14 of the
// vector's largest lose some, at most 2^-25 of that largest).
#include "kv8.h"
#include "launch.h"

#include <cmath>

using drt::AttnWhere;

namespace {

constexpr float A8_RESCALE_LOG2 = 8.f;
// A base beyond this is rounded by more than 2^-4: p' = 2^(fma(s, a, -base)) would then be off by
// that, without bound; with the product rounded first it never passes 2^8.
constexpr float A8_LARGE = 1048576.f;
constexpr int A8_QROW = 136;  // fp16 elements per query vector in LDS (+ 16 bytes)

DRT_DEV float a8_max_xor32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

struct A8Out {
  void* out;      // [rows][Hq * 128], bf16 or fp32
  float* o_part;  // [splits][Hkv][n_qv][128] (not OUT)
  float* ml_part; // [splits][Hkv][n_qv][2]
  int bf16;
};

// QT query tiles a wave, QW waves over query tiles, KW waves over keys (wave kw of a query tile takes key
// tiles kw, kw + KW, ...; their parts meet in LDS at the end). OUT: one key range, the
// result itself; otherwise a part for attn_combine.
template <int QT, int QW, int KW, bool OUT>
__global__ __launch_bounds__(64 * QW * KW, 2) void attn8_kernel(
    const uint16_t* __restrict__ q, const uint8_t* __restrict__ kv, int64_t kv_head_stride,
    const float* __restrict__ scales, int q_bf16, int n_rows, int Hq, int Hkv,
    int tiles_per_split, float c, const AttnWhere where, const A8Out ao) {
  constexpr int NW = QW * KW, THREADS = 64 * NW, NQ = 32 * QT * QW;
  constexpr int Q_BYTES = NQ * A8_QROW * 2, O_BYTES = 16384;  // O: a query tile's, one wave
  constexpr int MRG = KW > 1 ? (NW / 2) * (O_BYTES + 512) : 0;
  constexpr int OUT_BYTES = QW * O_BYTES;
  constexpr int LDS = Q_BYTES > MRG ? (Q_BYTES > OUT_BYTES ? Q_BYTES : OUT_BYTES)
                                    : (MRG > OUT_BYTES ? MRG : OUT_BYTES);
  static_assert(KW == 1 || QT == 1, "the key ways' merge holds one query tile a wave");
  __shared__ __align__(16) char smem[LDS];
  __shared__ float qpow[NQ];  // c times a query vector's power of two
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int qw = wave % QW, kw = wave / QW;
  const int G = Hq / Hkv, n_qv = n_rows * G;
  const int kvh = blockIdx.x % Hkv, split = blockIdx.x / Hkv;
  const int qt0 = blockIdx.y * (QW * QT);  // the work-group's first query tile
  const int n_tiles = (where.n_keys + 31) >> 5;

  // queries into LDS, 16 threads (eight elements each) a query vector
  for (int it = threadIdx.x; it < NQ * 16; it += THREADS) {
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
    if (ch == 0) qpow[v] = c * pw;
  }
  __syncthreads();

  const _Float16* ql = (const _Float16*)smem + (qw * QT * 32 + (lane & 31)) * A8_QROW + 8 * (lane >> 5);
  f16x8 qr[QT == 1 ? 8 : 1];  // one query tile: its operands stay in registers
  if (QT == 1) {
#pragma unroll
    for (int i = 0; i < 8; ++i) qr[QT == 1 ? i : 0] = *(const f16x8*)(ql + 16 * i);
  }
  int q_end[QT];
  float cq[QT], m_run[QT], l_run[QT];
  f32x16 o[QT][4];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int v = (qw * QT + t) * 32 + (lane & 31), qv = qt0 * 32 + v;
    q_end[t] = key_end_of(min(qv, n_qv - 1) / G, where);
    cq[t] = qpow[v];
    m_run[t] = -INFINITY;
    l_run[t] = 0.f;
#pragma unroll
    for (int hb = 0; hb < 4; ++hb) o[t][hb] = f32x16{};
  }
  // (ends never fall from row to row) keys every row of the wave sees, and any of them
  const int first_qv = min((qt0 + qw * QT) * 32, n_qv - 1);
  const int last_qv = min((qt0 + qw * QT + QT) * 32 - 1, n_qv - 1);
  const int wave_full = key_end_of(first_qv / G, where), wave_end = key_end_of(last_qv / G, where);
  const bool idle = (qt0 + qw * QT) * 32 >= n_qv;
  const int t_begin = split * tiles_per_split;
  const int t_end = idle ? 0 : min(min(n_tiles, t_begin + tiles_per_split), (wave_end + 31) >> 5);

  const uint8_t* base = kv + kvh * kv_head_stride + lane * 16;
  const float2* sc = (const float2*)(scales + kvh * (kv_head_stride / KV8_TILE) * 2);
  struct Tile {
    u32x4 k[4], v[4];
    float2 s;
  };
  auto load = [&](Tile& x, int t) {
    const uint8_t* p = base + (int64_t)t * KV8_TILE;
#pragma unroll
    for (int i = 0; i < 4; ++i) x.k[i] = *(const u32x4*)(p + i * 1024);
#pragma unroll
    for (int i = 0; i < 4; ++i) x.v[i] = *(const u32x4*)(p + 4096 + i * 1024);
    x.s = sc[t];
  };
  auto compute = [&](const Tile& x, int t) {
    const int key0 = t * 32;
    const float sk = x.s.x, sv = x.s.y;
    if (!(sk + sv < INFINITY)) {  // a tile that is NaN: so is every row that sees it
#pragma unroll
      for (int i = 0; i < QT; ++i)
        if (key0 < q_end[i]) {
          l_run[i] = NAN;
          if (m_run[i] == -INFINITY) m_run[i] = 0.f;
        }
      return;
    }
    const float lb = (float)((int)(__float_as_uint(sv) >> 23) - 127);  // sv = 2^lb
    const float inv_sv = __uint_as_float((254u << 23) - __float_as_uint(sv));
    f32x16 s[QT];
#pragma unroll
    for (int i = 0; i < QT; ++i) s[i] = f32x16{};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const f16x8 kf = kv8_to_f16(x.k[i >> 1][2 * (i & 1)], x.k[i >> 1][2 * (i & 1) + 1]);
#pragma unroll
      for (int j = 0; j < QT; ++j)
        s[j] = mfma_f16(kf, QT == 1 ? qr[QT == 1 ? i : 0] : *(const f16x8*)(ql + j * 32 * A8_QROW + 16 * i),
                        s[j]);
    }
    if (key0 + 32 > wave_full) {
#pragma unroll
      for (int j = 0; j < QT; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          s[j][r] = key0 + mfma_row(r, lane) < q_end[j] ? s[j][r] : -INFINITY;
    }
    f16x8 pf[QT][2];
#pragma unroll
    for (int j = 0; j < QT; ++j) {
      float tmax = s[j][0];
#pragma unroll
      for (int r = 1; r < 16; ++r) tmax = fmaxf(tmax, s[j][r]);
      // (above zero even where both powers of two are the least: no 0 * inf)
      float a = fmaxf(sk * cq[j], 1e-37f);
      const float u = fmaf(a8_max_xor32(tmax), a, lb);  // -inf: no visible key in the tile
      const bool up = u > m_run[j] + A8_RESCALE_LOG2;
      if (__ballot(up)) {
        const float alpha = up ? __builtin_amdgcn_exp2f(m_run[j] - u) : 1.f;  // 0 from -inf
        if (__ballot(up && m_run[j] != -INFINITY)) {
#pragma unroll
          for (int hb = 0; hb < 4; ++hb) o[j][hb] *= alpha;
        }
        l_run[j] *= alpha;
        m_run[j] = up ? u : m_run[j];
      }
      const float off = lb - (m_run[j] == -INFINITY ? 0.f : m_run[j]);
      if (__ballot(fabsf(m_run[j]) > A8_LARGE)) {  // scores rounded as the base was
#pragma unroll
        for (int r = 0; r < 16; ++r) s[j][r] *= a;
        a = 1.f;
      }
      float psum = 0.f;
#pragma unroll
      for (int kh = 0; kh < 2; ++kh)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float p = __builtin_amdgcn_exp2f(fmaf(s[j][kh * 8 + e], a, off));
          psum += p;
          pf[j][kh][e] = (_Float16)p;
        }
      l_run[j] = fmaf(psum, inv_sv, l_run[j]);
    }
#pragma unroll
    for (int hb = 0; hb < 4; ++hb)
#pragma unroll
      for (int kh = 0; kh < 2; ++kh) {
        const f16x8 vf = kv8_to_f16(x.v[hb][2 * kh], x.v[hb][2 * kh + 1]);
#pragma unroll
        for (int j = 0; j < QT; ++j) o[j][hb] = mfma_f16(vf, pf[j][kh], o[j][hb]);
      }
  };
  int t = t_begin + kw;
  if (t < t_end) {
    Tile a, b;
    load(a, t);
    for (;;) {
      if (t + KW < t_end) load(b, t + KW);
      compute(a, t);
      t += KW;
      if (t >= t_end) break;
      if (t + KW < t_end) load(a, t + KW);
      compute(b, t);
      t += KW;
      if (t >= t_end) break;
    }
  }
#pragma unroll
  for (int j = 0; j < QT; ++j) l_run[j] += __shfl_xor(l_run[j], 32, 64);

  // the key ways of a query tile in pairs
  if (KW > 1) {
    const int tile = qw;
#pragma unroll
    for (int half = KW / 2; half > 0; half >>= 1) {
      __syncthreads();  // the queries, or the round before, have been read
      if (kw >= half && kw < 2 * half) {
        f32x4* d = (f32x4*)(smem + ((kw - half) * QW + tile) * (O_BYTES + 512));
#pragma unroll
        for (int hb = 0; hb < 4; ++hb)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            d[(hb * 4 + r) * 64 + lane] =
                f32x4{o[0][hb][4 * r], o[0][hb][4 * r + 1], o[0][hb][4 * r + 2], o[0][hb][4 * r + 3]};
        ((float2*)((char*)d + O_BYTES))[lane] = make_float2(m_run[0], l_run[0]);
      }
      __syncthreads();
      if (kw < half) {
        const f32x4* d = (const f32x4*)(smem + (kw * QW + tile) * (O_BYTES + 512));
        const float2 ml = ((const float2*)((const char*)d + O_BYTES))[lane];
        const float mm = fmaxf(m_run[0], ml.x);
        const float w0 = m_run[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run[0] - mm);
        const float w1 = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - mm);
#pragma unroll
        for (int hb = 0; hb < 4; ++hb)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const f32x4 y = d[(hb * 4 + r) * 64 + lane];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              o[0][hb][4 * r + e] = fmaf(w1, y[e], w0 * o[0][hb][4 * r + e]);
          }
        l_run[0] = fmaf(w1, ml.y, w0 * l_run[0]);
        m_run[0] = mm;
      }
    }
  }
  __syncthreads();
  if (kw > 0) return;  // (no barrier follows)
  // Rows out: a query tile's O^T through 16 KiB of the wave's own, as 16-byte pieces (query v,
  // piece p at p ^ v: every bank in turn both ways), 16 lanes a query vector.
  f32x4* ot = (f32x4*)(smem + qw * O_BYTES);
#pragma unroll
  for (int j = 0; j < QT; ++j) {
    const int v0 = (qt0 + qw * QT + j) * 32;
#pragma unroll
    for (int hb = 0; hb < 4; ++hb)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        ot[(lane & 31) * 32 + ((hb * 8 + 2 * r + (lane >> 5)) ^ (lane & 31))] =
            f32x4{o[j][hb][4 * r], o[j][hb][4 * r + 1], o[j][hb][4 * r + 2], o[j][hb][4 * r + 3]};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int v = (lane >> 4) + 4 * i, ch = lane & 15, qv = v0 + v;
      const float m = __shfl(m_run[j], v, 64), l = __shfl(l_run[j], v, 64);
      f32x4 y0 = ot[v * 32 + ((2 * ch) ^ v)], y1 = ot[v * 32 + ((2 * ch + 1) ^ v)];
      if (qv >= n_qv) continue;
      if (OUT) {
        const float inv = 1.f / l;
        y0 *= inv;
        y1 *= inv;
        const int row = qv / G;
        const int64_t at = ((int64_t)row * Hq + kvh * G + (qv - row * G)) * 128 + ch * 8;
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
        const int64_t at = ((int64_t)split * Hkv + kvh) * n_qv + qv;
        *(f32x4*)(ao.o_part + at * 128 + ch * 8) = y0;
        *(f32x4*)(ao.o_part + at * 128 + ch * 8 + 4) = y1;
        if (ch == 0) *(float2*)(ao.ml_part + at * 2) = make_float2(m, l);
      }
    }
  }
}

}  // namespace

namespace drt {

Attn8Plan plan_attention8(int n_rows, int Hq, int Hkv, int n_keys) {
  Attn8Plan p;
  const int qtiles = (int)(((int64_t)n_rows * (Hq / Hkv) + 31) / 32);
  p.qw = qtiles == 1 ? 1 : qtiles == 2 ? 2 : 4;
  p.wide = qtiles > 4;
  const int per = p.qw;  // query tiles of a work-group
  p.qgroups = (qtiles + per - 1) / per;
  const int n_tiles = (n_keys + 31) / 32, kw = p.wide ? 1 : 8 / p.qw;
  const int64_t wgs = (int64_t)Hkv * p.qgroups;
  const int target = p.wide ? 512 : 256;
  int64_t splits = std::max<int64_t>(1, target / wgs);
  splits = std::min<int64_t>({splits, (n_tiles + kw - 1) / kw, 64});
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
  const float c = 1.44269504088896340736f / sqrtf(128.0f);
  float* ml = part ? part + (size_t)p.splits * n_rows * Hq * 128 : nullptr;
  const A8Out ao{out, part, ml, out_bf16};
  const dim3 grid((unsigned)(p.splits * Hkv), (unsigned)p.qgroups);
#define DRT_A8(QT, QW, KW, OUT)                                                               \
  hipLaunchKernelGGL((attn8_kernel<QT, QW, KW, OUT>), grid, dim3(64 * QW * KW), 0, s,         \
                     (const uint16_t*)q, (const uint8_t*)kv_layer, kv_head_stride, scales,    \
                     (int)q_bf16, n_rows, Hq, Hkv, p.tiles_per_split, c, where, ao)
#define DRT_A8O(QT, QW, KW)                                                                   \
  do { if (p.splits == 1) DRT_A8(QT, QW, KW, true); else DRT_A8(QT, QW, KW, false); } while (0)
  if (p.wide) DRT_A8O(1, 4, 1);
  else if (p.qw == 1) DRT_A8O(1, 1, 8);
  else if (p.qw == 2) DRT_A8O(1, 2, 4);
  else DRT_A8O(1, 4, 2);
#undef DRT_A8O
#undef DRT_A8
  DRT_HIP(hipGetLastError());
  if (p.splits > 1) attn_combine(part, ml, p.splits, n_rows, Hq, Hkv, out, out_bf16 ? 3 : 2, s);
}

}  // namespace drt
