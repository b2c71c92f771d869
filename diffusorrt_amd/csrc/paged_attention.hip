// Attention of a batch's new rows over their sequences' keys in the pages of a cache, for gfx950.
//
// Query vectors of one K/V head are flattened (row, head of the group) within a sequence and taken in
// units; keys come in the pages' 32-key tiles. A wave computes S^T = K Q^T and O^T += V^T P^T as 32x32x16
// products with a running base and sum per query vector: p = 2^(s c - base), c = log2(e) / sqrt(128),
// o = sum p v / sum p. The base is raised when a tile's largest exponent has gone more than 8 over what it
// was raised by last; any base gives the same quotient (PA_LIFT: which). p's rounding to the products'
// 16-bit type is the one rounding ahead of the sums; scores, base, sum and O are fp32.
//
// A list made on the host (paged_plan.h) gives every work-group its unit and its share of the keys, so
// sequences of any lengths fill the chip: nothing is padded to the longest, and a sequence alone is cut
// as finely as pays. Units cut along their keys leave parts that a second launch joins.
//
// The weights' type is the cache's, which the products' operands share: an fp32 result is off by 0.8 to
// 1.7 * 10^-4 of its size over an fp16 cache and 1.3 * 10^-3 over a bf16 one, a row by 2.5 * 10^-4 and 2.0 * 10^-3 at
// most in the cases measured (a bf16 result, whose own rounding is 1.7 * 10^-3, by 2.1 in all over a bf16 cache).
#include "cache_dev.h"
#include "launch.h"
#include "paged_plan.h"

namespace {

using drt::PagedJoin;
using drt::PagedPiece;

constexpr int PA_TILE = 16384;  // bytes
constexpr int PA_QROW = 136;    // 16-bit elements per query vector in LDS (+ 16 bytes)

// The largest exponent less the base, where it is raised. fp16 weights are 2^7 then and 2^15 at most, which
// keeps those of down to 2^-21 of the largest normal numbers (many small ones add up over a long sequence).
// bf16 ones, which have the exponents, are 2^-24 and 2^-16 at most: thousands of keys whose values are the
// type's largest do not overflow the sum ahead of its division.
template <int CT> constexpr float PA_LIFT = CT == 1 ? 7.f : -24.f;

struct PaArgs {
  const uint16_t* q;    // [rows][hq][128]
  const uint8_t* cache; // this layer
  const PagedPiece* pieces;
  const int32_t* first;  // (large kernel) a work-group's first piece
  const int32_t* table;  // a page's first tile of head 0
  int hq, hkv, tpp, masked, block;
  float c;               // log2(e) / sqrt(128)
  int out_bf16;
  void* out;             // [rows][hq * 128]
  float* o_part;         // [slot][hkv][32][128]
  float* ml_part;        // [slot][hkv][32][2]
};

// The piece of this work-group, by scalar loads.
DRT_DEV PagedPiece pa_piece(const PagedPiece* pieces, int i) {
  const auto* p = (const __attribute__((address_space(4))) int32_t*)(uintptr_t)(pieces + i);
  PagedPiece y;
  y.row0 = p[0];
  y.rows = p[1];
  y.pos0 = p[2];
  y.keys = p[3];
  y.prompt_len = p[4];
  y.vec0 = p[5];
  y.tile0 = p[6];
  y.tile1 = p[7];
  y.slot = p[8];
  y.table = p[9];
  y.last = p[10];
  y.wide = p[11];
  return y;
}

// The number of keys that the sequence's row sees, always the first ones.
DRT_DEV int pa_key_end(const PaArgs& x, const PagedPiece& y, int row) {
  if (!x.masked) return y.keys;
  const int p = y.pos0 + row;
  if (p < y.prompt_len) return min(y.keys, y.prompt_len);
  const uint32_t mine = (uint32_t)(p - y.prompt_len) / (uint32_t)x.block;
  return (int)min((int64_t)y.keys, y.prompt_len + ((int64_t)mine + 1) * x.block);
}

// c + the sum of eight weights as the products have them (so that the quotient of a few large weights is
// not off by their roundings: a row that one key takes gets that key's value itself).
DRT_DEV float pa_add8(const f16x8 p, float c) { return kv8_add8(p, c); }
DRT_DEV float pa_add8(const bf16x8 p, float c) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const bf16x2 one = {(__bf16)1.f, (__bf16)1.f};
  const u32x4 w = __builtin_bit_cast(u32x4, p);
  const uint32_t w0 = w[0], w1 = w[1], w2 = w[2], w3 = w[3];
  c = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w0), one, c, false);
  c = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w1), one, c, false);
  c = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w2), one, c, false);
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w3), one, c, false);
}

// The products of a tile's 32 head dims of V (two operands) with the weights of QT query tiles. part: keys
// that not every row sees are among the tile's, or lie behind the sequence's last, and may be anything.
template <int CT, int QT>
DRT_DEV void pa_values(u32x4 v0, u32x4 v1, const typename CacheT<CT>::vec (&pf)[QT][2], bool part, int key0,
                       const int (&end)[QT], int lane, f32x16* const (&o)[QT]) {
  typedef CacheT<CT> T;
  typedef typename T::vec vec;
  u32x4 vr[2] = {v0, v1};
  if (part) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    u16x2 most = {0, 0};
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t w = vr[i][e] & 0x7fff7fffu;
        most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, w));
      }
    constexpr unsigned short EXP = CT == 1 ? 0x7c00 : 0x7f80;
    if (__ballot(most[0] >= EXP || most[1] >= EXP)) ca_values_apart<CT, QT>(vr, key0, end, lane, o);
  }
#pragma unroll
  for (int kh = 0; kh < 2; ++kh)
#pragma unroll
    for (int j = 0; j < QT; ++j) *o[j] = T::mma(__builtin_bit_cast(vec, vr[kh]), pf[j][kh], *o[j]);
}

DRT_DEV void pa_store8(const PaArgs& x, int64_t at, f32x4 y0, f32x4 y1) {
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
}

// Units of 32 query vectors: eight waves over keys, wave kw takes tiles kw, kw + 8, ... of the piece,
// straight from memory into registers, the next while this is worked on. They meet in LDS at the end.
// Bound by the keys' bytes where those are many: one row x 16 heads over 131072 keys 96 us (537 MB at 5.8
// TB/s of the kernel's 92), 32 tokens x 28 heads over up to 16384 52 (251 MB at 5.2 of 48). A CU alone draws
// 55 GB/s so, 0.29 us a tile; where units of the same keys run beside one another tiles come from the L2,
// 0.15. One row over 1337 keys: 5.6 us, of which a tile each wave and the joins; 3.0 more joins its parts.
// Four waves a work-group (two of them a CU) are slower where memory bounds (131072 keys 118 us).
constexpr int PS_WAVES = 8;
template <int CT>
DRT_DEV void pa_few(const PaArgs& x, const PagedPiece& pc, uint16_t* q_lds, char* ring0, char* ring1, float2* ml) {
  typedef CacheT<CT> T;
  typedef typename T::vec vec;
  constexpr int PIECES = 32, WAVE_O = 32 * PIECES * 16;
  // (a wave's O, 16 KiB; four in each of the rings)
  auto o_of = [&](int w) { return (f32x4*)((w < 4 ? ring0 : ring1) + (w & 3) * WAVE_O); };
  const int lane = threadIdx.x & 63, tid = threadIdx.x;
  const int kw = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kvh = (int)(blockIdx.x % (uint32_t)x.hkv), G = x.hq / x.hkv;
  const int vecs = min(32, pc.rows * G - pc.vec0);
  auto row_of = [&](int v) { return (int)((uint32_t)(pc.vec0 + v) / (uint32_t)G); };
  auto offset_of = [&](int v) {  // of query vector v's head in q and out
    const int row = row_of(v);
    return ((int64_t)(pc.row0 + row) * x.hq + kvh * G + (pc.vec0 + v - row * G)) * 128;
  };

  // the queries (behind the last query vector it again: not used)
  const int v = tid >> 4, ch = tid & 15;
  const u32x4 qraw = *(const u32x4*)(x.q + offset_of(min(v, vecs - 1)) + ch * 8);

  // this wave's tiles: lane l holds the tile number in the layer of its (64 i + l)-th
  const int n = (pc.tile1 - pc.tile0 - kw + PS_WAVES - 1) / PS_WAVES;
  const int sh = __builtin_ctz(x.tpp);
  auto numbers = [&](int i) {
    const int t = min(pc.tile0 + kw + PS_WAVES * (i + lane), pc.tile1 - 1);
    return x.table[pc.table + (t >> sh)] + kvh * x.tpp + (t & (x.tpp - 1));
  };
  int held = n > 0 ? numbers(0) : 0;
  auto tile_at = [&](int i) {
    return x.cache + (int64_t)__builtin_amdgcn_readlane(held, i & 63) * PA_TILE + lane * 16;
  };
  u32x4 kr[8], vr[8];
  if (n > 0) {
    const uint8_t* p = tile_at(0);
#pragma unroll
    for (int i = 0; i < 8; ++i) kr[i] = *(const u32x4*)(p + i * 1024);
#pragma unroll
    for (int i = 0; i < 8; ++i) vr[i] = *(const u32x4*)(p + PA_TILE / 2 + i * 1024);
  }
  const int q_end[1] = {pa_key_end(x, pc, row_of(min(lane & 31, vecs - 1)))};
  // (ends never fall from row to row) keys that every row of the unit sees
  const int full_end = pa_key_end(x, pc, row_of(0));
  *(u32x4*)(q_lds + v * PA_QROW + ch * 8) = qraw;
  ca_lds_barrier();
  const uint16_t* ql = q_lds + (lane & 31) * PA_QROW + 8 * (lane >> 5);
  vec qr[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) qr[i] = *(const vec*)(ql + 16 * i);

  float m_run = -INFINITY, l_run = 0.f;
  float base = 0.f;     // m_run, or 0 before any key
  float scale = x.c;    // 1 where the base is large: the scores are then scaled as it was
  f32x16 o[4];
#pragma unroll
  for (int hb = 0; hb < 4; ++hb) o[hb] = f32x16{};
  for (int it = 0; it < n; ++it) {
    const int key0 = (pc.tile0 + kw + PS_WAVES * it) * 32;
    const int next = min(it + 1, n - 1);  // (the last tile's own again: loaded, not used)
    if ((next & 63) == 0 && next) held = numbers(next);
    const uint8_t* p = tile_at(next);
    f32x16 s = f32x16{};
#pragma unroll
    for (int i = 0; i < 8; ++i) s = T::mma(ca_operand<CT>(kr, i), qr[i], s);
#pragma unroll
    for (int i = 0; i < 8; ++i) kr[i] = *(const u32x4*)(p + i * 1024);
    const bool part = key0 + 32 > full_end;
    if (part) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = key0 + mfma_row(r, lane) < q_end[0] ? s[r] : -INFINITY;
    }
    float tmax = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) tmax = fmaxf(tmax, s[r]);
    const float u = ca_max_xor32(tmax) * x.c;  // -inf: no visible key
    const bool up = u - m_run > PA_LIFT<CT> + CA_RESCALE_LOG2;  // (exact where it matters)
    if (__ballot(up)) {
      const float to = up ? u - PA_LIFT<CT> : m_run;
      const float alpha = up ? __builtin_amdgcn_exp2f(m_run - to) : 1.f;  // 0 from -inf
#pragma unroll
      for (int hb = 0; hb < 4; ++hb) o[hb] *= alpha;
      l_run *= alpha;
      m_run = to;
      base = up ? to : base;
      scale = __ballot(fabsf(base) > CA_LARGE) ? 1.f : x.c;
    }
    if (scale == 1.f) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] *= x.c;
    }
    vec pf[1][2];
#pragma unroll
    for (int kh = 0; kh < 2; ++kh)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        pf[0][kh][e] = T::weight(__builtin_amdgcn_exp2f(fmaf(s[kh * 8 + e], scale, -base)));
    l_run = pa_add8(pf[0][1], pa_add8(pf[0][0], l_run));
#pragma unroll
    for (int hb = 0; hb < 4; ++hb) {
      f32x16* const at[1] = {&o[hb]};
      pa_values<CT, 1>(vr[2 * hb], vr[2 * hb + 1], pf, part, key0, q_end, lane, at);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) vr[i] = *(const u32x4*)(p + PA_TILE / 2 + i * 1024);
  }
  l_run += __shfl_xor(l_run, 32, 64);

  // The ways joined: every wave leaves its O in LDS as 16-byte pieces (query v, piece p at p ^ v: every
  // bank in turn both ways), then threads with eight head dims of a query vector add the ways'.
  {
    f32x4* d = o_of(kw);
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        d[(lane & 31) * PIECES + ((b * 8 + 2 * r + (lane >> 5)) ^ (lane & 15))] =
            f32x4{o[b][4 * r], o[b][4 * r + 1], o[b][4 * r + 2], o[b][4 * r + 3]};
    if (lane < 32) ml[kw * 32 + lane] = make_float2(m_run, l_run);
  }
  __syncthreads();
  if (v >= vecs) return;
  float2 w[PS_WAVES];
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int k = 0; k < PS_WAVES; ++k) {
    w[k] = ml[k * 32 + v];
    m = fmaxf(m, w[k].x);
  }
  f32x4 y0 = f32x4{}, y1 = f32x4{};
#pragma unroll
  for (int k = 0; k < PS_WAVES; ++k) {
    const f32x4* d = o_of(k) + v * PIECES;
    const float f = w[k].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(w[k].x - m);
    y0 += f * d[(2 * ch) ^ (v & 15)];
    y1 += f * d[(2 * ch + 1) ^ (v & 15)];
    l = fmaf(f, w[k].y, l);
  }
  if (pc.slot < 0) {
    const float inv = pc.tile1 == 0 ? 0.f : 1.f / l;  // (no key: zeros)
    pa_store8(x, offset_of(v) + ch * 8, y0 * inv, y1 * inv);
  } else {
    const int64_t at = ((int64_t)pc.slot * x.hkv + kvh) * 32 + v;
    *(f32x4*)(x.o_part + at * 128 + ch * 8) = y0;
    *(f32x4*)(x.o_part + at * 128 + ch * 8 + 4) = y1;
    if (ch == 0) *(float2*)(x.ml_part + at * 2) = make_float2(m, l);
  }
}

// Units of many query vectors: QW waves side by side of QT tiles of 32 (for all of which a key tile's operands
// are read once), for each of 8 / QW key ways, which take turns at the tiles. Tiles come by direct-to-LDS
// loads, one for the waves of a way together, the next while this is worked on; queries lie in LDS for
// all of it, some of them in registers.
// 64 query vectors (2 x 1 and four ways): 0.245 us a tile, 0.15 for 32 of them above; it begins and ends 2 us
// slower, so it takes over where keys are long (16 sequences of 32 rows x 16 heads 47 us, 50 above; 150 rows
// x 28 heads over 16000 keys 53 and 66, over 1300 17.7 and 11.2).
// 256 (4 x 2 and two ways): 0.74 us a tile. Bound by the matrix unit at the clock that the card's power
// leaves it: 2048 rows x 28 heads over 10240 keys 286 us, 1.13 PFLOP/s in the steps, as much as a large
// library product; the rest is the first and last 20 us of a work-group and rows that see fewer keys
// finishing early. With zeros for data it is 26 % faster. All 256 registers are taken and 6 (fp16) or 8 (bf16) more
// spilled: addresses of the queries' loads and LDS places, reloaded once a part and in no step, but each
// with a wait among those loads. Below, not faster: the two ways half a step apart with a barrier between,
// priorities around the products, five or six of eight query steps in registers.
template <int CT, int QW, int QT>
DRT_DEV void pa_shared(const PaArgs& x, const PagedPiece& pc, uint16_t* q_lds, char* ring0, char* ring1, float2* ml) {
  typedef CacheT<CT> T;
  typedef typename T::vec vec;
  constexpr int WAYS = 8 / QW, VW = 32 * QT, NQ = QW * VW;  // query vectors of a wave, of the unit
  constexpr int HELD = QT == 1 ? 8 : 4;  // steps of 16 head dims whose queries are in registers
  const int lane = threadIdx.x & 63, tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), qw = wave % QW, way = wave / QW;
  const int kvh = (int)(blockIdx.x % (uint32_t)x.hkv), G = x.hq / x.hkv;
  const int vecs = min(NQ, pc.rows * G - pc.vec0);
  auto row_of = [&](int v) { return (int)((uint32_t)(pc.vec0 + v) / (uint32_t)G); };
  auto offset_of = [&](int v) {
    const int row = row_of(v);
    return ((int64_t)(pc.row0 + row) * x.hq + kvh * G + (pc.vec0 + v - row * G)) * 128;
  };

  // this key way's tiles
  const int n_it = (pc.tile1 - pc.tile0 + WAYS - 1) / WAYS;       // of the work-group
  const int n = (pc.tile1 - pc.tile0 - way + WAYS - 1) / WAYS;    // of the way
  const int sh = __builtin_ctz(x.tpp);
  auto numbers = [&](int i) {
    const int t = min(pc.tile0 + way + WAYS * (i + lane), pc.tile1 - 1);
    return x.table[pc.table + (t >> sh)] + kvh * x.tpp + (t & (x.tpp - 1));
  };
  int held = n > 0 ? numbers(0) : 0;
  auto issue = [&](int i, char* dst) {  // this wave's share of the way's tile i
    if (i >= n) return;
    if ((i & 63) == 0 && i) held = numbers(i);
    const __amdgpu_buffer_rsrc_t src = __builtin_amdgcn_make_buffer_rsrc(
        (void*)(x.cache + (int64_t)__builtin_amdgcn_readlane(held, i & 63) * PA_TILE), 0, PA_TILE,
        0x00020000);
#pragma unroll
    for (int k = 0; k < 16 / QW; ++k)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          src, (__attribute__((address_space(3))) void*)(dst + way * PA_TILE + (qw * (16 / QW) + k) * 1024), 16,
          (uint32_t)((qw * (16 / QW) + k) * 1024 + lane * 16), 0, 0, 0);
  };
  issue(0, ring0);
  u32x4 qraw[NQ / 32];  // (behind the last query vector it again: not used)
#pragma unroll
  for (int it = 0; it < NQ / 32; ++it)
    qraw[it] = *(const u32x4*)(x.q + offset_of(min((it * 512 + tid) >> 4, vecs - 1)) + (tid & 15) * 8);
#pragma unroll
  for (int it = 0; it < NQ / 32; ++it)
    *(u32x4*)(q_lds + ((it * 512 + tid) >> 4) * PA_QROW + (tid & 15) * 8) = qraw[it];
  const uint16_t* ql = q_lds + (qw * VW + (lane & 31)) * PA_QROW + 8 * (lane >> 5);
  int q_end[QT];
#pragma unroll
  for (int j = 0; j < QT; ++j)
    q_end[j] = pa_key_end(x, pc, row_of(min(qw * VW + 32 * j + (lane & 31), vecs - 1)));
  // (ends never fall from row to row) keys that every row of the wave sees, and any of them
  const int full_end = pa_key_end(x, pc, row_of(min(qw * VW, vecs - 1)));
  const int wave_end = qw * VW < vecs ? pa_key_end(x, pc, row_of(min(qw * VW + VW - 1, vecs - 1))) : 0;

  float m_run[QT], l_run[QT], base[QT];  // base: m_run, or 0 before any key
  f32x16 o[QT][4];
#pragma unroll
  for (int j = 0; j < QT; ++j) {
    m_run[j] = -INFINITY;
    l_run[j] = base[j] = 0.f;
#pragma unroll
    for (int hb = 0; hb < 4; ++hb) o[j][hb] = f32x16{};
  }

  f32x16 s[QT];
  vec pf[QT][2];
  float scale = x.c;    // 1 where a base is large: the scores are then scaled as it was
  auto weights = [&] {  // of all query tiles, from their scores
    float u[QT], far = 0.f;
    bool up[QT], any = false;
#pragma unroll
    for (int j = 0; j < QT; ++j) {
      float tmax = s[j][0];
#pragma unroll
      for (int r = 1; r < 16; ++r) tmax = fmaxf(tmax, s[j][r]);
      u[j] = ca_max_xor32(tmax) * x.c;  // -inf: no visible key
      up[j] = u[j] - m_run[j] > PA_LIFT<CT> + CA_RESCALE_LOG2;
      any = any || up[j];
    }
    if (__ballot(any)) {
#pragma unroll
      for (int j = 0; j < QT; ++j) {
        const float to = up[j] ? u[j] - PA_LIFT<CT> : m_run[j];
        const float alpha = up[j] ? __builtin_amdgcn_exp2f(m_run[j] - to) : 1.f;  // 0 from -inf
#pragma unroll
        for (int hb = 0; hb < 4; ++hb) o[j][hb] *= alpha;
        l_run[j] *= alpha;
        m_run[j] = to;
        base[j] = up[j] ? to : base[j];
        far = fmaxf(far, fabsf(base[j]));
      }
      scale = __ballot(far > CA_LARGE) ? 1.f : x.c;
    }
    if (scale == 1.f) {
#pragma unroll
      for (int j = 0; j < QT; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[j][r] *= x.c;
    }
#pragma unroll
    for (int j = 0; j < QT; ++j) {
#pragma unroll
      for (int kh = 0; kh < 2; ++kh)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          pf[j][kh][e] =
              T::weight(__builtin_amdgcn_exp2f(fmaf(s[j][kh * 8 + e], scale, -base[j])));
      l_run[j] = pa_add8(pf[j][1], pa_add8(pf[j][0], l_run[j]));
    }
  };
  // A step is a tile of each way. ANY: one that not every row sees whole (the others' steps have queries in
  // registers, where two query tiles leave room for half of them).
  vec qr[QT][HELD];
  auto step = [&](int i, const char* here, char* next, auto any) {
    constexpr bool ANY = decltype(any)::value;
    const int key0 = (pc.tile0 + way + WAYS * i) * 32;
    const bool mine = ANY ? i < n && key0 < wave_end : wave_end > 0;
    const bool part = ANY && key0 + 32 > full_end;
    const uint16_t* kt = (const uint16_t*)(here + way * PA_TILE) + lane * 8;
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): its tile is here
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (i + 1 < n_it) issue(i + 1, next);
    if (mine) {
#pragma unroll
      for (int j = 0; j < QT; ++j) s[j] = f32x16{};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const vec kf = *(const vec*)(kt + e * 512);
#pragma unroll
        for (int j = 0; j < QT; ++j)
          s[j] = T::mma(kf, (!ANY || QT == 1) && e < HELD
                               ? qr[j][e < HELD ? e : 0]
                               : *(const vec*)(ql + j * 32 * PA_QROW + 16 * e),
                        s[j]);
      }
      if (part) {
#pragma unroll
        for (int j = 0; j < QT; ++j)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            s[j][r] = key0 + mfma_row(r, lane) < q_end[j] ? s[j][r] : -INFINITY;
      }
      weights();
#pragma unroll
      for (int hb = 0; hb < 4; ++hb) {
        f32x16* at[QT];
#pragma unroll
        for (int j = 0; j < QT; ++j) at[j] = &o[j][hb];
        pa_values<CT, QT>(*(const u32x4*)(kt + 4096 + hb * 1024),
                         *(const u32x4*)(kt + 4096 + hb * 1024 + 512), pf, part, key0, q_end, lane, at);
      }
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): this wave is done reading the slot
  };
  __syncthreads();  // the queries are in LDS
#pragma unroll
  for (int j = 0; j < QT; ++j)
#pragma unroll
    for (int e = 0; e < HELD; ++e) qr[j][e] = *(const vec*)(ql + j * 32 * PA_QROW + 16 * e);
  // (a whole number of both rings' steps) tiles that every row of the unit sees, of both ways
  const int whole = min(pa_key_end(x, pc, row_of(0)) >> 5, pc.tile1) - pc.tile0;
  const int n_whole = max(whole, 0) / WAYS & ~1;
  int it = 0;
  for (; it < n_whole; it += 2) {
    step(it, ring0, ring1, std::false_type{});
    step(it + 1, ring1, ring0, std::false_type{});
  }
  for (; it < n_it; it += 2) {
    step(it, ring0, ring1, std::true_type{});
    if (it + 1 >= n_it) break;
    step(it + 1, ring1, ring0, std::true_type{});
  }
#pragma unroll
  for (int j = 0; j < QT; ++j) l_run[j] += __shfl_xor(l_run[j], 32, 64);

  // The other ways' parts to the first, which has the same queries in the same registers, half a head
  // at a time; the first way's waves write theirs out, eight head dims a lane.
  constexpr int REGION = QT * 8192, IN_RING = WAYS * PA_TILE / REGION;
  static_assert((WAYS - 1) * QW <= 2 * IN_RING, "half a head of the other ways' queries fits the rings");
  auto region = [&](int w) {  // of way w's wave of these queries
    const int i = (w - 1) * QW + qw;
    return (i < IN_RING ? ring0 + i * REGION : ring1 + (i - IN_RING) * REGION) + lane * 16;
  };
  float f[QT][WAYS];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    __syncthreads();  // the rings, or the first half, have been read
    if (way) {
      char* const mine = region(way);
#pragma unroll
      for (int j = 0; j < QT; ++j) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const f32x16& y = o[j][2 * half + b];
            *(f32x4*)(mine + ((j * 2 + b) * 4 + r) * 1024) =
                f32x4{y[4 * r], y[4 * r + 1], y[4 * r + 2], y[4 * r + 3]};
          }
        if (half == 0 && lane < 32)
          ml[(way - 1) * NQ + qw * VW + j * 32 + lane] = make_float2(m_run[j], l_run[j]);
      }
    }
    __syncthreads();
    if (!way) {
#pragma unroll
      for (int j = 0; j < QT; ++j) {
        const int v = qw * VW + j * 32 + (lane & 31);
        if (half == 0) {
          float2 z[WAYS];
          z[0] = make_float2(m_run[j], l_run[j]);
          float m = m_run[j], l = 0.f;
#pragma unroll
          for (int w = 1; w < WAYS; ++w) {
            z[w] = ml[(w - 1) * NQ + v];
            m = fmaxf(m, z[w].x);
          }
#pragma unroll
          for (int w = 0; w < WAYS; ++w) {
            f[j][w] = z[w].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(z[w].x - m);
            l = fmaf(f[j][w], z[w].y, l);
          }
          m_run[j] = m;
          l_run[j] = l;
        }
        const float inv = pc.slot >= 0 ? 1.f : pc.tile1 == 0 ? 0.f : 1.f / l_run[j];  // (no key: zeros)
        const bool there = v < vecs;
        const int64_t part = ((int64_t)(pc.slot + (v >> 5)) * x.hkv + kvh) * 32 + (v & 31);
        const int64_t out = there ? offset_of(v) : 0;
        if (half == 0 && pc.slot >= 0 && there && lane < 32)
          *(float2*)(x.ml_part + part * 2) = make_float2(m_run[j], l_run[j]);
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int r = 0; r < 4; r += 2) {
            // dims 8 r + 4 (lane / 32) + 0..3 and 8 (r + 1) + ... become 8 (r + lane / 32) + 0..7
            f32x4 y[2];
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              const f32x16& z = o[j][2 * half + b];
              y[g] = f32x4{z[4 * (r + g)], z[4 * (r + g) + 1], z[4 * (r + g) + 2], z[4 * (r + g) + 3]} *
                     f[j][0];
#pragma unroll
              for (int w = 1; w < WAYS; ++w)
                y[g] += *(const f32x4*)(region(w) + ((j * 2 + b) * 4 + r + g) * 1024) * f[j][w];
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(y[0][e]),
                                                              __float_as_uint(y[1][e]), false, false);
              y[0][e] = __uint_as_float(w[0]);
              y[1][e] = __uint_as_float(w[1]);
            }
            const int hd = 64 * half + 32 * b + 8 * (r + (lane >> 5));
            if (!there) continue;
            if (pc.slot < 0) {
              pa_store8(x, out + hd, y[0] * inv, y[1] * inv);
            } else {
              *(f32x4*)(x.o_part + part * 128 + hd) = y[0];
              *(f32x4*)(x.o_part + part * 128 + hd + 4) = y[1];
            }
          }
      }
    }
  }
}

// (the buffer resource type is not known to the host pass: the bodies are device functions)
// (separate arrays: the compiler knows the slot being read is not one being filled)
template <int CT> __global__ __launch_bounds__(512, 2) void paged_attn_kernel(const PaArgs x) {
  __shared__ __align__(16) uint16_t q_lds[64 * PA_QROW];
  __shared__ __align__(1024) char ring0[4 * PA_TILE];
  __shared__ __align__(1024) char ring1[4 * PA_TILE];
  __shared__ float2 ml[8 * 32];
#if defined(__HIP_DEVICE_COMPILE__)
  const PagedPiece pc = pa_piece(x.pieces, (int)(blockIdx.x / (uint32_t)x.hkv));
  if (pc.wide) pa_shared<CT, 2, 1>(x, pc, q_lds, ring0, ring1, ml);
  else pa_few<CT>(x, pc, q_lds, ring0, ring1, ml);
#endif
}
template <int CT> __global__ __launch_bounds__(512, 2) void paged_attn_large_kernel(const PaArgs x) {
  __shared__ __align__(16) uint16_t q_lds[256 * PA_QROW];
  __shared__ __align__(1024) char ring0[2 * PA_TILE];
  __shared__ __align__(1024) char ring1[2 * PA_TILE];
  __shared__ float2 ml[256];
#if defined(__HIP_DEVICE_COMPILE__)
  for (int at = x.first[blockIdx.x / (uint32_t)x.hkv];; ++at) {
    const PagedPiece pc = pa_piece(x.pieces, at);
    pa_shared<CT, 4, 2>(x, pc, q_lds, ring0, ring1, ml);
    if (pc.last) return;
    __syncthreads();  // the next part's queries and tiles go where this one's O was
  }
#endif
}

// The parts of a unit joined: WIDE, a wave for each query vector, lane (sg, ch) adding head dims 8 ch ..
// + 8 of parts sg, sg + 4, ...; the four groups meet by lane exchanges. Otherwise sixteen lanes for each,
// four query vectors a wave. All loads of a batch of parts are on their way before their use. 3.0 to 4.3 us, a
// launch and one chain of loads. (Joined by the last work-group of a unit to arrive instead: 64 rows x 16
// heads over 2048 keys 16.8 us, 12.3 with this launch.)
template <bool WIDE>
__global__ __launch_bounds__(256) void paged_join_kernel(const PaArgs x, const PagedJoin* joins) {
  const int kvh = (int)(blockIdx.x % (uint32_t)x.hkv), G = x.hq / x.hkv;
  const PagedJoin y = joins[blockIdx.x / (uint32_t)x.hkv];
  const int lane = threadIdx.x & 63, ch = lane & 15, sg = WIDE ? lane >> 4 : 0;
  const int v = WIDE ? (int)blockIdx.y * 4 + (threadIdx.x >> 6) : (int)blockIdx.y * 16 + (threadIdx.x >> 4);
  if (v >= y.vecs) return;
  constexpr int SB = 4, STEP = WIDE ? 4 : 1;
  float m = -INFINITY, l = 0.f;
  f32x4 a0 = f32x4{}, a1 = f32x4{};
  for (int s0 = sg; s0 < y.parts; s0 += STEP * SB) {
    float2 ml[SB];
    f32x4 p0[SB], p1[SB];
#pragma unroll
    for (int j = 0; j < SB; ++j) {
      const int64_t slot = y.slot + (int64_t)y.step * min(s0 + STEP * j, y.parts - 1);
      const int64_t at = (slot * x.hkv + kvh) * 32 + v;
      ml[j] = *(const float2*)(x.ml_part + at * 2);
      p0[j] = *(const f32x4*)(x.o_part + at * 128 + 8 * ch);
      p1[j] = *(const f32x4*)(x.o_part + at * 128 + 8 * ch + 4);
    }
    float mb = m;
#pragma unroll
    for (int j = 0; j < SB; ++j) {
      if (s0 + STEP * j >= y.parts) {  // (the last part's again: 0 * infinity would be NaN)
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
  if (WIDE) {
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
  }
  const float inv = 1.f / l;  // (a unit that is cut has keys)
  const int row = (y.vec0 + v) / G;
  const int64_t at = ((int64_t)(y.row0 + row) * x.hq + kvh * G + (y.vec0 + v - row * G)) * 128 + 8 * ch;
  pa_store8(x, at, a0 * inv, a1 * inv);
}

}  // namespace

namespace drt {

size_t paged_part_bytes(int slots, int hkv) { return (size_t)slots * hkv * 32 * 130 * 4; }

void paged_attention(const PagedAttnCall& c, hipStream_t s) {
  PaArgs a{};
  a.q = (const uint16_t*)c.q;
  a.cache = (const uint8_t*)c.cache;
  a.table = c.list + c.table;
  a.hq = c.hq;
  a.hkv = c.hkv;
  a.tpp = c.tpp;
  a.masked = c.masked;
  a.block = c.block;
  a.c = 1.44269504088896340736f / sqrtf(128.0f);
  a.out_bf16 = c.out_type == 2;
  a.out = c.out;
  a.o_part = (float*)c.workspace;
  a.ml_part = a.o_part ? a.o_part + (size_t)c.slots * c.hkv * 32 * 128 : nullptr;
  if (c.n_small) {
    a.pieces = (const PagedPiece*)(c.list + c.small);
    const dim3 grid((unsigned)c.n_small * (unsigned)c.hkv);
    if (c.cache_bf16) hipLaunchKernelGGL(paged_attn_kernel<2>, grid, dim3(512), 0, s, a);
    else hipLaunchKernelGGL(paged_attn_kernel<1>, grid, dim3(512), 0, s, a);
    DRT_HIP(hipGetLastError());
  }
  if (c.n_large) {
    a.pieces = (const PagedPiece*)(c.list + c.large);
    a.first = c.list + c.first_large;
    const dim3 grid((unsigned)c.n_large * (unsigned)c.hkv);
    if (c.cache_bf16) hipLaunchKernelGGL(paged_attn_large_kernel<2>, grid, dim3(512), 0, s, a);
    else hipLaunchKernelGGL(paged_attn_large_kernel<1>, grid, dim3(512), 0, s, a);
    DRT_HIP(hipGetLastError());
  }
  if (c.n_joins) {
    // Few query vectors of many parts by a wave each, many of few by a quarter (both launches, us with a wave
    // and a quarter: one row over 16000 keys, 25 parts, 17.7 and 20.6; over 60000, 105 parts, 20.6 and 32.8;
    // 64 rows x 32 heads in 128 parts of 32 units 31.8 and 31.2).
    const bool wide = c.slots > 4 * c.n_joins || (int64_t)c.n_joins * c.hkv < 64;
    const unsigned n = (unsigned)c.n_joins * (unsigned)c.hkv;
    const PagedJoin* joins = (const PagedJoin*)(c.list + c.joins);
    if (wide) hipLaunchKernelGGL(paged_join_kernel<true>, dim3(n, 8), dim3(256), 0, s, a, joins);
    else hipLaunchKernelGGL(paged_join_kernel<false>, dim3(n, 2), dim3(256), 0, s, a, joins);
    DRT_HIP(hipGetLastError());
  }
}

}  // namespace drt
