// Attention of a batch's new rows over their sequences' keys in the pages of a cache, for gfx950.
//
// Query vectors of one K/V head are flattened (row, head of the group) within a sequence and taken in
// units; keys come in the pages' 32-key tiles. A wave computes S^T = K Q^T and O^T += V^T P^T as 32x32x16
// products with a running base and sum per query vector: p = 2^(s c - base), c = log2(e) / sqrt(128),
// o = sum p v / sum p. The base is raised when a tile's largest exponent exceeds it by more than 8
// (any base gives the same quotient; p <= 2^8). p's rounding to the products' 16-bit type is the one
// rounding ahead of the sums; scores, base, sum and O are fp32.
//
// A list made on the host (paged_plan.h) gives every work-group its unit and its share of the keys, so
// sequences of any lengths fill the chip: nothing is padded to the longest, and a sequence alone is cut
// as finely as pays. Units cut along their keys leave parts that a second launch joins.
#include "cache_dev.h"
#include "launch.h"
#include "paged_plan.h"

namespace {

using drt::PagedJoin;
using drt::PagedPiece;

constexpr int PA_TILE = 16384;  // bytes
constexpr int PA_QROW = 136;    // 16-bit elements per query vector in LDS (+ 16 bytes)

struct PaArgs {
  const uint16_t* q;    // [rows][hq][128]
  const uint8_t* cache; // this layer
  const PagedPiece* pieces;
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

// Whether any of a tile's V (16 bits) in this lane's registers is not finite.
template <int CT> DRT_DEV bool pa_any_not_finite(const u32x4 (&vr)[8]) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  u16x2 most = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t w = vr[i][e] & 0x7fff7fffu;
      most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, w));
    }
  constexpr unsigned short EXP = CT == 1 ? 0x7c00 : 0x7f80;
  return most[0] >= EXP || most[1] >= EXP;
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

// Units of 32 query vectors: KW waves over keys (wave kw takes tiles kw, kw + KW, ... of the piece; they
// meet in LDS at the end), a tile straight from memory into registers.
template <int CT, int KW>
__global__ __launch_bounds__(64 * KW, 2) void paged_attn_kernel(const PaArgs x) {
  typedef CacheT<CT> T;
  typedef typename T::vec vec;
  constexpr int THREADS = 64 * KW, PIECES = 32, WAVE_O = 32 * PIECES * 16;
  constexpr int Q_BYTES = 32 * PA_QROW * 2, O_BYTES = KW * WAVE_O;
  __shared__ __align__(16) char smem[Q_BYTES > O_BYTES ? Q_BYTES : O_BYTES];
  __shared__ float2 ml[KW][32];
  const int lane = threadIdx.x & 63, tid = threadIdx.x;
  const int kw = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kvh = (int)(blockIdx.x % (uint32_t)x.hkv), G = x.hq / x.hkv;
  const PagedPiece pc = pa_piece(x.pieces, (int)(blockIdx.x / (uint32_t)x.hkv));
  const int vecs = min(32, pc.rows * G - pc.vec0);
  auto row_of = [&](int v) { return (pc.vec0 + v) / G; };
  auto offset_of = [&](int v) {  // of query vector v's head in q and out
    const int row = row_of(v);
    return ((int64_t)(pc.row0 + row) * x.hq + kvh * G + (pc.vec0 + v - row * G)) * 128;
  };

  constexpr int QL = 512 / THREADS;
  static_assert(QL * THREADS == 512, "whole rounds of the queries");
  u32x4 qraw[QL];
#pragma unroll
  for (int it = 0; it < QL; ++it) {
    const int v = (it * THREADS + tid) >> 4;
    qraw[it] = u32x4{0u, 0u, 0u, 0u};
    if (v < vecs) qraw[it] = *(const u32x4*)(x.q + offset_of(v) + (tid & 15) * 8);
  }

  // this wave's tiles: lane l holds the tile number in the layer of its (64 i + l)-th
  const int n = (pc.tile1 - pc.tile0 - kw + KW - 1) / KW;
  const int sh = __builtin_ctz(x.tpp);
  auto numbers = [&](int i) {
    const int t = min(pc.tile0 + kw + KW * (i + lane), pc.tile1 - 1);
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
  const int q_end = pa_key_end(x, pc, row_of(min(lane & 31, vecs - 1)));
  // (ends never fall from row to row) keys that every row of the unit sees
  const int full_end = pa_key_end(x, pc, row_of(0));
#pragma unroll
  for (int it = 0; it < QL; ++it)
    *(u32x4*)(smem + (((it * THREADS + tid) >> 4) * PA_QROW + (tid & 15) * 8) * 2) = qraw[it];
  ca_lds_barrier();
  const uint16_t* ql = (const uint16_t*)smem + (lane & 31) * PA_QROW + 8 * (lane >> 5);
  vec qr[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) qr[i] = *(const vec*)(ql + 16 * i);

  float m_run = -INFINITY, l_run = 0.f;
  f32x16 o[4];
#pragma unroll
  for (int hb = 0; hb < 4; ++hb) o[hb] = f32x16{};
  for (int it = 0; it < n; ++it) {
    const int key0 = (pc.tile0 + kw + KW * it) * 32;
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
      for (int r = 0; r < 16; ++r) s[r] = key0 + mfma_row(r, lane) < q_end ? s[r] : -INFINITY;
    }
    float tmax = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) tmax = fmaxf(tmax, s[r]);
    const float u = ca_max_xor32(tmax) * x.c;  // -inf: no visible key
    const bool up = u > m_run + CA_RESCALE_LOG2;
    if (__ballot(up)) {
      const float alpha = up ? __builtin_amdgcn_exp2f(m_run - u) : 1.f;  // 0 from -inf
#pragma unroll
      for (int hb = 0; hb < 4; ++hb) o[hb] *= alpha;
      l_run *= alpha;
      m_run = up ? u : m_run;
    }
    const float mb = m_run == -INFINITY ? 0.f : m_run;
    float a = x.c;
    if (__ballot(fabsf(mb) > CA_LARGE)) {  // exponents rounded as the base was
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] *= a;
      a = 1.f;
    }
    float psum = 0.f;
    vec pf[2];
#pragma unroll
    for (int kh = 0; kh < 2; ++kh)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float w = __builtin_amdgcn_exp2f(fmaf(s[kh * 8 + e], a, -mb));
        psum += w;
        pf[kh][e] = T::weight(w);
      }
    l_run += psum;
    // What lies behind the sequence's last key, or is not for every row, may be anything
    if (part && __ballot(pa_any_not_finite<CT>(vr))) ca_values_apart<CT>(vr, key0, q_end, lane, o);
#pragma unroll
    for (int hb = 0; hb < 4; ++hb)
#pragma unroll
      for (int kh = 0; kh < 2; ++kh) o[hb] = T::mma(ca_operand<CT>(vr, hb * 2 + kh), pf[kh], o[hb]);
#pragma unroll
    for (int i = 0; i < 8; ++i) vr[i] = *(const u32x4*)(p + PA_TILE / 2 + i * 1024);
  }
  l_run += __shfl_xor(l_run, 32, 64);

  // The key ways joined: every wave leaves its O in LDS as 16-byte pieces (query v, piece p at p ^ v:
  // every bank in turn both ways), then threads with eight head dims of a query vector add the ways'.
  __syncthreads();  // the queries have been read
  {
    f32x4* d = (f32x4*)(smem + kw * WAVE_O);
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        d[(lane & 31) * PIECES + ((b * 8 + 2 * r + (lane >> 5)) ^ (lane & 15))] =
            f32x4{o[b][4 * r], o[b][4 * r + 1], o[b][4 * r + 2], o[b][4 * r + 3]};
    if (lane < 32) ml[kw][lane] = make_float2(m_run, l_run);
  }
  __syncthreads();
#pragma unroll
  for (int it = 0; it < QL; ++it) {
    const int v = (it * THREADS + tid) >> 4, ch = tid & 15;
    if (v >= vecs) continue;
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
      const f32x4* d = (const f32x4*)(smem + k * WAVE_O) + v * PIECES;
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
}

// The parts of a unit joined, a wave for each query vector: lane (sg, ch) adds head dims 8 ch .. + 8 of
// parts sg, sg + 4, ..., all of a batch's loads before their use, and the four groups meet by lane
// exchanges.
__global__ __launch_bounds__(256) void paged_join_kernel(const PaArgs x, const PagedJoin* joins) {
  const int kvh = (int)(blockIdx.x % (uint32_t)x.hkv), G = x.hq / x.hkv;
  const PagedJoin y = joins[blockIdx.x / (uint32_t)x.hkv];
  const int v = (int)blockIdx.y * 4 + (threadIdx.x >> 6);
  if (v >= y.vecs) return;
  const int lane = threadIdx.x & 63, ch = lane & 15, sg = lane >> 4;
  constexpr int SB = 4;
  float m = -INFINITY, l = 0.f;
  f32x4 a0 = f32x4{}, a1 = f32x4{};
  for (int s0 = sg; s0 < y.parts; s0 += 4 * SB) {
    float2 ml[SB];
    f32x4 p0[SB], p1[SB];
#pragma unroll
    for (int j = 0; j < SB; ++j) {
      const int64_t slot = y.slot + (int64_t)y.step * min(s0 + 4 * j, y.parts - 1);
      const int64_t at = (slot * x.hkv + kvh) * 32 + v;
      ml[j] = *(const float2*)(x.ml_part + at * 2);
      p0[j] = *(const f32x4*)(x.o_part + at * 128 + 8 * ch);
      p1[j] = *(const f32x4*)(x.o_part + at * 128 + 8 * ch + 4);
    }
    float mb = m;
#pragma unroll
    for (int j = 0; j < SB; ++j) {
      if (s0 + 4 * j >= y.parts) {  // (the last part's again: 0 * infinity would be NaN)
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
    if (c.cache_bf16) hipLaunchKernelGGL((paged_attn_kernel<2, 8>), grid, dim3(512), 0, s, a);
    else hipLaunchKernelGGL((paged_attn_kernel<1, 8>), grid, dim3(512), 0, s, a);
    DRT_HIP(hipGetLastError());
  }
  if (c.n_joins) {
    hipLaunchKernelGGL(paged_join_kernel, dim3((unsigned)c.n_joins * (unsigned)c.hkv, 8), dim3(256), 0,
                       s, a, (const PagedJoin*)(c.list + c.joins));
    DRT_HIP(hipGetLastError());
  }
}

}  // namespace drt
