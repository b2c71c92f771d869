// The paged cache's appends, and reading rows back.
//
// Pages hold the 32-key tiles of the contiguous cache (attention.hip has their layout), which a page never
// ends inside. A work-group owns the rows that a batch puts into one tile (PagedTile) for some of the
// heads: it turns the keys of its K/V heads on their way into the tile and the queries of its heads on
// theirs into the attention's operand type, or takes values in, eight keys of a head dim a store where the
// rows hold all eight. Rows around those stay as they are, so batches that write other rows of one tile
// may overlap in time.
// Bound by its bytes where there are many rows (three prompts, 1301 rows x 16 + 8 heads of bf16: 8.4 us, 21 MB
// at 2.5 TB/s; 4.5 to read them back), else by its launch and two rounds of loads (64 tokens x 28 + 4 heads
// of fp32 4.8 us, 2.5 to read them back).
#include "launch.h"
#include "paged_plan.h"
#include "rotary.h"

namespace {

using drt::PagedTile;

struct AppendArgs {
  const void *q, *k, *v;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;  // strides in elements
  const PagedTile* tiles;
  uint16_t* cache;  // this layer
  uint16_t* q_out;  // [rows][hq][128]
  const uint64_t* freq;
  float magnitude;
  int dim, half;  // dim 0: no rotation
  int hq, hkv, tpp;
};

// A work-group's tile, by scalar loads.
DRT_DEV PagedTile tile_of(const PagedTile* tiles, int i) {
  const auto* p = (const __attribute__((address_space(4))) int32_t*)(uintptr_t)(tiles + i);
  PagedTile t;
  t.tile = p[0];
  t.lo = p[1];
  t.hi = p[2];
  t.row = p[3];
  t.pos = p[4];
  return t;
}

// The 16-bit elements' position of (key, head dim) of V in a tile; K's eight dims are 16 bytes at
// ((hd / 8) * 32 + key) * 8.
DRT_DEV int v_group_at(int hd, int group) {  // group = 2 (key / 16) + ((key >> 2) & 1)
  return 4096 + ((((hd >> 5) * 2 + (group >> 1)) * 2 + (group & 1)) * 32 + (hd & 31)) * 8;
}
DRT_DEV int v_key_of(int group, int j) { return 16 * (group >> 1) + 4 * (group & 1) + (j & 3) + 8 * (j >> 2); }

// Keys and queries: a thread has one place (key of the tile, sixteen elements that make pairs, or eight
// that are not turned) of several heads, so it makes its cosines and sines once; four heads' loads are on
// their way at a time.
template <int DT, int CT>
DRT_DEV void append_turned(const AppendArgs& a, const PagedTile& t, int part, int parts) {
  const int n = t.hi - t.lo, tid = threadIdx.x;
  const int units = a.hkv + (a.q ? a.hq : 0);
  const int u0 = units * part / parts, u1 = units * (part + 1) / parts;
  const bool half = a.half && a.dim;
  const int turned = half ? a.dim / 16 : a.dim / 8;
  const int items = half ? 16 - turned : 16, per = n * items;
  const int groups = max(1, 256 / per), group = per < 256 ? tid / per : 0;
  if (group >= groups) return;
  constexpr int SIZE = DT == 0 ? 4 : 2, AT_ONCE = 4;
  for (int i = tid - group * per; i < per; i += 256) {
    const int kk = i / items, j = i - kk * items;
    const int c0 = half && j >= turned ? j + turned : j, up = half ? turned : 0;
    const bool turns = j < turned, pairs8 = turns && half;
    const int64_t row = t.row + kk;
    const char* const kp = (const char*)a.k + (row * a.k_row + c0 * 8) * SIZE;
    const char* const qp = (const char*)a.q + (row * a.q_row + c0 * 8) * SIZE;
    float x[AT_ONCE][8], y[AT_ONCE][8];
    auto take = [&](int u) {
#pragma unroll
      for (int b = 0; b < AT_ONCE; ++b) {  // (behind the last head it again: not stored)
        const int h = min(u + b * groups, u1 - 1);
        const char* const from =
            h < a.hkv ? kp + h * a.k_head * SIZE : qp + (h - a.hkv) * a.q_head * SIZE;
        rotary_load8<DT>(from, x[b]);
        if (pairs8) rotary_load8<DT>(from + up * 8 * SIZE, y[b]);
      }
    };
    take(u0 + group);
    float c[8], s[8];
    if (turns) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (half || e < 4) {
          const float2 cs = rotary_cos_sin(rotary_turn(a.freq[(half ? 8 : 4) * j + e], t.pos + kk));
          c[e] = cs.x * a.magnitude;
          s[e] = cs.y * a.magnitude;
        }
    }
    for (int u = u0 + group; u < u1;) {
#pragma unroll
      for (int b = 0; b < AT_ONCE; ++b) {
        const int h = u + b * groups;
        if (h >= u1) break;
        const bool key = h < a.hkv;
        const int step = key ? 32 * 8 : 8;  // from chunk to chunk
        uint16_t* const to =
            (key ? a.cache + ((int64_t)t.tile + (int64_t)h * a.tpp) * 8192 + (t.lo + kk) * 8
                 : a.q_out + (row * a.hq + h - a.hkv) * 128) + c0 * step;
        if (pairs8) {
#pragma unroll
          for (int e = 0; e < 8; ++e) rotary_turn_pair(x[b][e], y[b][e], c[e], s[e]);
          *(u32x4*)(to + up * step) = rotary_pack8<CT>(y[b]);
        } else if (turns) {
#pragma unroll
          for (int e = 0; e < 4; ++e) rotary_turn_pair(x[b][2 * e], x[b][2 * e + 1], c[e], s[e]);
        }
        *(u32x4*)to = rotary_pack8<CT>(x[b]);
      }
      u += groups * AT_ONCE;
      if (u < u1) take(u);
    }
  }
}

// Values: a thread has two head dims of eight keys that are side by side in the tile, of several heads.
template <int DT, int CT>
DRT_DEV void append_values(const AppendArgs& a, const PagedTile& t, int part, int parts) {
  const int n = t.hi - t.lo, hd = 2 * (threadIdx.x & 63), group = threadIdx.x >> 6;
  int keys = 0;  // which of this thread's eight are the batch's
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int kk = v_key_of(group, j) - t.lo;
    keys |= kk >= 0 && kk < n ? 1 << j : 0;
  }
  if (!keys) return;
  for (int head = a.hkv * part / parts; head < a.hkv * (part + 1) / parts; ++head) {
    float x[2][8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int kk = min(max(v_key_of(group, j) - t.lo, 0), n - 1);
      const int64_t at = (int64_t)(t.row + kk) * a.v_row + head * a.v_head + hd;
      rotary_load2<DT>(a.v, at, x[0][j], x[1][j]);
    }
    uint16_t* const to =
        a.cache + ((int64_t)t.tile + (int64_t)head * a.tpp) * 8192 + v_group_at(hd, group);
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      const u32x4 w = rotary_pack8<CT>(x[d]);
      if (keys == 255) {
        *(u32x4*)(to + 8 * d) = w;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (keys >> j & 1) to[8 * d + j] = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
      }
    }
  }
}

template <int DT, int CT>
__global__ __launch_bounds__(256) void paged_append_kernel(const AppendArgs a, int parts, int v_parts) {
  const PagedTile t = tile_of(a.tiles, blockIdx.x);
  if ((int)blockIdx.y < parts) append_turned<DT, CT>(a, t, blockIdx.y, parts);
  else append_values<DT, CT>(a, t, blockIdx.y - parts, v_parts);
}

// Rows back from their tiles: keys by the first `parts` work-groups of a tile, values by the others.
__global__ __launch_bounds__(256) void paged_load_kernel(const PagedTile* tiles, const uint16_t* cache,
                                                         int hkv, int tpp, uint16_t* k, uint16_t* v,
                                                         int parts) {
  const PagedTile t = tile_of(tiles, blockIdx.x);
  const bool keys = (int)blockIdx.y < parts;
  const int part = blockIdx.y - (keys ? 0 : parts), tid = threadIdx.x;
  const int h0 = hkv * part / parts, h1 = hkv * (part + 1) / parts, n = t.hi - t.lo;
  if (keys) {
    const int per = n * 16, all = per * (h1 - h0);
    for (int i = tid; i < all; i += 256) {
      const int h = i / per, r = i - h * per, kk = r >> 4, c = r & 15;
      const uint16_t* from = cache + ((int64_t)t.tile + (int64_t)(h0 + h) * tpp) * 8192;
      *(u32x4*)(k + ((int64_t)(t.row + kk) * hkv + h0 + h) * 128 + c * 8) =
          *(const u32x4*)(from + (c * 32 + t.lo + kk) * 8);
    }
    return;
  }
  const int hd = 2 * (tid & 63), group = tid >> 6;
  for (int head = h0; head < h1; ++head) {
    const uint16_t* from = cache + ((int64_t)t.tile + (int64_t)head * tpp) * 8192 + v_group_at(hd, group);
    const u32x4 w0 = *(const u32x4*)from, w1 = *(const u32x4*)(from + 8);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int kk = v_key_of(group, j) - t.lo;
      if (kk >= 0 && kk < n) {
        const uint32_t a = w0[j >> 1] >> (16 * (j & 1)), b = w1[j >> 1] >> (16 * (j & 1));
        *(uint32_t*)(v + ((int64_t)(t.row + kk) * hkv + head) * 128 + hd) = (a & 0xffffu) | b << 16;
      }
    }
  }
}

// Work-groups a tile that share its K/V heads: one each, or one for two where there are many tiles and half as
// many do (us a head each and two: loads of 125 tiles x 8 heads 5.9 and 6.9, 42 x 8 3.9 and 4.7, 16 x 8 3.3 and 4.1;
// 2000 x 8 100 and 101, its append 229 and 230 to 235).
int heads_of(int n_tiles, int hkv) { return (int64_t)n_tiles * hkv <= 1024 ? hkv : (hkv + 1) / 2; }

}  // namespace

namespace drt {

void paged_append(const AppendCall& c, hipStream_t s) {
  AppendArgs a{};
  a.q = c.q;
  a.k = c.k;
  a.v = c.v;
  a.q_row = c.q_row;
  a.q_head = c.q_head;
  a.k_row = c.k_row;
  a.k_head = c.k_head;
  a.v_row = c.v_row;
  a.v_head = c.v_head;
  a.tiles = (const PagedTile*)c.tiles;
  a.cache = (uint16_t*)c.cache;
  a.q_out = (uint16_t*)c.q_out;
  a.freq = c.rotary.freq;
  a.magnitude = c.rotary.magnitude;
  a.dim = c.rotary.dim;
  a.half = c.rotary.half;
  a.hq = c.hq;
  a.hkv = c.hkv;
  a.tpp = c.tpp;
  // A tile's work-groups: heads enough for a thread's four at once, by the rows a tile has on average
  const int per = std::max(1, c.rows / c.n_tiles) * (a.half && a.dim ? 16 - a.dim / 16 : 16);
  const int at_once = 4 * std::max(1, 256 / per), units = c.hkv + (c.q ? c.hq : 0);
  const int parts = (units + at_once - 1) / at_once, v_parts = heads_of(c.n_tiles, c.hkv);
  const dim3 grid((unsigned)c.n_tiles, (unsigned)(parts + v_parts));
#define DRT_PA1(DT, CT) \
  hipLaunchKernelGGL((paged_append_kernel<DT, CT>), grid, dim3(256), 0, s, a, parts, v_parts)
#define DRT_PA(DT)                                                    \
  do { if (c.cache_bf16) DRT_PA1(DT, 2); else DRT_PA1(DT, 1); } while (0)
  if (c.type == 0) DRT_PA(0);
  else if (c.type == 1) DRT_PA(1);
  else DRT_PA(2);
#undef DRT_PA
#undef DRT_PA1
  DRT_HIP(hipGetLastError());
}

void paged_load(const void* tiles, int n_tiles, const void* cache, int hkv, int tpp, void* k, void* v,
                hipStream_t s) {
  const int parts = heads_of(n_tiles, hkv);
  const dim3 grid((unsigned)n_tiles, (unsigned)(2 * parts));
  hipLaunchKernelGGL(paged_load_kernel, grid, dim3(256), 0, s, (const PagedTile*)tiles,
                     (const uint16_t*)cache, hkv, tpp, (uint16_t*)k, (uint16_t*)v, parts);
  DRT_HIP(hipGetLastError());
}

}  // namespace drt
