// The paged cache's appends, and reading rows back.
//
// Pages hold the 32-key tiles of the contiguous cache (attention.hip has their layout), which a page never
// ends inside. A work-group owns the rows that a batch puts into one tile (PagedTile) for some of the
// heads: it makes the cosines and sines of their positions once, in LDS, and turns the keys of its K/V
// heads on their way into the tile and the queries of its heads on theirs into the attention's operand
// type. Values go in as they are, eight keys of a head dim a store where the rows hold all eight.
// Rows around those stay as they are, so batches that write other rows of one tile may overlap in time.
// Bound by its bytes where there are many rows, else by its launch and three rounds of loads.
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

// The 16-bit elements' position of (key, head dim) of V in a tile; K's eight dims are 16 bytes at
// ((hd / 8) * 32 + key) * 8.
DRT_DEV int v_group_at(int hd, int group) {  // group = 2 (key / 16) + ((key >> 2) & 1)
  return 4096 + ((((hd >> 5) * 2 + (group >> 1)) * 2 + (group & 1)) * 32 + (hd & 31)) * 8;
}
DRT_DEV int v_key_of(int group, int j) { return 16 * (group >> 1) + 4 * (group & 1) + (j & 3) + 8 * (j >> 2); }

template <int DT, int CT>
__global__ __launch_bounds__(256) void paged_append_kernel(const AppendArgs a) {
  __shared__ float2 turns[32 * 64];
  const PagedTile t = a.tiles[blockIdx.x];
  const int part = blockIdx.y, parts = gridDim.y, tid = threadIdx.x;
  const int kv0 = a.hkv * part / parts, nkv = a.hkv * (part + 1) / parts - kv0;
  const int q0 = a.q ? a.hq * part / parts : 0, nq = a.q ? a.hq * (part + 1) / parts - q0 : 0;
  const int n = t.hi - t.lo, pairs = a.dim / 2;
  if (a.dim) {
    if ((tid & 63) < pairs) {
      const uint64_t f = a.freq[tid & 63];
      for (int kk = tid >> 6; kk < n; kk += 4) {
        const float2 cs = rotary_cos_sin(rotary_turn(f, t.pos + kk));
        turns[kk * 64 + (tid & 63)] = make_float2(cs.x * a.magnitude, cs.y * a.magnitude);
      }
    }
    __syncthreads();
  }
  // keys and queries: sixteen chunks of eight dims a head; two that make pairs go together (half layout)
  const bool half = a.half && a.dim;
  const int turned = half ? a.dim / 16 : a.dim / 8;
  const uint32_t items = half ? 16 - turned : 16, per_head = items * n, all = per_head * (nkv + nq);
  for (uint32_t i = tid; i < all; i += 256) {
    const uint32_t h = i / per_head, r = i - h * per_head;
    const int kk = (int)(r / items), j = (int)(r - (uint32_t)kk * items);
    const bool key = (int)h < nkv;
    const int head = key ? kv0 + (int)h : q0 + (int)h - nkv;
    const int64_t row = t.row + kk;
    const int64_t src = key ? row * a.k_row + head * a.k_head : row * a.q_row + head * a.q_head;
    const char* from = (const char*)(key ? a.k : a.q) + src * (DT == 0 ? 4 : 2);
    const int step = key ? 32 * 8 : 8;  // from chunk to chunk
    uint16_t* to = key ? a.cache + ((int64_t)t.tile + (int64_t)head * a.tpp) * 8192 + (t.lo + kk) * 8
                       : a.q_out + (row * a.hq + head) * 128;
    const int c0 = half && j >= turned ? j + turned : j;
    constexpr int BYTES = DT == 0 ? 32 : 16;
    float x[8], y[8];
    rotary_load8<DT>(from + c0 * BYTES, x);
    if (j < turned) {
      const float2* cs = turns + kk * 64;
      if (half) {
        rotary_load8<DT>(from + (c0 + turned) * BYTES, y);
#pragma unroll
        for (int e = 0; e < 8; ++e) rotary_turn_pair(x[e], y[e], cs[8 * j + e].x, cs[8 * j + e].y);
        *(u32x4*)(to + (c0 + turned) * step) = rotary_pack8<CT>(y);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          rotary_turn_pair(x[2 * e], x[2 * e + 1], cs[4 * j + e].x, cs[4 * j + e].y);
      }
    }
    *(u32x4*)(to + c0 * step) = rotary_pack8<CT>(x);
  }
  for (int i = tid; i < nkv * 512; i += 256) {
    const int hd = i & 127, group = (i >> 7) & 3, head = kv0 + (i >> 9);
    float x[8];
    bool all = true, any = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int kk = v_key_of(group, j) - t.lo;
      const bool in = kk >= 0 && kk < n;
      all = all && in;
      any = any || in;
    }
    if (!any) continue;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int kk = min(max(v_key_of(group, j) - t.lo, 0), n - 1);
      x[j] = rotary_load1<DT>(a.v, (int64_t)(t.row + kk) * a.v_row + head * a.v_head + hd);
    }
    uint16_t* to = a.cache + ((int64_t)t.tile + (int64_t)head * a.tpp) * 8192 + v_group_at(hd, group);
    const u32x4 w = rotary_pack8<CT>(x);
    if (all) {
      *(u32x4*)to = w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int kk = v_key_of(group, j) - t.lo;
        if (kk >= 0 && kk < n) to[j] = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
      }
    }
  }
}

__global__ __launch_bounds__(256) void paged_load_kernel(const PagedTile* tiles, const uint16_t* cache,
                                                         int hkv, int tpp, uint16_t* k, uint16_t* v) {
  const PagedTile t = tiles[blockIdx.x];
  const int part = blockIdx.y, parts = gridDim.y, tid = threadIdx.x;
  const int kv0 = hkv * part / parts, nkv = hkv * (part + 1) / parts - kv0;
  const uint32_t n = t.hi - t.lo, all = n * 16 * nkv;
  for (uint32_t i = tid; i < all; i += 256) {
    const uint32_t h = i / (16 * n), r = i - h * 16 * n, kk = r >> 4, c = r & 15;
    const int64_t at = ((int64_t)(t.row + kk) * hkv + kv0 + h) * 128;
    const uint16_t* from = cache + ((int64_t)t.tile + (int64_t)(kv0 + h) * tpp) * 8192;
    *(u32x4*)(k + at + c * 8) = *(const u32x4*)(from + (c * 32 + t.lo + kk) * 8);
  }
  for (int i = tid; i < nkv * 512; i += 256) {
    const int hd = i & 127, group = (i >> 7) & 3, head = kv0 + (i >> 9);
    const u32x4 w = *(const u32x4*)(cache + ((int64_t)t.tile + (int64_t)head * tpp) * 8192 +
                                    v_group_at(hd, group));
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int kk = v_key_of(group, j) - t.lo;
      if (kk >= 0 && kk < (int)n)
        v[((int64_t)(t.row + kk) * hkv + head) * 128 + hd] = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
    }
  }
}

// Work-groups a tile: as many as fill the chip twice, each with a K/V head at least.
int parts_of(int n_tiles, int hkv) { return std::max(1, std::min(hkv, (512 + n_tiles - 1) / n_tiles)); }

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
  const dim3 grid((unsigned)c.n_tiles, (unsigned)parts_of(c.n_tiles, c.hkv));
#define DRT_PA(DT)                                                                                 \
  do {                                                                                             \
    if (c.cache_bf16) hipLaunchKernelGGL((paged_append_kernel<DT, 2>), grid, dim3(256), 0, s, a);  \
    else hipLaunchKernelGGL((paged_append_kernel<DT, 1>), grid, dim3(256), 0, s, a);               \
  } while (0)
  if (c.type == 0) DRT_PA(0);
  else if (c.type == 1) DRT_PA(1);
  else DRT_PA(2);
#undef DRT_PA
  DRT_HIP(hipGetLastError());
}

void paged_load(const void* tiles, int n_tiles, const void* cache, int hkv, int tpp, void* k, void* v,
                hipStream_t s) {
  const dim3 grid((unsigned)n_tiles, (unsigned)parts_of(n_tiles, hkv));
  hipLaunchKernelGGL(paged_load_kernel, grid, dim3(256), 0, s, (const PagedTile*)tiles,
                     (const uint16_t*)cache, hkv, tpp, (uint16_t*)k, (uint16_t*)v);
  DRT_HIP(hipGetLastError());
}

}  // namespace drt
