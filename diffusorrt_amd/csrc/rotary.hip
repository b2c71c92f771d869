// Rotary positions of rows of heads (rotary.h has the angle and its cosine and sine).
//
// Bound by its bytes, each read and written once: a thread makes the cosines and sines of 8 pairs (half
// layout) or 4 (interleaved) once and turns those of one or two heads, 16 or 32 bytes a load. 8192 rows x 16 heads
// of bf16: 11.8 us, 67 MB at 5.7 TB/s (a large copy's 4.9 is of more than the last-level cache holds); 1000
// rows x 28 heads of fp32 7.0; one row 2.3, its launch.
#include "launch.h"
#include "rotary.h"

namespace {

struct RotateArgs {
  const void* x;
  void* y;
  int64_t x_row, x_head, y_row, y_head;  // strides in elements
  const int32_t* positions;              // null: pos0 + row
  const uint64_t* freq;                  // [dim / 2]
  float magnitude;
  int pos0, rows, heads, hd, dim, inverse;
  int items, groups, per;  // threads a head; groups of `per` heads
};

DRT_DEV float2 turn_at(const RotateArgs& a, int p, int pair) {
  float2 cs = rotary_cos_sin(rotary_turn(a.freq[pair], p));
  cs.x *= a.magnitude;
  cs.y *= a.inverse ? -a.magnitude : a.magnitude;
  return cs;
}

// dim a multiple of 16 (half) or 8 (interleaved), hd of 8.
template <int DT, bool HALF>
__global__ __launch_bounds__(256) void rotate_kernel(const RotateArgs a) {
  constexpr int SIZE = DT == 0 ? 4 : 2;
  const uint32_t id = blockIdx.x * 256u + threadIdx.x;
  const uint32_t per_row = (uint32_t)(a.items * a.groups), row = id / per_row;
  if (row >= (uint32_t)a.rows) return;
  const uint32_t in_row = id - row * per_row, group = in_row / (uint32_t)a.items;
  const int j = (int)(in_row - group * (uint32_t)a.items);
  const int h0 = (int)group * a.per, h1 = min(h0 + a.per, a.heads);
  const int turned = HALF ? a.dim / 16 : a.dim / 8;
  // the first element of this thread's eight, and (half) of their partners
  const int e0 = HALF && j >= turned ? 8 * (j + turned) : 8 * j, e1 = e0 + a.dim / 2;
  const char* x = (const char*)a.x + ((int64_t)row * a.x_row + (int64_t)h0 * a.x_head + e0) * SIZE;
  char* y = (char*)a.y + ((int64_t)row * a.y_row + (int64_t)h0 * a.y_head + e0) * SIZE;
  const int64_t dx = a.x_head * SIZE, dy = a.y_head * SIZE, up = (int64_t)(e1 - e0) * SIZE;
  if (j >= turned) {  // elements that are not turned
    for (int h = h0; h < h1; ++h, x += dx, y += dy) {
      float v[8];
      rotary_load8<DT>(x, v);
      rotary_store8<DT>(y, v);
    }
    return;
  }
  const int p = a.positions ? a.positions[row] : a.pos0 + (int)row;
  constexpr int PAIRS = HALF ? 8 : 4;
  float c[PAIRS], s[PAIRS];
#pragma unroll
  for (int i = 0; i < PAIRS; ++i) {
    const float2 cs = turn_at(a, p, PAIRS * j + i);
    c[i] = cs.x;
    s[i] = cs.y;
  }
  for (int h = h0; h < h1; ++h, x += dx, y += dy) {
    float u[8], v[8];
    rotary_load8<DT>(x, u);
    if (HALF) {
      rotary_load8<DT>(x + up, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) rotary_turn_pair(u[i], v[i], c[HALF ? i : 0], s[HALF ? i : 0]);
      rotary_store8<DT>(y + up, v);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) rotary_turn_pair(u[2 * i], u[2 * i + 1], c[i], s[i]);
    }
    rotary_store8<DT>(y, u);
  }
}

// Any even dim: a thread a pair, then one an element that is not turned. Bound by its index divisions and
// narrow loads: 4096 rows x 16 heads of bf16, 72 of 128 elements 24.6 us, 34 MB at 1.4 TB/s; 250 of 256 31.7.
template <int DT>
__global__ __launch_bounds__(256) void rotate_any_kernel(const RotateArgs a, bool half) {
  const int pairs = a.dim / 2, per_head = pairs + (a.hd - a.dim);
  const int64_t n = (int64_t)a.rows * a.heads * per_head;
  for (int64_t id = blockIdx.x * (int64_t)256 + threadIdx.x; id < n; id += gridDim.x * (int64_t)256) {
    const int j = (int)(id % per_head);
    const int64_t rh = id / per_head;
    const int row = (int)(rh / a.heads), head = (int)(rh % a.heads);
    const int64_t x = (int64_t)row * a.x_row + (int64_t)head * a.x_head;
    const int64_t y = (int64_t)row * a.y_row + (int64_t)head * a.y_head;
    if (j >= pairs) {
      const int e = a.dim + (j - pairs);
      rotary_store1<DT>(a.y, y + e, rotary_load1<DT>(a.x, x + e));
      continue;
    }
    const float2 cs = turn_at(a, a.positions ? a.positions[row] : a.pos0 + row, j);
    const int e0 = half ? j : 2 * j, e1 = half ? j + pairs : 2 * j + 1;
    float u = rotary_load1<DT>(a.x, x + e0), v = rotary_load1<DT>(a.x, x + e1);
    rotary_turn_pair(u, v, cs.x, cs.y);
    rotary_store1<DT>(a.y, y + e0, u);
    rotary_store1<DT>(a.y, y + e1, v);
  }
}

}  // namespace

namespace drt {

void rotate(const RotateCall& r, hipStream_t s) {
  RotateArgs a{};
  a.x = r.x;
  a.y = r.y;
  a.x_row = r.x_row;
  a.x_head = r.x_head;
  a.y_row = r.y_row;
  a.y_head = r.y_head;
  a.positions = r.positions;
  a.freq = r.rotary.freq;
  a.magnitude = r.rotary.magnitude;
  a.pos0 = r.pos0;
  a.rows = r.rows;
  a.heads = r.heads;
  a.hd = r.hd;
  a.dim = r.rotary.dim;
  a.inverse = r.inverse;
  const bool half = r.rotary.half;
  const int turned = half ? a.dim / 16 : a.dim / 8;
  if (a.hd % 8 == 0 && a.dim % (half ? 16 : 8) == 0) {
    const int rest = r.x == r.y ? 0 : (a.hd - a.dim) / 8;  // (in place they are there already)
    a.items = turned + rest;
    // Two heads a thread, which share the angles, where that leaves work for the chip (bf16, us with two and
    // one: 2048 rows x 16 heads 5.3 and 5.6, 4096 7.7 and 8.2, 8192 12.0 and 12.9, 65536 94 and 96, 1000 3.9 both;
    // four take 0 to 7 % longer than two, eight 2 to 50 %).
    a.per = (int64_t)a.rows * a.items * a.heads > 131072 ? 2 : 1;
    a.groups = (a.heads + a.per - 1) / a.per;
    const int64_t threads = (int64_t)a.rows * a.items * a.groups;
    require(threads <= INT32_MAX - 256, "rotate: too many rows for one call");
    const dim3 grid((unsigned)((threads + 255) / 256));
#define DRT_ROT(DT)                                                                          \
  do {                                                                                       \
    if (half) hipLaunchKernelGGL((rotate_kernel<DT, true>), grid, dim3(256), 0, s, a);       \
    else hipLaunchKernelGGL((rotate_kernel<DT, false>), grid, dim3(256), 0, s, a);           \
  } while (0)
    if (r.type == 0) DRT_ROT(0);
    else if (r.type == 1) DRT_ROT(1);
    else DRT_ROT(2);
#undef DRT_ROT
  } else {
    const int64_t n = (int64_t)a.rows * a.heads * (a.dim / 2 + a.hd - a.dim);
    const dim3 grid((unsigned)std::min<int64_t>((n + 255) / 256, 16384));
    if (r.type == 0) hipLaunchKernelGGL(rotate_any_kernel<0>, grid, dim3(256), 0, s, a, half);
    else if (r.type == 1) hipLaunchKernelGGL(rotate_any_kernel<1>, grid, dim3(256), 0, s, a, half);
    else hipLaunchKernelGGL(rotate_any_kernel<2>, grid, dim3(256), 0, s, a, half);
  }
  DRT_HIP(hipGetLastError());
}

}  // namespace drt
