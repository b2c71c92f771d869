// A batch of sequences over a paged cache: what the host checks, and the work list that the kernels of
// paged.hip and paged_attention.hip read. Plain host code (the kernels use its structures only).
//
// Pages are page_size keys (a power of two, whole 32-key tiles) of every K/V head, tiles as
// everywhere in this library: tile i of head h in page g is tile (g * hkv + h) * tpp + i of the layer,
// tpp = page_size / 32. The list holds pages as g * hkv * tpp, the tile that its head 0 begins with.
// Every index that a kernel takes from the list has been checked here against the cache and the rows.
#pragma once
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>
#include <vector>

namespace drt {

// A work-group's part of an attention: up to `vecs` query vectors (row * G + head of the group, G = hq
// / hkv) of one sequence over tiles [tile0, tile1) of its keys. Read by scalar loads: 64 bytes.
struct PagedPiece {
  int32_t row0, rows;        // the sequence's rows in the batch
  int32_t pos0, keys, prompt_len;
  int32_t vec0;              // first query vector of the unit, within the sequence
  int32_t tile0, tile1;
  int32_t slot;              // where its part goes (32 query vectors a slot); < 0: the whole unit
  int32_t table;             // the sequence's first page in the list
  int32_t unused[6];
};
// 32 query vectors of a unit whose keys are split: their parts are in slots slot, slot + step, ...
struct PagedJoin {
  int32_t row0, vec0, vecs, slot, step, parts;
  int32_t unused[2];
};
// Rows of one sequence in one tile: keys [lo, hi) of the tile are rows row.. of the batch.
struct PagedTile {
  int32_t tile;  // of head 0
  int32_t lo, hi, row, pos;
  int32_t unused[3];
};
static_assert(sizeof(PagedPiece) == 64 && sizeof(PagedJoin) == 32 && sizeof(PagedTile) == 32, "");

struct PagedBatchArgs {
  int32_t seqs = 0, width = 0;       // table [seqs][width]
  const int32_t *table = nullptr, *rows = nullptr, *keys = nullptr, *pos0 = nullptr,
                *prompt_len = nullptr;  // (prompt_len may be null: 0)
  int32_t page_size = 0, pages = 0, hq = 0, hkv = 0, masked = 0, block = 1;
};

// Where the parts of a list begin, in 32-bit words, and how many there are.
struct PagedPlanInfo {
  // appendable: every row lies inside its sequence's keys, and none in the tile of another sequence's
  int32_t rows = 0, appendable = 1;
  int32_t n_small = 0, n_large = 0, n_joins = 0, n_tiles = 0, slots = 0;
  int64_t small = 0, large = 0, joins = 0, tiles = 0, table = 0, words = 0;
};

constexpr int PAGED_VECS = 32;      // query vectors of a unit of the small kernel
constexpr int PAGED_VECS_L = 256;   // ... of the large one
// Sequences of up to so many query vectors a K/V head go to the small kernel.
constexpr int PAGED_SMALL = INT32_MAX;
constexpr int PAGED_CUS = 256;

// The number of keys that the row at position p sees, always the first ones.
inline int64_t paged_key_end(int64_t p, int64_t keys, bool masked, int64_t prompt_len, int64_t block) {
  if (!masked) return keys;
  if (p < prompt_len) return std::min(keys, prompt_len);
  return std::min(keys, prompt_len + ((p - prompt_len) / block + 1) * block);
}

// "" or what is wrong with a batch.
inline std::string paged_check(const PagedBatchArgs& a) {
  const auto at = [](int s) { return "sequence " + std::to_string(s) + ": "; };
  if (a.page_size < 32 || (a.page_size & (a.page_size - 1))) return "page_size must be a power of two from 32 on";
  if (a.seqs < 1 || a.width < 0 || !a.rows || !a.keys || !a.pos0 || (a.width && !a.table))
    return "a batch has a sequence at least, and rows, keys and positions of each";
  if (a.hkv < 1 || a.hq < 1 || a.hq % a.hkv) return "query heads must be a multiple of the K/V heads";
  if (a.pages < 1 || (int64_t)a.pages * a.hkv * (a.page_size / 32) > INT32_MAX)
    return "a layer has at most 2^31 - 1 tiles of 32 keys and one head";
  if (a.masked && a.block < 1) return "bad mask geometry";
  int64_t total = 0;
  for (int s = 0; s < a.seqs; ++s) {
    const int64_t rows = a.rows[s], keys = a.keys[s], pos0 = a.pos0[s];
    if (rows < 0 || keys < 0 || pos0 < 0 || pos0 + rows > INT32_MAX)
      return at(s) + "rows, keys and positions are whole numbers of 32 bits from zero on";
    if (a.prompt_len && a.prompt_len[s] < 0) return at(s) + "bad mask geometry";
    if (keys > INT32_MAX - 64) return at(s) + "too many keys";
    const int64_t need = (keys + a.page_size - 1) / a.page_size;
    if (need > a.width) return at(s) + "its keys need more pages than it lists";
    for (int64_t i = 0; i < need; ++i) {
      const int32_t g = a.table[(int64_t)s * a.width + i];
      if (g < 0 || g >= a.pages)
        return at(s) + "page " + std::to_string(g) + " is outside the cache's " + std::to_string(a.pages);
    }
    total += rows;
  }
  if (total < 1) return "a batch has a row at least";
  if (total * (a.hq / a.hkv) > INT32_MAX - 1024) return "too many rows for one batch";
  return "";
}

namespace paged_detail {

struct Unit {
  int seq, vec0, vecs;
  int64_t tiles;
  int parts;
};

// How a kernel's units are cut along their keys: the parts of each. Times in us: `fixed` a part, `tile`
// 32 keys of one, `join` for the second launch, `part` a part's 32 query vectors written and read;
// `at_once` work-groups run side by side.
struct Costs {
  double fixed, tile, join, part;
  int at_once;
};
inline void cut(std::vector<Unit>& units, int hkv, const Costs& c) {
  int64_t most = 0;
  for (const Unit& u : units) most = std::max(most, u.tiles);
  if (most < 2) return;
  double best = -1.;
  int64_t best_len = most;
  // lengths of a part from whole units down, each about a fifth shorter than the last
  for (int64_t len = most; len >= 1; len = std::min(len - 1, len * 4 / 5)) {
    double longest = 0., sum = 0.;
    int64_t extra = 0;
    for (const Unit& u : units) {
      const int64_t n = std::max<int64_t>(1, (u.tiles + len - 1) / len);
      if (n > 256) { sum = -1.; break; }
      const double one = c.fixed + c.tile * (double)((u.tiles + n - 1) / n);
      longest = std::max(longest, one);
      sum += one * (double)n;
      if (n > 1) extra += n * ((u.vecs + 31) / 32);
    }
    if (sum < 0.) break;
    const double us = std::max(longest, sum * hkv / c.at_once) +
                      (extra ? c.join + c.part * (double)extra * hkv : 0.);
    if (best < 0. || us < best) {
      best = us;
      best_len = len;
    }
  }
  for (Unit& u : units) u.parts = (int)std::max<int64_t>(1, (u.tiles + best_len - 1) / best_len);
}

}  // namespace paged_detail

// The list of a checked batch.
inline PagedPlanInfo paged_plan(const PagedBatchArgs& a, std::vector<int32_t>& out) {
  using namespace paged_detail;
  PagedPlanInfo p;
  const int G = a.hq / a.hkv, tpp = a.page_size / 32;
  std::vector<int32_t> row0(a.seqs);
  std::vector<int64_t> table0(a.seqs);
  std::vector<Unit> units[2];
  std::vector<PagedTile> tiles;
  std::vector<int32_t> written;  // the tiles' numbers, to find two rows in one place
  int64_t n_table = 0;
  for (int s = 0; s < a.seqs; ++s) {
    row0[s] = p.rows;
    p.rows += a.rows[s];
    table0[s] = n_table;
    n_table += (a.keys[s] + (int64_t)a.page_size - 1) / a.page_size;
    const int64_t vecs = (int64_t)a.rows[s] * G;
    const bool large = vecs > PAGED_SMALL;
    const int step = large ? PAGED_VECS_L : PAGED_VECS;
    for (int64_t v = 0; v < vecs; v += step) {
      const int n = (int)std::min<int64_t>(step, vecs - v);
      const int64_t end = paged_key_end(a.pos0[s] + (v + n - 1) / G, a.keys[s], a.masked != 0,
                                        a.prompt_len ? a.prompt_len[s] : 0, a.block);
      units[large].push_back(Unit{s, (int)v, n, (end + 31) / 32, 1});
    }
    // the tiles that rows inside the sequence's keys lie in
    const int32_t* pg = a.table + (int64_t)s * a.width;
    const int64_t last = std::min<int64_t>(a.keys[s], (int64_t)a.pos0[s] + a.rows[s]);
    if (a.rows[s] && last < (int64_t)a.pos0[s] + a.rows[s]) p.appendable = 0;
    for (int64_t pos = a.pos0[s]; pos < last;) {
      const int64_t t = pos / 32, end = std::min(last, (t + 1) * 32);
      PagedTile y{};
      y.tile = pg[t / tpp] * a.hkv * tpp + (int)(t % tpp);
      y.lo = (int)(pos % 32);
      y.hi = y.lo + (int)(end - pos);
      y.row = row0[s] + (int)(pos - a.pos0[s]);
      y.pos = (int)pos;
      tiles.push_back(y);
      pos = end;
    }
  }
  // (a tile is written by one work-group: two parts of one tile are refused even side by side)
  written.reserve(tiles.size());
  for (const PagedTile& t : tiles) written.push_back(t.tile);
  std::sort(written.begin(), written.end());
  if (std::adjacent_find(written.begin(), written.end()) != written.end()) p.appendable = 0;

  cut(units[0], a.hkv, Costs{3.0, 0.055, 4.0, 0.004, PAGED_CUS});
  cut(units[1], a.hkv, Costs{4.0, 0.9, 4.0, 0.004, PAGED_CUS});
  std::vector<PagedPiece> pieces[2];
  std::vector<PagedJoin> joins;
  int slot = 0;
  for (int k = 0; k < 2; ++k) {
    for (const Unit& u : units[k]) {
      const int s = u.seq, subs = (u.vecs + 31) / 32;
      for (int i = 0; i < u.parts; ++i) {
        PagedPiece y{};
        y.row0 = row0[s];
        y.rows = a.rows[s];
        y.pos0 = a.pos0[s];
        y.keys = a.keys[s];
        y.prompt_len = a.prompt_len ? a.prompt_len[s] : 0;
        y.vec0 = u.vec0;
        y.tile0 = (int)(u.tiles * i / u.parts);
        y.tile1 = (int)(u.tiles * (i + 1) / u.parts);
        y.slot = u.parts > 1 ? slot + i * subs : -1;
        y.table = (int)table0[s];
        pieces[k].push_back(y);
      }
      if (u.parts == 1) continue;
      for (int j = 0; j < subs; ++j) {
        PagedJoin y{};
        y.row0 = row0[s];
        y.vec0 = u.vec0 + 32 * j;
        y.vecs = std::min(32, u.vecs - 32 * j);
        y.slot = slot + j;
        y.step = subs;
        y.parts = u.parts;
        joins.push_back(y);
      }
      slot += subs * u.parts;
    }
    // the longest first (parts of one length keep their order: neighbours read the same keys)
    std::stable_sort(pieces[k].begin(), pieces[k].end(), [](const PagedPiece& x, const PagedPiece& y) {
      return x.tile1 - x.tile0 > y.tile1 - y.tile0;
    });
  }
  p.n_small = (int)pieces[0].size();
  p.n_large = (int)pieces[1].size();
  p.n_joins = (int)joins.size();
  p.n_tiles = (int)tiles.size();
  p.slots = slot;
  out.clear();
  auto put = [&](const void* data, size_t words) {
    const int64_t at = (int64_t)out.size();
    const int32_t* w = (const int32_t*)data;
    out.insert(out.end(), w, w + words);
    return at;
  };
  p.small = put(pieces[0].data(), pieces[0].size() * 16);
  p.large = put(pieces[1].data(), pieces[1].size() * 16);
  p.joins = put(joins.data(), joins.size() * 8);
  p.tiles = put(tiles.data(), tiles.size() * 8);
  p.table = (int64_t)out.size();
  for (int s = 0; s < a.seqs; ++s) {
    const int64_t n = (a.keys[s] + (int64_t)a.page_size - 1) / a.page_size;
    for (int64_t i = 0; i < n; ++i) out.push_back(a.table[(int64_t)s * a.width + i] * a.hkv * tpp);
  }
  p.words = (int64_t)out.size();
  return p;
}

}  // namespace drt
