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
#include <map>
#include <string>
#include <vector>

namespace drt {

// A part of an attention: a unit of query vectors (row * G + head of the group, G = hq / hkv) of one
// sequence over tiles [tile0, tile1) of its keys. A work-group of the large kernel does some that follow one
// another: the last of them says so. Read by scalar loads: 64 bytes.
struct PagedPiece {
  int32_t row0, rows;        // the sequence's rows in the batch
  int32_t pos0, keys, prompt_len;
  int32_t vec0;              // first query vector of the unit, within the sequence
  int32_t tile0, tile1;
  int32_t slot;              // where its part goes (32 query vectors a slot); < 0: the whole unit
  int32_t table;             // the sequence's first page in the list
  int32_t last;              // a work-group's last
  int32_t wide;              // (small kernel) its unit is of up to 64 query vectors, not 32
  int32_t unused[4];
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
  // work-groups of a K/V head for each kernel: of the small one a part each, of the large one from part
  // first_large[i] on to its last
  int32_t n_small = 0, n_large = 0, n_joins = 0, n_tiles = 0, slots = 0;
  int64_t small = 0, large = 0, first_large = 0;
  int64_t joins = 0, tiles = 0, table = 0, words = 0;
};

// Query vectors of a unit: of the small kernel, 32 or 64, and of the large one.
constexpr int PAGED_VECS = 32, PAGED_VECS_M = 64, PAGED_VECS_L = 256;
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
  if (a.hkv < 1 || a.hq < 1 || a.hq % a.hkv || a.hq > 16384)
    return "query heads must be a multiple of the K/V heads, 16384 at most";
  if (a.pages < 1 || a.pages > INT32_MAX / ((int64_t)a.hkv * (a.page_size / 32)))
    return "a layer has at most 2^31 - 1 tiles of 32 keys and one head";
  if (a.masked && a.block < 1) return "bad mask geometry";
  int64_t total = 0, listed = 0;
  for (int s = 0; s < a.seqs; ++s) listed += (std::max(a.keys[s], 0) + (int64_t)a.page_size - 1) / a.page_size;
  if (listed > INT32_MAX) return "too many pages for one batch";
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
  double beside = 1.;  // units of the sequence
};

// Times in us. A part: `fixed` (its queries in, its result out) and `tile` for 32 keys, on its CU; where
// units read the same keys side by side those come from the L2, else each is `alone` in waiting for memory;
// JOIN, LARGE_JOIN: the second launch that a cut needs. Of 181 batches of 1 to 48 sequences (1 to 1000 rows, 300 to
// 60000 keys, 16 heads on 8, 28 on 4, 32 on 2; profiles/paged_plan_batches.csv) what these times choose is
// 2.2 % slower on average than the fastest of both units at up to 15 lengths of parts, in 30 of them by more
// than 5 %, by 25 % at worst (48 tokens x 28 heads over 12000 keys: 134 us, 108 in parts a quarter as long).
struct Costs {
  double fixed, tile, alone;
};
constexpr Costs SMALL{5., 0.147, 0.143}, MEDIUM{7., 0.235, 0.13}, LARGE{12., 0.74, 0.};
constexpr double JOIN = 3.3, LARGE_JOIN = 20.;
// What the large kernel's equal shares are cut by: a tile counts for more than in a whole unit's time. Cut by
// LARGE, eight of ten batches take 0 to 2 % longer (700 rows x 28 heads over 16000 keys 200 us for 196, 2048 over
// 70000 1830 for 1821; 1400 rows x 64 heads beside tokens 933 for 947).
constexpr Costs LARGE_SHARES{12., 0.875, 0.};
// The part [tile0, tile1) of unit `unit` for work-group `group`.
struct Share {
  int unit, group;
  int64_t tile0, tile1;
};
// Units in their order as the shares of work-groups of equal time, `groups` of them at most. A share ends
// inside a unit where it must; not within the time of a part's fixed cost of the unit's ends, where the cut
// would cost what it saves.
inline std::vector<Share> cut(const std::vector<Unit>& units, int groups, const Costs& c) {
  std::vector<Share> out;
  double left = 0.;
  for (const Unit& u : units) left += c.fixed + c.tile * (double)u.tiles;
  int group = 0;
  const int64_t least = std::max<int64_t>(1, (int64_t)(c.fixed / c.tile));  // tiles worth a cut
  double mine = 0., quota = left / groups;
  for (int i = 0; i < (int)units.size(); ++i) {
    int64_t at = 0;
    const int64_t tiles = units[i].tiles;
    for (;;) {
      int64_t n = tiles - at;
      const double room = quota - mine - c.fixed;
      bool full = false;
      if (group + 1 < groups && room < c.tile * (double)n) {  // it does not all fit
        full = true;
        int64_t fit = room > 0. ? (int64_t)(room / c.tile) : 0;
        if (n - fit < least) fit = n;
        if (fit < least) fit = 0;
        if (fit == 0 && mine == 0.) fit = std::min(n, least);
        n = fit;
      }
      if (n > 0 || (tiles == 0 && !full)) {
        out.push_back(Share{i, group, at, at + n});
        mine += c.fixed + c.tile * (double)n;
        at += n;
      }
      if (full) {
        left -= mine;
        ++group;
        mine = 0.;
        // (what is left, evenly; a unit cut here begins once more)
        quota = (left + (at > 0 && at < tiles ? c.fixed : 0.)) / (groups - group);
        if (at > 0 && at < tiles) left += c.fixed;
      }
      if (at >= tiles && (tiles > 0 || n > 0 || !full)) break;
    }
  }
  return out;
}

// The time of work-groups, `slots` of them at once, the longest first, each where one before it ends; parts:
// (us, how many). Times within 4 % are taken as one, and many rounds as even ones: a plan is made once a step.
// (Places are an XCD's, to which a work-group belongs by its number: where some wait for one they end later
// than that by up to half of the longest of them.)
inline double makespan(std::vector<std::pair<double, int64_t>>& parts, int slots) {
  int64_t all = 0;
  double longest = 0., sum = 0.;
  for (const auto& y : parts) {
    all += y.second;
    longest = std::max(longest, y.first);
    sum += y.first * (double)y.second;
  }
  if (all <= slots) return longest;
  std::sort(parts.begin(), parts.end(), std::greater<std::pair<double, int64_t>>());
  double last = longest, waits = 0.;
  int64_t before = 0;
  for (const auto& y : parts) {
    before += y.second;
    if (before > slots) {
      waits = y.first;
      break;
    }
  }
  if (all <= 4 * slots) {
    std::map<double, int64_t> free_at{{0., slots}};
    for (size_t i = 0; i < parts.size();) {
      const double us = parts[i].first;
      int64_t n = 0;
      for (; i < parts.size() && parts[i].first > 0.96 * us; ++i) n += parts[i].second;
      while (n > 0) {
        const auto at = free_at.begin();
        const int64_t k = std::min(n, at->second);
        const double end = at->first + us;
        n -= k;
        at->second -= k;
        if (at->second == 0) free_at.erase(at);
        free_at[end] += k;
        last = std::max(last, end);
      }
    }
  }
  return std::max(last, sum / slots + 0.5 * waits);
}

// (us, longest part in tiles) of units that are cut into equal parts, each a work-group of its own, by the
// least time of all. all_us: what reading the keys of all sequences once takes; the nearer the work-groups'
// own time comes to that, the more they wait for one another.
inline std::pair<double, int64_t> part_length(const std::vector<Unit>& units, int hkv, double all_us) {
  std::vector<std::pair<double, int64_t>> parts;
  int64_t most = 0;
  for (const Unit& u : units) most = std::max(most, u.tiles);
  double best = -1.;
  int64_t best_len = std::max<int64_t>(1, most);
  for (int64_t len = best_len; len >= 1; len = std::min(len - 1, len * 3 / 4)) {
    parts.clear();
    int64_t cuts = 0, most_cuts = 0;
    for (const Unit& u : units) {
      const int64_t n = std::max<int64_t>(1, (u.tiles + len - 1) / len);
      const Costs& c = u.vecs > PAGED_VECS ? MEDIUM : SMALL;
      parts.emplace_back(c.fixed + (c.tile + c.alone / u.beside) * (double)((u.tiles + n - 1) / n), n * hkv);
      cuts += n > 1 ? n * ((u.vecs + 31) / 32) : 0;
      most_cuts = std::max(most_cuts, n);
    }
    if (most_cuts > 128) break;
    const double own = makespan(parts, PAGED_CUS), all = SMALL.fixed + all_us;
    const double us = std::sqrt(std::sqrt(own * own * own * own + all * all * all * all)) +
                      (cuts ? JOIN + 0.008 * (double)(cuts * hkv) : 0.);
    if (best < 0. || us < best) {
      best = us;
      best_len = len;
    }
    // (whole units that take no longer than all of the work spread evenly)
    if (len >= most) {
      double sum = 0.;
      for (const auto& y : parts) sum += y.first * (double)y.second;
      if (own <= 1.1 * std::max(all, sum / PAGED_CUS)) break;
    }
  }
  return {best, best_len};
}

// Units of the large kernel: each a work-group of its own, or all of them in equal shares whose parts are
// joined (0.009 us for 32 query vectors of a part written and read).
struct LargeTimes {
  double whole = 0., cut = 0.;
};
inline LargeTimes large_times(const std::vector<Unit>& units, int hkv) {
  LargeTimes y;
  if (units.empty()) return y;
  const int groups = std::max(1, PAGED_CUS / hkv);
  std::vector<std::pair<double, int64_t>> parts;
  double sum = 0.;
  for (const Unit& u : units) {
    parts.emplace_back(LARGE.fixed + LARGE.tile * (double)u.tiles, hkv);
    sum += parts.back().first;
  }
  y.whole = makespan(parts, PAGED_CUS);
  y.cut = sum / groups + LARGE.fixed + LARGE_JOIN + 0.009 * 8. * (double)(units.size() + groups) * hkv;
  return y;
}

// The order of the small kernel's pieces: the longest first (lengths within 8 tiles are one: 32 rows x 28 heads
// over 60000 keys 48.5 us, sorted to the tile 50.1). Work-groups go round the 8 XCDs, each with an
// L2 of its own, and a piece's K/V heads follow one another: pieces of one sequence's same keys (`same`) are
// put so that they come to the same XCDs, as long as there are others to take the places between (eight
// sequences of 9 rows x 28 heads over up to 2500 keys 12.1 us with their join, in the units' order 13.3; sixteen
// of 32 rows 52 and 54; 17 or 32 rows alone alike).
inline void side_by_side(std::vector<PagedPiece>& pieces, const std::vector<int>& same, int hkv) {
  int lanes = 8;
  for (int h = hkv; lanes > 1 && h % 2 == 0; h /= 2) lanes /= 2;
  std::vector<int> order(pieces.size()), count, lane_of;
  for (size_t i = 0; i < order.size(); ++i) order[i] = (int)i;
  std::stable_sort(order.begin(), order.end(), [&](int x, int y) {
    return (pieces[x].tile1 - pieces[x].tile0) / 8 > (pieces[y].tile1 - pieces[y].tile0) / 8;
  });
  for (const int y : same) {
    if (y >= (int)count.size()) count.resize(y + 1);
    ++count[y];
  }
  lane_of.assign(count.size(), -1);
  std::vector<std::vector<int>> lane(lanes);
  std::vector<size_t> size(lanes, 0);
  for (const int i : order) {
    int to = lane_of[same[i]];
    if (to < 0) {
      to = (int)(std::min_element(size.begin(), size.end()) - size.begin());
      // (of very many, each to a lane of its own: enough of them are beside one another)
      if (2 * lanes * (size_t)count[same[i]] <= pieces.size()) lane_of[same[i]] = to;
    }
    lane[to].push_back(i);
    size[to] += pieces[i].tile1 - pieces[i].tile0 + 20;
  }
  std::vector<PagedPiece> out;
  out.reserve(pieces.size());
  for (size_t i = 0; out.size() < pieces.size(); ++i)
    for (int l = 0; l < lanes; ++l)
      if (i < lane[l].size()) out.push_back(pieces[lane[l][i]]);
  pieces.swap(out);
}

}  // namespace paged_detail

// The list of a checked batch.
inline PagedPlanInfo paged_plan(const PagedBatchArgs& a, std::vector<int32_t>& out) {
  using namespace paged_detail;
  PagedPlanInfo p;
  const int G = a.hq / a.hkv, tpp = a.page_size / 32;
  std::vector<int32_t> row0(a.seqs);
  std::vector<int64_t> table0(a.seqs);
  std::vector<Unit> units[2], units64;
  std::vector<PagedTile> tiles;
  std::vector<int32_t> written;  // the tiles' numbers, to find two rows in one place
  int64_t n_table = 0;
  const auto unit_tiles = [&](int s, int64_t last_vec) {
    const int64_t end = paged_key_end(a.pos0[s] + last_vec / G, a.keys[s], a.masked != 0,
                                      a.prompt_len ? a.prompt_len[s] : 0, a.block);
    return (end + 31) / 32;
  };
  const auto units_of = [&](int s, int step, std::vector<Unit>& to) {
    const int64_t vecs = (int64_t)a.rows[s] * G;
    for (int64_t v = 0; v < vecs; v += step) {
      const int n = (int)std::min<int64_t>(step, vecs - v);
      to.push_back(Unit{s, (int)v, n, unit_tiles(s, v + n - 1), (double)((vecs + step - 1) / step)});
    }
  };
  // What reading the keys of all of the units' sequences once takes, at 5.3 TB/s.
  const auto read_us = [&](const std::vector<Unit>& of) {
    std::vector<int64_t> read(a.seqs, 0);
    int64_t all = 0;
    for (const Unit& u : of) read[u.seq] = std::max(read[u.seq], u.tiles);
    for (int64_t n : read) all += n;
    return 0.0031 * (double)(all * a.hkv);
  };
  // Sequences of many query vectors: by the large kernel where that takes less time than units of 64. (Work:
  // that of a CU, in tiles of 256 query vectors, about a us each. Of 40 of them no batch was faster there, of
  // 400 none was slower.)
  double work = 0.;
  bool others = false;
  for (int s = 0; s < a.seqs; ++s) {
    if ((int64_t)a.rows[s] * G >= PAGED_VECS_L) units_of(s, PAGED_VECS_L, units[1]);
    else others = others || a.rows[s];
  }
  for (const Unit& u : units[1]) work += (double)(u.tiles * a.hkv) / PAGED_CUS;
  const LargeTimes large_us = large_times(units[1], a.hkv);
  bool many = work > 400.;
  if (!many && work > 40.) {
    std::vector<Unit> small;
    for (int s = 0; s < a.seqs; ++s)
      if ((int64_t)a.rows[s] * G >= PAGED_VECS_L) units_of(s, PAGED_VECS_M, small);
    const double us = std::min(large_us.whole, large_us.cut) + (others ? 8. : 0.);
    double least = 0.;  // what any cut of them takes
    for (const Unit& u : small) least += (MEDIUM.fixed + MEDIUM.tile * (double)u.tiles) * a.hkv / PAGED_CUS;
    many = us < least || us < part_length(small, a.hkv, read_us(small)).first;
  }
  if (!many) units[1].clear();
  for (int s = 0; s < a.seqs; ++s) {
    row0[s] = p.rows;
    p.rows += a.rows[s];
    table0[s] = n_table;
    n_table += (a.keys[s] + (int64_t)a.page_size - 1) / a.page_size;
    const int64_t vecs = (int64_t)a.rows[s] * G;
    const bool large = many && vecs >= PAGED_VECS_L;
    if (!large) {
      units_of(s, PAGED_VECS, units[0]);
      units_of(s, PAGED_VECS_M, units64);
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

  std::vector<PagedPiece> pieces[2];
  std::vector<int32_t> first;
  std::vector<PagedJoin> joins;
  int slot = 0;
  for (int k = 0; k < 2; ++k) {
    if (units[k].empty()) continue;
    std::vector<Share> shares;
    std::vector<int> same;  // a number for each sequence and part of its keys: which a share has
    if (k == 0) {
      const auto longest = [](const Unit& x, const Unit& y) { return x.tiles > y.tiles; };
      std::stable_sort(units[0].begin(), units[0].end(), longest);
      const double all_us = read_us(units[0]);
      auto best = part_length(units[0], a.hkv, all_us);
      if (units64.size() < units[0].size()) {
        const auto other = part_length(units64, a.hkv, all_us);
        if (other.first < best.first) {
          best = other;
          units[0].swap(units64);
          std::stable_sort(units[0].begin(), units[0].end(), longest);
        }
      }
      const int64_t len = best.second;
      int group = 0, numbers = 0;
      std::vector<std::pair<int, int>> number(a.seqs);  // (of a sequence the first, how many)
      for (const Unit& u : units[0]) {
        int& n = number[u.seq].second;
        n = std::max(n, (int)((u.tiles + len - 1) / len));
      }
      for (auto& y : number) {
        y.first = numbers;
        numbers += std::max(1, y.second);
      }
      for (int i = 0; i < (int)units[0].size(); ++i) {
        const int64_t tiles = units[0][i].tiles, n = std::max<int64_t>(1, (tiles + len - 1) / len);
        for (int64_t j = 0; j < n; ++j) {
          shares.push_back(Share{i, group++, tiles * j / n, tiles * (j + 1) / n});
          same.push_back(number[units[0][i].seq].first + (int)j);
        }
      }
    } else {
      if (large_us.whole <= large_us.cut) {
        std::stable_sort(units[1].begin(), units[1].end(),
                         [](const Unit& x, const Unit& y) { return x.tiles > y.tiles; });
        for (int i = 0; i < (int)units[1].size(); ++i) shares.push_back(Share{i, i, 0, units[1][i].tiles});
      } else {
        shares = cut(units[1], std::max(1, PAGED_CUS / a.hkv), LARGE_SHARES);
      }
    }
    for (size_t i = 0; i < shares.size();) {
      size_t j = i;
      while (j < shares.size() && shares[j].unit == shares[i].unit) ++j;
      const Unit& u = units[k][shares[i].unit];
      const int s = u.seq, subs = (u.vecs + 31) / 32, parts = (int)(j - i), slot0 = slot;
      for (; i < j; ++i) {
        if (i == 0 || shares[i].group != shares[i - 1].group) {
          if (i) pieces[k].back().last = 1;
          if (k == 1) first.push_back((int32_t)pieces[k].size());
        }
        PagedPiece y{};
        y.row0 = row0[s];
        y.rows = a.rows[s];
        y.pos0 = a.pos0[s];
        y.keys = a.keys[s];
        y.prompt_len = a.prompt_len ? a.prompt_len[s] : 0;
        y.vec0 = u.vec0;
        y.tile0 = (int)shares[i].tile0;
        y.tile1 = (int)shares[i].tile1;
        y.slot = parts > 1 ? slot : -1;
        y.table = (int)table0[s];
        y.wide = u.vecs > PAGED_VECS;
        pieces[k].push_back(y);
        if (parts > 1) slot += subs;
      }
      for (int q = 0; parts > 1 && q < subs; ++q) {
        PagedJoin y{};
        y.row0 = row0[s];
        y.vec0 = u.vec0 + 32 * q;
        y.vecs = std::min(32, u.vecs - 32 * q);
        y.slot = slot0 + q;
        y.step = subs;
        y.parts = parts;
        joins.push_back(y);
      }
    }
    pieces[k].back().last = 1;
    if (k == 0) side_by_side(pieces[0], same, a.hkv);
  }
  p.n_small = (int)pieces[0].size();
  p.n_large = (int)first.size();
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
  p.first_large = put(first.data(), first.size());
  out.resize((out.size() + 15) / 16 * 16);
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
