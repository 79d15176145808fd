// The plan of a packed (ragged) prompt batch: which row tiles and key ranges its attention's
// workgroups take, and where every packed row goes.  Host code alone (standard C++, no HIP),
// so that it can be checked without a device.
#pragma once

#include <stdint.h>

#include <algorithm>
#include <vector>

namespace t2i_host {

constexpr int RG_ROWS = 128;    // (row, q head) pairs of a tile
constexpr int RG_KEYS = 64;     // keys of a block
constexpr int RG_ITEM = 8;      // words of a work item or merge entry
constexpr int RG_MERGE = 8;     // pairs of a merge entry
constexpr int RG_SLOTS = 512;   // workgroups that the chip holds: two a CU

// A work item: {first packed row of the sequence, its rows, slots before them, cache row,
// first pair of the tile, first key block, key block behind the last, part (-1: none)}.
// A bin is a workgroup (of every kv head): items bins[i] .. bins[i + 1] - 1, one after the other.
// A merge entry, for up to RG_MERGE pairs of a cut tile: {first packed row of the sequence, its
// rows, first pair of the tile, first part, parts, first of its pairs within the tile, 0, 0}.
struct PackedTable {
  std::vector<int32_t> row_pos, row_cache, items, bins, merges;
  int32_t n_parts = 0;
};

// Pair j of a sequence is its row j / G under q head j % G of a kv head (G q heads a kv head).
// Last key block + 1 that a tile of pairs [j0, j0 + RG_ROWS) can attend.
inline int tile_blocks(int64_t j0, int64_t pairs, int G, int start) {
  const int64_t last = std::min<int64_t>(j0 + RG_ROWS, pairs) - 1;
  return (int)((start + last / G + RG_KEYS) / RG_KEYS);
}

// Times in us that the choice below goes by, fitted to graph-launched calls (1 to 64 sequences, 1 to
// 4000 rows, 0 to 6000 slots before them, 8 kv heads of 2 and 4 q heads): a key block of a
// workgroup that has its CU alone, and its share of a CU that two workgroups fill; tiles of up
// to 32 pairs (one wave of four multiplies) wait for their loads longer, and the single row of a
// sequence takes half as many products again.
struct BlockTime { double alone, shared; };
inline BlockTime block_time(int64_t pairs, bool single_row) {
  return pairs > 32 ? BlockTime{1.35, 1.1} : single_row ? BlockTime{1.95, 1.45} : BlockTime{1.75, 1.35};
}
constexpr double RG_CUS = 256, ITEM_TIME = 2.5;       // ITEM_TIME: first loads and outputs
constexpr double CALL_TIME = 4, MERGE_TIME = 5;       // MERGE_TIME: a second launch
constexpr double PART_BYTES_PER_US = 1e7;             // parts written and read again

inline PackedTable packed_items(const int32_t* lengths, const int32_t* starts, const int32_t* cache_rows, int n, int G,
                                int Hkv);

// Two ways to hand the tiles out, whichever the times above say ends sooner:
//   whole: a workgroup a tile, longest first (the chip takes the next as slots come free);
//   even:  RG_SLOTS workgroups with equal shares of the tiles' key blocks, cut where a share
//          ends; the parts of a cut tile are joined by a second launch.
// Measured (us, whole / even; taken): 1999 rows from 6001, 32 / 8 heads 237 / 258 (whole); 1000 rows
// from 6001 151 / 132 (even); 32 x 500 rows 129 / 213 (whole); 2000 rows from 0, 16 / 8 47 / 42
// (even); 16 single rows from 4000, 4 q heads, 131 / 50, 4 of 2 126 / 19 (even); 4 x 300 rows 11.0 / 16.7 (whole).
inline PackedTable packed_table(const int32_t* lengths, const int32_t* starts, const int32_t* cache_rows, int n, int G,
                                int Hkv) {
  PackedTable t = packed_items(lengths, starts, cache_rows, n, G, Hkv);
  for (int i = 0; i < n; ++i)
    for (int32_t r = 0; r < lengths[i]; ++r) {
      t.row_pos.push_back(starts[i] + r);
      t.row_cache.push_back(cache_rows ? cache_rows[i] : i);
    }
  return t;
}

inline PackedTable packed_items(const int32_t* lengths, const int32_t* starts, const int32_t* cache_rows, int n, int G,
                                int Hkv) {
  struct Tile { int32_t seq, row0; int64_t j0, live; int32_t blocks; BlockTime time; };
  std::vector<Tile> tiles;
  int64_t row0 = 0;
  double work = 0, longest = 0;                        // a kv head's, and one tile's
  for (int i = 0; i < n; ++i) {
    const int64_t pairs = (int64_t)lengths[i] * G;
    for (int64_t j0 = 0; j0 < pairs; j0 += RG_ROWS) {
      const int64_t live = std::min<int64_t>(pairs - j0, RG_ROWS);
      tiles.push_back({i, (int32_t)row0, j0, live, tile_blocks(j0, pairs, G, starts[i]), block_time(live, lengths[i] == 1)});
      work += tiles.back().blocks * tiles.back().time.shared;
      longest = std::max(longest, tiles.back().blocks * tiles.back().time.alone);
    }
    row0 += lengths[i];
  }
  std::stable_sort(tiles.begin(), tiles.end(),
                   [](const Tile& a, const Tile& b) { return a.blocks * a.time.alone > b.blocks * b.time.alone; });
  const auto item = [&](PackedTable& t, const Tile& a, int k0, int k1, int part) {
    const int32_t w[RG_ITEM] = {a.row0, lengths[a.seq], starts[a.seq], cache_rows ? cache_rows[a.seq] : a.seq,
                                (int32_t)a.j0, k0, k1, part};
    t.items.insert(t.items.end(), w, w + RG_ITEM);
  };
  const auto close_bin = [](PackedTable& t) { t.bins.push_back((int32_t)(t.items.size() / RG_ITEM)); };
  PackedTable whole;
  whole.bins.push_back(0);
  for (const Tile& a : tiles) {
    item(whole, a, 0, a.blocks, -1);
    close_bin(whole);
  }
  const double heads = Hkv / RG_CUS;
  const double whole_time = CALL_TIME + std::max(longest + 1, work * heads + tiles.size() * heads * ITEM_TIME);
  // (no cut can end before the tiles' own work)
  if (whole_time <= CALL_TIME + MERGE_TIME + work * heads + tiles.size() * heads * ITEM_TIME) return whole;

  const int64_t slots = std::max(1, RG_SLOTS / Hkv);   // a kv head's
  // a share is at least two key blocks
  const int64_t n_even = std::max<int64_t>(1, std::min<int64_t>(slots, (int64_t)(work / (2 * 1.1))));
  const double share = work / n_even;
  PackedTable even;
  even.bins.push_back(0);
  double room = share, merged = 0;                     // of the open bin; pairs of all parts
  for (const Tile& a : tiles) {
    std::vector<size_t> at;                            // items of the tile
    for (int k0 = 0; k0 < a.blocks;) {
      const int left = a.blocks - k0;
      int take = (int)std::min<double>(left, std::max(1.0, room / a.time.shared + 0.5));
      if (left - take == 1) take = left;               // no part of a single block
      at.push_back(even.items.size());
      item(even, a, k0, k0 + take, -1);
      k0 += take;
      room -= take * a.time.shared;
      if (room < a.time.shared) {                      // the share is used up
        close_bin(even);
        room = std::max(room + share, a.time.shared);
      }
    }
    if (at.size() > 1) {
      for (size_t s = 0; s < at.size(); ++s) even.items[at[s] + 7] = even.n_parts + (int32_t)s;
      for (int32_t e = 0; e < a.live; e += RG_MERGE) {
        const int32_t m[RG_ITEM] = {a.row0, lengths[a.seq], (int32_t)a.j0, even.n_parts, (int32_t)at.size(), e, 0, 0};
        even.merges.insert(even.merges.end(), m, m + RG_ITEM);
      }
      even.n_parts += (int32_t)at.size();
      merged += (double)a.live * at.size();
    }
  }
  if (even.bins.back() != (int32_t)(even.items.size() / RG_ITEM)) close_bin(even);
  const double even_time = CALL_TIME + MERGE_TIME + std::max(share * 1.3, work * heads) +
                           even.items.size() / RG_ITEM * heads * ITEM_TIME + merged * Hkv * 1024 / PART_BYTES_PER_US;
  return whole_time <= even_time ? whole : even;
}

// A tree's attention: its contexts are on the device, where every workgroup finds its own even
// share of the batch's key blocks (of at least two blocks).  Shares of a kv head's tile, at most:
inline int tree_bins(int64_t B, int tiles_heads, int cap) {
  const int64_t most = B * ((cap + RG_KEYS - 1) / RG_KEYS) / 2;
  return (int)std::max<int64_t>(1, std::min<int64_t>(std::max(1, RG_SLOTS / tiles_heads), most));
}

}  // namespace t2i_host
