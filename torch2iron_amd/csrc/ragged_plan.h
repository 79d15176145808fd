// The plan of a packed (ragged) prompt batch: which row tiles and key ranges its attention's
// workgroups take, and where every packed row goes.  Host code alone (standard C++, no HIP),
// so that it can be checked without a device.
#pragma once

#include <stdint.h>

#include <algorithm>
#include <queue>
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

// Time of a key block of a tile, in twelfths of a full tile's: with fewer than 128 pairs some of
// the four waves have nothing to multiply, but the block's loads take nearly as long.
inline int64_t block_cost(int64_t pairs) { return pairs > 32 ? 12 : 11; }
constexpr int64_t TILE_COST = 3 * 12;     // first loads and outputs of an item
constexpr int64_t MERGE_COST = 8 * 12;    // a second launch that joins parts

// Two ways to hand the tiles out, whichever a count of their costs says ends sooner:
//   whole: a workgroup a tile, longest first (the chip takes the next as slots come free);
//   even:  RG_SLOTS workgroups with equal shares of the tiles' key blocks, cut where a share
//          ends; the parts of a cut tile are joined by a second launch.
inline PackedTable packed_table(const int32_t* lengths, const int32_t* starts, const int32_t* cache_rows, int n, int G,
                                int Hkv) {
  PackedTable t;
  struct Tile { int32_t seq, row0; int64_t j0; int32_t blocks; int64_t cost; };
  std::vector<Tile> tiles;
  int64_t row0 = 0, work = 0;
  for (int i = 0; i < n; ++i) {
    const int64_t pairs = (int64_t)lengths[i] * G;
    for (int64_t j0 = 0; j0 < pairs; j0 += RG_ROWS) {
      const int b = tile_blocks(j0, pairs, G, starts[i]);
      tiles.push_back({i, (int32_t)row0, j0, b, block_cost(std::min<int64_t>(pairs - j0, RG_ROWS))});
      work += b * tiles.back().cost;
    }
    for (int32_t r = 0; r < lengths[i]; ++r) {
      t.row_pos.push_back(starts[i] + r);
      t.row_cache.push_back(cache_rows ? cache_rows[i] : i);
    }
    row0 += lengths[i];
  }
  const auto item = [&](const Tile& a, int k0, int k1, int part) {
    const int32_t w[RG_ITEM] = {a.row0, lengths[a.seq], starts[a.seq], cache_rows ? cache_rows[a.seq] : a.seq,
                                (int32_t)a.j0, k0, k1, part};
    t.items.insert(t.items.end(), w, w + RG_ITEM);
  };
  std::stable_sort(tiles.begin(), tiles.end(),
                   [](const Tile& a, const Tile& b) { return a.blocks * a.cost > b.blocks * b.cost; });
  const int64_t slots = std::max(1, RG_SLOTS / Hkv);   // a kv head's
  int64_t whole = 0;                                   // when the last slot is done
  {
    std::priority_queue<int64_t, std::vector<int64_t>, std::greater<int64_t>> free_at;
    for (const Tile& a : tiles) {
      int64_t at = 0;
      if ((int64_t)free_at.size() >= slots) {
        at = free_at.top();
        free_at.pop();
      }
      free_at.push(at + a.blocks * a.cost + TILE_COST);
      whole = std::max(whole, at + a.blocks * a.cost + TILE_COST);
    }
  }
  // a share is at least two full key blocks
  const int64_t n_even = std::max<int64_t>(1, std::min<int64_t>(slots, work / (2 * 12)));
  const int64_t share = (work + n_even - 1) / n_even;
  const int64_t even = share + 2 * TILE_COST + MERGE_COST;
  t.bins.push_back(0);
  if (whole <= even) {
    for (const Tile& a : tiles) {
      item(a, 0, a.blocks, -1);
      t.bins.push_back((int32_t)(t.items.size() / RG_ITEM));
    }
    return t;
  }
  int64_t room = share;                                // of the open bin
  for (const Tile& a : tiles) {
    std::vector<int> cuts{0};
    std::vector<size_t> at;                            // items of the tile
    while (cuts.back() < a.blocks) {
      const int left = a.blocks - cuts.back();
      int take = (int)std::min<int64_t>(left, std::max<int64_t>(1, (room + a.cost / 2) / a.cost));
      if (left - take == 1) take = left;               // no part of a single block
      at.push_back(t.items.size());
      item(a, cuts.back(), cuts.back() + take, -1);
      cuts.push_back(cuts.back() + take);
      room -= take * a.cost;
      if (room < a.cost) {                             // the share is used up
        t.bins.push_back((int32_t)(t.items.size() / RG_ITEM));
        room += share;
        if (room < a.cost) room = a.cost;
      }
    }
    if (at.size() > 1) {
      for (size_t s = 0; s < at.size(); ++s) t.items[at[s] + 7] = t.n_parts + (int32_t)s;
      const int64_t live = std::min<int64_t>((int64_t)lengths[a.seq] * G - a.j0, RG_ROWS);
      for (int32_t e = 0; e < live; e += RG_MERGE) {
        const int32_t m[RG_ITEM] = {a.row0, lengths[a.seq], (int32_t)a.j0, t.n_parts, (int32_t)at.size(), e, 0, 0};
        t.merges.insert(t.merges.end(), m, m + RG_ITEM);
      }
      t.n_parts += (int32_t)at.size();
    }
  }
  if (t.bins.back() != (int32_t)(t.items.size() / RG_ITEM)) t.bins.push_back((int32_t)(t.items.size() / RG_ITEM));
  return t;
}

// A tree's attention: its contexts are on the device, where every workgroup finds its own even
// share of the batch's key blocks (of at least two blocks).  Shares of a kv head's tile, at most:
inline int tree_bins(int64_t B, int tiles_heads, int cap, int tile_rows) {
  const int64_t most = B * ((cap + RG_KEYS - 1) / RG_KEYS) / 2;
  return (int)std::max<int64_t>(1, std::min<int64_t>(std::max(1, (tile_rows == 128 ? 512 : 256) / tiles_heads), most));
}

}  // namespace t2i_host
