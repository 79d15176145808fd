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

// A work item: {first packed row of the sequence, its rows, slots before them, cache row,
// first pair of the tile, first key block, key block behind the last, part (-1: none)}.
// A merge entry: {first packed row, rows, first pair, first part, parts, 0, 0, 0}.
struct PackedTable {
  std::vector<int32_t> row_pos, row_cache, items, merges;
  int32_t n_parts = 0;
};

// Pair j of a sequence is its row j / G under q head j % G of a kv head (G q heads a kv head).
// Last key block + 1 that a tile of pairs [j0, j0 + RG_ROWS) can attend.
inline int tile_blocks(int64_t j0, int64_t pairs, int G, int start) {
  const int64_t last = std::min<int64_t>(j0 + RG_ROWS, pairs) - 1;
  return (int)((start + last / G + RG_KEYS) / RG_KEYS);
}

// Tiles of RG_ROWS pairs, each over all its keys or, where the batch has too few tiles to fill
// the chip (512 workgroups: two a CU) and this one has many key blocks, over parts of them that
// a second launch merges.  A part has at least 16 key blocks.  Longest items first, so that the
// short ones fill the tail.
inline PackedTable packed_table(const int32_t* lengths, const int32_t* starts, const int32_t* cache_rows, int n, int G,
                                int Hkv) {
  PackedTable t;
  struct Tile { int32_t seq, row0; int64_t j0; int32_t blocks; };
  std::vector<Tile> tiles;
  int64_t row0 = 0, work = 0;
  for (int i = 0; i < n; ++i) {
    const int64_t pairs = (int64_t)lengths[i] * G;
    for (int64_t j0 = 0; j0 < pairs; j0 += RG_ROWS) {
      tiles.push_back({i, (int32_t)row0, j0, tile_blocks(j0, pairs, G, starts[i])});
      work += tiles.back().blocks;
    }
    for (int32_t r = 0; r < lengths[i]; ++r) {
      t.row_pos.push_back(starts[i] + r);
      t.row_cache.push_back(cache_rows ? cache_rows[i] : i);
    }
    row0 += lengths[i];
  }
  const int64_t share = std::max<int64_t>(16, (work * Hkv + 511) / 512);   // key blocks of a workgroup
  struct Item { int32_t w[RG_ITEM]; };
  std::vector<Item> items;
  for (const Tile& a : tiles) {
    int parts = 1;
    if (2 * a.blocks >= 3 * share) parts = (int)((a.blocks + share / 2) / share);
    const int32_t crow = cache_rows ? cache_rows[a.seq] : a.seq;
    for (int s = 0; s < parts; ++s)
      items.push_back({{a.row0, lengths[a.seq], starts[a.seq], crow, (int32_t)a.j0,
                        (int32_t)((int64_t)a.blocks * s / parts), (int32_t)((int64_t)a.blocks * (s + 1) / parts),
                        parts > 1 ? t.n_parts + s : -1}});
    if (parts > 1) {
      const int32_t m[RG_ITEM] = {a.row0, lengths[a.seq], (int32_t)a.j0, t.n_parts, parts, 0, 0, 0};
      t.merges.insert(t.merges.end(), m, m + RG_ITEM);
      t.n_parts += parts;
    }
  }
  std::stable_sort(items.begin(), items.end(),
                   [](const Item& a, const Item& b) { return a.w[6] - a.w[5] > b.w[6] - b.w[5]; });
  for (const Item& a : items) t.items.insert(t.items.end(), a.w, a.w + RG_ITEM);
  return t;
}

// Parts of each tile of a tree's attention: from the sizes alone (the contexts are on the
// device), enough for 512 workgroups, each with at least four key blocks of a full cache.
inline int tree_splits(int64_t tiles, int cap) {
  const int64_t want = (512 + tiles - 1) / tiles;
  return (int)std::max<int64_t>(1, std::min<int64_t>(want, std::min(64, cap / (4 * RG_KEYS))));
}

}  // namespace t2i_host
