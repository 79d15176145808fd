// Attention of ragged batches over a KV cache in pages for gfx950:
//
//   * t2i_paged_plan: a step's plan, made on the device from each sequence's rows and context: where every
//     row goes, and which tiles and keys the attention's workgroups take;
//   * t2i_paged_qk_rope_kv: per-head q/k RMSNorm + RoPE and the write of k and v into their pages;
//   * t2i_paged_attention: causal GQA attention of prompt chunks, drafted tokens and single tokens.
//
// Slot j of sequence s is place j % P of page pages[s][j / P]; pools are [n_pages, Hkv, P, D], so that the slots
// of a page and kv head are contiguous.  Scores, softmax statistics and sums are fp32; weights enter P . V
// as t2i_packed_attention's do.
#include <math.h>

#include <algorithm>

#include "t2i_common.h"
#include "qk_prep.h"
#include "ragged_attend.h"

namespace t2i {

// ============================================================================
// the plan of a step
// ============================================================================
constexpr int PG_THREADS = 1024;
constexpr int PG_SEQS = 4096;                // sequences of a plan
constexpr int PG_TILE = 8;                   // words of a tile: {first row, rows, context, sequence, first pair, first unit, units, 0}
constexpr int PG_BIN = 4;                    // of a bin: {first tile (-1: none), first unit, unit behind the last, narrow ones among wide?}
constexpr int PG_MERGE = 8;                  // of a merge: {first row, rows (0: none), first pair, first part, first second part, parts, 0, 0}
constexpr int PG_NARROW = 32;                // pairs that one wave multiplies
constexpr int PG_ROW = 2;                    // of a row: {position (-1: none), sequence}

// A unit is a key block of a tile; all tiles' units stand in a row.
struct PagedPlanParams {
  const int32_t* row_starts;                 // [B + 1]
  const int32_t* ctx;                        // [B]
  int32_t* tiles;                            // [tiles_cap][PG_TILE]
  int32_t* bins;                             // [bins_cap][PG_BIN]
  int32_t* merges;                           // [merges_cap][PG_MERGE]: a cut tile's, at its number or at its last share's
  int32_t* row;                              // [rows][PG_ROW]
  int rows, B, G, Hkv, cap, tiles_cap, bins_cap, shares, merges_cap;
};

// Sums of the values of the threads before this one, and of all (LDS: one word a wave).
__device__ __forceinline__ int plan_scan(int v, int* s_wave, int& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const int u = __shfl_up(x, s, 64);
    if (lane >= s) x += u;
  }
  __syncthreads();                           // the words of the scan before are read
  if (lane == 63) s_wave[wave] = x;
  __syncthreads();
  int before = 0;
  all = 0;
  for (int w = 0; w < PG_THREADS / 64; ++w) {
    before += w < wave ? s_wave[w] : 0;
    all += s_wave[w];
  }
  return before + x - v;
}

// The sequence of the row ranges first[0 .. n] that holds `at`, the last of several that start there.
template <typename P>
__device__ __forceinline__ int plan_find(const P& first, int n, int at) {
  int lo = 0, hi = n;                        // first[lo] <= at < first[hi], as far as the array ascends
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (first[mid] <= at) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Rows of a sequence: 0 where its range does not lie in the batch.
__device__ __forceinline__ int plan_rows(const PagedPlanParams& p, int s) {
  const int a = p.row_starts[s], b = p.row_starts[s + 1];
  return a >= 0 && a <= b && b <= p.rows ? b - a : 0;
}

// Times in us that the choice below goes by: those of the packed plan (ragged_plan.h), in which a key block of a
// workgroup costs `alone` with a CU to itself and `shared` where two workgroups fill one.
__device__ __forceinline__ void plan_times(int pairs, float& alone, float& shared) {
  alone = pairs > PG_NARROW ? 1.35f : 1.95f;
  shared = pairs > PG_NARROW ? 1.1f : 1.45f;
}

// Workgroup 0: the tiles and how they are handed out; the others: a thread a row.  As in the packed plan a tile goes
// to a workgroup whole, longest first, or the units are cut into equal shares whose tiles' parts a second launch
// joins, whichever the times say ends sooner; here the device decides, so that a captured step may
// serve every later one.
// A chain of scans and look-ups in one workgroup, bound by their latency: one token 6 us, 32 single tokens 10.5, 16 x 5
// drafts 8.3, 4997 rows of 16 prompts 15 (from a graph; 12.0 for the 32 tokens behind an idle GPU), once a step of all
// layers.  A thread finds its own share (one after the other took 13.2 us for the 32 tokens), and shares are cut without
// 64-bit division.
__global__ __launch_bounds__(PG_THREADS) void paged_plan_kernel(const PagedPlanParams p) {
  const int tid = threadIdx.x;
  int falls = 0;                             // row_starts that do not ascend: no row is anyone's
  for (int s = tid; s < p.B; s += PG_THREADS) falls |= p.row_starts[s] < 0 || p.row_starts[s] > p.row_starts[s + 1] || p.row_starts[s + 1] > p.rows;
  const bool ascends = !__syncthreads_or(falls);
  if (blockIdx.x > 0) {
    const int row = (blockIdx.x - 1) * PG_THREADS + tid;
    if (row >= p.rows) return;
    const int s = plan_find(p.row_starts, p.B, row);
    const int n = plan_rows(p, s), r = row - p.row_starts[s], ctx = p.ctx[s];
    const bool ok = ascends && r >= 0 && r < n && ctx >= 0 && ctx <= p.cap - n;
    p.row[PG_ROW * row] = ok ? ctx + r : -1;
    p.row[PG_ROW * row + 1] = s;
    return;
  }
  __shared__ int s_first[PG_SEQS + 1];       // first tile of each sequence
  __shared__ int s_wave[PG_THREADS / 64], s_count[PG_THREADS];
  __shared__ int s_work, s_longest;          // times of all tiles (0.05 us), and of the longest (a float's bits)
  __shared__ int s_pairs, s_units, s_wide;   // pairs of all tiles; units of the longest; is any tile wider than PG_NARROW

  // ---- tiles of each sequence ----
  int n_tiles = 0;
  for (int base = 0; base < p.B; base += PG_THREADS) {
    const int s = base + tid;
    const int n = s < p.B && ascends ? (plan_rows(p, s) * p.G + RG_ROWS - 1) / RG_ROWS : 0;
    int all;
    const int at = plan_scan(n, s_wave, all);
    if (s < p.B) s_first[s] = n_tiles + at;
    n_tiles += all;
  }
  if (tid == 0) {
    s_first[p.B] = n_tiles;
    s_work = s_longest = s_pairs = s_units = s_wide = 0;
  }
  for (int i = tid; i < p.bins_cap; i += PG_THREADS) p.bins[PG_BIN * i] = -1;
  for (int i = tid; i < p.merges_cap; i += PG_THREADS) p.merges[PG_MERGE * i + 1] = 0;
  __syncthreads();

  // ---- the tiles, and their units in a row ----
  int total = 0;
  for (int base = 0; base < n_tiles; base += PG_THREADS) {
    const int t = base + tid;
    int units = 0, pairs = 0, row0 = 0, rows = 0, ctx = -1, s = 0, j0 = 0;
    if (t < n_tiles) {
      s = plan_find(s_first, p.B, t);
      row0 = p.row_starts[s];
      rows = plan_rows(p, s);
      j0 = (t - s_first[s]) * RG_ROWS;
      ctx = p.ctx[s];
      if (ctx < 0 || ctx > p.cap - rows) ctx = -1;         // zero rows: a unit without keys
      pairs = min(rows * p.G - j0, RG_ROWS);
      units = ctx < 0 ? 1 : (ctx + (j0 + pairs - 1) / p.G + RG_KEYS) / RG_KEYS;
    }
    int all;
    const int first = total + plan_scan(units, s_wave, all);
    if (t < n_tiles) {
      int32_t* w = p.tiles + (size_t)t * PG_TILE;
      w[0] = row0; w[1] = rows; w[2] = ctx; w[3] = s; w[4] = j0; w[5] = first; w[6] = units; w[7] = 0;
      if (t < PG_THREADS) s_count[t] = first;
      float alone, shared;
      plan_times(pairs, alone, shared);
      atomicAdd(&s_pairs, pairs);
      atomicMax(&s_units, units);
      if (pairs > PG_NARROW) s_wide = 1;
      atomicMax(&s_longest, __float_as_int(units * alone));   // positive floats order as integers
      atomicAdd(&s_work, (int)(units * shared * 20.0f + 0.5f));   // whole numbers: in any order the same sum
    }
    total += all;
  }
  __syncthreads();
  if (n_tiles == 0) return;

  // ---- whole tiles or even shares ----
  const float heads = p.Hkv / 256.0f, work = s_work * 0.05f, longest_time = __int_as_float(s_longest);
  const int n = max(1, min(p.shares, total / 2));          // shares, of at least two units
  const float whole_time = 4.0f + fmaxf(longest_time + 1.0f, work * heads + n_tiles * heads * 2.5f);
  const float merged = (float)s_pairs / n_tiles * (n + min(n, n_tiles));
  const float even_time = 9.0f + fmaxf(work / n * 1.3f, work * heads) + (n_tiles + n) * heads * 2.5f + merged * p.Hkv * 1024e-7f;
  if (whole_time <= even_time) {
    // longest first: a tile's place is the number of tiles of more units, by buckets of like ones
    const int longest = s_units;
    const auto bucket = [&](int units) { return (int)((float)(longest - units) / (float)longest * (PG_THREADS - 1)); };
    s_count[tid] = 0;
    __syncthreads();
    for (int base = 0; base < n_tiles; base += PG_THREADS) {
      const int t = base + tid;
      if (t < n_tiles) atomicAdd(&s_count[bucket(p.tiles[(size_t)t * PG_TILE + 6])], 1);
    }
    __syncthreads();
    const int mine = s_count[tid];
    int all;
    const int before = plan_scan(mine, s_wave, all);
    __syncthreads();
    s_count[tid] = before;
    __syncthreads();
    for (int base = 0; base < n_tiles; base += PG_THREADS) {
      const int t = base + tid;
      if (t >= n_tiles) continue;
      const int first = p.tiles[(size_t)t * PG_TILE + 5], units = p.tiles[(size_t)t * PG_TILE + 6];
      // (the order within a bucket is of no account: every tile is a workgroup's own)
      const int at = atomicAdd(&s_count[bucket(units)], 1);
      int32_t* w = p.bins + (size_t)at * PG_BIN;
      w[0] = t; w[1] = first; w[2] = first + units; w[3] = s_wide;
    }
    return;
  }
  // a thread a share: total i / n without 64-bit division (the remainder and n stay below 2^9)
  const int each = total / n, left = total - each * n;
  const auto run_start = [&](int i) { return each * i + left * i / n; };
  if (tid >= n) return;                                    // (shares are at most RG_SLOTS)
  const int from = run_start(tid), to = run_start(tid + 1);
  const auto first_unit = [&](int t) { return n_tiles <= PG_THREADS ? s_count[t] : p.tiles[(size_t)t * PG_TILE + 5]; };
  int t = 0;
  for (int hi = n_tiles; hi - t > 1;) {                    // the tile that holds the share's first unit
    const int mid = (t + hi) / 2;
    if (first_unit(mid) <= from) t = mid;
    else hi = mid;
  }
  int32_t* const bin = p.bins + (size_t)tid * PG_BIN;
  bin[0] = t; bin[1] = from; bin[2] = to; bin[3] = 0;
  const int32_t* const rec = p.tiles + (size_t)t * PG_TILE;
  const int first = rec[5], end = first + rec[6];
  if (from > first && to >= end) {                         // the share ends a tile that others began: its merge
    int run = min((int)((float)first * n / total), tid);   // the share that holds the tile's first unit, about; then exactly
    while (run_start(run + 1) <= first) ++run;
    while (run_start(run) > first) --run;
    int32_t* const w = p.merges + (size_t)(p.merges_cap < p.shares ? t : tid) * PG_MERGE;
    w[0] = rec[0]; w[2] = rec[4]; w[3] = 2 * run + (run_start(run) != first); w[4] = 2 * (run + 1); w[5] = tid - run + 1;
    w[1] = rec[1];
  }
}

// ============================================================================
// q/k RMSNorm + RoPE + the write into the pages
// ============================================================================
struct PagedPrepParams {
  const uint16_t* qkv;      // [rows, (Hq + 2 Hkv) * D]
  const uint16_t* qn;
  const uint16_t* kn;
  const uint16_t* rope;     // [>= cap, D] cos even / sin odd
  uint16_t* q;              // [rows, Hq, D]
  uint16_t* kc;             // [n_pages, Hkv, P, D]
  uint16_t* vc;
  const int32_t* row;       // the plan's rows
  const int32_t* pages;     // [B, max_pages]
  int B, Hq, Hkv, cap, max_pages, n_pages, page_shift, style;
  float eps;
};

constexpr int PG_PREP_NB = 2;

// One workgroup (4 waves) a row, as the contiguous caches' ragged_prep_kernel, whose bits it gives: only where a
// row goes is another matter.  The page's id is needed at the stores alone.  4997 rows of 16 / 8 heads 21 us (82 MB, 3.9 TB/s,
// as over a contiguous cache); up to 80 rows 4 us, a launch and three dependent loads.
__global__ __launch_bounds__(256) void paged_prep_kernel(const PagedPrepParams p) {
  constexpr int D = RG_D;
  const int row = blockIdx.x;
  const int lane = threadIdx.x & 63;
  const int pos = p.row[PG_ROW * row], s = p.row[PG_ROW * row + 1];
  if (pos < 0 || pos >= p.cap || s < 0 || s >= p.B) return;
  const int page = p.pages[(size_t)s * p.max_pages + (pos >> p.page_shift)];
  const int c = lane & 15;
  const int slot = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 4 + (lane >> 4);   // 0 .. 15
  const int nvec = p.Hq + 2 * p.Hkv;
  const uint16_t* src_row = p.qkv + (size_t)row * nvec * D;
  for (int base = 0; base < nvec; base += 16 * PG_PREP_NB) {
    u32x4 raw[PG_PREP_NB];
#pragma unroll
    for (int j = 0; j < PG_PREP_NB; ++j)
      raw[j] = prep_load(src_row + (size_t)min(base + 16 * j + slot, nvec - 1) * D, c, p.style);
    const u32x4 rp = *reinterpret_cast<const u32x4*>(p.rope + (size_t)pos * D + 8 * c);
    const u32x4 gqv = prep_load(p.qn, c, p.style);
    const u32x4 gkv = prep_load(p.kn, c, p.style);
#pragma unroll
    for (int j = 0; j < PG_PREP_NB; ++j) asm volatile("" : "+v"(raw[j]));   // every load before the first use
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < PG_PREP_NB; ++j) {
      const int vi = base + 16 * j + slot;     // uniform over the 16-lane row
      const bool isq = vi < p.Hq;
      const bool normed = vi < p.Hq + p.Hkv;   // q and k: RMSNorm + RoPE; v as is
      const u32x4 y = prep_vector(raw[j], rp, isq ? gqv : gkv, normed, p.style, p.eps);
      if (vi >= nvec || (!isq && (uint32_t)page >= (uint32_t)p.n_pages)) continue;
      const int h = vi - p.Hq - (normed ? 0 : p.Hkv);
      const size_t at = ((((size_t)page * p.Hkv + h) << p.page_shift) + (pos & ((1 << p.page_shift) - 1))) * D;
      prep_store(isq ? p.q + ((size_t)row * p.Hq + vi) * D : normed ? p.kc + at : p.vc + at, c, p.style, y);
    }
  }
}

// ============================================================================
// attention
// ============================================================================
struct PagedTables {
  const int32_t* tiles;
  const int32_t* bins;
  const int32_t* merges;
  int tiles_cap, B;
};

// NaN in the place of an item's results (a slot of its sequence stands in no page).
__device__ __forceinline__ void poison_item(const RaggedAttnParams& p, const RaggedItem& it, int h, int lane, int wave) {
  const int c = lane & 31, h2 = lane >> 5;
  const int j = it.j0 + wave * 32 + c;
  if (j >= it.pairs) return;
  wait_stores();                             // of the results
  if (it.part >= 0) {
    const size_t st = ((size_t)it.part * p.Hkv + h) * p.part_rows + wave * 32 + c;
    if (h2 == 0) p.part_ml[st] = float2{INFINITY, __uint_as_float(0x7FC00000u)};
    return;
  }
  const int t = j / p.G, head = h * p.G + (j - t * p.G);
  const size_t qrow = (size_t)it.row0 + t;
  for (int i = 0; i < RG_D / 16; ++i)
    *reinterpret_cast<u32x4*>(p.out + (qrow * p.Hq + head) * RG_D + h2 * (RG_D / 2) + 8 * i) =
        u32x4{0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u};
  if (p.out_sums && h2 == 0) p.out_sums[(size_t)head * p.rows + qrow] = __uint_as_float(0x7FC00000u);
}

// A workgroup takes a bin's units for one kv head, tile by tile.  Sequences of one tile (single tokens, drafted
// tokens, short chunks) multiply by weights of 16 bits: their products hide behind the loads.  Single tokens among the
// tiles of long chunks, one workgroup each, are as slow as their own chain of loads: they take the form with more
// of them on their way (two chunks of 509 and 701 rows with 24 tokens 146 -> 129 us).  Where they fill the chip themselves
// that form has more barriers for nothing (32 tokens 56.9 -> 58.7 us, 64 after 4090 slots 170 -> 179).
// What bounds it (16 / 8 and 32 / 8 heads, this launch alone):
//   tokens and drafts: memory.  64 tokens after 4090 slots 6.3 TB/s, 8 after 30000 6.5, of the 6.85 that a bulk read reaches; 32 after
//     409 to 4090 52 us (295 MB, 5.7 TB/s: shares of 9 blocks, whose first loads nothing hides), MFMA 12 % and VALU 15 % of
//     a SIMD's cycles.
//   1999 rows after 30001: 0.96-1.11 ms by the card, 0.91-1.06 PFLOP/s: MFMA 54 %, VALU 51 % at 1.7-1.9 GHz, as packed rows.
//   two chunks with 24 tokens: 122 us of 116 to 137 by the card and by what ran before, 2.8 TB/s and 0.52 PFLOP/s: the longest
//     chains of loads beside the chunks' products.
// Measured and dropped: wide tiles first (two chunks with 24 tokens 130 -> 158 us), wide and narrow ones in turn, so that a CU
// might run both (125-146 for 130-147 there, 16 chunks with 10 tokens 90 -> 92, in turns of four 94); bins that carry their
// first tile's words; heavier shares where a CU has one workgroup.
__global__ __launch_bounds__(64 * RG_WAVES, 2) void paged_attention_kernel(const RaggedAttnParams p, const PagedTables tab) {
  extern __shared__ __align__(256) uint16_t s_kv[];   // [buffer][K, V][key][dim]
  __shared__ uint32_t s_odd[RG_WAVES];                     // an item's pairs whose sums are not finite
  __shared__ int s_bad[RG_WAVES];                          // whether a wave met a page outside the pool
  const int h = blockIdx.x % p.Hkv;
  const int bin = blockIdx.x / p.Hkv;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int tile = tab.bins[(size_t)bin * PG_BIN];
  if (tile < 0) return;
  const int at0 = tab.bins[(size_t)bin * PG_BIN + 1], end = tab.bins[(size_t)bin * PG_BIN + 2];
  const bool among_wide = tab.bins[(size_t)bin * PG_BIN + 3] != 0;
  for (int at = at0; at < end && tile < tab.tiles_cap; ++tile) {
    const int32_t* w = tab.tiles + (size_t)tile * PG_TILE;
    RaggedItem it;
    it.row0 = w[0]; it.rows = w[1]; it.start = w[2]; it.crow = w[3];
    it.j0 = w[4]; it.kb0 = at - w[5];
    const int units = w[6], take = min(units - it.kb0, end - at);
    // a plan of other tensors is not followed (a start below 0 has no keys, however many its rows)
    if (it.row0 < 0 || it.rows < 1 || it.row0 + (long long)it.rows > p.rows || (it.start >= 0 && it.start > p.cap - it.rows) ||
        it.crow < 0 || it.crow >= tab.B || it.j0 < 0 || it.kb0 < 0 || take < 1)
      return;
    it.pairs = it.rows * p.G;
    if (it.j0 >= it.pairs) return;
    it.kb1 = it.kb0 + take;
    it.part = take == units ? -1 : 2 * bin + (at != at0);
    if (it.part >= p.n_parts) return;
    at += take;
    it.kend = it.start + (min(it.j0 + RG_ROWS, it.pairs) - 1) / p.G + 1;
    if (it.start < 0) it.kb1 = it.kb0;                     // does not fit its pages: zero rows
    else if (it.kb1 > (it.kend + RG_KEYS - 1) / RG_KEYS) return;

    const auto run = [&](auto fine, auto narrow) __attribute__((always_inline)) {
      constexpr bool FINE = decltype(fine)::value, NARROW = decltype(narrow)::value;
      if (NARROW) {                                          // blocks of 32 keys
        it.kb0 *= 2;
        it.kb1 = min(2 * it.kb1, (it.kend + 31) / 32);
      }
      bool bad = false;
      const uint32_t odd = attend_item<RG_PAGED, FINE, false, NARROW>(p, it, h, s_kv, lane, wave, 0, bad);
      if (it.kb0 >= it.kb1) return;
      // (a wave writes these words after a barrier of the item, behind which no wave reads the last item's)
      if (lane == 0) s_odd[wave] = odd, s_bad[wave] = bad;
      lds_barrier();                                         // the buffers are free
      uint32_t any = 0;
      int none = 0;
#pragma unroll
      for (int w = 0; w < RG_WAVES; ++w) any |= s_odd[w], none |= s_bad[w];
      if (__builtin_amdgcn_readfirstlane(none)) {
        poison_item(p, it, h, lane, wave);
        return;
      }
      if (!__builtin_amdgcn_readfirstlane(any)) return;
      (void)attend_item<RG_PAGED, FINE, true, NARROW>(p, it, h, s_kv, lane, wave, odd, bad);
      lds_barrier();
    };
    if (among_wide && it.pairs <= PG_NARROW) run(std::true_type{}, std::true_type{});
    else if (it.pairs <= RG_ROWS) run(std::true_type{}, std::false_type{});
    else run(std::false_type{}, std::false_type{});
  }
}

// The parts of a cut tile joined, as the contiguous caches' merge; LANES lanes a pair.  4 us behind 32 tokens, 6 behind 16 x 5
// drafts (a launch, the merge's words, two rounds of parts), 2-3 where nothing was cut.
template <int LANES>
__global__ __launch_bounds__(256) void paged_merge_kernel(const RaggedAttnParams p, const PagedTables tab) {
  constexpr int JOINED = 256 / LANES;        // pairs of a workgroup
  const int lane = threadIdx.x & (LANES - 1);
  const int h = blockIdx.x % p.Hkv;
  const int groups = p.part_rows / JOINED;
  const int group = blockIdx.x / p.Hkv % groups;
  const int32_t* w = tab.merges + (size_t)(blockIdx.x / p.Hkv / groups) * PG_MERGE;
  const int row0 = w[0], rows = w[1], j0 = w[2], first = w[3], second = w[4], parts = w[5];
  if (rows < 1 || row0 < 0 || row0 + (long long)rows > p.rows || j0 < 0 || first < 0 || parts < 2 || second < 0 ||
      first >= p.n_parts || second + 2 * (parts - 2) >= p.n_parts)
    return;
  const int at = group * JOINED + (int)threadIdx.x / LANES;
  const int j = j0 + at;
  if (j >= (long long)rows * p.G) return;      // a pair's lanes together
  const int t = j / p.G;
  join_parts<LANES>(p, h, at, first, second, 2, parts, (size_t)row0 + t, h * p.G + (j - t * p.G), lane);
}

}  // namespace t2i

// ============================================================================
// host side
// ============================================================================
using t2i_host::aligned16;
using t2i_host::fail;

namespace {

bool aligned4(const void* p) { return ((uintptr_t)p & 3u) == 0; }
constexpr long long INT_MOST = 0x7FFFFFFF;

// What a plan holds: words of each of its tables.
struct PlanSizes {
  int tiles, bins, shares, merges;
  int64_t words;
};
PlanSizes plan_sizes(int32_t rows, int32_t B, int32_t G, int32_t Hkv) {
  PlanSizes z;
  z.tiles = (int)((long long)rows * G / t2i_host::RG_ROWS + B);
  z.shares = std::max(1, t2i_host::RG_SLOTS / Hkv);
  z.bins = std::max(z.tiles, z.shares);
  z.merges = std::min(z.tiles, z.shares);
  z.words = (int64_t)z.tiles * t2i::PG_TILE + (int64_t)z.bins * t2i::PG_BIN + (int64_t)z.merges * t2i::PG_MERGE + (int64_t)rows * t2i::PG_ROW;
  return z;
}

int page_shift(int32_t page_slots) { return 31 - __builtin_clz(page_slots); }

// What every paged call takes.
int check_paged(int32_t rows, int32_t B, int32_t max_pages, int32_t page_slots, int32_t Hq, int32_t Hkv) {
  if (Hkv < 1 || Hq < Hkv || Hq % Hkv) return fail(T2I_ERR_SHAPE, "Hq=%d Hkv=%d invalid", Hq, Hkv);
  if (Hq > 1024) return fail(T2I_ERR_SHAPE, "Hq=%d exceeds 1024", Hq);
  if (page_slots < 16 || page_slots > 65536 || (page_slots & (page_slots - 1)))
    return fail(T2I_ERR_SHAPE, "pages of %d slots unsupported (a power of two from 16 to 65536)", page_slots);
  if (B < 1 || B > t2i::PG_SEQS) return fail(T2I_ERR_SHAPE, "%d sequences (1 to %d)", B, t2i::PG_SEQS);
  if (max_pages < 1 || (long long)max_pages * page_slots > 1 << 23)
    return fail(T2I_ERR_SHAPE, "%d pages of %d slots a sequence (at most 8388608 slots)", max_pages, page_slots);
  if (rows < 1 || (long long)rows * Hq > INT_MOST - t2i_host::RG_ROWS || rows > (1 << 24) - 1)
    return fail(T2I_ERR_SHAPE, "rows=%d of %d heads invalid", rows, Hq);
  const PlanSizes z = plan_sizes(rows, B, Hq / Hkv, Hkv);
  const long long blocks = ((long long)max_pages * page_slots + t2i_host::RG_KEYS - 1) / t2i_host::RG_KEYS;
  if (z.tiles * blocks * 32 > INT_MOST || (long long)z.bins * Hkv > 0xFFFFFFFFLL / 256)
    return fail(T2I_ERR_SHAPE, "rows=%d of %d sequences over %d slots are too many", rows, B, max_pages * page_slots);
  return T2I_OK;
}

int check_pool(int32_t n_pages, int32_t D, const void* pages, const void* k, const void* v, const int32_t* plan, int64_t plan_words,
               int64_t need) {
  if (!pages || !k || !v || !plan) return fail(T2I_ERR_NULL, "paged pointers must not be NULL");
  if (D != t2i::RG_D) return fail(T2I_ERR_SHAPE, "head_dim %d unsupported (only 128)", D);
  if (n_pages < 1) return fail(T2I_ERR_SHAPE, "%d pages invalid", n_pages);
  if (!aligned16(k) || !aligned16(v)) return fail(T2I_ERR_ALIGN, "the pools must be 16-byte aligned");
  if (!aligned4(pages) || !aligned4(plan)) return fail(T2I_ERR_ALIGN, "pages and plan must be 4-byte aligned");
  if (plan_words < need) return fail(T2I_ERR_WORKSPACE, "the plan holds %lld words, %lld needed", (long long)plan_words, (long long)need);
  return T2I_OK;
}

// The tables of a plan in its buffer.
struct PlanTables {
  int32_t *tiles, *bins, *merges, *row;
  PlanTables(const int32_t* plan, const PlanSizes& z) {
    tiles = const_cast<int32_t*>(plan);
    bins = tiles + (size_t)z.tiles * t2i::PG_TILE;
    merges = bins + (size_t)z.bins * t2i::PG_BIN;
    row = merges + (size_t)z.merges * t2i::PG_MERGE;
  }
};

int part_rows(int32_t rows, int32_t G) { return (int)std::min<long long>(t2i_host::RG_ROWS, ((long long)rows * G + 31) / 32 * 32); }

}  // namespace

extern "C" int64_t t2i_paged_plan_words(int32_t rows, int32_t n_seqs, int32_t Hq, int32_t Hkv) {
  if (check_paged(rows, n_seqs, 1, 16, Hq, Hkv)) return 0;
  return plan_sizes(rows, n_seqs, Hq / Hkv, Hkv).words;
}

extern "C" int t2i_paged_plan(const int32_t* row_starts, const int32_t* context_lens, int32_t n_seqs, int32_t rows,
                              int32_t max_pages, int32_t page_slots, int32_t Hq, int32_t Hkv, int32_t* plan,
                              int64_t plan_words, void* stream) {
  if (!row_starts || !context_lens || !plan) return fail(T2I_ERR_NULL, "row_starts, context_lens and plan must not be NULL");
  if (!aligned4(row_starts) || !aligned4(context_lens) || !aligned4(plan))
    return fail(T2I_ERR_ALIGN, "row_starts, context_lens and plan must be 4-byte aligned");
  if (int rc = check_paged(rows, n_seqs, max_pages, page_slots, Hq, Hkv)) return rc;
  const PlanSizes z = plan_sizes(rows, n_seqs, Hq / Hkv, Hkv);
  if (plan_words < z.words) return fail(T2I_ERR_WORKSPACE, "the plan holds %lld words, %lld needed", (long long)plan_words, (long long)z.words);
  const PlanTables t(plan, z);
  t2i::PagedPlanParams p{};
  p.row_starts = row_starts; p.ctx = context_lens; p.tiles = t.tiles; p.bins = t.bins; p.merges = t.merges; p.row = t.row;
  p.rows = rows; p.B = n_seqs; p.G = Hq / Hkv; p.Hkv = Hkv; p.cap = max_pages * page_slots;
  p.tiles_cap = z.tiles; p.bins_cap = z.bins; p.shares = z.shares; p.merges_cap = z.merges;
  const int groups = 1 + (rows + t2i::PG_THREADS - 1) / t2i::PG_THREADS;
  hipLaunchKernelGGL(t2i::paged_plan_kernel, dim3(groups), dim3(t2i::PG_THREADS), 0, reinterpret_cast<hipStream_t>(stream), p);
  return t2i_host::hip_status(hipGetLastError(), "paged plan launch");
}

extern "C" int t2i_paged_qk_rope_kv(const uint16_t* qkv, int32_t rows, const int32_t* plan, int64_t plan_words,
                                    const int32_t* pages, int32_t n_seqs, int32_t max_pages, int32_t n_pages,
                                    int32_t page_slots, int32_t Hq, int32_t Hkv, int32_t D, const uint16_t* q_norm,
                                    const uint16_t* k_norm, float eps, const uint16_t* rope, int32_t rope_style,
                                    uint16_t* q_out, uint16_t* k_pages, uint16_t* v_pages, void* stream) {
  if (!qkv || !q_norm || !k_norm || !rope || !q_out) return fail(T2I_ERR_NULL, "paged prep pointers must not be NULL");
  if (!aligned16(qkv) || !aligned16(q_norm) || !aligned16(k_norm) || !aligned16(rope) || !aligned16(q_out))
    return fail(T2I_ERR_ALIGN, "paged prep tensors must be 16-byte aligned");
  if (rope_style != 0 && rope_style != 1) return fail(T2I_ERR_VALUE, "rope_style must be 0 or 1");
  if (!(eps > 0.0f)) return fail(T2I_ERR_VALUE, "eps must be positive");
  if (int rc = check_paged(rows, n_seqs, max_pages, page_slots, Hq, Hkv)) return rc;
  const PlanSizes z = plan_sizes(rows, n_seqs, Hq / Hkv, Hkv);
  if (int rc = check_pool(n_pages, D, pages, k_pages, v_pages, plan, plan_words, z.words)) return rc;
  t2i::PagedPrepParams p{};
  p.qkv = qkv; p.qn = q_norm; p.kn = k_norm; p.rope = rope; p.q = q_out; p.kc = k_pages; p.vc = v_pages;
  p.row = PlanTables(plan, z).row; p.pages = pages; p.B = n_seqs; p.Hq = Hq; p.Hkv = Hkv; p.cap = max_pages * page_slots;
  p.max_pages = max_pages; p.n_pages = n_pages; p.page_shift = page_shift(page_slots); p.style = rope_style; p.eps = eps;
  hipLaunchKernelGGL(t2i::paged_prep_kernel, dim3(rows), dim3(256), 0, reinterpret_cast<hipStream_t>(stream), p);
  return t2i_host::hip_status(hipGetLastError(), "paged prep launch");
}

extern "C" size_t t2i_paged_attention_workspace_bytes(int32_t rows, int32_t Hq, int32_t Hkv) {
  if (rows < 1 || Hkv < 1 || Hq < Hkv || Hq % Hkv || Hq > 1024) return 0;
  const size_t parts = 2 * (size_t)std::max(1, t2i_host::RG_SLOTS / Hkv);
  return parts * Hkv * part_rows(rows, Hq / Hkv) * (t2i::RG_D * sizeof(float) + sizeof(float2));
}

extern "C" int t2i_paged_attention(const uint16_t* q, int32_t rows, const int32_t* plan, int64_t plan_words,
                                   const int32_t* pages, int32_t n_seqs, int32_t max_pages, int32_t n_pages,
                                   int32_t page_slots, int32_t Hq, int32_t Hkv, int32_t D, const uint16_t* k_pages,
                                   const uint16_t* v_pages, uint16_t* out, float* out_sums, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  if (!q || !out) return fail(T2I_ERR_NULL, "paged attention pointers must not be NULL");
  if (!aligned16(q) || !aligned16(out)) return fail(T2I_ERR_ALIGN, "paged attention tensors must be 16-byte aligned");
  if (!aligned4(out_sums)) return fail(T2I_ERR_ALIGN, "out_sums must be 4-byte aligned");
  if (int rc = check_paged(rows, n_seqs, max_pages, page_slots, Hq, Hkv)) return rc;
  const PlanSizes z = plan_sizes(rows, n_seqs, Hq / Hkv, Hkv);
  if (int rc = check_pool(n_pages, D, pages, k_pages, v_pages, plan, plan_words, z.words)) return rc;
  const size_t need = t2i_paged_attention_workspace_bytes(rows, Hq, Hkv);
  if (!workspace || workspace_bytes < need) return fail(T2I_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : 0, need);
  if (!aligned16(workspace)) return fail(T2I_ERR_ALIGN, "the workspace must be 16-byte aligned");
  t2i::RaggedAttnParams p{};
  p.q = q; p.kc = k_pages; p.vc = v_pages; p.out = out; p.out_sums = out_sums; p.rows = rows;
  p.Hq = Hq; p.Hkv = Hkv; p.G = Hq / Hkv; p.cap = max_pages * page_slots;
  p.pages = pages; p.max_pages = max_pages; p.n_pages = n_pages; p.page_shift = page_shift(page_slots);
  p.scale_log2 = (float)(1.4426950408889634 / sqrt((double)D));
  p.n_parts = 2 * z.shares;
  p.part_rows = part_rows(rows, p.G);
  p.part_o = reinterpret_cast<float*>(workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + (size_t)p.n_parts * Hkv * p.part_rows * t2i::RG_D);
  const PlanTables t(plan, z);
  const t2i::PagedTables tab{t.tiles, t.bins, t.merges, z.tiles, n_seqs};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  constexpr int LDS_BYTES = 2 * 2 * t2i::RG_KEYS * t2i::RG_D * 2;   // two buffers of K and V
  hipLaunchKernelGGL(t2i::paged_attention_kernel, dim3(z.bins * Hkv), dim3(64 * t2i::RG_WAVES), LDS_BYTES, s, p, tab);
  if (int rc = t2i_host::hip_status(hipGetLastError(), "paged attention launch")) return rc;
  // Tiles enough for all shares are mostly handed out whole, and then what this launch takes is its waves that find
  // nothing to do: a quarter of them with 8 lanes a pair (16 prompts of 37 to 1021 rows 36.9 -> 34.5 us).  Few tiles are
  // cut into many parts, which more lanes join sooner (a single token 10.6 us, with 8 lanes 11.6; 2 x 9 drafts 45.6, 48.8).
  const auto merge = [&](auto lanes) {
    constexpr int LANES = decltype(lanes)::value;
    hipLaunchKernelGGL(t2i::paged_merge_kernel<LANES>, dim3(z.merges * Hkv * (p.part_rows * LANES / 256)), dim3(256), 0, s, p, tab);
  };
  if (z.tiles >= z.shares) merge(std::integral_constant<int, 8>{});
  else merge(std::integral_constant<int, 32>{});
  return t2i_host::hip_status(hipGetLastError(), "paged attention merge launch");
}
