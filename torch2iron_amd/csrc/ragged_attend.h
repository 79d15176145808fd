// Attention of one tile of (row, q head) pairs over blocks of keys, and the join of its parts, for
// the ragged batches over a contiguous cache (packed prompts, drafted trees) and over a cache in pages.
#pragma once

#include <math.h>

#include "t2i_common.h"
#include "ragged_plan.h"

namespace t2i {

constexpr int RG_D = 128;
constexpr int RG_KEYS = t2i_host::RG_KEYS;
constexpr int RG_WAVES = 4;                  // waves of a workgroup of the attention, 32 pairs each
constexpr int RG_ROWS = t2i_host::RG_ROWS;
constexpr int RG_ITEM = t2i_host::RG_ITEM;
constexpr int TREE_NODES = 64;               // nodes of a tree: one lane of a wave each

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) short i16x4;

// ---- trees: a wave holds one, lane i its node i ----

// The parent of node `lane`, or -1 for a root (a parent outside [0, lane) makes one).
__device__ __forceinline__ int tree_parent(const int32_t* parents, int N, int lane) {
  const int p = parents[min(lane, N - 1)];
  return p >= 0 && p < lane ? p : -1;
}

// Nodes above the lane's node, whose parent is p, by doubling the steps: after k rounds a lane
// knows the nodes up to 2^k steps above it, and the one that stands there.
__device__ __forceinline__ unsigned long long tree_above(int p) {
  uint32_t lo = 0, hi = 0;
  if (p >= 0) (p < 32 ? lo : hi) = 1u << (p & 31);
#pragma unroll
  for (int k = 0; k < 6; ++k) {
    const int at = max(p, 0);
    const uint32_t l = __shfl(lo, at, 64), h = __shfl(hi, at, 64);
    const int q = __shfl(p, at, 64);
    if (p >= 0) {
      lo |= l;
      hi |= h;
      p = q;
    }
  }
  return (unsigned long long)hi << 32 | lo;
}

// A tree's nodes and context as the kernels take them: nodes = 0 where there is nothing to
// do; ok: the context and its nodes lie in the cache.
struct TreeSeq {
  int ctx, nodes;
  bool ok;
};
__device__ __forceinline__ TreeSeq tree_seq(const int32_t* ctx_lens, const int32_t* counts, int b, int N, int cap) {
  TreeSeq t;
  t.ctx = ctx_lens[b];
  t.nodes = counts ? max(0, min(counts[b], N)) : N;
  t.ok = t.ctx >= 0 && t.ctx <= cap - t.nodes;
  return t;
}

struct RaggedAttnParams {
  const uint16_t* q;        // [rows, Hq, D]
  const uint16_t* kc;       // [cache rows, Hkv, cap, D]
  const uint16_t* vc;
  uint16_t* out;            // [rows, Hq * D]
  float* out_sums;          // NULL, or [Hq, rows]: each head's sum of its bf16 context values
  float* part_o;            // [parts][Hkv][part_rows][D] unnormalised outputs of a part of the keys
  float2* part_ml;          // [parts][Hkv][part_rows] their running maximum and sum
  int2* cuts;               // trees: [B] first slot and last run of a cut sequence ({-1, }: it is in one piece)
  const int32_t* items;     // packed: [n_items][RG_ITEM]; merge: [n_merges][RG_ITEM]
  const int32_t* bins;      // packed: [n_bins + 1] each workgroup's first item
  const int32_t* parents;   // trees: [B, N]
  const int32_t* ctx;
  const int32_t* counts;
  long long rows;
  int n_cache, n_items, n_bins, n_parts, part_rows, Hq, Hkv, G, cap, B, N, tiles;
  float scale_log2;         // D^-1/2 * log2(e)
  // keys in pages: kc and vc are [n_pages, Hkv, 2^page_shift, D]
  const int32_t* pages;     // [B, max_pages] the page of each 2^page_shift slots of a sequence
  int max_pages, n_pages, page_shift;
};

// Where an item's keys stand, and which of them a row sees: a prompt's rows in a cache row (causal), a drafted
// tree's nodes in a cache row, or rows whose slots are in pages (causal).
enum RaggedForm { RG_PACKED, RG_TREE, RG_PAGED };

// A piece of work: the tile of a sequence's (row, q head of a kv head) pairs from j0 on, over key
// blocks kb0 .. kb1 - 1; keys from kend on are seen by none of its rows.
struct RaggedItem {
  int row0, rows, start, crow, kb0, kb1, part, kend, j0, pairs;
};

typedef __attribute__((ext_vector_type(4))) int i32x4;

// Until every LDS operation of this wave is done, and every wave is here.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}
// Until every vector memory operation of this wave is done, and every wave is here.
__device__ __forceinline__ void loads_done_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}
// Loads straight into LDS are written as asm, left in flight, because the compiler waits for
// every one of them before any read of LDS; loads_done_barrier covers them.  The compiler does
// not look into asm for hazards: M0 is written a wait state before the load that reads it, and
// an SGPR that a VALU instruction wrote is five wait states away from a load.
//
// 16 bytes a lane from byte `at` of a buffer into LDS at lds + 16 lane.
__device__ __forceinline__ void lds_load16(i32x4 rsrc, uint32_t at, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :: "s"(lds), "v"(at), "s"(rsrc) : "memory", "m0");
}
// 16 keys from a buffer, four an instruction, the lane's chunk of instruction i's at byte at[i]
// (from soff on, less 1024 i).  An instruction's offset counts for the memory address and for
// the LDS address.
// ONCE: past the caches' own order (nt), for keys that no other workgroup reads.
#define T2I_KEYS(mod)                                                                                             \
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\t"                                                                  \
               "buffer_load_dwordx4 %1, %5, %6 offen" mod " lds\n\t"                                              \
               "buffer_load_dwordx4 %2, %5, %6 offen offset:1024" mod " lds\n\t"                                  \
               "buffer_load_dwordx4 %3, %5, %6 offen offset:2048" mod " lds\n\t"                                  \
               "buffer_load_dwordx4 %4, %5, %6 offen offset:3072" mod " lds"                                      \
               :: "s"(lds), "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "s"(rsrc), "s"(soff) : "memory", "m0")
template <bool ONCE>
__device__ __forceinline__ void lds_load_keys(i32x4 rsrc, const uint32_t (&at)[4], uint32_t soff, uint32_t lds) {
  if constexpr (ONCE) {
    T2I_KEYS(" nt");
  } else {
    T2I_KEYS("");
  }
}
#undef T2I_KEYS
// The same for 8 keys.
__device__ __forceinline__ void lds_load_keys(i32x4 rsrc, const uint32_t (&at)[2], uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\t"
               "buffer_load_dwordx4 %1, %3, 0 offen nt lds\n\t"
               "buffer_load_dwordx4 %2, %3, 0 offen offset:1024 nt lds"
               :: "s"(lds), "v"(at[0]), "v"(at[1]), "s"(rsrc) : "memory", "m0");
}
// A buffer over everything from p on (every offset used is inside the cache: checked or clamped).
__device__ __forceinline__ i32x4 keys_rsrc(const void* p) {
  const uint64_t a = (uint64_t)(uintptr_t)p;
  return i32x4{(int)__builtin_amdgcn_readfirstlane((uint32_t)a),
               (int)(__builtin_amdgcn_readfirstlane((uint32_t)(a >> 32)) & 0xFFFF), -1, 0x00027000};
}
__device__ __forceinline__ uint32_t rg_lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}
// max / sum over the two lanes (c, c + 32) of a row, in both
__device__ __forceinline__ float pair_max(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float pair_sum(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// Two bf16 values, 0 in the place of infinities and NaN.
__device__ __forceinline__ uint32_t finite_or_zero(uint32_t w) {
  if ((w & 0x7F80u) == 0x7F80u) w &= 0xFFFF0000u;
  return (w & 0x7F800000u) == 0x7F800000u ? w & 0xFFFFu : w;
}

// An item of a workgroup, for one kv head: four waves of 32 pairs.  All products run transposed on
// the 32 x 32 x 16 MFMA, so that a lane (c = lane % 32, h2 = lane / 32) holds one pair's scores and
// outputs:
//   S^T = K Q^T: A = K from LDS (lane: key 32 n + c, dims 16 ks + 8 h2 ..), B = the wave's q
//     rows (registers); register i holds the score of key 32 n + 8 (i / 4) + 4 h2 + i % 4;
//   the online softmax per lane: the row's maximum from its two lanes by one lane swap, the
//     weights' sum left per lane until the end.  The reference m moves only when a maximum
//     passes it by 8 (weights up to 2^8, the same relative precision): after the first blocks
//     outputs are hardly ever rescaled;
//   O^T += V^T P^T: B = P^T straight from those registers, rounded to bf16 (16 keys a step, in
//     the order they stand in), A = V^T from LDS in that order by transposing reads
//     (ds_read_b64_tr_b16: four keys of one dim a lane out of V's own row order).
// FINE: what the rounding of the weights left is a second bf16 word and V is multiplied by both:
// weights of 16 bits, whose error the output's own rounding hides, normalised by their fp32 sum.  Trees
// and sequences of one row take it, since they stand in for decode steps, whose weights are fp32
// (16 x 26 nodes 46 -> 48 us, 8 x 64 nodes over 32k slots 270 -> 330, 16 single rows 32.8 -> 34.1); prompt
// rows round their weights once, as the batch form of the prompt pass does (8001 rows: 517 us,
// with FINE 713).
// In an MFMA a weight of 0 times an infinity or a NaN in V is a NaN, also for rows whose mask hides that
// key.  An item with sums that are not finite is therefore run again, MASKED: blocks that some row does
// not see whole and whose V holds such a value are multiplied key by key for the rows that attend it; FINE
// multiplies its second words by V without such values, since they may be 0 or negative.  (500 rows from
// 1500, 16 / 8 heads, without such values 32 us, with a NaN in the last slot 76, in the first 46; 1624 and
// 2384 where such rows were formed again from all of their keys.)
// K and V blocks go straight from memory into LDS, two buffers, one barrier a block; a row's
// 16-byte chunk ch stands at place ch ^ (row % 16) (K) or ch ^ 4 (row % 4) (V): 16 neighbouring
// lanes of a K read, 32 of a transposing read cover all banks (a load into LDS cannot pad rows,
// but each lane chooses what it loads; with ch ^ 2 (row % 8) for both, half of the cycles of
// LDS were bank conflicts).  Keys past the last one reload it: slots that no row attends are
// never read.
//   The buffers take 64 KB: two workgroups a CU.  Eight waves with four buffers, whose K and V come once
// for 256 pairs, gained nothing for trees of more than 128 pairs (this form / eight waves: 8 x 64 nodes, 4 q
// heads a kv head, 32k slots 318 / 325 us; 1 x 64 over 4k 26.9 / 29.3; 2 x 64 of 8 q heads over 20k 138 / 137).
// What bounds it (one MI355X; a bulk read reaches 6.7 TB/s, an 8192^3 product 1.21 PFLOP/s):
//   8001 rows from 0, 32 / 8 heads: 500-530 us, 0.99-1.05 PFLOP/s.  MFMAs take 54 % of a SIMD's
//     cycles and VALU instructions as many beside them, at the 1.8-1.9 GHz that the card holds
//     under this load; LDS 27 % of a CU's, no bank conflicts.
//   16 x 26 nodes over 901 to 4001 slots, 16 / 8 heads: 48 us with the merge; 42 without, in which
//     164 MB come from memory (3.9 TB/s) and waves wait 67 % of their time.
//   8 x 64 nodes over 15007 to 32003 slots, 32 / 8 heads: 318-345 us with the merge (10): MFMA 52 % of a
//     SIMD's cycles, a third of them for the second words; 781 MB, 2.4 TB/s.
//   16 prompts of 37 to 1021 rows: 29-32 us: first loads and outputs of items of up to 16 blocks.
// Measured and dropped: one half's softmax beside the other half's products (8 % slower), priorities
// around the products (1-3 %), scheduling groups and iglp (0-4 %), two waves sharing the blocks of a
// tile of up to 32 pairs (single rows 5 % faster, everything else 3-8 % slower: registers).
// Returns the wave's pairs (bit c) whose sums are not finite, which were not written; MASKED: writes `only` those.
// Pages: a wave's 16 keys of a block lie in one page (pages hold 16 2^n slots), whose id comes by a scalar load a
// block ahead; the buffer starts at its first slot, so that offsets stay small whatever the pool's size.  An id
// outside the pool is read as page 0 and raises `bad`.
// NARROW (pages, up to 32 pairs): one wave multiplies, and what counts is how much is on its way from memory.  Blocks of 32
// keys (kb0 and kb1 count those) in four buffers: three are loading while one is multiplied, where two buffers of
// 64 keys leave half of them.
template <RaggedForm FORM, bool FINE, bool MASKED, bool NARROW = false>
__device__ __forceinline__ uint32_t attend_item(const RaggedAttnParams& p, const RaggedItem& it, int h, uint16_t* s_kv, int lane,
                                                int wave, uint32_t only, bool& bad) {
  constexpr int D = RG_D;
  constexpr bool TREE = FORM == RG_TREE, PAGED = FORM == RG_PAGED;
  static_assert(!NARROW || PAGED);
  constexpr int KEYS = NARROW ? 32 : RG_KEYS, STAGES = NARROW ? 4 : 2;   // keys of a block, blocks in LDS
  constexpr int WKEYS = KEYS / RG_WAVES;       // keys of a block that a wave loads
  const int c = lane & 31, h2 = lane >> 5;

  // ---- K / V staging: a wave's instruction moves 4 keys (1 KB); 4 each of K and V a block ----
  const size_t cache_base = PAGED ? 0 : ((size_t)it.crow * p.Hkv + h) * (size_t)p.cap * D;
  const int srow = lane >> 4;                              // key within the instruction's four
  const int place = lane & 15;                             // where the lane's 16 bytes go in the key's row
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(rg_lds_address(s_kv) + wave * WKEYS * D * 2);
  constexpr int LOADS = WKEYS / 4;                         // instructions of a wave for K, and for V
  uint32_t kat[LOADS], vat[LOADS];                         // what the lane loads: byte in the block, less 1024 i
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int key = PAGED ? srow : wave * WKEYS + srow;    // pages: from the wave's first key on
    kat[i] = key * (D * 2) + 16 * (place ^ ((wave * WKEYS + 4 * i + srow) & 15));
    vat[i] = key * (D * 2) + 16 * (place ^ (4 * srow));
  }
  i32x4 krsrc = keys_rsrc(p.kc + cache_base), vrsrc = keys_rsrc(p.vc + cache_base);
  // pages: the wave's first key of a block (at most the last key there is), and its page
  auto wave_key = [&](int kb) __attribute__((always_inline)) { return min(kb * KEYS + wave * WKEYS, it.kend - 1) & -WKEYS; };
  auto page_of = [&](int kb) __attribute__((always_inline)) {
    typedef const __attribute__((address_space(4))) int32_t* scalar_ptr;
    return ((scalar_ptr)(uintptr_t)(p.pages + (size_t)it.crow * p.max_pages))[wave_key(kb) >> p.page_shift];
  };
  int page = 0;                                            // of the next block to load
  if (PAGED && it.kb0 < it.kb1) page = page_of(it.kb0);
  // K and V block kb into its buffer
  auto stage = [&](int kb) __attribute__((always_inline)) {
    const uint32_t lds = lds0 + ((kb - it.kb0) & (STAGES - 1)) * (4 * KEYS * D);
    if constexpr (PAGED) {
      const bool in = (uint32_t)page < (uint32_t)p.n_pages;
      bad |= !in;
      const size_t first = (((size_t)(in ? page : 0) * p.Hkv + h) << p.page_shift) + (wave_key(kb) & ((1 << p.page_shift) - 1));
      krsrc = keys_rsrc(p.kc + first * D);
      vrsrc = keys_rsrc(p.vc + first * D);
      page = page_of(min(kb + 1, it.kb1 - 1));
    }
    if ((kb + 1) * KEYS <= it.kend) {
      const uint32_t at = PAGED ? 0u : (uint32_t)kb * (KEYS * D * 2);
      if constexpr (NARROW) {
        lds_load_keys(krsrc, kat, lds);
        lds_load_keys(vrsrc, vat, lds + 2 * KEYS * D);
      } else if (it.pairs <= RG_ROWS) {                     // the sequence's only tile: its keys are read once
        lds_load_keys<true>(krsrc, kat, at, lds);
        lds_load_keys<true>(vrsrc, vat, at, lds + 2 * KEYS * D);
      } else {
        lds_load_keys<false>(krsrc, kat, at, lds);
        lds_load_keys<false>(vrsrc, vat, at, lds + 2 * KEYS * D);
      }
    } else {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int at = wave * WKEYS + 4 * i + srow;
        const uint32_t key = (uint32_t)(PAGED ? min(4 * i + srow, it.kend - 1 - wave_key(kb)) : min(kb * KEYS + at, it.kend - 1)) * (D * 2);
        lds_load16(krsrc, key + 16 * (place ^ (at & 15)), lds + i * 4 * D * 2);
        lds_load16(vrsrc, key + 16 * (place ^ (4 * srow)), lds + 2 * KEYS * D + i * 4 * D * 2);
      }
    }
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s)
    if (it.kb0 + s < it.kb1) stage(it.kb0 + s);

  // ---- this lane's pair, and its q row as the B operand ----
  const int j = it.j0 + wave * 32 + c;
  const bool wave_on = it.j0 + wave * 32 < it.pairs && (!MASKED || only);   // some pair of the wave is to be done
  const int jj = min(j, it.pairs - 1);
  const int t = jj / p.G;
  const int head = h * p.G + (jj - t * p.G);
  const size_t qrow = (size_t)it.row0 + t;
  u32x4 qb[8];
  {
    const uint16_t* src = p.q + (qrow * p.Hq + head) * D + 8 * h2;
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) qb[ks] = *reinterpret_cast<const u32x4*>(src + 16 * ks);
  }
  // positions of the wave's rows: first and last (wave-uniform), this lane's
  const int t_first = (it.j0 + wave * 32) / p.G;
  const int t_last = (min(it.j0 + wave * 32 + 32, it.pairs) - 1) / p.G;
  const int qpos = it.start + t;
  const int mask_from = TREE ? it.start : it.start + t_first + 1;   // keys below it are seen by every row
  const int wave_end = TREE ? it.kend : it.start + t_last + 1;      // keys from it on by none
  uint32_t seen_lo = 0, seen_hi = 0;                       // tree: the nodes that the lane's node attends
  if (TREE && it.kb1 * KEYS > it.start && it.kb0 < it.kb1) {
    const unsigned long long own = 1ull << lane;
    const unsigned long long s = tree_above(tree_parent(p.parents + (size_t)it.row0, p.N, lane)) | own;
    seen_lo = __shfl((uint32_t)s, t, 64);
    seen_hi = __shfl((uint32_t)(s >> 32), t, 64);
  }

  float m = -INFINITY, mref = 0.0f, l = 0.0f;              // mref: m, or 0 while m is -inf; l: of this lane's keys
  f32x16 o[4];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[dt][i] = 0.0f;

  // LDS offsets (elements): K row c of a 32-key tile, V rows by transposing reads
  const int kx = c & 15;
  const int vi = lane & 15, vrow = 4 * h2 + (vi >> 2);     // key of the 8 that the lane's read names
  const int vcol = 2 * ((lane >> 4) & 1) + ((vi & 3) >> 1);   // its 16-byte chunk within a 32-dim tile

  if constexpr (NARROW) {
    // The loop counts its own loads, four a block: nothing else may be on its way in it.  (Not known to the compiler,
    // which so waits for the q rows here and not at their use.)
    asm volatile("s_waitcnt vmcnt(0)"
                 : "+v"(qb[0]), "+v"(qb[1]), "+v"(qb[2]), "+v"(qb[3]), "+v"(qb[4]), "+v"(qb[5]), "+v"(qb[6]), "+v"(qb[7]) :: "memory");
  }
  for (int kb = it.kb0; kb < it.kb1; ++kb) {
    // this block is here, the buffer of the one before it free
    if constexpr (NARROW) {
      if (kb + 2 < it.kb1) asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      else if (kb + 1 < it.kb1) asm volatile("s_waitcnt vmcnt(4) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      else loads_done_barrier();
    } else {
      loads_done_barrier();
    }
    if (kb + STAGES - 1 < it.kb1) stage(kb + STAGES - 1);
    if (!wave_on || kb * KEYS >= wave_end) continue;
    const uint16_t* const bk = s_kv + ((kb - it.kb0) & (STAGES - 1)) * (2 * KEYS * D);
    const uint16_t* const bv = bk + KEYS * D;
    // ---- S^T = K Q^T ----
    f32x16 s[KEYS / 32];
#pragma unroll
    for (int n = 0; n < KEYS / 32; ++n) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[n][i] = 0.0f;
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) {
        const u32x4 ka = *reinterpret_cast<const u32x4*>(bk + (32 * n + c) * D + ((2 * ks + h2) ^ kx) * 8);
        s[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, ka),
                                                       __builtin_bit_cast(bf16x8, qb[ks]), s[n], 0, 0, 0);
      }
    }
    // ---- masks, only on blocks that some row does not see whole ----
    if (kb * KEYS + KEYS > mask_from) {
      if (TREE) {
        const int rel = kb * KEYS - it.start;           // node of the block's first key (negative: a context slot)
        const unsigned long long w = (unsigned long long)seen_hi << 32 | seen_lo;
        unsigned long long bm = rel >= 64 ? 0ull : rel >= 0 ? w >> rel : (w << -rel) | ((1ull << -rel) - 1);
        bm >>= 4 * h2;
#pragma unroll
        for (int n = 0; n < KEYS / 32; ++n)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (!((uint32_t)(bm >> (32 * n)) & (1u << (8 * (i / 4) + i % 4)))) s[n][i] = -INFINITY;
      } else {
        const int rel = qpos - kb * KEYS - 4 * h2;
#pragma unroll
        for (int n = 0; n < KEYS / 32; ++n)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (32 * n + 8 * (i / 4) + i % 4 > rel) s[n][i] = -INFINITY;
      }
    }
    // ---- online softmax (log2 domain) ----
    float mx = fmaxf(s[0][0], s[KEYS / 32 - 1][0]);
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, fmaxf(s[0][i], s[KEYS / 32 - 1][i]));
    mx = pair_max(mx) * p.scale_log2;
    if (__any(mx > m + (MASKED ? 0.0f : 8.0f))) {          // MASKED: no weight above 1, sums of huge values fit
      const float mn = fmaxf(m, mx);
      const float f = m > -INFINITY ? exp2_fast(m - mn) : 0.0f;
      l *= f;
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[dt][i] *= f;
      m = mn;
      mref = mn > -INFINITY ? mn : 0.0f;
    }
    // ---- MASKED: where V holds an infinity or a NaN, key by key for the rows that attend it ----
    if constexpr (MASKED) {
      if (kb * KEYS + KEYS > mask_from) {
        bool odd = false;
#pragma unroll 4
        for (int i = 0; i < KEYS / 4; ++i) {
          const u32x4 x = *reinterpret_cast<const u32x4*>(bv + 4 * i * D + 8 * lane);
#pragma unroll
          for (int e = 0; e < 4; ++e) odd |= finite_or_zero(x[e]) != x[e];
        }
        if (__any(odd)) {
          const uint32_t unseen = __float_as_uint(-1.0f);  // no weight
#pragma unroll
          for (int n = 0; n < KEYS / 32; ++n)
#pragma unroll 1
            for (int i = 0; i < 16; ++i) {
              const float x = s[n][i], e = exp2_fast(fmaf(x, p.scale_log2, -mref));
              const uint32_t w = x == -INFINITY ? unseen : __float_as_uint(FINE ? e : round_bf16(e));
              l += w == unseen ? 0.0f : __uint_as_float(w);
              const auto two = __builtin_amdgcn_permlane32_swap(w, w, false, false);
#pragma unroll 1
              for (int half = 0; half < 2; ++half) {
                const uint32_t wk = half ? two[1] : two[0], sees = wk == unseen ? 0u : ~0u;
                const float weight = __uint_as_float(wk & sees);
                const int key = 32 * n + 8 * (i / 4) + 4 * half + i % 4;
                const uint16_t* const v = bv + key * D + 4 * h2;
#pragma unroll
                for (int dt = 0; dt < 4; ++dt) {
                  __builtin_amdgcn_sched_barrier(0);       // a few reads at a time: registers
#pragma unroll
                  for (int g = 0; g < 4; ++g) {
                    const u32x2 y = *reinterpret_cast<const u32x2*>(v + ((4 * dt + g) ^ (4 * (key & 3))) * 8) & sees;
                    o[dt][4 * g] = fmaf(weight, bf16_lo(y.x), o[dt][4 * g]);
                    o[dt][4 * g + 1] = fmaf(weight, bf16_hi(y.x), o[dt][4 * g + 1]);
                    o[dt][4 * g + 2] = fmaf(weight, bf16_lo(y.y), o[dt][4 * g + 2]);
                    o[dt][4 * g + 3] = fmaf(weight, bf16_hi(y.y), o[dt][4 * g + 3]);
                  }
                }
              }
            }
          continue;
        }
      }
    }
    uint32_t pw[KEYS / 32][8], pr[KEYS / 32][8];                           // bf16 weights, two keys a word; what their rounding left
#pragma unroll
    for (int n = 0; n < KEYS / 32; ++n)
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const float e0 = exp2_fast(fmaf(s[n][i], p.scale_log2, -mref)), e1 = exp2_fast(fmaf(s[n][i + 1], p.scale_log2, -mref));
        const uint32_t w = pack_bf16x2(e0, e1);
        pw[n][i / 2] = w;
        if constexpr (FINE) {
          pr[n][i / 2] = pack_bf16x2(e0 - bf16_lo(w), e1 - bf16_hi(w));
          l += e0 + e1;
        } else {
          l = dot2_bf16(w, 0x3F803F80u, l);                // the rounded weights
        }
      }
    // ---- O^T += V^T P^T ----
#pragma unroll
    for (int u = 0; u < KEYS / 16; ++u) {
      const uint32_t* const w = pw[u / 2] + 4 * (u % 2);
      const uint32_t* const r = pr[u / 2] + 4 * (u % 2);
      bf16x8 va[4];
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) {
        const uint16_t* const v = bv + (16 * u + vrow) * D + ((4 * dt + vcol) ^ (4 * (vi >> 2))) * 8 + 4 * (vi & 1);
        typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
        const i16x4 a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(v));
        const i16x4 a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(v + 8 * D));
        const u32x2 b0 = __builtin_bit_cast(u32x2, a0), b1 = __builtin_bit_cast(u32x2, a1);
        va[dt] = __builtin_bit_cast(bf16x8, u32x4{b0.x, b0.y, b1.x, b1.y});
        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va[dt], __builtin_bit_cast(bf16x8, u32x4{w[0], w[1], w[2], w[3]}), o[dt], 0, 0, 0);
      }
      if constexpr (FINE) {
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) {
          if (MASKED) {                                    // a second word may be 0 or negative
            u32x4 x = __builtin_bit_cast(u32x4, va[dt]);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = finite_or_zero(x[e]);
            va[dt] = __builtin_bit_cast(bf16x8, x);
          }
          o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va[dt], __builtin_bit_cast(bf16x8, u32x4{r[0], r[1], r[2], r[3]}), o[dt], 0, 0, 0);
        }
      }
    }
  }

  // ---- outputs: register i of o[dt] is dim 32 dt + 8 (i / 4) + 4 h2 + i % 4 of the lane's pair ----
  if (!wave_on) return 0;
  l = pair_sum(l);
  if constexpr (!MASKED) {
    float finite = 0.0f * l;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) finite = fmaf(0.0f, o[dt][i], finite);
    const unsigned long long odd = __ballot(finite != finite);
    only = (uint32_t)(odd | odd >> 32);                    // bit c: the pair of lanes c and c + 32
  }
  const bool live = j < it.pairs && (only >> c & 1) == MASKED;
  if (it.part >= 0) {
    const size_t st = ((size_t)it.part * p.Hkv + h) * p.part_rows + wave * 32 + c;
    m = l != l ? INFINITY : m;                             // a row that saw a NaN stays one in the merge
    if (live && h2 == 0) p.part_ml[st] = float2{m, l};
    if (live && m > -INFINITY) {                           // else its outputs are not read
      float* dst = p.part_o + st * D + 4 * h2;
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<f32x4*>(dst + 32 * dt + 8 * g) = f32x4{o[dt][4 * g], o[dt][4 * g + 1], o[dt][4 * g + 2], o[dt][4 * g + 3]};
    }
    return only;
  }
  const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);   // nothing attended: a zero row; NaN stays
  uint16_t* const dst = p.out + (qrow * p.Hq + head) * D + 8 * h2;
  float hs = 0.0f;
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int g = 0; g < 4; g += 2) {
      uint32_t x[2], y[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        x[e] = pack_bf16x2(o[dt][4 * g + 2 * e] * inv, o[dt][4 * g + 2 * e + 1] * inv);
        y[e] = pack_bf16x2(o[dt][4 * g + 4 + 2 * e] * inv, o[dt][4 * g + 5 + 2 * e] * inv);
        hs += (bf16_lo(x[e]) + bf16_hi(x[e])) + (bf16_lo(y[e]) + bf16_hi(y[e]));
      }
      // lanes trade halves: each ends up with 8 neighbouring dims
      const auto a = __builtin_amdgcn_permlane32_swap(x[0], y[0], false, false);
      const auto b = __builtin_amdgcn_permlane32_swap(x[1], y[1], false, false);
      if (live) *reinterpret_cast<u32x4*>(dst + 32 * dt + 8 * g) = u32x4{a[0], b[0], a[1], b[1]};
    }
  if (p.out_sums) {
    hs = pair_sum(hs);
    if (live && h2 == 0) p.out_sums[(size_t)head * p.rows + qrow] = hs;
  }
  return only;
}

// The parts of a tile joined, for one (row, q head) pair: LANES lanes, 128 / LANES dims each; parts in their order
// (first, then second, second + step, ...), MERGE_AHEAD of them in flight, with a running maximum.
constexpr int MERGE_AHEAD = 4;
constexpr int MERGE_PAIRS = t2i_host::RG_MERGE;

template <int LANES>
__device__ __forceinline__ void join_parts(const RaggedAttnParams& p, int h, int at, int first, int second, int step, int parts,
                                           size_t qrow, int head, int lane) {
  constexpr int D = RG_D, PER = D / 4 / LANES;             // dims 4 lane + 4 LANES i
  float M = -INFINITY, l = 0.0f;
  f32x4 o[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < parts; s0 += MERGE_AHEAD) {
    float2 ml[MERGE_AHEAD];
    f32x4 v[MERGE_AHEAD][PER];
#pragma unroll
    for (int u = 0; u < MERGE_AHEAD; ++u) {
      const int s = min(s0 + u, parts - 1), part = s == 0 ? first : second + (s - 1) * step;
      const size_t st = ((size_t)part * p.Hkv + h) * p.part_rows + at;
      ml[u] = p.part_ml[st];
#pragma unroll
      for (int i = 0; i < PER; ++i) v[u][i] = *reinterpret_cast<const f32x4*>(p.part_o + st * D + 4 * lane + 4 * LANES * i);
    }
    float mn = M;
#pragma unroll
    for (int u = 0; u < MERGE_AHEAD; ++u) mn = fmaxf(mn, ml[u].x);
    const float f = state_weight(M, mn);
    l *= f;
#pragma unroll
    for (int i = 0; i < PER; ++i) o[i] *= f;
    M = mn;
#pragma unroll
    for (int u = 0; u < MERGE_AHEAD; ++u) {
      const bool some = s0 + u < parts && ml[u].x > -INFINITY;   // else nothing was attended, nor written
      const float g = exp2_fast(ml[u].x - M);
      l += some ? g * ml[u].y : 0.0f;
#pragma unroll
      for (int i = 0; i < PER; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] += some ? g * v[u][i][e] : 0.0f;
    }
  }
  const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
  float hs = 0.0f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const u32x2 w = u32x2{pack_bf16x2(o[i][0] * inv, o[i][1] * inv), pack_bf16x2(o[i][2] * inv, o[i][3] * inv)};
    *reinterpret_cast<u32x2*>(p.out + (qrow * p.Hq + head) * D + 4 * lane + 4 * LANES * i) = w;
    hs += (bf16_lo(w.x) + bf16_hi(w.x)) + (bf16_lo(w.y) + bf16_hi(w.y));
  }
  if (p.out_sums) {
    if constexpr (LANES == 32) {
      hs = row_sum16(hs);
      hs += __shfl_xor(hs, 16, 32);
    } else {
#pragma unroll
      for (int s = LANES / 2; s; s >>= 1) hs += __shfl_xor(hs, s, LANES);
    }
    if (lane == 0) p.out_sums[(size_t)head * p.rows + qrow] = hs;
  }
}

}  // namespace t2i
