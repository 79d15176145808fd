// Attention of ragged batches over the contiguous KV cache for gfx950:
//
//   * t2i_packed_qk_rope_kv / t2i_tree_qk_rope_kv: per-head q/k RMSNorm + RoPE and the
//     cache write of packed prompt rows, or of the nodes of drafted trees;
//   * t2i_packed_attention: causal GQA attention of packed rows of many sequences, each
//     with its own length and its own earlier slots;
//   * t2i_tree_attention: GQA attention of a tree of drafted tokens: a node attends the
//     sequence's context, the nodes above it and itself;
//   * t2i_tree_commit: the greedy walk down the drafted trees and the accepted path's K/V
//     rows moved to the front, in every layer.
//
// Scores, softmax statistics and sums are fp32.  The softmax weights of prompt rows enter the P . V
// product as bf16, as in t2i_prefill_attention (quantized_qwen3/model.py:277), and each row's
// normaliser sums those rounded weights, so that a row of equal values comes back exact; trees and
// sequences of one row, which stand in for decode steps, multiply by weights of 16 bits.
#include <math.h>

#include <exception>
#include <type_traits>

#include "t2i_common.h"
#include "qk_prep.h"
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

// ============================================================================
// q/k RMSNorm + RoPE + KV-cache write of ragged rows
// ============================================================================
struct RaggedPrepParams {
  const uint16_t* qkv;      // [rows, (Hq + 2 Hkv) * D]
  const uint16_t* qn;
  const uint16_t* kn;
  const uint16_t* rope;     // [>= cap, D] cos even / sin odd
  uint16_t* q;              // [rows, Hq, D]
  uint16_t* kc;             // [cache rows, Hkv, cap, D]
  uint16_t* vc;
  const int32_t* row_pos;   // packed: position (and slot) of each row, its cache row
  const int32_t* row_cache;
  const int32_t* parents;   // trees: [B, N]; slot = context + node, position = context + depth
  const int32_t* ctx;
  const int32_t* counts;
  int N, n_cache, Hq, Hkv, cap, style;
  float eps;
};

// One workgroup (4 waves) per row, a head vector to a 16-lane row of a wave, as
// prefill_prep_kernel (same bits): RG_PREP_NB batches of 16 vectors in flight.  A row whose
// position, slot or cache row lies outside the cache writes nothing.  Bound by HBM where rows are
// many, every byte read and written once (4997 rows, 16 / 8 heads: 21 us, 3.9 TB/s), by the latency
// of a workgroup's own chain where they are few (416 nodes: 4.9 us for 6.8 MB).
constexpr int RG_PREP_NB = 2;

template <bool TREE>
__global__ __launch_bounds__(256) void ragged_prep_kernel(const RaggedPrepParams p) {
  constexpr int D = RG_D;
  const int row = blockIdx.x;
  const int lane = threadIdx.x & 63;
  int pos, dst_slot, crow;
  if (TREE) {
    crow = row / p.N;
    const int node = row - crow * p.N;
    const TreeSeq t = tree_seq(p.ctx, p.counts, crow, p.N, p.cap);
    if (!t.ok || node >= t.nodes) return;
    dst_slot = t.ctx + node;
    pos = t.ctx;
    const int parent = tree_parent(p.parents + (size_t)crow * p.N, p.N, lane);
    for (int up = node; (up = __builtin_amdgcn_readlane(parent, up)) >= 0;) ++pos;   // a parent stands before its node
  } else {
    pos = dst_slot = p.row_pos[row];
    crow = p.row_cache[row];
    if (pos < 0 || pos >= p.cap || crow < 0 || crow >= p.n_cache) return;
  }
  const int c = lane & 15;
  const int slot = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 4 + (lane >> 4);   // 0 .. 15
  const int nvec = p.Hq + 2 * p.Hkv;
  const uint16_t* src_row = p.qkv + (size_t)row * nvec * D;
  for (int base = 0; base < nvec; base += 16 * RG_PREP_NB) {
    u32x4 raw[RG_PREP_NB];
#pragma unroll
    for (int j = 0; j < RG_PREP_NB; ++j)
      raw[j] = prep_load(src_row + (size_t)min(base + 16 * j + slot, nvec - 1) * D, c, p.style);
    const u32x4 rp = *reinterpret_cast<const u32x4*>(p.rope + (size_t)pos * D + 8 * c);
    const u32x4 gqv = prep_load(p.qn, c, p.style);
    const u32x4 gkv = prep_load(p.kn, c, p.style);
#pragma unroll
    for (int j = 0; j < RG_PREP_NB; ++j) asm volatile("" : "+v"(raw[j]));   // every load before the first use
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < RG_PREP_NB; ++j) {
      const int vi = base + 16 * j + slot;     // uniform over the 16-lane row
      const bool isq = vi < p.Hq;
      const bool normed = vi < p.Hq + p.Hkv;   // q and k: RMSNorm + RoPE; v as is
      const u32x4 y = prep_vector(raw[j], rp, isq ? gqv : gkv, normed, p.style, p.eps);
      if (vi >= nvec) continue;
      uint16_t* dst;
      if (isq) dst = p.q + ((size_t)row * p.Hq + vi) * D;
      else if (normed) dst = p.kc + (((size_t)crow * p.Hkv + (vi - p.Hq)) * p.cap + dst_slot) * D;
      else dst = p.vc + (((size_t)crow * p.Hkv + (vi - p.Hq - p.Hkv)) * p.cap + dst_slot) * D;
      prep_store(dst, c, p.style, y);
    }
  }
}

// ============================================================================
// attention
// ============================================================================
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
};

// A piece of work: the tile of a sequence's (row, q head of a kv head) pairs from j0 on, over key
// blocks kb0 .. kb1 - 1; keys from kend on are seen by none of its rows.
struct RaggedItem {
  int row0, rows, start, crow, kb0, kb1, part, kend, j0, pairs;
};

// The even shares of a batch of trees: the key blocks of all sequences in a row, cut into `n`
// equal runs.  A workgroup takes a run for one tile of pairs of one kv head; the tiles of a
// sequence stand beside each other on one XCD and read the same K and V at the same time, so
// memory gives them once (8 trees of two tiles over 32k slots, before weights had 16 bits: 307 us
// one tile after the other, 260 side by side).  A sequence that is cut leaves a part in each of its
// runs: slot 2 bin where it is the run's first piece, 2 bin + 1 where it is the last of several.
struct TreeWalk {
  int n, total, b, blocks, kb;         // n: runs; the next piece starts at block kb of sequence b
  TreeSeq seq;

  // Key blocks of a sequence; one for zero rows (nodes that do not fit the cache).
  __device__ __forceinline__ int blocks_of(const TreeSeq& t) const {
    return t.nodes == 0 ? 0 : t.ok ? (t.ctx + t.nodes + RG_KEYS - 1) / RG_KEYS : 1;
  }
  // (32-bit products: the host keeps total below 2^23 and n at 2^9 or less, so that total n < 2^32)
  __device__ __forceinline__ int run_start(int i) const { return (int)((uint32_t)total * (uint32_t)i / (uint32_t)n); }
  // the run that holds block x
  __device__ __forceinline__ int run_of(int x) const { return (int)(((uint32_t)(x + 1) * (uint32_t)n - 1) / (uint32_t)total); }

  // Sums of 64 sequences' blocks at a time; false where there is no such run.
  __device__ __forceinline__ bool begin(const RaggedAttnParams& p, int bin, int lane, int& at, int& end) {
    const auto scan = [&](int base) {          // blocks of sequences base .. base + lane
      int v = base + lane < p.B ? blocks_of(tree_seq(p.ctx, p.counts, base + lane, p.N, p.cap)) : 0;
#pragma unroll
      for (int s = 1; s < 64; s <<= 1) {
        const int u = __shfl_up(v, s, 64);
        if (lane >= s) v += u;
      }
      return v;
    };
    total = 0;
    for (int base = 0; base < p.B; base += 64) total += __builtin_amdgcn_readlane(scan(base), 63);
    n = max(1, min(p.n_bins, total / 2));
    if (bin >= n || total == 0) return false;
    at = run_start(bin);
    end = run_start(bin + 1);
    int before = 0;
    for (int base = 0;; base += 64) {          // ends: at < total
      const int v = scan(base), sum = __builtin_amdgcn_readlane(v, 63);
      if (before + sum > at) {
        const int first = __builtin_ctzll(__ballot(before + v > at));
        b = base + first;
        if (first) before += __builtin_amdgcn_readlane(v, first - 1);
        break;
      }
      before += sum;
    }
    seq = tree_seq(p.ctx, p.counts, b, p.N, p.cap);
    blocks = blocks_of(seq);
    kb = at - before;
    return true;
  }

  // The next piece of the run for a tile, and where it ends.
  __device__ __forceinline__ int next(const RaggedAttnParams& p, int bin, int tile, int h, int at0, int at, int end, RaggedItem& it) {
    while (kb == blocks) {                     // ends: blocks are left
      seq = tree_seq(p.ctx, p.counts, ++b, p.N, p.cap);
      blocks = blocks_of(seq);
      kb = 0;
    }
    const int take = min(blocks - kb, end - at);
    const bool whole = take == blocks;
    it.row0 = b * p.N;
    it.rows = seq.nodes;
    it.start = seq.ctx;
    it.crow = b;
    it.j0 = tile * RG_ROWS;
    it.pairs = seq.nodes * p.G;
    it.kend = seq.ctx + seq.nodes;
    it.kb0 = kb;
    it.kb1 = seq.ok ? kb + take : kb;
    it.part = whole ? -1 : (2 * bin + (at != at0)) * p.tiles + tile;
    if (h == 0 && tile == 0 && threadIdx.x == 0 && kb + take == blocks) {   // the sequence's last piece: what its merge reads
      const int first = at - kb, run = run_of(first);
      p.cuts[b] = int2{whole ? -1 : 2 * run + (run_start(run) != first), bin};
    }
    kb += take;
    return at + take;
  }
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
template <bool TREE, bool FINE, bool MASKED>
__device__ __forceinline__ uint32_t attend_item(const RaggedAttnParams& p, const RaggedItem& it, int h, uint16_t* s_kv, int lane,
                                                int wave, uint32_t only) {
  constexpr int D = RG_D;
  constexpr int WKEYS = RG_KEYS / RG_WAVES;    // keys of a block that a wave loads
  const int c = lane & 31, h2 = lane >> 5;

  // ---- K / V staging: a wave's instruction moves 4 keys (1 KB); 4 each of K and V a block ----
  const size_t cache_base = ((size_t)it.crow * p.Hkv + h) * (size_t)p.cap * D;
  const int srow = lane >> 4;                              // key within the instruction's four
  const int place = lane & 15;                             // where the lane's 16 bytes go in the key's row
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(rg_lds_address(s_kv) + wave * WKEYS * D * 2);
  constexpr int LOADS = WKEYS / 4;                         // instructions of a wave for K, and for V
  uint32_t kat[LOADS], vat[LOADS];                         // what the lane loads: byte in the block, less 1024 i
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    kat[i] = (wave * WKEYS + srow) * (D * 2) + 16 * (place ^ ((wave * WKEYS + 4 * i + srow) & 15));
    vat[i] = (wave * WKEYS + srow) * (D * 2) + 16 * (place ^ (4 * srow));
  }
  const i32x4 krsrc = keys_rsrc(p.kc + cache_base), vrsrc = keys_rsrc(p.vc + cache_base);
  // K and V block kb into its buffer
  auto stage = [&](int kb) __attribute__((always_inline)) {
    const uint32_t lds = lds0 + ((kb - it.kb0) & 1) * (4 * RG_KEYS * D);
    if ((kb + 1) * RG_KEYS <= it.kend) {
      const uint32_t at = (uint32_t)kb * (RG_KEYS * D * 2);
      if (it.pairs <= RG_ROWS) {                            // the sequence's only tile: its keys are read once
        lds_load_keys<true>(krsrc, kat, at, lds);
        lds_load_keys<true>(vrsrc, vat, at, lds + 2 * RG_KEYS * D);
      } else {
        lds_load_keys<false>(krsrc, kat, at, lds);
        lds_load_keys<false>(vrsrc, vat, at, lds + 2 * RG_KEYS * D);
      }
    } else {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int at = wave * WKEYS + 4 * i + srow;
        const uint32_t key = (uint32_t)min(kb * RG_KEYS + at, it.kend - 1) * (D * 2);
        lds_load16(krsrc, key + 16 * (place ^ (at & 15)), lds + i * 4 * D * 2);
        lds_load16(vrsrc, key + 16 * (place ^ (4 * srow)), lds + 2 * RG_KEYS * D + i * 4 * D * 2);
      }
    }
  };
  if (it.kb0 < it.kb1) stage(it.kb0);

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
  if (TREE && it.kb1 * RG_KEYS > it.start && it.kb0 < it.kb1) {
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

  for (int kb = it.kb0; kb < it.kb1; ++kb) {
    loads_done_barrier();                                  // this block is here, the buffer of the one before it free
    if (kb + 1 < it.kb1) stage(kb + 1);
    if (!wave_on || kb * RG_KEYS >= wave_end) continue;
    const uint16_t* const bk = s_kv + ((kb - it.kb0) & 1) * (2 * RG_KEYS * D);
    const uint16_t* const bv = bk + RG_KEYS * D;
    // ---- S^T = K Q^T ----
    f32x16 s[2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
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
    if (kb * RG_KEYS + RG_KEYS > mask_from) {
      if (TREE) {
        const int rel = kb * RG_KEYS - it.start;           // node of the block's first key (negative: a context slot)
        const unsigned long long w = (unsigned long long)seen_hi << 32 | seen_lo;
        unsigned long long bm = rel >= 64 ? 0ull : rel >= 0 ? w >> rel : (w << -rel) | ((1ull << -rel) - 1);
        bm >>= 4 * h2;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (!((uint32_t)(bm >> (32 * n)) & (1u << (8 * (i / 4) + i % 4)))) s[n][i] = -INFINITY;
      } else {
        const int rel = qpos - kb * RG_KEYS - 4 * h2;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (32 * n + 8 * (i / 4) + i % 4 > rel) s[n][i] = -INFINITY;
      }
    }
    // ---- online softmax (log2 domain) ----
    float mx = fmaxf(s[0][0], s[1][0]);
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, fmaxf(s[0][i], s[1][i]));
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
      if (kb * RG_KEYS + RG_KEYS > mask_from) {
        bool odd = false;
#pragma unroll 4
        for (int i = 0; i < RG_KEYS / 4; ++i) {
          const u32x4 x = *reinterpret_cast<const u32x4*>(bv + 4 * i * D + 8 * lane);
#pragma unroll
          for (int e = 0; e < 4; ++e) odd |= finite_or_zero(x[e]) != x[e];
        }
        if (__any(odd)) {
          const uint32_t unseen = __float_as_uint(-1.0f);  // no weight
#pragma unroll
          for (int n = 0; n < 2; ++n)
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
    uint32_t pw[2][8], pr[2][8];                           // bf16 weights, two keys a word; what their rounding left
#pragma unroll
    for (int n = 0; n < 2; ++n)
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
    for (int u = 0; u < 4; ++u) {
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

// A workgroup takes a bin's items for one kv head, one after the other.
template <bool TREE>
__global__ __launch_bounds__(64 * RG_WAVES, 2) void ragged_attention_kernel(const RaggedAttnParams p) {
  extern __shared__ __align__(256) uint16_t s_kv[];   // [buffer][K, V][key][dim]
  __shared__ uint32_t s_odd[RG_WAVES];                     // an item's pairs whose sums are not finite

  const int h = blockIdx.x % p.Hkv;
  const int tile = TREE ? blockIdx.x / p.Hkv % p.tiles : 0;
  const int bin = blockIdx.x / p.Hkv / (TREE ? p.tiles : 1);
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  int at = 0, end = 0;          // packed: items; trees: key blocks of the whole batch
  TreeWalk walk;
  if (TREE) {
    if (!walk.begin(p, bin, lane, at, end)) return;
  } else {
    at = max(p.bins[bin], 0);
    end = min(p.bins[bin + 1], p.n_items);
  }
  const int at0 = at;
  for (; at < end;) {
    RaggedItem it;
    if (TREE) {
      at = walk.next(p, bin, tile, h, at0, at, end, it);
      if (it.j0 >= it.pairs) continue;                       // this sequence has fewer tiles
    } else {
      const int32_t* w = p.items + (size_t)at * RG_ITEM;
      ++at;
      it.row0 = w[0]; it.rows = w[1]; it.start = w[2]; it.crow = w[3];
      it.j0 = w[4]; it.kb0 = w[5]; it.kb1 = w[6]; it.part = w[7];
      it.pairs = (int)((uint32_t)it.rows * (uint32_t)p.G);   // checked below
      // a table that does not fit the tensors is not followed
      if (it.row0 < 0 || it.rows < 1 || it.row0 + (long long)it.rows > p.rows || it.start < 0 ||
          it.start > p.cap - it.rows || it.crow < 0 || it.crow >= p.n_cache || it.j0 < 0 ||
          (long long)it.rows * p.G > 0x7FFFFFFF - RG_ROWS || it.j0 >= it.pairs || it.part >= p.n_parts)
        continue;
      it.kend = it.start + (min(it.j0 + RG_ROWS, it.pairs) - 1) / p.G + 1;
      it.kb0 = max(it.kb0, 0);
      it.kb1 = min(it.kb1, (it.kend + RG_KEYS - 1) / RG_KEYS);
    }

    const auto run = [&](auto fine) __attribute__((always_inline)) {
      constexpr bool FINE = decltype(fine)::value;
      const uint32_t odd = attend_item<TREE, FINE, false>(p, it, h, s_kv, lane, wave, 0);
      if (it.kb0 >= it.kb1) return;
      if (lane == 0) s_odd[wave] = odd;
      lds_barrier();                                         // the buffers are free
      uint32_t any = 0;
#pragma unroll
      for (int w = 0; w < RG_WAVES; ++w) any |= s_odd[w];
      if (!__builtin_amdgcn_readfirstlane(any)) return;
      (void)attend_item<TREE, FINE, true>(p, it, h, s_kv, lane, wave, odd);
      lds_barrier();
    };
    if (TREE || it.rows == 1) run(std::true_type{});
    else run(std::false_type{});
  }
}

// The parts of a tile joined: 32 lanes a (row, q head) pair, four dims each, eight pairs a
// workgroup; parts in their order, MERGE_AHEAD of them in flight, with a running maximum.  Bound
// by its loads' latency (16 trees of 26 nodes: 5.5-6 us, 9.6 with a wave a pair and two passes).
constexpr int MERGE_AHEAD = 4;
constexpr int MERGE_PAIRS = t2i_host::RG_MERGE;

template <bool TREE>
__global__ __launch_bounds__(256) void ragged_merge_kernel(const RaggedAttnParams p) {
  constexpr int D = RG_D;
  const int lane = threadIdx.x & 31;
  const int h = blockIdx.x % p.Hkv;
  const int idx = blockIdx.x / p.Hkv;
  int row0, rows, first, parts, second, step, j0, at = threadIdx.x >> 5;   // parts: first, then second, second + step, ...
  if (TREE) {
    const int groups = p.part_rows / MERGE_PAIRS, group = idx % groups;
    const int tile = idx / groups % p.tiles, b = idx / groups / p.tiles;
    row0 = b * p.N;
    rows = tree_seq(p.ctx, p.counts, b, p.N, p.cap).nodes;
    at += group * MERGE_PAIRS;
    j0 = tile * RG_ROWS;
    if (j0 + group * MERGE_PAIRS >= rows * p.G) return;   // nothing was written for it
    const int2 w = p.cuts[b];
    if (w.x < 0) return;                       // one piece: its rows are written
    first = w.x * p.tiles + tile;
    parts = w.y - w.x / 2 + 1;
    second = (w.x / 2 + 1) * 2 * p.tiles + tile;
    step = 2 * p.tiles;
  } else {
    const int32_t* w = p.items + (size_t)idx * RG_ITEM;
    row0 = w[0]; rows = w[1]; j0 = w[2]; first = w[3]; parts = w[4];
    at += w[5];
    second = first + 1;
    step = 1;
    if (row0 < 0 || rows < 1 || row0 + (long long)rows > p.rows || j0 < 0 || j0 > 0x7FFFFFFF - p.part_rows || first < 0 ||
        parts < 1 || first > p.n_parts - parts || w[5] < 0 || w[5] > p.part_rows - MERGE_PAIRS)
      return;
  }
  const int j = j0 + at;
  if (j >= (long long)rows * p.G) return;      // 32 lanes together
  const int t = j / p.G;
  const int head = h * p.G + (j - t * p.G);
  float M = -INFINITY, l = 0.0f;
  f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < parts; s0 += MERGE_AHEAD) {
    float2 ml[MERGE_AHEAD];
    f32x4 v[MERGE_AHEAD];
#pragma unroll
    for (int u = 0; u < MERGE_AHEAD; ++u) {
      const int s = min(s0 + u, parts - 1), part = s == 0 ? first : second + (s - 1) * step;
      const size_t st = ((size_t)part * p.Hkv + h) * p.part_rows + at;
      ml[u] = p.part_ml[st];
      v[u] = *reinterpret_cast<const f32x4*>(p.part_o + st * D + 4 * lane);
    }
    float mn = M;
#pragma unroll
    for (int u = 0; u < MERGE_AHEAD; ++u) mn = fmaxf(mn, ml[u].x);
    const float f = state_weight(M, mn);
    l *= f;
    o *= f;
    M = mn;
#pragma unroll
    for (int u = 0; u < MERGE_AHEAD; ++u) {
      const bool some = s0 + u < parts && ml[u].x > -INFINITY;   // else nothing was attended, nor written
      const float g = exp2_fast(ml[u].x - M);
      l += some ? g * ml[u].y : 0.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += some ? g * v[u][e] : 0.0f;
    }
  }
  const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
  const u32x2 w = u32x2{pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv)};
  const size_t qrow = (size_t)row0 + t;
  *reinterpret_cast<u32x2*>(p.out + (qrow * p.Hq + head) * D + 4 * lane) = w;
  if (p.out_sums) {
    float hs = row_sum16((bf16_lo(w.x) + bf16_hi(w.x)) + (bf16_lo(w.y) + bf16_hi(w.y)));
    hs += __shfl_xor(hs, 16, 32);
    if (lane == 0) p.out_sums[(size_t)head * p.rows + qrow] = hs;
  }
}

// ============================================================================
// the accepted path of a drafted tree
// ============================================================================
struct TreeCommitParams {
  const int32_t* tokens;    // [B, N]
  const int32_t* parents;
  const int32_t* picks;
  const int32_t* ctx;       // [B]
  const int32_t* counts;    // [B] or NULL
  uint16_t* kc;             // [layers, B, Hkv, cap, D]
  uint16_t* vc;
  int32_t* path;            // [B, N]
  int32_t* n_path;          // [B]
  int32_t* next;
  int32_t* ctx_out;
  int B, N, layers, Hkv, cap;
};

// A wave per (layer, sequence, kv head); lane i holds node i.  Every wave walks the tree itself
// (a ballot a step; the walk costs less than a hand-over), then moves its head's rows: four
// slots at a time, 16 lanes of 16 bytes each.  The path's nodes ascend, so entry e comes from a
// slot at or behind e: a group's writes never reach a slot that a later group reads.  Bound by the
// latency of its chain (nodes, walk, rows): 28 layers x 8 heads, 8 nodes 3.0 us, 32 sequences of 26
// nodes 6.6-6.8 us.
__global__ __launch_bounds__(256) void tree_commit_kernel(const TreeCommitParams p) {
  constexpr int D = RG_D;
  const int lane = threadIdx.x & 63;
  const long long id = (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (id >= (long long)p.layers * p.B * p.Hkv) return;
  const int b = (int)(id / p.Hkv % p.B);
  const TreeSeq t = tree_seq(p.ctx, p.counts, b, p.N, p.cap);
  const int at = b * p.N + min(lane, p.N - 1);
  const int token = p.tokens[at], pick = p.picks[at];
  const int parent = tree_parent(p.parents + (size_t)b * p.N, p.N, lane);
  int mine = -1, n = 0, cur = -1;
  if (t.ok && t.nodes > 0) {
    cur = 0;
    for (;;) {                                             // at most N steps: cur ascends
      if (lane == n) mine = cur;
      ++n;
      const int want = __builtin_amdgcn_readlane(pick, cur);
      const unsigned long long right = __ballot(lane < t.nodes && parent == cur && token == want);
      if (!right) break;
      cur = __builtin_ctzll(right);
    }
  }
  const int next = __builtin_amdgcn_readlane(pick, max(cur, 0));
  if (id < (long long)p.B * p.Hkv && id % p.Hkv == 0) {    // layer 0, head 0: the record
    if (lane < p.N) p.path[b * p.N + lane] = mine;
    if (lane == 0) {
      p.n_path[b] = n;
      p.next[b] = n ? next : -1;
      p.ctx_out[b] = t.ctx + n;
    }
  }
  const size_t base = (size_t)id * p.cap * D + (size_t)t.ctx * D + (lane & 15) * 8;
  for (int e0 = 0; e0 < n; e0 += 4) {
    const int e = e0 + (lane >> 4);
    const int from = __shfl(mine, e, 64);                  // e < 64
    if (e < n && from != e) {
      const u32x4 k = *reinterpret_cast<const u32x4*>(p.kc + base + (size_t)from * D);
      const u32x4 v = *reinterpret_cast<const u32x4*>(p.vc + base + (size_t)from * D);
      *reinterpret_cast<u32x4*>(p.kc + base + (size_t)e * D) = k;
      *reinterpret_cast<u32x4*>(p.vc + base + (size_t)e * D) = v;
    }
  }
}

}  // namespace t2i

// ============================================================================
// host side
// ============================================================================
using t2i_host::aligned16;
using t2i_host::fail;

namespace {

bool aligned4(const void* p) { return ((uintptr_t)p & 3u) == 0; }

int check_heads(int32_t Hq, int32_t Hkv, int32_t D, int32_t cap) {
  if (D != t2i::RG_D) return fail(T2I_ERR_SHAPE, "head_dim %d unsupported (only 128)", D);
  if (Hkv < 1 || Hq < Hkv || Hq % Hkv) return fail(T2I_ERR_SHAPE, "Hq=%d Hkv=%d invalid", Hq, Hkv);
  if (Hq > 1024) return fail(T2I_ERR_SHAPE, "Hq=%d exceeds 1024", Hq);
  // a kv head's rows of the cache are addressed with 32-bit byte offsets
  if (cap < 1 || cap > (1 << 23)) return fail(T2I_ERR_SHAPE, "ctx_cap=%d must be 1 to 8388608", cap);
  return T2I_OK;
}

// Pairs and parts stay below 2^31, the threads of a launch below 2^32.
bool too_many(long long n) { return n > 0x7FFFFFFFLL; }
bool past_grid(long long groups, int threads) { return groups > 0xFFFFFFFFLL / threads; }

size_t part_bytes(long long parts, int32_t Hkv, int32_t rows) {
  return (size_t)parts * Hkv * rows * (t2i::RG_D * sizeof(float) + sizeof(float2));
}

// The workspace's parts: outputs first, then the (max, sum) pairs; returns what follows them.
void* set_parts(t2i::RaggedAttnParams& p, void* ws, long long parts, int32_t rows) {
  p.part_rows = rows;
  p.part_o = reinterpret_cast<float*>(ws);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + (size_t)parts * p.Hkv * rows * t2i::RG_D);
  return p.part_ml + (size_t)parts * p.Hkv * rows;
}

constexpr int LDS_BYTES = 2 * 2 * t2i::RG_KEYS * t2i::RG_D * 2;   // two buffers of K and V

template <bool TREE>
int launch_attention(const t2i::RaggedAttnParams& p, long long groups, hipStream_t s) {
  hipLaunchKernelGGL(t2i::ragged_attention_kernel<TREE>, dim3(groups), dim3(64 * t2i::RG_WAVES), LDS_BYTES, s, p);
  return t2i_host::hip_status(hipGetLastError(), "ragged attention launch");
}

// A tree call's launch: tiles of a sequence, workgroups of a kv head, rows of a part's tile.
struct TreePlan {
  int tiles, bins, rows;
  size_t bytes;
};
TreePlan tree_plan(int32_t B, int32_t N, int32_t Hq, int32_t Hkv, int32_t cap) {
  TreePlan t;
  const int pairs = N * (Hq / Hkv);
  t.tiles = (pairs + t2i_host::RG_ROWS - 1) / t2i_host::RG_ROWS;
  t.bins = t2i_host::tree_bins(B, t.tiles * Hkv, cap);
  t.rows = std::min(t2i_host::RG_ROWS, (pairs + 31) / 32 * 32);
  t.bytes = part_bytes(2LL * t.bins * t.tiles, Hkv, t.rows) + (size_t)B * sizeof(int2);
  return t;
}

int check_prep(const void* qkv, const void* qn, const void* kn, const void* rope, const void* q, const void* kc,
               const void* vc, float eps, int32_t style) {
  if (!qkv || !qn || !kn || !rope || !q || !kc || !vc) return fail(T2I_ERR_NULL, "ragged prep pointers must not be NULL");
  if (!aligned16(qkv) || !aligned16(qn) || !aligned16(kn) || !aligned16(rope) || !aligned16(q) || !aligned16(kc) ||
      !aligned16(vc))
    return fail(T2I_ERR_ALIGN, "ragged prep tensors must be 16-byte aligned");
  if (style != 0 && style != 1) return fail(T2I_ERR_VALUE, "rope_style must be 0 or 1");
  if (!(eps > 0.0f)) return fail(T2I_ERR_VALUE, "eps must be positive");
  return T2I_OK;
}

int check_tree(const int32_t* parents, const int32_t* ctx, const int32_t* counts, int32_t B, int32_t N, int32_t cap) {
  if (!parents || !ctx) return fail(T2I_ERR_NULL, "parents and context_lens must not be NULL");
  if (!aligned4(parents) || !aligned4(ctx) || !aligned4(counts))
    return fail(T2I_ERR_ALIGN, "parents, context_lens and node_counts must be 4-byte aligned");
  if (B < 1 || N < 1 || N > t2i::TREE_NODES || N > cap)
    return fail(T2I_ERR_SHAPE, "B=%d N=%d invalid (1 to %d nodes, at most the cache's %d slots)", B, N, t2i::TREE_NODES, cap);
  return T2I_OK;
}

}  // namespace

extern "C" int t2i_packed_plan(const int32_t* lengths, const int32_t* starts, const int32_t* cache_rows, int32_t n,
                               int32_t Hq, int32_t Hkv, int32_t n_cache_rows, int32_t ctx_cap, int32_t* table,
                               int64_t table_words, int64_t* sizes) {
  if (!lengths || !starts || !sizes) return fail(T2I_ERR_NULL, "lengths, starts and sizes must not be NULL");
  if (int rc = check_heads(Hq, Hkv, t2i::RG_D, ctx_cap)) return rc;
  if (n < 1 || n_cache_rows < 1 || n > n_cache_rows)
    return fail(T2I_ERR_SHAPE, "%d sequences over %d cache rows invalid", n, n_cache_rows);
  try {
    std::vector<char> used(n_cache_rows, 0);
    long long rows = 0;
    for (int i = 0; i < n; ++i) {
      const int crow = cache_rows ? cache_rows[i] : i;
      if (lengths[i] < 0 || starts[i] < 0 || (long long)starts[i] + lengths[i] > ctx_cap)
        return fail(T2I_ERR_VALUE, "sequence %d: rows %d from slot %d exceed the cache (%d)", i, lengths[i], starts[i], ctx_cap);
      if (crow < 0 || crow >= n_cache_rows) return fail(T2I_ERR_VALUE, "sequence %d: cache row %d out of range", i, crow);
      if (used[crow]) return fail(T2I_ERR_VALUE, "sequence %d: cache row %d is another sequence's", i, crow);
      used[crow] = 1;
      rows += lengths[i];
    }
    if (too_many(rows * Hq)) return fail(T2I_ERR_SHAPE, "%lld packed rows are too many", rows);
    const t2i_host::PackedTable t = t2i_host::packed_table(lengths, starts, cache_rows, n, Hq / Hkv, Hkv);
    sizes[0] = (int64_t)t.row_pos.size();
    sizes[1] = (int64_t)t.items.size() / t2i::RG_ITEM;
    sizes[2] = (int64_t)t.merges.size() / t2i::RG_ITEM;
    sizes[3] = t.n_parts;
    sizes[4] = (int64_t)t.bins.size() - 1;
    sizes[5] = (int64_t)(2 * t.row_pos.size() + t.items.size() + t.merges.size() + t.bins.size());
    if (!table) return T2I_OK;
    if (table_words < sizes[5]) return fail(T2I_ERR_WORKSPACE, "the table holds %lld words, %lld needed", (long long)table_words, (long long)sizes[5]);
    for (const auto* v : {&t.row_pos, &t.row_cache, &t.items, &t.merges, &t.bins}) table = std::copy(v->begin(), v->end(), table);
    return T2I_OK;
  } catch (const std::exception& e) {
    return fail(T2I_ERR_WORKSPACE, "host memory for the plan: %s", e.what());
  }
}

extern "C" int t2i_packed_qk_rope_kv(const uint16_t* qkv, int32_t rows, const int32_t* row_pos, const int32_t* row_cache,
                                     int32_t n_cache_rows, int32_t Hq, int32_t Hkv, int32_t D, const uint16_t* q_norm,
                                     const uint16_t* k_norm, float eps, const uint16_t* rope, int32_t rope_style,
                                     uint16_t* q_out, uint16_t* k_cache, uint16_t* v_cache, int32_t ctx_cap, void* stream) {
  if (int rc = check_prep(qkv, q_norm, k_norm, rope, q_out, k_cache, v_cache, eps, rope_style)) return rc;
  if (!row_pos || !row_cache) return fail(T2I_ERR_NULL, "row_pos and row_cache must not be NULL");
  if (!aligned4(row_pos) || !aligned4(row_cache)) return fail(T2I_ERR_ALIGN, "row_pos and row_cache must be 4-byte aligned");
  if (int rc = check_heads(Hq, Hkv, D, ctx_cap)) return rc;
  if (rows < 1 || n_cache_rows < 1 || past_grid(rows, 256))
    return fail(T2I_ERR_SHAPE, "rows=%d cache rows=%d invalid", rows, n_cache_rows);
  t2i::RaggedPrepParams p{};
  p.qkv = qkv; p.qn = q_norm; p.kn = k_norm; p.rope = rope; p.q = q_out; p.kc = k_cache; p.vc = v_cache;
  p.row_pos = row_pos; p.row_cache = row_cache; p.n_cache = n_cache_rows;
  p.Hq = Hq; p.Hkv = Hkv; p.cap = ctx_cap; p.style = rope_style; p.eps = eps;
  hipLaunchKernelGGL(t2i::ragged_prep_kernel<false>, dim3(rows), dim3(256), 0, reinterpret_cast<hipStream_t>(stream), p);
  return t2i_host::hip_status(hipGetLastError(), "packed prep launch");
}

extern "C" size_t t2i_packed_attention_workspace_bytes(int64_t n_parts, int32_t Hkv) {
  return n_parts < 1 || Hkv < 1 || too_many(n_parts) ? 0 : part_bytes(n_parts, Hkv, t2i_host::RG_ROWS);
}

extern "C" int t2i_packed_attention(const uint16_t* q, int32_t rows, const int32_t* items, int32_t n_items,
                                    const int32_t* merges, int32_t n_merges, int32_t n_parts, const int32_t* bins,
                                    int32_t n_bins, int32_t Hq, int32_t Hkv, int32_t D, const uint16_t* k_cache,
                                    const uint16_t* v_cache, int32_t n_cache_rows, int32_t ctx_cap, uint16_t* out,
                                    float* out_sums, void* workspace, size_t workspace_bytes, void* stream) {
  if (!q || !items || !bins || !k_cache || !v_cache || !out) return fail(T2I_ERR_NULL, "packed attention pointers must not be NULL");
  if (int rc = check_heads(Hq, Hkv, D, ctx_cap)) return rc;
  if (rows < 1 || n_cache_rows < 1 || n_items < 1 || n_bins < 1 || n_merges < 0 || n_parts < 0 ||
      (n_parts > 0 && (n_merges < 1 || !merges)))
    return fail(T2I_ERR_SHAPE, "rows=%d items=%d bins=%d merges=%d parts=%d invalid", rows, n_items, n_bins, n_merges, n_parts);
  if (past_grid((long long)n_bins * Hkv, 256) || past_grid((long long)n_merges * Hkv, 256))
    return fail(T2I_ERR_SHAPE, "%d bins of %d kv heads exceed the grid", n_bins, Hkv);
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(out))
    return fail(T2I_ERR_ALIGN, "packed attention tensors must be 16-byte aligned");
  if (!aligned4(items) || !aligned4(merges) || !aligned4(bins) || !aligned4(out_sums))
    return fail(T2I_ERR_ALIGN, "tables and out_sums must be 4-byte aligned");
  const size_t need = part_bytes(n_parts, Hkv, t2i_host::RG_ROWS);
  if (need && (!workspace || workspace_bytes < need)) return fail(T2I_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : 0, need);
  if (need && !aligned16(workspace)) return fail(T2I_ERR_ALIGN, "the workspace must be 16-byte aligned");
  t2i::RaggedAttnParams p{};
  p.q = q; p.kc = k_cache; p.vc = v_cache; p.out = out; p.out_sums = out_sums; p.items = items; p.bins = bins;
  p.rows = rows; p.n_cache = n_cache_rows; p.n_items = n_items; p.n_bins = n_bins; p.n_parts = n_parts;
  p.Hq = Hq; p.Hkv = Hkv; p.G = Hq / Hkv; p.cap = ctx_cap;
  p.scale_log2 = (float)(1.4426950408889634 / sqrt((double)D));
  if (need) set_parts(p, workspace, n_parts, t2i_host::RG_ROWS);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (int rc = launch_attention<false>(p, (long long)n_bins * Hkv, s)) return rc;
  if (!need) return T2I_OK;
  p.items = merges;
  hipLaunchKernelGGL(t2i::ragged_merge_kernel<false>, dim3(n_merges * Hkv), dim3(256), 0, s, p);
  return t2i_host::hip_status(hipGetLastError(), "packed attention merge launch");
}

extern "C" int t2i_tree_qk_rope_kv(const uint16_t* qkv, const int32_t* parents, const int32_t* context_lens,
                                   const int32_t* node_counts, int32_t B, int32_t N, int32_t Hq, int32_t Hkv, int32_t D,
                                   const uint16_t* q_norm, const uint16_t* k_norm, float eps, const uint16_t* rope,
                                   int32_t rope_style, uint16_t* q_out, uint16_t* k_cache, uint16_t* v_cache,
                                   int32_t ctx_cap, void* stream) {
  if (int rc = check_prep(qkv, q_norm, k_norm, rope, q_out, k_cache, v_cache, eps, rope_style)) return rc;
  if (int rc = check_heads(Hq, Hkv, D, ctx_cap)) return rc;
  if (int rc = check_tree(parents, context_lens, node_counts, B, N, ctx_cap)) return rc;
  if (past_grid((long long)B * N, 256)) return fail(T2I_ERR_SHAPE, "B=%d N=%d exceed the grid", B, N);
  t2i::RaggedPrepParams p{};
  p.qkv = qkv; p.qn = q_norm; p.kn = k_norm; p.rope = rope; p.q = q_out; p.kc = k_cache; p.vc = v_cache;
  p.parents = parents; p.ctx = context_lens; p.counts = node_counts; p.N = N; p.n_cache = B;
  p.Hq = Hq; p.Hkv = Hkv; p.cap = ctx_cap; p.style = rope_style; p.eps = eps;
  hipLaunchKernelGGL(t2i::ragged_prep_kernel<true>, dim3(B * N), dim3(256), 0, reinterpret_cast<hipStream_t>(stream), p);
  return t2i_host::hip_status(hipGetLastError(), "tree prep launch");
}

extern "C" size_t t2i_tree_attention_workspace_bytes(int32_t B, int32_t N, int32_t Hq, int32_t Hkv, int32_t ctx_cap) {
  if (B < 1 || N < 1 || N > t2i::TREE_NODES || Hkv < 1 || Hq < Hkv || Hq % Hkv || Hq > 1024 || ctx_cap < N) return 0;
  return tree_plan(B, N, Hq, Hkv, ctx_cap).bytes;
}

extern "C" int t2i_tree_attention(const uint16_t* q, const int32_t* parents, const int32_t* context_lens,
                                  const int32_t* node_counts, int32_t B, int32_t N, int32_t Hq, int32_t Hkv, int32_t D,
                                  const uint16_t* k_cache, const uint16_t* v_cache, int32_t ctx_cap, uint16_t* out,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  if (!q || !k_cache || !v_cache || !out) return fail(T2I_ERR_NULL, "tree attention pointers must not be NULL");
  if (int rc = check_heads(Hq, Hkv, D, ctx_cap)) return rc;
  if (int rc = check_tree(parents, context_lens, node_counts, B, N, ctx_cap)) return rc;
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(out))
    return fail(T2I_ERR_ALIGN, "tree attention tensors must be 16-byte aligned");
  t2i::RaggedAttnParams p{};
  p.q = q; p.kc = k_cache; p.vc = v_cache; p.out = out; p.parents = parents; p.ctx = context_lens; p.counts = node_counts;
  const TreePlan t = tree_plan(B, N, Hq, Hkv, ctx_cap);
  p.rows = (long long)B * N; p.n_cache = B; p.Hq = Hq; p.Hkv = Hkv; p.G = Hq / Hkv; p.cap = ctx_cap; p.B = B; p.N = N;
  p.tiles = t.tiles;
  p.n_bins = t.bins;
  p.scale_log2 = (float)(1.4426950408889634 / sqrt((double)D));
  if (past_grid((long long)B * t.tiles * Hkv * (t.rows / t2i::MERGE_PAIRS), 256) || too_many((long long)B * N) ||
      (long long)B * ((ctx_cap + t2i::RG_KEYS - 1) / t2i::RG_KEYS) >= 1 << 23)
    return fail(T2I_ERR_SHAPE, "B=%d N=%d Hkv=%d over %d slots are too many", B, N, Hkv, ctx_cap);
  if (!workspace || workspace_bytes < t.bytes) return fail(T2I_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : 0, t.bytes);
  if (!aligned16(workspace)) return fail(T2I_ERR_ALIGN, "the workspace must be 16-byte aligned");
  p.cuts = reinterpret_cast<int2*>(set_parts(p, workspace, 2LL * t.bins * t.tiles, t.rows));
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (int rc = launch_attention<true>(p, (long long)t.bins * t.tiles * Hkv, s)) return rc;
  hipLaunchKernelGGL(t2i::ragged_merge_kernel<true>, dim3(B * t.tiles * Hkv * (t.rows / t2i::MERGE_PAIRS)), dim3(256), 0, s, p);
  return t2i_host::hip_status(hipGetLastError(), "tree attention merge launch");
}

extern "C" int t2i_tree_commit(const int32_t* tokens, const int32_t* parents, const int32_t* picks,
                               const int32_t* context_lens, const int32_t* node_counts, int32_t layers, int32_t B,
                               int32_t N, int32_t Hkv, int32_t D, uint16_t* k_cache, uint16_t* v_cache, int32_t ctx_cap,
                               int32_t* path, int32_t* path_counts, int32_t* next_tokens, int32_t* context_out,
                               void* stream) {
  if (!tokens || !picks || !k_cache || !v_cache || !path || !path_counts || !next_tokens || !context_out)
    return fail(T2I_ERR_NULL, "tree commit pointers must not be NULL");
  if (int rc = check_heads(Hkv, Hkv, D, ctx_cap)) return rc;
  if (int rc = check_tree(parents, context_lens, node_counts, B, N, ctx_cap)) return rc;
  if (layers < 1 || past_grid((long long)layers * B * Hkv, 64)) return fail(T2I_ERR_SHAPE, "layers=%d invalid", layers);
  if (!aligned4(tokens) || !aligned4(picks) || !aligned4(path) || !aligned4(path_counts) || !aligned4(next_tokens) || !aligned4(context_out))
    return fail(T2I_ERR_ALIGN, "token and count arrays must be 4-byte aligned");
  if (!aligned16(k_cache) || !aligned16(v_cache)) return fail(T2I_ERR_ALIGN, "caches must be 16-byte aligned");
  if (context_out == context_lens) return fail(T2I_ERR_VALUE, "context_out must not be context_lens (every wave reads it)");
  t2i::TreeCommitParams p{};
  p.tokens = tokens; p.parents = parents; p.picks = picks; p.ctx = context_lens; p.counts = node_counts;
  p.kc = k_cache; p.vc = v_cache; p.path = path; p.n_path = path_counts; p.next = next_tokens; p.ctx_out = context_out;
  p.B = B; p.N = N; p.layers = layers; p.Hkv = Hkv; p.cap = ctx_cap;
  const long long waves = (long long)layers * B * Hkv;
  hipLaunchKernelGGL(t2i::tree_commit_kernel, dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, reinterpret_cast<hipStream_t>(stream), p);
  return t2i_host::hip_status(hipGetLastError(), "tree commit launch");
}
