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
#include "ragged_attend.h"

namespace t2i {

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
      constexpr RaggedForm FORM = TREE ? RG_TREE : RG_PACKED;
      bool bad = false;
      const uint32_t odd = attend_item<FORM, FINE, false>(p, it, h, s_kv, lane, wave, 0, bad);
      if (it.kb0 >= it.kb1) return;
      if (lane == 0) s_odd[wave] = odd;
      lds_barrier();                                         // the buffers are free
      uint32_t any = 0;
#pragma unroll
      for (int w = 0; w < RG_WAVES; ++w) any |= s_odd[w];
      if (!__builtin_amdgcn_readfirstlane(any)) return;
      (void)attend_item<FORM, FINE, true>(p, it, h, s_kv, lane, wave, odd, bad);
      lds_barrier();
    };
    if (TREE || it.rows == 1) run(std::true_type{});
    else run(std::false_type{});
  }
}

// The parts of a tile joined: 32 lanes a (row, q head) pair, four dims each, eight pairs a
// workgroup; parts in their order, MERGE_AHEAD of them in flight, with a running maximum.  Bound
// by its loads' latency (16 trees of 26 nodes: 5.5-6 us, 9.6 with a wave a pair and two passes).
template <bool TREE>
__global__ __launch_bounds__(256) void ragged_merge_kernel(const RaggedAttnParams p) {
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
  join_parts<32>(p, h, at, first, second, step, parts, (size_t)row0 + t, head, lane);
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
