// Low-rank adapters of many requests beside a shared projection, for gfx950:
//
//   * t2i_adapter_plan: the rows of a step in the order of their adapters, made on the device;
//   * t2i_adapter_add: out[r] = y[r] + scale_a B_a (A_a x[r]) for every row r with adapter a, y being the shared
//     projection's output; or silu(gate) * up of that for paired columns.
//
// Two launches: h = scale A x, then out = y + B h.  h is kept as two bf16 words (16 bits): both meet in one MFMA
// of 16 ranks, whose 32 terms are B h_hi and B h_lo.
#include <math.h>

#include <algorithm>

#include "t2i_common.h"

namespace t2i {

constexpr int AD_THREADS = 1024;             // of the plan
constexpr int AD_MOST = 511;                 // adapters of a pool
constexpr int AD_TILE = 64;                  // rows of a tile: one adapter's
constexpr int AD_HEAD = 4;                   // words of a tile: {adapter (-1: none), its first place in the order, rows, 0},
constexpr int AD_REC = AD_HEAD + AD_TILE;    //   then its rows, so that one look at the plan gives all
constexpr int AD_PARTS = 4;                  // slices of a projection's columns

struct AdapterPlanParams {
  const int32_t* ids;                        // [M]
  int32_t* tiles;                            // [tiles_cap][AD_REC]
  int M, n, tiles_cap;
};

// Sums of the values of the threads before this one (LDS: one word a wave).
__device__ __forceinline__ int adapter_scan(int v, int* s_wave) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const int u = __shfl_up(x, s, 64);
    if (lane >= s) x += u;
  }
  __syncthreads();
  if (lane == 63) s_wave[wave] = x;
  __syncthreads();
  int before = 0;
  for (int w = 0; w < wave; ++w) before += s_wave[w];
  return before + x - v;
}

// One workgroup: a counting sort (by adapter, those rows last that have none) that keeps the rows of an adapter in their
// order.  A wave takes its share of the rows 64 at a time, adapter by adapter of those there are among them.  5 to 7 us for up
// to 4001 rows, 12 for 8192: latency, once a step of all projections.
__global__ __launch_bounds__(AD_THREADS) void adapter_plan_kernel(const AdapterPlanParams p) {
  extern __shared__ int s_count[];           // [16 waves][n + 1]: rows, then the next place, of a wave's adapter
  __shared__ int s_wave[AD_THREADS / 64], s_tile[AD_THREADS + 1], s_start[AD_THREADS + 1];
  constexpr int WAVES = AD_THREADS / 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int buckets = p.n + 1;
  for (int i = tid; i < WAVES * buckets; i += AD_THREADS) s_count[i] = 0;
  __syncthreads();
  const int share = ((p.M + WAVES - 1) / WAVES + 63) & ~63;
  const int from = wave * share, to = min(from + share, p.M);
  int* const mine = s_count + wave * buckets;
  // every adapter among 64 rows: its rows, and whether this lane's is one of them
  const auto walk = [&](auto each) {
    for (int base = from; base < to; base += 64) {
      const int row = base + lane;
      int id = row < to ? p.ids[row] : -2;
      if (row < to && (id < 0 || id >= p.n)) id = p.n;
      unsigned long long left = __ballot(row < to);
      while (left) {
        const int a = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
        const unsigned long long same = __ballot(id == a);
        each(row, a, same, id == a);
        left &= ~same;
      }
    }
  };
  walk([&](int, int a, unsigned long long same, bool) {
    if (lane == 0) mine[a] += __builtin_popcountll(same);
  });
  __syncthreads();
  int rows = 0;
  if (tid < buckets)
    for (int w = 0; w < WAVES; ++w) rows += s_count[w * buckets + tid];
  const int start = adapter_scan(rows, s_wave);
  const int tile = adapter_scan((rows + AD_TILE - 1) / AD_TILE, s_wave);
  if (tid < buckets) {
    int at = start;
    for (int w = 0; w < WAVES; ++w) {
      const int c = s_count[w * buckets + tid];
      s_count[w * buckets + tid] = at;
      at += c;
    }
    s_start[tid] = start;
    s_tile[tid] = tile;
    if (tid == buckets - 1) {
      s_start[buckets] = start + rows;
      s_tile[buckets] = tile + (rows + AD_TILE - 1) / AD_TILE;
    }
  }
  __syncthreads();
  for (int t = tid; t < p.tiles_cap; t += AD_THREADS) {
    int4 rec = int4{-1, 0, 0, 0};
    if (t < s_tile[buckets]) {
      int lo = 0, hi = buckets;              // the last bucket that starts at t or before
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (s_tile[mid] <= t) lo = mid;
        else hi = mid;
      }
      rec.x = lo < p.n ? lo : -1;
      rec.y = s_start[lo] + (t - s_tile[lo]) * AD_TILE;
      rec.z = min(s_start[lo + 1] - rec.y, AD_TILE);
    }
    *reinterpret_cast<int4*>(p.tiles + (size_t)t * AD_REC) = rec;
  }
  walk([&](int row, int a, unsigned long long same, bool is) {
    const int at = mine[a], in = at + __builtin_popcountll(same & ((1ull << lane) - 1)) - s_start[a];   // of its adapter's rows
    if (is) p.tiles[(size_t)(s_tile[a] + in / AD_TILE) * AD_REC + AD_HEAD + in % AD_TILE] = row;
    if (lane == 0) mine[a] = at + __builtin_popcountll(same);
  });
}

struct AdapterParams {
  const uint16_t* x;                         // [M, K]
  const uint16_t* y;                         // [M, N]
  uint16_t* out;                             // [M, N], or [M, N / 2]
  const uint16_t* a;                         // [n][parts * R / 16][K / 32][4 groups of 8 k][16 ranks][8 k], R a multiple of 16
  const uint16_t* b;                         // [n][N / 128 rounded up][R / 16][8 t][2 groups of 8 ranks][16 c][8 ranks]: column 8 c + t
  const float* scales;                       // [n] or NULL
  const int32_t* tiles;
  uint16_t* h;                               // [tiles * 4][parts * R / 16][hi 0-7, hi 8-15, lo 0-7, lo 8-15][16 rows][8 ranks]
  int M, K, N, n, R, rank, parts, ends[AD_PARTS], blocks, swiglu, tiles_cap;   // ends: column behind each slice
};

// A tile as the plan has it, checked; rows 0: nothing to do.
struct AdapterTile {
  int adapter, first, rows;
  const int32_t* row;
  // Row i (below AD_TILE) of the tile, its first one behind the last: read without waiting for the count.
  __device__ __forceinline__ int at(const AdapterParams& p, int i) const {
    const int r = row[i], r0 = row[0];
    return min(max(i < rows ? r : r0, 0), p.M - 1);
  }
};
__device__ __forceinline__ AdapterTile adapter_tile(const AdapterParams& p, int t) {
  const int32_t* const rec = p.tiles + (size_t)t * AD_REC;
  const int4 w = *reinterpret_cast<const int4*>(rec);
  AdapterTile r{w.x, w.y, w.z, rec + AD_HEAD};
  if (r.adapter >= p.n || r.first < 0 || r.rows < 0 || r.rows > AD_TILE || r.first > p.M - r.rows) r.rows = 0;
  return r;
}

// ============================================================================
// h = scale A x
// ============================================================================
// A workgroup 16 rows of a tile by NC x 16 ranks; its waves take 128 k in turn and meet in LDS.  A comes in the order
// that the MFMA takes it (1 KB a load instruction).  An operand's lanes want 16 rows of x at once: loaded that way four
// neighbouring lanes ask for four lines, and the loads alone took 16 us of 4001 rows' 19 (K 6144, two fragments of
// ranks).  So an instruction takes 256 bytes of four rows, and the rows turn into operands in the wave's own part of LDS, a
// row's 16-byte piece q at place q ^ row: 16 lanes of a write or a read cover all banks.
// Sixteen waves in place of eight gained nothing (4001 rows 22.0 us, 8192 56).
// 4001 rows 12-13 us (49 MB of x, 4 TB/s; nothing hides a wave's first and last loads: six rounds a wave), 8192 of K 2048
// 13 (34 MB), 331 5.3, 16 3.3 (two rounds of dependent loads).
constexpr int AD_WAVES = 8;

template <int NC>
__global__ __launch_bounds__(64 * AD_WAVES, 4) void adapter_shrink_kernel(const AdapterParams p) {
  constexpr int STEPS = 4, W = AD_WAVES;                   // steps of 32 k
  union Lds {
    uint16_t x[W][16 * 32 * STEPS];
    float part[W][NC][16][17];
  };
  __shared__ __align__(16) Lds lds;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // (workgroups go round the eight XCDs: those that share rows of x stand eight apart, behind one L2)
  const int block = blockIdx.x / 8 % p.blocks, rows16 = blockIdx.x / 8 / p.blocks * 8 + blockIdx.x % 8;
  const int sub = rows16 % (AD_TILE / 16), tile = rows16 / (AD_TILE / 16);
  const int c = lane & 15, g = lane >> 4;
  if (tile >= p.tiles_cap) return;
  const AdapterTile t = adapter_tile(p, tile);
  if (t.adapter < 0 || sub * 16 >= t.rows) return;
  const uint16_t* x[4];                                    // rows 4 q + g
#pragma unroll
  for (int q = 0; q < 4; ++q) x[q] = p.x + (size_t)t.at(p, sub * 16 + 4 * q + g) * p.K;
  const int groups = p.parts * p.R / 16, g0 = block * NC, steps = p.K / 32;
  const uint16_t* a[NC];
#pragma unroll
  for (int j = 0; j < NC; ++j) a[j] = p.a + ((size_t)t.adapter * groups + min(g0 + j, groups - 1)) * p.K * 16 + 8 * lane;
  f32x4 acc[NC];
#pragma unroll
  for (int j = 0; j < NC; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  u32x4 xv[4];
  const auto fetch = [&](int s0) __attribute__((always_inline)) {
    const int k = min(32 * s0 + 8 * c, p.K - 8);           // (what lies behind K is not multiplied)
#pragma unroll
    for (int q = 0; q < 4; ++q) xv[q] = *reinterpret_cast<const u32x4*>(x[q] + k);
  };
  if (STEPS * wave < steps) fetch(STEPS * wave);
  for (int s0 = STEPS * wave; s0 < steps; s0 += STEPS * W) {
    u32x4 av[STEPS][NC];
#pragma unroll
    for (int u = 0; u < STEPS; ++u)
#pragma unroll
      for (int j = 0; j < NC; ++j) av[u][j] = *reinterpret_cast<const u32x4*>(a[j] + (size_t)min(s0 + u, steps - 1) * 512);
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *reinterpret_cast<u32x4*>(&lds.x[wave][(4 * q + g) * 128 + 8 * (c ^ (4 * q + g))]) = xv[q];
    if (s0 + STEPS * W < steps) fetch(s0 + STEPS * W);
#pragma unroll
    for (int u = 0; u < STEPS; ++u) {
      if (s0 + u >= steps) break;
      const u32x4 xo = *reinterpret_cast<const u32x4*>(&lds.x[wave][c * 128 + 8 * ((4 * u + g) ^ c)]);
#pragma unroll
      for (int j = 0; j < NC; ++j)
        acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, xo), __builtin_bit_cast(bf16x8, av[u][j]), acc[j], 0, 0, 0);
    }
  }
  __syncthreads();                                         // the rows of x are done with
  // register e: row 4 g + e, rank c
#pragma unroll
  for (int j = 0; j < NC; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) lds.part[wave][j][4 * g + e][c] = acc[j][e];
  __syncthreads();
  const float scale = p.scales ? p.scales[t.adapter] : 1.0f;
  for (int e = threadIdx.x; e < NC * 256; e += 64 * W) {
    const int j = e >> 8, group = g0 + j, row = e >> 4 & 15, col = e & 15;
    if (group >= groups) continue;
    float h = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) h += lds.part[w][j][row][col];
    h = (16 * group + col) % p.R < p.rank ? h * scale : 0.0f;   // (a rank of the padding may be 0 times an infinity)
    const uint32_t hi = f32_to_bf16(h);
    const float left = h - bf16_to_f32(hi);
    uint16_t* const dst = p.h + (((size_t)tile * (AD_TILE / 16) + sub) * groups + group) * 512 + (col >> 3) * 128 + row * 8 + (col & 7);
    dst[0] = hi;
    dst[256] = fabsf(left) < INFINITY ? f32_to_bf16(left) : 0;   // an infinity stays one
  }
}

// ============================================================================
// out = y + B h
// ============================================================================
// A wave 16 rows of a tile by 128 columns; a workgroup the tile's 64 rows.  (Tiles of up to 16 rows with four times the columns
// a workgroup in place of three waves that leave at once: 64 single rows 9.8 us for 8.5, 32 x 5 17.2 for 16.4.)  B comes in
// the order that the MFMA takes it, and in one that leaves a lane (c, g) 8 neighbouring columns of rows 4 g .. 4 g + 3
// (register i of product t: column 8 c + t of row 4 g + i): y and out move as 256 bytes of four rows an instruction.  Of
// paired columns the even products are gate's, the odd ones up's. 8192 rows of rank 16 37 us (201 MB, 5.4 TB/s: the rate of
// a copy), 4001 of rank 32 8 (33 MB), 331 of rank 64 7.5 (23 MB: the plan's word, then B, then the results, one after the
// other), 16 3.  Higher ranks wait for B and h in the caches: 5100 rows of 12288 paired columns 38, 59, 85 us at rank 16,
// 64, 128.  B of 64 ranks in LDS for the four waves of a workgroup gained 4 % at rank 128 and 5 % for the 8192 rows and
// cost 2 to 3 % for 16 and 331 rows.
template <bool PAIRED>
__global__ __launch_bounds__(256) void adapter_expand_kernel(const AdapterParams p) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tile = blockIdx.x / p.blocks;
  const AdapterTile t = adapter_tile(p, tile);
  const int block = blockIdx.x % p.blocks, n0 = 128 * block, sub = wave;
  if (n0 >= p.N || sub * 16 >= t.rows) return;
  if (t.adapter < 0 && !p.swiglu && p.out == p.y) return;  // nothing to add in place
  const int c = lane & 15, g = lane >> 4;
  const int col = n0 + 8 * c;
  int row[4];
  u32x4 y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    row[i] = t.at(p, sub * 16 + 4 * g + i);
    y[i] = *reinterpret_cast<const u32x4*>(p.y + (size_t)row[i] * p.N + min(col, p.N - 8));
  }
  if (t.adapter < 0 && !p.swiglu) {                        // their bits, where a sum with 0 makes 0 of -0
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (col < p.N && sub * 16 + 4 * g + i < t.rows) *reinterpret_cast<u32x4*>(p.out + (size_t)row[i] * p.N + col) = y[i];
    return;
  }
  f32x4 acc[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) acc[k] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (t.adapter >= 0) {
    const int groups = p.parts * p.R / 16, steps = p.R / 16;
    int slice = 0;                                         // of the wave's columns
    if (!PAIRED)
      for (int s = 0; s < AD_PARTS - 1; ++s) slice += s < p.parts - 1 && n0 >= p.ends[s];
    const uint16_t* const h = p.h + (((size_t)tile * (AD_TILE / 16) + sub) * groups + slice * steps) * 512 + 8 * lane;
    const uint16_t* const b = p.b + ((size_t)t.adapter * ((p.N + 127) / 128) + block) * p.R * 128 + 8 * lane;
    // The operands of a step come while the one before it is multiplied.  Both halves of a wave take the same of B (for the
    // two words of h): a load brings two products' to the halves, and a swap gives either to both.
    u32x4 hv[2], bv[4];
    const auto fetch_h = [&](int s) __attribute__((always_inline)) {
      hv[0] = *reinterpret_cast<const u32x4*>(h + 512 * s);
      if (PAIRED) hv[1] = *reinterpret_cast<const u32x4*>(h + 512 * (s + steps));
    };
    const auto fetch_b = [&](int s, int k) __attribute__((always_inline)) { bv[k] = *reinterpret_cast<const u32x4*>(b + (4 * s + k) * 512); };
    const auto multiply = [&](int k, u32x4 w, u32x4 x0, u32x4 x1) __attribute__((always_inline)) {
      u32x4 w0, w1;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const auto both = __builtin_amdgcn_permlane32_swap(w[e], w[e], false, false);
        w0[e] = both[0];
        w1[e] = both[1];
      }
      acc[2 * k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x0), __builtin_bit_cast(bf16x8, w0), acc[2 * k], 0, 0, 0);
      acc[2 * k + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x1), __builtin_bit_cast(bf16x8, w1), acc[2 * k + 1], 0, 0, 0);
    };
    fetch_h(0);
#pragma unroll
    for (int k = 0; k < 4; ++k) fetch_b(0, k);
#pragma unroll 1
    for (int s = 1; s < steps; ++s) {
      const u32x4 x0 = hv[0], x1 = hv[PAIRED];
      fetch_h(s);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const u32x4 w = bv[k];
        fetch_b(s, k);
        multiply(k, w, x0, x1);
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) multiply(k, bv[k], hv[0], hv[PAIRED]);
  }
  if (col >= p.N) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (sub * 16 + 4 * g + i >= t.rows) break;
    float f[8];
    unpack8(y[i], f);
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] += acc[k][i];
    if (p.swiglu) {                                        // silu(gate) * up, rounded once (the exponential and the reciprocal are off by an ulp)
      float r[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) r[k] = f[2 * k] * __builtin_amdgcn_rcpf(1.0f + exp2_fast(-1.4426950408889634f * f[2 * k])) * f[2 * k + 1];
      *reinterpret_cast<u32x2*>(p.out + (size_t)row[i] * (p.N / 2) + col / 2) = u32x2{pack_bf16x2(r[0], r[1]), pack_bf16x2(r[2], r[3])};
    } else {
      *reinterpret_cast<u32x4*>(p.out + (size_t)row[i] * p.N + col) =
          u32x4{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])};
    }
  }
}

}  // namespace t2i

using t2i_host::aligned16;
using t2i_host::fail;

namespace {

bool aligned4(const void* p) { return ((uintptr_t)p & 3u) == 0; }

int tiles_cap(int32_t M, int32_t n) { return M / t2i::AD_TILE + std::min(n + 1, M); }
int64_t plan_words(int32_t M, int32_t n) { return (int64_t)tiles_cap(M, n) * t2i::AD_REC; }
int padded(int32_t rank) { return (rank + 15) / 16 * 16; }

int check_rows(int32_t M, int32_t n) {
  if (M < 1 || M > (1 << 24) - 1) return fail(T2I_ERR_SHAPE, "M=%d rows invalid", M);
  if (n < 1 || n > t2i::AD_MOST) return fail(T2I_ERR_SHAPE, "%d adapters (1 to %d)", n, t2i::AD_MOST);
  return T2I_OK;
}

}  // namespace

extern "C" int64_t t2i_adapter_plan_words(int32_t M, int32_t n_adapters) {
  return check_rows(M, n_adapters) ? 0 : plan_words(M, n_adapters);
}

extern "C" int t2i_adapter_plan(const int32_t* ids, int32_t M, int32_t n_adapters, int32_t* plan, int64_t words, void* stream) {
  if (!ids || !plan) return fail(T2I_ERR_NULL, "ids and plan must not be NULL");
  if (!aligned4(ids)) return fail(T2I_ERR_ALIGN, "ids must be 4-byte aligned");
  if (!aligned16(plan)) return fail(T2I_ERR_ALIGN, "the plan must be 16-byte aligned");
  if (int rc = check_rows(M, n_adapters)) return rc;
  if (words < plan_words(M, n_adapters))
    return fail(T2I_ERR_WORKSPACE, "the plan holds %lld words, %lld needed", (long long)words, (long long)plan_words(M, n_adapters));
  t2i::AdapterPlanParams p{};
  p.ids = ids; p.M = M; p.n = n_adapters; p.tiles_cap = tiles_cap(M, n_adapters);
  p.tiles = plan;
  const size_t lds = (size_t)(t2i::AD_THREADS / 64) * (n_adapters + 1) * sizeof(int);
  hipLaunchKernelGGL(t2i::adapter_plan_kernel, dim3(1), dim3(t2i::AD_THREADS), lds, reinterpret_cast<hipStream_t>(stream), p);
  return t2i_host::hip_status(hipGetLastError(), "adapter plan launch");
}

extern "C" size_t t2i_adapter_add_workspace_bytes(int32_t M, int32_t n_adapters, int32_t parts, int32_t rank) {
  if (check_rows(M, n_adapters) || parts < 1 || parts > t2i::AD_PARTS || rank < 1 || rank > 256) return 0;
  return (size_t)tiles_cap(M, n_adapters) * (t2i::AD_TILE / 16) * (parts * padded(rank) / 16) * 1024;
}

extern "C" int t2i_adapter_add(const uint16_t* y, const uint16_t* x, int32_t M, int32_t K, int32_t N, const int32_t* plan,
                               int64_t words, const uint16_t* a, const uint16_t* b, const float* scales, int32_t n_adapters,
                               int32_t rank, int32_t parts, const int32_t* widths, int32_t paired, int32_t swiglu,
                               uint16_t* out, void* workspace, size_t workspace_bytes, void* stream) {
  if (!y || !x || !plan || !a || !b || !out)
    return fail(T2I_ERR_NULL, "adapter_add pointers must not be NULL");
  if (!aligned16(y) || !aligned16(x) || !aligned16(plan) || !aligned16(a) || !aligned16(b) || !aligned16(out))
    return fail(T2I_ERR_ALIGN, "adapter_add tensors must be 16-byte aligned");
  if (!aligned4(scales)) return fail(T2I_ERR_ALIGN, "scales must be 4-byte aligned");
  if (int rc = check_rows(M, n_adapters)) return rc;
  if (K < 32 || K % 32 || N < 16 || N % 16 || K > 1 << 20 || N > 1 << 20)
    return fail(T2I_ERR_SHAPE, "K=%d N=%d unsupported (K %% 32, N %% 16)", K, N);
  if (rank < 1 || rank > 256) return fail(T2I_ERR_SHAPE, "rank %d unsupported (1 to 256)", rank);
  if (parts < 1 || parts > t2i::AD_PARTS || (paired && parts != 2))
    return fail(T2I_ERR_SHAPE, "%d slices unsupported (1 to %d, paired: 2)", parts, t2i::AD_PARTS);
  if (parts > 1 && !paired && !widths) return fail(T2I_ERR_NULL, "slices need widths");
  if (swiglu && !paired) return fail(T2I_ERR_VALUE, "SwiGLU needs paired columns");
  if (swiglu && out == y) return fail(T2I_ERR_VALUE, "SwiGLU has rows of N / 2: out must not be y");
  t2i::AdapterParams p{};
  if (!paired && parts > 1) {
    long long at = 0;
    for (int i = 0; i < parts; ++i) {
      if (widths[i] < 128 || widths[i] % 128) return fail(T2I_ERR_SHAPE, "a slice of %d columns (multiples of 128)", widths[i]);
      p.ends[i] = (int)(at += widths[i]);
      if (at > N) break;
    }
    if (at != N) return fail(T2I_ERR_SHAPE, "the slices hold %lld columns, N=%d", at, N);
  }
  if (words < plan_words(M, n_adapters))
    return fail(T2I_ERR_WORKSPACE, "the plan holds %lld words, %lld needed", (long long)words, (long long)plan_words(M, n_adapters));
  const size_t need = t2i_adapter_add_workspace_bytes(M, n_adapters, parts, rank);
  if (!workspace || workspace_bytes < need) return fail(T2I_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : 0, need);
  if (!aligned16(workspace)) return fail(T2I_ERR_ALIGN, "the workspace must be 16-byte aligned");
  const int cap = tiles_cap(M, n_adapters);
  p.x = x; p.y = y; p.out = out; p.a = a; p.b = b; p.scales = scales;
  p.tiles = plan; p.h = reinterpret_cast<uint16_t*>(workspace);
  p.M = M; p.K = K; p.N = N; p.n = n_adapters; p.tiles_cap = cap; p.R = padded(rank); p.rank = rank; p.parts = parts; p.swiglu = swiglu != 0;
  const int fragments = parts * p.R / 16, expand_blocks = (N + 127) / 128;
  if (((long long)cap * 4 + 8) * fragments > 0xFFFFFFFFLL / 1024 || (long long)cap * expand_blocks > 0xFFFFFFFFLL / 256)
    return fail(T2I_ERR_SHAPE, "M=%d N=%d rank=%d exceed the grid", M, N, rank);
  const uintptr_t y0 = (uintptr_t)y, out0 = (uintptr_t)out;
  const uintptr_t y_bytes = 2 * (uintptr_t)M * N, out_bytes = swiglu ? y_bytes / 2 : y_bytes;
  if (out0 != y0 && out0 < y0 + y_bytes && y0 < out0 + out_bytes)
    return fail(T2I_ERR_VALUE, "out must be y itself or lie beside it");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  // as many fragments of ranks a workgroup (up to four) as leave one for every CU (1, 2, 3, 4 of them, us: 331 rows
  // of 8 12.8, 13.0, 13.7, 14.5; 16 of 3 5.7, 6.1, 6.5, 6.5; 4001 of 2 21.5, 20.7; 8192 of 3 52.4, 53.8, 51.8)
  const int nc = (int)std::min<long long>(std::min(fragments, 4), std::max<long long>(1, ((long long)M * fragments + 4095) / 4096));
  p.blocks = (fragments + nc - 1) / nc;
  const dim3 grid((cap * 4 + 7) / 8 * 8 * p.blocks), threads(64 * t2i::AD_WAVES);
  switch (nc) {
    case 1: hipLaunchKernelGGL(t2i::adapter_shrink_kernel<1>, grid, threads, 0, s, p); break;
    case 2: hipLaunchKernelGGL(t2i::adapter_shrink_kernel<2>, grid, threads, 0, s, p); break;
    case 3: hipLaunchKernelGGL(t2i::adapter_shrink_kernel<3>, grid, threads, 0, s, p); break;
    default: hipLaunchKernelGGL(t2i::adapter_shrink_kernel<4>, grid, threads, 0, s, p); break;
  }
  if (int rc = t2i_host::hip_status(hipGetLastError(), "adapter shrink launch")) return rc;
  p.blocks = expand_blocks;
  if (paired) hipLaunchKernelGGL(t2i::adapter_expand_kernel<true>, dim3(cap * p.blocks), dim3(256), 0, s, p);
  else hipLaunchKernelGGL(t2i::adapter_expand_kernel<false>, dim3(cap * p.blocks), dim3(256), 0, s, p);
  return t2i_host::hip_status(hipGetLastError(), "adapter expand launch");
}
