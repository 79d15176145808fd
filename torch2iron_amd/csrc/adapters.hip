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
constexpr int AD_REC = 4;                    // words of a tile: {adapter (-1: none), its first place in the order, rows, 0}
constexpr int AD_PARTS = 4;                  // slices of a projection's columns

struct AdapterPlanParams {
  const int32_t* ids;                        // [M]
  int32_t* tiles;                            // [tiles_cap][AD_REC]
  int32_t* order;                            // [M] rows by adapter, those without one last
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

// One workgroup: a counting sort that keeps the rows of an adapter in their order.  A wave takes its share of
// the rows 64 at a time, adapter by adapter of those there are among them.
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
    reinterpret_cast<int4*>(p.tiles)[t] = rec;
  }
  walk([&](int row, int a, unsigned long long same, bool is) {
    const int at = mine[a];
    if (is) p.order[at + __builtin_popcountll(same & ((1ull << lane) - 1))] = row;
    if (lane == 0) mine[a] = at + __builtin_popcountll(same);
  });
}

struct AdapterParams {
  const uint16_t* x;                         // [M, K]
  const uint16_t* y;                         // [M, N]
  uint16_t* out;                             // [M, N], or [M, N / 2]
  const uint16_t* a;                         // [n, parts * R, K], R a multiple of 16
  const uint16_t* b;                         // [n, N, R]
  const float* scales;                       // [n] or NULL
  const int32_t* tiles;
  const int32_t* order;
  uint16_t* h;                               // [M][parts * R / 16][hi 16, lo 16]: rows in the plan's order
  int M, K, N, n, R, rank, parts, ends[AD_PARTS], blocks, swiglu;   // ends: column behind each slice
};

// A tile as the plan has it, checked; rows 0: nothing to do.
struct AdapterTile {
  int adapter, first, rows;
};
__device__ __forceinline__ AdapterTile adapter_tile(const AdapterParams& p, int t) {
  const int4 w = reinterpret_cast<const int4*>(p.tiles)[t];
  AdapterTile r{w.x, w.y, w.z};
  if (r.adapter >= p.n || r.first < 0 || r.rows < 0 || r.rows > AD_TILE || r.first > p.M - r.rows) r.rows = 0;
  return r;
}
__device__ __forceinline__ int adapter_row(const AdapterParams& p, int at) { return min(max(p.order[at], 0), p.M - 1); }

// ============================================================================
// h = scale A x
// ============================================================================
// A workgroup 16 rows of a tile by NC x 16 ranks; its waves share K and meet in LDS.  Both operands come straight from
// memory: lane (c, g) holds 8 neighbouring k of row c (x) and of rank c (A).
constexpr int AD_WAVES = 8;

template <int NC>
__global__ __launch_bounds__(64 * AD_WAVES) void adapter_shrink_kernel(const AdapterParams p) {
  __shared__ float s_part[AD_WAVES][NC][16][17];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int block = blockIdx.x % p.blocks, sub = blockIdx.x / p.blocks % (AD_TILE / 16);
  const AdapterTile t = adapter_tile(p, blockIdx.x / p.blocks / (AD_TILE / 16));
  if (t.adapter < 0 || sub * 16 >= t.rows) return;
  const int c = lane & 15, g = lane >> 4;
  const int ranks = p.parts * p.R, r0 = block * NC * 16;
  const uint16_t* const x = p.x + (size_t)adapter_row(p, t.first + min(sub * 16 + c, t.rows - 1)) * p.K + 8 * g;
  const uint16_t* a[NC];
#pragma unroll
  for (int j = 0; j < NC; ++j) a[j] = p.a + ((size_t)t.adapter * ranks + min(r0 + 16 * j + c, ranks - 1)) * p.K + 8 * g;
  const int steps = p.K / 32, k0 = wave * steps / AD_WAVES, k1 = (wave + 1) * steps / AD_WAVES;
  f32x4 acc[NC];
#pragma unroll
  for (int j = 0; j < NC; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int k = k0; k < k1; ++k) {
    const u32x4 xv = *reinterpret_cast<const u32x4*>(x + 32 * k);
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const u32x4 av = *reinterpret_cast<const u32x4*>(a[j] + 32 * k);
      acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, xv), __builtin_bit_cast(bf16x8, av), acc[j], 0, 0, 0);
    }
  }
  // register i: row 4 g + i, rank c
#pragma unroll
  for (int j = 0; j < NC; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) s_part[wave][j][4 * g + i][c] = acc[j][i];
  __syncthreads();
  const float scale = p.scales ? p.scales[t.adapter] : 1.0f;
  for (int e = threadIdx.x; e < NC * 256; e += 64 * AD_WAVES) {
    const int j = e >> 8, row = e >> 4 & 15, col = e & 15;
    const int rank = r0 + 16 * j + col;
    if (sub * 16 + row >= t.rows || rank >= ranks) continue;
    float h = 0.0f;
#pragma unroll
    for (int w = 0; w < AD_WAVES; ++w) h += s_part[w][j][row][col];
    h = rank % p.R < p.rank ? h * scale : 0.0f;            // (a rank of the padding may be 0 times an infinity)
    const uint32_t hi = f32_to_bf16(h);
    const float left = h - bf16_to_f32(hi);
    uint16_t* const dst = p.h + ((size_t)(t.first + sub * 16 + row) * ranks + (r0 + 16 * j)) * 2 + col;
    dst[0] = hi;
    dst[16] = fabsf(left) < INFINITY ? f32_to_bf16(left) : 0;   // an infinity stays one
  }
}

// ============================================================================
// out = y + B h
// ============================================================================
// A workgroup a tile by 256 columns, a wave 64 of them, 16 rows at a time.  Run transposed (B's rows as the
// MFMA's rows), with B's rows in an order that leaves a lane 16 neighbouring columns of one row:
// register i of part t holds column 16 g + 4 t + i (paired: gate 8 g + 4 (t % 2) + i for t < 2, up behind).
template <bool PAIRED>
__global__ __launch_bounds__(256) void adapter_expand_kernel(const AdapterParams p) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = (blockIdx.x % p.blocks * 4 + wave) * 64;
  const AdapterTile t = adapter_tile(p, blockIdx.x / p.blocks);
  if (n0 >= p.N || t.rows == 0) return;
  if (t.adapter < 0 && !p.swiglu && p.out == p.y) return;  // nothing to add in place
  const int c = lane & 15, g = lane >> 4;
  const int groups = p.parts * p.R / 16, steps = p.R / 16;
  int slice = 0;                                           // of the wave's columns
  if (!PAIRED)
    for (int s = 0; s < AD_PARTS - 1; ++s) slice += s < p.parts - 1 && n0 >= p.ends[s];
  const uint16_t* b[4];
#pragma unroll
  for (int t4 = 0; t4 < 4; ++t4) {
    const int col = PAIRED ? 2 * (4 * (t4 & 1) + (c & 3)) + (t4 >> 1) : 4 * t4 + (c & 3);
    b[t4] = p.b + ((size_t)max(t.adapter, 0) * p.N + min(n0 + 16 * (c >> 2) + col, p.N - 1)) * p.R + 8 * (g & 1);
  }
  const int col = n0 + 16 * g;                             // the lane's columns
  for (int sub = 0; sub * 16 < t.rows; ++sub) {
    const int at = t.first + min(sub * 16 + c, t.rows - 1);
    const int row = adapter_row(p, at);
    const bool live = sub * 16 + c < t.rows && col < p.N;
    u32x4 y0 = u32x4{0, 0, 0, 0}, y1 = y0;
    if (live) {
      y0 = *reinterpret_cast<const u32x4*>(p.y + (size_t)row * p.N + col);
      y1 = *reinterpret_cast<const u32x4*>(p.y + (size_t)row * p.N + col + 8);
    }
    f32x4 acc[4];
#pragma unroll
    for (int t4 = 0; t4 < 4; ++t4) acc[t4] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (t.adapter >= 0) {
      const uint16_t* const h = p.h + ((size_t)at * groups + slice * steps) * 32 + 8 * g;
      for (int s = 0; s < steps; ++s) {
        u32x4 hv[2];
        hv[0] = *reinterpret_cast<const u32x4*>(h + 32 * s);
        if (PAIRED) hv[1] = *reinterpret_cast<const u32x4*>(h + 32 * (s + steps));
#pragma unroll
        for (int t4 = 0; t4 < 4; ++t4) {
          const u32x4 bv = *reinterpret_cast<const u32x4*>(b[t4] + 16 * s);
          acc[t4] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, bv),
                                                            __builtin_bit_cast(bf16x8, hv[PAIRED ? t4 >> 1 : 0]), acc[t4], 0, 0, 0);
        }
      }
    }
    float f[16];
    {
      float lo[8], hi[8];
      unpack8(y0, lo);
      unpack8(y1, hi);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = lo[i], f[8 + i] = hi[i];
    }
#pragma unroll
    for (int e = 0; e < 16; ++e)
      f[e] += PAIRED ? acc[2 * (e & 1) + (e >> 3)][e >> 1 & 3] : acc[e >> 2][e & 3];
    if (!live) continue;
    if (p.swiglu) {                                        // silu(gate) * up, rounded once
      float r[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] = silu_f32(f[2 * i]) * f[2 * i + 1];
      *reinterpret_cast<u32x4*>(p.out + (size_t)row * (p.N / 2) + col / 2) =
          u32x4{pack_bf16x2(r[0], r[1]), pack_bf16x2(r[2], r[3]), pack_bf16x2(r[4], r[5]), pack_bf16x2(r[6], r[7])};
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        *reinterpret_cast<u32x4*>(p.out + (size_t)row * p.N + col + 8 * i) =
            u32x4{pack_bf16x2(f[8 * i], f[8 * i + 1]), pack_bf16x2(f[8 * i + 2], f[8 * i + 3]),
                  pack_bf16x2(f[8 * i + 4], f[8 * i + 5]), pack_bf16x2(f[8 * i + 6], f[8 * i + 7])};
    }
  }
}

}  // namespace t2i

using t2i_host::aligned16;
using t2i_host::fail;

namespace {

bool aligned4(const void* p) { return ((uintptr_t)p & 3u) == 0; }

int tiles_cap(int32_t M, int32_t n) { return M / t2i::AD_TILE + std::min(n + 1, M); }
int64_t plan_words(int32_t M, int32_t n) { return (int64_t)tiles_cap(M, n) * t2i::AD_REC + M; }
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
  p.tiles = plan; p.order = plan + (size_t)p.tiles_cap * t2i::AD_REC;
  const size_t lds = (size_t)(t2i::AD_THREADS / 64) * (n_adapters + 1) * sizeof(int);
  hipLaunchKernelGGL(t2i::adapter_plan_kernel, dim3(1), dim3(t2i::AD_THREADS), lds, reinterpret_cast<hipStream_t>(stream), p);
  return t2i_host::hip_status(hipGetLastError(), "adapter plan launch");
}

extern "C" size_t t2i_adapter_add_workspace_bytes(int32_t M, int32_t parts, int32_t rank) {
  if (M < 1 || parts < 1 || parts > t2i::AD_PARTS || rank < 1 || rank > 256) return 0;
  return (size_t)M * parts * padded(rank) * 4;
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
      if (widths[i] < 64 || widths[i] % 64) return fail(T2I_ERR_SHAPE, "a slice of %d columns (multiples of 64)", widths[i]);
      p.ends[i] = (int)(at += widths[i]);
      if (at > N) break;
    }
    if (at != N) return fail(T2I_ERR_SHAPE, "the slices hold %lld columns, N=%d", at, N);
  }
  if (words < plan_words(M, n_adapters))
    return fail(T2I_ERR_WORKSPACE, "the plan holds %lld words, %lld needed", (long long)words, (long long)plan_words(M, n_adapters));
  const size_t need = t2i_adapter_add_workspace_bytes(M, parts, rank);
  if (!workspace || workspace_bytes < need) return fail(T2I_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : 0, need);
  if (!aligned16(workspace)) return fail(T2I_ERR_ALIGN, "the workspace must be 16-byte aligned");
  const int cap = tiles_cap(M, n_adapters);
  p.x = x; p.y = y; p.out = out; p.a = a; p.b = b; p.scales = scales;
  p.tiles = plan; p.order = plan + (size_t)cap * t2i::AD_REC; p.h = reinterpret_cast<uint16_t*>(workspace);
  p.M = M; p.K = K; p.N = N; p.n = n_adapters; p.R = padded(rank); p.rank = rank; p.parts = parts; p.swiglu = swiglu != 0;
  const int fragments = parts * p.R / 16, expand_blocks = (N + 255) / 256;
  if ((long long)cap * 4 * fragments > 0xFFFFFFFFLL / 512 || (long long)cap * expand_blocks > 0xFFFFFFFFLL / 256)
    return fail(T2I_ERR_SHAPE, "M=%d N=%d rank=%d exceed the grid", M, N, rank);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  // few rows: 16 ranks a workgroup, so that there are enough of them
  if (M <= 256 || fragments == 1) {
    p.blocks = fragments;
    hipLaunchKernelGGL(t2i::adapter_shrink_kernel<1>, dim3(cap * 4 * p.blocks), dim3(64 * t2i::AD_WAVES), 0, s, p);
  } else {
    p.blocks = (fragments + 3) / 4;
    hipLaunchKernelGGL(t2i::adapter_shrink_kernel<4>, dim3(cap * 4 * p.blocks), dim3(64 * t2i::AD_WAVES), 0, s, p);
  }
  if (int rc = t2i_host::hip_status(hipGetLastError(), "adapter shrink launch")) return rc;
  p.blocks = expand_blocks;
  if (paired) hipLaunchKernelGGL(t2i::adapter_expand_kernel<true>, dim3(cap * p.blocks), dim3(256), 0, s, p);
  else hipLaunchKernelGGL(t2i::adapter_expand_kernel<false>, dim3(cap * p.blocks), dim3(256), 0, s, p);
  return t2i_host::hip_status(hipGetLastError(), "adapter expand launch");
}
