// Log probabilities of given tokens over rows of logits for gfx950, with each row's entropy
// and its top alternatives, in one pass over the logits (t2i_token_logprobs).
//
// With a reference m near the row's largest logit and y = (x - m) log2 e:
//   Z = sum 2^y,  T = sum 2^y y,  log p(t) = x_t - m - ln Z,  entropy = ln Z - (T / Z) ln 2.
// m, Z and T are kept as the pass goes: when y's reference falls by d (a larger m), Z and T follow
// it as Z 2^d and (T + d Z) 2^d.  A lane's m moves only when a logit passes it by LP_SLACK: weights
// up to e^LP_SLACK have the same relative precision, and after its first values a lane hardly
// ever stops for it.  fp32 throughout; the difference is taken before it is scaled, so
// that logits of any size (the type's lowest value as a mask among them) keep their places.
#include <math.h>

#include <algorithm>

#include "t2i_common.h"

namespace t2i {

constexpr int LP_WAVES = 4;
constexpr int LP_THREADS = 64 * LP_WAVES;
constexpr int LP_TOP = 32;                   // alternatives of a row: one lane of a wave each
constexpr int LP_UNROLL = 4;                 // 16-byte loads of a lane in flight
constexpr float LP_SLACK = 6.0f;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

typedef unsigned long long u64;

// What a part of a row leaves.
struct LpState {
  float m, z, t;
};

__device__ __forceinline__ LpState lp_join(LpState a, LpState b) {
  const float m = fmaxf(a.m, b.m);
  const float ms = m > -INFINITY ? m : 0.0f;   // nothing but -inf so far: every weight is 0
  // (an infinite maximum gives NaN here, as the definition does)
  const float da = a.m > -INFINITY ? (a.m - ms) * LOG2E : -INFINITY, db = b.m > -INFINITY ? (b.m - ms) * LOG2E : -INFINITY;
  const float fa = exp2_fast(da), fb = exp2_fast(db);
  LpState r;
  r.m = m;
  r.z = a.z * fa + b.z * fb;
  r.t = (a.t + fmaxf(da, -1e30f) * a.z) * fa + (b.t + fmaxf(db, -1e30f) * b.z) * fb;
  return r;
}

// A value and its index as one key: larger values first, among equals the lower index; NaN above
// every number, both zeros alike.
__device__ __forceinline__ u64 lp_key(float v, int index) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  const uint32_t o = v != v ? 0xFFFFFFFFu : (b & 0x80000000u ? ~b : b | 0x80000000u);
  return (u64)o << 32 | (0xFFFFFFFFu - (uint32_t)index);
}
__device__ __forceinline__ float lp_value(u64 key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return o == 0xFFFFFFFFu ? __uint_as_float(0x7FC00000u) : __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
__device__ __forceinline__ u64 lane_key(u64 v, int lane) {
  return (u64)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(v >> 32), lane) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((uint32_t)v, lane);
}

// A wave's best keys, descending, one a lane.  Keys below 2^32 stand for no value.
struct LpTop {
  u64 list = 0, last = 0;                    // last: the k-th key (uniform)
  float floor = __uint_as_float(0x7FC00000u);   // its value; NaN, which no comparison passes, while there is none
  __device__ __forceinline__ void set_last(int k) {
    last = lane_key(list, k - 1);
    floor = lp_value(last);
  }
  // The list from one key a lane, each in the place of its rank (all different).
  __device__ __forceinline__ void fill(u64 key, int k) {
    int rank = 0;
#pragma unroll 8
    for (int i = 0; i < 64; ++i) rank += lane_key(key, i) > key;
    list = (u64)(uint32_t)__builtin_amdgcn_ds_permute(4 * rank, (int)(key >> 32)) << 32 |
           (uint32_t)__builtin_amdgcn_ds_permute(4 * rank, (int)key);
    set_last(k);
  }
  __device__ __forceinline__ void insert(u64 x, int k, int lane) {
    const int pos = __builtin_popcountll(__ballot(list > x));
    // every lane's neighbour below (wave_shr:1)
    const u64 up = (u64)(uint32_t)__builtin_amdgcn_update_dpp(0, (int)(list >> 32), 0x138, 0xF, 0xF, false) << 32 |
                   (uint32_t)__builtin_amdgcn_update_dpp(0, (int)list, 0x138, 0xF, 0xF, false);
    list = lane < pos ? list : lane == pos ? x : up;
    set_last(k);
  }
  // every lane's key that belongs here (0: none)
  __device__ __forceinline__ void take(u64 key, int k, int lane) {
    u64 in = __ballot(key > last);
    while (in) {
      const int at = __builtin_ctzll(in);
      insert(lane_key(key, at), k, lane);
      in &= in - 1;
      in &= __ballot(key > last);
    }
  }
};

// Word i (modulo 4) of a 16-byte piece.
__device__ __forceinline__ uint32_t word_of(u32x4 v, int i) {
  const uint32_t a = i & 1 ? v.y : v.x, b = i & 1 ? v.w : v.z;
  return i & 2 ? b : a;
}

template <typename T>
struct LpType;
template <>
struct LpType<float> {
  static constexpr int PER = 4;              // values of a 16-byte piece
  static __device__ __forceinline__ void get(u32x4 v, float* f) {
    f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ float one(const void* p, size_t i) { return reinterpret_cast<const float*>(p)[i]; }
  // value i of a piece
  static __device__ __forceinline__ float pick(u32x4 v, int i) { return __uint_as_float(word_of(v, i)); }
};
struct LpBf16 {};
template <>
struct LpType<LpBf16> {
  static constexpr int PER = 8;
  static __device__ __forceinline__ void get(u32x4 v, float* f) {
    float g[8];
    unpack8(v, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = g[i];
  }
  static __device__ __forceinline__ float one(const void* p, size_t i) { return bf16_to_f32(reinterpret_cast<const uint16_t*>(p)[i]); }
  static __device__ __forceinline__ float pick(u32x4 v, int i) {
    const uint32_t w = word_of(v, i >> 1);
    return i & 1 ? bf16_hi(w) : bf16_lo(w);
  }
};
struct LpF16 {};
template <>
struct LpType<LpF16> {
  static constexpr int PER = 8;
  static __device__ __forceinline__ void get(u32x4 v, float* f) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = f16_to_f32(w[i] & 0xFFFFu);
      f[2 * i + 1] = f16_to_f32(w[i] >> 16);
    }
  }
  static __device__ __forceinline__ float one(const void* p, size_t i) { return f16_to_f32(reinterpret_cast<const uint16_t*>(p)[i]); }
  static __device__ __forceinline__ float pick(u32x4 v, int i) {
    const uint32_t w = word_of(v, i >> 1);
    return f16_to_f32(i & 1 ? w >> 16 : w & 0xFFFFu);
  }
};

struct LpParams {
  const void* logits;       // rows of V values, `stride` values apart
  const int32_t* tokens;    // [M] or NULL
  float* logprobs;          // [M]
  float* entropy;           // [M] or NULL
  float* top_logprobs;      // [M, k]
  int32_t* top_ids;         // [M, k]
  LpState* part;            // [M][splits]
  u64* part_top;            // [M][splits][k]
  long long stride;
  int M, V, k, splits;
};

// The row's results from its state and (lane i < k) its i-th best key.
__device__ __forceinline__ void lp_finish(const LpParams& p, int row, LpState st, float x_t, bool in_range, u64 best, int lane) {
  const float logz = logf(st.z);
  if (lane == 0) {
    if (p.logprobs) p.logprobs[row] = in_range ? (x_t - st.m) - logz : 0.0f;
    if (p.entropy) p.entropy[row] = logz - st.t / st.z * LN2;
  }
  if (lane < p.k) {
    p.top_logprobs[(size_t)row * p.k + lane] = (lp_value(best) - st.m) - logz;
    p.top_ids[(size_t)row * p.k + lane] = (int32_t)(0xFFFFFFFFu - (uint32_t)best);
  }
}

// One workgroup a (row, part of the row); waves take 16-byte pieces in turn, LP_UNROLL of them a
// lane in flight, and keep their own state and best list; both meet in LDS.  A wave's list
// starts as its lanes' largest values of the first pieces, in order; after that it looks at a
// piece's order only where a lane's largest value passes the k-th best of its own list and of
// the other waves' (which only grow, so an older one of them is as good).  2043 rows of 151936
// fp32 logits, 20 best: 225-238 us, 5.2-5.5 TB/s (a bulk read reaches 6.7), 217 without lists: VALU
// instructions in 87 % of a SIMD's cycles beside memory.  416 bf16 or fp16 rows: 32.5 us without best lists,
// 51-54 with 8 (7 of them the merge): VALU instructions, 83 % of a SIMD's cycles.
// Measured and dropped: twice the pieces on their way (1-14 % slower), lists of the waves joined by
// rank (2 %), fewer and longer parts (3-10 %).
template <typename T>
__global__ __launch_bounds__(LP_THREADS) void token_logprobs_kernel(const LpParams p) {
  using Ty = LpType<T>;
  constexpr int PER = Ty::PER;
  constexpr int SIZE = 16 / PER;
  const int row = blockIdx.x / p.splits;
  const int part = blockIdx.x - row * p.splits;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const char* const base = reinterpret_cast<const char*>(p.logits) + (size_t)row * p.stride * SIZE;
  // the row from its first 16-byte boundary on in whole pieces; up to PER - 1 values before and behind
  const int head = min((int)((16 - ((uintptr_t)base & 15)) & 15) / SIZE, p.V);
  const int pieces = (p.V - head) / PER;
  const int p0 = (int)((long long)pieces * part / p.splits), p1 = (int)((long long)pieces * (part + 1) / p.splits);
  const char* const src = base + (size_t)head * SIZE;

  LpState st{-INFINITY, 0.0f, 0.0f};
  LpTop top;
  // values v[0 .. n) of this lane (unused ones -inf, whose weight is 0); returns their maximum,
  // NaN where one is NaN
  auto add = [&](const float* v, int n) __attribute__((always_inline)) {
    float mx = v[0];
    for (int i = 1; i < n; ++i) mx = __builtin_elementwise_maximum(mx, v[i]);
    if (!(mx <= st.m + LP_SLACK)) {
      const float d = st.m > -INFINITY ? (st.m - mx) * LOG2E : mx != mx ? mx : -1e30f;   // z and t are 0 at first
      const float f = exp2_fast(d);
      st.t = (st.t + fmaxf(d, -1e30f) * st.z) * f;
      st.z *= f;
      st.m = mx;
    }
    const float ms = st.m > -INFINITY ? st.m : 0.0f;
    for (int i = 0; i < n; ++i) {
      const float y = fmaxf((v[i] - ms) * LOG2E, -200.0f);   // 2^-200 is 0: a finite number times no weight
      const float e = exp2_fast(y);
      st.z += e;
      st.t = fmaf(e, y, st.t);
    }
    return mx;
  };
  __shared__ float s_floor[LP_WAVES];
  if (lane == 0) s_floor[wave] = -INFINITY;
  __syncthreads();
  const int first = p0 + wave * 64 * LP_UNROLL;
  u32x4 ahead[LP_UNROLL];                      // the next pieces, on their way
  const auto load = [&](int q) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < LP_UNROLL; ++u)
      ahead[u] = *reinterpret_cast<const u32x4*>(src + (size_t)min(q + 64 * u + lane, p1 - 1) * 16);
  };
  if (first < p1) load(first);
  for (int q = first; q < p1; q += LP_WAVES * 64 * LP_UNROLL) {
    u32x4 raw[LP_UNROLL];
#pragma unroll
    for (int u = 0; u < LP_UNROLL; ++u) raw[u] = ahead[u];
    if (q + LP_WAVES * 64 * LP_UNROLL < p1) load(q + LP_WAVES * 64 * LP_UNROLL);
    u64 start = 0;                             // the lane's key that the list started with
    if (p.k && q == first) {
      float mx = -INFINITY;
      int at = -1;
#pragma unroll
      for (int u = 0; u < LP_UNROLL; ++u) {
        const int piece = q + 64 * u + lane;
        float v[PER];
        Ty::get(raw[u], v);
#pragma unroll
        for (int i = 0; i < PER; ++i)
          if (piece < p1 && (at < 0 || v[i] > mx || (v[i] != v[i] && mx == mx))) {
            mx = v[i];
            at = head + piece * PER + i;
          }
      }
      start = at < 0 ? (u64)(64 - lane) : lp_key(mx, at);
      top.fill(start, p.k);
    }
    float others = -INFINITY;
#pragma unroll
    for (int w = 0; w < LP_WAVES; ++w)
      others = fmaxf(others, __hip_atomic_load(&s_floor[w], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP));
    const float floor0 = top.floor;
    const bool full = q + 64 * LP_UNROLL <= p1;
#pragma unroll
    for (int u = 0; u < LP_UNROLL; ++u) {
      const int piece = q + 64 * u + lane;
      float v[PER];
      Ty::get(raw[u], v);
      if (!full) {                             // uniform
#pragma unroll
        for (int i = 0; i < PER; ++i) v[i] = piece < p1 ? v[i] : -INFINITY;
      }
      const float mx = add(v, PER);
      // a NaN passes; a value equal to the k-th best (a NaN where that is one) counts only beside
      // values that the list already holds from this piece, or at the start from later ones: others
      // stand behind it (2043 fp32 rows of nothing but NaN: 235 us, without this 3293)
      if (p.k) {
        const bool nan = top.last >> 32 == 0xFFFFFFFFu;
        u64 hit = __ballot(piece < p1 && !(mx < top.floor || ((mx == top.floor || nan) && !start) || mx < others));
        if (hit && q == first) {               // many lanes, at the start: value by value over all of them
#pragma unroll
          for (int i = 0; i < PER; ++i)
            if (__ballot(piece < p1 && !(v[i] < top.floor))) {
              const u64 key = lp_key(v[i], head + piece * PER + i);
              top.take(piece < p1 && key != start ? key : 0, p.k, lane);   // start is in the list
            }
          hit = 0;
        }
        for (; hit; hit &= hit - 1) {          // lane by lane: the values of its piece, one a lane
          const int from = __builtin_ctzll(hit);
          const u32x4 w = u32x4{(uint32_t)__builtin_amdgcn_readlane(raw[u].x, from), (uint32_t)__builtin_amdgcn_readlane(raw[u].y, from),
                                (uint32_t)__builtin_amdgcn_readlane(raw[u].z, from), (uint32_t)__builtin_amdgcn_readlane(raw[u].w, from)};
          top.take(lane < PER ? lp_key(Ty::pick(w, lane), head + (q + 64 * u + from) * PER + lane) : 0, p.k, lane);
        }
      }
    }
    if (p.k && lane == 0 && top.floor != floor0 && top.floor == top.floor)
      __hip_atomic_store(&s_floor[wave], top.floor, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
  }
  // the values outside the pieces: the first part's, by the first wave
  if (part == 0 && wave == 0) {
    const int tail = head + pieces * PER;      // lanes below 32: before the pieces, others behind
    const int i = lane < 32 ? lane : tail + lane - 32;
    const bool in = lane < 32 ? lane < head : i < p.V;
    const float v = in ? Ty::one(base, i) : -INFINITY;
    (void)add(&v, 1);
    if (p.k) top.take(in ? lp_key(v, i) : 0, p.k, lane);
  }

  // ---- lanes, then waves ----
#pragma unroll
  for (int s = 32; s; s >>= 1) st = lp_join(st, LpState{__shfl_xor(st.m, s, 64), __shfl_xor(st.z, s, 64), __shfl_xor(st.t, s, 64)});
  __shared__ LpState s_state[LP_WAVES];
  __shared__ u64 s_top[LP_WAVES][LP_TOP];
  if (lane == 0) s_state[wave] = st;
  if (lane < p.k) s_top[wave][lane] = top.list;
  __syncthreads();
  if (wave) return;
  for (int w = 1; w < LP_WAVES; ++w) {
    st = lp_join(st, s_state[w]);
    if (p.k) top.take(lane < p.k ? s_top[w][lane] : 0, p.k, lane);
  }
  if (p.splits > 1) {
    const size_t at = (size_t)row * p.splits + part;
    if (lane == 0) p.part[at] = st;
    if (lane < p.k) p.part_top[at * p.k + lane] = top.list;
    return;
  }
  const int t = p.tokens ? p.tokens[row] : -1;
  const bool in = t >= 0 && t < p.V;
  lp_finish(p, row, st, in ? Ty::one(base, t) : 0.0f, in, top.list, lane);
}

// The parts of a row joined: one wave a row, a lane every 64th part, then the lanes.
template <typename T>
__global__ __launch_bounds__(64) void token_logprobs_merge_kernel(const LpParams p) {
  using Ty = LpType<T>;
  const int row = blockIdx.x, lane = threadIdx.x;
  LpState st{-INFINITY, 0.0f, 0.0f};
  for (int s = lane; s < p.splits; s += 64) st = lp_join(st, p.part[(size_t)row * p.splits + s]);
#pragma unroll
  for (int s = 32; s; s >>= 1) st = lp_join(st, LpState{__shfl_xor(st.m, s, 64), __shfl_xor(st.z, s, 64), __shfl_xor(st.t, s, 64)});
  LpTop top;
  const u64* keys = p.part_top + (size_t)row * p.splits * p.k;
  // entry i of every part's list before entry i + 1 of any: the best come first, and where no
  // list's entry i belongs here none behind it does
  for (int i = 0; i < p.k; ++i) {
    bool some = false;
    for (int s0 = 0; s0 < p.splits; s0 += 64) {
      const u64 key = s0 + lane < p.splits ? keys[(size_t)(s0 + lane) * p.k + i] : 0;
      if (i == 0 && s0 == 0) {
        top.fill(key >> 32 ? key : (u64)(64 - lane), p.k);
        some = true;
      } else if (__ballot(key > top.last)) {
        top.take(key, p.k, lane);
        some = true;
      }
    }
    if (!some) break;
  }
  const char* const base = reinterpret_cast<const char*>(p.logits) + (size_t)row * p.stride * (16 / Ty::PER);
  const int t = p.tokens ? p.tokens[row] : -1;
  const bool in = t >= 0 && t < p.V;
  lp_finish(p, row, st, in ? Ty::one(base, t) : 0.0f, in, top.list, lane);
}

}  // namespace t2i

using t2i_host::fail;

namespace {

// Parts of a row: workgroups for four a CU in all, each with at least 2048 values.
int lp_splits(int M, int V) { return std::max(1, std::min((1024 + M - 1) / M, std::min(V / 2048, 256))); }

size_t lp_bytes(int M, int splits, int k) {
  return splits < 2 ? 0 : (size_t)M * splits * (((sizeof(t2i::LpState) + 4) & ~(size_t)7) + (size_t)k * sizeof(t2i::u64));
}

}  // namespace

extern "C" size_t t2i_token_logprobs_workspace_bytes(int32_t M, int32_t V, int32_t top_k) {
  if (M < 1 || V < 1 || top_k < 0 || top_k > t2i::LP_TOP) return 0;
  return lp_bytes(M, lp_splits(M, V), top_k);
}

extern "C" int t2i_token_logprobs(const void* logits, int32_t logits_type, int64_t row_stride, int32_t M, int32_t V,
                                  const int32_t* tokens, int32_t top_k, float* logprobs, float* entropy,
                                  float* top_logprobs, int32_t* top_ids, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  if (!logits || (tokens && !logprobs) || (top_k > 0 && (!top_logprobs || !top_ids)))
    return fail(T2I_ERR_NULL, "token_logprobs pointers must not be NULL");
  if (logits_type < T2I_LOGITS_FP32 || logits_type > T2I_LOGITS_FP16) return fail(T2I_ERR_VALUE, "logits_type %d unknown", logits_type);
  if (M < 1 || V < 1 || row_stride < V) return fail(T2I_ERR_SHAPE, "M=%d V=%d row stride %lld invalid", M, V, (long long)row_stride);
  if (top_k < 0 || top_k > t2i::LP_TOP || top_k > V) return fail(T2I_ERR_VALUE, "top_k=%d must be 0 to %d, at most V", top_k, t2i::LP_TOP);
  const uintptr_t size = logits_type == T2I_LOGITS_FP32 ? 4 : 2;
  if (((uintptr_t)logits % size) || (((uintptr_t)tokens | (uintptr_t)logprobs | (uintptr_t)entropy | (uintptr_t)top_logprobs | (uintptr_t)top_ids) & 3u))
    return fail(T2I_ERR_ALIGN, "token_logprobs arrays must be aligned to their values");
  const int splits = lp_splits(M, V);
  if ((long long)M * splits > 0xFFFFFFFFLL / t2i::LP_THREADS) return fail(T2I_ERR_SHAPE, "M=%d exceeds the grid", M);
  const size_t need = lp_bytes(M, splits, top_k);
  if (need && (!workspace || workspace_bytes < need)) return fail(T2I_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : 0, need);
  if (need && !t2i_host::aligned16(workspace)) return fail(T2I_ERR_ALIGN, "the workspace must be 16-byte aligned");
  t2i::LpParams p{};
  p.logits = logits; p.tokens = tokens; p.logprobs = tokens ? logprobs : nullptr; p.entropy = entropy;
  p.top_logprobs = top_logprobs; p.top_ids = top_ids; p.stride = row_stride; p.M = M; p.V = V; p.k = top_k; p.splits = splits;
  if (need) {   // keys (8 bytes) first, then the states (4-byte values)
    p.part_top = reinterpret_cast<t2i::u64*>(workspace);
    p.part = reinterpret_cast<t2i::LpState*>(p.part_top + (size_t)M * splits * top_k);
  }
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define T2I_LP(ty)                                                                                                        \
  hipLaunchKernelGGL((t2i::token_logprobs_kernel<ty>), dim3(M * splits), dim3(t2i::LP_THREADS), 0, s, p);                 \
  if (int rc = t2i_host::hip_status(hipGetLastError(), "token_logprobs launch")) return rc;                               \
  if (!need) return T2I_OK;                                                                                               \
  hipLaunchKernelGGL((t2i::token_logprobs_merge_kernel<ty>), dim3(M), dim3(64), 0, s, p);                                 \
  return t2i_host::hip_status(hipGetLastError(), "token_logprobs merge launch")
  switch (logits_type) {
    case T2I_LOGITS_FP32: { T2I_LP(float); }
    case T2I_LOGITS_BF16: { T2I_LP(t2i::LpBf16); }
    default: { T2I_LP(t2i::LpF16); }
  }
#undef T2I_LP
}
