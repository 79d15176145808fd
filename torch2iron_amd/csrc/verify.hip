// Drafted tokens held to the model's probabilities with given random numbers, and the next token drawn, for
// gfx950 (t2i_verify_drafts).
//
// Row i of a sequence gives p_i = softmax(x_i / T).  The draft y behind it, taken from q_i, stays where u_i q_i(y) <
// p_i(y); behind the first that does not, the next token comes from max(p_i - q_i, 0), else from the last
// row's p: the first token whose running sum passes u times the whole sum.  Tokens come out distributed as the
// model's own.  T <= 0: p is 1 at the first maximum.
//
// All weights and sums are fp64: a running sum over 150k tokens has borders every 1e-5 and less, and with
// weights of fp32 (errors of 1e-7, added over the tokens of a tail) a draw in some hundred would fall on the other
// side of one.  fp64 instructions run at the rate of fp32's here, and a weight takes about twenty.
#include <math.h>

#include <algorithm>

#include "t2i_common.h"

namespace t2i {

constexpr int VD_CHUNK = 1024;               // tokens whose sum is kept: a wave's, sixteen a lane
constexpr int VD_WAVES = 4;
constexpr int VD_THREADS = 64 * VD_WAVES;

struct VdChunk {
  double z;                                  // sum of exp((x - m) / T)
  float m;                                   // the largest logit
  int best;                                  // T <= 0: its first place
};

// What was decided for a sequence whose refused draft has probabilities (else one kernel goes on with it).
struct VdChoice {
  double z;
  float m;
  int row, mode, best;
};
enum VdMode { VD_NONE, VD_BEST, VD_ALL, VD_WITHOUT, VD_REST };   // no token; the best; by p; by p without the draft; by max(p - q, 0)

struct VdParams {
  const void* logits;                        // rows of V values, `stride` apart
  const int32_t* row_starts;                 // [B + 1]
  const int32_t* tokens;                     // [M]
  const float* uniforms;                     // [M]
  const float* probs;                        // rows of V, `probs_stride` apart, or NULL
  const float* temperatures;                 // [B] or NULL (1)
  int32_t* counts;                           // [B]
  int32_t* next;                             // [B]
  float* logprobs;                           // [M]
  VdChunk* chunks;                           // [M][n_chunks]
  double* rest;                              // [B][n_chunks] sums of max(p - q, 0)
  VdChoice* choice;                          // [B]
  long long stride, probs_stride;
  int M, V, B, n_chunks, splits;
};

// 2^y for y <= 0 or so (fp64, relative error 1e-14): the whole part as an exponent, 2^f = e^(f ln 2) by its Taylor
// series (|f| <= 1/2: the first term left out is 0.347^12 / 12! = 6e-15).  Below 2^-1100 (and for -inf) 0; NaN stays.
__device__ __forceinline__ double exp2_f64(double y) {
  y = y < -1100.0 ? -1100.0 : y;
  const double n = __builtin_rint(y);
  const double t = (y - n) * 0.69314718055994530942;
  double p = 1.0 / 39916800.0;
  p = __builtin_fma(p, t, 1.0 / 3628800.0);
  p = __builtin_fma(p, t, 1.0 / 362880.0);
  p = __builtin_fma(p, t, 1.0 / 40320.0);
  p = __builtin_fma(p, t, 1.0 / 5040.0);
  p = __builtin_fma(p, t, 1.0 / 720.0);
  p = __builtin_fma(p, t, 1.0 / 120.0);
  p = __builtin_fma(p, t, 1.0 / 24.0);
  p = __builtin_fma(p, t, 1.0 / 6.0);
  p = __builtin_fma(p, t, 0.5);
  p = __builtin_fma(p, t, 1.0);
  p = __builtin_fma(p, t, 1.0);
  return __builtin_amdgcn_ldexp(p, (int)n);
}

// exp((x - m) / T) with c = log2(e) / T; 0 for a logit of -inf, whatever m and c are
__device__ __forceinline__ double vd_weight(float x, float m, double c) {
  return x == -INFINITY ? 0.0 : exp2_f64(((double)x - (double)m) * c);
}

// log2(e) / T; a temperature that is not above 0 (greedy) counts as 1 where probabilities are formed
__device__ __forceinline__ double vd_scale(float t) { return 1.44269504088896340736 / (t > 0.0f ? (double)t : 1.0); }

__device__ __forceinline__ double vd_wave_sum(double v) {
#pragma unroll
  for (int s = 32; s; s >>= 1) v += __shfl_xor(v, s, 64);
  return v;
}
__device__ __forceinline__ float vd_wave_max(float v) {
#pragma unroll
  for (int s = 32; s; s >>= 1) v = fmaxf(v, __shfl_xor(v, s, 64));
  return v;
}
__device__ __forceinline__ int vd_wave_min(int v) {
#pragma unroll
  for (int s = 32; s; s >>= 1) v = min(v, __shfl_xor(v, s, 64));
  return v;
}

// ---- logits of the three types: a lane's pieces of 16 bytes, at any alignment of the values ----
struct VdBf16 {};
struct VdF16 {};
template <typename T>
struct VdType;
template <>
struct VdType<float> {
  static constexpr int SIZE = 4;
  static __device__ __forceinline__ void get(u32x4 v, float* f) {
    f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ float one(const char* p) { return *reinterpret_cast<const float*>(p); }
};
template <>
struct VdType<VdBf16> {
  static constexpr int SIZE = 2;
  static __device__ __forceinline__ void get(u32x4 v, float* f) {
    float g[8];
    unpack8(v, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = g[i];
  }
  static __device__ __forceinline__ float one(const char* p) { return bf16_to_f32(*reinterpret_cast<const uint16_t*>(p)); }
};
template <>
struct VdType<VdF16> {
  static constexpr int SIZE = 2;
  static __device__ __forceinline__ void get(u32x4 v, float* f) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = f16_to_f32(w[i] & 0xFFFFu);
      f[2 * i + 1] = f16_to_f32(w[i] >> 16);
    }
  }
  static __device__ __forceinline__ float one(const char* p) { return f16_to_f32(*reinterpret_cast<const uint16_t*>(p)); }
};

// Values first .. first + N - 1 of a row of V (N a 16-byte piece's or a multiple), -inf behind its end.
typedef u32x4 u32x4_any __attribute__((aligned(2)));
template <typename T, int N>
__device__ __forceinline__ void vd_load(const char* row, int first, int V, float (&f)[N]) {
  constexpr int SIZE = VdType<T>::SIZE, PER = 16 / SIZE;
  const char* const at = row + (size_t)first * SIZE;
  if (first <= V - N) {
#pragma unroll
    for (int i = 0; i < N / PER; ++i) VdType<T>::get(*reinterpret_cast<const u32x4_any*>(at + 16 * i), f + PER * i);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = first + i < V ? VdType<T>::one(at + i * SIZE) : -INFINITY;
  }
}

template <typename T>
__device__ __forceinline__ const char* vd_row(const VdParams& p, int row) {
  return reinterpret_cast<const char*>(p.logits) + (size_t)row * p.stride * VdType<T>::SIZE;
}

// The rows of a sequence; none where they do not lie in the batch.
__device__ __forceinline__ int vd_rows(const VdParams& p, int b, int& first) {
  first = p.row_starts[b];
  const int end = p.row_starts[b + 1];
  return first >= 0 && first <= end && end <= p.M ? end - first : 0;
}

// ============================================================================
// largest value and sum of every chunk of every row
// ============================================================================
// A wave a chunk: its logits in one go, the maximum, then the weights.  Lane l holds the pieces l, l + 64, ...
template <typename T>
__global__ __launch_bounds__(VD_THREADS) void verify_rows_kernel(const VdParams p) {
  constexpr int PER = 16 / VdType<T>::SIZE, PIECES = VD_CHUNK / 64 / PER;
  __shared__ int s_seq;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = blockIdx.x / p.splits;
  const int chunk = (blockIdx.x - row * p.splits) * VD_WAVES + wave;
  const char* const src = vd_row<T>(p, row);
  float x[PIECES][PER];
  if (chunk < p.n_chunks) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) vd_load<T>(src, chunk * VD_CHUNK + (64 * i + lane) * PER, p.V, x[i]);
  }
  // the row's sequence, for its temperature
  float t = 1.0f;
  if (p.temperatures) {
    if (threadIdx.x == 0) s_seq = -1;
    __syncthreads();
    for (int b = threadIdx.x; b < p.B; b += VD_THREADS)
      if (p.row_starts[b] <= row && row < p.row_starts[b + 1]) s_seq = b;
    __syncthreads();
    if (s_seq >= 0) t = p.temperatures[s_seq];
  }
  if (chunk >= p.n_chunks) return;
  const double c = vd_scale(t);
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < PIECES; ++i)
#pragma unroll
    for (int j = 0; j < PER; ++j) m = fmaxf(m, x[i][j]);
  m = vd_wave_max(m);
  double z = 0.0;
#pragma unroll
  for (int i = 0; i < PIECES; ++i)
#pragma unroll
    for (int j = 0; j < PER; ++j) z += vd_weight(x[i][j], m, c);
  z = vd_wave_sum(z);
  int best = 0;
  if (!(t > 0.0f)) {
    best = 0x7FFFFFFF;
#pragma unroll
    for (int i = PIECES - 1; i >= 0; --i)
#pragma unroll
      for (int j = PER - 1; j >= 0; --j)
        if (x[i][j] == m) best = chunk * VD_CHUNK + (64 * i + lane) * PER + j;
    best = vd_wave_min(best);
  }
  if (lane == 0) p.chunks[(size_t)row * p.n_chunks + chunk] = VdChunk{z, m, best};
  if (threadIdx.x == 0 && chunk == 0) p.logprobs[row] = 0.0f;
}

// ============================================================================
// which drafts stay
// ============================================================================
// A row's largest logit and sum (a wave; every lane receives them), and the first place of the largest.
__device__ __forceinline__ void vd_join(const VdParams& p, int row, double c, int lane, float& m, double& z, int& best) {
  const VdChunk* const at = p.chunks + (size_t)row * p.n_chunks;
  m = -INFINITY;
  for (int i = lane; i < p.n_chunks; i += 64) m = fmaxf(m, at[i].m);
  m = vd_wave_max(m);
  z = 0.0;
  best = 0x7FFFFFFF;
  for (int i = lane; i < p.n_chunks; i += 64) {
    const VdChunk s = at[i];
    z += s.m > -INFINITY ? s.z * vd_weight(s.m, m, c) : s.z;   // (nothing but -inf: 0; NaN stays)
    if (s.m == m) best = min(best, s.best);
  }
  z = vd_wave_sum(z);
  best = vd_wave_min(best);
}

// A workgroup's decision for sequence b: what its next token is drawn by, from which row.  Waves take rows in turn;
// each remembers the first of its rows behind which no draft stays.  WRITE: the log probabilities of the drafts that stay.
template <typename T, bool WRITE>
__device__ __forceinline__ VdChoice vd_decide(const VdParams& p, int b, int* s_row, VdChoice* s_choice) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int first;
  const int n = vd_rows(p, b, first);
  const float t = p.temperatures ? p.temperatures[b] : 1.0f;
  const bool greedy = !(t > 0.0f);
  const double c = vd_scale(t);
  if (threadIdx.x == 0) {
    *s_row = first + n - 1;
    *s_choice = VdChoice{0.0, 0.0f, -1, VD_NONE, 0};
  }
  __syncthreads();
  VdChoice mine{0.0, 0.0f, -1, VD_NONE, 0};
  for (int row = first + wave; row < first + n && mine.row < 0; row += VD_WAVES) {
    float m;
    double z;
    int best;
    vd_join(p, row, c, lane, m, z, best);
    const bool fine = z > 0.0 && z < INFINITY;             // no NaN, no +inf, not all -inf
    bool stays = false;
    float lp = 0.0f;
    if (row + 1 < first + n) {
      const int y = p.tokens[row + 1];
      if (fine && y >= 0 && y < p.V) {
        const float x = VdType<T>::one(vd_row<T>(p, row) + (size_t)y * VdType<T>::SIZE);
        const double q = p.probs ? (double)p.probs[(size_t)row * p.probs_stride + y] : 1.0;
        stays = greedy ? y == best : (double)p.uniforms[row] * q < vd_weight(x, m, c) / z;
        lp = (float)(((double)x - (double)m) * c * 0.69314718055994530942 - log(z));
      }
    }
    if (stays) {
      if (WRITE && lane == 0) p.logprobs[row] = lp;
    } else {
      const bool last = row + 1 == first + n;
      mine = VdChoice{z, m, row, !fine ? VD_NONE : greedy ? VD_BEST : last ? VD_ALL : p.probs ? VD_REST : VD_WITHOUT, best};
      if (lane == 0) atomicMin(s_row, row);
    }
  }
  __syncthreads();
  if (mine.row >= 0 && mine.row == *s_row && lane == 0) *s_choice = mine;
  __syncthreads();
  const VdChoice out = *s_choice;
  if (WRITE) {
    for (int row = out.row + 1 + (int)threadIdx.x; row < first + n; row += VD_THREADS) p.logprobs[row] = 0.0f;
    if (threadIdx.x == 0) p.counts[b] = out.row < 0 ? 0 : out.row - first;
  }
  return out;
}

// The weights by which a token is drawn.
struct VdWeights {
  double c, inv_z;
  float m;
  int mode, without;
  const float* q;                            // VD_REST: the row of draft probabilities
  __device__ __forceinline__ double of(float x, int at) const {
    const double e = vd_weight(x, m, c);
    if (mode == VD_REST) {
      const double w = e * inv_z - (double)q[at];
      return w > 0.0 ? w : 0.0;
    }
    return mode == VD_WITHOUT && at == without ? 0.0 : e;
  }
};

// The weights of a chunk of a row, four neighbouring tokens a thread of VD_THREADS.
template <typename T>
__device__ __forceinline__ void vd_four(const VdParams& p, const char* row, int chunk, const VdWeights& w, double (&v)[4]) {
  const int first = chunk * VD_CHUNK + 4 * (int)threadIdx.x;
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = first + j < p.V ? w.of(VdType<T>::one(row + (size_t)(first + j) * VdType<T>::SIZE), first + j) : 0.0;
}

// Sums over the workgroup: those of the threads before this one, and all.
__device__ __forceinline__ double vd_scan(double v, double* s_wave, double& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double x = v;
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const double u = __shfl_up(x, s, 64);
    if (lane >= s) x += u;
  }
  __syncthreads();
  if (lane == 63) s_wave[wave] = x;
  __syncthreads();
  double before = 0.0;
  all = 0.0;
  for (int w = 0; w < VD_WAVES; ++w) {
    if (w < wave) before += s_wave[w];
    all += s_wave[w];
  }
  const double up = __shfl_up(x, 1, 64);
  return before + (lane ? up : 0.0);
}

// The next token of sequence b, from what was decided: first the chunk, then the token within it.
template <typename T>
__device__ __forceinline__ void vd_pick(const VdParams& p, int b, VdChoice ch) {
  __shared__ double s_wave[VD_WAVES];
  __shared__ double s_before;
  __shared__ int s_chunk, s_last, s_token, s_some;
  int first;
  const int n = vd_rows(p, b, first);
  if (ch.mode == VD_NONE || ch.mode == VD_BEST) {          // (no rows: ch.row is -1)
    if (threadIdx.x == 0) {
      p.next[b] = ch.mode == VD_BEST ? ch.best : -1;
      if (ch.row >= 0) p.logprobs[ch.row] = ch.mode == VD_BEST ? (float)-log(ch.z) : __uint_as_float(0x7FC00000u);
    }
    return;
  }
  const char* const row = vd_row<T>(p, ch.row);
  VdWeights w;
  w.c = vd_scale(p.temperatures ? p.temperatures[b] : 1.0f);
  w.inv_z = 1.0 / ch.z;
  w.m = ch.m;
  w.mode = ch.mode;
  w.without = ch.row + 1 < first + n ? p.tokens[ch.row + 1] : -1;
  w.q = p.probs ? p.probs + (size_t)ch.row * p.probs_stride : nullptr;
  const VdChunk* const chunks = p.chunks + (size_t)ch.row * p.n_chunks;
  double without = 0.0, total = 0.0;
  const int odd = w.mode == VD_WITHOUT && w.without >= 0 && w.without < p.V ? w.without / VD_CHUNK : -1;
  if (odd >= 0) {                                          // the draft's own chunk, without it
    double v[4];
    vd_four<T>(p, row, odd, w, v);
    (void)vd_scan((v[0] + v[1]) + (v[2] + v[3]), s_wave, without);
  }
  const auto sum_of = [&](int i) {
    if (i >= p.n_chunks) return 0.0;
    if (w.mode == VD_REST) return p.rest[(size_t)b * p.n_chunks + i];
    return i == odd && w.mode == VD_WITHOUT ? without : chunks[i].m > -INFINITY ? chunks[i].z * vd_weight(chunks[i].m, w.m, w.c) : 0.0;
  };
  for (;;) {
    total = 0.0;
    for (int base = 0; base < p.n_chunks; base += VD_THREADS) {
      double all;
      (void)vd_scan(sum_of(base + threadIdx.x), s_wave, all);
      total += all;
    }
    if (total > 0.0 || w.mode == VD_ALL) break;
    w.mode = VD_ALL;                                       // nothing is left: by p itself
  }
  if (threadIdx.x == 0) {
    s_chunk = s_token = 0x7FFFFFFF;
    s_last = s_some = -1;
  }
  __syncthreads();
  const double target = (double)p.uniforms[first + n - 1] * total;
  double before = 0.0;
  for (int base = 0; base < p.n_chunks; base += VD_THREADS) {
    const int i = base + threadIdx.x;
    const double v = sum_of(i);
    double all;
    const double upto = before + vd_scan(v, s_wave, all);
    if (v > 0.0 && upto + v > target) atomicMin(&s_chunk, i);
    if (v > 0.0) atomicMax(&s_last, i);
    before += all;
    __syncthreads();
    if (s_chunk == i) s_before = upto;
    __syncthreads();
    if (s_chunk < 0x7FFFFFFF) break;
    if (s_last == i) s_before = upto;                      // u of 1 or more: the last token with a weight
    __syncthreads();
  }
  __syncthreads();
  const int chunk = s_chunk < 0x7FFFFFFF ? s_chunk : s_last;
  const double start = s_before;
  if (chunk < 0) {                                         // (a NaN among the draft's probabilities)
    if (threadIdx.x == 0) p.next[b] = -1;
    return;
  }
  double v[4], all;
  vd_four<T>(p, row, chunk, w, v);
  double upto = start + vd_scan((v[0] + v[1]) + (v[2] + v[3]), s_wave, all);
  const int at = chunk * VD_CHUNK + 4 * (int)threadIdx.x;
  bool found = false;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    upto += v[j];
    if (v[j] > 0.0) {
      if (!found && upto > target) atomicMin(&s_token, at + j), found = true;
      atomicMax(&s_some, at + j);
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    const int token = s_token < 0x7FFFFFFF ? s_token : s_some;
    p.next[b] = token;
    const float x = token >= 0 ? VdType<T>::one(row + (size_t)token * VdType<T>::SIZE) : 0.0f;
    p.logprobs[ch.row] = (float)(((double)x - (double)ch.m) * w.c * 0.69314718055994530942 - log(ch.z));
  }
}

// No draft probabilities: everything behind the rows' sums, a workgroup a sequence.
template <typename T>
__global__ __launch_bounds__(VD_THREADS) void verify_kernel(const VdParams p) {
  __shared__ int s_row;
  __shared__ VdChoice s_choice;
  const VdChoice ch = vd_decide<T, true>(p, blockIdx.x, &s_row, &s_choice);
  __syncthreads();
  vd_pick<T>(p, blockIdx.x, ch);
}

// With draft probabilities: first each chunk's sum of max(p - q, 0) behind a refused draft, `splits` workgroups a sequence
// (each decides for itself; the first writes it down), a wave a chunk.
template <typename T>
__global__ __launch_bounds__(VD_THREADS) void verify_rest_kernel(const VdParams p) {
  __shared__ int s_row;
  __shared__ VdChoice s_choice;
  const int b = blockIdx.x / p.splits, split = blockIdx.x - b * p.splits;
  VdChoice ch;
  if (split == 0) {
    ch = vd_decide<T, true>(p, b, &s_row, &s_choice);
    if (threadIdx.x == 0) p.choice[b] = ch;
  } else {
    ch = vd_decide<T, false>(p, b, &s_row, &s_choice);
  }
  if (ch.mode != VD_REST) return;
  constexpr int PER = 16 / VdType<T>::SIZE, PIECES = VD_CHUNK / 64 / PER;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const double c = vd_scale(p.temperatures ? p.temperatures[b] : 1.0f), inv_z = 1.0 / ch.z;
  const char* const row = vd_row<T>(p, ch.row);
  const float* const q = p.probs + (size_t)ch.row * p.probs_stride;
  for (int chunk = split * VD_WAVES + wave; chunk < p.n_chunks; chunk += p.splits * VD_WAVES) {
    double z = 0.0;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int first = chunk * VD_CHUNK + (64 * i + lane) * PER;
      float x[PER], y[PER];
      vd_load<T>(row, first, p.V, x);
      vd_load<float>(reinterpret_cast<const char*>(q), first, p.V, y);
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const double w = vd_weight(x[j], ch.m, c) * inv_z - (double)y[j];
        z += first + j < p.V && w > 0.0 ? w : 0.0;
      }
    }
    z = vd_wave_sum(z);
    if (lane == 0) p.rest[(size_t)b * p.n_chunks + chunk] = z;
  }
}
template <typename T>
__global__ __launch_bounds__(VD_THREADS) void verify_pick_kernel(const VdParams p) {
  vd_pick<T>(p, blockIdx.x, p.choice[blockIdx.x]);
}

}  // namespace t2i

using t2i_host::fail;

namespace {

int vd_chunks(int V) { return (int)(((long long)V + t2i::VD_CHUNK - 1) / t2i::VD_CHUNK); }

size_t vd_bytes(int M, int V, int B, bool probs) {
  const size_t n = vd_chunks(V);
  return (size_t)M * n * sizeof(t2i::VdChunk) + (probs ? (size_t)B * (n * sizeof(double) + sizeof(t2i::VdChoice)) : 0);
}

}  // namespace

extern "C" size_t t2i_verify_drafts_workspace_bytes(int32_t M, int32_t V, int32_t n_seqs, int32_t with_probs) {
  return M < 1 || V < 1 || n_seqs < 1 ? 0 : vd_bytes(M, V, n_seqs, with_probs != 0);
}

extern "C" int t2i_verify_drafts(const void* logits, int32_t logits_type, int64_t row_stride, int32_t M, int32_t V,
                                 const int32_t* row_starts, int32_t n_seqs, const int32_t* tokens, const float* uniforms,
                                 const float* draft_probs, int64_t probs_stride, const float* temperatures,
                                 int32_t* counts, int32_t* next_tokens, float* logprobs, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  if (!logits || !row_starts || !tokens || !uniforms || !counts || !next_tokens || !logprobs)
    return fail(T2I_ERR_NULL, "verify_drafts pointers must not be NULL");
  if (logits_type < T2I_LOGITS_FP32 || logits_type > T2I_LOGITS_FP16) return fail(T2I_ERR_VALUE, "logits_type %d unknown", logits_type);
  if (M < 1 || V < 1 || n_seqs < 1 || row_stride < V || (draft_probs && probs_stride < V))
    return fail(T2I_ERR_SHAPE, "M=%d V=%d sequences=%d row strides %lld, %lld invalid", M, V, n_seqs, (long long)row_stride, (long long)probs_stride);
  const uintptr_t size = logits_type == T2I_LOGITS_FP32 ? 4 : 2;
  if (((uintptr_t)logits % size) ||
      (((uintptr_t)row_starts | (uintptr_t)tokens | (uintptr_t)uniforms | (uintptr_t)draft_probs | (uintptr_t)temperatures |
        (uintptr_t)counts | (uintptr_t)next_tokens | (uintptr_t)logprobs) & 3u))
    return fail(T2I_ERR_ALIGN, "verify_drafts arrays must be aligned to their values");
  t2i::VdParams p{};
  p.n_chunks = vd_chunks(V);
  p.splits = (p.n_chunks + t2i::VD_WAVES - 1) / t2i::VD_WAVES;
  if ((long long)M * p.splits > 0xFFFFFFFFLL / t2i::VD_THREADS || n_seqs > 1 << 20)
    return fail(T2I_ERR_SHAPE, "M=%d rows of %d logits, %d sequences exceed the grid", M, V, n_seqs);
  const size_t need = vd_bytes(M, V, n_seqs, draft_probs != nullptr);
  if (!workspace || workspace_bytes < need) return fail(T2I_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : 0, need);
  if (!t2i_host::aligned16(workspace)) return fail(T2I_ERR_ALIGN, "the workspace must be 16-byte aligned");
  p.logits = logits; p.row_starts = row_starts; p.tokens = tokens; p.uniforms = uniforms; p.probs = draft_probs;
  p.temperatures = temperatures; p.counts = counts; p.next = next_tokens; p.logprobs = logprobs;
  p.stride = row_stride; p.probs_stride = probs_stride; p.M = M; p.V = V; p.B = n_seqs;
  p.chunks = reinterpret_cast<t2i::VdChunk*>(workspace);
  p.choice = reinterpret_cast<t2i::VdChoice*>(p.chunks + (size_t)M * p.n_chunks);
  p.rest = reinterpret_cast<double*>(p.choice + (draft_probs ? n_seqs : 0));
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  // workgroups of a sequence's rest: about two a CU in all
  const int rest_splits = std::max(1, std::min(p.splits, (512 + n_seqs - 1) / n_seqs));
#define T2I_VD(ty)                                                                                                       \
  hipLaunchKernelGGL((t2i::verify_rows_kernel<ty>), dim3(M * p.splits), dim3(t2i::VD_THREADS), 0, s, p);                 \
  if (int rc = t2i_host::hip_status(hipGetLastError(), "verify_drafts launch")) return rc;                               \
  if (!draft_probs) {                                                                                                    \
    hipLaunchKernelGGL((t2i::verify_kernel<ty>), dim3(n_seqs), dim3(t2i::VD_THREADS), 0, s, p);                          \
    return t2i_host::hip_status(hipGetLastError(), "verify_drafts launch");                                              \
  }                                                                                                                      \
  p.splits = rest_splits;                                                                                                \
  hipLaunchKernelGGL((t2i::verify_rest_kernel<ty>), dim3(n_seqs * rest_splits), dim3(t2i::VD_THREADS), 0, s, p);         \
  if (int rc = t2i_host::hip_status(hipGetLastError(), "verify_drafts launch")) return rc;                               \
  hipLaunchKernelGGL((t2i::verify_pick_kernel<ty>), dim3(n_seqs), dim3(t2i::VD_THREADS), 0, s, p);                       \
  return t2i_host::hip_status(hipGetLastError(), "verify_drafts launch")
  switch (logits_type) {
    case T2I_LOGITS_FP32: { T2I_VD(float); }
    case T2I_LOGITS_BF16: { T2I_VD(t2i::VdBf16); }
    default: { T2I_VD(t2i::VdF16); }
  }
#undef T2I_VD
}
