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
constexpr int VD_WAVES = 4;                  // waves of a workgroup over the rows
constexpr int VD_BLOCK = 1024;               // threads of a workgroup over a sequence: a thread a token of a chunk
constexpr int VD_HELD = 4;                   // chunks of a lane that stay in registers: rows of up to 262144 tokens

struct VdChunk {
  double z;                                  // sum of exp((x - m) / T)
  float m;                                   // the largest logit
  int best;                                  // T <= 0: its first place
};

// What was decided for a sequence: the row that its next token comes from, by which weights, and all that the draw needs.
struct VdChoice {
  double c, inv_z, log_z;                    // the row's scale and sum
  double start, target;                      // the sum before the chunk, and the one that the token's has to pass
  float m, u;                                // its largest logit, the number for the draw
  int row, mode, best, draft, chunk;         // row -1: no rows; draft: the refused one (-1: none); chunk: -1 not found yet
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
  int M, V, B, n_chunks, splits;             // workgroups of a row (of a sequence)
};

// ---- exp((x - m) / T) in fp64 ----
// With y = (x - m) 256 log2(e) / T = 256 n + j + f (j of 0 .. 255, |f| <= 1/2): 2^n 2^(j / 256) 2^(f / 256), the second from a
// table in LDS, the third 1 + f times the quadratic of the smallest largest error there is (2.4e-14).  A third of the
// instructions of a series for 2^(y / 256 - n).  (A table of 32 with no bank twice and a degree more, 8e-14: 122 bf16 rows
// 24.9 -> 24.2 us, 432 of fp32 86.5 -> 84.)
constexpr int VD_EXP = 256, VD_LOG = 8;
constexpr double VD_P1 = 0.002707606174062412, VD_P2 = 3.665566060705425e-06, VD_P3 = 3.3083022204273407e-09;
__device__ __forceinline__ double vd_fraction(double f) {
  return __builtin_fma(__builtin_fma(__builtin_fma(VD_P3, f, VD_P2), f, VD_P1), f, 1.0);
}

// The table: s_exp[j] = 2^(j / 256) by the series of e^t (the first term left out is 0.7^17 / 17! = 7e-18), and s_add[j] the
// same with j 2^12 taken from its high word, so that 2^n comes with an addition.  A barrier behind it is the caller's.
__device__ __forceinline__ void vd_table(double* s_exp, double* s_add = nullptr) {
  if (threadIdx.x < VD_EXP) {
    const double t = (double)threadIdx.x * (0.69314718055994530942 / VD_EXP);
    double p = 1.0;
#pragma unroll
    for (int k = 16; k > 0; --k) p = __builtin_fma(p * t, 1.0 / k, 1.0);
    s_exp[threadIdx.x] = p;
    if (s_add) s_add[threadIdx.x] = __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, p) - ((uint64_t)threadIdx.x << (52 - VD_LOG)));
  }
}

// 2^(y / 256): 0 far below; an infinite y gives NaN.
__device__ __forceinline__ double vd_exp(double y, const double* s_exp) {
  const double k = __builtin_rint(y);
  int n;
  asm("v_cvt_i32_f64 %0, %1" : "=v"(n) : "v"(k));          // (saturates)
  return __builtin_amdgcn_ldexp(vd_fraction(y - k) * s_exp[n & (VD_EXP - 1)], n >> VD_LOG);
}

// z + 2^(d c / 256), for a row's sums: -2^18 < d c < 2^20.  The whole part k = 256 n + j comes out of the low bits of
// d c + 1.5 2^52, and k 2^12, added to the high word of the table's value, is j 2^12 + n 2^20: n more in its exponent.
// The constants stay in registers (an instruction takes one from elsewhere, and copies would be a tenth of all).
struct VdAdd {
  double c, whole, p[3];
  const u32x2* table;
  __device__ __forceinline__ VdAdd(double scale, const double* s_add) : c(scale), whole(6755399441055744.0), p{VD_P3, VD_P2, VD_P1} {
    table = reinterpret_cast<const u32x2*>(s_add);
    asm("" : "+v"(c), "+v"(whole), "+v"(p[0]), "+v"(p[1]), "+v"(p[2]));
  }
  __device__ __forceinline__ double operator()(double d, double z) const {
    const double s = __builtin_fma(d, c, whole);
    const double f = __builtin_fma(d, c, whole - s);
    const uint32_t k = __builtin_bit_cast(u32x2, s).x;
    u32x2 e = table[k & (VD_EXP - 1)];
    e.y += k << (20 - VD_LOG);
    double v = __builtin_fma(p[0], f, p[1]);
    v = __builtin_fma(v, f, p[2]);
    v = __builtin_fma(v, f, 1.0);
    return __builtin_fma(v, __builtin_bit_cast(double, e), z);
  }
};

// exp((x - m) / T) with c = 256 log2(e) / T; 0 for a logit of -inf, whatever m and c are
__device__ __forceinline__ double vd_weight(float x, float m, double c, const double* s_exp) {
  const double w = vd_exp(((double)x - (double)m) * c, s_exp);
  return x == -INFINITY ? 0.0 : w;
}

// 256 log2(e) / T; a temperature that is not above 0 (greedy) counts as 1 where probabilities are formed
__device__ __forceinline__ double vd_scale(float t) { return VD_EXP * 1.44269504088896340736 / (t > 0.0f ? (double)t : 1.0); }
// log p of a logit x, given the row's m and z
__device__ __forceinline__ float vd_logprob(float x, float m, double c, double log_z) {
  return (float)(((double)x - (double)m) * c * (0.69314718055994530942 / VD_EXP) - log_z);
}

// ---- sums, maxima and minima of a wave, in every lane ----
template <int CTRL, int ROWS>
__device__ __forceinline__ double vd_shift(double v) {     // 0 where there is no lane to take from
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, ROWS, 0xF, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, ROWS, 0xF, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// the sum of the lanes up to this one
__device__ __forceinline__ double vd_upto(double v) {
  v += vd_shift<0x111, 0xF>(v);              // row_shr 1, 2, 4, 8: within 16 lanes
  v += vd_shift<0x112, 0xF>(v);
  v += vd_shift<0x114, 0xF>(v);
  v += vd_shift<0x118, 0xF>(v);
  v += vd_shift<0x142, 0xA>(v);              // row_bcast 15: into rows 1 and 3
  v += vd_shift<0x143, 0xC>(v);              // row_bcast 31: into rows 2 and 3
  return v;
}
__device__ __forceinline__ double vd_lane(double v, int lane) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  return __builtin_bit_cast(double, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), lane) << 32 |
                                        (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, lane));
}
__device__ __forceinline__ double vd_wave_sum(double v) { return vd_lane(vd_upto(v), 63); }
__device__ __forceinline__ float vd_wave_max(float v) {
  v = row_max16(v);
  return fmaxf(fmaxf(__int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 0)), __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 16))),
               fmaxf(__int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 32)), __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 48))));
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

// The rows of a sequence, none where they do not lie in the batch.
__device__ __forceinline__ int vd_rows(const VdParams& p, int b, int& first) {
  first = p.row_starts[b];
  const int end = p.row_starts[b + 1];
  return first >= 0 && first <= end && end <= p.M ? end - first : 0;
}

// ============================================================================
// largest value and sum of every chunk of every row
// ============================================================================
// A wave takes every step-th chunk of a row, the next one's logits on their way while it adds the weights of one: the largest
// logit first, then the weights.  Lane l holds the pieces l, l + 64, ... of a chunk (16 bytes, at any alignment of the values).
// 122 rows of 151936 bf16 logits 16-17 us (37 MB, VALU 81 % of a SIMD's cycles at 1.9 GHz), 432 of fp32 56 (262 MB,
// 4.7 TB/s, VALU 78 %).
// Without the weights it takes 11 and 48 us: launch, a wave's first loads, the reductions.  No difference to the largest
// logit (an instruction of 20 less) gained nothing; chunks two ahead (25.9 us for the whole call) and five waves a SIMD (93
// for 83 us of fp32) lost.
template <typename T>
__global__ __launch_bounds__(64 * VD_WAVES) void verify_rows_kernel(const VdParams p) {
  constexpr int PER = 16 / VdType<T>::SIZE, PIECES = VD_CHUNK / 64 / PER;
  __shared__ double s_exp[VD_EXP], s_add[VD_EXP];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = blockIdx.x / p.splits;
  const int from = (blockIdx.x - row * p.splits) * VD_WAVES + wave, step = p.splits * VD_WAVES;   // all waves side by side
  const int whole = p.V / VD_CHUNK;                        // chunks that lie in the row to their end
  const char* const src = vd_row<T>(p, row) + (size_t)lane * 16;
  u32x4 next[PIECES];
  const auto fetch = [&](int chunk) {
    if (chunk < whole) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i)
        next[i] = *reinterpret_cast<const u32x4_any*>(src + (size_t)chunk * (VD_CHUNK * VdType<T>::SIZE) + 1024 * i);
    }
  };
  fetch(from);
  // the row's sequence, for its temperature: the last that starts at the row or before it
  float t = 1.0f;
  if (p.temperatures) {
    int s = -1;
    for (int base = 0; base < p.B; base += 64)
      s += __builtin_popcountll(__ballot(base + lane < p.B && p.row_starts[min(base + lane, p.B - 1)] <= row));
    if (s >= 0) t = p.temperatures[s];
  }
  vd_table(s_exp, s_add);
  __syncthreads();
  const double c = vd_scale(t);
  const VdAdd add(c, s_add);
  const float down = t > 0.0f ? 690.0f * t : 690.0f;       // 690 / ln 2 = 995.5 powers of two
  for (int chunk = from; chunk < p.n_chunks; chunk += step) {
    float x[PIECES][PER];
    if (chunk < whole) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) VdType<T>::get(next[i], x[i]);
    } else {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) vd_load<T>(vd_row<T>(p, row), chunk * VD_CHUNK + (64 * i + lane) * PER, p.V, x[i]);
    }
    fetch(chunk + step);
    float m = -INFINITY, low = INFINITY;
#pragma unroll
    for (int i = 0; i < PIECES; ++i)
#pragma unroll
      for (int j = 0; j < PER; j += 2) {
        m = fmaxf(fmaxf(x[i][j], x[i][j + 1]), m);
        low = fminf(fminf(x[i][j], x[i][j + 1]), low);
      }
    m = vd_wave_max(m);
    double z = 0.0;
    if (m < INFINITY && !__ballot(!(m - low < down)) && c < 1e6) {   // (a NaN makes z one)
      const double md = (double)m;
#pragma unroll
      for (int i = 0; i < PIECES; ++i)
#pragma unroll
        for (int j = 0; j < PER; ++j) z = add((double)x[i][j] - md, z);
    } else {                                               // masked tokens, the row's end, infinities; temperatures near 0
#pragma unroll
      for (int i = 0; i < PIECES; ++i)
#pragma unroll
        for (int j = 0; j < PER; ++j) z += vd_weight(x[i][j], m, c, s_exp);
    }
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
  }
  if (threadIdx.x == 0 && from == 0) p.logprobs[row] = 0.0f;
}

// ============================================================================
// which drafts stay
// ============================================================================
// A row's largest logit and sum (a wave; every lane receives them), and the first place of the largest; part: this lane's
// chunks (lane, lane + 64, ...) in units of the row's largest weight.
__device__ __forceinline__ void vd_join(const VdParams& p, int row, double c, const double* s_exp, bool greedy, int lane, float& m,
                                        double& z, int& best, double (&part)[VD_HELD]) {
  const VdChunk* const at = p.chunks + (size_t)row * p.n_chunks;
  VdChunk held[VD_HELD];
#pragma unroll
  for (int i = 0; i < VD_HELD; ++i) held[i] = at[min(64 * i + lane, p.n_chunks - 1)];
  m = -INFINITY;
#pragma unroll
  for (int i = 0; i < VD_HELD; ++i) m = fmaxf(m, held[i].m);
  for (int i = 64 * VD_HELD + lane; i < p.n_chunks; i += 64) m = fmaxf(m, at[i].m);
  m = vd_wave_max(m);
  double sum = 0.0;
  best = 0x7FFFFFFF;
  const auto add = [&](const VdChunk& s) {
    const double w = s.m > -INFINITY ? s.z * vd_weight(s.m, m, c, s_exp) : s.z;   // (nothing but -inf: 0; NaN stays)
    sum += w;
    if (s.m == m) best = min(best, s.best);
    return w;
  };
#pragma unroll
  for (int i = 0; i < VD_HELD; ++i) part[i] = 64 * i + lane < p.n_chunks ? add(held[i]) : 0.0;
  for (int i = 64 * VD_HELD + lane; i < p.n_chunks; i += 64) (void)add(at[i]);
  z = vd_wave_sum(sum);
  if (greedy) best = vd_wave_min(best);
}

// The chunk of the token that ch's number draws, by a wave that holds all the row's parts; left open where the draft's
// chunk holds hardly anything else (the difference would not be exact), or no chunk is found.
__device__ __forceinline__ void vd_chunk_of(VdChoice& ch, double (&part)[VD_HELD], double taken, int V, int lane) {
  bool open = false;
  double total = 0.0, upto[VD_HELD], before[VD_HELD];
#pragma unroll
  for (int i = 0; i < VD_HELD; ++i) {
    if (ch.mode == VD_WITHOUT && ch.draft >= 0 && ch.draft < V && ch.draft / VD_CHUNK == 64 * i + lane) {
      const double left = part[i] - taken;
      open = !(left > 1e-3 * part[i]);
      part[i] = left;
    }
    upto[i] = vd_upto(part[i]);
    before[i] = total;
    total += vd_lane(upto[i], 63);
  }
  if (__ballot(open) || !(total > 0.0)) return;
  const double target = (double)ch.u * total;
#pragma unroll
  for (int i = VD_HELD - 1; i >= 0; --i) {
    const unsigned long long hit = __ballot(part[i] > 0.0 && before[i] + upto[i] > target);
    if (!hit) continue;
    const int at = __builtin_ctzll(hit);
    ch.chunk = 64 * i + at;
    ch.start = at ? before[i] + vd_lane(upto[i], at - 1) : before[i];
    ch.target = target;
  }
}

// A workgroup's decision for sequence b: what its next token is drawn by, from which row (with the draw 6.3 us for 32
// sequences of four drafts: five loads that depend on each other).  Waves take rows in turn; each remembers the first of
// its rows behind which no draft stays, and its parts: where the token comes from p itself (or p without the draft) the
// wave of that row finds the chunk too, without another look at memory.  WRITE: the log probabilities of the drafts that
// stay.
template <typename T, bool WRITE>
__device__ __forceinline__ VdChoice vd_decide(const VdParams& p, int b, const double* s_exp, int* s_row, VdChoice* s_choice) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int first, falls = 0;                                    // row_starts that do not ascend: ranges could overlap
  for (int s = threadIdx.x; s < p.B; s += VD_BLOCK) falls |= p.row_starts[s] < 0 || p.row_starts[s] > p.row_starts[s + 1] || p.row_starts[s + 1] > p.M;
  int n = vd_rows(p, b, first);
  const float t = p.temperatures ? p.temperatures[b] : 1.0f;
  const float draw = n ? p.uniforms[first + n - 1] : 0.0f;
  const bool greedy = !(t > 0.0f);
  const double c = vd_scale(t);
  VdChoice mine{c, 0.0, 0.0, 0.0, 0.0, 0.0f, draw, -1, VD_NONE, 0, -1, -1};
  double part[VD_HELD] = {}, taken = 0.0;                  // of the row of `mine`; the draft's weight
  if (threadIdx.x == 0) {
    *s_row = first + n - 1;
    *s_choice = mine;
  }
  if (__syncthreads_or(falls)) n = 0;                      // (also the table's barrier)
  for (int row = first + wave; row < first + n && mine.row < 0; row += VD_BLOCK / 64) {
    const bool last = row + 1 == first + n;
    const int y = last ? -1 : p.tokens[row + 1];
    const bool in = y >= 0 && y < p.V;
    const float x = in ? VdType<T>::one(vd_row<T>(p, row) + (size_t)y * VdType<T>::SIZE) : 0.0f;
    const double q = in && p.probs ? (double)p.probs[(size_t)row * p.probs_stride + y] : 1.0;
    const double u = (double)p.uniforms[row];
    float m;
    double z;
    int best;
    vd_join(p, row, c, s_exp, greedy, lane, m, z, best, part);
    taken = in ? vd_weight(x, m, c, s_exp) : 0.0;
    const bool fine = z > 0.0 && z < INFINITY;             // no NaN, no +inf, not all -inf
    const bool stays = fine && in && (greedy ? y == best : u * q * z < taken);
    if (stays) {
      if (WRITE && lane == 0) p.logprobs[row] = vd_logprob(x, m, c, log(z));
    } else {
      mine = VdChoice{c, 1.0 / z, log(z), 0.0, 0.0, m, draw, row, !fine ? VD_NONE : greedy ? VD_BEST : last ? VD_ALL : p.probs ? VD_REST : VD_WITHOUT,
                      best, y, -1};
      if (lane == 0) atomicMin(s_row, row);                // (a lane a wave)
    }
  }
  __syncthreads();
  const int at = *s_row;
  if (mine.row >= 0 && mine.row == at) {
    if ((mine.mode == VD_ALL || mine.mode == VD_WITHOUT) && p.n_chunks <= 64 * VD_HELD) vd_chunk_of(mine, part, taken, p.V, lane);
    if (lane == 0) *s_choice = mine;
  }
  if (WRITE) {
    for (int row = at + 1 + (int)threadIdx.x; row < first + n; row += VD_BLOCK) p.logprobs[row] = 0.0f;
    if (threadIdx.x == 0) p.counts[b] = n ? at - first : 0;
  }
  __syncthreads();
  return *s_choice;
}

// The weights by which a token is drawn, in units of 1 / z where there are draft probabilities.
struct VdWeights {
  double c, inv_z;
  float m;
  int mode, without;
  const float* q;                            // VD_REST: the row of draft probabilities
  const double* s_exp;
  __device__ __forceinline__ double of(float x, int at) const {
    const double e = vd_weight(x, m, c, s_exp);
    if (mode == VD_REST) {
      const double w = e * inv_z - (double)q[at];
      return w > 0.0 ? w : 0.0;
    }
    return mode == VD_WITHOUT && at == without ? 0.0 : e;
  }
};

constexpr int VD_BLOCK_WAVES = VD_BLOCK / 64;

// Sums over the workgroup of VD_BLOCK: those of the threads before this one, and all.
__device__ __forceinline__ double vd_scan(double v, double* s_wave, double& all) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const double x = vd_upto(v);
  __syncthreads();
  if (lane == 63) s_wave[wave] = x;
  __syncthreads();
  // every wave's 16 lanes hold the waves' sums
  const double w = s_wave[lane & (VD_BLOCK_WAVES - 1)];
  const double up = vd_upto(lane < VD_BLOCK_WAVES ? w : 0.0);
  all = vd_lane(up, VD_BLOCK_WAVES - 1);
  const double before = wave ? vd_lane(up, wave - 1) : 0.0;
  return before + vd_shift<0x138, 0xF>(x);                 // wave_shr 1
}

// The first and the last thread of the workgroup of which `hit` and `some` hold (none: past every one, -1).
struct VdEnds {
  int first, last;
};
__device__ __forceinline__ VdEnds vd_ends(bool hit, bool some, int2* s_ends) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned long long h = __ballot(hit), s = __ballot(some);
  __syncthreads();                                         // the words of the call before are read
  if (lane == 0)
    s_ends[wave] = int2{h ? 64 * wave + __builtin_ctzll(h) : 0x7FFFFFFF, s ? 64 * wave + 63 - __builtin_clzll(s) : -1};
  __syncthreads();
  const int2 w = s_ends[lane & (VD_BLOCK_WAVES - 1)];
  const uint32_t f = (uint32_t)__ballot(lane < VD_BLOCK_WAVES && w.x < 0x7FFFFFFF);
  const uint32_t l = (uint32_t)__ballot(lane < VD_BLOCK_WAVES && w.y >= 0);
  return VdEnds{f ? __builtin_amdgcn_readlane(w.x, __builtin_ctz(f)) : 0x7FFFFFFF,
                l ? __builtin_amdgcn_readlane(w.y, 31 - __builtin_clz(l)) : -1};
}

// The next token of sequence b, from what was decided: first the chunk, then the token within it.
template <typename T>
__device__ __forceinline__ void vd_pick(const VdParams& p, int b, VdChoice ch, const double* s_exp) {
  __shared__ double s_wave[VD_BLOCK_WAVES];
  __shared__ double s_before;
  __shared__ int2 s_ends[VD_BLOCK_WAVES];
  if (ch.mode == VD_NONE || ch.mode == VD_BEST) {
    if (threadIdx.x == 0) {
      p.next[b] = ch.mode == VD_BEST ? ch.best : -1;
      if (ch.row >= 0) p.logprobs[ch.row] = ch.mode == VD_BEST ? (float)-ch.log_z : __uint_as_float(0x7FC00000u);
    }
    return;
  }
  const char* const row = vd_row<T>(p, ch.row);
  const VdChunk* const chunks = p.chunks + (size_t)ch.row * p.n_chunks;
  const double* const rest = p.rest + (size_t)b * p.n_chunks;
  VdWeights w;
  w.c = ch.c;
  w.inv_z = ch.inv_z;
  w.m = ch.m;
  w.mode = ch.mode;
  w.without = ch.draft;
  w.q = p.probs ? p.probs + (size_t)ch.row * p.probs_stride : nullptr;
  w.s_exp = s_exp;
  float x = 0.0f;                                          // the logit of this thread's token of a chunk
  const auto token_weight = [&](int chunk) {
    const int at = chunk * VD_CHUNK + (int)threadIdx.x;
    if (at >= p.V) return 0.0;
    x = VdType<T>::one(row + (size_t)at * VdType<T>::SIZE);
    return w.of(x, at);
  };
  int chunk = ch.chunk;
  double start = ch.start, target = ch.target;
  if (chunk < 0) {                                         // not found yet: from the sums of the chunks
    double without = 0.0;
    const int odd = w.mode == VD_WITHOUT && w.without >= 0 && w.without < p.V ? w.without / VD_CHUNK : -1;
    if (odd >= 0) (void)vd_scan(token_weight(odd), s_wave, without);   // the draft's own chunk, without it
    const auto sum_of = [&](int i) {
      if (i >= p.n_chunks) return 0.0;
      if (w.mode == VD_REST) return rest[i];
      const VdChunk s = chunks[i];
      return i == odd && w.mode == VD_WITHOUT ? without : s.m > -INFINITY ? s.z * vd_weight(s.m, w.m, w.c, s_exp) : 0.0;
    };
    double total, v = 0.0, upto = 0.0;                       // (rows of up to 2^20 tokens: one round, kept for the search)
    for (;;) {
      total = 0.0;
      for (int base = 0; base < p.n_chunks; base += VD_BLOCK) {
        double all;
        v = sum_of(base + threadIdx.x);
        upto = vd_scan(v, s_wave, all);
        total += all;
      }
      if (total > 0.0 || w.mode == VD_ALL) break;
      w.mode = VD_ALL;                                       // nothing is left: by p itself
    }
    target = (double)ch.u * total;
    double before = 0.0;
    for (int base = 0; base < p.n_chunks; base += VD_BLOCK) {
      double all = 0.0;
      if (p.n_chunks > VD_BLOCK) {
        v = sum_of(base + threadIdx.x);
        upto = before + vd_scan(v, s_wave, all);
      }
      const VdEnds e = vd_ends(v > 0.0 && upto + v > target, v > 0.0, s_ends);
      const int at = e.first < 0x7FFFFFFF ? e.first : e.last;   // a number of 1 or more: the last with a weight
      if (at >= 0) {
        chunk = base + at;
        if ((int)threadIdx.x == at) s_before = upto;
      }
      before += all;
      if (e.first < 0x7FFFFFFF) break;
    }
    if (chunk < 0) {                                       // (a NaN among the draft's probabilities)
      if (threadIdx.x == 0) {
        p.next[b] = -1;
        p.logprobs[ch.row] = __uint_as_float(0x7FC00000u);
      }
      return;
    }
    __syncthreads();
    start = s_before;
  }
  double all;
  const double mine = token_weight(chunk);
  const double to = start + vd_scan(mine, s_wave, all) + mine;
  const VdEnds e = vd_ends(mine > 0.0 && to > target, mine > 0.0, s_ends);
  const int at = e.first < 0x7FFFFFFF ? e.first : e.last;
  if ((int)threadIdx.x == max(at, 0)) {
    p.next[b] = at < 0 ? -1 : chunk * VD_CHUNK + at;
    p.logprobs[ch.row] = at < 0 ? __uint_as_float(0x7FC00000u) : vd_logprob(x, ch.m, w.c, ch.log_z);
  }
}

// Everything behind the rows' sums, a workgroup a sequence; but where a refused draft has probabilities only the
// decision, which the next two launches go on with.
template <typename T>
__global__ __launch_bounds__(VD_BLOCK) void verify_kernel(const VdParams p) {
  __shared__ double s_exp[VD_EXP];
  __shared__ int s_row;
  __shared__ VdChoice s_choice;
  vd_table(s_exp);
  const VdChoice ch = vd_decide<T, true>(p, blockIdx.x, s_exp, &s_row, &s_choice);
  if (p.probs && threadIdx.x == 0) p.choice[blockIdx.x] = ch;
  if (ch.mode != VD_REST) vd_pick<T>(p, blockIdx.x, ch, s_exp);
}

// Each chunk's sum of max(p - q, 0) behind a refused draft, `splits` workgroups a sequence, a wave a chunk (64 rows 12.5 us,
// the row and its draft probabilities, 52 MB: one chunk's loads a wave, and launch).
template <typename T>
__device__ __forceinline__ void vd_rest(const VdParams& p, int b, const VdChoice& ch, int first, int step, const double* s_exp) {
  constexpr int PER = 16 / VdType<T>::SIZE, PIECES = VD_CHUNK / 64 / PER;
  const int lane = threadIdx.x & 63;
  const char* const row = vd_row<T>(p, ch.row);
  const float* const q = p.probs + (size_t)ch.row * p.probs_stride;
  for (int chunk = first; chunk < p.n_chunks; chunk += step) {
    float x[PIECES][PER], y[PIECES][PER];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int at = chunk * VD_CHUNK + (64 * i + lane) * PER;
      vd_load<T>(row, at, p.V, x[i]);
      vd_load<float>(reinterpret_cast<const char*>(q), at, p.V, y[i]);
    }
    double z = 0.0;
#pragma unroll
    for (int i = 0; i < PIECES; ++i)
#pragma unroll
      for (int j = 0; j < PER; ++j) {                      // (behind the row's end y is -inf, and the weight is left out)
        const double w = vd_weight(x[i][j], ch.m, ch.c, s_exp) * ch.inv_z - (double)y[i][j];
        z += w > 0.0 && y[i][j] > -INFINITY ? w : 0.0;
      }
    z = vd_wave_sum(z);
    if (lane == 0) p.rest[(size_t)b * p.n_chunks + chunk] = z;
  }
}
template <typename T>
__global__ __launch_bounds__(64 * VD_WAVES) void verify_rest_kernel(const VdParams p) {
  __shared__ double s_exp[VD_EXP];
  const int b = blockIdx.x / p.splits, split = blockIdx.x - b * p.splits;
  const VdChoice ch = p.choice[b];
  if (ch.mode != VD_REST) return;
  vd_table(s_exp);
  __syncthreads();
  vd_rest<T>(p, b, ch, split * VD_WAVES + (threadIdx.x >> 6), p.splits * VD_WAVES, s_exp);
}
// Few sequences: each of these workgroups decides for itself, and the first writes it down (or draws at once where
// there is no rest), which saves a launch.
template <typename T>
__global__ __launch_bounds__(VD_BLOCK) void verify_decide_rest_kernel(const VdParams p) {
  __shared__ double s_exp[VD_EXP];
  __shared__ int s_row;
  __shared__ VdChoice s_choice;
  const int b = blockIdx.x / p.splits, split = blockIdx.x - b * p.splits;
  VdChoice ch;
  vd_table(s_exp);
  if (split == 0) {
    ch = vd_decide<T, true>(p, b, s_exp, &s_row, &s_choice);
    if (threadIdx.x == 0) p.choice[b] = ch;
    if (ch.mode != VD_REST) vd_pick<T>(p, b, ch, s_exp);
  } else {
    ch = vd_decide<T, false>(p, b, s_exp, &s_row, &s_choice);
  }
  if (ch.mode == VD_REST) vd_rest<T>(p, b, ch, split * VD_BLOCK_WAVES + (threadIdx.x >> 6), p.splits * VD_BLOCK_WAVES, s_exp);
}
template <typename T>
__global__ __launch_bounds__(VD_BLOCK) void verify_pick_kernel(const VdParams p) {
  __shared__ double s_exp[VD_EXP];
  vd_table(s_exp);
  const VdChoice ch = p.choice[blockIdx.x];
  if (ch.mode != VD_REST) return;            // (drawn already)
  __syncthreads();
  vd_pick<T>(p, blockIdx.x, ch, s_exp);
}

}  // namespace t2i

using t2i_host::fail;

namespace {

int vd_chunks(int V) { return (int)(((long long)V + t2i::VD_CHUNK - 1) / t2i::VD_CHUNK); }

// Workgroups of a row.  A wave takes two chunks, one after the other, where that leaves enough waves for all CUs
// (us of the whole call for 1, 2, 4, 8 chunks: 16 fp32 rows of 151936 11.1, 12.1, 14.4, 20.4; 120 21.8, 22.4, 23.2, 26.5;
// 432 86.2, 83.7, 84.6, 86.1; bf16, 61 rows 16.7, 16.8, 18.2, 21.7; 122 25.2, 24.3, 24.7, 28.8; 250 31.2, 29.7, 30.8,
// 32.3).
int vd_splits(int M, int n_chunks) {
  const long long run = (long long)M * n_chunks < 16384 ? 1 : 2;
  return (int)((n_chunks + t2i::VD_WAVES * run - 1) / (t2i::VD_WAVES * run));
}

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
  p.splits = vd_splits(M, p.n_chunks);
  if ((long long)M * p.splits > 0xFFFFFFFFLL / (64 * t2i::VD_WAVES) || n_seqs > 1 << 16)
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
  // few sequences: their workgroups decide for themselves, so long as all of them run at once (this way / a launch more, us: 1
  // sequence of four drafts 13.2 / 14.2, 8 21.7 / 23.9, 24 29.1 / 33.2, and 48, which have 480 workgroups, 50.9 / 50.0)
  const int wide = (p.n_chunks + t2i::VD_BLOCK_WAVES - 1) / t2i::VD_BLOCK_WAVES;
  const bool fused = draft_probs && (long long)n_seqs * wide <= 256;
#define T2I_VD_LAUNCH(kernel, ty, groups, threads)                                                                    \
  hipLaunchKernelGGL((t2i::kernel<ty>), dim3(groups), dim3(threads), 0, s, p);                                        \
  if (int rc = t2i_host::hip_status(hipGetLastError(), "verify_drafts launch")) return rc
#define T2I_VD(ty)                                                                                                    \
  T2I_VD_LAUNCH(verify_rows_kernel, ty, M * p.splits, 64 * t2i::VD_WAVES);                                            \
  if (!fused) { T2I_VD_LAUNCH(verify_kernel, ty, n_seqs, t2i::VD_BLOCK); }                                            \
  if (!draft_probs) return T2I_OK;                                                                                    \
  if (fused) {                                                                                                        \
    p.splits = wide;                                                                                                  \
    T2I_VD_LAUNCH(verify_decide_rest_kernel, ty, n_seqs * p.splits, t2i::VD_BLOCK);                                   \
  } else {                                                                                                            \
    p.splits = std::max(1, std::min((p.n_chunks + t2i::VD_WAVES - 1) / t2i::VD_WAVES, (4096 + n_seqs - 1) / n_seqs)); \
    T2I_VD_LAUNCH(verify_rest_kernel, ty, n_seqs * p.splits, 64 * t2i::VD_WAVES);                                     \
  }                                                                                                                   \
  T2I_VD_LAUNCH(verify_pick_kernel, ty, n_seqs, t2i::VD_BLOCK);                                                       \
  return T2I_OK
  switch (logits_type) {
    case T2I_LOGITS_FP32: { T2I_VD(float); }
    case T2I_LOGITS_BF16: { T2I_VD(t2i::VdBf16); }
    default: { T2I_VD(t2i::VdF16); }
  }
#undef T2I_VD
#undef T2I_VD_LAUNCH
}
