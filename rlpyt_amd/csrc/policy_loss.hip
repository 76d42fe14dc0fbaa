// Clipped policy loss with a KL term and an entropy bonus over a softmax policy given by its logits [N, V],
// forward and backward in one pass, and the log-probabilities that it takes as inputs.
//
//   logp = l_a - lse(l)     r = exp(logp - old_logp)     d = ref_logp - logp
//   pi = -min(r A, clip(r, 1 - lo, 1 + hi) A)     kl = e^d - d - 1     H = -sum_j p_j log p_j
//   loss = sum_n w_n (pi + c_kl kl - c_H H) / sum_n w_n
//   dl_j = w / sum w [ c 1_{j = a} + p_j (c_H (log p_j + H) - c) ]     c = dpi/dlogp - c_kl (e^d - 1)
//
// Memory bound: the floor reads and writes the logits once.  A row is kept in registers (of a group of lanes for
// V <= 128, of a wave up to 8 KB, of a workgroup up to 256 KB) between the softmax statistics and the gradient.  Longer rows,
// and batches of so few rows that one workgroup each leaves the chip idle, are split over workgroups: one
// launch for the statistics of the parts, one that joins them and reads the row again for the gradient.
//
// Measured, against 4.64 TB/s of a large copy: 8192 x 32000 bf16 (a fifth of the rows padded) 200 us, 226 being what a copy
// of all its logits takes; 96 x 100003 f32, split, 11.5 + 16.5 us for a floor of 16.5; 8192 x 18 f32 8 us with the
// sum of the weights, and 4 for the sums over the rows.
//
// Sums over a row are f32 per lane and in a fixed order (no atomics); what is done once per row is in 64 bits, on f32
// logarithms and exponentials of reduced arguments: kl ~ d^2 / 2 cancels in 32.  Exponents are in base 2 and come from one fma,
// t = x log2(e) - m with m the rounded product of the largest logit; what that rounding took is put back per row.  Where m is
// so large that its rounding could be a large exponent itself (a row of masks), t = (x - largest) log2(e).  -inf
// logits: t = -inf, e^t = 0, and 0 * t is kept 0 by taking t no lower than -300.  NaN goes through to the loss.
#include <math.h>

#include <algorithm>

#include "common.h"
#include "policy_loss_plan.h"

namespace rlpyt {
namespace {

template <typename E>
struct Row16 {   // 16 bytes of a row; rows of odd length start anywhere, global loads need only the element's alignment
  static constexpr int n = 16 / sizeof(E);
  typedef E vec __attribute__((ext_vector_type(n)));
  struct __attribute__((packed, aligned(sizeof(E)))) raw { vec v; };
};

struct LossArgs {
  const void* logits;
  int64_t row_stride;             // elements
  const int64_t* action;
  const float *old_logp, *advantage, *ref_logp, *valid;   // ref_logp, valid: may be null
  void* grad;                     // [N, V] dense, or null
  float *logp, *entropy;          // [N] each, or null
  double* rows;                   // [n, 4]: w pi, w kl, w H, w clipped of a row (or workgroup), or null (log-probabilities only)
  const double* denom;            // sum of valid, or null: N, or summed by every workgroup for itself
  struct Stats* parts;            // split rows: statistics of the parts [N, P]
  int64_t N, n0, n_rows;          // a launch takes the rows n0 .. n0 + n_rows - 1
  int V, part;                    // part: elements of a row's part, a multiple of 8
  double lo, hi, c_kl, c_ent, g_scale;
};

constexpr float kLog2e = 1.44269504088896340736f;
constexpr double kLn2 = 0.69314718055994530942;
constexpr float kFloor = -300.f;   // 2^-300 is 0 in f32

__device__ __forceinline__ float exp_of(float t) { return __builtin_amdgcn_exp2f(t); }
__device__ __forceinline__ float bounded(float t) { return fmaxf(t, kFloor); }

// Softmax statistics of some logits: with t = x log2(e) - m,  s = sum 2^t,  u = sum 2^t t; m = -inf: none.  m is a float, the
// rounded product of the largest logit, up to kFused, and the product itself (48 bits) beyond.
struct Stats {
  double m;
  float s, u;
};
constexpr float kFused = 1 << 20;   // (rounded by 2^-5 at most)
__device__ __forceinline__ float scaled(float largest) { return largest * kLog2e; }
__device__ __forceinline__ Stats join(const Stats& p, const Stats& q) {
  Stats r;
  r.m = fmax(p.m, q.m);
  if (r.m == -INFINITY) return Stats{-INFINITY, p.s + q.s, 0.f};   // (NaN sums stay)
  const float dp = bounded((float)(p.m - r.m)), dq = bounded((float)(q.m - r.m)), fp = exp_of(dp), fq = exp_of(dq);
  r.s = fmaf(fp, p.s, fq * q.s);
  r.u = fp * fmaf(dp, p.s, p.u) + fq * fmaf(dq, q.s, q.u);
  return r;
}
template <int G>
__device__ __forceinline__ Stats group_join(Stats v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) {
    Stats q;
    q.m = __shfl_xor(v.m, o, kWave), q.s = __shfl_xor(v.s, o, kWave), q.u = __shfl_xor(v.u, o, kWave);
    v = join(v, q);
  }
  return v;
}
template <int G>
__device__ __forceinline__ float group_max(float m) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, kWave));
  return m;
}

// log(s) to 2^-24 absolute: s = 2^k f with f in [1, 2)
__device__ __forceinline__ double log_of(float s) {
  const int k = (int)(__float_as_uint(s) >> 23) - 127;
  if (!(s >= 1.f && s < 3e38f)) return log((double)s);   // (the largest term of a row's sum is 1)
  return (double)k * kLn2 + (double)logf(__uint_as_float((__float_as_uint(s) & 0x7fffffu) | 0x3f800000u));
}
// e^d - d - 1 >= 0, to ~ 2^-20 relative: the series where it cancels
__device__ __forceinline__ double kl_of(double d) {
  if (fabs(d) > 0.5) {
    const double e = (double)expf((float)d);
    return e == INFINITY ? e : e - d - 1.0;   // (d may be infinite itself)
  }
  double v = 1.0;                     // d^12 / 12! is left out
#pragma unroll
  for (int k = 11; k >= 3; --k) v = fma(v, d * (1.0 / k), 1.0);
  return 0.5 * d * d * v;
}

// What the mean divides by; every thread of the workgroup has to come here.
__device__ __forceinline__ double weights(const float* __restrict__ valid, int64_t N, const double* denom, double* scratch) {
  if (!valid) return (double)N;
  if (denom) return *denom;
  double v = 0.0;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < N; i += blockDim.x) v += (double)valid[i];
  v = wave_sum(v);
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.0;
  for (int i = 0; i < (int)(blockDim.x >> 6); ++i) v += scratch[i];
  return v;
}

// What follows from a row's statistics: its terms of the loss, and its gradient as 2^t (k1 t + k0), + ka at the action, with
// t = (x - base) log2(e) - m, of which one is 0.
struct RowOut {
  double pi, kl, ent, clipped;
  float logp, entropy, base, m, k1, k0, ka;
};
__device__ __forceinline__ RowOut row_terms(const LossArgs& p, int64_t n, float w, const Stats& st, float xa,
                                            bool in_range, double denom) {
  RowOut o = {};
  if (st.m == -INFINITY && st.s == 0.f) {   // every logit is -inf: no distribution, the row adds nothing and has no gradient
    o.logp = -INFINITY;
    return o;
  }
  if (fabs(st.m) <= (double)kFused) o.m = (float)st.m;
  else o.base = (float)(st.m / (double)kLog2e);   // (the largest logit again, to its last bit)
  // natural logarithms: x - lse = (x log2(e) - m) ln 2 - log(s)
  const double logs = log_of(st.s), mean = (double)st.u / (double)st.s * kLn2;
  const double H = logs - mean;
  const double lp = in_range ? ((double)xa * (double)kLog2e - st.m) * kLn2 - logs : (double)NAN;
  o.logp = (float)lp;
  o.entropy = (float)H;
  if (!p.rows) return o;
  const double A = (double)p.advantage[n], r = (double)expf((float)(lp - (double)p.old_logp[n]));
  const double rc = fmin(fmax(r, 1.0 - p.lo), 1.0 + p.hi);
  double c = 0.0;
  if (A != 0.0 || r != r) {
    const double plain = r * A, clip = rc * A;
    o.pi = -(plain < clip ? plain : clip);
    if (plain != plain) o.pi = plain;
    if (!(plain > clip)) c = -plain;
  }
  o.clipped = r != rc ? 1.0 : 0.0;
  if (p.ref_logp) {
    const double d = (double)p.ref_logp[n] - lp;
    o.kl = kl_of(d);
    if (p.c_kl != 0.0) c -= p.c_kl * (d == -INFINITY ? -1.0 : o.kl + d);   // e^d - 1
  }
  o.ent = H;
  const double g = denom != 0.0 ? p.g_scale * (double)w / denom : 0.0, gs = g / (double)st.s;
  o.k1 = (float)(gs * p.c_ent * kLn2);
  o.k0 = (float)(gs * (p.c_ent * (H - logs) - c));
  o.ka = (float)(g * c);
  o.pi *= w, o.kl *= w, o.ent *= w, o.clipped *= w;
  return o;
}

// ---- V <= K G: G lanes a row, K elements a lane, R rows one after the other ---------------------------------
// What is done once per row is ~150 operations in 64 bits, as much as the rest of 50 elements: lane r of a group does row r's.
// Joins the values of G lanes (8 or 16) within the vector unit, lane permutations as operands; every lane gets the result.
template <int CTRL>
__device__ __forceinline__ float permuted(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int G, typename F>
__device__ __forceinline__ float joined(float v, F f) {
  v = f(v, permuted<0xb1>(v));               // lanes 1 0 3 2
  v = f(v, permuted<0x4e>(v));               // lanes 2 3 0 1
  v = f(v, permuted<0x141>(v));              // 8 lanes mirrored
  if (G == 16) v = f(v, permuted<0x140>(v));   // 16 lanes mirrored
  return v;
}

template <typename ET, int G, int K, int R>
__global__ __launch_bounds__(256) void loss_group_kernel(const LossArgs p) {
  typedef typename Elem<ET>::type E;
  constexpr int each = 256 / G;           // groups of a workgroup, and rows of a round
  __shared__ double sums[4 * 16], ws[4];
  const int sub = threadIdx.x & (G - 1);
  const int64_t first = p.n0 + (int64_t)blockIdx.x * (each * R) + threadIdx.x / G, end = p.n0 + p.n_rows;
  const int64_t own = first + sub * each;    // the row whose terms this lane works out
  const bool mine = sub < R && own < end;
  const float w = mine ? (p.valid ? p.valid[own] : 1.f) : 0.f;
  const int64_t action = w != 0.f ? p.action[own] : -1;
  const bool in_range = action >= 0 && action < p.V;
  const float xa = in_range ? (float)((const E*)p.logits)[own * p.row_stride + action] : 0.f;
  float t[R][K];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const bool live = __shfl(w, r, G) != 0.f;   // padded rows are not read
    const E* row = (const E*)p.logits + (first + r * each) * p.row_stride;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int j = sub + k * G;
      t[r][k] = live && j < p.V ? (float)row[j] : -INFINITY;
    }
  }
  const double denom = weights(p.valid, p.N, p.denom, ws);
  Stats st = {-INFINITY, 0.f, 0.f};
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float m = t[r][0], s = 0.f, u = 0.f;
#pragma unroll
    for (int k = 1; k < K; ++k) m = fmaxf(m, t[r][k]);
    m = joined<G>(m, [](float a, float b) { return fmaxf(a, b); });
    const float from = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const float x = (t[r][k] - from) * kLog2e, e = exp_of(x);
      t[r][k] = bounded(x);
      s += e;
      u = fmaf(e, t[r][k], u);
    }
    s = joined<G>(s, [](float a, float b) { return a + b; });
    u = joined<G>(u, [](float a, float b) { return a + b; });
    if (sub == r) st = Stats{(double)m * (double)kLog2e, s, u};
  }
  RowOut o = {};
  if (w != 0.f) {
    o = row_terms(p, own, w, st, xa, in_range, denom);
    if (p.logp) p.logp[own] = o.logp, p.entropy[own] = o.entropy;
  }
  if (p.grad) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float k1 = __shfl(o.k1, r, G), k0 = __shfl(o.k0, r, G), ka = __shfl(o.ka, r, G);
      const int a = __shfl(in_range ? (int)action : -1, r, G);
      E* g = (E*)p.grad + (first + r * each) * p.V;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int j = sub + k * G;
        float v = exp_of(t[r][k]) * fmaf(k1, t[r][k], k0);   // (2^-300 is 0 too)
        if (j == a) v += ka;
        if (j < p.V && first + r * each < end) g[j] = (E)v;
      }
    }
  }
  if (!p.rows) return;
  double v[4] = {o.pi, o.kl, o.ent, o.clipped};
  block_sum<4>(v, sums);
  if (threadIdx.x == 0)
    for (int k = 0; k < 4; ++k) p.rows[(p.n0 / (each * R) + blockIdx.x) * 4 + k] = v[k];
}

// ---- a row held by one workgroup of NT threads, R x 16 bytes a thread -------------------------------------
template <typename E>
__device__ __forceinline__ typename Row16<E>::vec load16(const E* __restrict__ row, int j, int V) {
  typedef typename Row16<E>::vec vec;
  constexpr int n = Row16<E>::n;
  if (j + n <= V) return reinterpret_cast<const typename Row16<E>::raw*>(row + j)->v;
  vec v;
#pragma unroll
  for (int k = 0; k < n; ++k) v[k] = j + k < V ? row[j + k] : (E)-INFINITY;
  return v;
}
template <typename E>
__device__ __forceinline__ void store16(E* __restrict__ row, int j, int V, typename Row16<E>::vec v) {
  constexpr int n = Row16<E>::n;
  if (j + n <= V) {
    reinterpret_cast<typename Row16<E>::raw*>(row + j)->v = v;
    return;
  }
#pragma unroll
  for (int k = 0; k < n; ++k)
    if (j + k < V) row[j + k] = v[k];
}
template <typename E>
__device__ __forceinline__ typename Row16<E>::vec grad16(typename Row16<E>::vec x, int j, int64_t a,
                                                         const RowOut& o) {
  constexpr int n = Row16<E>::n;
  float g[n];
#pragma unroll
  for (int k = 0; k < n; ++k) {
    const float t = fmaf((float)x[k], kLog2e, -o.m);
    g[k] = exp_of(t) * fmaf(o.k1, bounded(t), o.k0);
  }
  if ((uint64_t)(a - j) < (uint64_t)n) {
#pragma unroll
    for (int k = 0; k < n; ++k)
      if (j + k == a) g[k] += o.ka;
  }
  typename Row16<E>::vec v;
#pragma unroll
  for (int k = 0; k < n; ++k) v[k] = (E)g[k];
  return v;
}
// Logits of a row whose largest one is beyond kFused, less that one.  (Rounded: nothing where they are near each other, and
// further away e^t is 0.)
template <typename E, int R>
__device__ __forceinline__ void rebase(typename Row16<E>::vec (&x)[R], float base) {
  if (base == 0.f) return;
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int k = 0; k < Row16<E>::n; ++k) x[r][k] = (E)((float)x[r][k] - base);
}
// Keeps the compiler from holding the floats of one pass over a row's registers for the next: they are converted again, and
// two workgroups of 1024 fit a CU, one loading while the other computes.
template <typename E, int R>
__device__ __forceinline__ void forget(typename Row16<E>::vec (&x)[R]) {
#pragma unroll
  for (int r = 0; r < R; ++r) {
    uint4 v = __builtin_bit_cast(uint4, x[r]);
    asm volatile("" : "+v"(v.x), "+v"(v.y), "+v"(v.z), "+v"(v.w));
    x[r] = __builtin_bit_cast(typename Row16<E>::vec, v);
  }
}
// statistics of the vectors of a wave
template <typename E, int R>
__device__ __forceinline__ Stats wave_stats(typename Row16<E>::vec (&x)[R]) {
  constexpr int n = Row16<E>::n;
  float m = -INFINITY;
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int k = 0; k < n; ++k) m = fmaxf(m, (float)x[r][k]);
  forget<E, R>(x);
  m = group_max<kWave>(m);
  Stats st = {(double)scaled(m), 0.f, 0.f};
  auto add = [&](float t) {
    const float e = exp_of(t);
    st.s += e;
    st.u = fmaf(e, bounded(t), st.u);
  };
  if (m == -INFINITY || fabsf(scaled(m)) <= kFused) {
    const float from = m == -INFINITY ? 0.f : scaled(m);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int k = 0; k < n; ++k) add(fmaf((float)x[r][k], kLog2e, -from));
  } else {
    st.m = (double)m * (double)kLog2e;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int k = 0; k < n; ++k) add(((float)x[r][k] - m) * kLog2e);
  }
  st.s = wave_sum(st.s);
  st.u = wave_sum(st.u);
  return st;
}
// joins the waves' statistics; every thread gets the result
template <int NT>
__device__ __forceinline__ Stats block_join(const Stats& st, Stats* lds) {
  constexpr int NW = NT / kWave;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  if (lane == 0) lds[w] = st;
  __syncthreads();
  Stats v = lane < NW ? lds[lane] : Stats{-INFINITY, 0.f, 0.f};
  v = group_join<NW>(v);
  v.m = __shfl(v.m, 0, kWave), v.s = __shfl(v.s, 0, kWave), v.u = __shfl(v.u, 0, kWave);
  return v;
}

template <typename ET, int NT, int R>
__global__ __launch_bounds__(NT) void loss_row_kernel(const LossArgs p) {
  typedef typename Elem<ET>::type E;
  typedef typename Row16<E>::vec vec;
  constexpr int n16 = Row16<E>::n;
  __shared__ Stats lds[NT / kWave];
  __shared__ RowOut out;
  __shared__ double ws[NT / kWave];
  const int64_t n = p.n0 + blockIdx.x;
  const float w = p.valid ? p.valid[n] : 1.f;
  E* g = p.grad ? (E*)p.grad + n * p.V : nullptr;
  if (w == 0.f) {   // a padded row: not read, no gradient
    if (g) {
      vec zero;
#pragma unroll
      for (int k = 0; k < n16; ++k) zero[k] = (E)0.f;
      for (int r = 0; r < R; ++r) {
        const int j = (r * NT + threadIdx.x) * n16;
        if (j < p.V) store16<E>(g, j, p.V, zero);
      }
    }
    if (p.rows && threadIdx.x < 4) p.rows[n * 4 + threadIdx.x] = 0.0;
    return;
  }
  const E* row = (const E*)p.logits + n * p.row_stride;
  const int64_t a = p.action[n];
  const bool in_range = a >= 0 && a < p.V;
  const float xa = in_range ? (float)row[a] : 0.f;
  vec x[R];
#pragma unroll
  for (int r = 0; r < R; ++r) x[r] = load16<E>(row, (r * NT + threadIdx.x) * n16, p.V);
  const double denom = weights(p.valid, p.N, p.denom, ws);
  const Stats st = block_join<NT>(wave_stats<E, R>(x), lds);
  forget<E, R>(x);
  if (threadIdx.x == 0) {
    out = row_terms(p, n, w, st, xa, in_range, denom);
    if (p.logp) p.logp[n] = out.logp, p.entropy[n] = out.entropy;
    if (p.rows) p.rows[n * 4] = out.pi, p.rows[n * 4 + 1] = out.kl, p.rows[n * 4 + 2] = out.ent, p.rows[n * 4 + 3] = out.clipped;
  }
  if (!g) return;
  __syncthreads();
  const RowOut o = out;
  rebase<E, R>(x, o.base);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int j = (r * NT + threadIdx.x) * n16;
    if (j < p.V) store16<E>(g, j, p.V, grad16<E>(x[r], j, a, o));
  }
}

// ---- a row held by one wave, R x 16 bytes a lane ----------------------------------------------------------
template <typename ET, int R>
__global__ __launch_bounds__(256) void loss_wave_kernel(const LossArgs p) {
  typedef typename Elem<ET>::type E;
  typedef typename Row16<E>::vec vec;
  constexpr int n16 = Row16<E>::n;
  __shared__ double sums[4][4], ws[4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t n = p.n0 + (int64_t)blockIdx.x * 4 + wave;
  const bool on = n < p.n0 + p.n_rows;
  const float w = on ? (p.valid ? p.valid[n] : 1.f) : 0.f;
  const double denom = weights(p.valid, p.N, p.denom, ws);
  RowOut o = {};
  if (w != 0.f) {
    const E* row = (const E*)p.logits + n * p.row_stride;
    const int64_t a = p.action[n];
    const bool in_range = a >= 0 && a < p.V;
    const float xa = in_range ? (float)row[a] : 0.f;
    vec x[R];
#pragma unroll
    for (int r = 0; r < R; ++r) x[r] = load16<E>(row, (r * kWave + lane) * n16, p.V);
    o = row_terms(p, n, w, wave_stats<E, R>(x), xa, in_range, denom);
    forget<E, R>(x);
    if (lane == 0 && p.logp) p.logp[n] = o.logp, p.entropy[n] = o.entropy;
    if (p.grad) {
      E* g = (E*)p.grad + n * p.V;
      rebase<E, R>(x, o.base);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int j = (r * kWave + lane) * n16;
        if (j < p.V) store16<E>(g, j, p.V, grad16<E>(x[r], j, a, o));
      }
    }
  } else if (on && p.grad) {
    vec zero;
#pragma unroll
    for (int k = 0; k < n16; ++k) zero[k] = (E)0.f;
    for (int j = lane * n16; j < p.V; j += kWave * n16) store16<E>((E*)p.grad + n * p.V, j, p.V, zero);
  }
  if (!p.rows) return;
  if (lane == 0) sums[0][wave] = o.pi, sums[1][wave] = o.kl, sums[2][wave] = o.ent, sums[3][wave] = o.clipped;
  __syncthreads();
  if (threadIdx.x < 4) {
    const double* v = sums[threadIdx.x];
    p.rows[(p.n0 / 4 + blockIdx.x) * 4 + threadIdx.x] = v[0] + v[1] + v[2] + v[3];
  }
}

// ---- rows split over workgroups ----------------------------------------------------------------------------
constexpr int kSplitThreads = 256, kSplitVecs = 4;   // vectors in flight per thread

template <typename ET>
__global__ __launch_bounds__(kSplitThreads) void loss_parts_kernel(const LossArgs p, int P) {
  typedef typename Elem<ET>::type E;
  typedef typename Row16<E>::vec vec;
  constexpr int n16 = Row16<E>::n, step = kSplitThreads * kSplitVecs * n16;
  __shared__ Stats lds[kSplitThreads / kWave];
  const int64_t n = p.n0 + blockIdx.x / P;
  const int i = blockIdx.x % P;
  if (p.valid && p.valid[n] == 0.f) return;
  const E* row = (const E*)p.logits + n * p.row_stride;
  const int begin = i * p.part, end = min(p.V, begin + p.part);
  Stats st = {-INFINITY, 0.f, 0.f};
  for (int j0 = begin; j0 < end; j0 += step) {
    vec x[kSplitVecs];
#pragma unroll
    for (int r = 0; r < kSplitVecs; ++r) x[r] = load16<E>(row, j0 + (r * kSplitThreads + threadIdx.x) * n16, end);
    st = join(st, wave_stats<E, kSplitVecs>(x));
  }
  st = block_join<kSplitThreads>(st, lds);
  if (threadIdx.x == 0) p.parts[n * P + i] = st;
}

template <typename ET>
__global__ __launch_bounds__(kSplitThreads) void loss_join_kernel(const LossArgs p, int P, int blocks) {
  typedef typename Elem<ET>::type E;
  typedef typename Row16<E>::vec vec;
  constexpr int n16 = Row16<E>::n, step = kSplitThreads * n16;
  __shared__ Stats lds[kSplitThreads / kWave];
  __shared__ RowOut out;
  __shared__ double ws[kSplitThreads / kWave];
  const int64_t n = p.n0 + blockIdx.x / blocks;   // blocks per row: P, or 1 without a gradient
  const int part = blockIdx.x % blocks;
  const float w = p.valid ? p.valid[n] : 1.f;
  const bool live = w != 0.f;
  const bool first = part == 0;
  const int64_t a = live ? p.action[n] : -1;
  const E* row = (const E*)p.logits + n * p.row_stride;
  if (live) {
    Stats st = {-INFINITY, 0.f, 0.f};
    for (int i = threadIdx.x; i < P; i += kSplitThreads) st = join(st, p.parts[n * P + i]);
    const double denom = weights(p.valid, p.N, p.denom, ws);
    st = block_join<kSplitThreads>(group_join<kWave>(st), lds);
    if (threadIdx.x == 0) {
      const bool in_range = a >= 0 && a < p.V;
      out = row_terms(p, n, w, st, in_range ? (float)row[a] : 0.f, in_range, denom);
      if (first && p.logp) p.logp[n] = out.logp, p.entropy[n] = out.entropy;
    }
  } else if (threadIdx.x == 0) {
    out = RowOut{};
  }
  if (threadIdx.x == 0 && first && p.rows)
    p.rows[n * 4] = out.pi, p.rows[n * 4 + 1] = out.kl, p.rows[n * 4 + 2] = out.ent, p.rows[n * 4 + 3] = out.clipped;
  if (!p.grad) return;
  __syncthreads();
  const RowOut o = out;
  E* g = (E*)p.grad + n * p.V;
  const int begin = part * p.part, end = min(p.V, begin + p.part);
  for (int j = begin + threadIdx.x * n16; j < end; j += step) {
    vec v[1];
    if (live) {
      v[0] = load16<E>(row, j, end);
      rebase<E, 1>(v, o.base);
      v[0] = grad16<E>(v[0], j, a, o);
    } else {
#pragma unroll
      for (int k = 0; k < n16; ++k) v[0][k] = (E)0.f;
    }
    store16<E>(g, j, end, v[0]);
  }
}

// ---- sums over the rows -------------------------------------------------------------------------------------
// One workgroup adds up to kSumRows rows; of more (a million samples took it 0.3 ms) kSumBlocks add a share each, first.
constexpr int kSumRows = 16384, kSumBlocks = 256;

template <typename T, int K>
__global__ __launch_bounds__(1024) void loss_sum_kernel(const T* __restrict__ in, int64_t n, double* __restrict__ out) {
  __shared__ double scratch[K * 16];
  double v[K] = {};
#pragma unroll 4
  for (int64_t i = (int64_t)blockIdx.x * 1024 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 1024)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += (double)in[i * K + k];
  block_sum<K>(v, scratch);
  if (threadIdx.x == 0)
    for (int k = 0; k < K; ++k) out[blockIdx.x * K + k] = v[k];
}

__global__ __launch_bounds__(1024) void loss_finish_kernel(const double* __restrict__ rows, int64_t n,
                                                           const double* __restrict__ denom,
                                                           const float* __restrict__ valid, int64_t N, double c_kl,
                                                           double c_ent, float* __restrict__ loss,
                                                           float* __restrict__ scalars) {
  __shared__ double scratch[4 * 16], ws[16];
  const double d = weights(valid, N, denom, ws);
  double v[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < n; i += 1024)
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] += rows[i * 4 + k];
  block_sum<4>(v, scratch);
  if (threadIdx.x != 0) return;
  const double inv = d != 0.0 ? 1.0 / d : 0.0;   // nothing valid: a loss of 0
  for (int k = 0; k < 4; ++k) v[k] *= inv;
  *loss = scalars[0] = (float)(v[0] + (c_kl != 0.0 ? c_kl * v[1] : 0.0) - c_ent * v[2]);
  for (int k = 0; k < 4; ++k) scalars[1 + k] = (float)v[k];
}

// grad *= *scale * factor, in place; nothing is read or written where that is 1 (hence a grid that the chip holds at once).
template <typename ET>
__global__ __launch_bounds__(256) void loss_scale_kernel(void* __restrict__ x, int64_t n,
                                                         const float* __restrict__ scale, float factor) {
  typedef typename Elem<ET>::type E;
  E* g = (E*)x;
  typedef typename Row16<E>::vec vec;
  constexpr int n16 = Row16<E>::n;
  const float f = *scale * factor;
  if (f == 1.f) return;
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * n16; i < n; i += (int64_t)gridDim.x * 256 * n16) {
    if (i + n16 <= n) {
      vec v = *reinterpret_cast<const vec*>(g + i);
#pragma unroll
      for (int k = 0; k < n16; ++k) v[k] = (E)((float)v[k] * f);
      *reinterpret_cast<vec*>(g + i) = v;
    } else {
      for (int64_t k = i; k < n; ++k) g[k] = (E)((float)g[k] * f);
    }
  }
}

// ------------------------------------------------------------------------------------ host side
enum { F32 = 0, BF16 = 1, F16 = 2 };

template <typename ET, int R>
void launch_groups(const LossArgs& p, hipStream_t s) {
  const int V = p.V;
  const dim3 grid((unsigned)ceil_div(p.n_rows, 256 / group_lanes(V) * R));
  if (V <= 8) RL_LAUNCH((loss_group_kernel<ET, 8, 1, R>), grid, dim3(256), 0, s, p);
  else if (V <= 32) RL_LAUNCH((loss_group_kernel<ET, 8, 4, R>), grid, dim3(256), 0, s, p);
  else if (V <= 64) RL_LAUNCH((loss_group_kernel<ET, 16, 4, R>), grid, dim3(256), 0, s, p);
  else RL_LAUNCH((loss_group_kernel<ET, 16, 8, R>), grid, dim3(256), 0, s, p);
}

template <typename ET>
int run(LossArgs p, const LossPlan& q, hipStream_t s) {
  typedef typename Elem<ET>::type E;
  const int V = p.V;
  const int64_t vecs = ceil_div((int64_t)V, (int64_t)Row16<E>::n);
  if (V <= kGroupV) {
    if (group_rows(p.N) == 1) launch_groups<ET, 1>(p, s);
    else launch_groups<ET, 4>(p, s);
  } else if (V * (int64_t)sizeof(E) <= kWaveBytes) {
    const dim3 grid((unsigned)ceil_div(p.n_rows, 4));
    if (vecs <= 64) RL_LAUNCH((loss_wave_kernel<ET, 1>), grid, dim3(256), 0, s, p);
    else if (vecs <= 128) RL_LAUNCH((loss_wave_kernel<ET, 2>), grid, dim3(256), 0, s, p);
    else if (vecs <= 256) RL_LAUNCH((loss_wave_kernel<ET, 4>), grid, dim3(256), 0, s, p);
    else RL_LAUNCH((loss_wave_kernel<ET, 8>), grid, dim3(256), 0, s, p);
  } else if (q.P == 0) {
    const dim3 grid((unsigned)p.n_rows);
    if (vecs <= 1024) RL_LAUNCH((loss_row_kernel<ET, 256, 4>), grid, dim3(256), 0, s, p);
    else if (vecs <= 2048) RL_LAUNCH((loss_row_kernel<ET, 512, 4>), grid, dim3(512), 0, s, p);
    else if (vecs <= 4096) RL_LAUNCH((loss_row_kernel<ET, 1024, 4>), grid, dim3(1024), 0, s, p);
    else if (vecs <= 8192) RL_LAUNCH((loss_row_kernel<ET, 1024, 8>), grid, dim3(1024), 0, s, p);
    else RL_LAUNCH((loss_row_kernel<ET, 1024, 16>), grid, dim3(1024), 0, s, p);
  } else {
    const int blocks = p.grad ? q.P : 1;
    RL_LAUNCH((loss_parts_kernel<ET>), dim3((unsigned)(p.n_rows * q.P)), dim3(kSplitThreads), 0, s, p, q.P);
    RL_LAUNCH((loss_join_kernel<ET>), dim3((unsigned)(p.n_rows * blocks)), dim3(kSplitThreads), 0, s, p, q.P, blocks);
  }
  RL_LAUNCH_CHECK();
  return RLPYT_OK;
}

int element_size(int dtype) { return dtype == F32 ? 4 : 2; }

int run_all(int dtype, LossArgs p, const LossPlan& q, hipStream_t s) {
  const int64_t slice = slice_rows(q);
  for (p.n0 = 0; p.n0 < p.N; p.n0 += slice) {
    p.n_rows = std::min(slice, p.N - p.n0);
    int rc;
    if (dtype == F32) rc = run<float>(p, q, s);
    else if (dtype == BF16) rc = run<Bf16>(p, q, s);
    else rc = run<Half>(p, q, s);
    if (rc != RLPYT_OK) return rc;
  }
  return RLPYT_OK;
}

// workspace: sum of valid | sums of shares | 4 partial sums per row or workgroup | statistics of the parts
constexpr int64_t kRowsOffset = 16 + kSumBlocks * 4 * (int64_t)sizeof(double);
int64_t parts_offset(const LossPlan& q) { return kRowsOffset + q.partials * 4 * (int64_t)sizeof(double); }

}  // namespace
}  // namespace rlpyt

using namespace rlpyt;

extern "C" int64_t rlpyt_policy_loss_workspace_bytes(int dtype, int64_t N, int64_t V) {
  if (dtype < F32 || dtype > F16 || N <= 0 || V <= 0) return kRowsOffset;
  const LossPlan q = plan_of(N, V, element_size(dtype));
  return parts_offset(q) + N * q.P * (int64_t)sizeof(Stats);
}

extern "C" int rlpyt_policy_kl_loss_fwd_bwd(int dtype, const void* logits, int64_t row_stride,
                                            const int64_t* action, const float* old_logp,
                                            const float* advantage, const float* ref_logp, const float* valid,
                                            int64_t N, int64_t V, double clip_low, double clip_high,
                                            double kl_coeff, double entropy_coeff, double grad_scale, float* loss,
                                            float* scalars, void* grad, void* workspace, rlpyt_stream_t stream) {
  RL_CHECK_ARG(dtype >= F32 && dtype <= F16, RLPYT_EINVAL, "rlpyt_policy_kl_loss_fwd_bwd: unknown dtype %d", dtype);
  RL_CHECK_ARG(N >= 0 && V > 0 && V <= (1 << 30), RLPYT_ESHAPE,
               "rlpyt_policy_kl_loss_fwd_bwd: N=%ld V=%ld out of range", (long)N, (long)V);
  RL_CHECK_ARG(loss && scalars && workspace, RLPYT_EINVAL, "rlpyt_policy_kl_loss_fwd_bwd: null pointer");
  RL_CHECK_ARG(N == 0 || (logits && action && old_logp && advantage), RLPYT_EINVAL,
               "rlpyt_policy_kl_loss_fwd_bwd: null pointer");
  hipStream_t s = (hipStream_t)stream;
  const LossPlan q = plan_of(N, V, element_size(dtype));
  LossArgs p = {};
  p.logits = logits, p.row_stride = row_stride, p.action = action, p.old_logp = old_logp, p.advantage = advantage;
  p.ref_logp = ref_logp, p.valid = valid, p.grad = grad;
  double *denom = (double*)workspace, *shares = (double*)((char*)workspace + 16);
  p.rows = (double*)((char*)workspace + kRowsOffset);
  // The sum of the weights: by every workgroup where that is few numbers altogether, else in a launch of its own, which costs 4 us of
  // the call.  On the device, f32 without a gradient, by every workgroup and in a launch: 1024 x 18 11.7 and 12.1 us, 8192 x 18 12.0 and
  // 12.0, 16384 x 18 13.4 and 12.7, 30000 x 18 19.0 and 16.1; 2048 x 500 10.7 and 11.1, 4096 x 500 12.4 and 12.1; 1024 x 3000 12.2 and
  // 12.3, 2048 x 3000 15.3 and 14.7.
  const bool fold = q.groups(N) * N <= (int64_t)1 << 21;
  p.denom = valid && !fold ? denom : nullptr;
  p.parts = (Stats*)((char*)workspace + parts_offset(q));
  p.N = N, p.V = (int)V, p.part = q.part;
  p.lo = clip_low, p.hi = clip_high, p.c_kl = kl_coeff, p.c_ent = entropy_coeff, p.g_scale = grad_scale;
  if (p.denom && N > kSumRows) {
    RL_LAUNCH((loss_sum_kernel<float, 1>), dim3(kSumBlocks), dim3(1024), 0, s, valid, N, shares);
    RL_LAUNCH((loss_sum_kernel<double, 1>), dim3(1), dim3(1024), 0, s, shares, kSumBlocks, denom);
  } else if (p.denom) {
    RL_LAUNCH((loss_sum_kernel<float, 1>), dim3(1), dim3(1024), 0, s, valid, N, denom);
  }
  const int rc = run_all(dtype, p, q, s);
  if (rc != RLPYT_OK) return rc;
  const double* rows = p.rows;
  int64_t sums = N ? q.partials : 0;
  if (sums > kSumRows) {
    RL_LAUNCH((loss_sum_kernel<double, 4>), dim3(kSumBlocks), dim3(1024), 0, s, rows, sums, shares);
    rows = shares, sums = kSumBlocks;
  }
  RL_LAUNCH(loss_finish_kernel, dim3(1), dim3(1024), 0, s, rows, sums, p.denom, valid, N, kl_coeff,
            entropy_coeff, loss, scalars);
  RL_LAUNCH_CHECK();
  return RLPYT_OK;
}

extern "C" int rlpyt_action_logp(int dtype, const void* logits, int64_t row_stride, const int64_t* action,
                                 int64_t N, int64_t V, float* logp, float* entropy, void* workspace,
                                 rlpyt_stream_t stream) {
  RL_CHECK_ARG(dtype >= F32 && dtype <= F16, RLPYT_EINVAL, "rlpyt_action_logp: unknown dtype %d", dtype);
  RL_CHECK_ARG(N >= 0 && V > 0 && V <= (1 << 30), RLPYT_ESHAPE, "rlpyt_action_logp: N=%ld V=%ld out of range",
               (long)N, (long)V);
  if (N == 0) return RLPYT_OK;
  RL_CHECK_ARG(logits && action && logp && entropy && workspace, RLPYT_EINVAL, "rlpyt_action_logp: null pointer");
  const LossPlan q = plan_of(N, V, element_size(dtype));
  LossArgs p = {};
  p.logits = logits, p.row_stride = row_stride, p.action = action, p.logp = logp, p.entropy = entropy;
  p.parts = (Stats*)((char*)workspace + parts_offset(q));
  p.N = N, p.V = (int)V, p.part = q.part;
  return run_all(dtype, p, q, (hipStream_t)stream);
}

extern "C" int rlpyt_scale_unless_one(int dtype, void* x, int64_t n, const float* scale, float factor,
                                      rlpyt_stream_t stream) {
  RL_CHECK_ARG(dtype >= F32 && dtype <= F16, RLPYT_EINVAL, "rlpyt_scale_unless_one: unknown dtype %d", dtype);
  RL_CHECK_ARG(n >= 0, RLPYT_ESHAPE, "rlpyt_scale_unless_one: n=%ld out of range", (long)n);
  if (n == 0) return RLPYT_OK;
  RL_CHECK_ARG(x && scale, RLPYT_EINVAL, "rlpyt_scale_unless_one: null pointer");
  RL_CHECK_ARG(RL_ALIGNED16(x), RLPYT_ESHAPE, "rlpyt_scale_unless_one: x must be 16-byte aligned");
  hipStream_t s = (hipStream_t)stream;
  const int per = 256 * (16 / element_size(dtype));
  const dim3 grid((unsigned)std::min<int64_t>(1024, ceil_div(n, per)));
  if (dtype == F32) RL_LAUNCH((loss_scale_kernel<float>), grid, dim3(256), 0, s, x, n, scale, factor);
  else if (dtype == BF16) RL_LAUNCH((loss_scale_kernel<Bf16>), grid, dim3(256), 0, s, x, n, scale, factor);
  else RL_LAUNCH((loss_scale_kernel<Half>), grid, dim3(256), 0, s, x, n, scale, factor);
  RL_LAUNCH_CHECK();
  return RLPYT_OK;
}
