// Gated linear recurrence over [T, B, D] sequences, its backward pass and its one-step form.
//
//   z_t = sigmoid(gate_t)      h_t = (1 - z_t) k_t h_{t-1} + z_t x_t      k_t = 0 where reset, else 1
//   G_t = dh_t + (1 - z_{t+1}) k_{t+1} G_{t+1}     dx_t = z_t G_t
//   dgate_t = G_t (x_t - k_t h_{t-1}) z_t (1 - z_t)     dh_0 = k_0 (1 - z_0) G_0
//
// Each step is the map h -> A h + H of one channel, and maps compose: (A2, H2) after (A1, H1) is
// (A2 A1, A2 H1 + H2).  A wave takes kL consecutive steps of 64 x V channels into registers, reduces
// them to one map, hands it to the workgroup's other waves (consecutive steps of the same channels)
// through LDS, folds the maps before its own into the state it starts from and runs its steps again
// from registers: the streams are read once.  Memory bound (~25 vector operations per element against
// 6 .. 12 bytes).  Where B D channels are too few to fill the chip, time is cut into segments as well: a first
// launch reduces every segment to its map (it reads the streams without writing), the main launch folds the
// maps of the segments before its own.  No workgroup ever waits for another one.
//
// Measured, against 4.64 TB/s of a large copy: 128 x 256 x 512 bf16 forward 25 us (103 MB, 4.1 TB/s), backward 38 us (170 MB,
// 4.5); 65536 x 1 x 1024 bf16 in 64 segments 75 + 75 us forward, 62 + 150 backward, where one pass over the streams
// would take 87 and 145; 85 x 32 x 512 f32 7.7 and 10.8 us, most of it latency (256 workgroups, two windows each).
//
// A reset forgets whatever came before, also a state that is not finite: such a map carries A = -1
// (a product of sigmoids is never negative) and composes as "H alone", not as 0 * h.
//
// States, maps and sums are 32 bits; x, gate, h and the gradients are f32, bf16 or f16 and each output is
// rounded once.  The backward pass starts from f32 states kept every kKeep steps and recomputes the others:
// reading h back would be 2 (4) bytes per element more and, for 16-bit streams, a rounded state.
#include <algorithm>

#include "common.h"

namespace rlpyt {
namespace {

constexpr int kL = 8;         // steps per wave and window
constexpr int kMaxWaves = 8;  // waves (consecutive kL-step chunks) per workgroup
constexpr int kKeep = 32;     // distance of the kept states: every window of 4 or 8 waves starts at one

// V values next to each other, at any multiple of the element's size (global memory asks for no more)
template <typename E, int V>
struct Vec {
  typedef E type __attribute__((ext_vector_type(V)));
  struct __attribute__((packed, aligned(sizeof(E)))) raw { type v; };
};
template <typename E, int V>
__device__ __forceinline__ typename Vec<E, V>::type load(const E* p) {
  return reinterpret_cast<const typename Vec<E, V>::raw*>(p)->v;
}
template <typename E, int V>
__device__ __forceinline__ void store(E* p, typename Vec<E, V>::type v) {
  reinterpret_cast<typename Vec<E, V>::raw*>(p)->v = v;
}

struct Stream {   // one [T, B, D] tensor: unit stride along D, element strides along T and B
  int64_t ts, bs;
};

// z = 1 / (1 + e^-g) and a = 1 - z.  The larger of the two is known to 5 x 2^-24, the other, about e^-|g|, to (1.3 |g| + 5) 2^-24
// relative: its exponent is rounded once, and three more operations for what that takes would come on ~25 per element.  (v_rcp alone
// leans one way, and the a's go into long products; a large gate is cut where z is 1 and a is nothing beside it; a NaN stays one.)
__device__ __forceinline__ void gates(float g, float& z, float& a) {
  float t = g * 1.44269504088896340736f;
  t = t > 120.f ? 120.f : t;
  const float e = __builtin_amdgcn_exp2f(t), d = 1.f + e, q = __builtin_amdgcn_rcpf(d);
  a = fmaf(fmaf(-d, q, 1.f), q, q);
  z = g > 0.f ? 1.f - a : e * a;
}

__device__ __forceinline__ float fold(float c, float A, float H) {
  return __float_as_int(A) < 0 ? H : fmaf(A, c, H);   // (-0 too: a product behind a reset may vanish)
}

// A of two maps, one after the other
__device__ __forceinline__ float chain(float A1, float A2) {
  return (__float_as_int(A1) | __float_as_int(A2)) < 0 ? -1.f : A1 * A2;
}

struct Args {
  const void *x, *gate, *dh;       // dh: backward only; strides 0 are fine
  void *h, *dx, *dgate;            // h: forward only
  Stream xs, gs, hs, dxs, dgs;     // hs: of h (forward) / dh (backward)
  const float* first;              // h0 (forward) / dhn (backward) [B D] or null
  float* last;                     // hn (forward) / dh0 (backward) [B D] or null
  const uint8_t* reset;            // [T, B] or null
  const int64_t* lengths;          // [B] or null
  float* chk;                      // f32 states before steps 0, kKeep, 2 kKeep, .. [ceil(T / kKeep), B D] or null
  float2* agg;                     // maps of the segments [S, B D]
  int T, B, D;
  int seg;                         // steps per segment, a multiple of the window
};

// What a lane needs to know about its V channels.
struct Lane {
  int64_t c;       // channel b D + d
  int b, d, end;   // end: steps of this sequence
  bool on;
};

template <int V, bool LEN>
__device__ __forceinline__ Lane lane_of(const Args& p) {
  Lane l;
  const int per_row = (p.D + V - 1) / V;
  const int64_t i = (int64_t)blockIdx.x * kWave + (threadIdx.x & 63);
  l.on = i < (int64_t)p.B * per_row;
  l.b = l.on ? (int)(i / per_row) : 0;
  // the last lane of a row of odd length takes a channel of its neighbour again, with the same results
  l.d = min((int)(i - (int64_t)l.b * per_row) * V, p.D - V);
  if (!l.on) l.d = 0;
  l.c = (int64_t)l.b * p.D + l.d;
  l.end = p.T;
  if (LEN) l.end = (int)min((int64_t)p.T, max((int64_t)0, p.lengths[l.b]));
  return l;
}

// kL rows from step t0 on; rows behind the last one are read as the last one and masked by the caller.
template <typename E, int V>
__device__ __forceinline__ void load_chunk(const E* __restrict__ base, int64_t ts, int t0, int last,
                                           typename Vec<E, V>::type (&out)[kL]) {
#pragma unroll
  for (int i = 0; i < kL; ++i)
    out[i] = load<E, V>(base + (int64_t)min(t0 + i, last) * ts);
}

// The reset bytes of kL steps, fetched like the streams, and as bits: the state is cleared before step t0 + i.
__device__ __forceinline__ void load_resets(const Args& p, const Lane& l, int t0, uint8_t (&r)[kL]) {
#pragma unroll
  for (int i = 0; i < kL; ++i) r[i] = p.reset[(int64_t)min(t0 + i, p.T - 1) * p.B + l.b];
}
__device__ __forceinline__ uint32_t reset_bits(const uint8_t (&r)[kL], int t0, int end) {
  uint32_t clear = 0;
#pragma unroll
  for (int i = 0; i < kL; ++i) clear |= (uint32_t)(r[i] != 0 && t0 + i < end) << i;
  return clear;
}

// Steps behind the end hold the state and add nothing: a gate of -inf (z = 0, a = 1).
template <typename E, int V>
__device__ __forceinline__ void mask_chunk(typename Vec<E, V>::type (&gr)[kL], typename Vec<E, V>::type (&other)[kL], int t0,
                                           int end) {
#pragma unroll
  for (int i = 0; i < kL; ++i)
    if (t0 + i >= end) {
#pragma unroll
      for (int k = 0; k < V; ++k) gr[i][k] = (E)-INFINITY, other[i][k] = (E)0.f;
    }
}

// The maps before (forward) or behind (backward) segment s, folded into the state this segment starts
// from.  Wave w folds an equal share of them, the shares are joined through LDS.
template <int V, bool FWD>
__device__ __forceinline__ void segment_carry(const Args& p, const Lane& l, int s, int S, int W, int w,
                                              float2 (*lds)[kWave * V], float (&carry)[V]) {
  const int lane = threadIdx.x & 63;
  const int64_t C = (int64_t)p.B * p.D;
#pragma unroll
  for (int k = 0; k < V; ++k) carry[k] = (l.on && p.first) ? p.first[l.c + k] : 0.f;
  const int n = FWD ? s : S - 1 - s;           // segments to fold, nearest to the start first
  if (n == 0) return;                          // (the same for the whole workgroup)
  const int lo = (int)((int64_t)n * w / W), hi = (int)((int64_t)n * (w + 1) / W);
  float A[V], H[V];
#pragma unroll
  for (int k = 0; k < V; ++k) A[k] = 1.f, H[k] = 0.f;
  if (l.on) {
#pragma unroll 8
    for (int j = lo; j < hi; ++j) {
      const float2* q = p.agg + (int64_t)(FWD ? j : S - 1 - j) * C + l.c;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float2 m = q[k];
        H[k] = fold(H[k], m.x, m.y);
        A[k] = chain(A[k], m.x);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < V; ++k) lds[w][lane * V + k] = float2{A[k], H[k]};
  __syncthreads();
  for (int j = 0; j < W; ++j) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float2 m = lds[j][lane * V + k];
      carry[k] = fold(carry[k], m.x, m.y);
    }
  }
  __syncthreads();
}

// Forward.  AGG: reduce the segment to its map, write nothing else.
template <typename ET, int V, bool RESET, bool LEN, bool AGG>
__global__ __launch_bounds__(64 * kMaxWaves) void gated_scan_fwd_kernel(const Args p) {
  typedef typename Elem<ET>::type E;
  typedef typename Vec<E, V>::type VE;
  __shared__ float2 lds[2][kMaxWaves][kWave * V];
  const Lane l = lane_of<V, LEN>(p);
  const int lane = threadIdx.x & 63, W = blockDim.x >> 6;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int s = blockIdx.y;
  const int64_t C = (int64_t)p.B * p.D;
  const E* xb = (const E*)p.x + (int64_t)l.b * p.xs.bs + l.d;
  const E* gb = (const E*)p.gate + (int64_t)l.b * p.gs.bs + l.d;
  E* hb = AGG ? nullptr : (E*)p.h + (int64_t)l.b * p.hs.bs + l.d;
  const int begin = s * p.seg, stop = (int)min((int64_t)p.T, (int64_t)begin + p.seg);
  const int end = LEN ? min(l.end, stop) : stop;
  float carry[V], total[V];      // AGG: carry is the map's H, total its A
  if (!AGG) {
    segment_carry<V, true>(p, l, s, gridDim.y, W, w, lds[0], carry);
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) carry[k] = 0.f, total[k] = 1.f;
  }
  const int step = W * kL;
  VE xr[kL], gr[kL];
  uint8_t rr[kL];
  if (RESET) load_resets(p, l, begin + w * kL, rr);
  load_chunk<E, V>(xb, p.xs.ts, begin + w * kL, p.T - 1, xr);
  load_chunk<E, V>(gb, p.gs.ts, begin + w * kL, p.T - 1, gr);
  int buf = 0;
  for (int t0 = begin; t0 < stop; t0 += step, buf ^= 1) {
    const int tc = t0 + w * kL;
    float a[kL][V], b[kL][V], A[V], H[V];
    const uint32_t clear = RESET ? reset_bits(rr, tc, end) : 0u;
    // most chunks hold kL steps of every channel and no reset
    const bool whole = !(LEN ? __any(tc + kL > end) : tc + kL > end), plain = whole && !(RESET && __any(clear != 0));
    if (!whole) mask_chunk<E, V>(gr, xr, tc, end);
#pragma unroll
    for (int k = 0; k < V; ++k) A[k] = 1.f, H[k] = 0.f;
#pragma unroll
    for (int i = 0; i < kL; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        float z;
        gates((float)gr[i][k], z, a[i][k]);
        b[i][k] = z * (float)xr[i][k];
      }
    if (!RESET || plain) {
#pragma unroll
      for (int i = 0; i < kL; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) H[k] = fmaf(a[i][k], H[k], b[i][k]), A[k] *= a[i][k];
    } else {
#pragma unroll
      for (int i = 0; i < kL; ++i) {
        const bool c = clear >> i & 1;
#pragma unroll
        for (int k = 0; k < V; ++k) {
          H[k] = c ? b[i][k] : fmaf(a[i][k], H[k], b[i][k]);
          A[k] = c ? -1.f : A[k] * a[i][k];     // (keeps its sign)
        }
      }
    }
    // the next window's loads fly over the exchange and the second run
    if (t0 + step < stop) {
      if (RESET) load_resets(p, l, tc + step, rr);
      load_chunk<E, V>(xb, p.xs.ts, tc + step, p.T - 1, xr);
      load_chunk<E, V>(gb, p.gs.ts, tc + step, p.T - 1, gr);
    }
#pragma unroll
    for (int k = 0; k < V; ++k) lds[buf][w][lane * V + k] = float2{A[k], H[k]};
    __syncthreads();   // the other buffer is free again: every wave has passed its last read of it
    float h[V];
#pragma unroll
    for (int k = 0; k < V; ++k) h[k] = carry[k];
    for (int j = 0; j < W; ++j) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float2 m = lds[buf][j][lane * V + k];
        carry[k] = fold(carry[k], m.x, m.y);
        if (AGG) total[k] = chain(total[k], m.x);
        if (!AGG && j + 1 == w) h[k] = carry[k];
      }
    }
    if (AGG) continue;
    if (p.chk && tc % kKeep == 0 && tc < stop && l.on) {
      typename Vec<float, V>::type v;
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] = h[k];
      store<float, V>(p.chk + (int64_t)(tc / kKeep) * C + l.c, v);
    }
    E* o = hb + (int64_t)tc * p.hs.ts;
    if (plain) {
#pragma unroll
      for (int i = 0; i < kL; ++i) {
        VE v;
#pragma unroll
        for (int k = 0; k < V; ++k) h[k] = fmaf(a[i][k], h[k], b[i][k]), v[k] = (E)h[k];
        if (l.on) store<E, V>(o + i * p.hs.ts, v);
      }
      continue;
    }
#pragma unroll
    for (int i = 0; i < kL; ++i) {
      VE v;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        if (RESET && (clear >> i & 1)) h[k] = b[i][k];
        else h[k] = fmaf(a[i][k], h[k], b[i][k]);
        v[k] = (E)(LEN && tc + i >= end ? 0.f : h[k]);
      }
      if (tc + i < stop && l.on) store<E, V>(o + i * p.hs.ts, v);
    }
  }
  if (w == 0 && l.on) {
    if (AGG) {
#pragma unroll
      for (int k = 0; k < V; ++k) p.agg[(int64_t)s * C + l.c + k] = float2{total[k], carry[k]};
    } else if (p.last && s == (int)gridDim.y - 1) {
#pragma unroll
      for (int k = 0; k < V; ++k) p.last[l.c + k] = carry[k];
    }
  }
}

// Backward, from the last window to the first.  The map of a step acts on R_t = (1 - z_{t+1}) k_{t+1}
// G_{t+1}, what comes from behind: R_{t-1} = a_t k_t (dh_t + R_t).
template <typename ET, int V, bool RESET, bool LEN, bool AGG>
__global__ __launch_bounds__(64 * kMaxWaves) void gated_scan_bwd_kernel(const Args p) {
  typedef typename Elem<ET>::type E;
  typedef typename Vec<E, V>::type VE;
  __shared__ float2 lds[2][kMaxWaves][kWave * V];
  __shared__ float ldh[2][AGG ? 1 : kMaxWaves][kWave * V];   // the maps' H, forward
  const Lane l = lane_of<V, LEN>(p);
  const int lane = threadIdx.x & 63, W = blockDim.x >> 6;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int s = blockIdx.y;
  const int64_t C = (int64_t)p.B * p.D;
  const E* xb = (const E*)p.x + (int64_t)l.b * p.xs.bs + l.d;
  const E* gb = (const E*)p.gate + (int64_t)l.b * p.gs.bs + l.d;
  const E* db = (const E*)p.dh + (int64_t)l.b * p.hs.bs + l.d;
  const int begin = s * p.seg, stop = (int)min((int64_t)p.T, (int64_t)begin + p.seg);
  const int end = LEN ? min(l.end, stop) : stop;
  float carry[V], total[V];
  if (!AGG) {
    segment_carry<V, false>(p, l, s, gridDim.y, W, w, lds[0], carry);
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) carry[k] = 0.f, total[k] = 1.f;
  }
  const int step = W * kL;
  const int windows = (stop - begin + step - 1) / step;
  VE xr[kL], gr[kL], dr[kL];
  uint8_t rr[kL];
  {
    const int tc = begin + (windows - 1) * step + w * kL;
    if (RESET) load_resets(p, l, tc, rr);
    if (!AGG) load_chunk<E, V>(xb, p.xs.ts, tc, p.T - 1, xr);
    load_chunk<E, V>(gb, p.gs.ts, tc, p.T - 1, gr);
    load_chunk<E, V>(db, p.hs.ts, tc, p.T - 1, dr);
  }
  int buf = 0;
  for (int n = windows - 1; n >= 0; --n, buf ^= 1) {
    const int tc = begin + n * step + w * kL;
    float a[kL][V], z[kL][V], x[kL][V], d[kL][V], A[V], R[V], H[V];
    const uint32_t clear = RESET ? reset_bits(rr, tc, end) : 0u;
    const bool whole = !(LEN ? __any(tc + kL > end) : tc + kL > end), plain = whole && !(RESET && __any(clear != 0));
    if (!whole) {
      mask_chunk<E, V>(gr, dr, tc, end);
      if (!AGG) mask_chunk<E, V>(gr, xr, tc, end);
    }
    float h[V];                    // the state this window starts from; every wave folds up to its own steps
    if (!AGG) {
      const typename Vec<float, V>::type v = load<float, V>(p.chk + (int64_t)((tc - w * kL) / kKeep) * C + l.c);
#pragma unroll
      for (int k = 0; k < V; ++k) h[k] = v[k];
    }
#pragma unroll
    for (int k = 0; k < V; ++k) A[k] = 1.f, R[k] = 0.f, H[k] = 0.f;
#pragma unroll
    for (int i = 0; i < kL; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        gates((float)gr[i][k], z[i][k], a[i][k]);
        d[i][k] = (float)dr[i][k];
        if (!AGG) x[i][k] = (float)xr[i][k];
      }
    if (!RESET || plain) {
#pragma unroll
      for (int i = kL - 1; i >= 0; --i)
#pragma unroll
        for (int k = 0; k < V; ++k) R[k] = a[i][k] * (d[i][k] + R[k]), A[k] *= a[i][k];
      if (!AGG)
#pragma unroll
        for (int i = 0; i < kL; ++i)
#pragma unroll
          for (int k = 0; k < V; ++k) H[k] = fmaf(a[i][k], H[k], z[i][k] * x[i][k]);
    } else {
#pragma unroll
      for (int i = kL - 1; i >= 0; --i) {
        const bool c = clear >> i & 1;
#pragma unroll
        for (int k = 0; k < V; ++k) {
          R[k] = c ? 0.f : a[i][k] * (d[i][k] + R[k]);
          A[k] = c ? -1.f : A[k] * a[i][k];     // (keeps its sign)
        }
      }
      if (!AGG)
#pragma unroll
        for (int i = 0; i < kL; ++i) {
          const bool c = clear >> i & 1;
#pragma unroll
          for (int k = 0; k < V; ++k) H[k] = fmaf(a[i][k], c ? 0.f : H[k], z[i][k] * x[i][k]);
        }
    }
    if (n > 0) {
      if (RESET) load_resets(p, l, tc - step, rr);
      if (!AGG) load_chunk<E, V>(xb, p.xs.ts, tc - step, p.T - 1, xr);
      load_chunk<E, V>(gb, p.gs.ts, tc - step, p.T - 1, gr);
      load_chunk<E, V>(db, p.hs.ts, tc - step, p.T - 1, dr);
    }
#pragma unroll
    for (int k = 0; k < V; ++k) {
      lds[buf][w][lane * V + k] = float2{A[k], R[k]};
      if (!AGG) ldh[buf][w][lane * V + k] = H[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < V; ++k) R[k] = carry[k];
    for (int j = W - 1; j >= 0; --j) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float2 m = lds[buf][j][lane * V + k];
        carry[k] = fold(carry[k], m.x, m.y);
        if (AGG) total[k] = chain(total[k], m.x);
        if (!AGG && j - 1 == w) R[k] = carry[k];
      }
    }
    if (AGG) continue;
    for (int j = 0; j < w; ++j)
#pragma unroll
      for (int k = 0; k < V; ++k) h[k] = fold(h[k], lds[buf][j][lane * V + k].x, ldh[buf][j][lane * V + k]);
    E* ox = (E*)p.dx + (int64_t)l.b * p.dxs.bs + l.d + (int64_t)tc * p.dxs.ts;
    E* og = (E*)p.dgate + (int64_t)l.b * p.dgs.bs + l.d + (int64_t)tc * p.dgs.ts;
    // x becomes dgate_t / G_t
    if (plain) {
#pragma unroll
      for (int i = 0; i < kL; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float b = z[i][k] * x[i][k];
          x[i][k] = (x[i][k] - h[k]) * (z[i][k] * a[i][k]);
          h[k] = fmaf(a[i][k], h[k], b);
        }
#pragma unroll
      for (int i = kL - 1; i >= 0; --i) {
        VE vx, vg;
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float G = d[i][k] + R[k];
          vx[k] = (E)(z[i][k] * G);
          vg[k] = (E)(x[i][k] * G);
          R[k] = a[i][k] * G;
        }
        if (l.on) {
          store<E, V>(ox + i * p.dxs.ts, vx);
          store<E, V>(og + i * p.dgs.ts, vg);
        }
      }
      continue;
    }
#pragma unroll
    for (int i = 0; i < kL; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        if (RESET && (clear >> i & 1)) h[k] = 0.f;
        const float b = z[i][k] * x[i][k];
        x[i][k] = (x[i][k] - h[k]) * (z[i][k] * a[i][k]);
        h[k] = fmaf(a[i][k], h[k], b);
      }
#pragma unroll
    for (int i = kL - 1; i >= 0; --i) {
      VE vx, vg;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const bool live = !LEN || tc + i < end;
        const float G = d[i][k] + R[k];
        vx[k] = (E)(live ? z[i][k] * G : 0.f);
        vg[k] = (E)(live ? x[i][k] * G : 0.f);
        R[k] = RESET && (clear >> i & 1) ? 0.f : a[i][k] * G;
      }
      if (tc + i < stop && l.on) {
        store<E, V>(ox + i * p.dxs.ts, vx);
        store<E, V>(og + i * p.dgs.ts, vg);
      }
    }
  }
  if (w == 0 && l.on) {
    if (AGG) {
#pragma unroll
      for (int k = 0; k < V; ++k) p.agg[(int64_t)s * C + l.c + k] = float2{total[k], carry[k]};
    } else if (p.last && s == 0) {
#pragma unroll
      for (int k = 0; k < V; ++k) p.last[l.c + k] = carry[k];
    }
  }
}

// One step: read x, gate and the state, write the state and the output; one lane per V channels.
template <typename ET, int V>
__global__ __launch_bounds__(256) void gated_scan_step_kernel(
    const void* __restrict__ xp, int64_t xbs, const void* __restrict__ gp, int64_t gbs,
    const uint8_t* __restrict__ reset, float* __restrict__ state, void* __restrict__ yp, int64_t C, int D) {
  typedef typename Elem<ET>::type E;
  const E *x = (const E*)xp, *gate = (const E*)gp;
  E* y = (E*)yp;
  typedef typename Vec<E, V>::type VE;
  typedef typename Vec<float, V>::type VF;
  const int64_t c = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V;
  if (c >= C) return;
  const int64_t b = c / D, d = c - b * D;
  const VE xv = *reinterpret_cast<const VE*>(x + b * xbs + d);
  const VE gv = *reinterpret_cast<const VE*>(gate + b * gbs + d);
  VF h = *reinterpret_cast<const VF*>(state + c);
  const bool clear = reset && reset[b];
  VE o;
#pragma unroll
  for (int k = 0; k < V; ++k) {
    float z, a;
    gates((float)gv[k], z, a);
    const float in = z * (float)xv[k];
    h[k] = clear ? in : fmaf(a, h[k], in);
    o[k] = (E)h[k];
  }
  *reinterpret_cast<VF*>(state + c) = h;
  *reinterpret_cast<VE*>(y + c) = o;
}

// ------------------------------------------------------------------------------------ host side
enum { F32 = 0, BF16 = 1, F16 = 2 };

struct Plan {
  int W, S, seg;
};

// A lane takes 4 bytes of a row: two 16-bit channels.  (8 bytes of f32: 192 registers, and a scan of 85 x 32 x 512 took 24 us
// both ways instead of 20.)
int channels(int size, int64_t D) { return size == 2 && D > 1 ? 2 : 1; }
int64_t tiles_of(int64_t B, int64_t D, int V) { return ceil_div(B * ceil_div(D, V), kWave); }

// W: waves that share the channels of one tile: 4 where the tiles fill the chip, else 8 (or what T needs).  S: segments
// along time.  A single segment reads the streams once; S > 1 reads them twice and adds a launch each way, so it needs idle CUs
// and windows that S segments take off the chain.  Both directions in f32 (bf16), one segment -> split: 48 tiles of 128 steps 12.6 ->
// 16.1 us (15.5 -> 18.8), of 256 20.5 -> 16.9 (26.5 -> 20.0); 64 of 256 21.0 -> 17.7 (26.7 -> 20.5); 96 of 256 21.9 -> 22.8 (27.9 -> 31), of
// 512 38.3 -> 36.4 (49.7 -> 50.2), of 1024 69 -> 56 (92 -> 73); 128 of 512 38.3 -> 40.9 (49.8 -> 54.6), of 1024 69 -> 69 (92 -> 88),
// of 2048 145 -> 134 (179 -> 157); 144 of 2048 153 -> 175 (184 -> 218).
Plan plan_of(int64_t T, int64_t tiles) {
  Plan q;
  q.W = (int)std::min<int64_t>(tiles >= 512 ? 4 : kMaxWaves, std::max<int64_t>(1, ceil_div(T, kL)));
  const int64_t window = (int64_t)q.W * kL, windows = std::max<int64_t>(1, ceil_div(T, window));
  int64_t S = 1;
  if (tiles <= 128 && windows >= (tiles <= 64 ? 4 : tiles <= 96 ? 8 : 16)) S = std::min<int64_t>({windows, ceil_div(512, tiles), (int64_t)256});
  const int64_t seg = ceil_div(windows, S) * window;
  q.S = (int)std::max<int64_t>(1, ceil_div(T, seg));
  q.seg = (int)std::min<int64_t>(seg, (int64_t)1 << 30);
  return q;
}

// Whether every row start is aligned to V elements.
bool fits(const void* ptr, Stream st, int D, int V, int size) {
  return ((uintptr_t)ptr & (V * size - 1)) == 0 && st.ts % V == 0 && st.bs % V == 0 && D % V == 0;
}

template <bool FWD, typename ET, int V, bool RESET, bool LEN>
int launch(const Args& p, const Plan& q, int64_t tiles, hipStream_t s) {
  const dim3 block(64 * q.W), grid((unsigned)tiles, (unsigned)q.S);
  if (FWD) {
    if (q.S > 1) RL_LAUNCH((gated_scan_fwd_kernel<ET, V, RESET, LEN, true>), grid, block, 0, s, p);
    RL_LAUNCH((gated_scan_fwd_kernel<ET, V, RESET, LEN, false>), grid, block, 0, s, p);
  } else {
    if (q.S > 1) RL_LAUNCH((gated_scan_bwd_kernel<ET, V, RESET, LEN, true>), grid, block, 0, s, p);
    RL_LAUNCH((gated_scan_bwd_kernel<ET, V, RESET, LEN, false>), grid, block, 0, s, p);
  }
  RL_LAUNCH_CHECK();
  return RLPYT_OK;
}

template <bool FWD, typename ET, int V>
int dispatch(const Args& p, hipStream_t s) {
  const int64_t tiles = tiles_of(p.B, p.D, V);
  const Plan q = plan_of(p.T, tiles);
  Args a = p;
  a.seg = q.seg;
  if (p.reset && p.lengths) return launch<FWD, ET, V, true, true>(a, q, tiles, s);
  if (p.reset) return launch<FWD, ET, V, true, false>(a, q, tiles, s);
  if (p.lengths) return launch<FWD, ET, V, false, true>(a, q, tiles, s);
  return launch<FWD, ET, V, false, false>(a, q, tiles, s);
}

template <bool FWD, typename ET>
int pick(const Args& p, hipStream_t s) {
  typedef typename Elem<ET>::type E;
  if constexpr (sizeof(E) == 2) {
    if (channels(2, p.D) == 2) return dispatch<FWD, ET, 2>(p, s);
  }
  return dispatch<FWD, ET, 1>(p, s);
}

bool sizes_ok(int64_t T, int64_t B, int64_t D) {
  // (a launch holds less than 2^32 threads: 8 per channel at most)
  return T >= 0 && B >= 0 && D >= 0 && T < (1 << 30) && B < (1 << 30) && D < (1 << 30) &&
         (B == 0 || D == 0 || B * D <= (int64_t)1 << 28);
}

}  // namespace
}  // namespace rlpyt

using namespace rlpyt;

extern "C" int64_t rlpyt_gated_scan_state_rows(int64_t T) { return T <= 0 ? 0 : ceil_div(T, kKeep); }

extern "C" int64_t rlpyt_gated_scan_workspace_bytes(int64_t T, int64_t B, int64_t D) {
  if (!sizes_ok(T, B, D) || T == 0 || B == 0 || D == 0) return 0;
  int64_t S = 1;      // (of either element size)
  for (int size : {2, 4}) S = std::max<int64_t>(S, plan_of(T, tiles_of(B, D, channels(size, D))).S);
  return S > 1 ? S * B * D * (int64_t)sizeof(float2) : 0;
}

extern "C" int rlpyt_gated_scan_fwd(int dtype, const void* x, int64_t x_ts, int64_t x_bs, const void* gate,
                                    int64_t g_ts, int64_t g_bs, const float* h0, const uint8_t* reset,
                                    const int64_t* lengths, void* h, int64_t h_ts, int64_t h_bs, float* hn,
                                    float* states, int64_t T, int64_t B, int64_t D, void* workspace,
                                    rlpyt_stream_t stream) {
  RL_CHECK_ARG(dtype >= F32 && dtype <= F16, RLPYT_EINVAL, "rlpyt_gated_scan_fwd: unknown dtype %d", dtype);
  RL_CHECK_ARG(sizes_ok(T, B, D), RLPYT_ESHAPE, "rlpyt_gated_scan_fwd: T=%ld B=%ld D=%ld out of range",
               (long)T, (long)B, (long)D);
  if (T == 0 || B == 0 || D == 0) return RLPYT_OK;
  RL_CHECK_ARG(x && gate && h, RLPYT_EINVAL, "rlpyt_gated_scan_fwd: null pointer");
  RL_CHECK_ARG(workspace || rlpyt_gated_scan_workspace_bytes(T, B, D) == 0, RLPYT_EINVAL,
               "rlpyt_gated_scan_fwd: null workspace");
  Args p = {};
  p.x = x, p.gate = gate, p.h = h;
  p.xs = {x_ts, x_bs}, p.gs = {g_ts, g_bs}, p.hs = {h_ts, h_bs};
  p.first = h0, p.last = hn, p.reset = reset, p.lengths = lengths, p.chk = states;
  p.agg = (float2*)workspace;
  p.T = (int)T, p.B = (int)B, p.D = (int)D;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == F32) return pick<true, float>(p, s);
  if (dtype == BF16) return pick<true, Bf16>(p, s);
  return pick<true, Half>(p, s);
}

extern "C" int rlpyt_gated_scan_bwd(int dtype, const void* x, int64_t x_ts, int64_t x_bs, const void* gate,
                                    int64_t g_ts, int64_t g_bs, const void* dh, int64_t d_ts, int64_t d_bs,
                                    const float* dhn, const uint8_t* reset, const int64_t* lengths,
                                    const float* states, void* dx, int64_t dx_ts, int64_t dx_bs, void* dgate,
                                    int64_t dg_ts, int64_t dg_bs, float* dh0, int64_t T, int64_t B, int64_t D,
                                    void* workspace, rlpyt_stream_t stream) {
  RL_CHECK_ARG(dtype >= F32 && dtype <= F16, RLPYT_EINVAL, "rlpyt_gated_scan_bwd: unknown dtype %d", dtype);
  RL_CHECK_ARG(sizes_ok(T, B, D), RLPYT_ESHAPE, "rlpyt_gated_scan_bwd: T=%ld B=%ld D=%ld out of range",
               (long)T, (long)B, (long)D);
  if (T == 0 || B == 0 || D == 0) return RLPYT_OK;
  RL_CHECK_ARG(x && gate && dh && states && dx && dgate, RLPYT_EINVAL, "rlpyt_gated_scan_bwd: null pointer");
  RL_CHECK_ARG(workspace || rlpyt_gated_scan_workspace_bytes(T, B, D) == 0, RLPYT_EINVAL,
               "rlpyt_gated_scan_bwd: null workspace");
  Args p = {};
  p.x = x, p.gate = gate, p.dh = dh, p.dx = dx, p.dgate = dgate;
  p.xs = {x_ts, x_bs}, p.gs = {g_ts, g_bs}, p.hs = {d_ts, d_bs}, p.dxs = {dx_ts, dx_bs}, p.dgs = {dg_ts, dg_bs};
  p.first = dhn, p.last = dh0, p.reset = reset, p.lengths = lengths, p.chk = const_cast<float*>(states);
  p.agg = (float2*)workspace;
  p.T = (int)T, p.B = (int)B, p.D = (int)D;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == F32) return pick<false, float>(p, s);
  if (dtype == BF16) return pick<false, Bf16>(p, s);
  return pick<false, Half>(p, s);
}

namespace {
template <typename ET>
int step_of(const void* x, int64_t xbs, const void* gate, int64_t gbs, const uint8_t* reset, float* state,
            void* y, int64_t B, int64_t D, hipStream_t s) {
  typedef typename Elem<ET>::type E;
  const Stream xs = {0, xbs}, gs = {0, gbs}, dense = {0, D};
  const int64_t C = B * D;
  const int size = (int)sizeof(E);
  const bool wide = fits(x, xs, (int)D, 2, size) && fits(gate, gs, (int)D, 2, size) && fits(y, dense, (int)D, 2, size) &&
                    fits(state, dense, (int)D, 2, 4);
  if (wide)
    RL_LAUNCH((gated_scan_step_kernel<ET, 2>), dim3((unsigned)ceil_div(C, 512)), dim3(256), 0, s, x, xbs,
              gate, gbs, reset, state, y, C, (int)D);
  else
    RL_LAUNCH((gated_scan_step_kernel<ET, 1>), dim3((unsigned)ceil_div(C, 256)), dim3(256), 0, s, x, xbs,
              gate, gbs, reset, state, y, C, (int)D);
  RL_LAUNCH_CHECK();
  return RLPYT_OK;
}
}  // namespace

extern "C" int rlpyt_gated_scan_step(int dtype, const void* x, int64_t x_bs, const void* gate, int64_t g_bs,
                                     const uint8_t* reset, float* state, void* y, int64_t B, int64_t D,
                                     rlpyt_stream_t stream) {
  RL_CHECK_ARG(dtype >= F32 && dtype <= F16, RLPYT_EINVAL, "rlpyt_gated_scan_step: unknown dtype %d", dtype);
  RL_CHECK_ARG(sizes_ok(1, B, D), RLPYT_ESHAPE, "rlpyt_gated_scan_step: B=%ld D=%ld out of range", (long)B, (long)D);
  if (B == 0 || D == 0) return RLPYT_OK;
  RL_CHECK_ARG(x && gate && state && y, RLPYT_EINVAL, "rlpyt_gated_scan_step: null pointer");
  hipStream_t s = (hipStream_t)stream;
  if (dtype == F32) return step_of<float>(x, x_bs, gate, g_bs, reset, state, y, B, D, s);
  if (dtype == BF16) return step_of<Bf16>(x, x_bs, gate, g_bs, reset, state, y, B, D, s);
  return step_of<Half>(x, x_bs, gate, g_bs, reset, state, y, B, D, s);
}
