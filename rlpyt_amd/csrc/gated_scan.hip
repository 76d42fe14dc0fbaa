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
// A reset forgets whatever came before, also a state that is not finite: such a map carries A = -1
// (a product of sigmoids is never negative) and composes as "H alone", not as 0 * h.
//
// States, maps and sums are 32 bits; x, gate, h and the gradients are f32, bf16 or f16 and each output is
// rounded once.  The backward pass starts from f32 states kept every kL steps and recomputes the others:
// reading h back would be 2 (4) bytes per element more and, for 16-bit streams, a rounded state.
#include <algorithm>

#include "common.h"

namespace rlpyt {
namespace {

constexpr int kL = 8;         // steps per wave and window = distance of the kept states
constexpr int kMaxWaves = 8;  // waves (consecutive kL-step chunks) per workgroup

template <typename E, int V>
struct Vec {
  typedef E type __attribute__((ext_vector_type(V)));
  typedef float ftype __attribute__((ext_vector_type(V)));
};

struct Stream {   // one [T, B, D] tensor: unit stride along D, element strides along T and B
  int64_t ts, bs;
};

// 1 / (1 + e^-g) and its complement, both to f32's relative accuracy
__device__ __forceinline__ void gates(float g, float& z, float& a) {
  const float e = __expf(-fabsf(g));          // NaN gates stay NaN
  const float r = __builtin_amdgcn_rcpf(1.f + e), s = e * r;
  z = g >= 0.f ? r : s;
  a = g >= 0.f ? s : r;
  if (g != g) z = a = g;
}

__device__ __forceinline__ float fold(float c, float A, float H) {
  return A < 0.f ? H : fmaf(A, c, H);
}

struct Args {
  const void *x, *gate, *dh;       // dh: backward only; strides 0 are fine
  void *h, *dx, *dgate;            // h: forward only
  Stream xs, gs, hs, dxs, dgs;     // hs: of h (forward) / dh (backward)
  const float* first;              // h0 (forward) / dhn (backward) [B D] or null
  float* last;                     // hn (forward) / dh0 (backward) [B D] or null
  const uint8_t* reset;            // [T, B] or null
  const int64_t* lengths;          // [B] or null
  float* chk;                      // f32 states before steps 0, kL, 2 kL, .. [ceil(T / kL), B D] or null
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
  const int64_t C = (int64_t)p.B * p.D;
  l.c = ((int64_t)blockIdx.x * kWave + (threadIdx.x & 63)) * V;
  l.on = l.c < C;                              // V divides D: a lane is in or out as a whole
  const int64_t c = l.on ? l.c : 0;
  l.b = (int)(c / p.D);
  l.d = (int)(c - (int64_t)l.b * p.D);
  l.end = p.T;
  if (LEN) l.end = (int)min((int64_t)p.T, max((int64_t)0, p.lengths[l.b]));
  return l;
}

// kL rows from step t0 on; rows behind the last one are read as the last one and masked by the caller.
template <typename E, int V>
__device__ __forceinline__ void load_chunk(const E* __restrict__ base, int64_t ts, int t0, int last,
                                           typename Vec<E, V>::type (&out)[kL]) {
  typedef typename Vec<E, V>::type VE;
#pragma unroll
  for (int i = 0; i < kL; ++i)
    out[i] = *reinterpret_cast<const VE*>(base + (int64_t)min(t0 + i, last) * ts);
}

// Bit i: the state is cleared before step t0 + i.
__device__ __forceinline__ uint32_t load_resets(const Args& p, const Lane& l, int t0, int end) {
  uint32_t clear = 0;
#pragma unroll
  for (int i = 0; i < kL; ++i) {
    const bool r = p.reset[(int64_t)min(t0 + i, p.T - 1) * p.B + l.b] != 0;
    clear |= (uint32_t)(r && t0 + i < end) << i;
  }
  return clear;
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
    for (int j = lo; j < hi; ++j) {
      const float2* q = p.agg + (int64_t)(FWD ? j : S - 1 - j) * C + l.c;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float2 m = q[k];
        H[k] = fold(H[k], m.x, m.y);
        A[k] = m.x < 0.f || A[k] < 0.f ? -1.f : A[k] * m.x;
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
template <typename E, int V, bool RESET, bool LEN, bool AGG>
__global__ __launch_bounds__(64 * kMaxWaves) void gated_scan_fwd_kernel(const Args p) {
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
  load_chunk<E, V>(xb, p.xs.ts, begin + w * kL, p.T - 1, xr);
  load_chunk<E, V>(gb, p.gs.ts, begin + w * kL, p.T - 1, gr);
  int buf = 0;
  for (int t0 = begin; t0 < stop; t0 += step, buf ^= 1) {
    const int tc = t0 + w * kL;
    float a[kL][V], b[kL][V], A[V], H[V];
    const uint32_t clear = RESET ? load_resets(p, l, tc, end) : 0u;
#pragma unroll
    for (int k = 0; k < V; ++k) A[k] = 1.f, H[k] = 0.f;
#pragma unroll
    for (int i = 0; i < kL; ++i) {
      const bool live = tc + i < end;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        float z, q;
        gates((float)gr[i][k], z, q);
        a[i][k] = live ? q : 1.f;
        b[i][k] = live ? z * (float)xr[i][k] : 0.f;
        if (RESET && (clear >> i & 1)) {
          A[k] = -1.f;
          H[k] = b[i][k];
        } else {
          H[k] = fmaf(a[i][k], H[k], b[i][k]);
          A[k] = A[k] < 0.f ? -1.f : A[k] * a[i][k];
        }
      }
    }
    // the next window's loads fly over the exchange and the second run
    if (t0 + step < stop) {
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
        if (AGG) total[k] = m.x < 0.f || total[k] < 0.f ? -1.f : total[k] * m.x;
        if (!AGG && j + 1 == w) h[k] = carry[k];
      }
    }
    if (AGG) continue;
    if (p.chk && tc < stop && l.on) {
      typedef typename Vec<float, V>::type VF;
      VF v;
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] = h[k];
      *reinterpret_cast<VF*>(p.chk + (int64_t)(tc / kL) * C + l.c) = v;
    }
    E* o = hb + (int64_t)tc * p.hs.ts;
#pragma unroll
    for (int i = 0; i < kL; ++i) {
      VE v;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        if (RESET && (clear >> i & 1)) h[k] = b[i][k];
        else h[k] = fmaf(a[i][k], h[k], b[i][k]);
        v[k] = (E)(LEN && tc + i >= end ? 0.f : h[k]);
      }
      if (tc + i < stop && l.on) *reinterpret_cast<VE*>(o + i * p.hs.ts) = v;
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
template <typename E, int V, bool RESET, bool LEN, bool AGG>
__global__ __launch_bounds__(64 * kMaxWaves) void gated_scan_bwd_kernel(const Args p) {
  typedef typename Vec<E, V>::type VE;
  __shared__ float2 lds[2][kMaxWaves][kWave * V];
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
  {
    const int tc = begin + (windows - 1) * step + w * kL;
    if (!AGG) load_chunk<E, V>(xb, p.xs.ts, tc, p.T - 1, xr);
    load_chunk<E, V>(gb, p.gs.ts, tc, p.T - 1, gr);
    load_chunk<E, V>(db, p.hs.ts, tc, p.T - 1, dr);
  }
  int buf = 0;
  for (int n = windows - 1; n >= 0; --n, buf ^= 1) {
    const int tc = begin + n * step + w * kL;
    float a[kL][V], z[kL][V], e[kL][V], d[kL][V], A[V], R[V];
    const uint32_t clear = RESET ? load_resets(p, l, tc, end) : 0u;
    float h[V];
#pragma unroll
    for (int k = 0; k < V; ++k) h[k] = 0.f;
    if (!AGG && tc < stop && l.on) {
      typedef typename Vec<float, V>::type VF;
      const VF v = *reinterpret_cast<const VF*>(p.chk + (int64_t)(tc / kL) * C + l.c);
#pragma unroll
      for (int k = 0; k < V; ++k) h[k] = v[k];
    }
#pragma unroll
    for (int i = 0; i < kL; ++i) {
      const bool live = tc + i < end;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        gates((float)gr[i][k], z[i][k], a[i][k]);
        if (!live) a[i][k] = 1.f, z[i][k] = 0.f;
        d[i][k] = live ? (float)dr[i][k] : 0.f;
        if (!AGG) {
          if (RESET && (clear >> i & 1)) h[k] = 0.f;
          const float x = live ? (float)xr[i][k] : 0.f;
          e[i][k] = (x - h[k]) * z[i][k] * a[i][k];
          h[k] = fmaf(a[i][k], h[k], z[i][k] * x);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < V; ++k) A[k] = 1.f, R[k] = 0.f;
#pragma unroll
    for (int i = kL - 1; i >= 0; --i) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        if (RESET && (clear >> i & 1)) {
          A[k] = -1.f;
          R[k] = 0.f;
        } else {
          R[k] = a[i][k] * (d[i][k] + R[k]);
          A[k] = A[k] < 0.f ? -1.f : A[k] * a[i][k];
        }
      }
    }
    if (n > 0) {
      if (!AGG) load_chunk<E, V>(xb, p.xs.ts, tc - step, p.T - 1, xr);
      load_chunk<E, V>(gb, p.gs.ts, tc - step, p.T - 1, gr);
      load_chunk<E, V>(db, p.hs.ts, tc - step, p.T - 1, dr);
    }
#pragma unroll
    for (int k = 0; k < V; ++k) lds[buf][w][lane * V + k] = float2{A[k], R[k]};
    __syncthreads();
#pragma unroll
    for (int k = 0; k < V; ++k) R[k] = carry[k];
    for (int j = W - 1; j >= 0; --j) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float2 m = lds[buf][j][lane * V + k];
        carry[k] = fold(carry[k], m.x, m.y);
        if (AGG) total[k] = m.x < 0.f || total[k] < 0.f ? -1.f : total[k] * m.x;
        if (!AGG && j - 1 == w) R[k] = carry[k];
      }
    }
    if (AGG) continue;
    E* ox = (E*)p.dx + (int64_t)l.b * p.dxs.bs + l.d + (int64_t)tc * p.dxs.ts;
    E* og = (E*)p.dgate + (int64_t)l.b * p.dgs.bs + l.d + (int64_t)tc * p.dgs.ts;
#pragma unroll
    for (int i = kL - 1; i >= 0; --i) {
      VE vx, vg;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const bool live = !LEN || tc + i < end;
        const float G = d[i][k] + R[k];
        vx[k] = (E)(live ? z[i][k] * G : 0.f);
        vg[k] = (E)(live ? e[i][k] * G : 0.f);
        R[k] = RESET && (clear >> i & 1) ? 0.f : a[i][k] * G;
      }
      if (tc + i < stop && l.on) {
        *reinterpret_cast<VE*>(ox + i * p.dxs.ts) = vx;
        *reinterpret_cast<VE*>(og + i * p.dgs.ts) = vg;
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
template <typename E, int V>
__global__ __launch_bounds__(256) void gated_scan_step_kernel(
    const E* __restrict__ x, int64_t xbs, const E* __restrict__ gate, int64_t gbs,
    const uint8_t* __restrict__ reset, float* __restrict__ state, E* __restrict__ y, int64_t C, int D) {
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

// W: waves that share the channels of one tile, at most kMaxWaves.  S: segments along time.  A single
// segment reads the streams once; S > 1 reads them twice and adds a launch, so it is taken only where the tiles alone
// leave most of the 256 CUs idle.
Plan plan_of(int64_t T, int64_t tiles) {
  Plan q;
  q.W = (int)std::min<int64_t>(kMaxWaves, std::max<int64_t>(1, ceil_div(T, kL)));
  const int64_t window = (int64_t)q.W * kL, windows = std::max<int64_t>(1, ceil_div(T, window));
  int64_t S = 1;
  if (tiles < 128) S = std::min<int64_t>({windows, ceil_div(512, tiles), (int64_t)256});
  const int64_t seg = ceil_div(windows, S) * window;
  q.S = (int)std::max<int64_t>(1, ceil_div(T, seg));
  q.seg = (int)std::min<int64_t>(seg, (int64_t)1 << 30);
  return q;
}

// The widest vector (<= 4 bytes of 16-bit, 4 .. 8 bytes of f32 elements) that every row start is aligned to.
bool fits(const void* ptr, Stream st, int D, int V, int size) {
  return ((uintptr_t)ptr & (V * size - 1)) == 0 && st.ts % V == 0 && st.bs % V == 0 && D % V == 0;
}

template <bool FWD, typename E, int V, bool RESET, bool LEN>
int launch(const Args& p, const Plan& q, int64_t tiles, hipStream_t s) {
  const dim3 block(64 * q.W), grid((unsigned)tiles, (unsigned)q.S);
  if (FWD) {
    if (q.S > 1) RL_LAUNCH((gated_scan_fwd_kernel<E, V, RESET, LEN, true>), grid, block, 0, s, p);
    RL_LAUNCH((gated_scan_fwd_kernel<E, V, RESET, LEN, false>), grid, block, 0, s, p);
  } else {
    if (q.S > 1) RL_LAUNCH((gated_scan_bwd_kernel<E, V, RESET, LEN, true>), grid, block, 0, s, p);
    RL_LAUNCH((gated_scan_bwd_kernel<E, V, RESET, LEN, false>), grid, block, 0, s, p);
  }
  RL_LAUNCH_CHECK();
  return RLPYT_OK;
}

template <bool FWD, typename E, int V>
int dispatch(const Args& p, hipStream_t s) {
  const int64_t tiles = ceil_div((int64_t)p.B * p.D, (int64_t)kWave * V);
  const Plan q = plan_of(p.T, tiles);
  Args a = p;
  a.seg = q.seg;
  if (p.reset && p.lengths) return launch<FWD, E, V, true, true>(a, q, tiles, s);
  if (p.reset) return launch<FWD, E, V, true, false>(a, q, tiles, s);
  if (p.lengths) return launch<FWD, E, V, false, true>(a, q, tiles, s);
  return launch<FWD, E, V, false, false>(a, q, tiles, s);
}

template <bool FWD, typename E>
int pick(const Args& p, hipStream_t s) {
  const int size = (int)sizeof(E);
  const bool wide = fits(p.x, p.xs, p.D, 2, size) && fits(p.gate, p.gs, p.D, 2, size) &&
                    fits(FWD ? p.h : p.dh, p.hs, p.D, 2, size) &&
                    (FWD || (fits(p.dx, p.dxs, p.D, 2, size) && fits(p.dgate, p.dgs, p.D, 2, size)));
  if (wide) return dispatch<FWD, E, 2>(p, s);
  return dispatch<FWD, E, 1>(p, s);
}

bool sizes_ok(int64_t T, int64_t B, int64_t D) {
  // (a launch holds less than 2^32 threads: 8 per channel at most)
  return T >= 0 && B >= 0 && D >= 0 && T < (1 << 30) && B < (1 << 30) && D < (1 << 30) &&
         (B == 0 || D == 0 || B * D <= (int64_t)1 << 28);
}

}  // namespace
}  // namespace rlpyt

using namespace rlpyt;

extern "C" int64_t rlpyt_gated_scan_state_rows(int64_t T) { return T <= 0 ? 0 : ceil_div(T, kL); }

extern "C" int64_t rlpyt_gated_scan_workspace_bytes(int64_t T, int64_t B, int64_t D) {
  if (!sizes_ok(T, B, D) || T == 0 || B == 0 || D == 0) return 0;
  // the narrow variant has more tiles, hence fewer segments: the wide one's count bounds both
  const Plan q = plan_of(T, ceil_div(B * D, (int64_t)kWave * 2));
  const Plan n = plan_of(T, ceil_div(B * D, (int64_t)kWave));
  const int64_t S = std::max(q.S, n.S);
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
  if (dtype == BF16) return pick<true, __bf16>(p, s);
  return pick<true, _Float16>(p, s);
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
  if (dtype == BF16) return pick<false, __bf16>(p, s);
  return pick<false, _Float16>(p, s);
}

namespace {
template <typename E>
int step_of(const void* x, int64_t xbs, const void* gate, int64_t gbs, const uint8_t* reset, float* state,
            void* y, int64_t B, int64_t D, hipStream_t s) {
  const Stream xs = {0, xbs}, gs = {0, gbs}, dense = {0, D};
  const int64_t C = B * D;
  const int size = (int)sizeof(E);
  const bool wide = fits(x, xs, (int)D, 2, size) && fits(gate, gs, (int)D, 2, size) && fits(y, dense, (int)D, 2, size) &&
                    fits(state, dense, (int)D, 2, 4);
  if (wide)
    RL_LAUNCH((gated_scan_step_kernel<E, 2>), dim3((unsigned)ceil_div(C, 512)), dim3(256), 0, s, (const E*)x, xbs,
              (const E*)gate, gbs, reset, state, (E*)y, C, (int)D);
  else
    RL_LAUNCH((gated_scan_step_kernel<E, 1>), dim3((unsigned)ceil_div(C, 256)), dim3(256), 0, s, (const E*)x, xbs,
              (const E*)gate, gbs, reset, state, (E*)y, C, (int)D);
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
  if (dtype == BF16) return step_of<__bf16>(x, x_bs, gate, g_bs, reset, state, y, B, D, s);
  return step_of<_Float16>(x, x_bs, gate, g_bs, reset, state, y, B, D, s);
}
