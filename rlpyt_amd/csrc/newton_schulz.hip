// Orthogonalising matrices by Newton-Schulz products, as an optimizer does with its update:
//
//   X_0 = G / (|G|_F + eps), transposed where G is tall      A = X X^T      Q = a I + b A + c A A      X <- Q X
//
// `steps` times; the singular values of X go towards 1, its singular vectors stay.  m = min, n = max of a matrix'
// sides: 2 m^2 n + 2 m^3 + 2 m^2 n operations a step, of which the two symmetric products need half.
//
// The polynomial multiplies small singular values by `a` a step (3.44^5 = 484 over five): an error of 2^-11 relative to |X|
// (one f16 or bf16 product) would end as large as they are.  So every factor is held as two f16 pieces, hi + lo = 22 bits,
// and a product is hi hi + hi lo + lo hi on the f16 matrix pipe with f32 accumulation: three instructions of 16 x the f32
// instruction's rate.  X, A and Q are stored times 2^12, which keeps the lo pieces out of f16's subnormals (entries of X are
// ~ 1 / sqrt(m n)); their spectral norms are < 8, which the host checks for the given coefficients.
//
// Storage of a factor with K columns (padded to the tile side, pads are 0): per row and 32 columns, 64 bytes of hi and 64 of lo.
// All products are row-times-row ("A B^T"): X X^T takes X, A A takes A (symmetric), Q X takes Q and X^T, so an epilogue
// writes its tile both ways.  Symmetric products compute the tiles on and above the diagonal and mirror them.
// The matrices of a list go through each launch together: 2 + 3 steps launches for up to 32 of them.
#include <limits.h>
#include <math.h>

#include <algorithm>

#include "common.h"

namespace rlpyt {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kMats = 32;            // matrices of one launch (the table is a kernel argument)
constexpr int kBK = 32;              // columns of a stage
constexpr float kScale = 4096.f;     // 2^12, of every stored factor
constexpr int kNormBlocks = 256;     // partial sums of squares per matrix
constexpr int kCUs = 256;

struct Mat {
  const void* in;                    // [rows, cols], row stride ld
  void* out;                         // [rows, cols] dense
  int64_t ld;
  int rows, cols;
  int mp, np;                        // padded sides of X: min and max
  int tall;
  _Float16 *x, *xt[2], *a, *q;       // X [mp, np], X^T [np, mp] (two: read and written), A, Q [mp, mp]
  double* norm;                      // [kNormBlocks]
};
// The first launch gets the table as its argument and leaves it in the workspace for the others: an argument is read from the
// host's memory, 3 KB of it by every launch.
enum { LOAD = 0, SYM = 1, FULL = 2 };
struct Mats {
  Mat m[kMats];
  int first[3][kMats];               // first tile of a matrix: of ns_load_kernel, of symmetric and of full products; INT_MAX behind n
};

__device__ __forceinline__ int find(const Mats* __restrict__ t, int kind, int tile) {
  const bool behind = (threadIdx.x & 63) < kMats && t->first[kind][threadIdx.x & (kMats - 1)] <= tile;
  return __builtin_amdgcn_readfirstlane(__popcll(__ballot(behind)) - 1);
}

__global__ __launch_bounds__(256) void ns_table_kernel(const Mats t, Mats* __restrict__ table) {
  for (int i = threadIdx.x; i < (int)(sizeof(Mats) / 4); i += 256) ((uint32_t*)table)[i] = ((const uint32_t*)&t)[i];
}

template <typename E>
__global__ __launch_bounds__(256) void ns_norm_kernel(const Mats t, Mats* __restrict__ table) {
  constexpr int n16 = 16 / sizeof(E);
  typedef E vec __attribute__((ext_vector_type(n16)));
  __shared__ double scratch[16];
  if (blockIdx.x == 0 && blockIdx.y == 0)
    for (int i = threadIdx.x; i < (int)(sizeof(Mats) / 4); i += 256) ((uint32_t*)table)[i] = ((const uint32_t*)&t)[i];
  const Mat& M = t.m[blockIdx.y];
  const int64_t total = (int64_t)M.rows * M.cols, first = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const E* in = (const E*)M.in;
  double v[1] = {0.0};
  auto add = [&](E x) {
    const double g = (double)(float)x;
    v[0] = fma(g, g, v[0]);
  };
  if (M.ld == M.cols && ((uintptr_t)in & 15) == 0) {
    constexpr int U = 4;               // loads in flight
    const int64_t step = kNormBlocks * 256, n = total / n16;
    for (int64_t i = first; i < n; i += U * step) {
      vec x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int k = 0; k < n16; ++k) x[u][k] = (E)0.f;
        if (i + u * step < n) x[u] = ((const vec*)in)[i + u * step];
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int k = 0; k < n16; ++k) add(x[u][k]);
    }
    if (blockIdx.x == 0 && threadIdx.x < total % n16) add(in[total - 1 - threadIdx.x]);
  } else {
    for (int64_t i = first; i < total; i += kNormBlocks * 256) {
      const int64_t r = i / M.cols;
      add(in[r * M.ld + (i - r * M.cols)]);
    }
  }
  block_sum<1>(v, scratch);
  if (threadIdx.x == 0) M.norm[blockIdx.x] = v[0];
}

// element (r, k) of a factor with K (padded) columns: hi at the returned index, lo 32 behind it
__device__ __forceinline__ int64_t at(int64_t r, int k, int K) { return (r * (K >> 5) + (k >> 5)) * 64 + (k & 31); }

__device__ __forceinline__ void split(float v, _Float16& hi, _Float16& lo) {
  hi = (_Float16)v;
  lo = (_Float16)(v - (float)hi);
}

// X_0 and its transpose from 32 x 32 tiles of the input
template <typename E>
__global__ __launch_bounds__(256) void ns_load_kernel(const Mats* __restrict__ t, double eps) {
  __shared__ float tile[32][33];
  __shared__ float factor;
  const int i = find(t, LOAD, blockIdx.x);
  const Mat M = t->m[i];
  if (threadIdx.x < kWave) {
    double s = 0.0;
    for (int k = threadIdx.x; k < kNormBlocks; k += kWave) s += M.norm[k];
    s = wave_sum(s);
    if (threadIdx.x == 0) factor = (float)((double)kScale / (sqrt(s) + eps));
  }
  __syncthreads();
  const int block = blockIdx.x - t->first[LOAD][i], tn = M.np / 32;
  const int r0 = block / tn * 32, c0 = block % tn * 32;      // rows, columns of X
  const int lx = threadIdx.x & 31, ly = threadIdx.x >> 5;
  for (int k = ly; k < 32; k += 8) {   // coalesced along the input's rows
    const int r = M.tall ? c0 + k : r0 + k, c = M.tall ? r0 + lx : c0 + lx;
    float v = 0.f;
    if (r < M.rows && c < M.cols) v = (float)((const E*)M.in)[(int64_t)r * M.ld + c] * factor;
    if (M.tall) tile[lx][k] = v;
    else tile[k][lx] = v;
  }
  __syncthreads();
  for (int k = ly; k < 32; k += 8) {
    _Float16 hi, lo;
    split(tile[k][lx], hi, lo);
    _Float16* p = M.x + at(r0 + k, c0 + lx, M.np);
    p[0] = hi, p[32] = lo;
    split(tile[lx][k], hi, lo);
    p = M.xt[0] + at(c0 + k, r0 + lx, M.mp);
    p[0] = hi, p[32] = lo;
  }
}

enum { GRAM = 0, POLY = 1, NEXT = 2, LAST = 3 };

__device__ __forceinline__ f32x16 mfma(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

struct Where {
  int mat, tr, tc;    // matrix, tile row, tile column
};

// The tile with this number in a launch.  Symmetric products count the tiles on and above the diagonal, row by row.
template <int MODE, int T>
__device__ __forceinline__ Where where(const Mats* __restrict__ t, int tile) {
  constexpr int kind = MODE < NEXT ? SYM : FULL;
  Where w;
  w.mat = find(t, kind, tile);
  const Mat& M = t->m[w.mat];
  int k = tile - t->first[kind][w.mat];
  if (MODE == GRAM || MODE == POLY) {
    const int nt = M.mp / T;
    w.tr = 0;
    while (k >= nt - w.tr) k -= nt - w.tr, ++w.tr;
    w.tc = w.tr + k;
  } else {
    const int nt = M.mp / T;           // column by column
    w.tc = k / nt;
    w.tr = k - w.tc * nt;
  }
  return w;
}

// Workgroups go round the 8 XCDs; the tiles of one XCD's workgroups are neighbours, which share rows of the factors in its L2.
__device__ __forceinline__ int neighbours(int block, int n) {
  const int xcd = block & 7, each = n >> 3, more = n & 7;
  return xcd * each + min(xcd, more) + (block >> 3);
}

struct Coeffs {
  float a, b, c;
};

// Writes a 32 x 32 block of a product (times 2^24): D[row = (r & 3) + 8 (r >> 2) + 4 (l >> 5)][column = l & 31],
// with its upper left corner at (row0, col0).  both: also the other way round.
template <int MODE, typename E>
__device__ __forceinline__ void write_block(const Mat& M, int cur, const Coeffs& f, const f32x16& acc, int row0, int col0,
                                            bool both) {
  const int lane = threadIdx.x & 63, col = col0 + (lane & 31);
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int row = row0 + 8 * g + 4 * (lane >> 5);
    f16x4 hi, lo, ah, al;
    if (MODE == POLY) {                // A is symmetric: 4 entries of a row instead of a column
      const _Float16* p = M.a + at(col, row, M.mp);
      ah = *(const f16x4*)p, al = *(const f16x4*)(p + 32);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float v = acc[4 * g + r];
      if (MODE == LAST) {
        v *= 1.f / (kScale * kScale);
        const int orow = M.tall ? col : row + r, ocol = M.tall ? row + r : col;
        if (orow < M.rows && ocol < M.cols) ((E*)M.out)[(int64_t)orow * M.cols + ocol] = (E)v;
        continue;
      }
      if (MODE == POLY) {
        v = fmaf(f.c, v * (1.f / kScale), f.b * ((float)ah[r] + (float)al[r]));
        if (row + r == col) v += f.a * kScale;
      } else {
        v *= 1.f / kScale;
      }
      _Float16 vh, vl;
      split(v, vh, vl);
      hi[r] = vh, lo[r] = vl;
      _Float16* o = (MODE == GRAM ? M.a : MODE == POLY ? M.q : M.x) + at(row + r, col, MODE == NEXT ? M.np : M.mp);
      o[0] = vh, o[32] = vl;
    }
    if (MODE == LAST || !both) continue;
    _Float16* o = (MODE == GRAM ? M.a : MODE == POLY ? M.q : M.xt[cur ^ 1]) + at(col, row, M.mp);   // 4 consecutive columns
    *(f16x4*)o = hi;
    *(f16x4*)(o + 32) = lo;
  }
}

// This wave's loads but the last N have arrived and its reads of LDS are done; then the workgroup's barrier.  (__syncthreads
// waits for all loads.)
template <int N>
__device__ __forceinline__ void wait_and_sync() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// A workgroup's tile of T x T: waves, 32 x 32 blocks of a wave, LDS stages of 2 T rows x 128 bytes.  What bounds a stage is the
// LDS: a wave reads its rows of both factors, the loads write them.  128: 64 + 32 KB a stage against 768 cycles of matrix pipe,
// at 128 bytes a cycle all of it; 256: half of that per operation, but a matrix of 4096 has just one tile for
// each CU.  64: for few tiles.
// NS stages: two for 256 and 128.  64 x 64 tiles come where the chip is not full and a load's way from another XCD's
// results (1 us) is what counts: 4, or 8 with one workgroup a CU.
template <int T>
struct Shape {
  static constexpr int waves = T == 256 ? 8 : 4, cols = waves / 2;                   // 2 rows of waves
  static constexpr int nx = T / 64, ny = T / 32 / cols;
  static constexpr int passes = T / (8 * waves);                                     // load instructions of a wave per factor
};

// One T x T tile of P Q^T per workgroup, the factors loaded straight from memory to LDS.  The 16-byte pieces of an LDS row are
// permuted by its row number, so that the 8 lanes that are served together read 8 different ones.
// Tiles from `full` on are split along K into S slices of a workgroup each, whose sums go to `part`, 16 values of a lane
// together, for ns_finish_kernel: the tiles that would make a round of their own on an idle chip.
template <int MODE, int T, int NS, typename E>
__global__ __launch_bounds__(Shape<T>::waves * 64) void ns_product_kernel(const Mats* __restrict__ t, int cur, Coeffs f,
                                                                         int full, int S, float* __restrict__ part) {
  typedef Shape<T> G;
  constexpr int NX = G::nx, NY = G::ny, L = 2 * G::passes;
  __shared__ __attribute__((aligned(16))) uint8_t lds[NS][2][T * 128];
  const int q = (int)blockIdx.x - full;
  const Where at_ = where<MODE, T>(t, q < 0 ? neighbours(blockIdx.x, full) : full + q / S);
  const Mat M = t->m[at_.mat];
  const int tr = at_.tr, tc = at_.tc;
  const int K = MODE == GRAM ? M.np : M.mp;
  const _Float16* P = MODE == GRAM ? M.x : MODE == POLY ? M.a : M.q;
  const _Float16* Q = MODE == GRAM ? M.x : MODE == POLY ? M.a : M.xt[cur];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // a load instruction of a wave fills 1 KB = 8 rows; lane -> row l >> 3, piece (l & 7) ^ (row & 7)
  const int64_t pitch = (int64_t)K * 4;   // bytes of a row
  const uint8_t *src[2];
  src[0] = (const uint8_t*)P + (int64_t)(tr * T + wave * 8 + (lane >> 3)) * pitch + ((lane & 7) ^ (lane >> 3)) * 16;
  src[1] = (const uint8_t*)Q + (int64_t)(tc * T + wave * 8 + (lane >> 3)) * pitch + ((lane & 7) ^ (lane >> 3)) * 16;
  auto stage = [&](int s, int k) {
#pragma unroll
    for (int o = 0; o < 2; ++o)
#pragma unroll
      for (int j = 0; j < G::passes; ++j)
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) void*)(src[o] + (int64_t)(8 * G::waves * j) * pitch + (int64_t)k * 128),
            (__attribute__((address_space(3))) void*)(&lds[s][o][(8 * G::waves * j + wave * 8) * 128]), 16, 0, 0);
  };
  f32x16 acc[NX][NY];
#pragma unroll
  for (int x = 0; x < NX; ++x)
#pragma unroll
    for (int y = 0; y < NY; ++y)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[x][y][r] = 0.f;
  const int wr = wave / G::cols * (32 * NX), wc = wave % G::cols * (32 * NY);
  const int steps = K / kBK;
  const int slice = q < 0 ? 0 : q % S;
  const int begin = q < 0 ? 0 : (int)((int64_t)steps * slice / S);
  const int end = q < 0 ? steps : (int)((int64_t)steps * (slice + 1) / S);
#pragma unroll
  for (int i = 0; i < NS - 1; ++i)
    if (begin + i < end) stage(i, begin + i);
  int s = 0;
  for (int k = begin; k < end; ++k, s = s + 1 == NS ? 0 : s + 1) {
    // stage k has arrived (up to NS - 2 behind it may be on their way), and stage k - 1 has been read
    const int behind = end - 1 - k;
    if (NS == 2 || behind == 0) wait_and_sync<0>();
    else if (behind >= NS - 2) wait_and_sync<(NS - 2) * L>();
    else if (NS > 4 && behind >= 4) wait_and_sync<4 * L>();
    else if (NS > 4 && behind >= 2) wait_and_sync<2 * L>();
    else wait_and_sync<L>();
    if (k + NS - 1 < end) stage(s == 0 ? NS - 1 : s - 1, k + NS - 1);
    const uint8_t* lp = lds[s][0];
    const uint8_t* lq = lds[s][1];
#pragma unroll
    for (int h = 0; h < 2; ++h) {      // 16 columns
      f16x8 ph[NX], pl[NX], qh[NY], ql[NY];
      const int piece = h * 2 + (lane >> 5);
#pragma unroll
      for (int x = 0; x < NX; ++x) {
        const int r = wr + 32 * x + (lane & 31);
        ph[x] = *(const f16x8*)(lp + r * 128 + (piece ^ (r & 7)) * 16);
        pl[x] = *(const f16x8*)(lp + r * 128 + ((piece + 4) ^ (r & 7)) * 16);
      }
#pragma unroll
      for (int y = 0; y < NY; ++y) {
        const int r = wc + 32 * y + (lane & 31);
        qh[y] = *(const f16x8*)(lq + r * 128 + (piece ^ (r & 7)) * 16);
        ql[y] = *(const f16x8*)(lq + r * 128 + ((piece + 4) ^ (r & 7)) * 16);
      }
#pragma unroll
      for (int x = 0; x < NX; ++x)
#pragma unroll
        for (int y = 0; y < NY; ++y) acc[x][y] = mfma(pl[x], qh[y], acc[x][y]);
#pragma unroll
      for (int x = 0; x < NX; ++x)
#pragma unroll
        for (int y = 0; y < NY; ++y) acc[x][y] = mfma(ph[x], ql[y], acc[x][y]);
#pragma unroll
      for (int x = 0; x < NX; ++x)
#pragma unroll
        for (int y = 0; y < NY; ++y) acc[x][y] = mfma(ph[x], qh[y], acc[x][y]);
    }
  }
#pragma unroll
  for (int x = 0; x < NX; ++x)
#pragma unroll
    for (int y = 0; y < NY; ++y) {
      if (q < 0) {
        write_block<MODE, E>(M, cur, f, acc[x][y], tr * T + wr + 32 * x, tc * T + wc + 32 * y, MODE >= NEXT || tr != tc);
      } else {
        const int block = (wr / 32 + x) * (T / 32) + wc / 32 + y;
        *(f32x16*)(part + (((int64_t)(q / S) * (T / 32) * (T / 32) + block) * S + slice) * 1024 + lane * 16) = acc[x][y];
      }
    }
}

// Adds the slices of the split tiles, in order: one wave per 32 x 32 block.
template <int MODE, int T, typename E>
__global__ __launch_bounds__(64) void ns_finish_kernel(const Mats* __restrict__ t, int cur, Coeffs f, int full, int S,
                                                       const float* __restrict__ part) {
  constexpr int N = T / 32;
  const int tile = blockIdx.x / (N * N), block = blockIdx.x % (N * N);
  const Where w = where<MODE, T>(t, full + tile);
  f32x16 acc;
#pragma unroll
  for (int r = 0; r < 16; ++r) acc[r] = 0.f;
  const float* p = part + (int64_t)blockIdx.x * S * 1024 + threadIdx.x * 16;
#pragma unroll 4
  for (int k = 0; k < S; ++k) acc += *(const f32x16*)(p + (int64_t)k * 1024);
  write_block<MODE, E>(t->m[w.mat], cur, f, acc, w.tr * T + block / N * 32, w.tc * T + block % N * 32,
                       MODE >= NEXT || w.tr != w.tc);
}

// ------------------------------------------------------------------------------------ host side
enum { F32 = 0, BF16 = 1, F16 = 2 };

int pad(int64_t v, int unit) { return (int)(ceil_div(v, unit) * unit); }

// bytes of one matrix' factors
int64_t factor_bytes(const Mat& m) {
  return (3 * (int64_t)m.mp * m.np + 2 * (int64_t)m.mp * m.mp) * 4 + kNormBlocks * (int64_t)sizeof(double);
}

int64_t tiles_of(const Mat& m, bool symmetric, int T) {
  const int64_t nt = m.mp / T;
  return symmetric ? nt * (nt + 1) / 2 : nt * (m.np / T);
}

// Matrices that go through the launches together, as the host sees them.
struct List {
  Mats t;
  int n, unit;        // matrices; what their sides are padded to
  int place[kMats];   // in the caller's list
};

// How a product of all matrices is launched.
struct Launch {
  int T;            // tile side
  int tiles, full;  // tiles, and how many of them are not split
  int S;            // slices of the others
  double cost;      // in rounds of 128 x 128 tiles
  int groups() const { return full + (tiles - full) * S; }
  int64_t part_floats() const { return (int64_t)(tiles - full) * S * T * T; }
};

// The workgroups that the chip holds at a time (2 a CU, of T = 256 one) make a round.  The tiles of whole rounds are not
// split.  Those left over are, where they would leave two thirds of the chip idle: into as many slices as the chip has
// room for, of at least 12 stages.
Launch launch_with(const List& l, int mode, int T) {
  Launch r = {T, 0, 0, 1, 0.0};
  int64_t tiles = 0, steps = 0;
  for (int i = 0; i < l.n; ++i) {
    tiles += tiles_of(l.t.m[i], mode < NEXT, T);
    steps = std::max<int64_t>(steps, (mode == GRAM ? l.t.m[i].np : l.t.m[i].mp) / kBK);
  }
  const int64_t round = (T == 256 ? 1 : 2) * kCUs, rest = tiles % round;
  r.tiles = r.full = (int)tiles;
  int64_t S = rest ? std::min(round / rest, steps / 12) : 1;
  if (S > 8) S &= ~7;               // slice k of all tiles on XCD k mod 8: each reads its columns only
  if (S >= 3) r.full = (int)(tiles - rest), r.S = (int)S;
  r.cost = (double)(tiles / round) + (rest ? (S >= 3 ? 0.1 + 1.0 / S : 1.0) : 0.0);
  if (T == 256) r.cost *= 1.7;      // (4 times the tile, by twice the waves: 2 at the same rate)
  return r;
}

Launch launch_of(const List& l, int mode) {
  if (l.unit == 64) return launch_with(l, mode, 64);
  const Launch r = launch_with(l, mode, 128);
  if (l.unit == 128) return r;
  const Launch q = launch_with(l, mode, 256);
  return q.cost < r.cost ? q : r;
}

template <int MODE, int T, int NS, typename E>
void product_with(const Launch& r, const Mats* t, int cur, const Coeffs& f, float* part, hipStream_t s) {
  RL_LAUNCH((ns_product_kernel<MODE, T, NS, E>), dim3((unsigned)r.groups()), dim3(Shape<T>::waves * 64), 0, s, t, cur, f,
            r.full, r.S, part);
  if (r.tiles > r.full)
    RL_LAUNCH((ns_finish_kernel<MODE, T, E>), dim3((unsigned)((r.tiles - r.full) * (T / 32) * (T / 32))), dim3(64), 0, s, t,
              cur, f, r.full, r.S, part);
}

// `first` of the table counts tiles of one side: a launch of 256 x 256 tiles takes the second table
template <int MODE, typename E>
void product(const List& l, const Mats* table, int cur, const Coeffs& f, float* part, hipStream_t s) {
  const Launch r = launch_of(l, MODE);
  if (r.T == 256) product_with<MODE, 256, 2, E>(r, table + 1, cur, f, part, s);
  else if (r.T == 128) product_with<MODE, 128, 2, E>(r, table, cur, f, part, s);
  else if (r.groups() > kCUs) product_with<MODE, 64, 4, E>(r, table, cur, f, part, s);
  else product_with<MODE, 64, 8, E>(r, table, cur, f, part, s);
}

void number_tiles(List& l, int T) {
  int sum[3] = {0, 0, 0};
  for (int i = 0; i < kMats; ++i) {
    for (int k = 0; k < 3; ++k) l.t.first[k][i] = i < l.n ? sum[k] : INT_MAX;
    if (i >= l.n) continue;
    sum[LOAD] += (l.t.m[i].mp / 32) * (l.t.m[i].np / 32);
    sum[SYM] += (int)tiles_of(l.t.m[i], true, T);
    sum[FULL] += (int)tiles_of(l.t.m[i], false, T);
  }
}

template <typename E>
int run(List& l, int steps, const Coeffs& f, double eps, Mats* table, float* part, hipStream_t s) {
  int tiles = 0;
  for (int i = 0; i < l.n; ++i) tiles += (l.t.m[i].mp / 32) * (l.t.m[i].np / 32);
  if (l.unit == 256) {
    number_tiles(l, 256);
    RL_LAUNCH((ns_table_kernel), dim3(1), dim3(256), 0, s, l.t, table + 1);
  }
  number_tiles(l, l.unit == 64 ? 64 : 128);
  RL_LAUNCH((ns_norm_kernel<E>), dim3(kNormBlocks, l.n), dim3(256), 0, s, l.t, table);
  RL_LAUNCH((ns_load_kernel<E>), dim3((unsigned)tiles), dim3(256), 0, s, table, eps);
  for (int k = 0; k < steps; ++k) {
    product<GRAM, float>(l, table, 0, f, part, s);
    product<POLY, float>(l, table, 0, f, part, s);
    if (k + 1 < steps) product<NEXT, float>(l, table, k & 1, f, part, s);
    else product<LAST, E>(l, table, k & 1, f, part, s);
  }
  RL_LAUNCH_CHECK();
  return RLPYT_OK;
}

// The matrices lo .. of a list that go together (at most kMats, empty ones left out) and what their sides are padded to;
// -> where the next ones start.  64 where 128 x 128 tiles would be too few for the chip, 256 where 256 x 256 ones are enough
// and the larger pads cost less than those tiles gain.
int gather(const int64_t* rows, const int64_t* cols, int n, int lo, List& l) {
  l.n = 0;
  for (; lo < n && l.n < kMats; ++lo) {
    if (rows[lo] == 0 || cols[lo] == 0) continue;
    l.place[l.n] = lo;
    Mat& m = l.t.m[l.n++];
    m = Mat{};
    m.rows = (int)rows[lo], m.cols = (int)cols[lo];
    m.tall = m.rows > m.cols;
  }
  auto pads = [&](int unit) {
    l.unit = unit;
    int64_t sum = 0;
    for (int i = 0; i < l.n; ++i) {
      Mat& m = l.t.m[i];
      m.mp = pad(std::min(m.rows, m.cols), unit), m.np = pad(std::max(m.rows, m.cols), unit);
      sum += (int64_t)m.mp * m.np;
    }
    return sum;
  };
  const int64_t wide = pads(256), usual = pads(128);
  if (usual < (int64_t)kCUs * 128 * 128) pads(64);
  else if (wide >= (int64_t)kCUs * 256 * 256 && wide < usual + usual / 16) pads(256);
  return lo;
}

int64_t part_floats(const List& l) {
  int64_t most = 0;
  for (int mode = GRAM; mode <= NEXT; ++mode) most = std::max(most, launch_of(l, mode).part_floats());
  return most;
}

// workspace: two tables | sums of slices | the matrices' factors
constexpr int64_t kTables = 2 * sizeof(Mats);
static_assert(sizeof(Mats) % 16 == 0 && sizeof(Mats) + 16 <= 4096, "an argument, and aligned pieces behind two of them");

}  // namespace
}  // namespace rlpyt

using namespace rlpyt;

namespace {
constexpr int64_t kMaxSide = 1 << 16;   // f16 keeps the lo pieces of ~ 1 / sqrt(m n) entries up to here

bool sides_ok(const int64_t* rows, const int64_t* cols, int n) {
  for (int i = 0; i < n; ++i)
    if (rows[i] < 0 || cols[i] < 0 || rows[i] > kMaxSide || cols[i] > kMaxSide) return false;
  return true;
}
}  // namespace

extern "C" int64_t rlpyt_orthogonalize_workspace_bytes(const int64_t* rows_host, const int64_t* cols_host, int n) {
  if (n <= 0 || !rows_host || !cols_host || !sides_ok(rows_host, cols_host, n)) return 0;
  int64_t most = 0;
  List l;
  for (int lo = 0; lo < n;) {     // (one group after the other, in the same workspace)
    lo = gather(rows_host, cols_host, n, lo, l);
    int64_t bytes = kTables + part_floats(l) * (int64_t)sizeof(float);
    for (int i = 0; i < l.n; ++i) bytes += factor_bytes(l.t.m[i]);
    if (l.n) most = std::max(most, bytes);
  }
  return most;
}

extern "C" int rlpyt_orthogonalize(int dtype, const void* const* in_host, const int64_t* ld_host,
                                   void* const* out_host, const int64_t* rows_host, const int64_t* cols_host, int n,
                                   int steps, float a, float b, float c, double eps, void* workspace,
                                   rlpyt_stream_t stream) {
  RL_CHECK_ARG(dtype >= F32 && dtype <= F16, RLPYT_EINVAL, "rlpyt_orthogonalize: unknown dtype %d", dtype);
  RL_CHECK_ARG(n >= 0 && steps >= 1 && steps <= 100, RLPYT_EINVAL, "rlpyt_orthogonalize: n=%d, steps=%d out of range",
               n, steps);
  if (n == 0) return RLPYT_OK;
  RL_CHECK_ARG(in_host && ld_host && out_host && rows_host && cols_host, RLPYT_EINVAL,
               "rlpyt_orthogonalize: null table");
  // the spectral norms of X and of the polynomial along the way, from the scalar recurrence on a grid of singular values
  for (int i = 0; i <= 1024; ++i) {
    double x = i / 1024.0;
    for (int k = 0; k < steps; ++k) {
      const double p = a + (b + c * x * x) * x * x;
      x *= p;
      RL_CHECK_ARG(fabs(x) < 8.0 && fabs(p) < 8.0 && x * x < 8.0, RLPYT_EINVAL,
                   "rlpyt_orthogonalize: coefficients (%g, %g, %g) leave the range of the stored factors", a, b, c);
    }
  }
  RL_CHECK_ARG(sides_ok(rows_host, cols_host, n), RLPYT_ESHAPE,
               "rlpyt_orthogonalize: sides of 0 to %ld are supported", (long)kMaxSide);
  bool any = false;
  for (int i = 0; i < n; ++i) {
    if (rows_host[i] * cols_host[i] == 0) continue;
    any = true;
    RL_CHECK_ARG(in_host[i] && out_host[i] && workspace, RLPYT_EINVAL, "rlpyt_orthogonalize: null pointer (matrix %d)", i);
  }
  if (!any) return RLPYT_OK;
  List l;
  for (int lo = 0; lo < n;) {
    lo = gather(rows_host, cols_host, n, lo, l);
    if (l.n == 0) break;
    Mats* table = (Mats*)workspace;
    float* part = (float*)((uint8_t*)workspace + kTables);
    uint8_t* ws = (uint8_t*)(part + part_floats(l));
    for (int i = 0; i < l.n; ++i) {
      Mat& m = l.t.m[i];
      m.in = in_host[l.place[i]], m.out = out_host[l.place[i]], m.ld = ld_host[l.place[i]];
      const int64_t big = (int64_t)m.mp * m.np * 2, small = (int64_t)m.mp * m.mp * 2;   // halves
      m.x = (_Float16*)ws;
      m.xt[0] = m.x + big, m.xt[1] = m.xt[0] + big;
      m.a = m.xt[1] + big, m.q = m.a + small;
      m.norm = (double*)(m.q + small);
      ws += factor_bytes(m);
    }
    const Coeffs f = {a, b, c};
    int rc;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == F32) rc = run<float>(l, steps, f, eps, table, part, s);
    else if (dtype == BF16) rc = run<__bf16>(l, steps, f, eps, table, part, s);
    else rc = run<_Float16>(l, steps, f, eps, table, part, s);
    if (rc != RLPYT_OK) return rc;
  }
  return RLPYT_OK;
}
