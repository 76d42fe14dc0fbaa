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
// The matrices of a list go through each launch together: up to 32 of them in 2 launches and 3 a step, and one more for a product
// whose sums are split.
//
// Measured: 4096 x 4096, a symmetric product 206 us (1.0 PF/s of f16 operations, half of them counted), a full one 365 us (1.13);
// a library's f16 product of 8192 reaches 1.2.  512 x 3456 with three small ones: 11 + 4 (X X^T, in four slices), 9 and 16 us a
// step, of which 1.5 to 3 are matrix instructions; the rest is the way of the tiles from L2 and the launches' own latency.
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
  _Float16 *x, *xt0, *xt1, *a, *q;   // X [mp, np], X^T [np, mp] (two: read and written), A, Q [mp, mp]
  double* norm;                      // [kNormBlocks]
  // (an array here puts a kernel's copy of this struct into scratch memory: 128 x 128 took 84 us instead of 75)
  __device__ _Float16* xt(int k) const { return k ? xt1 : xt0; }
};
// The first launch gets the table as its argument and leaves it in the workspace for the others: an argument is read from the
// host's memory, 3 KB of it by every launch.
enum { LOAD = 0, SYM = 1, FULL = 4, KINDS = 7 };   // (SYM, FULL: + 0, 1, 2 for tiles of 64, 128, 256)
struct Mats {
  Mat m[kMats];
  int first[KINDS][kMats];           // first tile of a matrix: of ns_load_kernel, of symmetric and full products; INT_MAX behind the last
};

__device__ __forceinline__ int find(const Mats* __restrict__ t, int kind, int tile) {
  const bool behind = (threadIdx.x & 63) < kMats && t->first[kind][threadIdx.x & (kMats - 1)] <= tile;
  return __builtin_amdgcn_readfirstlane(__popcll(__ballot(behind)) - 1);
}

template <typename ET>
__global__ __launch_bounds__(256) void ns_norm_kernel(const Mats t, Mats* __restrict__ table) {
  typedef typename Elem<ET>::type E;
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

// element (r, k) of a factor with K (padded) columns: hi at the returned index, lo 32 behind it.  (Rows of an odd number of
// 128-byte lines, so that one column's lines spread over more of the L2's channels, made no difference.)
__device__ __forceinline__ int64_t at(int64_t r, int k, int K) { return (r * (K >> 5) + (k >> 5)) * 64 + (k & 31); }

__device__ __forceinline__ void split(float v, _Float16& hi, _Float16& lo) {
  hi = (_Float16)v;
  lo = (_Float16)(v - (float)hi);
}

// X_0 and its transpose from 32 x 32 tiles of the input
template <typename ET>
__global__ __launch_bounds__(256) void ns_load_kernel(const Mats* __restrict__ t, double eps) {
  typedef typename Elem<ET>::type E;
  __shared__ float tile[32][33];
  __shared__ double factor;
  const int i = find(t, LOAD, blockIdx.x);
  const Mat M = t->m[i];
  if (threadIdx.x < kWave) {
    double s = 0.0;
    for (int k = threadIdx.x; k < kNormBlocks; k += kWave) s += M.norm[k];
    s = wave_sum(s);
    if (threadIdx.x == 0) factor = s > 0.0 ? (double)kScale / (sqrt(s) + eps) : s;   // (a NaN stays one)
  }
  __syncthreads();
  const int block = blockIdx.x - t->first[LOAD][i], tn = M.np / 32;
  const int r0 = block / tn * 32, c0 = block % tn * 32;      // rows, columns of X
  const int lx = threadIdx.x & 31, ly = threadIdx.x >> 5;
  for (int k = ly; k < 32; k += 8) {   // coalesced along the input's rows
    const int r = M.tall ? c0 + k : r0 + k, c = M.tall ? r0 + lx : c0 + lx;
    float v = 0.f;
    if (r < M.rows && c < M.cols) v = (float)((double)(float)((const E*)M.in)[(int64_t)r * M.ld + c] * factor);
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
    p = M.xt0 + at(c0 + k, r0 + lx, M.mp);
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
  constexpr int kind = (MODE < NEXT ? SYM : FULL) + (T == 256 ? 2 : T == 128 ? 1 : 0);
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
    _Float16* o = (MODE == GRAM ? M.a : MODE == POLY ? M.q : M.xt(cur ^ 1)) + at(col, row, M.mp);   // 4 consecutive columns
    *(f16x4*)o = hi;
    *(f16x4*)(o + 32) = lo;
  }
}

// Eight results (times 2^24) next to each other along a row of the product, ROW, or down a column, from (row, col) on, which
// the mirrored or transposed factor holds along its row.
template <int MODE, bool ROW, typename E>
__device__ __forceinline__ void write8(const Mat& M, int cur, const Coeffs& f, const float (&sum)[8], int row, int col) {
  const int r = ROW ? row : col, k = ROW ? col : row;    // row and first column where they are stored
  if (MODE == LAST) {
    if (r >= M.rows || k >= M.cols) return;
    struct __attribute__((packed, aligned(sizeof(E)))) raw {
      E v[8];
    } v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v.v[i] = (E)(sum[i] * (1.f / (kScale * kScale)));
    E* o = (E*)M.out + (int64_t)r * M.cols + k;
    if (k + 8 <= M.cols) {
      *reinterpret_cast<raw*>(o) = v;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (k + i < M.cols) o[i] = v.v[i];
    }
    return;
  }
  const int K = MODE == NEXT && ROW ? M.np : M.mp;
  f16x8 hi, lo, ah, al;
  if (MODE == POLY) {
    const _Float16* p = M.a + at(r, k, K);
    ah = *(const f16x8*)p, al = *(const f16x8*)(p + 32);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float v = sum[i] * (1.f / kScale);
    if (MODE == POLY) {
      v = fmaf(f.c, v, f.b * ((float)ah[i] + (float)al[i]));
      if (r == k + i) v += f.a * kScale;
    }
    _Float16 vh, vl;
    split(v, vh, vl);
    hi[i] = vh, lo[i] = vl;
  }
  _Float16* o = (MODE == GRAM ? M.a : MODE == POLY ? M.q : ROW ? M.x : M.xt(cur ^ 1)) + at(r, k, K);
  *(f16x8*)o = hi;
  *(f16x8*)(o + 32) = lo;
}
// Which ways a tile is written.
template <int MODE>
__device__ __forceinline__ bool by_rows(const Mat& M) {
  return MODE != LAST || !M.tall;
}
template <int MODE>
__device__ __forceinline__ bool by_columns(const Mat& M, const Where& w) {
  return MODE == NEXT || (MODE == LAST ? M.tall != 0 : w.tr != w.tc);
}

// This wave's loads but the last N have arrived and its reads of LDS are done; then the workgroup's barrier.  (__syncthreads
// waits for all loads.)
template <int N>
__device__ __forceinline__ void wait_and_sync() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// A workgroup's tile of T x T: waves, 32 x 32 blocks of a wave, NS LDS stages of 2 T rows x 128 bytes.
// 256 and 128 (two stages): where the chip is full.  128 moves 96 KB through the LDS a stage, against 768 cycles of matrix
// pipe, and twice 256's bytes from L2 per operation; but a matrix of 4096 has just one tile of 256 for each CU.
// 64: for few tiles.  What counts then is the time of a stage on its own (reads of the LDS, then three dependent
// products, twice: ~900 cycles) and a load's way from another XCD's results (1 us): four stages, and where one workgroup
// has a CU for itself, G = 2 sets of four waves that take every other 32 columns and add up in the end (128: eight waves).
template <int T, int G>
struct Shape {
  static constexpr int sets = T == 64 ? G : 1, waves = T == 256 ? 8 : T == 128 ? 4 * G : 4;         // waves of a set: 2 rows of
  static constexpr int cols = waves / 2, threads = waves * sets * 64;
  static constexpr int nx = T / 64, ny = T / 32 / cols;
  static constexpr int passes = T / (8 * waves);                                     // load instructions of a wave per factor
};
constexpr int kPitch = 65;   // floats of a row of a 64 x 64 tile in LDS: rows and columns are read without conflicts

// Where piece k of a row of 8 lies, and which piece lies at place k.  (The loads' row is taken within its pass of 8 x waves rows.)
__device__ __forceinline__ int place(int row, int k) { return k ^ ((row >> 1) & 7); }

// One T x T tile of P Q^T per workgroup, the factors loaded straight from memory to LDS.  The 16-byte pieces of an LDS row are
// permuted (place()), so that the 16 lanes that a read serves together hit all 64 banks: 16 rows have 8 permutations, of
// the even and of the odd ones, which are 128 bytes apart.  (Permuted by row & 7: half of all reads took 4 cycles more.)
// Tiles from `full` on are split along K into S slices of a workgroup each, whose sums go to `part` for ns_finish_kernel: the
// tiles that would make a round of their own on an idle chip.
template <int MODE, int T, int G_, int NS, typename ET>
__global__ __launch_bounds__((Shape<T, G_>::threads)) void ns_product_kernel(const Mats* __restrict__ t, int cur, Coeffs f,
                                                                          int full, int S, float* __restrict__ part) {
  typedef typename Elem<ET>::type E;
  typedef Shape<T, G_> G;
  constexpr int NX = G::nx, NY = G::ny, L = 2 * G::passes, KG = G::sets;
  __shared__ __attribute__((aligned(16))) uint8_t lds[NS][KG][2][T * 128];
  const int q = (int)blockIdx.x - full;
  const Where at_ = where<MODE, T>(t, q < 0 ? neighbours(blockIdx.x, full) : full + q / S);
  const Mat M = t->m[at_.mat];
  const int tr = at_.tr, tc = at_.tc;
  const int K = MODE == GRAM ? M.np : M.mp;
  const _Float16* P = MODE == GRAM ? M.x : MODE == POLY ? M.a : M.q;
  const _Float16* Q = MODE == GRAM ? M.x : MODE == POLY ? M.a : M.xt(cur);
  const int lane = threadIdx.x & 63;
  const int set = KG == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / G::waves;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) - set * G::waves;
  // a load instruction of a wave fills 1 KB = 8 rows; lane -> row l >> 3 of them, and the piece that belongs at its place
  const int64_t pitch = (int64_t)K * 4;   // bytes of a row
  const int lrow = wave * 8 + (lane >> 3), lpiece = place(lrow, lane & 7);
  const uint8_t* src[2];
  src[0] = (const uint8_t*)P + (int64_t)(tr * T + lrow) * pitch + set * 128 + lpiece * 16;
  src[1] = (const uint8_t*)Q + (int64_t)(tc * T + lrow) * pitch + set * 128 + lpiece * 16;
  auto stage = [&](int s, int k) {
#pragma unroll
    for (int o = 0; o < 2; ++o)
#pragma unroll
      for (int j = 0; j < G::passes; ++j)
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) void*)(src[o] + (int64_t)(8 * G::waves * j) * pitch + (int64_t)k * (KG * 128)),
            (__attribute__((address_space(3))) void*)(&lds[s][set][o][(8 * G::waves * j + wave * 8) * 128]), 16, 0, 0);
  };
  f32x16 acc[NX][NY];
#pragma unroll
  for (int x = 0; x < NX; ++x)
#pragma unroll
    for (int y = 0; y < NY; ++y)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[x][y][r] = 0.f;
  const int wr = wave / G::cols * (32 * NX), wc = wave % G::cols * (32 * NY);
  const int steps = K / (kBK * KG);     // (K is a multiple of 64)
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
    else wait_and_sync<L>();
    if (k + NS - 1 < end) stage(s == 0 ? NS - 1 : s - 1, k + NS - 1);
    const uint8_t* lp = lds[s][set][0];
    const uint8_t* lq = lds[s][set][1];
#pragma unroll
    for (int h = 0; h < 2; ++h) {      // 16 columns
      f16x8 ph[NX], pl[NX], qh[NY], ql[NY];
      const int piece = h * 2 + (lane >> 5);
#pragma unroll
      for (int x = 0; x < NX; ++x) {
        const int r = wr + 32 * x + (lane & 31);
        ph[x] = *(const f16x8*)(lp + r * 128 + place(r, piece) * 16);
        pl[x] = *(const f16x8*)(lp + r * 128 + place(r, piece + 4) * 16);
      }
#pragma unroll
      for (int y = 0; y < NY; ++y) {
        const int r = wc + 32 * y + (lane & 31);
        qh[y] = *(const f16x8*)(lq + r * 128 + place(r, piece) * 16);
        ql[y] = *(const f16x8*)(lq + r * 128 + place(r, piece + 4) * 16);
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
  if constexpr (T == 64) {     // through LDS, to rows and columns of 8
    static_assert(NS * 2 * T * 128 >= T * kPitch * (int)sizeof(float), "the sets' sums fit the stages");
    float* tile = (float*)&lds[0][0][0][0];
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 16; ++r)
      tile[set * (T * kPitch) + (wr + (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5)) * kPitch + wc + (lane & 31)] = acc[0][0][r];
    __syncthreads();
    const bool rows = by_rows<MODE>(M), columns = by_columns<MODE>(M, at_);
    for (int i = threadIdx.x; i < T * T / 8; i += G::threads) {
      const int a = i >> 3, b = (i & 7) * 8;
      float v[8];
      if (rows || q >= 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v[j] = tile[a * kPitch + b + j];
          if (KG == 2) v[j] += tile[T * kPitch + a * kPitch + b + j];
        }
        if (q < 0) {
          write8<MODE, true, E>(M, cur, f, v, tr * T + a, tc * T + b);
        } else {
          float4* o = (float4*)(part + ((int64_t)(q / S) * S + slice) * (T * T) + a * T + b);
          o[0] = float4{v[0], v[1], v[2], v[3]};
          o[1] = float4{v[4], v[5], v[6], v[7]};
        }
      }
      if (columns && q < 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v[j] = tile[(b + j) * kPitch + a];
          if (KG == 2) v[j] += tile[T * kPitch + (b + j) * kPitch + a];
        }
        write8<MODE, false, E>(M, cur, f, v, tr * T + b, tc * T + a);
      }
    }
  } else {
#pragma unroll
    for (int x = 0; x < NX; ++x)
#pragma unroll
      for (int y = 0; y < NY; ++y) {
        if (q < 0) {
          write_block<MODE, E>(M, cur, f, acc[x][y], tr * T + wr + 32 * x, tc * T + wc + 32 * y, MODE >= NEXT || tr != tc);
        } else {     // 16 values of a lane together
          const int block = (wr / 32 + x) * (T / 32) + wc / 32 + y;
          *(f32x16*)(part + (((int64_t)(q / S) * (T / 32) * (T / 32) + block) * S + slice) * 1024 + lane * 16) = acc[x][y];
        }
      }
  }
}

// Adds the slices of the split tiles, in order: a wave per 32 x 32 block of T = 256 and 128,
template <int MODE, int T, typename ET>
__global__ __launch_bounds__(64) void ns_finish_kernel(const Mats* __restrict__ t, int cur, Coeffs f, int full, int S,
                                                       const float* __restrict__ part) {
  typedef typename Elem<ET>::type E;
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

// and 16 rows of a 64 x 64 tile by a workgroup of two waves.
__global__ __launch_bounds__(128) void ns_finish64_kernel(const Mats* __restrict__ t, int full, int S,
                                                          const float* __restrict__ part) {
  constexpr int T = 64, R = 16;
  __shared__ float tile[R][kPitch];
  const int split = blockIdx.x / (T / R), band = blockIdx.x % (T / R);
  const Where w = where<GRAM, T>(t, full + split);
  const Mat M = t->m[w.mat];
  const int a = threadIdx.x >> 3, b = (threadIdx.x & 7) * 8;
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const float* p = part + (int64_t)split * S * (T * T) + (band * R + a) * T + b;
#pragma unroll 4
  for (int k = 0; k < S; ++k) {
    const float4 x = *(const float4*)(p + (int64_t)k * (T * T)), y = *(const float4*)(p + (int64_t)k * (T * T) + 4);
    v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w;
    v[4] += y.x, v[5] += y.y, v[6] += y.z, v[7] += y.w;
  }
  write8<GRAM, true, float>(M, 0, Coeffs{}, v, w.tr * T + band * R + a, w.tc * T + b);
  if (w.tr == w.tc) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) tile[a][b + j] = v[j];
  __syncthreads();
  const int col = threadIdx.x >> 1, r0 = (threadIdx.x & 1) * 8;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = tile[r0 + j][col];
  write8<GRAM, false, float>(M, 0, Coeffs{}, v, w.tr * T + band * R + r0, w.tc * T + col);
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

// The shapes that a product is compiled for.  per_cu: workgroups that a CU holds (LDS); stage: us of a stage of 32 columns
// where nothing else bounds it, as measured.
struct Variant {
  int T, G, per_cu;
  double stage;
};
constexpr Variant kVariants[] = {{64, 2, 1, 0.27}, {64, 1, 2, 0.42}, {128, 2, 1, 0.95}, {128, 1, 2, 1.2}, {256, 1, 1, 2.85}};

// How a product of all matrices is launched.
struct Launch {
  Variant v;
  int tiles, full;  // tiles, and how many of them are not split
  int S;            // slices of the others
  double us;        // estimated
  int groups() const { return full + (tiles - full) * S; }
  int64_t part_floats() const { return (int64_t)(tiles - full) * S * v.T * v.T; }
};

// The workgroups that the chip holds at a time make a round.  Tiles of whole rounds are not split; those left over may be,
// into slices of at least 8 stages, where their sums' way through memory costs less than an idle chip.  (Of the 64-tiles only
// X X^T's: the other products' sums over m columns are long enough only where larger tiles are faster.)  A stage takes the
// variant's time or what the loads of all CUs need for its bytes (measured: 8.7 TB/s, from 128 x 128 tiles on 10.8); a launch
// has 3.5 us around its stages, and a second round on CUs that hold one workgroup 2.5 of its own.
Launch launch_with(const List& l, int mode, const Variant& v) {
  double work = 0.0;
  int64_t tiles = 0, longest = 0;
  for (int i = 0; i < l.n; ++i) {
    const int64_t n = tiles_of(l.t.m[i], mode < NEXT, v.T), steps = (mode == GRAM ? l.t.m[i].np : l.t.m[i].mp) / kBK;
    tiles += n;
    work += (double)n * steps;
    longest = std::max(longest, steps);
  }
  const int64_t round = (int64_t)v.per_cu * kCUs, rest = tiles % round, full = tiles - rest;
  const double average = work / tiles;
  auto stage = [&](int64_t groups) {
    return std::max(v.stage, (double)std::min(groups, round) * v.T * 256 / (v.T == 64 ? 8.7e6 : 10.8e6));
  };
  const double rounds = (double)(full / round), own = v.per_cu == 1 ? 2.5 : 0.0;
  const double whole = full ? rounds * average * stage(full) + (rounds - (rest ? 0 : 1)) * own : 0.0;
  Launch r = {v, (int)tiles, (int)tiles, 1, 3.5 + whole + (rest ? longest * stage(rest) : 0.0)};
  const bool may = rest && (mode == GRAM || v.T > 64);
  for (int64_t S = 2; may && S <= std::min<int64_t>(round / rest, longest / 8); S += S < 8 ? 1 : 8) {   // (from 8 on by 8: slice k
    // of all tiles on XCD k mod 8, which reads its columns only)
    const double us = 3.5 + whole + (double)longest / S * stage(rest * S) + 4.5 + rest * S * v.T * v.T * 8 / 4e6;
    if (us < r.us) r.full = (int)full, r.S = (int)S, r.us = us;
  }
  return r;
}

Launch launch_of(const List& l, int mode) {
  Launch best = {};
  for (const Variant& v : kVariants) {
    if (v.T > l.unit) continue;
    const Launch r = launch_with(l, mode, v);
    if (best.tiles == 0 || r.us < best.us) best = r;
  }
  return best;
}

template <int MODE, int T, int G, int NS, typename ET>
void product_with(const Launch& r, const Mats* t, int cur, const Coeffs& f, float* part, hipStream_t s) {
  RL_LAUNCH((ns_product_kernel<MODE, T, G, NS, ET>), dim3((unsigned)r.groups()), dim3(Shape<T, G>::threads), 0, s, t, cur, f,
            r.full, r.S, part);
  const int split = r.tiles - r.full;
  if (split == 0) return;
  if constexpr (T > 64)
    RL_LAUNCH((ns_finish_kernel<MODE, T, ET>), dim3((unsigned)(split * (T / 32) * (T / 32))), dim3(64), 0, s, t, cur, f,
              r.full, r.S, part);
  else if constexpr (MODE == GRAM)
    RL_LAUNCH(ns_finish64_kernel, dim3((unsigned)(split * 4)), dim3(128), 0, s, t, r.full, r.S, part);
}

template <int MODE, typename ET>
void product(const List& l, const Mats* table, int cur, const Coeffs& f, float* part, hipStream_t s) {
  const Launch r = launch_of(l, MODE);
  if (r.v.T == 256) product_with<MODE, 256, 1, 2, ET>(r, table, cur, f, part, s);
  else if (r.v.T == 128 && r.v.G == 1) product_with<MODE, 128, 1, 2, ET>(r, table, cur, f, part, s);
  else if (r.v.T == 128) product_with<MODE, 128, 2, 4, ET>(r, table, cur, f, part, s);
  else if (r.v.G == 1) product_with<MODE, 64, 1, 4, ET>(r, table, cur, f, part, s);
  else product_with<MODE, 64, 2, 4, ET>(r, table, cur, f, part, s);
}

template <typename ET>
int run(List& l, int steps, const Coeffs& f, double eps, Mats* table, float* part, hipStream_t s) {
  int64_t sum[KINDS] = {};
  for (int i = 0; i < kMats; ++i) {
    for (int k = 0; k < KINDS; ++k) l.t.first[k][i] = i < l.n ? (int)sum[k] : INT_MAX;
    if (i >= l.n) continue;
    const Mat& m = l.t.m[i];
    sum[LOAD] += (int64_t)(m.mp / 32) * (m.np / 32);
    for (int k = 0; k < 3 && (64 << k) <= l.unit; ++k)
      sum[SYM + k] += tiles_of(m, true, 64 << k), sum[FULL + k] += tiles_of(m, false, 64 << k);
  }
  RL_LAUNCH((ns_norm_kernel<ET>), dim3(kNormBlocks, l.n), dim3(256), 0, s, l.t, table);
  RL_LAUNCH((ns_load_kernel<ET>), dim3((unsigned)sum[LOAD]), dim3(256), 0, s, table, eps);
  for (int k = 0; k < steps; ++k) {
    product<GRAM, float>(l, table, 0, f, part, s);
    product<POLY, float>(l, table, 0, f, part, s);
    if (k + 1 < steps) product<NEXT, float>(l, table, k & 1, f, part, s);
    else product<LAST, ET>(l, table, k & 1, f, part, s);
  }
  RL_LAUNCH_CHECK();
  return RLPYT_OK;
}

// The matrices lo .. of a list that go together (at most kMats, empty ones left out) and what their sides are padded to, 64,
// 128 or 256: what is expected to take the least time, with the tiles that this allows; -> where the next ones start.
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
  if (l.n == 0) return lo;
  auto with = [&](int unit) {
    l.unit = unit;
    for (int i = 0; i < l.n; ++i) {
      Mat& m = l.t.m[i];
      m.mp = pad(std::min(m.rows, m.cols), unit), m.np = pad(std::max(m.rows, m.cols), unit);
    }
    return launch_of(l, GRAM).us + launch_of(l, POLY).us + launch_of(l, NEXT).us;
  };
  int unit = 64;
  double least = with(64);
  for (int u : {128, 256}) {
    const double us = with(u);
    if (us < least) least = us, unit = u;
  }
  with(unit);
  return lo;
}

int64_t part_floats(const List& l) {
  int64_t most = 0;
  for (int mode = GRAM; mode <= NEXT; ++mode) most = std::max(most, launch_of(l, mode).part_floats());
  return most;
}

// workspace: table | sums of slices | the matrices' factors
constexpr int64_t kTables = sizeof(Mats);
static_assert(sizeof(Mats) % 16 == 0 && sizeof(Mats) + 16 <= 4096, "an argument, and aligned pieces behind it");

}  // namespace
}  // namespace rlpyt

using namespace rlpyt;

namespace {
constexpr int64_t kMaxSide = 1 << 16;   // f16 keeps the lo pieces of ~ 1 / sqrt(m n) entries up to here

// Whether the spectral norms of X, A and Q stay in the range of the stored factors: singular values in [0, top] go to
// |x p(x^2)|, largest at top or where (x p(x^2))' = 0, p(y) = a + b y + c y^2.
bool stays_bounded(double a, double b, double c, int steps) {
  const double half = -0.5 * (3.0 * b + copysign(sqrt(9.0 * b * b - 20.0 * a * c), b));
  const double places[] = {half / (5.0 * c), a / half, -b / (2.0 * c)};    // the last one: p' = 0 (none: NaN or infinite)
  auto p = [&](double y) { return a + (b + c * y) * y; };
  double top = 1.0;
  for (int k = 0; k < steps; ++k) {
    const double end = top * top;
    double q = std::max(fabs(a), fabs(p(end))), x = top * fabs(p(end));
    for (double y : places)
      if (y > 0.0 && y < end) q = std::max(q, fabs(p(y))), x = std::max(x, sqrt(y) * fabs(p(y)));
    if (!(fabs(a) < 8.0 && q < 8.0 && x * x < 8.0)) return false;
    top = x;
  }
  return true;
}

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
  RL_CHECK_ARG(stays_bounded(a, b, c, steps), RLPYT_EINVAL,
               "rlpyt_orthogonalize: coefficients (%g, %g, %g) leave the range of the stored factors", a, b, c);
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
      m.xt0 = m.x + big, m.xt1 = m.xt0 + big;
      m.a = m.xt1 + big, m.q = m.a + small;
      m.norm = (double*)(m.q + small);
      ws += factor_bytes(m);
    }
    const Coeffs f = {a, b, c};
    int rc;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == F32) rc = run<float>(l, steps, f, eps, table, part, s);
    else if (dtype == BF16) rc = run<Bf16>(l, steps, f, eps, table, part, s);
    else rc = run<Half>(l, steps, f, eps, table, part, s);
    if (rc != RLPYT_OK) return rc;
  }
  return RLPYT_OK;
}
