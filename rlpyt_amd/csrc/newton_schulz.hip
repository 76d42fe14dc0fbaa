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
// Storage of a factor with K columns (padded to 128, pads are 0): per row and 32 columns, 64 bytes of hi and 64 of lo.
// All products are row-times-row ("A B^T"): X X^T takes X, A A takes A (symmetric), Q X takes Q and X^T, so an epilogue
// writes its tile both ways.  Symmetric products compute the tiles on and above the diagonal and mirror them.
// The matrices of a list go through each launch together: 2 + 3 steps launches for up to 32 of them.
#include <math.h>

#include <algorithm>

#include "common.h"

namespace rlpyt {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kMats = 32;            // matrices of one launch (the table is a kernel argument)
constexpr int kTile = 128;           // tile of a product, and what the sides are padded to
constexpr int kBK = 32;              // columns of a stage
constexpr float kScale = 4096.f;     // 2^12, of every stored factor
constexpr int kNormBlocks = 64;      // partial sums of squares per matrix

struct Mat {
  const void* in;                    // [rows, cols], row stride ld
  void* out;                         // [rows, cols] dense
  int64_t ld;
  int rows, cols;
  int mp, np;                        // padded sides of X: min and max
  int tall;
  int tiles;                         // first workgroup of this matrix in a launch
  _Float16 *x, *xt[2], *a, *q;       // X [mp, np], X^T [np, mp] (two: read and written), A, Q [mp, mp]
  double* norm;                      // [kNormBlocks]
};
struct Mats {
  Mat m[kMats];
  int n;
};

__device__ __forceinline__ int find(const Mats& t, int block) {
  int i = 0;
  while (i + 1 < t.n && block >= t.m[i + 1].tiles) ++i;
  return i;
}

template <typename E>
__global__ __launch_bounds__(256) void ns_norm_kernel(const Mats t) {
  __shared__ double scratch[16];
  const Mat& M = t.m[blockIdx.y];
  const int64_t total = (int64_t)M.rows * M.cols;
  double v[1] = {0.0};
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += kNormBlocks * 256) {
    const int64_t r = i / M.cols;
    const double g = (double)(float)((const E*)M.in)[r * M.ld + (i - r * M.cols)];
    v[0] = fma(g, g, v[0]);
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
__global__ __launch_bounds__(256) void ns_load_kernel(const Mats t, double eps) {
  __shared__ float tile[32][33];
  __shared__ float factor;
  const int i = find(t, blockIdx.x);
  const Mat& M = t.m[i];
  if (threadIdx.x < kWave) {
    double s = M.norm[threadIdx.x];
    s = wave_sum(s);
    if (threadIdx.x == 0) factor = (float)((double)kScale / (sqrt(s) + eps));
  }
  __syncthreads();
  const int block = blockIdx.x - M.tiles, tn = M.np / 32;
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

// One 128 x 128 tile of P Q^T per workgroup: 4 waves of 64 x 64, two stages of 128 + 128 rows x 128 bytes in LDS, loaded
// straight from memory.  The 16-byte pieces of an LDS row are permuted by its row number, so that the 8 lanes that
// are served together read 8 different ones.
template <int MODE, typename E>
__global__ __launch_bounds__(256) void ns_product_kernel(const Mats t, int cur, float ca, float cb, float cc) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[2][2][kTile * 128];
  const int i = find(t, blockIdx.x);
  const Mat& M = t.m[i];
  int block = blockIdx.x - M.tiles;
  int tr, tc;
  if (MODE == GRAM || MODE == POLY) {   // tiles on and above the diagonal, row by row
    const int nt = M.mp / kTile;
    tr = 0;
    while (block >= nt - tr) block -= nt - tr, ++tr;
    tc = tr + block;
  } else {
    const int nt = M.np / kTile;
    tr = block / nt;
    tc = block % nt;
  }
  const int K = MODE == GRAM ? M.np : M.mp;
  const _Float16* P = MODE == GRAM ? M.x : MODE == POLY ? M.a : M.q;
  const _Float16* Q = MODE == GRAM ? M.x : MODE == POLY ? M.a : M.xt[cur];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // a load instruction of a wave fills 1 KB = 8 rows; lane -> row l >> 3, piece (l & 7) ^ (row & 7)
  const int64_t pitch = (int64_t)K * 4;   // bytes of a row
  const uint8_t *src[2];
  src[0] = (const uint8_t*)P + (int64_t)(tr * kTile + wave * 8 + (lane >> 3)) * pitch + ((lane & 7) ^ (lane >> 3)) * 16;
  src[1] = (const uint8_t*)Q + (int64_t)(tc * kTile + wave * 8 + (lane >> 3)) * pitch + ((lane & 7) ^ (lane >> 3)) * 16;
  auto stage = [&](int s, int k) {
#pragma unroll
    for (int o = 0; o < 2; ++o)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) void*)(src[o] + (int64_t)(32 * j) * pitch + (int64_t)k * 128),
            (__attribute__((address_space(3))) void*)(&lds[s][o][(32 * j + wave * 8) * 128]), 16, 0, 0);
  };
  f32x16 acc[2][2];
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int y = 0; y < 2; ++y)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[x][y][r] = 0.f;
  const int wr = (wave >> 1) * 64, wc = (wave & 1) * 64;
  const int steps = K / kBK;
  stage(0, 0);
  for (int k = 0; k < steps; ++k) {
    __syncthreads();      // this stage has arrived, and the other one has been read
    if (k + 1 < steps) stage((k + 1) & 1, k + 1);
    const uint8_t* lp = lds[k & 1][0];
    const uint8_t* lq = lds[k & 1][1];
#pragma unroll
    for (int h = 0; h < 2; ++h) {      // 16 columns
      f16x8 ph[2], pl[2], qh[2], ql[2];
      const int piece = h * 2 + (lane >> 5);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int rp = wr + 32 * x + (lane & 31), rq = wc + 32 * x + (lane & 31);
        ph[x] = *(const f16x8*)(lp + rp * 128 + ((piece) ^ (rp & 7)) * 16);
        pl[x] = *(const f16x8*)(lp + rp * 128 + ((piece + 4) ^ (rp & 7)) * 16);
        qh[x] = *(const f16x8*)(lq + rq * 128 + ((piece) ^ (rq & 7)) * 16);
        ql[x] = *(const f16x8*)(lq + rq * 128 + ((piece + 4) ^ (rq & 7)) * 16);
      }
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) acc[x][y] = mfma(pl[x], qh[y], acc[x][y]);
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) acc[x][y] = mfma(ph[x], ql[y], acc[x][y]);
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) acc[x][y] = mfma(ph[x], qh[y], acc[x][y]);
    }
  }
  // D[row = (r & 3) + 8 (r >> 2) + 4 (l >> 5)][column = l & 31], times 2^24
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int row0 = tr * kTile + wr + 32 * x + 4 * (lane >> 5), col = tc * kTile + wc + 32 * y + (lane & 31);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int row = row0 + 8 * g;
        f16x4 hi, lo;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float v = acc[x][y][4 * g + r];
          if (MODE == POLY) {
            const _Float16* p = M.a + at(row + r, col, M.mp);
            v = fmaf(cc, v * (1.f / kScale), cb * ((float)p[0] + (float)p[32]));
            if (row + r == col) v += ca * kScale;
          } else if (MODE == LAST) {
            v *= 1.f / (kScale * kScale);
            const int orow = M.tall ? col : row + r, ocol = M.tall ? row + r : col;
            if (orow < M.rows && ocol < M.cols) ((E*)M.out)[(int64_t)orow * M.cols + ocol] = (E)v;
            continue;
          } else {
            v *= 1.f / kScale;
          }
          _Float16 vh, vl;
          split(v, vh, vl);
          hi[r] = vh, lo[r] = vl;
          _Float16* o = (MODE == GRAM ? M.a : MODE == POLY ? M.q : M.x) +
                        at(row + r, col, MODE == NEXT ? M.np : M.mp);
          o[0] = vh, o[32] = vl;
        }
        if (MODE == LAST) continue;
        if (MODE == NEXT || tr != tc) {   // the other way round: 4 consecutive columns
          _Float16* o = (MODE == GRAM ? M.a : MODE == POLY ? M.q : M.xt[cur ^ 1]) + at(col, row, M.mp);
          *(f16x4*)o = hi;
          *(f16x4*)(o + 32) = lo;
        }
      }
    }
}

// ------------------------------------------------------------------------------------ host side
enum { F32 = 0, BF16 = 1, F16 = 2 };

int pad(int64_t v) { return (int)(ceil_div(v, kTile) * kTile); }

// bytes of one matrix' factors
int64_t factor_bytes(int64_t rows, int64_t cols) {
  const int64_t mp = pad(std::min(rows, cols)), np = pad(std::max(rows, cols));
  return (3 * mp * np + 2 * mp * mp) * 4 + kNormBlocks * (int64_t)sizeof(double);
}

template <typename E>
int run(Mats& t, int steps, float a, float b, float c, double eps, hipStream_t s) {
  RL_LAUNCH((ns_norm_kernel<E>), dim3(kNormBlocks, t.n), dim3(256), 0, s, t);
  auto grid = [&](auto tiles) {
    int64_t sum = 0;
    for (int i = 0; i < t.n; ++i) {
      t.m[i].tiles = (int)sum;
      sum += tiles(t.m[i]);
    }
    return dim3((unsigned)sum);
  };
  const dim3 load = grid([](const Mat& m) { return (int64_t)(m.mp / 32) * (m.np / 32); });
  RL_LAUNCH((ns_load_kernel<E>), load, dim3(256), 0, s, t, eps);
  for (int k = 0; k < steps; ++k) {
    const dim3 sym = grid([](const Mat& m) {
      const int64_t nt = m.mp / kTile;
      return nt * (nt + 1) / 2;
    });
    RL_LAUNCH((ns_product_kernel<GRAM, float>), sym, dim3(256), 0, s, t, 0, a, b, c);
    RL_LAUNCH((ns_product_kernel<POLY, float>), sym, dim3(256), 0, s, t, 0, a, b, c);
    const dim3 full = grid([](const Mat& m) { return (int64_t)(m.mp / kTile) * (m.np / kTile); });
    if (k + 1 < steps) RL_LAUNCH((ns_product_kernel<NEXT, float>), full, dim3(256), 0, s, t, k & 1, a, b, c);
    else RL_LAUNCH((ns_product_kernel<LAST, E>), full, dim3(256), 0, s, t, k & 1, a, b, c);
  }
  RL_LAUNCH_CHECK();
  return RLPYT_OK;
}

}  // namespace
}  // namespace rlpyt

using namespace rlpyt;

namespace {
constexpr int64_t kMaxSide = 1 << 16;   // f16 keeps the lo pieces of ~ 1 / sqrt(m n) entries up to here
}

extern "C" int64_t rlpyt_orthogonalize_workspace_bytes(const int64_t* rows_host, const int64_t* cols_host, int n) {
  int64_t bytes = 0;
  for (int i = 0; i < n; ++i) {
    if (rows_host[i] <= 0 || cols_host[i] <= 0) continue;
    bytes += factor_bytes(rows_host[i], cols_host[i]);
  }
  return bytes;
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
  for (int i = 0; i < n; ++i) {
    RL_CHECK_ARG(rows_host[i] >= 0 && cols_host[i] >= 0 && rows_host[i] <= kMaxSide && cols_host[i] <= kMaxSide,
                 RLPYT_ESHAPE, "rlpyt_orthogonalize: matrix %d is %ld x %ld", i, (long)rows_host[i], (long)cols_host[i]);
    RL_CHECK_ARG(rows_host[i] * cols_host[i] == 0 || (in_host[i] && out_host[i] && workspace), RLPYT_EINVAL,
                 "rlpyt_orthogonalize: null pointer (matrix %d)", i);
  }
  uint8_t* ws = (uint8_t*)workspace;
  for (int lo = 0; lo < n;) {
    Mats t = {};
    for (; lo < n && t.n < kMats; ++lo) {
      if (rows_host[lo] == 0 || cols_host[lo] == 0) continue;
      Mat& m = t.m[t.n++];
      m.in = in_host[lo], m.out = out_host[lo], m.ld = ld_host[lo];
      m.rows = (int)rows_host[lo], m.cols = (int)cols_host[lo];
      m.tall = m.rows > m.cols;
      m.mp = pad(std::min(m.rows, m.cols)), m.np = pad(std::max(m.rows, m.cols));
      const int64_t big = (int64_t)m.mp * m.np * 2, small = (int64_t)m.mp * m.mp * 2;   // halves
      m.x = (_Float16*)ws;
      m.xt[0] = m.x + big, m.xt[1] = m.xt[0] + big;
      m.a = m.xt[1] + big, m.q = m.a + small;
      m.norm = (double*)(m.q + small);
      ws += factor_bytes(m.rows, m.cols);
    }
    if (t.n == 0) break;
    int rc;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == F32) rc = run<float>(t, steps, a, b, c, eps, s);
    else if (dtype == BF16) rc = run<__bf16>(t, steps, a, b, c, eps, s);
    else rc = run<_Float16>(t, steps, a, b, c, eps, s);
    if (rc != RLPYT_OK) return rc;
  }
  return RLPYT_OK;
}
