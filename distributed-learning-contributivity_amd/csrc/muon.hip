// Orthogonalised update of weight matrices by Newton-Schulz products, and the Muon step (gfx950).
// include/mplc_hip_ops.h states the operators.
//
// With k = min(rows, cols) and L = max(rows, cols), X is kept as [L][k], so that the k x k side is A = X^T X and a step is
// X <- X P, P = a I + b A + c A^2: products with a polynomial epilogue on the tiled core of mma.h.
//
// Precision.  Small singular values grow by up to a^steps (485 for the usual five steps), and so do the rounding errors
// beside them: 16-bit products would be off by percents for a spectrum that decays.  All matrices are therefore held as
// split fp16 (22 bits) and multiplied with three fp16 matrix instructions, which keeps fp32's accuracy at about twice
// fp32's matrix rate.  The ranges are known by construction - |X| <= 2 (checked on the host for the given
// coefficients), |A| <= 4, |P| and its products by their bounds - so each matrix has one power-of-two scale that uses
// fp16's range without overflow.
//
// Gram space.  A phase of s steps needs X only twice: A = X^T X, then s - 1 times (P A P, which is the next step's A, and
// Q <- P Q) on k x k matrices, then X <- X Q.  Errors of A are amplified inside a phase, so a phase has at most 3 steps
// and the next one starts from the Gram matrix of its own X: against 64 bits, phases of 3 and 2 are as exact as five
// single steps in fp32, one phase of 5 is 10 to 50 times worse.  Used where L >= 1.5 k, where it takes fewer products.
#include <math.h>

#include "mma.h"
#include "mplc_hip.h"
#include "xcd.h"

namespace {

using namespace mma;

constexpr float X_SCALE = 16384.f;  // |X| <= 2
constexpr float A_SCALE = 8192.f;   // |A|, |P A| <= 4
constexpr int NORM_CHUNKS = 256;

// Split fp16 of a matrix times its scale.  Rows of 32-column blocks, 32 hi then 32 lo: both planes' pieces of a tile lie in
// one 128-byte line (planes of their own cost each operand along r half a line, fetched twice).
struct Planes {
  uint16_t* p;
  int64_t stride;  // elements of one model
  int ld;          // elements of a row: 2 * (columns rounded up to 32)
};
__device__ __forceinline__ int64_t plane_at(const Planes& p, int g, int64_t m, int n) {
  return g * p.stride + m * p.ld + ((n >> 5) << 6) + (n & 31);
}

__device__ __forceinline__ void split(float v, uint16_t& hi, uint16_t& lo) {
  hi = f32_to_f16(v);
  lo = f32_to_f16(v - f16_to_f32(hi));
}
__device__ __forceinline__ void store_planes(const Planes& p, int g, int64_t m, int n, f32x4 v) {
  uint16_t h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) split(v[i], h[i], l[i]);
  uint16_t* at = p.p + plane_at(p, g, m, n);  // n is a multiple of 4: 8-byte aligned
  u32x2 a, b;
  a[0] = h[0] | (uint32_t)h[1] << 16;
  a[1] = h[2] | (uint32_t)h[3] << 16;
  b[0] = l[0] | (uint32_t)l[1] << 16;
  b[1] = l[2] | (uint32_t)l[3] << 16;
  *reinterpret_cast<u32x2*>(at) = a;
  *reinterpret_cast<u32x2*>(at + 32) = b;
}
__device__ __forceinline__ f32x4 load_planes(const Planes& p, int g, int64_t m, int n) {
  const uint16_t* at = p.p + plane_at(p, g, m, n);
  const u32x2 a = *reinterpret_cast<const u32x2*>(at), b = *reinterpret_cast<const u32x2*>(at + 32);
  f32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    v[i] = f16_to_f32((uint16_t)(a[i >> 1] >> (16 * (i & 1)))) + f16_to_f32((uint16_t)(b[i >> 1] >> (16 * (i & 1))));
  return v;
}

// ------------------------------------------------------------------------------------------ the update U and its norm
struct Source {
  const void* g;
  int64_t g_stride, g_ld;
  float* m;  // NULL: U = g
  int64_t m_stride, m_ld;
  float beta;
  int nesterov, rows, cols;
};

// U at (r, c .. c + 3), `valid` of them inside, in two steps, so that several groups' loads are on their way at a time.
struct Raw {
  f32x4 g, m;
};
// N groups at at(j, r, c, valid); the momentum's loads stand in one branch, which the compiler waits for as a whole
template <Kind K, bool WIDE, int N, typename At> __device__ __forceinline__ void raw4(Raw (&x)[N], const Source& s, int g, At at) {
  typedef typename Elem<K>::T T;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    int r, c, valid;
    at(j, r, c, valid);
    x[j].g = load4<K, WIDE>(reinterpret_cast<const T*>(s.g) + g * s.g_stride + r * s.g_ld + c, valid);
  }
  if (s.m)
#pragma unroll
    for (int j = 0; j < N; ++j) {
      int r, c, valid;
      at(j, r, c, valid);
      x[j].m = load4<F32, WIDE>(s.m + g * s.m_stride + r * s.m_ld + c, valid);
    }
}
// FIRST: the pass that updates the momentum
template <bool FIRST> __device__ __forceinline__ f32x4 update4(const Source& s, Raw x, int g, int64_t r, int c, int valid) {
  if (s.m == nullptr) return x.g;
  if (FIRST) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x.m[i] = s.beta * x.m[i] + x.g[i];
    store4<F32>(s.m + g * s.m_stride + r * s.m_ld + c, x.m, valid);
  }
  f32x4 u;
#pragma unroll
  for (int i = 0; i < 4; ++i) u[i] = s.nesterov ? s.beta * x.m[i] + x.g[i] : x.m[i];
  return u;
}

// Walks a matrix's groups of 4 columns, NT threads side by side, without a division per group.
struct Walk {
  int r, c4, dr, dc, n4;
  __device__ __forceinline__ Walk(int first, int step, int n4_) : n4(n4_) {
    r = first / n4;
    c4 = first - r * n4;
    dr = step / n4;
    dc = step - dr * n4;
  }
  __device__ __forceinline__ void next() {
    r += dr;
    c4 += dc;
    if (c4 >= n4) {
      c4 -= n4;
      ++r;
    }
  }
};

__device__ __forceinline__ double block_sum(double v, double* part) {  // part: 4 doubles; every thread gets the sum
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  return (part[0] + part[1]) + (part[2] + part[3]);
}

// X_SCALE / |U| from |U|^2; 0 for U = 0, NaN where U is not finite
__device__ __forceinline__ double inverse_norm(double square) {
  if (square == 0.) return 0.;
  if (!(square < (double)INFINITY)) return (double)NAN;
  return (double)X_SCALE / sqrt(square);
}

// |U|^2 in 64 bits (neither 1e-30 nor 1e30 leaves the range), one partial sum per workgroup, NORM_CHUNKS at most per model
template <Kind K> __global__ __launch_bounds__(256) void norm_kernel(const Source s, double* sums) {
  __shared__ double part[4];
  const int g = blockIdx.y;
  double sum = 0.;
  by_width(s.cols, [&](auto wide) {
    for (Walk w(blockIdx.x * 256 + threadIdx.x, gridDim.x * 256, (s.cols + 3) >> 2); w.r < s.rows;) {
      Raw x[4];
      int r[4], c[4];
#pragma unroll
      for (int j = 0; j < 4; ++j, w.next()) {  // behind the last row: the last one again, not used
        r[j] = w.r;
        c[j] = w.c4 * 4;
      }
      raw4<K, decltype(wide)::value>(x, s, g, [&](int j, int& row, int& col, int& valid) {
        row = min(r[j], s.rows - 1);
        col = c[j];
        valid = s.cols - col;
      });
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (r[j] < s.rows) {
          const f32x4 v = update4<true>(s, x[j], g, r[j], c[j], s.cols - c[j]);
#pragma unroll
          for (int i = 0; i < 4; ++i) sum += (double)v[i] * (double)v[i];
        }
    }
  });
  sum = block_sum(sum, part);
  if (threadIdx.x == 0) sums[(int64_t)g * gridDim.x + blockIdx.x] = sum;
}

// X_0 as planes of L = rows rows, the columns behind k zero
template <Kind K> __global__ __launch_bounds__(256) void start_kernel(const Source s, const double* sums, int chunks, const Planes x) {
  __shared__ double part[4];
  const int g = blockIdx.y;
  const double inv = inverse_norm(block_sum(threadIdx.x < chunks ? sums[(int64_t)g * chunks + threadIdx.x] : 0., part));
  by_width(s.cols, [&](auto wide) {
    for (Walk w(blockIdx.x * 256 + threadIdx.x, gridDim.x * 256, x.ld >> 3); w.r < s.rows;) {
      Raw u[4];
      int r[4], c[4];
#pragma unroll
      for (int j = 0; j < 4; ++j, w.next()) {  // behind the last row or column: the last ones again, not used
        r[j] = w.r;
        c[j] = w.c4 * 4;
      }
      raw4<K, decltype(wide)::value>(u, s, g, [&](int j, int& row, int& col, int& valid) {
        row = min(r[j], s.rows - 1);
        col = c[j] < s.cols ? c[j] : (s.cols - 1) & ~3;
        valid = s.cols - col;
      });
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (r[j] < s.rows) {
          f32x4 v = update4<false>(s, u[j], g, r[j], c[j], s.cols - c[j]);
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = c[j] < s.cols ? (float)((double)v[i] * inv) : 0.f;
          store_planes(x, g, r[j], c[j], v);
        }
    }
  });
}

// The same with L = cols: 64 x 64 tiles, transposed through LDS
template <Kind K> __global__ __launch_bounds__(256) void start_wide_kernel(const Source s, const double* sums, int chunks, const Planes x) {
  __shared__ double part[4];
  __shared__ float tile[64][65];
  const int g = blockIdx.z;
  const double inv = inverse_norm(block_sum(threadIdx.x < chunks ? sums[(int64_t)g * chunks + threadIdx.x] : 0., part));
  const int l0 = blockIdx.x * 64, k0 = blockIdx.y * 64;
  const int q = (threadIdx.x & 15) * 4, ty = threadIdx.x >> 4;
  by_width(s.cols, [&](auto wide) {
    Raw u[4];
    const int in = l0 + q < s.cols ? l0 + q : (s.cols - 1) & ~3;
    raw4<K, decltype(wide)::value>(u, s, g, [&](int j, int& row, int& col, int& valid) {
      row = min(k0 + ty + 16 * j, s.rows - 1);
      col = in;
      valid = s.cols - in;
    });
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = ty + 16 * j;
      const f32x4 v = update4<false>(s, u[j], g, k0 + i, l0 + q, s.cols - l0 - q);
      const bool inside = k0 + i < s.rows && l0 + q < s.cols;
#pragma unroll
      for (int e = 0; e < 4; ++e) tile[q + e][i] = inside ? (float)((double)v[e] * inv) : 0.f;
    }
  });
  __syncthreads();
  for (int i = ty; i < 64; i += 16)
    if (l0 + i < s.cols && k0 + q < (x.ld >> 1)) {
      f32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = k0 + q + e < s.rows ? tile[i][q + e] : 0.f;
      store_planes(x, g, l0 + i, k0 + q, v);
    }
}

// ------------------------------------------------------------------------------------------ products
enum Epi { PLANES, POLY, PARTIAL, OUT, STEP };

struct Prod {
  Planes a, b;
  int m, n, r, models, tiles_m, tiles_n, splits, per_split;
  int symmetric;     // the result is: tiles above the diagonal are not computed but written twice
  float alpha;       // value = alpha * sum
  Planes out;        // PLANES, POLY: value times the output's scale (in alpha)
  Planes add;        // POLY: A, whose square the product is
  float ca, cb, cc;  // POLY: out = ca I + cb A + cc sum, times the scales
  float* partial;    // PARTIAL: [split][model][m][n]
  void* dst;         // OUT: the result; STEP: the weights
  int64_t dst_stride, dst_ld;
  int transposed;    // OUT, STEP: dst is [n][m]
  float keep, step;  // STEP: w = keep w - step value
};

// tile i of those at and below the diagonal: (0,0) (1,0) (1,1) (2,0) ...
__device__ __forceinline__ void lower_tile(int i, int& tm, int& tn) {
  tm = (int)((sqrtf(8.f * i + 1.f) - 1.f) * 0.5f);
  while (tm * (tm + 1) / 2 > i) --tm;
  while ((tm + 1) * (tm + 2) / 2 <= i) ++tm;
  tn = i - tm * (tm + 1) / 2;
}

// GRAM: both operands are X and the sum runs over its rows.  Bound by the latency of a tile's step and the two epilogues of a
// mirrored tile where the k x k products give a CU one workgroup: 16 x 512^3 takes 22 to 29 us, 3 x 777^3 16 to 18, the matrix cores
// busy 17 to 27 % of the CUs' cycles.  2 x 2048 x 2048, five steps: 1.46 ms, 236 TFLOP/s of the 341 that split fp16 allows,
// busy 34 to 57 %.
template <Kind K, bool GRAM, Epi E, int WM, int WN, int FM, int FN, int STAGES>
__global__ __launch_bounds__(64 * WM * WN) void product_kernel(const Prod p) {
  typedef Block<F16, GRAM, GRAM, WM, WN, FM, FN, 64, 2, STAGES> B;
  __shared__ __attribute__((aligned(16))) char lds[B::LDS_BYTES];
  int64_t b = xcd_block();
  int tm, tn;
  if (p.symmetric) {
    const int tiles = p.tiles_m * (p.tiles_m + 1) / 2;
    lower_tile((int)(b % tiles), tm, tn);
    b /= tiles;
  } else {
    tn = (int)(b % p.tiles_n);
    b /= p.tiles_n;
    tm = (int)(b % p.tiles_m);
    b /= p.tiles_m;
  }
  const int sp = (int)(b % p.splits), g = (int)(b / p.splits);
  const int m0 = tm * B::BM, n0 = tn * B::BN;
  const int rend = GRAM ? p.r : p.a.ld / 2;  // along r: zeros behind p.r
  const int nk = (rend + B::BK - 1) / B::BK;
  const int first = sp * p.per_split, last = min(nk, first + p.per_split);
  Operand<uint16_t> oa, ob;
  oa.p = p.a.p + g * p.a.stride;
  oa.ld = p.a.ld;
  oa.rows = GRAM ? p.a.ld / 2 : p.m;  // whole chunks of columns: the planes' padding is zero
  ob.p = p.b.p + g * p.b.stride;
  ob.ld = p.b.ld;
  ob.rows = GRAM ? p.b.ld / 2 : p.n;
  B blk;
  blk.clear();
  blk.run(lds, oa, ob, m0, n0, first * B::BK, min(rend, last * B::BK), true);
  if constexpr (E == PARTIAL) {
    float* out = p.partial + ((int64_t)sp * p.models + g) * p.m * p.n;
    blk.each_row(lds, m0, n0, [](int, int) { return 0; }, [&](int m, int n, f32x4 v, int) {
      if (m < p.m && n < p.n) store4<F32>(out + (int64_t)m * p.n + n, v, p.n - n);
    });
  } else if constexpr (E == PLANES || E == POLY) {
    // the same for a tile and its mirror image; zeros behind the last column
    auto before = [&](int m, int n) {
      return E == POLY && m < p.m && n < p.n ? load_planes(p.add, g, m, n) : f32x4{0.f, 0.f, 0.f, 0.f};
    };
    auto result = [&](int m, int n, f32x4 v, f32x4 x) {
      if (m >= p.m || n >= p.out.ld / 2) return;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (E == POLY) v[i] = p.cc * v[i] + (p.cb * x[i] + (n + i == m ? p.ca : 0.f));
        else v[i] *= p.alpha;
        if (n + i >= p.n) v[i] = 0.f;
      }
      store_planes(p.out, g, m, n, v);
    };
    blk.each_row(lds, m0, n0, before, result);
    if (p.symmetric && tm != tn) {
      __syncthreads();
      blk.each_column(lds, m0, n0, before, result);
    }
  } else {
    typedef typename Elem<K>::T T;
    T* dst = reinterpret_cast<T*>(p.dst) + g * p.dst_stride;
    const int rows = p.transposed ? p.n : p.m, cols = p.transposed ? p.m : p.n;
    auto result = [&](int r, int c, f32x4 v, auto w) {
      if (r >= rows || c >= cols) return;
      v *= p.alpha;
      if constexpr (E == STEP)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = p.keep * w[i] - p.step * v[i];
      store4<K>(dst + r * p.dst_ld + c, v, cols - c);
    };
    auto finish = [&](auto before) {
      if (p.transposed) blk.each_column(lds, m0, n0, before, result);
      else blk.each_row(lds, m0, n0, before, result);
    };
    if constexpr (E == STEP)
      by_width(cols, [&](auto wide) {
        finish([&](int r, int c) {
          return r < rows && c < cols ? load4<K, decltype(wide)::value>(dst + r * p.dst_ld + c, cols - c) : f32x4{0.f, 0.f, 0.f, 0.f};
        });
      });
    else finish([](int, int) { return 0; });
  }
}

// the Gram matrix from its partial sums, added in order: 64 x 64 tiles at and below the diagonal, the others mirrored
__global__ __launch_bounds__(256) void join_kernel(const Prod p) {
  __shared__ float tile[64][65];
  const int g = blockIdx.y;
  int tm, tn;
  lower_tile(blockIdx.x, tm, tn);
  const int m0 = tm * 64, n0 = tn * 64;
  const float* src = p.partial + (int64_t)g * p.m * p.n;
  const int64_t step = (int64_t)p.models * p.m * p.n;
  const int q = (threadIdx.x & 15) * 4;
  by_width(p.n, [&](auto wide) {
    for (int i = threadIdx.x >> 4; i < 64; i += 16) {
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
      const int m = m0 + i, n = n0 + q;
      if (m < p.m && n < p.n) {
        const float* at = src + (int64_t)m * p.n + n;
#pragma unroll 4
        for (int s = 0; s < p.splits; ++s) v += load4<F32, decltype(wide)::value>(at + s * step, p.n - n);
        v *= p.alpha;
      }
      if (m < p.m && n < p.out.ld / 2) store_planes(p.out, g, m, n, v);
#pragma unroll
      for (int e = 0; e < 4; ++e) tile[q + e][i] = v[e];
    }
  });
  if (tm == tn) return;
  __syncthreads();
  for (int i = threadIdx.x >> 4; i < 64; i += 16) {
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = tile[i][q + e];
    if (n0 + i < p.n && m0 + q < p.out.ld / 2) store_planes(p.out, g, n0 + i, m0 + q, v);
  }
}

// ------------------------------------------------------------------------------------------ matrices that fit in LDS
// One workgroup does everything for one model: U (and the momentum) is read once, X stays in LDS in fp32, and so do the
// k x k matrices; all products on v_mfma_f32_16x16x4.  Bound by the latency of that chain: 30 x 288 x 32 in 23 us, 1023 x
// 128 x 10 with its momentum and weights in 16 us.  Such a matrix needs 10 MFLOP or less, so what counts is that one
// launch replaces 20.  KT: k in tiles of 16.  Rows of S = 16 KT + 4 floats put the 16 rows of a fragment on different banks.
// A fragment of 16 r is one 16-byte read per lane: lane (i, h) holds r = 4 h .. 4 h + 3 and instruction e takes its
// element e - the order of r is free as long as both operands agree.
struct Small {
  Source src;
  int L, k, tall, steps, phases;
  float a, b, c;
  void* dst;
  int64_t dst_stride, dst_ld;
  float keep, step;
};

constexpr int small_scratch(int KT) {  // floats: T, P and Q, or four waves' partial Gram tiles
  const int mats = 3 * 16 * KT * (16 * KT + 4), parts = 4 * 256 * (KT * (KT + 1) / 2);
  return mats > parts ? mats : parts;
}

template <int KT> struct SmallBlock {
  static constexpr int KP = 16 * KT, S = KP + 4;
  static __device__ __forceinline__ f32x4 frag(const float* m, int row, int s, int lane) {
    return *reinterpret_cast<const f32x4*>(m + (row + (lane & 15)) * S + 16 * s + 4 * (lane >> 4));
  }
  // tile (ti, tj) of lhs rhs^T
  static __device__ __forceinline__ f32x4 tile(const float* lhs, const float* rhs, int ti, int tj, int lane) {
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < KT; ++s) {
      const f32x4 a = frag(lhs, ti * 16, s, lane), b = frag(rhs, tj * 16, s, lane);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], acc, 0, 0, 0);
    }
    return acc;
  }
  // out = f(row, col, lhs rhs) for symmetric matrices that commute; out is neither
  template <typename F> static __device__ __forceinline__ void product(float* out, const float* lhs, const float* rhs, F f) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int t = wave; t < KT * KT; t += 4) {
      const int ti = t / KT, tj = t % KT;
      const f32x4 v = tile(lhs, rhs, ti, tj, lane);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = ti * 16 + (lane >> 4) * 4 + e, col = tj * 16 + (lane & 15);
        out[row * S + col] = f(row, col, v[e]);
      }
    }
    __syncthreads();
  }
  // A = X^T X; rows of X dealt to the waves, four at a time; the waves' sums added in order
  static __device__ __forceinline__ void gram(float* A, const float* X, float* scratch, int Lp) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    constexpr int TILES = KT * (KT + 1) / 2;
    f32x4 acc[TILES];
#pragma unroll
    for (int i = 0; i < TILES; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int l = wave * 4; l < Lp; l += 16) {
      float f[KT];
#pragma unroll
      for (int t = 0; t < KT; ++t) f[t] = X[(l + (lane >> 4)) * S + t * 16 + (lane & 15)];
      int i = 0;
#pragma unroll
      for (int ti = 0; ti < KT; ++ti)
#pragma unroll
        for (int tj = 0; tj <= ti; ++tj, ++i) acc[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(f[ti], f[tj], acc[i], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < TILES; ++i) *reinterpret_cast<f32x4*>(scratch + ((wave * TILES + i) * 64 + lane) * 4) = acc[i];
    __syncthreads();
    for (int i = wave; i < TILES; i += 4) {
      const float* at = scratch + (i * 64 + lane) * 4;
      f32x4 v = *reinterpret_cast<const f32x4*>(at);
#pragma unroll
      for (int w = 1; w < 4; ++w) v += *reinterpret_cast<const f32x4*>(at + w * TILES * 256);
      int ti = 0;
      while ((ti + 1) * (ti + 2) / 2 <= i) ++ti;
      const int tj = i - ti * (ti + 1) / 2;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = ti * 16 + (lane >> 4) * 4 + e, col = tj * 16 + (lane & 15);
        A[row * S + col] = v[e];
        if (ti != tj) A[col * S + row] = v[e];
      }
    }
    __syncthreads();
  }
  // X = X Q, each wave its own rows
  static __device__ __forceinline__ void apply(float* X, const float* Q, int Lp) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int r = wave * 16; r < Lp; r += 64) {
      f32x4 v[KT];
#pragma unroll
      for (int t = 0; t < KT; ++t) v[t] = tile(X + r * S, Q, 0, t, lane);
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) X[(r + (lane >> 4) * 4 + e) * S + t * 16 + (lane & 15)] = v[t][e];
    }
    __syncthreads();
  }
};

template <Kind K, int KT, Epi E> __global__ __launch_bounds__(256) void small_kernel(const Small p) {
  typedef SmallBlock<KT> B;
  typedef typename Elem<K>::T T;  // of U
  constexpr int S = B::S, MAT = B::KP * S;
  extern __shared__ __attribute__((aligned(16))) float sm[];
  __shared__ double part[4];
  const int g = blockIdx.x, tid = threadIdx.x;
  const int Lp = (p.L + 15) & ~15;
  float* X = sm;
  float* A = X + Lp * S;
  float* scratch = A + MAT;
  const Source& s = p.src;
  const int n4 = (s.cols + 3) >> 2;
  for (int i = tid * 4; i < Lp * S; i += 1024) *reinterpret_cast<f32x4*>(X + i) = f32x4{0.f, 0.f, 0.f, 0.f};
  __syncthreads();
  double sum = 0.;
  by_width(s.cols, [&](auto wide) {
    for (Walk w(tid, 256, n4); w.r < s.rows;) {
      Raw x[4];
      int r[4], c[4];
#pragma unroll
      for (int j = 0; j < 4; ++j, w.next()) {  // behind the last row: the last one again, not used
        r[j] = w.r;
        c[j] = w.c4 * 4;
      }
      raw4<K, decltype(wide)::value>(x, s, g, [&](int j, int& row, int& col, int& valid) {
        row = min(r[j], s.rows - 1);
        col = c[j];
        valid = s.cols - col;
      });
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (r[j] < s.rows) {
          const f32x4 v = update4<true>(s, x[j], g, r[j], c[j], s.cols - c[j]);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (c[j] + e < s.cols) {
              X[p.tall ? r[j] * S + c[j] + e : (c[j] + e) * S + r[j]] = v[e];
              sum += (double)v[e] * (double)v[e];
            }
        }
    }
  });
  const double inv = inverse_norm(block_sum(sum, part)) * (1. / X_SCALE);
  for (int i = tid * 4; i < Lp * S; i += 1024) {
    f32x4 v = *reinterpret_cast<f32x4*>(X + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (float)((double)v[e] * inv);
    *reinterpret_cast<f32x4*>(X + i) = v;
  }
  __syncthreads();
  int done = 0;
  for (int ph = 0; ph < p.phases; ++ph) {
    const int n = (p.steps - done + (p.phases - ph) - 1) / (p.phases - ph);
    done += n;
    B::gram(A, X, scratch, Lp);
    float *P = scratch, *T1 = scratch + MAT, *Q = scratch + 2 * MAT;
    for (int i = 0; i < n; ++i) {
      float* cur = i == 0 ? Q : P;
      B::product(cur, A, A, [&](int row, int col, float v) {
        return p.c * v + (p.b * A[row * S + col] + (row == col ? p.a : 0.f));
      });
      auto same = [](int, int, float v) { return v; };
      if (i + 1 < n) {
        B::product(T1, cur, A, same);
        B::product(A, T1, cur, same);
      }
      if (i > 0) {
        B::product(T1, P, Q, same);
        float* h = Q;
        Q = T1;
        T1 = h;
      }
    }
    B::apply(X, Q, Lp);
  }
  typedef typename Elem<E == STEP ? F32 : K>::T O;
  O* dst = reinterpret_cast<O*>(p.dst) + g * p.dst_stride;
  for (Walk w(tid, 256, n4); w.r < s.rows; w.next()) {
    const int c = w.c4 * 4;
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = c + e < s.cols ? X[p.tall ? w.r * S + c + e : (c + e) * S + w.r] : 0.f;
    O* at = dst + w.r * p.dst_ld + c;
    if constexpr (E == STEP) {
      const f32x4 old = load4<F32, false>(at, s.cols - c);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = p.keep * old[e] - p.step * v[e];
      store4<F32>(at, v, s.cols - c);
    } else {
      store4<K>(at, v, s.cols - c);
    }
  }
}

// ------------------------------------------------------------------------------------------ narrow matrices: k <= 128
// U is read three times and nothing of its size but the result is written: the Gram matrix of U itself (whose trace is
// |U|^2: no pass for the norm), the Gram matrix of U Q1 formed on the way, and the result U (Q1 Q2).  What is between runs
// on one workgroup per model with all k x k matrices in LDS.  45 x 9216 x 128 fp32: 68, 127 and 103 us, where their bytes at a
// copy's rate or their products need 44, 60 and 89.  A workgroup alone on its CU passes three or four barriers per piece
// of rows with nothing to fill them, and the second pass spends 47 % of its LDS cycles in bank conflicts (Y, read across).
// KP: k padded to 64 or 128; a workgroup of 8 waves takes TR = 16384 / KP rows l of X at a time, the next ones on their
// way in registers.  TALL: L = rows.  Before |U| is known, a workgroup scales by a power of two that it raises (with what
// it has summed) when a larger value comes: split fp16 holds any range.
constexpr int NARROW_THREADS = 512;  // with Q in LDS: one workgroup per CU
constexpr int GRAM_THREADS = 256;    // without: several, whose conversions and products overlap

struct Square {  // planes of a KP x KP matrix as they lie in LDS, hi then lo, one after the other for each model
  char* p;
};

struct Narrow {
  Source src;
  int L, k, chunks, rows_per;  // chunks per model, rows l of one
  float* partial;              // [model][chunk][tile][1024]
  int* exponent;               // [model][chunk]
  double* inv;                 // [model] 1 / |U|
  Square q;                    // [model] Q
  float q_scale;
  void* dst;
  int64_t dst_stride, dst_ld;
  float keep, step;
};

// an LDS matrix of 16-bit elements with rows of RB bytes, read along its rows (chunks of 16 bytes exchanged by row)
template <int RB> __device__ __forceinline__ int along(int row, int elem) {
  const int s = RB >= 256 ? row & 15 : (row >> 1) & 7;
  return row * RB + (((elem >> 3) ^ s) << 4) + (elem & 7) * 2;
}
template <int RB> __device__ __forceinline__ u32x4 frag_along(const char* m, int row, int ks, int lane) {
  return *reinterpret_cast<const u32x4*>(m + along<RB>(row + (lane & 31), (2 * ks + (lane >> 5)) * 8));
}
// read across its rows (rows of RB + 64 bytes)
template <int RB> __device__ __forceinline__ u32x4 frag_across(const char* m, int i, int ks, int lane) {
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  const int q = lane & 15, r = (2 * ks + (lane >> 5)) * 8 + (q >> 2);
  const char* a = m + r * (RB + 64) + (i + (lane & 16) + 4 * (q & 3)) * 2;
  const u32x2 w0 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(a)));
  const u32x2 w1 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(a + 4 * (RB + 64))));
  u32x4 v;
  v[0] = w0[0]; v[1] = w0[1]; v[2] = w1[0]; v[3] = w1[1];
  return v;
}
__device__ __forceinline__ void put_split(char* hi, char* lo, f32x4 v) {
  uint16_t h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) split(v[i], h[i], l[i]);
  u32x2 a, b;
  a[0] = h[0] | (uint32_t)h[1] << 16;
  a[1] = h[2] | (uint32_t)h[3] << 16;
  b[0] = l[0] | (uint32_t)l[1] << 16;
  b[1] = l[2] | (uint32_t)l[3] << 16;
  *reinterpret_cast<u32x2*>(hi) = a;
  *reinterpret_cast<u32x2*>(lo) = b;
}
__device__ __forceinline__ void mfma3(f32x16& d, const u32x4* a, const u32x4* b) {  // a, b: hi and lo
  mfma<F16>(d, b[1], a[0], 0);
  mfma<F16>(d, b[0], a[1], 0);
  mfma<F16>(d, b[0], a[0], 0);
}

// TR rows l of U in registers, as 4-element pieces of U's rows
template <Kind K, int KP, bool TALL, int NT> struct Piece {
  static constexpr int TR = 32 * NT / KP, N = 8;
  static constexpr int RB = (TALL ? KP : TR) * 2;            // a stored row
  static constexpr int ACROSS = (TALL ? TR : KP) * (RB + 64);  // bytes of a plane
  static constexpr int ALONG = (TALL ? TR : KP) * RB;
  f32x4 u[N];
  static __device__ __forceinline__ void place(int j, int& row, int& col) {  // of the stored tile
    constexpr int PER = RB / 8;
    const int c = threadIdx.x + j * NT;
    row = c / PER;
    col = (c % PER) * 4;
  }
  Raw raw[N];
  __device__ __forceinline__ bool inside(int j, int l0, int lend, int k, int& r, int& c, int& valid) const {
    int row, col;
    place(j, row, col);
    r = TALL ? l0 + row : row;
    c = TALL ? col : l0 + col;
    valid = (TALL ? k : lend) - c;
    return r < (TALL ? lend : k) && valid > 0;
  }
  // asks for the rows, and takes what has come
  __device__ __forceinline__ void ask(const Source& s, int g, int l0, int lend, int k) {
    // what is not inside reads the first element's group, and is not used; a wide matrix's row goes on behind a chunk
    raw4<K, true>(raw, s, g, [&](int j, int& r, int& c, int& valid) {
      const bool in = inside(j, l0, lend, k, r, c, valid);
      r = in ? r : 0;
      valid = in ? (TALL ? valid : s.cols - c) : 4;
      c = in ? c : 0;
    });
  }
  template <bool FIRST> __device__ __forceinline__ void take(const Source& s, int g, int l0, int lend, int k) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      int r, c, valid;
      const bool in = inside(j, l0, lend, k, r, c, valid);
      f32x4 v = raw[j].g;
      if (s.m && (!FIRST || in)) v = update4<FIRST>(s, raw[j], g, r, c, valid);
#pragma unroll
      for (int e = 0; e < 4; ++e) u[j][e] = in && e < valid ? v[e] : 0.f;
    }
  }
  // planes for a sum over l (GRAM) or over k: whichever of the stored rows' directions that is
  template <bool GRAM, typename F> __device__ __forceinline__ void store(char* lds, F scaled) const {
    constexpr bool IS_ACROSS = GRAM == TALL;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      int row, col;
      place(j, row, col);
      const int at = IS_ACROSS ? row * (RB + 64) + col * 2 : along<RB>(row, col);
      f32x4 v = u[j];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = scaled(v[e]);
      put_split(lds + at, lds + (IS_ACROSS ? ACROSS : ALONG) + at, v);
    }
  }
};

// Gram tiles of 32 x 32 at and below the diagonal, at most 3 per wave; KP = 64: every wave has all 3 and its own l,
// KP = 128: groups of 4 waves share the tiles and have their own l
template <int KP, int NT> struct GramTiles {
  static constexpr int TILES = KP == 128 ? 10 : 3, GROUPS = KP == 128 ? NT / 256 : NT / 64, STEP = KP == 128 ? 4 : 1;
  static constexpr int KS = 32 * NT / KP / 16 / GROUPS;  // k-steps of a wave
  f32x16 acc[3];
  int ti[3], tj[3], n, group;
  __device__ __forceinline__ void init() {
    const int wave = threadIdx.x >> 6, member = KP == 128 ? wave & 3 : 0;
    group = KP == 128 ? wave >> 2 : wave;
    n = 0;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const int t = member + i * STEP;
      ti[i] = tj[i] = 0;
      if (t < TILES) {
        lower_tile(t, ti[i], tj[i]);
        n = i + 1;
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][e] = 0.f;
    }
  }
  // frag(plane, i, ks): of rows i .. i + 31 of X^T
  template <typename F> __device__ __forceinline__ void add(F frag) {
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int ks = group * KS + s;
#pragma unroll
      for (int i = 0; i < 3; ++i)
        if (i < n) {
          const u32x4 a[2] = {frag(0, ti[i] * 32, ks), frag(1, ti[i] * 32, ks)};
          const u32x4 b[2] = {frag(0, tj[i] * 32, ks), frag(1, tj[i] * 32, ks)};
          mfma3(acc[i], a, b);
        }
    }
  }
  // the groups' sums, added in order, to out [tile][1024]: value (m, n) of a tile at lane (m | ..) * 16 + ..
  __device__ __forceinline__ void finish(char* lds, float* out) {
    float* buf = reinterpret_cast<float*>(lds);
    const int lane = threadIdx.x & 63, member = KP == 128 ? (threadIdx.x >> 6) & 3 : 0;
    for (int gr = 0; gr < GROUPS; ++gr) {
      __syncthreads();
      if (group == gr)
#pragma unroll
        for (int i = 0; i < 3; ++i)
          if (i < n)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              f32x4* at = reinterpret_cast<f32x4*>(buf + (member + i * STEP) * 1024 + q * 256 + lane * 4);
              f32x4 v;
#pragma unroll
              for (int e = 0; e < 4; ++e) v[e] = acc[i][4 * q + e];
              *at = gr ? *at + v : v;
            }
    }
    __syncthreads();
    for (int i = threadIdx.x * 4; i < TILES * 1024; i += NT * 4)
      *reinterpret_cast<f32x4*>(out + i) = *reinterpret_cast<const f32x4*>(buf + i);
  }
};

// pass 1: the momentum; partial Gram matrices of U
template <Kind K, int KP, bool TALL> __global__ __launch_bounds__(GRAM_THREADS) void narrow_gram_kernel(const Narrow p) {
  typedef Piece<K, KP, TALL, GRAM_THREADS> Pc;
  typedef GramTiles<KP, GRAM_THREADS> Gt;
  constexpr int BYTES = 2 * (TALL ? Pc::ACROSS : Pc::ALONG), SUM = Gt::TILES * 4096;
  __shared__ __attribute__((aligned(16))) char lds[BYTES > SUM ? BYTES : SUM];
  __shared__ float most[GRAM_THREADS / 64];
  const int g = blockIdx.y, chunk = blockIdx.x, lane = threadIdx.x & 63;
  const int begin = chunk * p.rows_per, end = begin + min(p.L - begin, p.rows_per);  // no sum passes L
  Pc pc;
  Gt gt;
  gt.init();
  int exponent = -300;  // values are below 2^(exponent + 14); nothing seen yet
  pc.ask(p.src, g, begin, end, p.k);
  for (int l0 = begin; l0 < end; l0 += Pc::TR) {
    pc.template take<true>(p.src, g, l0, end, p.k);
    float mx = 0.f;
#pragma unroll
    for (int j = 0; j < Pc::N; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) mx = fmaxf(mx, fabsf(pc.u[j][e]));
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor(mx, d, 64));
    if (lane == 0) most[threadIdx.x >> 6] = mx;
    __syncthreads();  // also: the last tile's planes are read
#pragma unroll
    for (int w = 0; w < GRAM_THREADS / 64; ++w) mx = fmaxf(mx, most[w]);
    int e;
    frexpf(mx, &e);  // mx < 2^e
    e = mx > 0.f ? (mx < INFINITY ? e : 128) - 14 : -300;
    if (e > exponent) {
      if (exponent > -300)
#pragma unroll
        for (int i = 0; i < 3; ++i)
#pragma unroll
          for (int v = 0; v < 16; ++v) gt.acc[i][v] = ldexpf(gt.acc[i][v], 2 * (exponent - e));
      exponent = e;
    }
    const int down = exponent > -300 ? -exponent : 0;
    pc.template store<true>(lds, [&](float v) { return ldexpf(v, down); });
    __syncthreads();
    if (l0 + Pc::TR < end) pc.ask(p.src, g, l0 + Pc::TR, end, p.k);
    gt.add([&](int plane, int i, int ks) {
      if constexpr (TALL) return frag_across<Pc::RB>(lds + plane * Pc::ACROSS, i, ks, lane);
      else return frag_along<Pc::RB>(lds + plane * Pc::ALONG, i, ks, lane);
    });
  }
  const int64_t slot = (int64_t)g * p.chunks + chunk;
  gt.finish(lds, p.partial + slot * (Gt::TILES * 1024));
  if (threadIdx.x == 0) p.exponent[slot] = exponent;
}

// the chunks' partial sums, added in order at the largest exponent, into the first chunk's place
__global__ __launch_bounds__(256) void narrow_join_kernel(float* partial, const int* exponent, int chunks, int n) {
  const int g = blockIdx.y, i = (blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  float* at = partial + (int64_t)g * chunks * n + i;
  int top = -300;
  if (exponent)
    for (int c = 0; c < chunks; ++c) top = max(top, exponent[(int64_t)g * chunks + c]);
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  for (int c0 = 0; c0 < chunks; c0 += 8) {
    f32x4 x[8];
#pragma unroll
    for (int c = 0; c < 8; ++c)
      if (c0 + c < chunks) x[c] = *reinterpret_cast<const f32x4*>(at + (int64_t)(c0 + c) * n);
#pragma unroll
    for (int c = 0; c < 8; ++c)
      if (c0 + c < chunks) {
        if (exponent) {
          const int d = 2 * (exponent[(int64_t)g * chunks + c0 + c] - top);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[c][e] = ldexpf(x[c][e], d);
        }
        v += x[c];
      }
  }
  *reinterpret_cast<f32x4*>(at) = v;
}

template <int KP> __device__ __forceinline__ void load_square(char* lds, const Square& q, int g) {
  constexpr int BYTES = KP * KP * 4;
  const char* src = q.p + (int64_t)g * BYTES;
  for (int i = threadIdx.x * 16; i < BYTES; i += blockDim.x * 16)
    *reinterpret_cast<u32x4*>(lds + i) = *reinterpret_cast<const u32x4*>(src + i);
}

// passes 2 and 3: Y = U Q / |U| by TR rows.  GRAM: partial Gram matrices of Y; otherwise Y is the result.
template <Kind K, int KP, bool TALL, bool GRAM, Epi E>
__global__ __launch_bounds__(NARROW_THREADS) void narrow_apply_kernel(const Narrow p) {
  typedef Piece<K, KP, TALL, NARROW_THREADS> Pc;
  typedef GramTiles<KP, NARROW_THREADS> Gt;
  constexpr int TR = Pc::TR, QB = KP * KP * 2, YB = TR * (KP * 2 + 64);
  constexpr int XB = TALL ? Pc::ALONG : Pc::ACROSS;  // a plane of U
  constexpr int OUT_LD = TALL ? 68 : 36, OUT = 8 * (TALL ? 32 : 64) * OUT_LD * 4;
  constexpr int A = 2 * XB, B = GRAM ? 2 * YB : OUT, SUM = GRAM ? Gt::TILES * 4096 : 0;
  constexpr int REST = A > B ? A : B;
  __shared__ __attribute__((aligned(16))) char lds[2 * QB + (REST > SUM ? REST : SUM)];
  char* const xs = lds + 2 * QB;
  const int g = blockIdx.y, chunk = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int begin = chunk * p.rows_per, end = begin + min(p.L - begin, p.rows_per);  // no sum passes L
  const int wr = KP == 128 ? wave >> 1 : wave, wc = KP == 128 ? wave & 1 : 0;  // 32 rows l, 64 columns
  const double inv = p.inv[g] * (double)X_SCALE;
  const float back = GRAM ? 1.f / p.q_scale : 1.f / (X_SCALE * p.q_scale);
  Pc pc;
  Gt gt;
  if constexpr (GRAM) gt.init();
  pc.ask(p.src, g, begin, end, p.k);
  load_square<KP>(lds, p.q, g);
  for (int l0 = begin; l0 < end; l0 += TR) {
    pc.template take<false>(p.src, g, l0, end, p.k);
    __syncthreads();  // the last tile is done with
    pc.template store<false>(xs, [&](float v) { return (float)((double)v * inv); });
    __syncthreads();
    if (l0 + TR < end) pc.ask(p.src, g, l0 + TR, end, p.k);
    f32x16 acc[2];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[j][e] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KP / 16; ++ks) {
      u32x4 x[2];
#pragma unroll
      for (int pl = 0; pl < 2; ++pl) {
        if constexpr (TALL) x[pl] = frag_along<Pc::RB>(xs + pl * XB, wr * 32, ks, lane);
        else x[pl] = frag_across<Pc::RB>(xs + pl * XB, wr * 32, ks, lane);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const u32x4 q[2] = {frag_along<KP * 2>(lds, wc * 64 + j * 32, ks, lane), frag_along<KP * 2>(lds + QB, wc * 64 + j * 32, ks, lane)};
        // a lane gets 4 consecutive columns of a row l; the result of a wide matrix: 4 consecutive l of a column
        if (GRAM || TALL) mfma3(acc[j], x, q);
        else mfma3(acc[j], q, x);
      }
    }
    __syncthreads();  // U is read: its place takes Y
    if constexpr (GRAM) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          f32x4 v;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = acc[j][4 * q + e] * back;
          const int at = (wr * 32 + (lane & 31)) * (KP * 2 + 64) + (wc * 64 + j * 32 + 8 * q + 4 * (lane >> 5)) * 2;
          put_split(xs + at, xs + YB + at, v);
        }
      __syncthreads();
      gt.add([&](int plane, int i, int ks) { return frag_across<KP * 2>(xs + plane * YB, i, ks, lane); });
    } else {
      typedef typename Elem<E == STEP ? F32 : K>::T O;
      O* dst = reinterpret_cast<O*>(p.dst) + g * p.dst_stride;
      float* buf = reinterpret_cast<float*>(xs) + wave * (TALL ? 32 : 64) * OUT_LD;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          f32x4 v;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = acc[j][4 * q + e] * back;
          // TALL: row l, columns j; otherwise row n of 64, columns l
          const int row = (TALL ? 0 : j * 32) + (lane & 31), col = (TALL ? j * 32 : 0) + 8 * q + 4 * (lane >> 5);
          *reinterpret_cast<f32x4*>(buf + row * OUT_LD + col) = v;
        }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      constexpr int PERROW = TALL ? 16 : 8;
#pragma unroll
      for (int i = 0; i < (TALL ? 32 : 64); i += 64 / PERROW) {
        const int row = i + lane / PERROW, col = (lane % PERROW) * 4;
        f32x4 v = *reinterpret_cast<const f32x4*>(buf + row * OUT_LD + col);
        const int r = TALL ? l0 + wr * 32 + row : wc * 64 + row, c = TALL ? wc * 64 + col : l0 + wr * 32 + col;
        const int rend = TALL ? end : p.k, cend = TALL ? p.k : end;
        if (r < rend && c < cend) {
          O* at = dst + r * p.dst_ld + c;
          if constexpr (E == STEP) {
            const f32x4 old = load4<F32, true>(at, cend - c);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = p.keep * old[e] - p.step * v[e];
            store4<F32>(at, v, cend - c);
          } else {
            store4<K>(at, v, cend - c);
          }
        }
      }
    }
  }
  if constexpr (GRAM) gt.finish(xs, p.partial + ((int64_t)g * p.chunks + chunk) * (Gt::TILES * 1024));
}

// The steps of a phase on one workgroup: 8 or 5 products that wait for one another, 24 to 33 us for k = 128 whatever the batch
// up to 256 models.  Matrices live in registers (as the matrix instruction leaves them) and, as
// planes, in the two places of LDS when they are operands.
struct Chain {
  const float* partial;  // [model][chunk], joined into the first chunk's
  const int* exponent;  // first phase: A = sum / trace; NULL: A = sum / X_SCALE^2
  int chunks, n;
  double* inv;
  float a, b, c;
  float p_scale[3], q_scale[3];  // of step i
  Square before;                 // Q of the phase before (NULL: none)
  float before_scale;
  Square q;                      // the product of all Q so far
  float total_scale;
};

template <int KP> __global__ __launch_bounds__(KP * 4) void chain_kernel(const Chain p) {
  constexpr int NT = KP * 4, F = KP == 128 ? 2 : 1, RB = KP * 2, MAT = KP * RB;
  constexpr int TILES = GramTiles<KP, 256>::TILES;
  __shared__ __attribute__((aligned(16))) char lds[4 * MAT];
  const int g = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  char *const s1 = lds, *const s2 = lds + 2 * MAT;
  const int mb = (wave / 2) * 32, nb = (wave % 2) * 32 * F;
  const int row = mb + (lane & 31), col0 = nb + 4 * (lane >> 5);
  typedef f32x16 Mat[F];
  auto put = [&](char* to, const Mat& v, float scale) {
#pragma unroll
    for (int j = 0; j < F; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        f32x4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = v[j][4 * q + e] * scale;
        const int at = along<RB>(row, col0 + j * 32 + 8 * q);
        put_split(to + at, to + MAT + at, x);
      }
  };
  auto multiply = [&](Mat& v, const char* x, const char* y, float scale) {
#pragma unroll
    for (int j = 0; j < F; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) v[j][e] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KP / 16; ++ks) {
      const u32x4 a[2] = {frag_along<RB>(x, mb, ks, lane), frag_along<RB>(x + MAT, mb, ks, lane)};
#pragma unroll
      for (int j = 0; j < F; ++j) {
        const u32x4 b[2] = {frag_along<RB>(y, nb + j * 32, ks, lane), frag_along<RB>(y + MAT, nb + j * 32, ks, lane)};
        mfma3(v[j], a, b);
      }
    }
#pragma unroll
    for (int j = 0; j < F; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) v[j][e] *= scale;
  };

  // A: the tiles at and below the diagonal, mirrored through LDS
  int top = -300;
  if (p.exponent)
    for (int c = 0; c < p.chunks; ++c) top = max(top, p.exponent[(int64_t)g * p.chunks + c]);
  float* sum = reinterpret_cast<float*>(lds);  // [KP][KP + 4]
  static_assert(KP * (KP + 4) * 4 <= 4 * MAT, "the Gram matrix fits");
  for (int i = threadIdx.x * 4; i < TILES * 1024; i += NT * 4) {
    const int tile = i >> 10, in = i & 1023, q = in >> 8, ln = (in & 255) >> 2;
    const f32x4 v = *reinterpret_cast<const f32x4*>(p.partial + (int64_t)g * p.chunks * (TILES * 1024) + i);
    int ti, tj;
    lower_tile(tile, ti, tj);
    const int m = ti * 32 + (ln & 31), n = tj * 32 + 8 * q + 4 * (ln >> 5);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (ti != tj || n + e <= m) sum[m * (KP + 4) + n + e] = v[e];
      if (ti != tj || n + e < m) sum[(n + e) * (KP + 4) + m] = v[e];
    }
  }
  __syncthreads();
  float unit = 1.f / (X_SCALE * X_SCALE);
  if (p.exponent) {
    double trace = 0.;
    for (int i = 0; i < KP; ++i) trace += (double)sum[i * (KP + 4) + i];
    double inv = 0.;
    unit = 0.f;
    if (!(trace < (double)INFINITY)) inv = unit = NAN;
    else if (trace > 0.) {
      unit = (float)(1. / trace);
      inv = ldexp(1. / sqrt(trace), -top);
    }
    if (threadIdx.x == 0) p.inv[g] = inv;
  }
  Mat A, Q, T;
#pragma unroll
  for (int j = 0; j < F; ++j)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(sum + row * (KP + 4) + col0 + j * 32 + 8 * q);
#pragma unroll
      for (int e = 0; e < 4; ++e) A[j][4 * q + e] = x[e] * unit;
    }
  __syncthreads();
  put(s1, A, A_SCALE);
  __syncthreads();
  float q_scale = 1.f;
  for (int i = 0; i < p.n; ++i) {
    Mat P;
    const float ps = p.p_scale[i];
    multiply(P, s1, s1, 1.f / (A_SCALE * A_SCALE));  // P = a I + b A + c A^2
#pragma unroll
    for (int j = 0; j < F; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int col = col0 + j * 32 + 8 * (e >> 2) + (e & 3);
        P[j][e] = p.c * P[j][e] + (p.b * A[j][e] + (row == col ? p.a : 0.f));
      }
    put(s2, P, ps);
    __syncthreads();
    if (i + 1 < p.n) multiply(T, s2, s1, 1.f / (ps * A_SCALE));  // T = P A
    if (i == 0) {
#pragma unroll
      for (int j = 0; j < F; ++j) Q[j] = P[j];
    } else {  // Q = P Q
      __syncthreads();
      put(s1, Q, q_scale);
      __syncthreads();
      multiply(Q, s2, s1, 1.f / (ps * q_scale));
    }
    q_scale = p.q_scale[i];
    if (i + 1 < p.n) {  // A = T P
      __syncthreads();
      put(s1, T, A_SCALE);
      __syncthreads();
      multiply(A, s1, s2, 1.f / (A_SCALE * ps));
      __syncthreads();
      put(s1, A, A_SCALE);
      __syncthreads();
    }
  }
  if (p.before.p) {  // times the phase before
    __syncthreads();
    load_square<KP>(s1, p.before, g);
    put(s2, Q, q_scale);
    __syncthreads();
    multiply(Q, s2, s1, 1.f / (q_scale * p.before_scale));
  }
  __syncthreads();
  put(s1, Q, p.total_scale);
  __syncthreads();
  char* out = p.q.p + (int64_t)g * (2 * MAT);
  for (int i = threadIdx.x * 16; i < 2 * MAT; i += NT * 16)
    *reinterpret_cast<u32x4*>(out + i) = *reinterpret_cast<const u32x4*>(s1 + i);
}

// ------------------------------------------------------------------------------------------ host
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
size_t align16(size_t v) { return (v + 15) & ~(size_t)15; }

// Multiply-adds per cycle and CU of split products (measured on large ones)
// The last: one workgroup per CU with twice the tiles in flight, for products too small for two.
constexpr TileShape SHAPES[4] = {{256, 256, 1, 300.f}, {128, 128, 2, 250.f}, {64, 64, 2, 140.f}, {128, 128, 1, 200.f}};

// LDS of small_kernel, 0 where the matrix does not fit
size_t small_bytes(int L, int k) {
  if (k > 64) return 0;
  const int kt = (k + 15) / 16, s = 16 * kt + 4;
  const int64_t bytes = ((int64_t)((L + 15) & ~15) * s + 16 * kt * s + small_scratch(kt)) * 4;
  return bytes <= 160 * 1024 - 256 ? (size_t)bytes : 0;
}

struct Space {
  int k, L, ld, phases, chunks;
  int planned;  // the number of models that sums are split for
  size_t small;
  int narrow, rows_per;  // KP of the narrow form (0: not used), rows l of a chunk
  Choice gram;
  size_t sums, x, square, partial, total;  // bytes of one of each
  int n_x;
};

Choice shape_for(int64_t models, int64_t m, int64_t n, int64_t r, bool symmetric, bool can_split) {
  Choice best = {};
  double least = 0;
  for (int s = 0; s < 4; ++s) {  // choose() per shape, its tiles halved where the result is symmetric
    TileShape one = SHAPES[s];
    const int64_t t = ceil_div(m, one.bm);
    const int64_t tiles = symmetric ? t * (t + 1) / 2 : t * ceil_div(n, one.bn);
    double cost;
    Choice c = choose(&one, 1, models * tiles, one.bm, one.bn, r, ceil_div(r, 32), can_split, &cost);
    c.tile = s;
    c.tiles_m = t;
    c.tiles_n = symmetric ? t : ceil_div(n, one.bn);
    if (s == 0 || cost < least) {
      least = cost;
      best = c;
    }
  }
  return best;
}

int64_t blocks_of(const Choice& c, int64_t models, bool symmetric) {
  return (symmetric ? c.tiles_m * (c.tiles_m + 1) / 2 : c.tiles_m * c.tiles_n) * models * c.splits;
}

bool space(const mplc_muon_t& t, Space& s) {
  if (t.n_models < 0 || t.n_models > 65535 || t.rows < 1 || t.cols < 1 || t.dtype < 0 || t.dtype > 2) return false;
  if (t.steps < 1 || t.steps > 16) return false;
  s = Space{};
  s.planned = t.invariant ? 16 : t.n_models;
  s.k = t.rows < t.cols ? t.rows : t.cols;
  s.L = t.rows < t.cols ? t.cols : t.rows;
  s.ld = 2 * ((s.k + 31) & ~31);
  s.phases = 2 * (int64_t)s.L >= 3 * (int64_t)s.k ? (t.steps + 2) / 3 : t.steps;
  s.small = small_bytes(s.L, s.k);
  if (s.small) {  // reading X again costs nothing here: phases of two steps lose less to the Gram matrix's error
    s.phases = (t.steps + 1) / 2;
    return true;
  }
  if (s.k <= 128 && t.steps <= 6 && t.cols >= 4) {  // two phases of three steps at most; whole groups of columns
    s.narrow = s.k <= 64 ? 64 : 128;
    s.phases = (t.steps + 2) / 3;
    const int64_t tr = 16384 / s.narrow, pieces = ceil_div(s.L, tr);
    // about one workgroup per CU and round, whole pieces, at least two per workgroup where there are many
    int64_t per = ceil_div(pieces * s.planned, 512);
    if (per > pieces) per = pieces;
    per = per < 1 ? 1 : ceil_div(pieces, ceil_div(pieces, per));  // chunks of one size
    s.rows_per = (int)(per * tr);
    s.chunks = (int)ceil_div(s.L, s.rows_per);
    const size_t G = (size_t)t.n_models, tiles = s.narrow == 128 ? 10 : 3;
    s.sums = align16(G * s.chunks * sizeof(int)) + align16(G * sizeof(double));
    s.partial = align16(G * s.chunks * tiles * 4096);
    s.square = G * s.narrow * s.narrow * 4;
    s.total = s.sums + s.partial + 2 * s.square;
    return true;
  }
  s.n_x = s.phases > 1 ? 2 : 1;
  const int64_t groups = (int64_t)t.rows * ceil_div(t.cols, 4);
  if (groups > (int64_t)1 << 30) return false;
  const int64_t most = s.planned >= 16 ? 64 : NORM_CHUNKS;
  s.chunks = (int)(ceil_div(groups, 1024) < most ? ceil_div(groups, 1024) : most);
  s.gram = shape_for(s.planned, s.k, s.k, s.L, true, true);
  const size_t G = (size_t)t.n_models;
  s.sums = align16(G * s.chunks * sizeof(double));
  s.x = align16(G * s.L * s.ld * 2);
  s.square = align16(G * s.k * s.ld * 2);
  s.partial = s.gram.splits > 1 ? align16(G * s.gram.splits * (size_t)s.k * s.k * sizeof(float)) : 0;
  s.total = s.sums + s.n_x * s.x + 6 * s.square + s.partial;
  return ceil_div(s.L, 64) * ceil_div(s.k, 64) * (int64_t)t.n_models <= (1 << 23) &&
         blocks_of(s.gram, t.n_models, true) <= (1 << 23) && ceil_div(s.k, 64) <= 65535;
}

// largest |a s + b s^3 + c s^5| for s in [0, r]
double poly_bound(double a, double b, double c, double r) {
  auto f = [&](double s) { return fabs(s * (a + s * s * (b + s * s * c))); };
  double best = f(r);
  auto at = [&](double q) {
    if (q > 0 && sqrt(q) < r) best = fmax(best, f(sqrt(q)));
  };
  if (c == 0) {
    if (b != 0) at(-a / (3 * b));
  } else {
    const double d = 9 * b * b - 20 * a * c;
    if (d >= 0) {
      at((-3 * b + sqrt(d)) / (10 * c));
      at((-3 * b - sqrt(d)) / (10 * c));
    }
  }
  return best;
}
// largest |a + b q + c q^2| for q in [0, r^2]
double factor_bound(double a, double b, double c, double r) {
  auto f = [&](double q) { return fabs(a + q * (b + q * c)); };
  double best = fmax(f(0), f(r * r));
  if (c != 0 && -b / (2 * c) > 0 && -b / (2 * c) < r * r) best = fmax(best, f(-b / (2 * c)));
  return best;
}
// the largest power of two that keeps `bound` inside fp16
float scale_for(double bound) {
  int e = (int)floor(log2(60000. / fmax(bound, 1e-6)));
  if (e > 15) e = 15;
  return (float)ldexp(1., e);
}

template <Kind K, bool GRAM, Epi E> hipError_t product(Prod p, const Choice& c, hipStream_t s) {
  p.tiles_m = (int)c.tiles_m;
  p.tiles_n = (int)c.tiles_n;
  p.splits = c.splits;
  p.per_split = c.per_split;
  const dim3 grid((unsigned)blocks_of(c, p.models, p.symmetric));
  if (c.tile == 0) product_kernel<K, GRAM, E, 2, 4, 4, 2, 2><<<grid, 512, 0, s>>>(p);
  else if (c.tile == 1) product_kernel<K, GRAM, E, 2, 2, 2, 2, 2><<<grid, 256, 0, s>>>(p);
  else if (c.tile == 2) product_kernel<K, GRAM, E, 2, 2, 1, 1, 4><<<grid, 256, 0, s>>>(p);
  else product_kernel<K, GRAM, E, 2, 2, 2, 2, 4><<<grid, 256, 0, s>>>(p);
  return hipGetLastError();
}

template <Kind K, int KT, Epi E> int launch_small(const Small& p, const Space& sp, int models, hipStream_t s) {
  if (sp.small > 48 * 1024) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&small_kernel<K, KT, E>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)sp.small);
    if (e != hipSuccess) return (int)e;
  }
  small_kernel<K, KT, E><<<dim3((unsigned)models), 256, sp.small, s>>>(p);
  return (int)hipGetLastError();
}

template <Kind K, Epi E> int run_small(const mplc_muon_t& t, const Space& sp, const Source& src, hipStream_t s) {
  Small p = {src, sp.L, sp.k, t.rows >= t.cols, t.steps, sp.phases, t.a, t.b, t.c, t.out, t.out_stride, t.out_ld, 0.f, 0.f};
  if (E == STEP) {
    p.dst = t.w;
    p.dst_stride = t.w_stride;
    p.dst_ld = t.w_ld;
    p.keep = (float)(1. - (double)t.lr * t.weight_decay);
    p.step = t.lr * t.scale;
  }
  switch ((sp.k + 15) / 16) {
    case 1: return launch_small<K, 1, E>(p, sp, t.n_models, s);
    case 2: return launch_small<K, 2, E>(p, sp, t.n_models, s);
    case 3: return launch_small<K, 3, E>(p, sp, t.n_models, s);
    default: return launch_small<K, 4, E>(p, sp, t.n_models, s);
  }
}

template <Kind K, int KP, bool TALL, Epi E>
int launch_narrow(const mplc_muon_t& t, const Space& sp, const Source& src, hipStream_t s) {
  char* ws = reinterpret_cast<char*>(t.workspace);
  Narrow p = {};
  p.src = src;
  p.L = sp.L;
  p.k = sp.k;
  p.chunks = sp.chunks;
  p.rows_per = sp.rows_per;
  p.exponent = reinterpret_cast<int*>(ws);
  ws += align16((size_t)t.n_models * sp.chunks * sizeof(int));
  p.inv = reinterpret_cast<double*>(ws);
  ws += align16((size_t)t.n_models * sizeof(double));
  p.partial = reinterpret_cast<float*>(ws);
  ws += sp.partial;
  Square q[2];
  for (int i = 0; i < 2; ++i) {
    q[i].p = ws;
    ws += sp.square;
  }
  if (E == STEP) {
    p.dst = t.w;
    p.dst_stride = t.w_stride;
    p.dst_ld = t.w_ld;
    p.keep = (float)(1. - (double)t.lr * t.weight_decay);
    p.step = t.lr * t.scale;
  } else {
    p.dst = t.out;
    p.dst_stride = t.out_stride;
    p.dst_ld = t.out_ld;
  }
  const dim3 grid((unsigned)sp.chunks, (unsigned)t.n_models);
  hipError_t err;
  double r = 1., total = 1.;
  int done = 0;
  for (int ph = 0; ph < sp.phases; ++ph) {
    if (ph == 0) narrow_gram_kernel<K, KP, TALL><<<grid, GRAM_THREADS, 0, s>>>(p);
    else narrow_apply_kernel<K, KP, TALL, true, E><<<grid, NARROW_THREADS, 0, s>>>(p);
    if ((err = hipGetLastError()) != hipSuccess) return (int)err;
    if (sp.chunks > 1) {
      constexpr int n = GramTiles<KP, 256>::TILES * 1024;
      narrow_join_kernel<<<dim3(n / 1024, (unsigned)t.n_models), 256, 0, s>>>(p.partial, ph == 0 ? p.exponent : nullptr,
                                                                              sp.chunks, n);
      if ((err = hipGetLastError()) != hipSuccess) return (int)err;
    }
    Chain c = {p.partial, ph == 0 ? p.exponent : nullptr, sp.chunks, (t.steps - done + (sp.phases - ph) - 1) / (sp.phases - ph),
               p.inv, t.a, t.b, t.c, {}, {}, {}, 0.f, {}, 0.f};
    double bound = 1.;
    for (int i = 0; i < c.n; ++i) {
      const double pb = factor_bound(t.a, t.b, t.c, r);
      bound *= pb;
      c.p_scale[i] = scale_for(pb);
      c.q_scale[i] = scale_for(bound);
      r = poly_bound(t.a, t.b, t.c, r);
    }
    total *= bound;
    if (ph > 0) {
      c.before = q[0];
      c.before_scale = p.q_scale;
    }
    c.q = q[ph];
    c.total_scale = scale_for(total);
    chain_kernel<KP><<<dim3((unsigned)t.n_models), KP * 4, 0, s>>>(c);
    if ((err = hipGetLastError()) != hipSuccess) return (int)err;
    p.q = q[ph];
    p.q_scale = c.total_scale;
    done += c.n;
  }
  narrow_apply_kernel<K, KP, TALL, false, E><<<grid, NARROW_THREADS, 0, s>>>(p);
  return (int)hipGetLastError();
}

template <Kind K, Epi E> int run_narrow(const mplc_muon_t& t, const Space& sp, const Source& src, hipStream_t s) {
  const bool tall = t.rows >= t.cols;
  if (sp.narrow == 64) return tall ? launch_narrow<K, 64, true, E>(t, sp, src, s) : launch_narrow<K, 64, false, E>(t, sp, src, s);
  return tall ? launch_narrow<K, 128, true, E>(t, sp, src, s) : launch_narrow<K, 128, false, E>(t, sp, src, s);
}

template <Kind K, Epi LAST> int run(const mplc_muon_t& t, const Space& sp, const Source& src, hipStream_t s) {
  if (sp.small) return run_small<K, LAST>(t, sp, src, s);
  if (sp.narrow) return run_narrow<K, LAST>(t, sp, src, s);
  char* ws = reinterpret_cast<char*>(t.workspace);
  double* sums = reinterpret_cast<double*>(ws);
  ws += sp.sums;
  auto planes = [&](size_t bytes, int64_t stride) {
    Planes p = {reinterpret_cast<uint16_t*>(ws), stride, sp.ld};
    ws += bytes;
    return p;
  };
  Planes X[2], S[6];
  for (int i = 0; i < sp.n_x; ++i) X[i] = planes(sp.x, (int64_t)sp.L * sp.ld);
  for (int i = 0; i < 6; ++i) S[i] = planes(sp.square, (int64_t)sp.k * sp.ld);
  float* partial = reinterpret_cast<float*>(ws);
  hipError_t err;
  norm_kernel<K><<<dim3(sp.chunks, t.n_models), 256, 0, s>>>(src, sums);
  if ((err = hipGetLastError()) != hipSuccess) return (int)err;
  const bool tall = t.rows >= t.cols;
  if (tall) {
    const int64_t n = ceil_div((int64_t)t.rows * ceil_div(t.cols, 4), 1024);
    start_kernel<K><<<dim3((unsigned)(n < 1024 ? n : 1024), (unsigned)t.n_models), 256, 0, s>>>(src, sums, sp.chunks, X[0]);
  } else {
    start_wide_kernel<K><<<dim3((unsigned)ceil_div(sp.L, 64), (unsigned)ceil_div(sp.k, 64), (unsigned)t.n_models), 256, 0, s>>>(
        src, sums, sp.chunks, X[0]);
  }
  if ((err = hipGetLastError()) != hipSuccess) return (int)err;

  Prod base = {};
  base.models = t.n_models;
  const Choice small = shape_for(sp.planned, sp.k, sp.k, sp.k, true, false);
  const Choice apply = shape_for(sp.planned, sp.L, sp.k, sp.k, false, false);
  const double a = t.a, b = t.b, c = t.c;
  double r = 1.;
  int done = 0, x = 0;
  for (int ph = 0; ph < sp.phases; ++ph) {
    const int n = (t.steps - done + (sp.phases - ph) - 1) / (sp.phases - ph);
    Planes A = S[0], A2 = S[1], P = S[2], T = S[3], Q = S[4], Q2 = S[5];
    Prod p = base;  // A = X^T X
    p.a = p.b = X[x];
    p.m = p.n = sp.k;
    p.r = sp.L;
    p.symmetric = 1;
    p.alpha = A_SCALE / (X_SCALE * X_SCALE);
    p.out = A;
    p.partial = partial;
    if (sp.gram.splits > 1) {
      if ((err = product<F32, true, PARTIAL>(p, sp.gram, s)) != hipSuccess) return (int)err;
      p.splits = sp.gram.splits;
      const int64_t jt = ceil_div(sp.k, 64);
      join_kernel<<<dim3((unsigned)(jt * (jt + 1) / 2), (unsigned)t.n_models), 256, 0, s>>>(p);
      if ((err = hipGetLastError()) != hipSuccess) return (int)err;
    } else if ((err = product<F32, true, PLANES>(p, sp.gram, s)) != hipSuccess) {
      return (int)err;
    }
    auto square = [&](const Planes& l, float ls, const Planes& m, float ms, const Planes& o, float os) {
      Prod q = base;
      q.a = l;
      q.b = m;
      q.m = q.n = q.r = sp.k;
      q.symmetric = 1;
      q.alpha = os / (ls * ms);
      q.out = o;
      return product<F32, false, PLANES>(q, small, s);
    };
    double qbound = 1.;
    float q_scale = 1.f;
    for (int i = 0; i < n; ++i) {
      const double pb = factor_bound(a, b, c, r);
      const float p_scale = scale_for(pb);
      Prod q = base;  // P = a I + b A + c A^2
      q.a = q.b = q.add = A;
      q.m = q.n = q.r = sp.k;
      q.ca = t.a * p_scale;
      q.cb = t.b * (p_scale / A_SCALE);
      q.cc = t.c * (p_scale / (A_SCALE * A_SCALE));
      q.symmetric = 1;
      q.out = i == 0 ? Q : P;
      if ((err = product<F32, false, POLY>(q, small, s)) != hipSuccess) return (int)err;
      qbound *= pb;
      const Planes& cur = q.out;
      const float new_scale = i == 0 ? p_scale : scale_for(qbound);
      if (i + 1 < n) {  // the next step's A = P A P
        if ((err = square(cur, p_scale, A, A_SCALE, T, A_SCALE)) != hipSuccess) return (int)err;
        if ((err = square(T, A_SCALE, cur, p_scale, A2, A_SCALE)) != hipSuccess) return (int)err;
        const Planes h = A;
        A = A2;
        A2 = h;
      }
      if (i > 0) {
        if ((err = square(P, p_scale, Q, q_scale, Q2, new_scale)) != hipSuccess) return (int)err;
        const Planes h = Q;
        Q = Q2;
        Q2 = h;
      }
      q_scale = new_scale;
      r = poly_bound(a, b, c, r);
    }
    p = base;  // X <- X Q
    p.a = X[x];
    p.b = Q;
    p.m = sp.L;
    p.n = p.r = sp.k;
    if (ph + 1 < sp.phases) {
      p.alpha = 1.f / q_scale;
      p.out = X[1 - x];
      err = product<F32, false, PLANES>(p, apply, s);
      x = 1 - x;
    } else {
      p.alpha = 1.f / (X_SCALE * q_scale);
      p.transposed = !tall;
      if (LAST == OUT) {
        p.dst = t.out;
        p.dst_stride = t.out_stride;
        p.dst_ld = t.out_ld;
        err = product<K, false, OUT>(p, apply, s);
      } else {
        p.dst = t.w;
        p.dst_stride = t.w_stride;
        p.dst_ld = t.w_ld;
        p.keep = (float)(1. - (double)t.lr * t.weight_decay);
        p.step = t.lr * t.scale;
        err = product<F32, false, STEP>(p, apply, s);
      }
    }
    if (err != hipSuccess) return (int)err;
    done += n;
  }
  return MPLC_OK;
}

int check(const mplc_muon_t* t, Space& sp) {
  if (t == nullptr || !space(*t, sp)) return MPLC_E_ARG;
  if (!(fabsf(t->a) < 1e3f && fabsf(t->b) < 1e3f && fabsf(t->c) < 1e3f)) return MPLC_E_ARG;
  double r = 1.;
  for (int i = 0; i < t->steps; ++i) {
    r = poly_bound(t->a, t->b, t->c, r);
    if (!(r <= 2.)) return MPLC_E_ARG;
  }
  if (t->n_models == 0) return MPLC_OK;
  if (t->g == nullptr || t->g_ld < t->cols) return MPLC_E_ARG;
  if (((uintptr_t)t->workspace & 15) != 0) return MPLC_E_ARG;
  if (sp.total && (t->workspace == nullptr || t->workspace_bytes < sp.total)) return MPLC_E_WORKSPACE;
  return MPLC_OK;
}

template <Epi LAST> int dispatch(const mplc_muon_t& t, const Space& sp, const Source& src, void* stream) {
  hipStream_t s = (hipStream_t)stream;
  if (t.dtype == MPLC_DTYPE_F32) return run<F32, LAST>(t, sp, src, s);
  if (t.dtype == MPLC_DTYPE_BF16) return run<BF16, LAST>(t, sp, src, s);
  return run<F16, LAST>(t, sp, src, s);
}

}  // namespace

extern "C" size_t mplc_muon_workspace_bytes(const mplc_muon_t* t) {
  Space sp;
  return t != nullptr && space(*t, sp) ? sp.total : 0;
}

extern "C" int mplc_orthogonalize(const mplc_muon_t* t, void* stream) {
  Space sp;
  const int st = check(t, sp);
  if (st != MPLC_OK || t->n_models == 0) return st;
  if (t->out == nullptr || t->out_ld < t->cols) return MPLC_E_ARG;
  const Source src = {t->g, t->g_stride, t->g_ld, nullptr, 0, 0, 0.f, 0, t->rows, t->cols};
  return dispatch<OUT>(*t, sp, src, stream);
}

extern "C" int mplc_muon_step(const mplc_muon_t* t, void* stream) {
  Space sp;
  const int st = check(t, sp);
  if (st != MPLC_OK || t->n_models == 0) return st;
  if (t->m == nullptr || t->m_ld < t->cols || t->w == nullptr || t->w_ld < t->cols) return MPLC_E_ARG;
  const Source src = {t->g, t->g_stride, t->g_ld, t->m, t->m_stride, t->m_ld, t->beta, t->nesterov, t->rows, t->cols};
  return dispatch<STEP>(*t, sp, src, stream);
}
