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

struct Planes {  // split fp16 of a matrix times its scale
  uint16_t* hi;
  uint16_t* lo;
  int64_t stride;  // elements of one model
  int ld;
};

__device__ __forceinline__ void split(float v, uint16_t& hi, uint16_t& lo) {
  hi = f32_to_f16(v);
  lo = f32_to_f16(v - f16_to_f32(hi));
}
__device__ __forceinline__ void store_planes(const Planes& p, int g, int64_t m, int n, f32x4 v) {
  uint16_t h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) split(v[i], h[i], l[i]);
  const int64_t at = g * p.stride + m * p.ld + n;  // n and ld are multiples of 4: 8-byte aligned
  u32x2 a, b;
  a[0] = h[0] | (uint32_t)h[1] << 16;
  a[1] = h[2] | (uint32_t)h[3] << 16;
  b[0] = l[0] | (uint32_t)l[1] << 16;
  b[1] = l[2] | (uint32_t)l[3] << 16;
  *reinterpret_cast<u32x2*>(p.hi + at) = a;
  *reinterpret_cast<u32x2*>(p.lo + at) = b;
}
__device__ __forceinline__ f32x4 load_planes(const Planes& p, int g, int64_t m, int n) {
  const int64_t at = g * p.stride + m * p.ld + n;
  const u32x2 a = *reinterpret_cast<const u32x2*>(p.hi + at), b = *reinterpret_cast<const u32x2*>(p.lo + at);
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

// U at (r, c .. c + 3), `valid` of them inside; FIRST: the pass that updates the momentum
template <Kind K, bool FIRST> __device__ __forceinline__ f32x4 update4(const Source& s, int g, int64_t r, int c, int valid) {
  typedef typename Elem<K>::T T;
  f32x4 u = load4<K>(reinterpret_cast<const T*>(s.g) + g * s.g_stride + r * s.g_ld + c, valid);
  if (s.m == nullptr) return u;
  float* pm = s.m + g * s.m_stride + r * s.m_ld + c;
  f32x4 m = load4<F32>(pm, valid);
  if (FIRST) {
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = s.beta * m[i] + u[i];
    store4<F32>(pm, m, valid);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) u[i] = s.nesterov ? s.beta * m[i] + u[i] : m[i];
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
  for (Walk w(blockIdx.x * 256 + threadIdx.x, gridDim.x * 256, (s.cols + 3) >> 2); w.r < s.rows; w.next()) {
    const f32x4 v = update4<K, true>(s, g, w.r, w.c4 * 4, s.cols - w.c4 * 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) sum += (double)v[i] * (double)v[i];
  }
  sum = block_sum(sum, part);
  if (threadIdx.x == 0) sums[(int64_t)g * gridDim.x + blockIdx.x] = sum;
}

// X_0 as planes [L][ld]; L = rows
template <Kind K> __global__ __launch_bounds__(256) void start_kernel(const Source s, const double* sums, int chunks, const Planes x) {
  __shared__ double part[4];
  const int g = blockIdx.y;
  const double inv = inverse_norm(block_sum(threadIdx.x < chunks ? sums[(int64_t)g * chunks + threadIdx.x] : 0., part));
  for (Walk w(blockIdx.x * 256 + threadIdx.x, gridDim.x * 256, (s.cols + 3) >> 2); w.r < s.rows; w.next()) {
    f32x4 v = update4<K, false>(s, g, w.r, w.c4 * 4, s.cols - w.c4 * 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (float)((double)v[i] * inv);
    store_planes(x, g, w.r, w.c4 * 4, v);
  }
}

// The same with L = cols: 64 x 64 tiles, transposed through LDS
template <Kind K> __global__ __launch_bounds__(256) void start_wide_kernel(const Source s, const double* sums, int chunks, const Planes x) {
  __shared__ double part[4];
  __shared__ float tile[64][65];
  const int g = blockIdx.z;
  const double inv = inverse_norm(block_sum(threadIdx.x < chunks ? sums[(int64_t)g * chunks + threadIdx.x] : 0., part));
  const int l0 = blockIdx.x * 64, k0 = blockIdx.y * 64;
  const int q = (threadIdx.x & 15) * 4, ty = threadIdx.x >> 4;
  for (int i = ty; i < 64; i += 16) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (k0 + i < s.rows && l0 + q < s.cols) v = update4<K, false>(s, g, k0 + i, l0 + q, s.cols - l0 - q);
#pragma unroll
    for (int e = 0; e < 4; ++e) tile[q + e][i] = (float)((double)v[e] * inv);
  }
  __syncthreads();
  for (int i = ty; i < 64; i += 16)
    if (l0 + i < s.cols && k0 + q < x.ld) {
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

template <Kind K, Epi E> __device__ __forceinline__ void write_result(const Prod& p, int g, int m, int n, f32x4 v) {
  typedef typename Elem<K>::T T;
  T* dst = reinterpret_cast<T*>(p.dst) + g * p.dst_stride;
  if (!p.transposed) {
    T* at = dst + m * p.dst_ld + n;
    if constexpr (E == STEP) {
      const f32x4 w = load4<K>(at, p.n - n);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = p.keep * w[i] - p.step * v[i];
    }
    store4<K>(at, v, p.n - n);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < p.n) {
        T* at = dst + (n + i) * p.dst_ld + m;
        if constexpr (E == STEP) *at = from_f32<K>(p.keep * to_f32<K>(*at) - p.step * v[i]);
        else *at = from_f32<K>(v[i]);
      }
  }
}

// tile i of those at and below the diagonal: (0,0) (1,0) (1,1) (2,0) ...
__device__ __forceinline__ void lower_tile(int i, int& tm, int& tn) {
  tm = (int)((sqrtf(8.f * i + 1.f) - 1.f) * 0.5f);
  while (tm * (tm + 1) / 2 > i) --tm;
  while ((tm + 1) * (tm + 2) / 2 <= i) ++tm;
  tn = i - tm * (tm + 1) / 2;
}

// planes at (n .. n + 3, m): the mirror image of a tile below the diagonal
__device__ __forceinline__ void store_planes_mirrored(const Planes& p, int g, int m, int n, int N, f32x4 v) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n + i < N) {
      const int64_t at = g * p.stride + (int64_t)(n + i) * p.ld + m;
      split(v[i], p.hi[at], p.lo[at]);
    }
}

// GRAM: both operands are X and the sum runs over its rows
template <Kind K, bool GRAM, Epi E, int WM, int WN, int FM, int FN>
__global__ __launch_bounds__(64 * WM * WN) void product_kernel(const Prod p) {
  typedef Block<F16, GRAM, GRAM, WM, WN, FM, FN, 64, 2> B;
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
  const int nk = (p.r + B::BK - 1) / B::BK;
  const int first = sp * p.per_split, last = min(nk, first + p.per_split);
  Operand<uint16_t> oa, ob;
  oa.p[0] = p.a.hi + g * p.a.stride;
  oa.p[1] = p.a.lo + g * p.a.stride;
  oa.ld = p.a.ld;
  oa.rows = p.m;
  ob.p[0] = p.b.hi + g * p.b.stride;
  ob.p[1] = p.b.lo + g * p.b.stride;
  ob.ld = p.b.ld;
  ob.rows = p.n;
  B blk;
  blk.clear();
  blk.run(lds, oa, ob, m0, n0, first * B::BK, min(p.r, last * B::BK));
  auto value = [&](int m, int n, f32x4 v) {
    if constexpr (E == POLY) {
      const f32x4 a = load_planes(p.add, g, m, n);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = p.cc * v[i] + p.cb * a[i];
        if (n + i == m) v[i] += p.ca;
      }
    } else if constexpr (E != PARTIAL) {
      v *= p.alpha;
    }
    if constexpr (E == PLANES || E == POLY)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i >= p.n) v[i] = 0.f;
    return v;
  };
  auto result = [&](int m, int n, f32x4 v) {
    if (m >= p.m || n >= p.n) return;
    v = value(m, n, v);
    if constexpr (E == PARTIAL)
      store4<F32>(p.partial + ((int64_t)sp * p.models + g) * p.m * p.n + (int64_t)m * p.n + n, v, p.n - n);
    else if constexpr (E == PLANES || E == POLY) store_planes(p.out, g, m, n, v);
    else write_result<K, E>(p, g, m, n, v);
  };
  if ((E == OUT || E == STEP) && p.transposed) blk.each(m0, n0, result);
  else blk.each_row(lds, m0, n0, result);
  if constexpr (E == PLANES || E == POLY)
    if (p.symmetric && tm != tn)
      blk.each(m0, n0, [&](int m, int n, f32x4 v) {
        if (m < p.m && n < p.n) store_planes_mirrored(p.out, g, m, n, p.n, value(m, n, v));
      });
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
  for (int i = threadIdx.x >> 4; i < 64; i += 16) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    const int m = m0 + i, n = n0 + q;
    if (m < p.m && n < p.n) {
      const float* at = src + (int64_t)m * p.n + n;
      v = load4<F32>(at, p.n - n);
      for (int s = 1; s < p.splits; ++s) v += load4<F32>(at + s * step, p.n - n);
      v *= p.alpha;
      store_planes(p.out, g, m, n, v);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) tile[q + e][i] = v[e];
  }
  if (tm == tn) return;
  __syncthreads();
  for (int i = threadIdx.x >> 4; i < 64; i += 16) {
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = tile[i][q + e];
    if (n0 + i < p.n && m0 + q < p.m) store_planes(p.out, g, n0 + i, m0 + q, v);
  }
}

// ------------------------------------------------------------------------------------------ matrices that fit in LDS
// One workgroup does everything for one model: U (and the momentum) is read once, X stays in LDS in fp32, and so do the
// k x k matrices; all products on v_mfma_f32_16x16x4.  Such a matrix needs 10 MFLOP or less, so what counts is that one
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
  for (Walk w(tid, 256, n4); w.r < s.rows; w.next()) {
    const int c = w.c4 * 4;
    const f32x4 v = update4<K, true>(s, g, w.r, c, s.cols - c);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (c + e < s.cols) {
        X[p.tall ? w.r * S + c + e : (c + e) * S + w.r] = v[e];
        sum += (double)v[e] * (double)v[e];
      }
  }
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
      const f32x4 old = load4<F32>(at, s.cols - c);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = p.keep * old[e] - p.step * v[e];
      store4<F32>(at, v, s.cols - c);
    } else {
      store4<K>(at, v, s.cols - c);
    }
  }
}

// ------------------------------------------------------------------------------------------ host
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
size_t align16(size_t v) { return (v + 15) & ~(size_t)15; }

// Multiply-adds per cycle and CU of split products (measured on large ones)
constexpr TileShape SHAPES[3] = {{256, 256, 1, 280.f}, {128, 128, 2, 205.f}, {64, 64, 3, 120.f}};

// LDS of small_kernel, 0 where the matrix does not fit
size_t small_bytes(int L, int k) {
  if (k > 64) return 0;
  const int kt = (k + 15) / 16, s = 16 * kt + 4;
  const int64_t bytes = ((int64_t)((L + 15) & ~15) * s + 16 * kt * s + small_scratch(kt)) * 4;
  return bytes <= 160 * 1024 - 256 ? (size_t)bytes : 0;
}

struct Space {
  int k, L, ld, phases, chunks;
  size_t small;
  Choice gram;
  size_t sums, x, square, partial, total;  // bytes of one of each
  int n_x;
};

Choice shape_for(int64_t models, int64_t m, int64_t n, int64_t r, bool symmetric, bool can_split) {
  Choice best = {};
  double least = 0;
  for (int s = 0; s < 3; ++s) {  // choose() per shape, its tiles halved where the result is symmetric
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
  s.k = t.rows < t.cols ? t.rows : t.cols;
  s.L = t.rows < t.cols ? t.cols : t.rows;
  s.ld = (s.k + 7) & ~7;
  s.phases = 2 * (int64_t)s.L >= 3 * (int64_t)s.k ? (t.steps + 2) / 3 : t.steps;
  s.small = small_bytes(s.L, s.k);
  if (s.small) {  // reading X again costs nothing here: phases of two steps lose less to the Gram matrix's error
    s.phases = (t.steps + 1) / 2;
    return true;
  }
  s.n_x = s.phases > 1 ? 2 : 1;
  const int64_t groups = (int64_t)t.rows * ceil_div(t.cols, 4);
  if (groups > (int64_t)1 << 30) return false;
  const int64_t most = t.n_models >= 16 ? 64 : NORM_CHUNKS;
  s.chunks = (int)(ceil_div(groups, 1024) < most ? ceil_div(groups, 1024) : most);
  s.gram = shape_for(t.n_models, s.k, s.k, s.L, true, true);
  const size_t G = (size_t)t.n_models;
  s.sums = align16(G * s.chunks * sizeof(double));
  s.x = align16(G * s.L * s.ld * 2) * 2;       // both planes
  s.square = align16(G * s.k * s.ld * 2) * 2;
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
  if (c.tile == 0) product_kernel<K, GRAM, E, 2, 4, 4, 2><<<grid, 512, 0, s>>>(p);
  else if (c.tile == 1) product_kernel<K, GRAM, E, 2, 2, 2, 2><<<grid, 256, 0, s>>>(p);
  else product_kernel<K, GRAM, E, 2, 2, 1, 1><<<grid, 256, 0, s>>>(p);
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

template <Kind K, Epi LAST> int run(const mplc_muon_t& t, const Space& sp, const Source& src, hipStream_t s) {
  if (sp.small) return run_small<K, LAST>(t, sp, src, s);
  char* ws = reinterpret_cast<char*>(t.workspace);
  double* sums = reinterpret_cast<double*>(ws);
  ws += sp.sums;
  auto planes = [&](size_t bytes, int64_t stride) {
    Planes p = {reinterpret_cast<uint16_t*>(ws), reinterpret_cast<uint16_t*>(ws + bytes / 2), stride, sp.ld};
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
  const Choice small = shape_for(t.n_models, sp.k, sp.k, sp.k, true, false);
  const Choice apply = shape_for(t.n_models, sp.L, sp.k, sp.k, false, false);
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
