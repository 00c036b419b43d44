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
constexpr int NORM_CHUNKS = 64;

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

// U at (r, c); FIRST: the pass that updates the momentum
template <Kind K, bool FIRST> __device__ __forceinline__ float update_at(const Source& s, int g, int r, int c) {
  typedef typename Elem<K>::T T;
  const float v = to_f32<K>(reinterpret_cast<const T*>(s.g)[g * s.g_stride + r * s.g_ld + c]);
  if (s.m == nullptr) return v;
  float* pm = s.m + g * s.m_stride + r * s.m_ld + c;
  float m = *pm;
  if (FIRST) {
    m = s.beta * m + v;
    *pm = m;
  }
  return s.nesterov ? s.beta * m + v : m;
}

// |U|^2 in 64 bits (neither 1e-30 nor 1e30 leaves the range), NORM_CHUNKS partial sums per model
template <Kind K> __global__ __launch_bounds__(256) void norm_kernel(const Source s, double* sums) {
  __shared__ double part[4];
  const int g = blockIdx.y;
  const int64_t n = (int64_t)s.rows * s.cols;
  double sum = 0.;
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < n; t += (int64_t)gridDim.x * 256) {
    const int r = (int)(t / s.cols), c = (int)(t - (int64_t)r * s.cols);
    const double v = update_at<K, true>(s, g, r, c);
    sum += v * v;
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) sum += __shfl_down(sum, d, 64);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) sums[(int64_t)g * gridDim.x + blockIdx.x] = (part[0] + part[1]) + (part[2] + part[3]);
}

// X_SCALE / |U|; 0 for U = 0, NaN where U is not finite
__device__ __forceinline__ double inverse_norm(const double* sums, int g, int chunks) {
  double sum = 0.;
  for (int i = 0; i < chunks; ++i) sum += sums[(int64_t)g * chunks + i];
  if (sum == 0.) return 0.;
  if (!(sum < (double)INFINITY)) return (double)NAN;
  return (double)X_SCALE / sqrt(sum);
}

// X_0 as planes [L][ld], its columns behind k zero.  TALL: rows = L.  32 x 32 tiles, transposed through LDS where not.
template <Kind K, bool TALL>
__global__ __launch_bounds__(256) void start_kernel(const Source s, const double* sums, int chunks, const Planes x) {
  __shared__ float tile[32][33];
  const int g = blockIdx.z;
  const double inv = inverse_norm(sums, g, chunks);
  const int L = TALL ? s.rows : s.cols, k = TALL ? s.cols : s.rows;
  const int l0 = blockIdx.x * 32, k0 = blockIdx.y * 32;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  for (int i = ty; i < 32; i += 8) {
    const int r = TALL ? l0 + i : k0 + i, c = TALL ? k0 + tx : l0 + tx;
    float v = 0.f;
    if (r < s.rows && c < s.cols) v = (float)((double)update_at<K, false>(s, g, r, c) * inv);
    if (TALL) tile[i][tx] = v;
    else tile[tx][i] = v;
  }
  __syncthreads();
  const int row = threadIdx.x >> 3, col = (threadIdx.x & 7) * 4;
  if (l0 + row < L && k0 + col < x.ld) {
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = k0 + col + e < k ? tile[row][col + e] : 0.f;
    store_planes(x, g, l0 + row, k0 + col, v);
  }
}

// ------------------------------------------------------------------------------------------ products
enum Epi { PLANES, POLY, PARTIAL, OUT, STEP };

struct Prod {
  Planes a, b;
  int m, n, r, models, tiles_m, tiles_n, splits, per_split;
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

// GRAM: both operands are X and the sum runs over its rows
template <Kind K, bool GRAM, Epi E, int W, int F>
__global__ __launch_bounds__(64 * W * W) void product_kernel(const Prod p) {
  typedef Block<F16, GRAM, GRAM, W, W, F, F, 64, 2> B;
  __shared__ __attribute__((aligned(16))) char lds[B::LDS_BYTES];
  int64_t b = xcd_block();
  const int tn = (int)(b % p.tiles_n);
  b /= p.tiles_n;
  const int tm = (int)(b % p.tiles_m);
  b /= p.tiles_m;
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
  auto result = [&](int m, int n, f32x4 v) {
    if (m >= p.m || n >= p.n) return;
    if constexpr (E == PARTIAL) {
      store4<F32>(p.partial + ((int64_t)sp * p.models + g) * p.m * p.n + (int64_t)m * p.n + n, v, p.n - n);
    } else if constexpr (E == PLANES) {
      v *= p.alpha;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i >= p.n) v[i] = 0.f;
      store_planes(p.out, g, m, n, v);
    } else if constexpr (E == POLY) {
      const f32x4 a = load_planes(p.add, g, m, n);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = p.cc * v[i] + p.cb * a[i];
        if (n + i == m) v[i] += p.ca;
        if (n + i >= p.n) v[i] = 0.f;
      }
      store_planes(p.out, g, m, n, v);
    } else {
      v *= p.alpha;
      write_result<K, E>(p, g, m, n, v);
    }
  };
  if ((E == OUT || E == STEP) && p.transposed) blk.each(m0, n0, result);
  else blk.each_row(lds, m0, n0, result);
}

// the Gram matrix from its partial sums, added in order
__global__ __launch_bounds__(256) void join_kernel(const Prod p) {
  const int n4 = p.out.ld >> 2;
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (t >= (int64_t)p.m * n4) return;
  const int g = blockIdx.y, m = (int)(t / n4), n = (int)(t % n4) * 4;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (n < p.n) {
    const float* src = p.partial + (int64_t)g * p.m * p.n + (int64_t)m * p.n + n;
    const int64_t step = (int64_t)p.models * p.m * p.n;
    v = load4<F32>(src, p.n - n);
    for (int s = 1; s < p.splits; ++s) v += load4<F32>(src + s * step, p.n - n);
    v *= p.alpha;
  }
  store_planes(p.out, g, m, n, v);
}

// ------------------------------------------------------------------------------------------ host
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
size_t align16(size_t v) { return (v + 15) & ~(size_t)15; }

struct Space {
  int k, L, ld, phases, gram_splits, gram_per_split, chunks;
  size_t sums, x, square, partial, total;  // bytes of one of each
  int n_x;
};

bool wide_tile(int64_t tiles128) { return tiles128 >= 64; }

bool space(const mplc_muon_t& t, Space& s) {
  if (t.n_models < 0 || t.n_models > 65535 || t.rows < 1 || t.cols < 1 || t.dtype < 0 || t.dtype > 2) return false;
  if (t.steps < 1 || t.steps > 16) return false;
  s = Space{};
  s.k = t.rows < t.cols ? t.rows : t.cols;
  s.L = t.rows < t.cols ? t.cols : t.rows;
  s.ld = (s.k + 7) & ~7;
  s.phases = 2 * (int64_t)s.L >= 3 * (int64_t)s.k ? (t.steps + 2) / 3 : t.steps;
  s.n_x = s.phases > 1 ? 2 : 1;
  const int64_t elems = (int64_t)t.rows * t.cols;
  s.chunks = (int)(ceil_div(elems, 4096) < NORM_CHUNKS ? ceil_div(elems, 4096) : NORM_CHUNKS);
  const int64_t t64 = ceil_div(s.k, 64), t128 = ceil_div(s.k, 128);
  const int64_t tiles = (s.k <= 64 ? t64 * t64 : t128 * t128) * t.n_models;
  const int64_t nk = ceil_div(s.L, 32);
  int64_t splits = 1;
  if (tiles < 512 && tiles > 0) {  // two workgroups per CU, at least 8 tiles of r each
    splits = ceil_div(512, tiles);
    if (splits > nk / 8) splits = nk / 8;
    if (splits > 64) splits = 64;
    if (splits < 1) splits = 1;
  }
  s.gram_per_split = (int)ceil_div(nk, splits);
  s.gram_splits = (int)ceil_div(nk, s.gram_per_split);
  const size_t G = (size_t)t.n_models;
  s.sums = align16(G * s.chunks * sizeof(double));
  s.x = align16(G * s.L * s.ld * 2) * 2;       // both planes
  s.square = align16(G * s.k * s.ld * 2) * 2;
  s.partial = s.gram_splits > 1 ? align16(G * s.gram_splits * (size_t)s.k * s.k * sizeof(float)) : 0;
  s.total = s.sums + s.n_x * s.x + 6 * s.square + s.partial;
  const int64_t most = ceil_div(s.L, 64) * ceil_div(s.k, 64) * (int64_t)t.n_models;
  return most <= (1 << 23) && tiles * s.gram_splits <= (1 << 23) && ceil_div(s.k, 32) <= 65535;
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

template <Kind K, bool GRAM, Epi E> hipError_t product(Prod p, hipStream_t s) {
  const int64_t big = ceil_div(p.m, 128) * ceil_div(p.n, 128) * p.models;
  const bool wide = GRAM ? p.m > 64 : (p.n > 64 && wide_tile(big));
  const int b = wide ? 128 : 64;
  p.tiles_m = (int)ceil_div(p.m, b);
  p.tiles_n = (int)ceil_div(p.n, b);
  if (!GRAM) {
    p.splits = 1;
    p.per_split = (int)ceil_div(p.r, 32);
  }
  const dim3 grid((unsigned)((int64_t)p.tiles_m * p.tiles_n * p.splits * p.models));
  if (wide) product_kernel<K, GRAM, E, 2, 2><<<grid, 256, 0, s>>>(p);
  else product_kernel<K, GRAM, E, 2, 1><<<grid, 256, 0, s>>>(p);
  return hipGetLastError();
}

template <Kind K, Epi LAST> int run(const mplc_muon_t& t, const Space& sp, const Source& src, hipStream_t s) {
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
  const dim3 sg((unsigned)ceil_div(sp.L, 32), (unsigned)ceil_div(sp.k, 32), (unsigned)t.n_models);
  if (tall) start_kernel<K, true><<<sg, 256, 0, s>>>(src, sums, sp.chunks, X[0]);
  else start_kernel<K, false><<<sg, 256, 0, s>>>(src, sums, sp.chunks, X[0]);
  if ((err = hipGetLastError()) != hipSuccess) return (int)err;

  Prod base = {};
  base.models = t.n_models;
  base.splits = 1;
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
    p.splits = sp.gram_splits;
    p.per_split = sp.gram_per_split;
    p.alpha = A_SCALE / (X_SCALE * X_SCALE);
    p.out = A;
    p.partial = partial;
    if (p.splits > 1) {
      if ((err = product<K, true, PARTIAL>(p, s)) != hipSuccess) return (int)err;
      join_kernel<<<dim3((unsigned)ceil_div((int64_t)sp.k * (sp.ld / 4), 256), (unsigned)t.n_models), 256, 0, s>>>(p);
      if ((err = hipGetLastError()) != hipSuccess) return (int)err;
    } else if ((err = product<K, true, PLANES>(p, s)) != hipSuccess) {
      return (int)err;
    }
    auto square = [&](const Planes& l, float ls, const Planes& m, float ms, const Planes& o, float os) {
      Prod q = base;
      q.a = l;
      q.b = m;
      q.m = q.n = q.r = sp.k;
      q.alpha = os / (ls * ms);
      q.out = o;
      return product<K, false, PLANES>(q, s);
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
      q.out = i == 0 ? Q : P;
      if ((err = product<K, false, POLY>(q, s)) != hipSuccess) return (int)err;
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
      err = product<K, false, PLANES>(p, s);
      x = 1 - x;
    } else {
      p.alpha = 1.f / (X_SCALE * q_scale);
      p.transposed = !tall;
      if (LAST == OUT) {
        p.dst = t.out;
        p.dst_stride = t.out_stride;
        p.dst_ld = t.out_ld;
        err = product<K, false, OUT>(p, s);
      } else {
        p.dst = t.w;
        p.dst_stride = t.w_stride;
        p.dst_ld = t.w_ld;
        p.keep = (float)(1. - (double)t.lr * t.weight_decay);
        p.step = t.lr * t.scale;
        err = product<F32, false, STEP>(p, s);
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
  if (t->workspace == nullptr || t->workspace_bytes < sp.total) return MPLC_E_WORKSPACE;
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
