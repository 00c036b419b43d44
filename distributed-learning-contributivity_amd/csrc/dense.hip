// Dense layer batched over models (gfx950): y[g] = act(x[g] w[g] + b[g]) + r[g] and its gradients, any size, fp32 / bf16 /
// fp16, ragged row counts, one input shared by all models.  include/mplc_hip_ops.h states the operator.
//
// All three products run on the tiled core of mma.h without a copy or a transposition of an operand:
//   forward  y  [row][out] = sum over in  of x[row][in]  w[in][out]    A along r, B across r
//   dx          [row][in]  = sum over out of dz[row][out] w[in][out]   A along r, B along r
//   dw          [in][out]  = sum over row of x[row][in]  dz[row][out]  A across r, B across r
// A shared input's dx sums over the models inside the same product: r runs over (model, out).
//
// Few tiles and a long sum (a training batch's rows against 9216 inputs): r is split over workgroups, the fp32 partial
// sums go through the workspace and a second kernel adds them in order and applies the epilogue.
//
// act'(z) needs dz as an operand of two products: one pass computes it, rounds it to the operands' type and sums its
// columns (db) on the way, in fp32, per 64 rows, the blocks of rows added in order.  The rounding is a choice: a 16-bit matrix
// instruction takes 16-bit operands, and a second plane for the rest of dz would double both products (8192 x 4096 x 4096 bf16:
// 520 us more beside 990).  It raises the error of 16-bit dx and dw from that of their own rounding alone, 1.7e-3 in bf16 and
// 2.1e-4 in fp16, to 2.3e-3 and 2.9e-4 (Frobenius norm); z stays fp32, as its rounding would enter dz through act' as well.
#include <math.h>

#include "mma.h"
#include "mplc_hip.h"
#include "xcd.h"

namespace {

using namespace mma;

struct Epilogue {
  const void* bias;
  int64_t bias_stride;
  const void* res;
  int64_t res_stride, res_ld;
  void* out;
  int64_t out_stride, out_ld;
  float* z;
  int64_t z_stride, z_ld;
  int act;
};

struct Product {
  const void* a;
  int64_t a_stride, a_ld;
  const void* b;
  int64_t b_stride, b_ld;
  int m, n, r;           // sizes of one model's product
  int models, segments;
  int joined;            // one product, r runs over (segments, r): counts limit a segment's rows, every row is written
  const int32_t* counts;
  int count_is_r;        // counts limit r (dw), not m
  int tiles_m, tiles_n, nk, splits, per_split;  // nk: units of r; per_split: units of a split
  int aligned;           // 16-byte rows: tiles go straight into LDS
  int b_cols;            // across r: columns of B that may be read (n, or its padding too)
  float* partial;        // [split][model][m][n] where splits > 1
};

__device__ __forceinline__ int count_of(const int32_t* counts, int g, int most) {
  if (counts == nullptr) return most;
  const int c = counts[g];
  return c < 0 ? 0 : (c > most ? most : c);
}

// Standard normal: the probability of values below z and its density.  The tail below -|z| is exp(-z^2 / 2) t (c0 + c1 t + ..
// + c8 t^8) with t = 1 / (1 + 0.28 |z|): the coefficients were fitted here to the least relative error over |z| <= 64
// (9.1e-8), so that gelu keeps its digits far in the negative tail, where an error that is small beside 1 alone would be larger
// than the result.  In fp32 the square and its product with log2(e) / 2 are carried in two parts, as their rounding would be
// multiplied by z^2: relative error of the tail 4.2e-7, and 7.5e-6 without (enough for 16-bit results).
template <Kind K> __device__ __forceinline__ float normal(float z, float& density) {
  const float a = fminf(fabsf(z), 64.f), s = a * a;
  float e;
  if constexpr (K == F32) {
    constexpr double L = 0.72134752044448170;
    const float h = s * (float)L;
    const float l = __builtin_fmaf(__builtin_fmaf(a, a, -s), (float)L, __builtin_fmaf(s, (float)(L - (float)L), __builtin_fmaf(s, (float)L, -h)));
    e = __builtin_amdgcn_exp2f(-h);
    e = __builtin_fmaf(e, l * -0.69314718056f, e);
  } else {
    e = __expf(-0.5f * s);
  }
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.28f, a, 1.f));
  constexpr float c[9] = {0.11170406639575958f, 0.11169082671403885f, 0.10321412980556488f, 0.08275685459375381f, 0.07594385743141174f,
                          -0.012980633415281773f, 0.10007699579000473f, -0.09832608699798584f, 0.02592002972960472f};
  float q = c[8];
#pragma unroll
  for (int i = 7; i >= 0; --i) q = __builtin_fmaf(q, t, c[i]);
  const float tail = e * t * q;
  density = 0.39894228040143268f * e;
  return z < 0.f ? tail : 1.f - tail;
}

// far in the negative tail the result is 0, at -infinity too
template <Kind K> __device__ __forceinline__ float activate(int act, float z) {
  switch (act) {
    case MPLC_ACT_RELU: return z < 0.f ? 0.f : z;
    case MPLC_ACT_GELU: {
      float density;
      const float p = normal<K>(z, density);
      return z < -64.f ? 0.f : z * p;
    }
    case MPLC_ACT_SILU: return z < -1e4f ? 0.f : z / (1.f + __expf(-z));
    default: return z;
  }
}
template <Kind K> __device__ __forceinline__ float slope(int act, float z) {
  switch (act) {
    case MPLC_ACT_RELU: return z > 0.f ? 1.f : 0.f;
    case MPLC_ACT_GELU: {
      if (fabsf(z) > 64.f) return z > 0.f ? 1.f : 0.f;
      float density;
      const float p = normal<K>(z, density);
      return p + z * density;
    }
    case MPLC_ACT_SILU: {
      if (fabsf(z) > 1e4f) return z > 0.f ? 1.f : 0.f;
      const float s = 1.f / (1.f + __expf(-z));
      return s * (1.f + z * (1.f - s));
    }
    default: return 1.f;
  }
}

template <Kind K, bool WIDE> __device__ __forceinline__ f32x4 residual_at(const Epilogue& e, int g, int m, int n, int N) {
  typedef typename Elem<K>::T T;
  return e.res ? load4<K, WIDE>(reinterpret_cast<const T*>(e.res) + g * e.res_stride + m * e.res_ld + n, N - n)
               : f32x4{0.f, 0.f, 0.f, 0.f};
}
template <Kind K, bool WIDE> __device__ __forceinline__ f32x4 bias_at(const Epilogue& e, int g, int n, int N) {
  typedef typename Elem<K>::T T;
  return e.bias ? load4<K, WIDE>(reinterpret_cast<const T*>(e.bias) + g * e.bias_stride + n, N - n) : f32x4{0.f, 0.f, 0.f, 0.f};
}
// x w of 4 columns n .. of row m of model g -> z, y
template <Kind K>
__device__ __forceinline__ void finish(const Epilogue& e, int g, int m, int n, int N, f32x4 v, f32x4 bias, f32x4 res) {
  typedef typename Elem<K>::T T;
  const int valid = N - n;
  if (e.bias) v += bias;
  if (e.z) store4<F32>(e.z + g * e.z_stride + m * e.z_ld + n, v, valid);
  if (e.act != MPLC_ACT_NONE)
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = activate<K>(e.act, v[i]);
  if (e.res) v += res;
  store4<K>(reinterpret_cast<T*>(e.out) + g * e.out_stride + m * e.out_ld + n, v, valid);
}

// Tile order of one product: 8 tile rows at a time, column by column, so that the workgroups in flight on an XCD share
// their rows of A and columns of B in its L2.
__device__ __forceinline__ void tile_of(int idx, int tm, int tn, int& m, int& n) {
  const int band = idx / (8 * tn), first = band * 8;
  const int size = tm - first < 8 ? tm - first : 8;
  const int in = idx - band * 8 * tn;
  m = first + in % size;
  n = in / size;
}

constexpr int unit_of(Kind k) { return k == F32 ? 32 : 64; }  // what a split takes whole numbers of

// One tile of a product, or of a split of its sum.  Bound by the matrix cores where there are tiles for all CUs.  8192 x 4096 x
// 4096 bf16 on 256 x 256 tiles, products alone: 285 / 260 / 263 us (forward / dx / dw), 960 to 1060 TFLOP/s.  In a training
// step with gelu, residual and z: 371 / 266 / 283 us, 740 / 1035 / 970 TFLOP/s - with one workgroup per CU nothing hides the
// forward's epilogue.  fp32 on 128 x 128: 130 TFLOP/s.
template <Kind K, bool AA, bool BA, int WM, int WN, int FM, int FN, int BKB, int STAGES>
__global__ __launch_bounds__(64 * WM * WN) void product_kernel(const Product p, const Epilogue e) {
  typedef typename Elem<K>::T T;
  typedef Block<K, AA, BA, WM, WN, FM, FN, BKB, 1, STAGES> B;
  __shared__ __attribute__((aligned(16))) char lds[B::LDS_BYTES];
  int64_t b = xcd_block();
  const int tiles = p.tiles_m * p.tiles_n;
  int tm, tn;
  tile_of((int)(b % tiles), p.tiles_m, p.tiles_n, tm, tn);
  b /= tiles;
  const int split = (int)(b % p.splits), g = (int)(b / p.splits);
  const int m0 = tm * B::BM, n0 = tn * B::BN;
  const bool seg = !AA && !BA && p.joined;  // dx
  const int cnt = seg ? p.m : count_of(p.counts, g, p.count_is_r ? p.r : p.m);
  const int M = p.count_is_r ? p.m : cnt, R = p.count_is_r ? cnt : p.r;
  if (m0 >= M) return;
  const int64_t first = (int64_t)split * p.per_split, last = first + p.per_split;  // units of r
  const T* pa = reinterpret_cast<const T*>(p.a) + g * p.a_stride;
  const T* pb = reinterpret_cast<const T*>(p.b) + g * p.b_stride;
  B blk;
  blk.clear();
  if (seg) {
    // unit u of (model, r) as a tile of (model, r)
    const int nk = (R + B::BK - 1) / B::BK;
    auto tile_at = [&](int64_t u) {
      const int64_t s = u / p.nk;
      return s >= p.segments ? (int64_t)p.segments * nk : s * nk + min(nk, (int)(u - s * p.nk) * (unit_of(K) / B::BK));
    };
    const int64_t from = tile_at(first), to = tile_at(last);
    auto at = [&](int s, Operand<T>& a, Operand<T>& o, int& r0) {
      a.p = pa + s * p.a_stride;
      o.p = pb + s * p.b_stride;
      a.ld = p.a_ld;
      o.ld = p.b_ld;
      a.rows = p.m;
      o.rows = p.n;
      r0 = 0;
    };
    if (p.aligned && p.counts == nullptr && R % B::BK == 0) {
      if (from < to) blk.ring(lds, m0, n0, nk, from, to, at);
    } else {
      auto piece = [&](int s, Operand<T>& a, Operand<T>& o, int& r0, int& rend) {
        at(s, a, o, r0);
        rend = R;
        return count_of(p.counts, s, p.m);
      };
      blk.through_registers(lds, m0, n0, nk, from, to, piece);
      // A zero in the place of a row behind a count, times an infinite or NaN weight, is NaN: once more, row by row.  (The
      // tiles of short sums would lose a workgroup per CU to its registers; with counts they are not taken.)
      if constexpr (BKB != 64)
        if (p.counts != nullptr && blk.not_finite(lds)) {
          blk.clear();
          blk.masked(lds, m0, n0, nk, from, to, piece);
        }
    }
  } else {
    const Operand<T> a = {pa, p.a_ld, M}, o = {pb, p.b_ld, BA ? p.b_cols : p.n};
    blk.run(lds, a, o, m0, n0, (int)min((int64_t)R, first * unit_of(K)), (int)min((int64_t)R, last * unit_of(K)), p.aligned);
  }
  if (p.splits > 1) {
    float* out = p.partial + ((int64_t)split * p.models + g) * p.m * p.n;
    blk.each_row(lds, m0, n0, [](int, int) { return 0; }, [&](int m, int n, f32x4 v, int) {
      if (m < M && n < p.n) store4<F32>(out + (int64_t)m * p.n + n, v, p.n - n);
    });
  } else {
    by_width(p.n, [&](auto wide) {
      constexpr bool W = decltype(wide)::value;
      const int nl = n0 + B::lane_column();
      const f32x4 bias = nl < p.n ? bias_at<K, W>(e, g, nl, p.n) : f32x4{0.f, 0.f, 0.f, 0.f};
      blk.each_row(
          lds, m0, n0,
          [&](int m, int n) { return m < M && n < p.n ? residual_at<K, W>(e, g, m, n, p.n) : f32x4{0.f, 0.f, 0.f, 0.f}; },
          [&](int m, int n, f32x4 v, f32x4 res) {
            if (m < M && n < p.n) finish<K>(e, g, m, n, p.n, v, bias, res);
          });
    });
  }
}

// Bound by the weights' stream: 8 x 1 row, 4096 -> 4097, 538 MB in 108 us, 5.0 TB/s from unaligned rows.
// Few rows (ROWS at most) of large fp32 weights that no 16-byte load takes whole: the weights stream through once and the
// product is a few multiply-adds per element, so there is nothing for the matrix cores to share.  A wave takes 256 columns, 4
// a lane, and every fourth group of 8 r; a row's x[r] is one value for the whole wave, from LDS.  Each lane keeps 8 loads of w
// on their way.
template <int ROWS> __global__ __launch_bounds__(256) void rows_kernel(const Product p, const Epilogue e) {
  constexpr Kind K = F32;
  constexpr int STEP = 512;  // r whose x is staged at a time
  __shared__ float xs[STEP][ROWS];
  __shared__ f32x4 part[4][ROWS][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t b = xcd_block();
  const int tn = (int)(b % p.tiles_n), split = (int)(b / p.tiles_n % p.splits), g = (int)(b / p.tiles_n / p.splits);
  const int M = count_of(p.counts, g, p.m);
  if (M == 0) return;
  const int c = (tn * 64 + lane) * 4, in = c < p.n ? c : (p.n - 1) & ~3;
  const int first = split * p.per_split * unit_of(K), last = min(p.r, first + p.per_split * unit_of(K));
  const float* x = reinterpret_cast<const float*>(p.a) + g * p.a_stride;
  const float* w = reinterpret_cast<const float*>(p.b) + g * p.b_stride + in;
  f32x4 acc[ROWS];
#pragma unroll
  for (int m = 0; m < ROWS; ++m) acc[m] = f32x4{0.f, 0.f, 0.f, 0.f};
  by_width(p.n, [&](auto wide) {
    for (int r0 = first; r0 < last; r0 += STEP) {
      const int n = min(STEP, last - r0);
      __syncthreads();
      for (int i = threadIdx.x; i < ROWS * STEP; i += 256) {
        const int m = i / STEP, r = i % STEP;
        xs[r][m] = m < M && r < n ? x[m * p.a_ld + r0 + r] : 0.f;
      }
      __syncthreads();
      for (int r = wave * 8; r < n; r += 32) {
        f32x4 v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)  // behind the last r: the last one again, not added
          v[i] = load4<K, decltype(wide)::value>(w + min(r0 + r + i, last - 1) * p.b_ld, p.n - in);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (r + i < n)
#pragma unroll
            for (int m = 0; m < ROWS; ++m) acc[m] += xs[r + i][m] * v[i];
        }
      }
    }
  });
#pragma unroll
  for (int m = 0; m < ROWS; ++m) part[wave][m][lane] = acc[m];
  __syncthreads();
  by_width(p.n, [&](auto wide) {
    constexpr bool W = decltype(wide)::value;
    for (int m = wave; m < ROWS; m += 4)
      if (m < M && c < p.n) {
        f32x4 v = part[0][m][lane] + part[1][m][lane];
        v += part[2][m][lane] + part[3][m][lane];
        if (p.splits > 1)
          store4<F32>(p.partial + (((int64_t)split * p.models + g) * p.m + m) * p.n + c, v, p.n - c);
        else
          finish<K>(e, g, m, c, p.n, v, bias_at<K, W>(e, g, c, p.n), residual_at<K, W>(e, g, m, c, p.n));
      }
  });
}

// adds the partial sums of one product in order and finishes it
template <Kind K> __global__ __launch_bounds__(256) void join_kernel(const Product p, const Epilogue e) {
  const int n4 = (p.n + 3) >> 2;
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (t >= (int64_t)p.m * n4) return;
  const int g = blockIdx.y, m = (int)(t / n4), n = (int)(t % n4) * 4;
  if (!p.count_is_r && !p.joined && m >= count_of(p.counts, g, p.m)) return;
  const float* src = p.partial + (int64_t)g * p.m * p.n + (int64_t)m * p.n + n;
  const int64_t step = (int64_t)p.models * p.m * p.n;
  by_width(p.n, [&](auto wide) {
    constexpr bool W = decltype(wide)::value;
    const f32x4 bias = bias_at<K, W>(e, g, n, p.n), res = residual_at<K, W>(e, g, m, n, p.n);
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < p.splits; s0 += 8) {  // 8 loads in flight; behind the last split the last again, not added
      f32x4 x[8];
#pragma unroll
      for (int s = 0; s < 8; ++s) x[s] = load4<F32, W>(src + (s0 + s < p.splits ? s0 + s : p.splits - 1) * step, p.n - n);
#pragma unroll
      for (int s = 0; s < 8; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += s0 + s < p.splits ? x[s][i] : 0.f;
    }
    finish<K>(e, g, m, n, p.n, v, bias, res);
  });
}

constexpr int DZ_ROWS = 64;  // rows summed by one workgroup

// dz = dy act'(z) and the sums of its columns over DZ_ROWS rows.  A wave takes LANES groups of 4 columns of 64 / LANES
// rows at a time (a narrow matrix would leave lanes idle), 4 such passes in flight.  Bound by HBM: 8192 x 4096 bf16,
// gelu, 268 MB in 61 us, 4.4 TB/s.
template <Kind K, int LANES>
__global__ __launch_bounds__(256) void dz_kernel(const void* dy_, int64_t dy_stride, int64_t dy_ld, const float* z,
                                                 int64_t z_stride, int64_t z_ld, int act, int rows, int n,
                                                 const int32_t* counts, void* dz_, int dz_ld, float* sums, void* db_,
                                                 int64_t db_stride) {
  typedef typename Elem<K>::T T;
  constexpr int STEP = 4 * (64 / LANES);  // rows of a pass of the workgroup
  __shared__ f32x4 part[4][LANES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int g = blockIdx.z, c = (blockIdx.y * LANES + lane % LANES) * 4;
  const int cnt = count_of(counts, g, rows);
  const int r0 = blockIdx.x * DZ_ROWS, r1 = min(cnt, r0 + DZ_ROWS);
  const T* dy = reinterpret_cast<const T*>(dy_) + g * dy_stride;
  T* dz = dz_ ? reinterpret_cast<T*>(dz_) + (int64_t)g * rows * dz_ld : nullptr;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  if (c < n)
    by_width(n, [&](auto wide) {
      constexpr bool W = decltype(wide)::value;
      for (int r = r0 + wave * (64 / LANES) + lane / LANES; r < r1; r += 4 * STEP) {
        f32x4 d[4], zz[4];
        // rows behind the last one are the last one again, and not counted
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i] = load4<K, W>(dy + min(r + STEP * i, r1 - 1) * dy_ld + c, n - c);
        if (act != MPLC_ACT_NONE)
#pragma unroll
          for (int i = 0; i < 4; ++i) zz[i] = load4<F32, W>(z + g * z_stride + min(r + STEP * i, r1 - 1) * z_ld + c, n - c);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (r + STEP * i < r1) {
            if (act != MPLC_ACT_NONE) {
#pragma unroll
              for (int e = 0; e < 4; ++e) d[i][e] *= slope<K>(act, zz[i][e]);
              if (dz) store4<K>(dz + (int64_t)(r + STEP * i) * dz_ld + c, d[i], n - c);
            }
            sum += d[i];
          }
      }
    });
  if (sums == nullptr && db_ == nullptr) return;
#pragma unroll
  for (int d = 32; d >= LANES; d >>= 1)
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] += __shfl_xor(sum[e], d, 64);
  if (lane < LANES) part[wave][lane] = sum;
  __syncthreads();
  if (wave == 0 && lane < LANES && c < n) {
    f32x4 v = part[0][lane] + part[1][lane];
    v += part[2][lane] + part[3][lane];
    if (sums) store4<F32>(sums + ((int64_t)g * gridDim.x + blockIdx.x) * n + c, v, n - c);
    else store4<K>(reinterpret_cast<T*>(db_) + g * db_stride + c, v, n - c);
  }
}

// db from the blocks' sums: 64 columns a workgroup, its waves take every fourth block
template <Kind K>
__global__ __launch_bounds__(256) void db_kernel(const float* sums, int blocks, int n, int rows, const int32_t* counts,
                                                 void* db_, int64_t db_stride) {
  typedef typename Elem<K>::T T;
  __shared__ float part[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int g = blockIdx.y, c = blockIdx.x * 64 + lane;
  const int nb = min(blocks, (count_of(counts, g, rows) + DZ_ROWS - 1) / DZ_ROWS);
  float v = 0.f;
  if (c < n)
    for (int i = wave; i < nb; i += 32) {
      float x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = i + 4 * k < nb ? sums[((int64_t)g * blocks + i + 4 * k) * n + c] : 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) v += x[k];
    }
  part[wave][lane] = v;
  __syncthreads();
  if (wave == 0 && c < n)
    reinterpret_cast<T*>(db_)[g * db_stride + c] = from_f32<K>((part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]));
}

// ---------------------------------------------------------------------------------------------- host
enum Form { FORWARD, DX, DW };

struct Plan {
  int cfg;  // place in SHAPES_16 / SHAPES_F32; 5: short sums; 6: few rows
  Product p;
  int64_t blocks;
  size_t partial_bytes;
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Multiply-adds per cycle and CU (measured on large products; 0: shape not built).  256 x 256 in fp32 would leave one
// wave per SIMD without gaining anything: the fp32 matrix rate is reached by 128 x 128.
constexpr TileShape SHAPES_16[5] = {{128, 128, 2, 640.f}, {64, 64, 3, 330.f}, {32, 128, 2, 280.f}, {256, 256, 1, 900.f},
                                    {64, 128, 3, 450.f}};
constexpr TileShape SHAPES_F32[5] = {{128, 128, 2, 115.f}, {64, 64, 4, 105.f}, {32, 128, 3, 95.f}, {256, 256, 1, 0.f},
                                     {64, 128, 3, 108.f}};

// Tile and split of one product.
bool plan(const mplc_dense_t& t, Form form, Plan& out) {
  Product p = {};
  const bool shared_dx = form == DX && t.x_shared;
  p.models = shared_dx ? 1 : t.n_models;
  p.segments = shared_dx ? t.n_models : 1;
  p.joined = shared_dx && (t.n_models > 1 || t.counts);  // a row behind one model's count gets 0 like any that none reaches
  p.m = form == DW ? t.in : t.rows;
  p.n = form == DX ? t.in : t.out;
  p.r = form == FORWARD ? t.in : form == DX ? t.out : t.rows;
  p.counts = t.counts;
  p.count_is_r = form == DW;
  const bool f32 = t.dtype == MPLC_DTYPE_F32;
  p.nk = (int)ceil_div(p.r, f32 ? unit_of(F32) : unit_of(BF16));
  const int64_t units = (int64_t)p.nk * p.segments;
  if (units > INT32_MAX) return false;
  const Choice c = choose(f32 ? SHAPES_F32 : SHAPES_16, 5, p.models, p.m, p.n, (int64_t)p.r * p.segments, units, true);
  out.cfg = c.tile;
  // A short sum is bound by its operands' latency and its result's stores: tiles of half the length leave LDS for three
  // workgroups per CU (45 x 9216 x 128 from 51 rows: fp32 106 us against 118, fp16 47 against 92).
  if ((c.tile == 0 || c.tile == 3) && p.nk <= 2 && !(p.joined && p.counts)) out.cfg = 5;
  p.splits = c.splits;
  p.per_split = c.per_split;
  // Few rows of large fp32 weights whose rows are no whole 16 bytes.  8 x 1 row, 4096 -> 4097: 108 us against 147 on the tiles, 64
  // x 2, 2304 -> 513: 39 against 68; 8 rows: 10 to 20 % faster.  Below 4 M weights the tiles' shorter start counts (1 x 1, 2304
  // -> 513: 8.4 against 9.5 us).  16-bit weights stream faster through the tiles, cut rows too (81 x 2, 3256 -> 653 fp16: 77
  // against 87 us, with 8 rows 77 against 137), and so do whole rows (8 x 1, 4096 -> 4096 fp32: 94 against 98).  Decided by
  // sizes alone, as the workspace is: where `out` is whole 16 bytes but the base or ld is not, the tiles take them.
  if (form == FORWARD && f32 && p.m <= 8 && p.n >= 128 && p.n % 4 != 0 && (int64_t)p.models * p.r * p.n >= 1 << 22) {
    // 256 columns a workgroup; r split until there are 4 workgroups per CU, at least 128 r each
    out.cfg = 6;
    p.tiles_m = 1;
    p.tiles_n = (int)ceil_div(p.n, 256);
    const int64_t blocks = (int64_t)p.tiles_n * p.models, least = 128 / unit_of(F32);
    int64_t splits = ceil_div(1024, blocks > 0 ? blocks : 1);
    if (splits > p.nk / least) splits = p.nk / least;
    if (splits < 1) splits = 1;
    p.per_split = (int)(p.nk > 0 ? ceil_div(p.nk, splits) : 1);
    p.splits = (int)(p.nk > 0 ? ceil_div(p.nk, p.per_split) : 1);
    if (blocks * p.splits > (1 << 23)) return false;
    out.blocks = blocks * p.splits;
    out.partial_bytes = p.splits > 1 ? (size_t)p.splits * p.models * p.m * p.n * sizeof(float) : 0;
    out.p = p;
    return true;
  }
  p.tiles_m = (int)(out.cfg == 5 ? ceil_div(p.m, 128) : c.tiles_m);
  p.tiles_n = (int)(out.cfg == 5 ? ceil_div(p.n, 128) : c.tiles_n);
  const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n * p.models;
  if (tiles * c.splits > (1 << 23)) return false;
  out.blocks = tiles * p.splits;
  out.partial_bytes = p.splits > 1 ? (size_t)p.splits * p.models * p.m * p.n * sizeof(float) : 0;
  out.p = p;
  return true;
}

template <Kind K, bool AA, bool BA> hipError_t launch(Plan& pl, const Epilogue& e, hipStream_t s) {
  const int ch = K == F32 ? 4 : 8;
  auto fits = [&](const void* base, int64_t stride, int64_t ld) {
    return ((uintptr_t)base & 15) == 0 && stride % ch == 0 && ld % ch == 0;
  };
  pl.p.aligned = fits(pl.p.a, pl.p.a_stride, pl.p.a_ld) && fits(pl.p.b, pl.p.b_stride, pl.p.b_ld) &&
                 (!AA || pl.p.m % ch == 0) && (!BA || pl.p.b_cols % ch == 0);
  const dim3 grid((unsigned)pl.blocks);
  if (pl.cfg == 6) {
    if constexpr (!AA && BA && K == F32) {  // the forward product
      if (pl.p.m <= 1) rows_kernel<1><<<grid, 256, 0, s>>>(pl.p, e);
      else if (pl.p.m <= 2) rows_kernel<2><<<grid, 256, 0, s>>>(pl.p, e);
      else if (pl.p.m <= 4) rows_kernel<4><<<grid, 256, 0, s>>>(pl.p, e);
      else rows_kernel<8><<<grid, 256, 0, s>>>(pl.p, e);
    }
  } else if (pl.cfg == 0) product_kernel<K, AA, BA, 2, 2, 2, 2, 128, 2><<<grid, 256, 0, s>>>(pl.p, e);
  else if (pl.cfg == 1) product_kernel<K, AA, BA, 2, 2, 1, 1, 128, 3><<<grid, 256, 0, s>>>(pl.p, e);
  else if (pl.cfg == 4) product_kernel<K, AA, BA, 1, 4, 2, 1, 128, 2><<<grid, 256, 0, s>>>(pl.p, e);
  else if (pl.cfg == 3) {
    if constexpr (K != F32) product_kernel<K, AA, BA, 2, 4, 4, 2, 128, 2><<<grid, 512, 0, s>>>(pl.p, e);
  }
  else if (pl.cfg == 5) product_kernel<K, AA, BA, 2, 2, 2, 2, 64, 3><<<grid, 256, 0, s>>>(pl.p, e);
  else product_kernel<K, AA, BA, 1, 4, 1, 1, 128, 3><<<grid, 256, 0, s>>>(pl.p, e);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess || pl.p.splits == 1) return err;
  const dim3 jg((unsigned)ceil_div((int64_t)pl.p.m * ((pl.p.n + 3) / 4), 256), (unsigned)pl.p.models);
  join_kernel<K><<<jg, 256, 0, s>>>(pl.p, e);
  return hipGetLastError();
}

size_t align16(size_t v) { return (v + 15) & ~(size_t)15; }

bool sizes_ok(const mplc_dense_t& t) {
  if (t.n_models < 0 || t.rows < 0 || t.in < 1 || t.out < 1) return false;
  if (t.dtype < 0 || t.dtype > 2 || t.activation < 0 || t.activation > 3) return false;
  return t.n_models <= 65535;
}
// a tensor of [models][rows][cols]: rows may not overlap one another
bool view_ok(const void* p, int64_t ld, int cols) { return p != nullptr && ld >= cols; }

struct BackwardSpace {
  Plan dx, dw;
  size_t dz, sums, partial, total;
  int dz_ld, blocks;
};

bool backward_space(const mplc_dense_t& t, BackwardSpace& s) {
  s = BackwardSpace{};
  const size_t size = t.dtype == MPLC_DTYPE_F32 ? 4 : 2;
  s.dz_ld = (t.out + 7) & ~7;
  s.blocks = (int)ceil_div(t.rows, DZ_ROWS);
  if ((t.dx || t.dw) && t.activation != MPLC_ACT_NONE)
    s.dz = align16((size_t)t.n_models * t.rows * s.dz_ld * size);
  if (t.db && s.blocks > 1) s.sums = align16((size_t)t.n_models * s.blocks * t.out * sizeof(float));
  size_t partial = 0;
  if (t.dx) {
    if (!plan(t, DX, s.dx)) return false;
    partial = s.dx.partial_bytes;
  }
  if (t.dw) {
    if (!plan(t, DW, s.dw)) return false;
    partial = partial > s.dw.partial_bytes ? partial : s.dw.partial_bytes;
  }
  s.partial = align16(partial);  // dx's partial sums are joined before dw's are written: one place for both
  s.total = s.dz + s.sums + s.partial;
  return s.blocks <= (1 << 23) && ceil_div(t.out, 256) <= 65535;  // the grid of dz_kernel
}

template <Kind K> int forward(const mplc_dense_t& t, const Plan& pl0, hipStream_t s) {
  Plan pl = pl0;
  pl.p.a = t.x;
  pl.p.a_stride = t.x_shared ? 0 : t.x_stride;
  pl.p.a_ld = t.x_ld;
  pl.p.b = t.w;
  pl.p.b_stride = t.w_stride;
  pl.p.b_ld = t.w_ld;
  pl.p.b_cols = pl.p.n;
  pl.p.partial = reinterpret_cast<float*>(t.workspace);
  Epilogue e = {t.bias, t.bias_stride, t.residual, t.residual_stride, t.residual_ld, t.y, t.y_stride, t.y_ld,
                t.z, t.z_stride, t.z_ld, t.activation};
  return (int)launch<K, false, true>(pl, e, s);
}

template <Kind K> int backward(const mplc_dense_t& t, BackwardSpace& sp, hipStream_t s) {
  char* ws = reinterpret_cast<char*>(t.workspace);
  void* dz = sp.dz ? ws : nullptr;
  float* sums = sp.sums ? reinterpret_cast<float*>(ws + sp.dz) : nullptr;
  float* partial = reinterpret_cast<float*>(ws + sp.dz + sp.sums);
  hipError_t err;
  if (dz || t.db) {
    const int lanes = t.out > 128 ? 64 : t.out > 64 ? 32 : 16;
    const dim3 grid((unsigned)(sp.blocks ? sp.blocks : 1), (unsigned)ceil_div(t.out, 4 * lanes), (unsigned)t.n_models);
    auto go = [&](auto kernel) {
      kernel<<<grid, 256, 0, s>>>(t.dy, t.dy_stride, t.dy_ld, t.z, t.z_stride, t.z_ld, t.activation, t.rows, t.out,
                                  t.counts, dz, sp.dz_ld, sums, sums ? nullptr : t.db, t.db_stride);
    };
    if (lanes == 64) go(dz_kernel<K, 64>);
    else if (lanes == 32) go(dz_kernel<K, 32>);
    else go(dz_kernel<K, 16>);
    if ((err = hipGetLastError()) != hipSuccess) return (int)err;
    if (sums) {
      db_kernel<K><<<dim3((unsigned)ceil_div(t.out, 64), (unsigned)t.n_models), 256, 0, s>>>(
          sums, sp.blocks, t.out, t.rows, t.counts, t.db, t.db_stride);
      if ((err = hipGetLastError()) != hipSuccess) return (int)err;
    }
  }
  const void* d = dz ? dz : t.dy;
  const int64_t d_stride = dz ? (int64_t)t.rows * sp.dz_ld : t.dy_stride, d_ld = dz ? sp.dz_ld : t.dy_ld;
  if (t.dx && t.rows > 0) {
    Plan& pl = sp.dx;
    pl.p.a = d;
    pl.p.a_stride = d_stride;
    pl.p.a_ld = d_ld;
    pl.p.b = t.w;
    pl.p.b_stride = t.w_stride;
    pl.p.b_ld = t.w_ld;
    pl.p.partial = partial;
    Epilogue e = {};
    e.out = t.dx;
    e.out_stride = t.x_shared ? 0 : t.dx_stride;
    e.out_ld = t.dx_ld;
    if ((err = launch<K, false, false>(pl, e, s)) != hipSuccess) return (int)err;
  }
  if (t.dw) {
    Plan& pl = sp.dw;
    pl.p.a = t.x;
    pl.p.a_stride = t.x_shared ? 0 : t.x_stride;
    pl.p.a_ld = t.x_ld;
    pl.p.b_cols = dz ? sp.dz_ld : pl.p.n;
    pl.p.b = d;
    pl.p.b_stride = d_stride;
    pl.p.b_ld = d_ld;
    pl.p.partial = partial;
    Epilogue e = {};
    e.out = t.dw;
    e.out_stride = t.dw_stride;
    e.out_ld = t.dw_ld;
    if ((err = launch<K, true, true>(pl, e, s)) != hipSuccess) return (int)err;
  }
  return MPLC_OK;
}

}  // namespace

extern "C" size_t mplc_dense_forward_workspace_bytes(const mplc_dense_t* t) {
  Plan pl;
  if (t == nullptr || !sizes_ok(*t) || !plan(*t, FORWARD, pl)) return 0;
  return pl.partial_bytes;
}

extern "C" size_t mplc_dense_backward_workspace_bytes(const mplc_dense_t* t) {
  BackwardSpace s;
  if (t == nullptr || !sizes_ok(*t) || !backward_space(*t, s)) return 0;
  return s.total;
}

extern "C" int mplc_dense_forward(const mplc_dense_t* t, void* stream) {
  if (t == nullptr || !sizes_ok(*t)) return MPLC_E_ARG;
  if (t->n_models == 0 || t->rows == 0) return MPLC_OK;
  if (!view_ok(t->x, t->x_ld, t->in) || !view_ok(t->w, t->w_ld, t->out) || !view_ok(t->y, t->y_ld, t->out))
    return MPLC_E_ARG;
  if ((t->residual && t->residual_ld < t->out) || (t->z && t->z_ld < t->out)) return MPLC_E_ARG;
  Plan pl;
  if (!plan(*t, FORWARD, pl)) return MPLC_E_SHAPE;
  if (pl.partial_bytes && (t->workspace == nullptr || t->workspace_bytes < pl.partial_bytes)) return MPLC_E_WORKSPACE;
  if (((uintptr_t)t->workspace & 15) != 0) return MPLC_E_ARG;
  hipStream_t s = (hipStream_t)stream;
  if (t->dtype == MPLC_DTYPE_F32) return forward<F32>(*t, pl, s);
  if (t->dtype == MPLC_DTYPE_BF16) return forward<BF16>(*t, pl, s);
  return forward<F16>(*t, pl, s);
}

extern "C" int mplc_dense_backward(const mplc_dense_t* t, void* stream) {
  if (t == nullptr || !sizes_ok(*t)) return MPLC_E_ARG;
  if (t->n_models == 0) return t->x_shared && t->dx && t->rows > 0 ? MPLC_E_SHAPE : MPLC_OK;
  if (t->rows > 0) {
    if (!view_ok(t->dy, t->dy_ld, t->out)) return MPLC_E_ARG;
    if (t->activation != MPLC_ACT_NONE && !view_ok(t->z, t->z_ld, t->out)) return MPLC_E_ARG;
    if (t->dx && (!view_ok(t->w, t->w_ld, t->out) || t->dx_ld < t->in)) return MPLC_E_ARG;
    if (t->dw && !view_ok(t->x, t->x_ld, t->in)) return MPLC_E_ARG;
  }
  if (t->dw && t->dw_ld < t->out) return MPLC_E_ARG;
  BackwardSpace sp;
  if (!backward_space(*t, sp)) return MPLC_E_SHAPE;
  if (sp.total && (t->workspace == nullptr || t->workspace_bytes < sp.total)) return MPLC_E_WORKSPACE;
  if (((uintptr_t)t->workspace & 15) != 0) return MPLC_E_ARG;
  hipStream_t s = (hipStream_t)stream;
  if (t->dtype == MPLC_DTYPE_F32) return backward<F32>(*t, sp, s);
  if (t->dtype == MPLC_DTYPE_BF16) return backward<BF16>(*t, sp, s);
  return backward<F16>(*t, sp, s);
}

extern "C" int64_t mplc_ops_layout(int what) {
  return what == 0 ? (int64_t)sizeof(mplc_dense_t) : what == 1 ? (int64_t)sizeof(mplc_muon_t) : -1;
}
