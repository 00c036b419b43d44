// Tiled matrix products on the CDNA4 matrix cores, shared by the dense layer (dense.hip) and the orthogonalised update
// (muon.hip).
//
// D[m][n] = sum over r of A[m][r] B[n][r], with either operand stored "along r" (element (i, r) at i * ld + r) or
// "across r" (at r * ld + i); three element kinds: fp32 (v_mfma_f32_32x32x2), bf16 and fp16 (v_mfma_f32_32x32x16); all
// sums fp32.
//
// Split fp16 (PL = 2 planes): a value v is held as hi = fp16(v), lo = fp16(v - hi), 22 bits together, and a product
// takes three matrix instructions (hi hi, hi lo, lo hi; lo lo is below 2^-24 of the product).  Values must be scaled
// into fp16's range by the caller.  It reaches fp32's accuracy at a third of the fp16 rate, about twice the fp32 rate.
//
// One workgroup computes a BM x BN tile over tiles of r, BKB bytes of an operand "along r" long.  Where the operands'
// rows are 16-byte aligned their tiles go from memory into LDS directly (global_load_lds, no registers), in a ring of
// STAGES tiles, whose loads run ahead by STAGES - 1 tiles; one barrier per tile.  Other operands, and the last tile of an
// r that no tile divides, go through registers.
//
// LDS.  A tile is a sequence of 16-byte chunks, row by row; which chunk of a row is at which place is exchanged by row
// (XOR), so that the rows that one pass of a read touches fall on different banks: along r, the 16 rows of a
// ds_read_b128; across r, the 4 rows of a ds_read_b64_tr_b16 (which transposes 4 x 16 elements inside 16 lanes) or the
// two of an fp32 fragment's ds_read_b32.
//
// The matrix instruction is issued as B A^T, so that a lane ends up with 4 consecutive columns n of one row m (wide
// stores and wide reads of the residual) instead of 4 rows of one column.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace mma {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

enum Kind { F32 = 0, BF16 = 1, F16 = 2 };

template <Kind K> struct Elem { typedef uint16_t T; };
template <> struct Elem<F32> { typedef float T; };

__device__ __forceinline__ float bf16_to_f32(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
__device__ __forceinline__ uint16_t f32_to_bf16(float v) {
  union { __bf16 b; uint16_t u; } c;
  c.b = (__bf16)v;  // round to nearest even
  return c.u;
}
__device__ __forceinline__ float f16_to_f32(uint16_t v) {
  union { uint16_t u; _Float16 h; } c;
  c.u = v;
  return (float)c.h;
}
__device__ __forceinline__ uint16_t f32_to_f16(float v) {
  union { uint16_t u; _Float16 h; } c;
  c.h = (_Float16)v;
  return c.u;
}
template <Kind K> __device__ __forceinline__ float to_f32(typename Elem<K>::T v) {
  if constexpr (K == F32) return v;
  else if constexpr (K == BF16) return bf16_to_f32(v);
  else return f16_to_f32(v);
}
template <Kind K> __device__ __forceinline__ typename Elem<K>::T from_f32(float v) {
  if constexpr (K == F32) return v;
  else if constexpr (K == BF16) return f32_to_bf16(v);
  else return f32_to_f16(v);
}

// vectors at any element's place (gfx950 global memory takes unaligned loads; as one vector type each, which the
// compiler does not take apart)
typedef uint32_t u32x4a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2a2 __attribute__((ext_vector_type(2), aligned(2)));
typedef float f32x4a4 __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ u32x4 load16(const void* p) { return *reinterpret_cast<const u32x4a2*>(p); }

// `n` valid elements from p (n <= 0: none), the rest zero
template <Kind K> __device__ __forceinline__ u32x4 load16_edge(const typename Elem<K>::T* p, int n) {
  constexpr int CH = 16 / sizeof(typename Elem<K>::T);
  if (n >= CH) return load16(p);
  u32x4 r = {0, 0, 0, 0};
  if constexpr (K == F32) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < n) r[e] = __float_as_uint(p[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) r[e >> 1] |= (uint32_t)p[e] << (16 * (e & 1));
  }
  return r;
}

// a chunk's elements from place n on, at the front, zeros behind them
template <typename T> __device__ __forceinline__ u32x4 drop_front(u32x4 v, int n) {
  const int bits = n * (int)sizeof(T) * 8, d = bits & 63;
  uint64_t lo = v[0] | (uint64_t)v[1] << 32, hi = v[2] | (uint64_t)v[3] << 32;
  lo = bits & 64 ? hi : lo;
  hi = bits & 64 ? 0 : hi;
  lo = d ? lo >> d | hi << (64 - d) : lo;
  hi >>= d;
  return u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
}

// 4 consecutive elements starting at p, n >= 1 of them valid, the others 0, without a branch: the compiler waits for what
// each branch has loaded, one latency after the other.  WIDE: the row has 4 elements or more, and one load that ends at the
// row's end takes a cut group; otherwise the last element is read again in the place of those that are not there.
template <Kind K, bool WIDE> __device__ __forceinline__ f32x4 load4(const typename Elem<K>::T* p, int n) {
  f32x4 r;
  if constexpr (WIDE) {
    const int d = n >= 4 ? 0 : 4 - n;
    if constexpr (K == F32) {
      r = *reinterpret_cast<const f32x4a4*>(p - d);
    } else {
      const u32x2 t = *reinterpret_cast<const u32x2a2*>(p - d);
#pragma unroll
      for (int e = 0; e < 4; ++e) r[e] = to_f32<K>((uint16_t)(t[e >> 1] >> (16 * (e & 1))));
    }
    const bool two = d & 2, one = d & 1;
    r[0] = two ? r[2] : r[0];
    r[1] = two ? r[3] : r[1];
    r[2] = two ? 0.f : r[2];
    r[3] = two ? 0.f : r[3];
    r[0] = one ? r[1] : r[0];
    r[1] = one ? r[2] : r[1];
    r[2] = one ? r[3] : r[2];
    r[3] = one ? 0.f : r[3];
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      r[e] = to_f32<K>(p[e < n ? e : n - 1]);
      r[e] = e < n ? r[e] : 0.f;
    }
  }
  return r;
}
// f(true or false) for WIDE, chosen once
template <typename F> __device__ __forceinline__ void by_width(int columns, F f) {
  if (columns >= 4) f(std::true_type{});
  else f(std::false_type{});
}
template <Kind K> __device__ __forceinline__ void store4(typename Elem<K>::T* p, f32x4 v, int n) {
  if (n >= 4) {
    if constexpr (K == F32) {
      *reinterpret_cast<f32x4a4*>(p) = v;
    } else {
      u32x2 t;
      t[0] = (uint32_t)from_f32<K>(v[0]) | ((uint32_t)from_f32<K>(v[1]) << 16);
      t[1] = (uint32_t)from_f32<K>(v[2]) | ((uint32_t)from_f32<K>(v[3]) << 16);
      *reinterpret_cast<u32x2a2*>(p) = t;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (e < n) p[e] = from_f32<K>(v[e]);
  }
}

// fp32: instruction e of 4 takes r = e (lanes 0-31) and r = 4 + e (lanes 32-63) of the fragments' 8
template <Kind K> __device__ __forceinline__ void mfma(f32x16& d, const u32x4& a, const u32x4& b, int e) {
  if constexpr (K == F32) {
    d = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[e]), __uint_as_float(b[e]), d, 0, 0, 0);
  } else if constexpr (K == BF16) {
    d = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), d, 0, 0, 0);
  } else {
    d = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), d, 0, 0, 0);
  }
}

// One operand of the product as the kernel sees it.  Two planes lie in one row, in blocks of 32 elements of the one and
// then of the other.
template <typename T> struct Operand {
  const T* p;
  int64_t ld;
  int rows;        // valid i
};

// The tile of one operand: BT rows i by BK r.
template <Kind K, bool ACROSS, int BT, int BKB, int NT, int PL> struct Tile {
  typedef typename Elem<K>::T T;
  static constexpr int CH = 16 / sizeof(T);              // elements of a chunk
  static constexpr int BK = BKB / sizeof(T);             // r per tile
  static constexpr int RPC = ACROSS ? BT / CH : BK / CH; // chunks of a stored row
  static constexpr int ROWB = RPC * 16;
  static constexpr int CHUNKS = BT * BK / CH;
  static constexpr int PER = CHUNKS / NT;
  static constexpr int PLANE_BYTES = CHUNKS * 16;
  static constexpr int BYTES = PL * PLANE_BYTES;
  static_assert(CHUNKS % NT == 0, "whole chunks per thread");

  const T* ptr[PL][PER];
  int live[PER];  // ACROSS: valid elements of the chunk's columns

  // place of chunk ch of a row, and the chunk at a place
  __device__ __forceinline__ static int swz(int row, int ch) {
    if constexpr (!ACROSS) return BKB == 128 ? ch ^ ((row >> 1) & 7) : ch ^ ((row >> 2) & 3);
    else if constexpr (K == F32) return RPC >= 16 ? ch ^ (((row >> 2) & 1) << 3) : ch;
    else return RPC >= 16 ? ch ^ ((row & 3) << 2) : RPC == 8 ? ch ^ (((row >> 1) & 1) << 2) : ch;
  }
  __device__ __forceinline__ static void place(int j, int tid, int& row, int& ch) {
    const int c = tid + j * NT;
    row = c / RPC;
    ch = swz(row, c % RPC);
  }

  // Points at the tile of rows [i0, i0 + BT) and r = r0 ...  Rows behind o.rows (never stored) repeat the last one, so
  // that only the end of r needs checks; chunks of columns across r behind o.rows read the row's first ones, and a chunk
  // that o.rows cuts is read from where it ends at the row's end.
  __device__ __forceinline__ void seek(const Operand<T>& o, int i0, int r0, int tid) {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      int row, ch;
      place(j, tid, row, ch);
      int64_t off;
      if constexpr (ACROSS) {
        const int i = i0 + ch * CH;
        live[j] = o.rows - i;
        off = (int64_t)(r0 + row) * o.ld + (live[j] > 0 ? column(i) : 0) - (o.rows >= CH ? behind(j) : 0);
      } else {
        off = (int64_t)min(i0 + row, o.rows - 1) * o.ld + column(r0 + ch * CH);
      }
#pragma unroll
      for (int p = 0; p < PL; ++p) ptr[p][j] = o.p + off + 32 * p;
    }
  }
  // ACROSS: elements of the chunk that are not there
  __device__ __forceinline__ int behind(int j) const { return live[j] > 0 && live[j] < CH ? CH - live[j] : 0; }
  __device__ __forceinline__ void advance(int64_t ld) {
#pragma unroll
    for (int p = 0; p < PL; ++p)
#pragma unroll
      for (int j = 0; j < PER; ++j) ptr[p][j] += ACROSS ? BK * ld : BK * PL;
  }
  static_assert(PL == 1 || BK == 32, "a tile along r is a block of each plane");
  __device__ __forceinline__ static int column(int c) { return PL == 1 ? c : ((c >> 5) << 6) + (c & 31); }
  // the whole tile at ptr into LDS; counts as PL * PER loads of the wave
  __device__ __forceinline__ void fetch(char* lds, int tid) const {
    typedef __attribute__((address_space(3))) uint32_t lds_u32;
    typedef __attribute__((address_space(1))) const uint32_t glb_u32;
#pragma unroll
    for (int p = 0; p < PL; ++p)
#pragma unroll
      for (int j = 0; j < PER; ++j)
        __builtin_amdgcn_global_load_lds((glb_u32*)ptr[p][j], (lds_u32*)(lds + p * PLANE_BYTES + (j * NT + (tid & ~63)) * 16), 16, 0, 0);
  }
  // the tile at ptr, of which `left` r are valid (left >= BK: all); columns (ACROSS, uniform): WHOLE, no chunk of them is
  // cut; CUT, one may be; FEW, there are fewer than a chunk's; rows at or behind `rows` contribute nothing
  enum Columns { WHOLE, CUT, FEW };
  static __device__ __forceinline__ Columns columns(int i0, int rows) {
    return !ACROSS || i0 + BT <= rows || rows % CH == 0 ? WHOLE : rows >= CH ? CUT : FEW;
  }
  struct Regs {
    u32x4 v[PL][PER];
  };
  // ld, rend: of the operand; where the tile is cut, every load still is one of whole chunks that ends inside the operand,
  // without a branch (the compiler waits for what each branch has loaded, one latency after the other: forward of 24 x 128
  // rows, 1001 -> 1027 bf16, 28 us against 55 with cut chunks loaded by elements)
  __device__ __forceinline__ void load(Regs& reg, int left, Columns cols, int64_t ld, int rend, int i0, int rows, bool drop,
                                       int tid) const {
    if (left >= BK && cols != FEW) {
#pragma unroll
      for (int p = 0; p < PL; ++p)
#pragma unroll
        for (int j = 0; j < PER; ++j) reg.v[p][j] = load16(ptr[p][j]);
    } else if (ACROSS ? cols != FEW : rend >= CH) {
      // along r: a chunk that r's end cuts, or that lies behind it, is read from where it ends there; across r: rows
      // behind the end read the last one
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        int row, ch;
        place(j, tid, row, ch);
        const int64_t back = ACROSS ? (row < left ? 0 : (row - left + 1) * ld) : max(0, CH - (left - ch * CH));
#pragma unroll
        for (int p = 0; p < PL; ++p) reg.v[p][j] = load16(ptr[p][j] - back);
      }
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        int row, ch;
        place(j, tid, row, ch);
        const int n = left - ch * CH;
        const bool there = ACROSS ? row < left : n > 0;
#pragma unroll
        for (int p = 0; p < PL; ++p) {
          u32x4 v = reg.v[p][j];
          if constexpr (!ACROSS) v = drop_front<T>(v, n > 0 && n < CH ? CH - n : 0);
#pragma unroll
          for (int e = 0; e < 4; ++e) reg.v[p][j][e] = there ? v[e] : 0;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        int row, ch;
        place(j, tid, row, ch);
        const int n = ACROSS ? (row < left ? live[j] : 0) : left - ch * CH;
#pragma unroll
        for (int p = 0; p < PL; ++p) reg.v[p][j] = load16_edge<K>(ptr[p][j], n);
      }
    }
    if constexpr (ACROSS)
      if (cols == CUT)
#pragma unroll
        for (int j = 0; j < PER; ++j)
#pragma unroll
          for (int p = 0; p < PL; ++p) reg.v[p][j] = drop_front<T>(reg.v[p][j], behind(j));
    if constexpr (!ACROSS)
      if (drop)
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          int row, ch;
          place(j, tid, row, ch);
          if (i0 + row >= rows)
#pragma unroll
            for (int p = 0; p < PL; ++p) reg.v[p][j] = u32x4{0, 0, 0, 0};
        }
  }
  __device__ __forceinline__ void store(const Regs& reg, char* lds, int tid) const {
#pragma unroll
    for (int j = 0; j < PER; ++j)
#pragma unroll
      for (int p = 0; p < PL; ++p) *reinterpret_cast<u32x4*>(lds + p * PLANE_BYTES + (tid + j * NT) * 16) = reg.v[p][j];
  }
  // the fragment of rows [i, i + 32) for k-step ks (2 chunks of r)
  __device__ __forceinline__ static u32x4 frag(const char* lds, int plane, int i, int ks, int lane) {
    const char* base = lds + plane * PLANE_BYTES;
    if constexpr (!ACROSS) {
      const int row = i + (lane & 31);
      return *reinterpret_cast<const u32x4*>(base + row * ROWB + swz(row, 2 * ks + (lane >> 5)) * 16);
    } else if constexpr (K == F32) {
      const int r = (2 * ks + (lane >> 5)) * 4, col = i + (lane & 31);
      const float* f = reinterpret_cast<const float*>(base + r * ROWB + swz(r, col >> 2) * 16) + (col & 3);
      u32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = __float_as_uint(f[e * (ROWB / 4)]);
      return v;
    } else {
      // 16 lanes fetch 4 rows of 16 elements (lane q of them: row q / 4, elements 4 (q % 4) ..) and lane q receives
      // element q of the 4 rows; twice, for 8 r
      const int q = lane & 15;
      const int r = (2 * ks + (lane >> 5)) * 8 + (q >> 2), col = i + (lane & 16) + 4 * (q & 3);
      const char* a = base + r * ROWB + swz(r, col >> 3) * 16 + (col & 7) * 2;
      typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
      const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(a));
      const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(a + 4 * ROWB));
      const u32x2 w0 = __builtin_bit_cast(u32x2, v0), w1 = __builtin_bit_cast(u32x2, v1);
      u32x4 v;
      v[0] = w0[0]; v[1] = w0[1]; v[2] = w1[0]; v[3] = w1[1];
      return v;
    }
  }
};

// Waits for the wave's own LDS accesses.
__device__ __forceinline__ void wait_lds() {
  __builtin_amdgcn_s_waitcnt(15 | (7 << 4) | (0 << 8) | (3 << 14));
  asm volatile("" ::: "memory");
}
__device__ __forceinline__ void barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
// Waits until at most N of the wave's loads are on their way, and keeps later LDS accesses behind that.
template <int N> __device__ __forceinline__ void wait_loads() {
  static_assert(N < 64, "six bits");
  __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));
  asm volatile("" ::: "memory");
}

// A workgroup of WM x WN waves, each FM x FN fragments of 32 x 32.
template <Kind K, bool A_ACROSS, bool B_ACROSS, int WM_, int WN_, int FM_, int FN_, int BKB, int PL, int STAGES>
struct Block {
  typedef typename Elem<K>::T T;
  static constexpr int WM = WM_, WN = WN_, FM = FM_, FN = FN_;
  static constexpr int NT = 64 * WM * WN;
  static constexpr int BM = 32 * WM * FM, BN = 32 * WN * FN;
  typedef Tile<K, A_ACROSS, BM, BKB, NT, PL> TA;
  typedef Tile<K, B_ACROSS, BN, BKB, NT, PL> TB;
  static constexpr int BK = TA::BK;
  static constexpr int STAGE = TA::BYTES + TB::BYTES;
  static constexpr int LDS_BYTES = STAGES * STAGE;
  static_assert(STAGES >= 2, "one tile in use, one on its way");

  f32x16 acc[FM][FN];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  }

  struct Frags {
    u32x4 a[PL][FM], b[PL][FN];
  };
  __device__ __forceinline__ static void read(Frags& f, const char* la, const char* lb, int ks, int lane, int wm, int wn) {
#pragma unroll
    for (int p = 0; p < PL; ++p) {
#pragma unroll
      for (int i = 0; i < FM; ++i) f.a[p][i] = TA::frag(la, p, (wm * FM + i) * 32, ks, lane);
#pragma unroll
      for (int j = 0; j < FN; ++j) f.b[p][j] = TB::frag(lb, p, (wn * FN + j) * 32, ks, lane);
    }
  }
  // The products of one step, in two parts: what follows the first part is issued behind instructions that are already
  // under way.  Consecutive instructions write different accumulators: none waits for the one before it.
  template <bool FIRST> __device__ __forceinline__ void multiply(const Frags& f) {
    if constexpr (PL == 2) {  // small terms first
      if constexpr (FIRST) {
        each_pair([&](int i, int j) { mfma<K>(acc[i][j], f.b[1][j], f.a[0][i], 0); });
      } else {
        each_pair([&](int i, int j) { mfma<K>(acc[i][j], f.b[0][j], f.a[1][i], 0); });
        each_pair([&](int i, int j) { mfma<K>(acc[i][j], f.b[0][j], f.a[0][i], 0); });
      }
    } else if constexpr (K == F32) {
#pragma unroll
      for (int e = FIRST ? 0 : 1; e < (FIRST ? 1 : 4); ++e)
        each_pair([&](int i, int j) { mfma<K>(acc[i][j], f.b[0][j], f.a[0][i], e); });
    } else {
      each_pair([&](int i, int j) {
        if ((i == 0) == FIRST) mfma<K>(acc[i][j], f.b[0][j], f.a[0][i], 0);
      });
    }
  }
  // One tile's products.  The fragments of step ks + 1 are on their way while the matrix cores work on step ks, across
  // the tile's end too: turn() - called once every read of this tile has arrived - makes the next tile's LDS ready and
  // returns it (nullptr: no more), so neither its barrier nor its first reads leave the matrix cores idle.
  static constexpr int KS = BKB / 32;
  static constexpr bool PIPE = PL * (FM + FN) <= 8;  // registers for two sets of fragments
  static_assert(KS % 2 == 0, "the sets alternate");
  Frags f[PIPE ? 2 : 1];
  __device__ __forceinline__ void first(const char* cur, int lane, int wm, int wn) {
    if constexpr (PIPE) read(f[0], cur, cur + TA::BYTES, 0, lane, wm, wn);
  }
  template <typename Turn> __device__ __forceinline__ void compute(const char* cur, int lane, int wm, int wn, Turn turn) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      if constexpr (PIPE) {
        // the wait for this step's fragments stands before the next one's are asked for, so it is for them alone
        multiply<true>(f[ks & 1]);
        __builtin_amdgcn_sched_barrier(0);
        if (ks + 1 < KS) {
          read(f[(ks + 1) & 1], cur, cur + TA::BYTES, ks + 1, lane, wm, wn);
        } else {
          wait_lds();
          const char* next = turn();
          if (next) read(f[0], next, next + TA::BYTES, 0, lane, wm, wn);
        }
        __builtin_amdgcn_sched_barrier(0);
        multiply<false>(f[ks & 1]);
        __builtin_amdgcn_sched_barrier(0);
      } else {
        read(f[0], cur, cur + TA::BYTES, ks, lane, wm, wn);
        if (ks + 1 == KS) {
          wait_lds();
          turn();
        }
        multiply<true>(f[0]);
        multiply<false>(f[0]);
      }
    }
  }

  template <typename F> __device__ __forceinline__ static void each_pair(F f) {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) f(i, j);
  }

  // acc += the sum over [r0, rend); A.rows, B.rows > 0.  aligned: bases and lds are multiples of 16 bytes, and the
  // columns of an operand across r whole chunks.
  __device__ __forceinline__ void run(char* lds, const Operand<T>& A, const Operand<T>& B, int m0, int n0, int r0,
                                      int rend, bool aligned) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (r0 >= rend) return;
    const int n = (rend - r0) / BK;
    if (!aligned) {
      through_registers(lds, m0, n0, (rend - r0 + BK - 1) / BK, 0, (rend - r0 + BK - 1) / BK,
                        [&](int, Operand<T>& a, Operand<T>& b, int& first, int& end) {
                          a = A;
                          b = B;
                          first = r0;
                          end = rend;
                          return A.rows;
                        });
      return;
    }
    // the cut tile's loads go first, where there are registers for them: they have arrived when the others are done
    const int cut = r0 + n * BK;
    typename TA::Regs ra;
    typename TB::Regs rb;
    TA ta;
    TB tb;
    constexpr bool EARLY = PL == 1 && BM * BN < 256 * 256;
    auto load_cut = [&]() {
      ta.seek(A, m0, cut, tid);
      tb.seek(B, n0, cut, tid);
      ta.load(ra, rend - cut, TA::WHOLE, A.ld, rend, m0, 0, false, tid);
      tb.load(rb, rend - cut, TB::WHOLE, B.ld, rend, n0, 0, false, tid);
    };
    if (EARLY && cut < rend) load_cut();
    if (n > 0)
      ring(lds, m0, n0, n, 0, n, [&](int, Operand<T>& a, Operand<T>& b, int& first) {
        a = A;
        b = B;
        first = r0;
      });
    if (cut < rend) {
      if (!EARLY) load_cut();
      ta.store(ra, lds, tid);
      tb.store(rb, lds + TA::BYTES, tid);
      __syncthreads();
      first(lds, lane, wave / WN, wave % WN);
      compute(lds, lane, wave / WN, wave % WN, []() -> const char* { return nullptr; });
      __syncthreads();
    }
  }

  // acc += the sum over tiles [from, to) of pieces of n whole tiles each: at(s, A, B, r0) says where piece s is
  template <typename At>
  __device__ __forceinline__ void ring(char* lds, int m0, int n0, int n, int64_t from, int64_t to, At at) {
    constexpr int LOADS = PL * (TA::PER + TB::PER);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = wave / WN, wn = wave % WN;
    const int all = (int)(to - from);
    TA ta;
    TB tb;
    Operand<T> A, B;
    int r0, s = (int)(from / n), t = (int)(from - (int64_t)s * n), issued = 0;
    auto seek = [&]() {
      at(s, A, B, r0);
      ta.seek(A, m0, r0 + t * BK, tid);
      tb.seek(B, n0, r0 + t * BK, tid);
    };
    auto fetch = [&](char* to) {
      ta.fetch(to, tid);
      tb.fetch(to + TA::BYTES, tid);
      ++issued;
      if (++t == n) {
        t = 0;
        ++s;
        if (issued < all) seek();
      } else {
        ta.advance(A.ld);
        tb.advance(B.ld);
      }
    };
    seek();
#pragma unroll
    for (int i = 0; i < STAGES; ++i)
      if (i < all) fetch(lds + i * STAGE);
    if (issued == STAGES) wait_loads<(STAGES - 1) * LOADS>();  // the first tile's
    else wait_loads<0>();
    barrier();
    first(lds, lane, wm, wn);
    int stage = 0;
    for (int it = 0; it < all; ++it) {
      char* cur = lds + stage * STAGE;
      stage = stage + 1 == STAGES ? 0 : stage + 1;
      char* nxt = lds + stage * STAGE;
      compute(cur, lane, wm, wn, [&]() -> const char* {
        if (it + 1 == all) return nullptr;
        if (issued - it == STAGES) wait_loads<(STAGES - 2) * LOADS>();  // the next tile's, not the ones behind it
        else wait_loads<0>();
        barrier();  // everyone's part of the next tile is there, and everyone has read this one
        if (issued < all) fetch(cur);
        return nxt;
      });
    }
    __syncthreads();
  }

  // The same through registers, pieces of n tiles of which the last may be cut: at(s, A, B, r0, rend) returns how many
  // rows of A take part in piece s (the others are zeros, and contribute nothing where B is finite).
  template <typename At>
  __device__ __forceinline__ void through_registers(char* lds, int m0, int n0, int n, int64_t from, int64_t to, At at) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = wave / WN, wn = wave % WN;
    if (n <= 0 || to <= from) return;
    const int all = (int)(to - from);
    TA ta;
    TB tb;
    typename TA::Regs ra;
    typename TB::Regs rb;
    Operand<T> A, B;
    int r0, rend, rows, s = (int)(from / n), t = (int)(from - (int64_t)s * n);
    typename TA::Columns cols_a;
    typename TB::Columns cols_b;
    auto seek = [&]() {
      rows = at(s, A, B, r0, rend);
      ta.seek(A, m0, r0 + t * BK, tid);
      tb.seek(B, n0, r0 + t * BK, tid);
      cols_a = TA::columns(m0, A.rows);
      cols_b = TB::columns(n0, B.rows);
    };
    auto load = [&]() {
      const int left = rend - r0 - t * BK;
      ta.load(ra, left, cols_a, A.ld, rend, m0, rows, rows < min(A.rows, m0 + BM), tid);
      tb.load(rb, left, cols_b, B.ld, rend, n0, 0, false, tid);
    };
    seek();
    load();
    ta.store(ra, lds, tid);
    tb.store(rb, lds + TA::BYTES, tid);
    __syncthreads();
    first(lds, lane, wm, wn);
    for (int it = 0; it < all; ++it) {
      char* cur = lds + (it & 1) * STAGE;
      char* nxt = lds + ((it + 1) & 1) * STAGE;
      const bool more = it + 1 < all;
      if (more) {
        if (++t == n) {
          t = 0;
          ++s;
          seek();
        } else {
          ta.advance(A.ld);
          tb.advance(B.ld);
        }
        load();
      }
      compute(cur, lane, wm, wn, [&]() -> const char* {
        if (!more) return nullptr;
        ta.store(ra, nxt, tid);  // everyone has read what was there: the tile before this one
        tb.store(rb, nxt + TA::BYTES, tid);
        wait_lds();
        barrier();
        return nxt;
      });
    }
    __syncthreads();
  }

  // whether any of the workgroup's sums is not finite
  __device__ __forceinline__ bool not_finite(char* lds) const {
    bool bad = false;
    each_pair([&](int i, int j) {
#pragma unroll
      for (int e = 0; e < 16; ++e) bad |= !(fabsf(acc[i][j][e]) < INFINITY);
    });
    int* any = reinterpret_cast<int*>(lds);
    if (threadIdx.x == 0) *any = 0;
    __syncthreads();
    if (bad) *any = 1;
    __syncthreads();
    const bool result = *any != 0;
    __syncthreads();
    return result;
  }

  // The sum of through_registers() in the same order, rows that take no part in a piece left as they are whatever B holds:
  // nothing is read ahead, and each matrix instruction's result is taken row by row.
  template <typename At>
  __device__ __forceinline__ void masked(char* lds, int m0, int n0, int n, int64_t from, int64_t to, At at) {
    static_assert(PL == 1, "one plane");
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = wave / WN, wn = wave % WN;
    if (n <= 0) return;
    for (int64_t pos = from; pos < to; ++pos) {
      Operand<T> A, B;
      int r0, rend;
      const int s = (int)(pos / n), t = (int)(pos - (int64_t)s * n);
      const int rows = at(s, A, B, r0, rend), left = rend - r0 - t * BK;
      if (rows <= m0) continue;
      {
        TA ta;
        typename TA::Regs ra;
        ta.seek(A, m0, r0 + t * BK, tid);
        ta.load(ra, left, TA::columns(m0, A.rows), A.ld, rend, m0, rows, rows < min(A.rows, m0 + BM), tid);
        ta.store(ra, lds, tid);
      }
      {
        TB tb;
        typename TB::Regs rb;
        tb.seek(B, n0, r0 + t * BK, tid);
        tb.load(rb, left, TB::columns(n0, B.rows), B.ld, rend, n0, 0, false, tid);
        tb.store(rb, lds + TA::BYTES, tid);
      }
      __syncthreads();
#pragma unroll 1
      for (int ks = 0; ks < KS; ++ks)
        each_pair([&](int i, int j) {
          const u32x4 a = TA::frag(lds, 0, (wm * FM + i) * 32, ks, lane);
          const u32x4 b = TB::frag(lds + TA::BYTES, 0, (wn * FN + j) * 32, ks, lane);
          f32x16 d = acc[i][j];
#pragma unroll
          for (int e = 0; e < (K == F32 ? 4 : 1); ++e) mfma<K>(d, b, a, e);
          const bool part = m0 + (wm * FM + i) * 32 + (lane & 31) < rows;
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[i][j][e] = part ? d[e] : acc[i][j][e];
        });
      __syncthreads();
    }
  }

  // the first of the columns, from n0, that each_row() gives this lane
  static __device__ __forceinline__ int lane_column() {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    return (wave % WN) * FN * 32 + (lane % (8 * FN)) * 4;
  }

  // f(m, n, v, x): 4 consecutive columns n .. n + 3 of row m, neighbouring lanes at neighbouring columns, 32 FN of a row,
  // through the wave's own part of LDS (which run() has left): stores cover whole lines.  pre(m, n) loads what f adds, for
  // all rows of a pass before any of them is stored.
  template <typename P, typename F> __device__ __forceinline__ void each_row(char* lds, int m0, int n0, P pre, F f) const {
    constexpr int LD = 32 * FN + 4;  // floats; the rows one pass writes fall on different banks
    constexpr int PERROW = 8 * FN, ROWS = 64 / PERROW, N = 32 / ROWS;
    static_assert(WM * WN * 32 * LD * 4 <= LDS_BYTES, "the epilogue's rows fit");
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = wave / WN, wn = wave % WN;
    float* buf = reinterpret_cast<float*>(lds) + wave * 32 * LD;
    const int col = (lane % PERROW) * 4, n = n0 + wn * FN * 32 + col;
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int mi = m0 + (wm * FM + i) * 32 + lane / PERROW;
      decltype(pre(0, 0)) x[N];
#pragma unroll
      for (int r = 0; r < N; ++r) x[r] = pre(mi + r * ROWS, n);
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          f32x4 v;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = acc[i][j][4 * q + e];
          *reinterpret_cast<f32x4*>(buf + (lane & 31) * LD + j * 32 + 8 * q + 4 * (lane >> 5)) = v;
        }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int r = 0; r < N; ++r)
        f(mi + r * ROWS, n, *reinterpret_cast<const f32x4*>(buf + (r * ROWS + lane / PERROW) * LD + col), x[r]);
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
  }

  // The same for the transposed result: f(n, m, v, x) with 4 consecutive rows m .. m + 3 of column n.
  template <typename P, typename F> __device__ __forceinline__ void each_column(char* lds, int m0, int n0, P pre, F f) const {
    constexpr int W = FM < 2 ? FM : 2;  // 32 W rows at a time
    constexpr int LD = 32 * W + 4, PERROW = 8 * W, ROWS = 64 / PERROW, N = 32 / ROWS;
    static_assert(WM * WN * 32 * LD * 4 <= LDS_BYTES && FM % W == 0, "the epilogue's rows fit");
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = wave / WN, wn = wave % WN;
    float* buf = reinterpret_cast<float*>(lds) + wave * 32 * LD;
    const int col = (lane % PERROW) * 4;
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int i = 0; i < FM; i += W) {
        const int m = m0 + (wm * FM + i) * 32 + col, nj = n0 + (wn * FN + j) * 32 + lane / PERROW;
        decltype(pre(0, 0)) x[N];
#pragma unroll
        for (int r = 0; r < N; ++r) x[r] = pre(nj + r * ROWS, m);
#pragma unroll
        for (int w = 0; w < W; ++w)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            buf[(8 * (e >> 2) + 4 * (lane >> 5) + (e & 3)) * LD + w * 32 + (lane & 31)] = acc[i + w][j][e];
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int r = 0; r < N; ++r)
          f(nj + r * ROWS, m, *reinterpret_cast<const f32x4*>(buf + (r * ROWS + lane / PERROW) * LD + col), x[r]);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
      }
  }
};

// ------------------------------------------------------------------------------------------ host: tile and split
struct TileShape {
  int bm, bn, per_cu;  // workgroups of it that a CU holds
  float rate;          // multiply-adds per cycle and CU of one CU full of them
};
struct Choice {
  int tile, splits, per_split;  // per_split: units of the sum per split
  int64_t tiles_m, tiles_n;
};

// The tile shape and the split of a product of `models` matrices m x n over r, whose sum comes in `units` pieces: the one
// with the least estimated cycles.  Counted are the rounds in which the workgroups run on 256 CUs, the products of padded
// tiles at the shape's measured rate, a fixed cost per workgroup, and for a split the partial sums' traffic (about 2 KB
// per cycle) and the second launch.
inline Choice choose(const TileShape* shapes, int n_shapes, int64_t models, int64_t m, int64_t n, int64_t r, int64_t units,
                     bool can_split, double* cost = nullptr) {
  Choice best = {};
  double least = 0;
  for (int s = 0; s < n_shapes; ++s) {
    const TileShape& t = shapes[s];
    if (t.rate <= 0) continue;
    const int64_t tm = (m + t.bm - 1) / t.bm, tn = (n + t.bn - 1) / t.bn, tiles = tm * tn * models;
    for (int64_t want = 1; want <= 64 && (want == 1 || (can_split && want <= units)); want *= 2) {
      int64_t per = (units + want - 1) / want;
      if (per < 1) per = 1;
      const int64_t splits = units > 0 ? (units + per - 1) / per : 1;
      if (want > 1 && splits * 2 <= want) continue;
      const double share = (double)r * per / (units > 0 ? units : 1);
      const int64_t blocks = tiles * splits;
      // a CU that holds fewer workgroups than it could runs them faster, down to one at 60 % of the full rate
      const int64_t full = blocks / (256 * t.per_cu), rest = blocks - full * 256 * t.per_cu;
      const double one = (double)t.bm * t.bn * share / t.rate + 2500;
      double cycles = full * t.per_cu * one;
      if (rest > 0) {
        const int64_t k = (rest + 255) / 256;
        cycles += one * (k > 1 ? k : (t.per_cu > 1 ? 1.6 : 1.0));
      }
      if (splits > 1) cycles += 8000 + (double)models * m * n * 4 * (splits + 1) / 2000;
      if (best.splits == 0 || cycles < least) {
        least = cycles;
        best = Choice{s, (int)splits, (int)per, tm, tn};
      }
    }
  }
  if (cost) *cost = least;
  return best;
}

}  // namespace mma
