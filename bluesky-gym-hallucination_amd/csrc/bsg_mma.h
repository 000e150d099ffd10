// Matrix-core fragments shared by the memory operators (bsg_delta.hip, bsg_attention.hip).
//
// One product step is D[16][16] += A[16][32] B[32][16] on one wave, for fp32 or bf16 operands
// and fp32 accumulators.  Lane l (m = l & 15, g = l >> 4) holds eight k-values of row m of A,
// the same eight of column m of B, and D[4g + r][m], r = 0..3.  A product does not care which
// eight k-values a lane group holds as long as A and B agree, and two orders are used:
//   "run":  k = 8g + j                                (eight consecutive values of a row)
//   "tile": k = 4g + j (j < 4), 16 + 4g + j - 4 (j >= 4)
// The tile order is the one in which two stacked D tiles lie in registers, so the result of one
// product is the B operand of the next without leaving them (scores -> probabilities -> output,
// state -> state).
//
// fp32 operands go through v_mfma_f32_16x16x4_f32 (exact fp32 products; the j-th of eight
// instructions takes the lane's j-th value).  bf16 operands take one v_mfma_f32_16x16x32_bf16.
// An fp32 value that meets a bf16 operand is split into bf16 parts (Wide): value = p0 + p1 + p2,
// each part the rounding of what the ones before left, 8 bits a part, so three parts hold the
// fp32 value and two hold it to 2^-17.
#ifndef BSG_MMA_H_
#define BSG_MMA_H_

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace bsg {
namespace mma {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16;
typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));

template <class T> struct FragOf;
template <> struct FragOf<float> { typedef f32x8 F; typedef f32x4 H; };
template <> struct FragOf<bf16> { typedef bf16x8 F; typedef bf16x4 H; };
template <class T> using Frag = typename FragOf<T>::F;   // a lane's eight k-values
template <class T> using Half = typename FragOf<T>::H;   // four of them

// an fp32-valued operand next to operands of type T
template <class T, int N> struct Wide { Frag<T> p[N]; };
template <class T, int N> struct Parts { static constexpr int n = N; };
template <int N> struct Parts<float, N> { static constexpr int n = 1; };
template <class T, int N> using WideOf = Wide<T, Parts<T, N>::n>;

__device__ __forceinline__ void mma(f32x4& d, const bf16x8& a, const bf16x8& b) {
  d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, d, 0, 0, 0);
}
__device__ __forceinline__ void mma(f32x4& d, const f32x8& a, const f32x8& b) {
#pragma unroll
  for (int j = 0; j < 8; ++j) d = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], d, 0, 0, 0);
}
// one operand exact in T, the other wide
template <class T, int N>
__device__ __forceinline__ void mma(f32x4& d, const Frag<T>& a, const Wide<T, N>& b) {
#pragma unroll
  for (int i = N - 1; i >= 0; --i) mma(d, a, b.p[i]);
}
template <class T, int N>
__device__ __forceinline__ void mma(f32x4& d, const Wide<T, N>& a, const Frag<T>& b) {
#pragma unroll
  for (int i = N - 1; i >= 0; --i) mma(d, a.p[i], b);
}
// both wide: the parts' products down to the order that a part has
template <class T, int N>
__device__ __forceinline__ void mma(f32x4& d, const Wide<T, N>& a, const Wide<T, N>& b) {
#pragma unroll
  for (int s = N - 1; s >= 0; --s)
#pragma unroll
    for (int i = 0; i <= s; ++i) mma(d, a.p[i], b.p[s - i]);
}
// the same for several D that share B, a part at a time: products of one D do not wait for each other
template <class T, int M, int N>
__device__ __forceinline__ void mma_all(f32x4 (&d)[M], const Frag<T> (&a)[M], const Wide<T, N>& b) {
#pragma unroll
  for (int i = N - 1; i >= 0; --i)
#pragma unroll
    for (int j = 0; j < M; ++j) mma(d[j], a[j], b.p[i]);
}
// D[16][16] += A[16][16] B[16][16] in fp32: a[r] = A[m][4g + r], b[r] = B[4g + r][m], which is
// how a D tile lies in registers
__device__ __forceinline__ void mma16(f32x4& d, const f32x4& a, const f32x4& b) {
#pragma unroll
  for (int r = 0; r < 4; ++r) d = __builtin_amdgcn_mfma_f32_16x16x4f32(a[r], b[r], d, 0, 0, 0);
}

// ---- loads of a lane's eight k-values ------------------------------------------------------
__device__ __forceinline__ f32x8 join(const f32x4& a, const f32x4& b) {
  return f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}
__device__ __forceinline__ bf16x8 join(const bf16x4& a, const bf16x4& b) {
  return bf16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}
// from a row (16-byte aligned at k0 + 8g), run order
template <class T>
__device__ __forceinline__ Frag<T> load_run(const T* row, int k0, int g) {
  return *reinterpret_cast<const Frag<T>*>(row + k0 + 8 * g);
}
// from a row, tile order
template <class T>
__device__ __forceinline__ Frag<T> load_tile(const T* row, int k0, int g) {
  return join(*reinterpret_cast<const Half<T>*>(row + k0 + 4 * g),
              *reinterpret_cast<const Half<T>*>(row + k0 + 16 + 4 * g));
}
// from column m0 + m of a row-major LDS tile whose rows are k, tile order.  bf16: the transposing
// LDS read; the 16 lanes of a group address four rows of 16 values (lane i: row i / 4, values
// 4 (i % 4)..+3) and lane i receives column i.
__device__ __forceinline__ f32x8 load_col(const float* s, int ld, int k0, int m0, int lane) {
  const int m = lane & 15, g = lane >> 4;
  const float* p = s + (k0 + 4 * g) * ld + m0 + m;
  const float* q = p + 16 * ld;
  return f32x8{p[0], p[ld], p[2 * ld], p[3 * ld], q[0], q[ld], q[2 * ld], q[3 * ld]};
}
__device__ __forceinline__ bf16x8 load_col(const bf16* s, int ld, int k0, int m0, int lane) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  const int i = lane & 15, g = lane >> 4;
  const bf16* p = s + (k0 + 4 * g + (i >> 2)) * ld + m0 + 4 * (i & 3);
  const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p));
  const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 16 * ld));
  return join(__builtin_bit_cast(bf16x4, a), __builtin_bit_cast(bf16x4, b));
}

// ---- conversions ---------------------------------------------------------------------------
// two values to bf16, a in the low half: one instruction (value by value it is two and one to join them)
__device__ __forceinline__ uint32_t pair(float a, float b) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
}
template <class T, int N>
__device__ __forceinline__ void split(Wide<T, N>& w, const f32x8& x);
__device__ __forceinline__ void split(Wide<float, 1>& w, const f32x8& x) { w.p[0] = x; }
template <int N>
__device__ __forceinline__ void split(Wide<bf16, N>& w, const f32x8& x) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  f32x8 rest = x;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    u32x4 part;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      part[j] = pair(rest[2 * j], rest[2 * j + 1]);
      rest[2 * j] -= __uint_as_float(part[j] << 16);
      rest[2 * j + 1] -= __uint_as_float(part[j] & 0xffff0000u);
    }
    w.p[i] = __builtin_bit_cast(bf16x8, part);
  }
}
template <class T> __device__ __forceinline__ Frag<T> round_frag(const f32x8& x);
template <> __device__ __forceinline__ f32x8 round_frag<float>(const f32x8& x) { return x; }
template <> __device__ __forceinline__ bf16x8 round_frag<bf16>(const f32x8& x) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(bf16x8, u32x4{pair(x[0], x[1]), pair(x[2], x[3]), pair(x[4], x[5]), pair(x[6], x[7])});
}
__device__ __forceinline__ f32x8 widen(const f32x8& x) { return x; }
__device__ __forceinline__ f32x8 widen(const bf16x8& x) {
  f32x8 r;
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = (float)x[j];
  return r;
}
__device__ __forceinline__ f32x4 widen(const f32x4& x) { return x; }
__device__ __forceinline__ f32x4 widen(const bf16x4& x) {
  return f32x4{(float)x[0], (float)x[1], (float)x[2], (float)x[3]};
}
template <class T>
__device__ __forceinline__ void store4(T* p, const f32x4& x) {   // 4 T's, aligned to their size
  Half<T> h;
#pragma unroll
  for (int r = 0; r < 4; ++r) h[r] = (T)x[r];
  *reinterpret_cast<Half<T>*>(p) = h;
}

// Values per 16-byte access, and the LDS row pitch for rows of n values: 16 bytes more than the
// row, so that the 16 rows a fragment load touches start in different banks.
template <class T> struct Vec { static constexpr int n = 16 / (int)sizeof(T); };
template <class T> __host__ __device__ constexpr int pitch(int n) { return n + Vec<T>::n; }

// sum / max over the four lane groups (the rows of a D tile): lanes 16 and 32 apart trade places
__device__ __forceinline__ float sum_groups(float x) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
__device__ __forceinline__ float max_groups(float x) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// An R x N tile on its way from memory to LDS through registers: loaded while the one before it is
// computed.  Rows behind `rows` (at least 1) become zeros; in their place the last one is read.
template <class T, int R, int N, int NT>
struct Fetch {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  static constexpr int V = Vec<T>::n, ROW = N / V, n = (R * ROW + NT - 1) / NT;
  u32x4 x[n];
  __device__ __forceinline__ void load(const T* p, int64_t stride, int rows, int tid) {
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const int at = tid + i * NT, r = at / ROW, c = at % ROW * V;
      x[i] = *reinterpret_cast<const u32x4*>(p + min(r, rows - 1) * stride + c);
    }
  }
  __device__ __forceinline__ void store(T* s, int rows, int tid) const {
    if (rows >= R) {
#pragma unroll
      for (int i = 0; i < n; ++i) put(s, tid + i * NT, x[i]);
    } else {
#pragma unroll
      for (int i = 0; i < n; ++i) put(s, tid + i * NT, (tid + i * NT) / ROW < rows ? x[i] : u32x4{0, 0, 0, 0});
    }
  }
  static __device__ __forceinline__ void put(T* s, int at, const u32x4& v) {
    const int r = at / ROW, c = at % ROW * V;
    if (R * ROW % NT == 0 || r < R) *reinterpret_cast<u32x4*>(s + r * pitch<T>(N) + c) = v;
  }
};

}  // namespace mma
}  // namespace bsg
#endif  // BSG_MMA_H_
