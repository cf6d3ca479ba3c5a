// Products whose matrix depends on the column (lora*.hip, moe.hip): element types, the argument records shared with
// dplasma_amd/ops/indexed_ops.py, and fragments for the matrix instructions.
//
// Matrices are column-major with one token per column, so a token's features are contiguous: X(c, t) = X[t * ldx + c].
#pragma once
#include "common.h"

enum { DPL_H = 6, DPL_B = 7 };  // fp16, bf16: precisions of these operators only

template <typename T> struct Num {
  typedef float acc;
};
template <> struct Num<double> {
  typedef double acc;
};
template <typename T> __device__ inline typename Num<T>::acc widen(T v) { return (typename Num<T>::acc)v; }

struct LoraArgs {
  long long ldw, ldx, lda, ldb, ldy, lddx, ldda, lddb;
  const void *W, *X, *A, *B, *ids, *scale, *dY;  // scale null: ones
  void *Y, *dX, *dA, *dB, *ws;                   // forward: Y; gradient: dY in, dX / dA / dB out (each may be null)
  double alpha, beta;
  long long ws_bytes;
  int prec, T, K, N, r, L;
};

struct MoeArgs {
  long long ldg, ld1, ld2, ldx, ldy;
  const void *G, *W1, *W2, *X;
  void *Y, *ws;
  double alpha, beta;
  long long ws_bytes;
  int prec, T, H, I, E, topk, norm, pad;
};

// ---------------------------------------------------------------- fragments of 16 bytes
// A lane holds 16 bytes of a row: E elements that are contiguous along the contraction.  Lane group q = lane / 16 holds
// the q-th 16 bytes of 64, so one fragment of a 16-row operand is KS = 4 E long, and the matrix instruction that takes
// element i of every lane contracts the indices {E q + i}: any order will do as long as both operands use the same.
//   h, b: one 16x16x32 instruction;   s: four 16x16x4;   d: two 16x16x4
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef __bf16 b8_t __attribute__((ext_vector_type(8)));
typedef int i4_t __attribute__((ext_vector_type(4)));
typedef double d2_t __attribute__((ext_vector_type(2)));

template <typename T> struct Op;
template <> struct Op<__bf16> {
  typedef b8_t vec;
  typedef f4_t out;
  static constexpr int E = 8, KS = 32;
  static __device__ inline out mma(vec a, vec b, out c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Op<_Float16> {
  typedef h8_t vec;
  typedef f4_t out;
  static constexpr int E = 8, KS = 32;
  static __device__ inline out mma(vec a, vec b, out c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <> struct Op<float> {
  typedef f4_t vec;
  typedef f4_t out;
  static constexpr int E = 4, KS = 16;
  static __device__ inline out mma(vec a, vec b, out c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    return c;
  }
};
template <> struct Op<double> {
  typedef d2_t vec;
  typedef d4_t out;
  static constexpr int E = 2, KS = 8;
  static __device__ inline out mma(vec a, vec b, out c) {
#pragma unroll
    for (int i = 0; i < 2; ++i) c = __builtin_amdgcn_mfma_f64_16x16x4f64(a[i], b[i], c, 0, 0, 0);
    return c;
  }
};
// row of a 16 x 16 result that register i of a lane holds (its column is lane % 16)
template <typename T> __device__ inline int out_row(int lane, int i) {
  return sizeof(T) == 8 ? (lane >> 4) + 4 * i : 4 * (lane >> 4) + i;
}

// E elements from any element address
template <typename T> __device__ inline typename Op<T>::vec load_vec(const T* p) {
  typename Op<T>::vec v;
  __builtin_memcpy(&v, p, 16);
  return v;
}
// the same with zeros from the m-th element on
template <typename T> __device__ inline typename Op<T>::vec load_part(const T* p, int m) {
  if (m >= Op<T>::E) return load_vec(p);
  typename Op<T>::vec v;
#pragma unroll
  for (int i = 0; i < Op<T>::E; ++i) v[i] = i < m ? p[i] : (T)0;
  return v;
}

// the vector, or zeros
template <typename V> __device__ inline V keep(V v, bool in) {
  i4_t b = __builtin_bit_cast(i4_t, v);
#pragma unroll
  for (int i = 0; i < 4; ++i) b[i] = in ? b[i] : 0;
  return __builtin_bit_cast(V, b);
}

// ---------------------------------------------------------------- intermediates between two products
// A 32-bit result that is the next product's operand.  For h and b it goes to the 16-bit matrix instructions as two
// bf16 numbers, hi + lo: 16 bits of it (off by at most 2^-16 of itself) over the whole range of 32-bit numbers -- one
// 16-bit number would keep 8 bits, or overflow past 65504 in fp16 where the plain 32-bit intermediate does not.  The
// second product's own operand is exact in one bf16 (b) or two (h); of the four products of an h pair the smallest
// (lo lo, below 2^-16) is left out.  s and d keep their own type.
template <typename T> struct Mid {  // h, b
  typedef __bf16 elem;
  static constexpr int PARTS = 2;
  static __device__ inline void put(elem* hi, elem* lo, float v) {
    const __bf16 h = (__bf16)v;
    // an infinity has no remainder (inf - inf would make it NaN)
    const float rest = v - (float)h;
    *hi = h;
    *lo = (__bf16)(__builtin_isfinite(rest) ? rest : 0.f);
  }
};
template <> struct Mid<float> {
  typedef float elem;
  static constexpr int PARTS = 1;
  static __device__ inline void put(elem* hi, elem*, float v) { *hi = v; }
};
template <> struct Mid<double> {
  typedef double elem;
  static constexpr int PARTS = 1;
  static __device__ inline void put(elem* hi, elem*, double v) { *hi = v; }
};
// The other operand of a Mid product: one vector, or hi and lo for h.
template <typename T> struct MidOp {
  typedef typename Op<typename Mid<T>::elem>::vec vec;
  vec f;
  __device__ inline void set(typename Op<T>::vec v) { f = v; }
  __device__ inline typename Op<T>::out mma(vec hi, vec lo, typename Op<T>::out c) const {
    c = Op<T>::mma(f, hi, c);
    return Mid<T>::PARTS == 2 ? Op<T>::mma(f, lo, c) : c;
  }
  // the intermediate as the first operand
  __device__ inline typename Op<T>::out mma_first(vec hi, vec lo, typename Op<T>::out c) const {
    c = Op<T>::mma(hi, f, c);
    return Mid<T>::PARTS == 2 ? Op<T>::mma(lo, f, c) : c;
  }
};
template <> struct MidOp<_Float16> {
  typedef b8_t vec;
  vec f, g;
  // 11 bits: the upper 8 by truncation, the rest exactly in the second number (none beside an infinity)
  __device__ inline void set(h8_t v) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = (float)v[i], h = __uint_as_float(__float_as_uint(x) & 0xffff0000u), rest = x - h;
      f[i] = (__bf16)h;
      g[i] = (__bf16)(rest == rest ? rest : 0.f);
    }
  }
  __device__ inline f4_t mma(vec hi, vec lo, f4_t c) const {
    c = Op<__bf16>::mma(f, hi, c);
    c = Op<__bf16>::mma(f, lo, c);
    return Op<__bf16>::mma(g, hi, c);
  }
  __device__ inline f4_t mma_first(vec hi, vec lo, f4_t c) const {
    c = Op<__bf16>::mma(hi, f, c);
    c = Op<__bf16>::mma(lo, f, c);
    return Op<__bf16>::mma(hi, g, c);
  }
};

// ---------------------------------------------------------------- workspace cursor
struct Carve {
  char* p;
  size_t used = 0;
  template <typename T> T* take(size_t n) {
    T* q = (T*)(p ? p + used : nullptr);
    used += (n * sizeof(T) + 255) & ~(size_t)255;
    return q;
  }
};
