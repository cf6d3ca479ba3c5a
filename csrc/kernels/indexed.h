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
// A 32-bit result that is the next product's operand.  It lies in memory as it is (64 bits in d).  For h and b it goes to
// the 16-bit matrix instructions as three bf16 numbers of 8 bits each whose sum it is, over the whole range of 32-bit
// numbers: nothing is rounded between the two products.  The second product's own operand is exact in one bf16 (b) or two
// (h), so three or six products of the instruction's are the exact product.  s and d take it as it is.
//
// Mem: a lane's intermediates as they come from memory, Op<T>::E of them.
template <typename T> struct Mem {  // h, b
  f4_t v[2];
  __device__ inline void load(const float* p) {
    v[0] = load_vec(p);
    v[1] = load_vec(p + 4);
  }
  // zeros from the m-th on
  __device__ inline void load_to(const float* p, int m) {
    v[0] = load_part(p, m);
    v[1] = load_part(p + 4, m - 4);
  }
};
template <> struct Mem<float> {
  f4_t v;
  __device__ inline void load(const float* p) { v = load_vec(p); }
  __device__ inline void load_to(const float* p, int m) { v = load_part(p, m); }
};
template <> struct Mem<double> {
  d2_t v;
  __device__ inline void load(const double* p) { v = load_vec(p); }
  __device__ inline void load_to(const double* p, int m) { v = load_part(p, m); }
};
// Mid: the same as operands.
template <typename T> struct Mid {  // h, b
  b8_t part[3];
  __device__ inline void set(const Mem<T>& m) {
    i4_t w[3];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      unsigned u[3][2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        // by truncation: 8 bits, then the exact rest's 8, then the last 8.  An infinity has no rest (inf - inf would make
        // it NaN)
        const float x = m.v[i / 2][i % 2 * 2 + e];
        u[0][e] = __float_as_uint(x);
        float rest = x - __uint_as_float(u[0][e] & 0xffff0000u);
        rest = rest == rest ? rest : 0.f;
        u[1][e] = __float_as_uint(rest);
        u[2][e] = __float_as_uint(rest - __uint_as_float(u[1][e] & 0xffff0000u));
      }
#pragma unroll
      for (int p = 0; p < 3; ++p) w[p][i] = (int)__builtin_amdgcn_perm(u[p][1], u[p][0], 0x07060302);  // both upper halves
    }
#pragma unroll
    for (int p = 0; p < 3; ++p) part[p] = __builtin_bit_cast(b8_t, w[p]);
  }
};
template <> struct Mid<float> {
  f4_t part;
  __device__ inline void set(const Mem<float>& m) { part = m.v; }
};
template <> struct Mid<double> {
  d2_t part;
  __device__ inline void set(const Mem<double>& m) { part = m.v; }
};
// The other operand of a Mid product, which is a sum of N of the instruction's: product k adds the k-th (product_first: with
// the intermediate as the instruction's first operand).  One after the other on the same accumulators they would wait for
// each other, so kernels with several accumulators put the loop over k outside.
template <typename T> struct MidOp {  // s, d
  static constexpr int N = 1;
  typename Op<T>::vec f;
  __device__ inline void set(typename Op<T>::vec v) { f = v; }
  __device__ inline typename Op<T>::out product(int, const Mid<T>& m, typename Op<T>::out c) const { return Op<T>::mma(f, m.part, c); }
  __device__ inline typename Op<T>::out product_first(int, const Mid<T>& m, typename Op<T>::out c) const { return Op<T>::mma(m.part, f, c); }
};
template <> struct MidOp<__bf16> {
  static constexpr int N = 3;
  b8_t f;
  __device__ inline void set(b8_t v) { f = v; }
  __device__ inline f4_t product(int k, const Mid<__bf16>& m, f4_t c) const { return Op<__bf16>::mma(f, m.part[k], c); }
  __device__ inline f4_t product_first(int k, const Mid<__bf16>& m, f4_t c) const { return Op<__bf16>::mma(m.part[k], f, c); }
};
template <> struct MidOp<_Float16> {
  static constexpr int N = 6;
  b8_t f, g;
  // 11 bits: the upper 8 by truncation, the rest exactly in the second number (none beside an infinity)
  __device__ inline void set(h8_t v) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = (float)v[i], h = __uint_as_float(__float_as_uint(x) & 0xffff0000u), rest = x - h;
      f[i] = (__bf16)h;
      g[i] = (__bf16)(rest == rest ? rest : 0.f);
    }
  }
  __device__ inline f4_t product(int k, const Mid<_Float16>& m, f4_t c) const { return Op<__bf16>::mma(k < 3 ? f : g, m.part[k % 3], c); }
  __device__ inline f4_t product_first(int k, const Mid<_Float16>& m, f4_t c) const { return Op<__bf16>::mma(m.part[k % 3], k < 3 ? f : g, c); }
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
