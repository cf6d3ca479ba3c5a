// Launchers and shared pieces of gemm_lora's kernels (lora*.hip).
#pragma once
#include "indexed.h"

// 16 bytes per lane from memory to LDS (lane i to lds + 16 i; lds is the same for the whole wave).  The buffer form reads
// base[off + soff ..], zeros where that is past `bytes`.
// The kernels that use these have all their LDS in one object: with two the compiler tells their accesses apart, and then
// waits for every load to LDS that is under way before it reads the object that they go to.  The waits are the kernels'.
__device__ inline void dma_buffer(const void* base, unsigned bytes, void* lds, unsigned off, int soff) {
#ifdef __HIP_DEVICE_COMPILE__
  __builtin_amdgcn_raw_ptr_buffer_load_lds(__builtin_amdgcn_make_buffer_rsrc((void*)base, 0, bytes, 0x00020000),
                                           (__attribute__((address_space(3))) void*)lds, 16, off, soff, 0, 0);
#endif
}
__device__ inline void dma_global(const void* p, void* lds) {
#ifdef __HIP_DEVICE_COMPILE__
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)p,
                                   (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
#endif
}

// The transposing LDS read: of a group of 16 lanes lane i gets, as element j, element i % 4 of what lane 4 j + i / 4 points
// at.  A function of its own, with a restricted pointer, for the alias scope: without one the compiler waits for every
// load to LDS that is under way before the read (dX, bf16, 100 tokens, 4096 x 4096: 45.1 us with those waits, 26.8
// without; 16384 tokens, 16384 -> 4096: 1.15 PFLOP/s, 1.38).
typedef short s4_t __attribute__((ext_vector_type(4)));
__device__ inline s4_t read_turned(const char* __restrict__ p) {
#ifdef __HIP_DEVICE_COMPILE__
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4_t*)p);
#else
  return s4_t{};
#endif
}

template <int N> struct Int {
  static constexpr int value = N;
};

// The rows p[0 .. ROWS) against x by one wave, its lanes along the rows; every lane gets the sums.  4 loads of a row are
// under way at a time (with 8 the low-rank vectors of 48 tokens, K = 4096, took 2.5 us longer).
template <int ROWS, typename T>
__device__ inline void wave_dots(const T* const* p, const T* x, int K, typename Num<T>::acc* out) {
  typedef typename Num<T>::acc R;
  typedef typename Op<T>::vec V;
  constexpr int E = Op<T>::E, STEP = 64 * E;
  R s[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) s[i] = 0;
  int k = (threadIdx.x & 63) * E, left = K / STEP;
  auto run = [&](auto width) {
    constexpr int U = decltype(width)::value;
    V a[U][ROWS], b[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int i = 0; i < ROWS; ++i) a[u][i] = load_vec(p[i] + k + u * STEP);
      b[u] = load_vec(x + k + u * STEP);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < ROWS; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) s[i] = fma((R)a[u][i][e], (R)b[u][e], s[i]);
    k += U * STEP;
    left -= U;
  };
  while (left >= 4) run(Int<4>());
  if (left >= 2) run(Int<2>());
  if (left) run(Int<1>());
  if (k < K) {
    const V b = load_part(x + k, K - k);
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const V a = load_part(p[i] + k, K - k);
#pragma unroll
      for (int e = 0; e < E; ++e) s[i] = fma((R)a[e], (R)b[e], s[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    for (int o = 32; o; o >>= 1) s[i] += __shfl_xor(s[i], o);
    out[i] = s[i];
  }
}

// T <= 64, forward (lora_few.hip)
size_t lora_few_ws(const LoraArgs& g);
int lora_few(const LoraArgs& g, hipStream_t st);

// Low-rank vectors of every token, 32-bit numbers (64 in d) for the next product (Mem<T>).
//   by_token:    [t * rp + j], zeros for j in r .. rp (rp: r in whole matrix steps)
//   by_adapter:  [j * tp + pos[t]], the tokens of an adapter next to each other (the gradients of its factors)
// Nothing is written for a token without an adapter, and nothing of it is used.
struct LowOut {
  void *by_token, *by_adapter;  // null: not asked for
  const int* pos;
  long long tp;
  int rp;
};

template <typename T> __device__ inline void put_low(const LowOut& o, int t, int j, typename Num<T>::acc v) {
  typedef typename Num<T>::acc R;
  if (o.by_token) ((R*)o.by_token)[(long long)t * o.rp + j] = v;
  if (o.by_adapter) ((R*)o.by_adapter)[j * o.tp + o.pos[t]] = v;
}
template <typename T> __device__ inline void pad_low(const LowOut& o, int t, int j) {
  typedef typename Num<T>::acc R;
  if (o.by_token) ((R*)o.by_token)[(long long)t * o.rp + j] = R(0);
}

static inline int low_pitch(int prec, int r) {
  const int ks = prec == DPL_D ? 8 : prec == DPL_S ? 16 : 32;
  return cdiv(r, ks) * ks;
}
static inline size_t mid_bytes(int prec) { return prec == DPL_D ? 8 : 4; }

// out(t, j) = s_l sum_c x[t*ldx + c] F[(l*r + j)*ldf + c],  l = ids[t], for one or two sets of the same tokens.
struct LowArgs {
  const void *x, *F, *scale;
  const int* ids;
  long long ldx, ldf;
  int prec, nt, C, r, L;
  LowOut out;
};
int lora_low(const LowArgs* sets, int n, hipStream_t st);

// y[t*ldy + n] = alpha (sum_c x[t*ldx + c] W(n, c) + sum_j low(t, j) F[(l*N + n)*ldf + j]) + beta y[t*ldy + n];
// nt: W(n, c) = W[n*ldw + c], else W[c*ldw + n]
struct TileArgs {
  const void *x, *W, *F, *low;  // low: by token
  const int* ids;
  void* y;
  long long ldx, ldw, ldf, ldy;
  double alpha, beta;
  int prec, T, C, N, r, rp, L;
};
int lora_tile(const TileArgs& a, bool nt, hipStream_t st);

// Gradient (lora_grad.hip).
size_t lora_grad_ws(const LoraArgs& g);
int lora_grad(const LoraArgs& g, hipStream_t st);
