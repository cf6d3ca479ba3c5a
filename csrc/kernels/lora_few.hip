// gemm_lora for a few tokens (T <= 64): the weights are read once and everything else hides behind that.
#include "lora.h"

namespace {

// S[t*r + j] = s_l sum_k x[t*ldx + k] A_l[j*lda + k], one wave per (t, j).
template <typename T>
__global__ __launch_bounds__(256) void k_few_low(const T* __restrict__ x, long long ldx, const T* __restrict__ A,
                                                 long long lda, const int* __restrict__ ids,
                                                 const typename Num<T>::acc* __restrict__ scale, int K, int r, int L,
                                                 typename Num<T>::acc* __restrict__ S) {
  typedef typename Num<T>::acc R;
  constexpr int E = Op<T>::E;
  const int t = blockIdx.x, j = blockIdx.y * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int l = ids[t];
  if (j >= r) return;
  R s = 0;
  if ((unsigned)l < (unsigned)L) {
    const T* a = A + ((long long)l * r + j) * lda;
    const T* p = x + (long long)t * ldx;
#pragma unroll 4
    for (int k = lane * E; k < K; k += 64 * E) {
      const typename Op<T>::vec u = load_part(a + k, K - k), v = load_part(p + k, K - k);
#pragma unroll
      for (int i = 0; i < E; ++i) s = fma((R)u[i], (R)v[i], s);
    }
    for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
    s *= scale ? scale[l] : R(1);
  }
  if (lane == 0) S[(long long)t * r + j] = s;
}

// 16 NF output features per workgroup, the contraction split over 8 waves and joined in LDS; G groups of 16 tokens.
// W's fragments go straight from memory to the matrix instruction (each element is used by one wave once); x comes
// from the caches.  A wave has one batch of fragments under way after another, as large as the registers of one
// workgroup per CU allow; what the adapters' parts need is asked for before and beside them.
template <int N> struct Int {
  static constexpr int value = N;
};
constexpr int S_MAX = 64;  // r up to which the low-rank vectors go through LDS

template <typename T, int G, int NF>
__global__ __launch_bounds__(512) void k_few_apply(const T* __restrict__ x, long long ldx, const T* __restrict__ W,
                                                   long long ldw, const T* __restrict__ B, long long ldb,
                                                   const int* __restrict__ ids,
                                                   const typename Num<T>::acc* __restrict__ S, int nt, int K, int N,
                                                   int r, int L, typename Num<T>::acc alpha,
                                                   typename Num<T>::acc beta, T* __restrict__ y, long long ldy) {
  typedef typename Num<T>::acc R;
  typedef typename Op<T>::vec V;
  constexpr int E = Op<T>::E, KS = Op<T>::KS, ROW = 16 * NF, LANES = 512 / ROW;  // tokens finished at a time
  constexpr int TI = (16 * G + LANES - 1) / LANES, SI = 16 * G * S_MAX / 512;
  __shared__ R red[8][16 * G][ROW + 1], low[16 * G * S_MAX];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, q = lane >> 4, c = lane & 15;
  const int n0 = blockIdx.x * ROW;
  const int steps = (K + KS - 1) / KS, s0 = steps * w / 8, s1 = steps * (w + 1) / 8, whole = min(s1, K / KS);
  typename Op<T>::out acc[NF][G];
#pragma unroll
  for (int f = 0; f < NF; ++f)
#pragma unroll
    for (int g = 0; g < G; ++g) acc[f][g] = typename Op<T>::out{R(0), R(0), R(0), R(0)};
  const T *pw[NF], *px[G];
#pragma unroll
  for (int f = 0; f < NF; ++f) pw[f] = W + (long long)min(n0 + 16 * f + c, N - 1) * ldw + q * E;
#pragma unroll
  for (int g = 0; g < G; ++g) px[g] = x + (long long)min(16 * g + c, nt - 1) * ldx + q * E;
  // this thread finishes feature n of tokens tid / ROW + LANES k
  const int col = tid % ROW, n = n0 + col;
  int lid[TI];
#pragma unroll
  for (int k = 0; k < TI; ++k) {
    const int t = tid / ROW + LANES * k;
    lid[k] = L > 0 && t < nt ? ids[t] : -1;
    if ((unsigned)lid[k] >= (unsigned)L) lid[k] = -1;
  }
  R sv[SI];
  if (r <= S_MAX && L > 0) {
#pragma unroll
    for (int k = 0; k < SI; ++k)
      if (tid + 512 * k < nt * r) sv[k] = S[tid + 512 * k];
  }
  int s = s0;
  auto run = [&](auto width) {
    constexpr int U = decltype(width)::value;
    V a[U][NF], b[U][G];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int f = 0; f < NF; ++f) a[u][f] = load_vec(pw[f] + (long long)(s + u) * KS);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int g = 0; g < G; ++g) b[u][g] = load_vec(px[g] + (long long)(s + u) * KS);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int f = 0; f < NF; ++f) acc[f][g] = Op<T>::mma(a[u][f], b[u][g], acc[f][g]);
    s += U;
  };
  if constexpr (G == 1)
    while (s + 16 <= whole) run(Int<16>());
  if constexpr (sizeof(T) < 8)
    while (s + 8 <= whole) run(Int<8>());
  while (s + 4 <= whole) run(Int<4>());
  while (s + 2 <= whole) run(Int<2>());
  if (s < whole) run(Int<1>());
  for (; s < s1; ++s) {
    const int left = K - s * KS - q * E;
    V a[NF];
#pragma unroll
    for (int f = 0; f < NF; ++f) a[f] = load_part(pw[f] + (long long)s * KS, left);
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const V b = load_part(px[g] + (long long)s * KS, left);
#pragma unroll
      for (int f = 0; f < NF; ++f) acc[f][g] = Op<T>::mma(a[f], b, acc[f][g]);
    }
  }
  // the first two vectors of the adapters' rows, on their way during the join
  const int nv = min(2, r / E);
  V bv[TI][2];
#pragma unroll
  for (int k = 0; k < TI; ++k)
    if (lid[k] >= 0 && n < N) {
      const T* b = B + ((long long)lid[k] * N + n) * ldb;
#pragma unroll
      for (int v = 0; v < 2; ++v)
        if (v < nv) bv[k][v] = load_vec(b + v * E);
    }
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
      for (int i = 0; i < 4; ++i) red[w][16 * g + c][16 * f + out_row<T>(lane, i)] = acc[f][g][i];
  if (r <= S_MAX && L > 0) {
#pragma unroll
    for (int k = 0; k < SI; ++k)
      if (tid + 512 * k < nt * r) low[tid + 512 * k] = sv[k];
  }
  __syncthreads();
  if (n >= N) return;
#pragma unroll
  for (int k = 0; k < TI; ++k) {
    const int t = tid / ROW + LANES * k;
    if (t >= nt) continue;
    R v = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) v += red[i][t][col];
    if (lid[k] >= 0) {
      const T* b = B + ((long long)lid[k] * N + n) * ldb;
      auto add = [&](const R* p) {
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (e < nv) {
#pragma unroll
            for (int i = 0; i < E; ++i) v = fma(p[e * E + i], (R)bv[k][e][i], v);
          }
        int j = nv * E;
#pragma unroll 2
        for (; j + E <= r; j += E) {
          const V f = load_vec(b + j);
#pragma unroll
          for (int i = 0; i < E; ++i) v = fma(p[j + i], (R)f[i], v);
        }
        for (; j < r; ++j) v = fma(p[j], widen(b[j]), v);
      };
      if (r <= S_MAX) add(&low[t * r]);
      else add(S + (long long)t * r);
    }
    T* o = &y[(long long)t * ldy + n];
    R u = alpha == R(0) ? R(0) : alpha * v;
    if (beta != R(0)) u += beta * widen(*o);
    *o = (T)u;
  }
}

template <typename T> int run(const LoraArgs& g, hipStream_t st) {
  typedef typename Num<T>::acc R;
  R* S = (R*)g.ws;
  const T *X = (const T*)g.X, *A = (const T*)g.A, *B = (const T*)g.B, *W = (const T*)g.W;
  const int* ids = (const int*)g.ids;
  if (g.L > 0) k_few_low<T><<<dim3(g.T, cdiv(g.r, 4)), 256, 0, st>>>(X, g.ldx, A, g.lda, ids, (const R*)g.scale, g.K, g.r, g.L, S);
  // two fragments of features for a fragment of tokens where that leaves a workgroup for every CU: x is read half as
  // often, and what a CU can have under way is the bound (48 tokens, 4096 x 8192: 43.4 us with one, 30.6 with two; 48
  // tokens, 4096 x 4096: 23.2 with one, 27.0 with two)
  const int nf = sizeof(T) < 8 && g.T > 16 && g.N >= 32 * 256 ? 2 : 1;
  auto apply = [&](auto kernel) {
    kernel<<<cdiv(g.N, 16 * nf), 512, 0, st>>>(X, g.ldx, W, g.ldw, B, g.ldb, ids, S, g.T, g.K, g.N, g.r, g.L, (R)g.alpha, (R)g.beta,
                                          (T*)g.Y, g.ldy);
  };
  if constexpr (sizeof(T) < 8)
    if (nf == 2) {
      if (g.T <= 32) apply(k_few_apply<T, 2, 2>);
      else if (g.T <= 48) apply(k_few_apply<T, 3, 2>);
      else apply(k_few_apply<T, 4, 2>);
      return (int)hipGetLastError();
    }
  if (g.T <= 16) apply(k_few_apply<T, 1, 1>);
  else if (g.T <= 32) apply(k_few_apply<T, 2, 1>);
  else if (g.T <= 48) apply(k_few_apply<T, 3, 1>);
  else apply(k_few_apply<T, 4, 1>);
  return (int)hipGetLastError();
}

}  // namespace

size_t lora_few_ws(const LoraArgs& g) { return (size_t)g.T * g.r * (g.prec == DPL_D ? 8 : 4); }

int lora_few(const LoraArgs& g, hipStream_t st) {
  switch (g.prec) {
    case DPL_S: return run<float>(g, st);
    case DPL_D: return run<double>(g, st);
    case DPL_H: return run<_Float16>(g, st);
    case DPL_B: return run<__bf16>(g, st);
  }
  return -1;
}
