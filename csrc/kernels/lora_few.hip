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

// 16 output features per workgroup, the contraction split over 8 waves and joined in LDS; G groups of 16 tokens.
// W's fragments go straight from memory to the matrix instruction (each element is used by one wave once); x comes
// from the caches.
template <typename T, int G>
__global__ __launch_bounds__(512) void k_few_apply(const T* __restrict__ x, long long ldx, const T* __restrict__ W,
                                                   long long ldw, const T* __restrict__ B, long long ldb,
                                                   const int* __restrict__ ids,
                                                   const typename Num<T>::acc* __restrict__ S, int nt, int K, int N,
                                                   int r, int L, typename Num<T>::acc alpha,
                                                   typename Num<T>::acc beta, T* __restrict__ y, long long ldy) {
  typedef typename Num<T>::acc R;
  typedef typename Op<T>::vec V;
  constexpr int E = Op<T>::E, KS = Op<T>::KS, U = G == 1 ? 8 : G == 2 ? 6 : 4;
  __shared__ R red[8][16 * G][17];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, q = lane >> 4, c = lane & 15;
  const int n0 = blockIdx.x * 16;
  const int steps = (K + KS - 1) / KS, each = (steps + 7) / 8;
  const int s0 = min(steps, w * each), s1 = min(steps, s0 + each);
  typename Op<T>::out acc[G];
#pragma unroll
  for (int g = 0; g < G; ++g) acc[g] = typename Op<T>::out{R(0), R(0), R(0), R(0)};
  const T* pw = W + (long long)min(n0 + c, N - 1) * ldw + q * E;
  const T* px[G];
#pragma unroll
  for (int g = 0; g < G; ++g) px[g] = x + (long long)min(16 * g + c, nt - 1) * ldx + q * E;
  const int whole = min(s1, K / KS);  // steps without an end of the rows in them
  int s = s0;
  for (; s + U <= whole; s += U) {
    V a[U], b[U][G];
#pragma unroll
    for (int u = 0; u < U; ++u) a[u] = load_vec(pw + (long long)(s + u) * KS);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int g = 0; g < G; ++g) b[u][g] = load_vec(px[g] + (long long)(s + u) * KS);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int g = 0; g < G; ++g) acc[g] = Op<T>::mma(a[u], b[u][g], acc[g]);
  }
  for (; s < s1; ++s) {
    const int left = K - s * KS - q * E;
    const V a = load_part(pw + (long long)s * KS, left);
#pragma unroll
    for (int g = 0; g < G; ++g) acc[g] = Op<T>::mma(a, load_part(px[g] + (long long)s * KS, left), acc[g]);
  }
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int i = 0; i < 4; ++i) red[w][16 * g + c][out_row<T>(lane, i)] = acc[g][i];
  __syncthreads();
  const int n = n0 + c;
  if (n >= N) return;
  for (int t = tid >> 4; t < nt; t += 32) {
    R v = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) v += red[k][t][c];
    const int l = ids[t];
    if ((unsigned)l < (unsigned)L) {
      const T* b = B + ((long long)l * N + n) * ldb;
      const R* p = S + (long long)t * r;
      for (int j = 0; j < r; j += E) {
        const V f = load_part(b + j, r - j);
#pragma unroll
        for (int i = 0; i < E; ++i)
          if (j + i < r) v = fma(p[j + i], (R)f[i], v);
      }
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
  auto apply = [&](auto kernel) {
    kernel<<<cdiv(g.N, 16), 512, 0, st>>>(X, g.ldx, W, g.ldw, B, g.ldb, ids, S, g.T, g.K, g.N, g.r, g.L, (R)g.alpha, (R)g.beta,
                                          (T*)g.Y, g.ldy);
  };
  if (g.T <= 16) apply(k_few_apply<T, 1>);
  else if (g.T <= 32) apply(k_few_apply<T, 2>);
  else apply(k_few_apply<T, 4>);
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
