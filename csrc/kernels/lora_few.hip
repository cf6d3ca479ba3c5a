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
  const int t = blockIdx.x, j = blockIdx.y * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int l = ids[t];
  if (j >= r) return;
  R s = 0;
  if ((unsigned)l < (unsigned)L) {
    const T* a = A + ((long long)l * r + j) * lda;
    wave_dots<1>(&a, x + (long long)t * ldx, K, &s);
    s *= scale ? scale[l] : R(1);
  }
  if (lane == 0) S[(long long)t * r + j] = s;
}

// One token: rows of W and of its adapter's A against x, one wave per row with its lanes along K (whole lines).  8 waves
// take the workgroup's 8 M features (M: 1 or 2) while 8 others make the low-rank vector, every workgroup for itself: A
// then comes from the caches, and that is less than a second launch and the way of the vector through memory, as long
// as a workgroup has not much more of A to read than of W and one wave's loads of W are enough to fill the memory:
//   2048 x 2048: r 16 5.9 us against 8.9 with two launches, r 64 9.5 us both ways
//   4096 x 4096: r 16 10.6 against 12.9, r 64 14.4 against 13.4;  4096 x 16384, r 8: 46.6 against 31.7
constexpr int ONE_R = 32, ONE_N = 4096;

template <typename T>
__global__ __launch_bounds__(1024) void k_one(const T* __restrict__ x, const T* __restrict__ W, long long ldw,
                                              const T* __restrict__ A, long long lda, const T* __restrict__ B,
                                              long long ldb, const int* __restrict__ ids,
                                              const typename Num<T>::acc* __restrict__ scale, int K, int N, int r, int L,
                                              int M, typename Num<T>::acc alpha, typename Num<T>::acc beta,
                                              T* __restrict__ y) {
  typedef typename Num<T>::acc R;
  __shared__ R low[ONE_R];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int l = L > 0 ? ids[0] : -1;
  const bool has = (unsigned)l < (unsigned)L;
  if (w >= 8) {
    if (has) {
      const T* a = A + (long long)l * r * lda;
      const R f = scale ? scale[l] : R(1);
      for (int j = w - 8; j < r; j += 16) {
        const T* p[2] = {a + j * lda, a + min(j + 8, r - 1) * lda};
        R v[2];
        wave_dots<2>(p, x, K, v);
        if (lane == 0) {
          low[j] = f * v[0];
          if (j + 8 < r) low[j + 8] = f * v[1];
        }
      }
    }
    __syncthreads();
    return;
  }
  const int n = blockIdx.x * M * 8 + w, n2 = M > 1 ? n + 8 : N;
  R v[2] = {0, 0}, f[2] = {0, 0};
  const T* p[2] = {W + min(n, N - 1) * ldw, W + min(n2, N - 1) * ldw};
  if (n2 < N) wave_dots<2>(p, x, K, v);
  else if (n < N) wave_dots<1>(p, x, K, v);
  if (has && lane < r) {
    if (n < N) f[0] = widen(B[((long long)l * N + n) * ldb + lane]);
    if (n2 < N) f[1] = widen(B[((long long)l * N + n2) * ldb + lane]);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int at = i ? n2 : n;
    R u = has && lane < r ? low[lane] * f[i] : R(0);
    for (int o = 32; o; o >>= 1) u += __shfl_xor(u, o);
    if (lane == 0 && at < N) {
      R z = alpha == R(0) ? R(0) : alpha * (v[i] + u);
      if (beta != R(0)) z += beta * widen(y[at]);
      y[at] = (T)z;
    }
  }
}

// 16 NF output features per workgroup, the contraction split over 8 waves and joined in LDS; G groups of 16 tokens.
// W's fragments go straight from memory to the matrix instruction (each element is used by one wave once); what the
// adapters' parts need is asked for before and beside them.  x comes from the caches, and that is what bounds more than
// a few tokens: 16 rows x 64 bytes a load, as the matrix instruction takes it, come out of the L2 at 37 GB/s per CU, whole
// lines at 115 to 130.
//   LINES (x's rows begin at multiples of 16 bytes): x in steps of 128 bytes of a row through a ring of LDS buffers that
//     each wave fills for itself, straight from memory (rows laid out as in k_tile); W four steps ahead in registers.
//   else: x in fragments from any address, in batches as large as the registers of one workgroup per CU allow.
// (T x K x N, us without and with LINES: 48 x 4096 x 8192 30.5, 27.3; 48 x 4096 x 4096 23.0, 16.4; 48 x 1024 x 4096 12.0,
// 10.8; 16 x 4096 x 8192 24.5, 20.5; 16 x 1024 x 4096 9.0, 9.2.)  What is left at 48 x 4096 x 8192: the launch of the
// low-rank vectors, 4 us, and one round of workgroups in which W comes at 3.2 TB/s, 67 MB in 21 us.
constexpr int S_MAX = 64;  // r up to which the low-rank vectors go through LDS

template <typename T, int G, int NF, bool LINES>
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
  constexpr int RING = G == 4 ? 2 : 3, SLOT = G * 2048, RED = 8 * 16 * G * (ROW + 1) * (int)sizeof(R);
  constexpr int MAIN = LINES && 8 * RING * SLOT > RED ? 8 * RING * SLOT : RED;
  __shared__ __attribute__((aligned(1024))) char sm[MAIN + 16 * G * S_MAX * sizeof(R)];
  R* low = (R*)(sm + MAIN);
  R(*red)[16 * G][ROW + 1] = (R(*)[16 * G][ROW + 1])sm;
  const int tid = threadIdx.x, lane = tid & 63, q = lane >> 4, c = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n0 = blockIdx.x * ROW;
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
  if constexpr (LINES) {
    constexpr int BK = 2 * KS, WL = 2 * NF, XL = 2 * G;  // loads of a step
    constexpr unsigned NOWHERE = 0x80000000u;
    const int units = (K + 4 * BK - 1) / (4 * BK), d0 = units * w / 8 * 4, d1 = units * (w + 1) / 8 * 4;
    char* ring = sm + w * RING * SLOT;
    const int xr = lane >> 3, xc = (lane & 7) ^ xr;
    unsigned ox[XL];
#pragma unroll
    for (int k = 0; k < XL; ++k) ox[k] = (unsigned)(min(8 * k + xr, nt - 1) * (int)ldx + xc * E) * sizeof(T);
    const unsigned xbytes = (unsigned)(((nt - 1) * ldx + K) * (long long)sizeof(T));
    auto stage = [&](int d) {  // past K: zeros
      const bool in = d * BK + xc * E < K;
      char* b = ring + d % RING * SLOT;
#pragma unroll
      for (int k = 0; k < XL; ++k) dma_buffer(x, xbytes, b + k * 1024, in ? ox[k] : NOWHERE, d * BK * (int)sizeof(T));
    };
    V a[4][2][NF];
    auto weights = [&](V(*v)[NF], int d) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int f = 0; f < NF; ++f) v[h][f] = load_vec(pw[f] + min((2 * d + h) * KS, K - E - q * E));
    };
    const int fx = c * 128 + ((q ^ (c & 7)) << 4);
    auto step = [&](const V(*v)[NF], int d) {
      const char* b = ring + d % RING * SLOT;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bool in = (2 * d + h) * KS + q * E < K;
        V z[G];
#pragma unroll
        for (int g = 0; g < G; ++g) z[g] = *(const V*)(b + (fx ^ 64 * h) + g * 2048);
#pragma unroll
        for (int f = 0; f < NF; ++f) {
          const V m = keep(v[h][f], in);
#pragma unroll
          for (int g = 0; g < G; ++g) acc[f][g] = Op<T>::mma(m, z[g], acc[f][g]);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    if (d0 < d1) {
      // A step's x is asked for RING - 1 steps ahead, its weights four, and a wait is for the step's x: for all but what
      // was asked for after it.  The first requests come in the order that the counts of the loop expect.
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (u >= 5 - RING) stage(d0 + u - (5 - RING));
        weights(a[u], d0 + u);
      }
      int d = d0;
      for (; d + 8 <= d1; d += 4) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          asm volatile("s_waitcnt vmcnt(%0)" ::"n"(WL + (RING - 2) * (XL + WL)) : "memory");
          step(a[u], d + u);
          stage(d + u + RING - 1);
          weights(a[u], d + u + 4);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      auto last = [&](auto at) {
        constexpr int U = decltype(at)::value;
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(XL * ((U + RING - 2 < 3 ? U + RING - 2 : 3) - U) + WL * (RING - 1 > U ? RING - 1 - U : 0)) : "memory");
        step(a[U], d + U);
        if (U + RING - 1 < 4) stage(d + U + RING - 1);
        __builtin_amdgcn_sched_barrier(0);
      };
      last(Int<0>());
      last(Int<1>());
      last(Int<2>());
      last(Int<3>());
    }
    __syncthreads();  // the rings give way to the join
  } else {
    const int steps = (K + KS - 1) / KS, s0 = steps * w / 8, s1 = steps * (w + 1) / 8, whole = min(s1, K / KS);
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
  if (g.T == 1 && g.r <= ONE_R && g.N <= ONE_N) {
    const int M = g.N <= 8 * 256 ? 1 : 2;  // a workgroup per CU at most
    k_one<T><<<cdiv(g.N, 8 * M), 1024, 0, st>>>(X, W, g.ldw, A, g.lda, B, g.ldb, ids, (const R*)g.scale, g.K, g.N, g.r, g.L, M,
                                               (R)g.alpha, (R)g.beta, (T*)g.Y);
    return (int)hipGetLastError();
  }
  if (g.L > 0) k_few_low<T><<<dim3(g.T, cdiv(g.r, 4)), 256, 0, st>>>(X, g.ldx, A, g.lda, ids, (const R*)g.scale, g.K, g.r, g.L, S);
  // two fragments of features for a fragment of tokens where that leaves a workgroup for every CU: x is read half as often
  // (48 tokens, 4096 x 8192: 32.3 us with one, 27.3 with two; 48 tokens, 4096 x 4096: 16.4 with one, 20.7 with two; 16
  // tokens, 4096 x 8192: 20.5 and 21.8)
  const int nf = sizeof(T) < 8 && g.T > 16 && g.N >= 32 * 256 ? 2 : 1;
  auto apply = [&](auto kernel) {
    kernel<<<cdiv(g.N, 16 * nf), 512, 0, st>>>(X, g.ldx, W, g.ldw, B, g.ldb, ids, S, g.T, g.K, g.N, g.r, g.L, (R)g.alpha, (R)g.beta,
                                          (T*)g.Y, g.ldy);
  };
  const int groups = cdiv(g.T, 16);
  if constexpr (sizeof(T) < 8) {
    const bool lines = ((uintptr_t)X | (uintptr_t)(g.ldx * sizeof(T))) % 16 == 0 && g.K % Op<T>::E == 0 && g.K >= (groups > 1 ? 16 : 64) * Op<T>::KS &&
                       g.ldx * (long long)sizeof(T) * 64 < (1ll << 30);
    auto pick = [&](auto f, auto l) {
      constexpr int F = decltype(f)::value;
      constexpr bool L = decltype(l)::value;
      if constexpr (F == 1) if (groups == 1) return apply(k_few_apply<T, 1, F, L>);
      groups <= 2 ? apply(k_few_apply<T, 2, F, L>) : groups == 3 ? apply(k_few_apply<T, 3, F, L>) : apply(k_few_apply<T, 4, F, L>);
    };
    if (nf == 2) lines ? pick(Int<2>(), Int<1>()) : pick(Int<2>(), Int<0>());
    else lines ? pick(Int<1>(), Int<1>()) : pick(Int<1>(), Int<0>());
  } else {
    groups == 1 ? apply(k_few_apply<T, 1, 1, false>) : groups == 2 ? apply(k_few_apply<T, 2, 1, false>)
    : groups == 3 ? apply(k_few_apply<T, 3, 1, false>) : apply(k_few_apply<T, 4, 1, false>);
  }
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
