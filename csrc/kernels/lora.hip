// Projection with low-rank adapters of many requests, and its gradient.
//
//   y_t  = alpha (W^T x_t + s_l B_l^T A_l^T x_t) + beta y_t            l = ids[t]; outside 0..L-1: no adapter
//   dx_t = alpha (W dy_t + s_l A_l B_l dy_t)
//   dA_l = alpha s_l sum_{t: ids[t]=l} x_t (B_l dy_t)^T                dB_l = alpha s_l sum_t (A_l^T x_t) dy_t^T
//
// Layouts (element offsets): W[n*ldw + k], X[t*ldx + k], Y[t*ldy + n], A_l[(l*r + j)*lda + k], B_l[(l*N + n)*ldb + j].
//
// Here: the entry points, and the gradient in s and d.  The forward product of few tokens is in lora_few.hip, that of many
// and the low-rank vectors in lora_tile.hip, the gradient in h and b in lora_grad.hip.
//
// Steps: the low-rank vectors S = s_l A_l^T x (and P = s_l B_l dy) of every token into the workspace, then the shared
// product with the adapter's part added to the same accumulators.  Nothing of one adapter ever meets another's token:
// where the rows of a tile use several adapters, each adapter's part is formed apart and kept by a select, so an
// infinity or NaN in one adapter stays with its own tokens.
#include "lora.h"

namespace {

template <typename R> __device__ inline R scale_of(const R* scale, int l) { return scale ? scale[l] : R(1); }

// Adapter ids of 64 rows in LDS, and the rows that name an adapter first.
__device__ inline unsigned long long tile_ids(int* sid, unsigned long long* sfirst, const int* ids, int t0, int T, int L) {
  const int tid = threadIdx.x;
  if (tid < 64) {
    int l = t0 + tid < T ? ids[t0 + tid] : -1;
    if ((unsigned)l >= (unsigned)L) l = -1;
    sid[tid] = l;
    bool first = l >= 0;
    for (int j = 0; j < 64; ++j) {  // every lane of the wave takes part in the shuffle
      const int o = __shfl(l, j);
      if (j < tid && o == l) first = false;
    }
    const unsigned long long m = __ballot(first);
    if (tid == 0) *sfirst = m;
  }
  __syncthreads();
  return *sfirst;
}

// Low-rank vectors: out[t*r + j] = s_l sum_c x[t*ldx + c] F_l(j, c); zero without an adapter.
// SF: F_l(j, c) = F[(l*r + j)*ldf + c] (A), else F[(l*C + c)*ldf + j] (B).
template <typename T, bool SF>
__global__ __launch_bounds__(256) void k_lora_low(const T* __restrict__ x, long long ldx, const T* __restrict__ F,
                                                  long long ldf, const int* __restrict__ ids,
                                                  const typename Num<T>::acc* __restrict__ scale, int nt, int C, int r,
                                                  int L, typename Num<T>::acc* __restrict__ out) {
  typedef typename Num<T>::acc R;
  __shared__ TileLds<R> s;
  __shared__ int sid[64];
  __shared__ unsigned long long sfirst;
  const int t0 = blockIdx.x * 64, j0 = blockIdx.y * 64;
  unsigned long long todo = tile_ids(sid, &sfirst, ids, t0, nt, L);
  TileAcc<R> acc;
  acc.zero();
  acc.each([&](int i, int j, R&) {
    if (t0 + i < nt && j0 + j < r && sid[i] < 0) out[(long long)(t0 + i) * r + j0 + j] = R(0);
  });
  for (; todo; todo &= todo - 1) {
    const int l = sid[__builtin_ctzll(todo)];
    acc.zero();
    const T* f = F + (long long)l * (SF ? r : C) * ldf;
    tile_product<true, SF>(
        s, acc, C, [&](int i, int c) { return t0 + i < nt ? widen(x[(long long)(t0 + i) * ldx + c]) : R(0); },
        [&](int j, int c) {
          return j0 + j < r ? widen(SF ? f[(long long)(j0 + j) * ldf + c] : f[(long long)c * ldf + j0 + j]) : R(0);
        });
    const R sc = scale_of(scale, l);
    acc.each([&](int i, int j, R& v) {
      if (t0 + i < nt && j0 + j < r && sid[i] == l) out[(long long)(t0 + i) * r + j0 + j] = sc * v;
    });
  }
}

// dx[t*ldy + n] = alpha (sum_c x[t*ldx + c] W[c*ldw + n] + sum_j low[t*r + j] F[(l*r + j)*ldf + n]),  x: dy, F: A
template <typename T>
__global__ __launch_bounds__(256) void k_lora_apply(const T* __restrict__ x, long long ldx, const T* __restrict__ W,
                                                    long long ldw, const T* __restrict__ F, long long ldf,
                                                    const int* __restrict__ ids,
                                                    const typename Num<T>::acc* __restrict__ low, int nt, int C, int N,
                                                    int r, int L, typename Num<T>::acc alpha, T* __restrict__ y,
                                                    long long ldy) {
  typedef typename Num<T>::acc R;
  __shared__ TileLds<R> s;
  __shared__ int sid[64];
  __shared__ unsigned long long sfirst;
  const int n0 = blockIdx.x * 64, t0 = blockIdx.y * 64;
  unsigned long long todo = tile_ids(sid, &sfirst, ids, t0, nt, L);
  TileAcc<R> acc, part;
  acc.zero();
  tile_product<true, false>(
      s, acc, C, [&](int i, int c) { return t0 + i < nt ? widen(x[(long long)(t0 + i) * ldx + c]) : R(0); },
      [&](int n, int c) { return n0 + n < N ? widen(W[(long long)c * ldw + n0 + n]) : R(0); });
  for (; todo; todo &= todo - 1) {
    const int l = sid[__builtin_ctzll(todo)];
    part.zero();
    const T* f = F + (long long)l * r * ldf;
    tile_product<true, false>(
        s, part, r,
        [&](int i, int c) { return t0 + i < nt && sid[i] == l ? low[(long long)(t0 + i) * r + c] : R(0); },
        [&](int n, int c) { return n0 + n < N ? widen(f[(long long)c * ldf + n0 + n]) : R(0); });
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int row = (threadIdx.x >> 7) * 32 + i * 16 + Mfma16<R>::row(threadIdx.x & 63, q);
          const R sum = acc.v[i][j][q] + part.v[i][j][q];
          acc.v[i][j][q] = sid[row] == l ? sum : acc.v[i][j][q];
        }
  }
  acc.each([&](int i, int n, R& v) {
    if (t0 + i < nt && n0 + n < N) y[(long long)(t0 + i) * ldy + n0 + n] = (T)(alpha == R(0) ? R(0) : alpha * v);
  });
}

// Tokens in the order of their adapters: off[l] tokens have a smaller adapter id, perm[off[l] ..] lists adapter l's
// tokens in their own order.  One workgroup per adapter reads all ids, so the order never depends on timing.
__global__ __launch_bounds__(256) void k_lora_sort(const int* __restrict__ ids, int nt, int L, int* __restrict__ off,
                                                   int* __restrict__ perm) {
  __shared__ int part[4], base;
  const int l = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  int below = 0;
  for (int t = tid; t < nt; t += 256) {
    const int id = ids[t];
    below += id >= 0 && id < l;
  }
  for (int o = 32; o; o >>= 1) below += __shfl_down(below, o);
  if (lane == 0) part[w] = below;
  __syncthreads();
  if (tid == 0) base = part[0] + part[1] + part[2] + part[3];
  __syncthreads();
  if (tid == 0) off[l] = base;
  for (int t0 = 0; t0 < nt; t0 += 256) {
    const bool mine = t0 + tid < nt && ids[t0 + tid] == l;
    const unsigned long long m = __ballot(mine);
    __syncthreads();  // everybody has read base and part of the round before
    if (lane == 0) part[w] = __popcll(m);
    __syncthreads();
    int at = base;
    for (int v = 0; v < w; ++v) at += part[v];
    if (mine) perm[at + __popcll(m & ((1ull << lane) - 1))] = t0 + tid;
    __syncthreads();
    if (tid == 0) base += part[0] + part[1] + part[2] + part[3];
  }
  __syncthreads();
  if (tid == 0 && l == L - 1) off[L] = base;
}

// Gradient of an adapter's factor: g(j, c) = alpha sum_{t of l} low[t*r + j] z[t*ldz + c];
// JC: out[(l*r + j)*ldo + c] (dA), else out[(l*C + c)*ldo + j] (dB).
template <typename T, bool JC>
__global__ __launch_bounds__(256) void k_lora_outer(const T* __restrict__ z, long long ldz,
                                                    const typename Num<T>::acc* __restrict__ low,
                                                    const int* __restrict__ off, const int* __restrict__ perm, int C,
                                                    int r, typename Num<T>::acc alpha, T* __restrict__ out,
                                                    long long ldo) {
  typedef typename Num<T>::acc R;
  __shared__ TileLds<R> s;
  const int c0 = blockIdx.x * 64, j0 = blockIdx.y * 64, l = blockIdx.z;
  const int first = off[l], n = off[l + 1] - first;
  const int* rows = perm + first;
  TileAcc<R> acc;
  acc.zero();
  tile_product<false, false>(
      s, acc, n, [&](int j, int t) { return j0 + j < r ? low[(long long)rows[t] * r + j0 + j] : R(0); },
      [&](int c, int t) { return c0 + c < C ? widen(z[(long long)rows[t] * ldz + c0 + c]) : R(0); });
  acc.each([&](int j, int c, R& v) {
    if (j0 + j < r && c0 + c < C) {
      const R o = alpha == R(0) ? R(0) : alpha * v;
      out[JC ? ((long long)l * r + j0 + j) * ldo + c0 + c : ((long long)l * C + c0 + c) * ldo + j0 + j] = (T)o;
    }
  });
}

template <typename T> struct PlainWs {
  typename Num<T>::acc *S, *P;
  int *off, *perm;
  size_t bytes;
  PlainWs(const LoraArgs& g, void* ws) {
    Carve c{(char*)ws};
    S = c.take<typename Num<T>::acc>((size_t)g.T * g.r);
    P = c.take<typename Num<T>::acc>((size_t)g.T * g.r);
    off = c.take<int>(g.L + 1);
    perm = c.take<int>(g.T);
    bytes = c.used;
  }
};

template <typename T> int run_grad(const LoraArgs& g, hipStream_t st) {
  typedef typename Num<T>::acc R;
  PlainWs<T> w(g, g.ws);
  if ((size_t)g.ws_bytes < w.bytes) return -2;
  const int tt = cdiv(g.T, 64), rt = cdiv(g.r, 64);
  const T *X = (const T*)g.X, *A = (const T*)g.A, *B = (const T*)g.B, *W = (const T*)g.W, *dY = (const T*)g.dY;
  const int* ids = (const int*)g.ids;
  const R* scale = (const R*)g.scale;
  if (g.L > 0 && g.T > 0) k_lora_low<T, false><<<dim3(tt, rt), 256, 0, st>>>(dY, g.ldy, B, g.ldb, ids, scale, g.T, g.N, g.r, g.L, w.P);
  if (g.dX && g.T > 0 && g.K > 0)
    k_lora_apply<T><<<dim3(cdiv(g.K, 64), tt), 256, 0, st>>>(dY, g.ldy, W, g.ldw, A, g.lda, ids, w.P, g.T, g.N, g.K, g.r, g.L,
                                                             (R)g.alpha, (T*)g.dX, g.lddx);
  if ((g.dA || g.dB) && g.L > 0) {
    k_lora_sort<<<g.L, 256, 0, st>>>(ids, g.T, g.L, w.off, w.perm);
    if (g.dA && g.K > 0)
      k_lora_outer<T, true><<<dim3(cdiv(g.K, 64), rt, g.L), 256, 0, st>>>(X, g.ldx, w.P, w.off, w.perm, g.K, g.r, (R)g.alpha, (T*)g.dA, g.ldda);
    if (g.dB && g.N > 0) {
      if (g.T > 0) k_lora_low<T, true><<<dim3(tt, rt), 256, 0, st>>>(X, g.ldx, A, g.lda, ids, scale, g.T, g.K, g.r, g.L, w.S);
      k_lora_outer<T, false><<<dim3(cdiv(g.N, 64), rt, g.L), 256, 0, st>>>(dY, g.ldy, w.S, w.off, w.perm, g.N, g.r, (R)g.alpha, (T*)g.dB, g.lddb);
    }
  }
  return (int)hipGetLastError();
}

// T > 64: the low-rank vectors, then the shared product that adds the adapters' parts
struct ForwardWs {
  char *hi, *lo;
  int rp;
  size_t bytes;
  ForwardWs(const LoraArgs& g, void* ws) {
    rp = low_pitch(g.prec, g.r);
    const size_t n = (size_t)g.T * rp * mid_bytes(g.prec);
    Carve c{(char*)ws};
    hi = c.take<char>(n);
    lo = c.take<char>(n);
    bytes = c.used;
  }
};

int forward(const LoraArgs& g, hipStream_t st) {
  if (g.T <= 64) return (size_t)g.ws_bytes < lora_few_ws(g) ? -2 : lora_few(g, st);
  ForwardWs w(g, g.ws);
  if ((size_t)g.ws_bytes < w.bytes) return -2;
  const int* ids = (const int*)g.ids;
  if (g.L > 0) {
    const LowArgs a{g.X, g.A, g.scale, ids, g.ldx, g.lda, g.prec, g.T, g.K, g.r, g.L, {w.hi, w.lo, nullptr, nullptr, nullptr, 0, w.rp}};
    const int rc = lora_low(&a, 1, st);
    if (rc) return rc;
  }
  return lora_tile({g.X, g.W, g.B, w.hi, w.lo, ids, g.Y, g.ldx, g.ldw, g.ldb, g.ldy, g.alpha, g.beta, g.prec, g.T, g.K, g.N, g.r, w.rp, g.L}, true, st);
}

}  // namespace

DPL_API int dpl_lora_args_bytes() { return (int)sizeof(LoraArgs); }

DPL_API long long dpl_lora_ws_bytes(const LoraArgs* g, int grad) {
  if (!grad) return (long long)(g->T <= 64 ? lora_few_ws(*g) : ForwardWs(*g, nullptr).bytes);
  switch (g->prec) {
    case DPL_S: return (long long)PlainWs<float>(*g, nullptr).bytes;
    case DPL_D: return (long long)PlainWs<double>(*g, nullptr).bytes;
  }
  return (long long)lora_grad_ws(*g);
}

DPL_API int dpl_lora(const LoraArgs* g, hipStream_t st) { return g->T == 0 || g->N == 0 ? 0 : forward(*g, st); }

DPL_API int dpl_lora_grad(const LoraArgs* g, hipStream_t st) {
  switch (g->prec) {
    case DPL_S: return run_grad<float>(*g, st);
    case DPL_D: return run_grad<double>(*g, st);
    case DPL_H:
    case DPL_B: return lora_grad_half(*g, st);
  }
  return -1;
}
