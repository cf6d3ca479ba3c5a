// A whole mixture-of-experts layer for a few tokens.
//
//   z = G^T x (in 64 bits), p = softmax(z), the top k of z (ties: the lowest index), w = p or p / sum of the chosen p
//   y = alpha sum_j w_j W2_e^T (silu(g) * u) + beta y,      [g; u] = W1_e^T x,  e = the j-th choice
//
// Layouts (element offsets): G[e*ldg + h], W1_e[(e*2I + i)*ld1 + h] (gate rows, then up rows), W2_e[(e*H + h)*ld2 + i],
// X[t*ldx + h], Y[t*ldy + h].  Slot t*k + j is the j-th choice of token t.
#include "indexed.h"

namespace {

constexpr int MAX_E = 4096;  // logits of one token in LDS, in 64 bits

// One workgroup per token.  The choice lies next to a border where two logits nearly agree, so they are summed in 64
// bits: two orders of summation then give the same experts unless the logits agree to ~1e-16.  A logit that is NaN
// counts as the largest (its token's output is NaN either way), so the chosen experts are always valid and distinct.
template <typename T>
__global__ __launch_bounds__(256) void k_moe_route(const T* __restrict__ x, long long ldx, const T* __restrict__ G,
                                                   long long ldg, int H, int E, int topk, int norm,
                                                   int* __restrict__ ids, typename Num<T>::acc* __restrict__ wt) {
  typedef typename Num<T>::acc R;
  __shared__ double z[MAX_E];
  const int t = blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  for (int e = w; e < E; e += 4) {
    double s = 0;
    for (int h = lane; h < H; h += 64) s = fma((double)widen(x[(long long)t * ldx + h]), (double)widen(G[(long long)e * ldg + h]), s);
    for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
    if (lane == 0) z[e] = s;
  }
  __syncthreads();
  if (w) return;
  // softmax denominators over all experts, then over the chosen ones
  double top = -INFINITY;
  for (int e = lane; e < E; e += 64) top = fmax(top, z[e]);
  for (int o = 32; o; o >>= 1) top = fmax(top, __shfl_xor(top, o));
  double sum = 0;
  for (int e = lane; e < E; e += 64) sum += exp(z[e] - top);
  for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
  double chosen = 0;
  unsigned long long taken = 0;  // bit q: expert lane + 64 q of this lane is taken
  for (int pass = 0; pass < 2; ++pass) {
    taken = 0;
    for (int j = 0; j < topk; ++j) {
      double best = 0;
      int at = E;  // nothing yet
      for (int e = lane, q = 0; e < E; e += 64, ++q) {
        if (taken >> q & 1) continue;
        const double v = z[e] != z[e] ? INFINITY : z[e];
        if (at == E || v > best) best = v, at = e;
      }
      for (int o = 32; o; o >>= 1) {
        const double b = __shfl_xor(best, o);
        const int a = __shfl_xor(at, o);
        if (a < E && (at == E || b > best || (b == best && a < at))) best = b, at = a;
      }
      if ((at & 63) == lane) taken |= 1ull << (at >> 6);
      const double p = exp(z[at] - top) / sum;
      if (pass == 0) {
        chosen += p;
      } else if (lane == 0) {
        ids[(long long)t * topk + j] = at;
        wt[(long long)t * topk + j] = (R)(norm ? p / chosen : p);
      }
    }
  }
}

// The slots of expert e, 64 at a time from the `skip`-th on, in slot order; returns how many the expert has in all.
__device__ inline int slots_of(int* list, int* count, const int* ids, int n, int e, int skip) {
  if (threadIdx.x < 64) {
    int have = 0;
    for (int s0 = 0; s0 < n; s0 += 64) {
      const int s = s0 + (int)threadIdx.x;
      const bool mine = s < n && ids[s] == e;
      const unsigned long long m = __ballot(mine);
      const int at = have + __popcll(m & ((1ull << threadIdx.x) - 1)) - skip;
      if (mine && at >= 0 && at < 64) list[at] = s;
      have += __popcll(m);
    }
    if (threadIdx.x == 0) *count = have;
  }
  __syncthreads();
  return *count;
}

// act[slot*I + i] = silu(g_i) u_i for the slots of expert blockIdx.y
template <typename T>
__global__ __launch_bounds__(256) void k_moe_up(const T* __restrict__ x, long long ldx, const T* __restrict__ W1,
                                                long long ld1, const int* __restrict__ ids, int n, int topk, int H,
                                                int I, typename Num<T>::acc* __restrict__ act) {
  typedef typename Num<T>::acc R;
  __shared__ TileLds<R> s;
  __shared__ int list[64], count;
  const int e = blockIdx.y, i0 = blockIdx.x * 64;
  const T* w = W1 + (long long)e * 2 * I * ld1;
  int total = 1;
  for (int skip = 0; skip < total; skip += 64) {
    __syncthreads();
    total = slots_of(list, &count, ids, n, e, skip);
    if (skip >= total) return;
    const int m = min(64, total - skip);
    TileAcc<R> g, u;
    g.zero();
    u.zero();
    for (int half = 0; half < 2; ++half)
      tile_product<true, true>(
          s, half ? u : g, H, [&](int q, int h) { return q < m ? widen(x[(long long)(list[q] / topk) * ldx + h]) : R(0); },
          [&](int i, int h) { return i0 + i < I ? widen(w[(long long)(half * I + i0 + i) * ld1 + h]) : R(0); });
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int q = 0; q < 4; ++q) u.v[a][b][q] *= g.v[a][b][q] / (R(1) + exp(-g.v[a][b][q]));
    u.each([&](int q, int i, R& v) {
      if (q < m && i0 + i < I) act[(long long)list[q] * I + i0 + i] = v;
    });
  }
}

// part[slot*H + h] = sum_i act[slot*I + i] W2_e(h, i)
template <typename T>
__global__ __launch_bounds__(256) void k_moe_down(const typename Num<T>::acc* __restrict__ act,
                                                  const T* __restrict__ W2, long long ld2, const int* __restrict__ ids,
                                                  int n, int H, int I, typename Num<T>::acc* __restrict__ part) {
  typedef typename Num<T>::acc R;
  __shared__ TileLds<R> s;
  __shared__ int list[64], count;
  const int e = blockIdx.y, h0 = blockIdx.x * 64;
  const T* w = W2 + (long long)e * H * ld2;
  int total = 1;
  for (int skip = 0; skip < total; skip += 64) {
    __syncthreads();
    total = slots_of(list, &count, ids, n, e, skip);
    if (skip >= total) return;
    const int m = min(64, total - skip);
    TileAcc<R> acc;
    acc.zero();
    tile_product<true, true>(
        s, acc, I, [&](int q, int i) { return q < m ? act[(long long)list[q] * I + i] : R(0); },
        [&](int h, int i) { return h0 + h < H ? widen(w[(long long)(h0 + h) * ld2 + i]) : R(0); });
    acc.each([&](int q, int h, R& v) {
      if (q < m && h0 + h < H) part[(long long)list[q] * H + h0 + h] = v;
    });
  }
}

template <typename T>
__global__ __launch_bounds__(256) void k_moe_join(const typename Num<T>::acc* __restrict__ part,
                                                  const typename Num<T>::acc* __restrict__ wt, int topk, int H,
                                                  typename Num<T>::acc alpha, typename Num<T>::acc beta,
                                                  T* __restrict__ y, long long ldy) {
  typedef typename Num<T>::acc R;
  const int h = blockIdx.x * 256 + threadIdx.x;
  const long long t = blockIdx.y;
  if (h >= H) return;
  R v = 0;
  for (int j = 0; j < topk; ++j) v += wt[t * topk + j] * part[(t * topk + j) * H + h];
  R o = alpha == R(0) ? R(0) : alpha * v;
  if (beta != R(0)) o += beta * widen(y[t * ldy + h]);
  y[t * ldy + h] = (T)o;
}

template <typename T> struct MoeWs {
  typename Num<T>::acc *wt, *act, *part;
  int* ids;
  size_t bytes;
  MoeWs(const MoeArgs& g, void* ws) {
    Carve c{(char*)ws};
    const size_t n = (size_t)g.T * g.topk;
    ids = c.take<int>(n);
    wt = c.take<typename Num<T>::acc>(n);
    act = c.take<typename Num<T>::acc>(n * g.I);
    part = c.take<typename Num<T>::acc>(n * g.H);
    bytes = c.used;
  }
};

template <typename T> int run(const MoeArgs& g, hipStream_t st) {
  typedef typename Num<T>::acc R;
  MoeWs<T> w(g, g.ws);
  if ((size_t)g.ws_bytes < w.bytes) return -2;
  const T *X = (const T*)g.X, *W1 = (const T*)g.W1, *W2 = (const T*)g.W2;
  const int n = g.T * g.topk;
  k_moe_route<T><<<g.T, 256, 0, st>>>(X, g.ldx, (const T*)g.G, g.ldg, g.H, g.E, g.topk, g.norm, w.ids, w.wt);
  if (g.I > 0) k_moe_up<T><<<dim3(cdiv(g.I, 64), g.E), 256, 0, st>>>(X, g.ldx, W1, g.ld1, w.ids, n, g.topk, g.H, g.I, w.act);
  k_moe_down<T><<<dim3(cdiv(g.H, 64), g.E), 256, 0, st>>>(w.act, W2, g.ld2, w.ids, n, g.H, g.I, w.part);
  k_moe_join<T><<<dim3(cdiv(g.H, 256), g.T), 256, 0, st>>>(w.part, w.wt, g.topk, g.H, (R)g.alpha, (R)g.beta, (T*)g.Y, g.ldy);
  return (int)hipGetLastError();
}

}  // namespace

DPL_API int dpl_moe_args_bytes() { return (int)sizeof(MoeArgs); }

DPL_API long long dpl_moe_ws_bytes(const MoeArgs* g) {
  return (long long)(g->prec == DPL_D ? MoeWs<double>(*g, nullptr).bytes : MoeWs<float>(*g, nullptr).bytes);
}

DPL_API int dpl_moe(const MoeArgs* g, hipStream_t st) {
  if (g->T == 0 || g->H == 0) return 0;
  if (g->E < 1 || g->E > MAX_E || g->topk < 1 || g->topk > g->E) return -1;
  switch (g->prec) {
    case DPL_S: return run<float>(*g, st);
    case DPL_D: return run<double>(*g, st);
    case DPL_H: return run<_Float16>(*g, st);
    case DPL_B: return run<__bf16>(*g, st);
  }
  return -1;
}
