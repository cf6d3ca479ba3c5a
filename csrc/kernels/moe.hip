// A whole mixture-of-experts layer for a few tokens, in three launches.
//
//   z = G^T x (in 64 bits), p = softmax(z), the top k of z (ties: the lowest index), w = p or p / sum of the chosen p
//   y = alpha sum_j w_j W2_e^T (silu(g) * u) + beta y,      [g; u] = W1_e^T x,  e = the j-th choice
//
// Layouts (element offsets): G[e*ldg + h], W1_e[(e*2I + i)*ld1 + h] (gate rows, then up rows), W2_e[(e*H + h)*ld2 + i],
// X[t*ldx + h], Y[t*ldy + h].  Slot t*k + j is the j-th choice of token t.
//
// The chosen experts' weights are what has to be read: their fragments go from memory straight to the matrix
// instruction (a weight is used by one wave once), the tokens come from the caches.
#include <type_traits>
#include "indexed.h"

namespace {

constexpr int MAX_E = 4096;    // logits of one token in LDS, in 64 bits
constexpr int MAX_K = 256;
constexpr int PARTS = 1024;    // slots times splits of the second product that a workgroup joins in LDS

// ---------------------------------------------------------------- router
// Four experts per wave; the last workgroup of a token to arrive chooses.  The choice lies next to a border where two
// logits nearly agree, so they are summed in 64 bits: two orders of summation then give the same experts unless the
// logits agree to ~1e-16.  A logit that is NaN counts as the largest (its token's output is NaN either way), so the
// chosen experts are always valid and distinct.
template <typename R>
__device__ inline void choose(const double* z, int E, int topk, int norm, int* ids, R* wt) {
  const int lane = threadIdx.x & 63;
  double top = -INFINITY;
  for (int e = lane; e < E; e += 64) top = fmax(top, z[e]);
  for (int o = 32; o; o >>= 1) top = fmax(top, __shfl_xor(top, o));
  double sum = 0;
  for (int e = lane; e < E; e += 64) sum += exp(z[e] - top);
  for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
  double chosen = 0;
  for (int pass = norm ? 0 : 1; pass < 2; ++pass) {
    unsigned long long taken = 0;  // bit q: expert lane + 64 q of this lane is taken
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
        ids[j] = at;
        wt[j] = (R)(norm ? p / chosen : p);
      }
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void k_moe_route(const T* __restrict__ x, long long ldx, const T* __restrict__ G,
                                                   long long ldg, int H, int E, int topk, int norm, double* zs,
                                                   int* arrived, int* __restrict__ ids,
                                                   typename Num<T>::acc* __restrict__ wt) {
  constexpr int V = Op<T>::E;
  __shared__ double z[MAX_E];
  __shared__ int last;
  const int t = blockIdx.y, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int e0 = (blockIdx.x * 4 + w) * 4, ne = min(4, E - e0);
  const T* px = x + (long long)t * ldx;
  double s[4] = {0, 0, 0, 0};
  if (ne > 0) {
    const T* g[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) g[k] = G + (long long)min(e0 + k, E - 1) * ldg;
#pragma unroll 2
    for (int h = lane * V; h < H; h += 64 * V) {
      const typename Op<T>::vec a = load_part(px + h, H - h);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const typename Op<T>::vec b = load_part(g[k] + h, H - h);
#pragma unroll
        for (int i = 0; i < V; ++i) s[k] = fma((double)widen(a[i]), (double)widen(b[i]), s[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      for (int o = 32; o; o >>= 1) s[k] += __shfl_xor(s[k], o);
  }
  if (gridDim.x > 1) {  // the others' logits come through memory
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (lane == k && k < ne) __hip_atomic_store(&zs[(long long)t * E + e0 + k], s[k], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
      last = __hip_atomic_fetch_add(&arrived[t], 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == (int)gridDim.x - 1;
      if (last) __hip_atomic_store(&arrived[t], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next run
    }
    __syncthreads();
    if (!last) return;
    for (int e = threadIdx.x; e < E; e += 256) z[e] = __hip_atomic_load(&zs[(long long)t * E + e], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (lane == k && k < ne) z[e0 + k] = s[k];
  }
  __syncthreads();
  if (w == 0) choose(z, E, topk, norm, ids + (long long)t * topk, wt + (long long)t * topk);
}

// ---------------------------------------------------------------- experts in use
// bits: one for each expert that a slot in ids[0 .. n) names.
template <int THREADS> __device__ inline void mark_experts(unsigned* bits, const int* ids, int n, int E) {
  for (int k = threadIdx.x; k < MAX_E / 32; k += THREADS) bits[k] = 0;
  __syncthreads();
  for (int s = threadIdx.x; s < n; s += THREADS) atomicOr(&bits[ids[s] >> 5], 1u << (ids[s] & 31));
  __syncthreads();
}
// The a-th expert in use (-1: there are fewer) and their number, for a whole wave.
__device__ inline int nth_expert(const unsigned* bits, int a, int& count) {
  const int lane = threadIdx.x & 63;
  const unsigned u = bits[2 * lane], v = bits[2 * lane + 1];
  const int mine = __popc(u) + __popc(v);
  int upto = mine;
  for (int o = 1; o < 64; o <<= 1) {
    const int b = __shfl_up(upto, o);
    if (lane >= o) upto += b;
  }
  count = __shfl(upto, 63);
  int e = -1, skip = a - (upto - mine);
  if (skip >= 0 && skip < mine) {
    unsigned long long m = (unsigned long long)v << 32 | u;
    for (; skip; --skip) m &= m - 1;
    e = 64 * lane + __builtin_ctzll(m);
  }
  const unsigned long long who = __ballot(e >= 0);
  return who ? __shfl(e, __builtin_ctzll(who)) : -1;
}

// The slots of expert e in slot order, the `skip`-th to the (skip + 63)-th into list; returns their number in all.
__device__ inline int slots_of(int* list, const int* ids, int n, int e, int skip) {
  const int lane = threadIdx.x & 63;
  int have = 0;
  for (int s0 = 0; s0 < n; s0 += 64) {
    const int s = s0 + lane;
    const bool mine = s < n && ids[s] == e;
    const unsigned long long m = __ballot(mine);
    const int at = have + __popcll(m & ((1ull << lane) - 1)) - skip;
    if (mine && at >= 0 && at < 64) list[at] = s;
    have += __popcll(m);
  }
  return have;
}

template <typename T> struct MoeWs {
  typedef typename Num<T>::acc R;
  typedef typename Mid<T>::elem M;
  int *arrived, *ids;
  R* wt;
  double* zs;
  M *hi, *lo = nullptr;
  size_t bytes;
  MoeWs(const MoeArgs& g, void* ws) {
    Carve c{(char*)ws};
    const size_t n = (size_t)g.T * g.topk;
    arrived = c.take<int>(g.T);  // first: zero before the first run
    ids = c.take<int>(n);
    wt = c.take<R>(n);
    zs = c.take<double>((size_t)g.T * g.E);
    hi = c.take<M>(n * g.I);
    if (Mid<T>::PARTS == 2) lo = c.take<M>(n * g.I);
    bytes = c.used;
  }
};

// ---------------------------------------------------------------- first product
// act(slot, i) = silu(g_i) u_i for 16 i of one expert in use: 16 gate and 16 up rows, H split over 8 waves and joined in
// LDS; up to G groups of 16 slots at a time.
template <typename T, int G>
__device__ inline void up_product(typename Op<T>::out (&acc)[2][G], const T* x, long long ldx, const T* wg, const T* wu,
                                  const int* list, int m, int topk, int H, int s0, int s1) {
  typedef typename Num<T>::acc R;
  typedef typename Op<T>::vec V;
  constexpr int E = Op<T>::E, KS = Op<T>::KS, U = G == 1 ? 8 : G == 2 ? 4 : 3;
  const int lane = threadIdx.x & 63, q = lane >> 4, c16 = lane & 15;
#pragma unroll
  for (int g = 0; g < G; ++g) acc[0][g] = acc[1][g] = typename Op<T>::out{R(0), R(0), R(0), R(0)};
  const T* px[G];
#pragma unroll
  for (int g = 0; g < G; ++g) px[g] = x + (long long)(list[min(16 * g + c16, m - 1)] / topk) * ldx + q * E;
  const int whole = min(s1, H / KS);
  int s = s0;
  for (; s + U <= whole; s += U) {
    V a[U], b[U], v[U][G];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      a[u] = load_vec(wg + (long long)(s + u) * KS);
      b[u] = load_vec(wu + (long long)(s + u) * KS);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int g = 0; g < G; ++g) v[u][g] = load_vec(px[g] + (long long)(s + u) * KS);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int g = 0; g < G; ++g) {
        acc[0][g] = Op<T>::mma(a[u], v[u][g], acc[0][g]);
        acc[1][g] = Op<T>::mma(b[u], v[u][g], acc[1][g]);
      }
  }
  for (; s < s1; ++s) {
    const int left = H - s * KS - q * E;
    const V a = load_part(wg + (long long)s * KS, left), b = load_part(wu + (long long)s * KS, left);
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const V v = load_part(px[g] + (long long)s * KS, left);
      acc[0][g] = Op<T>::mma(a, v, acc[0][g]);
      acc[1][g] = Op<T>::mma(b, v, acc[1][g]);
    }
  }
}

template <typename T, int GM>
__global__ __launch_bounds__(512) void k_moe_up(const T* __restrict__ x, long long ldx, const T* __restrict__ W1,
                                                long long ld1, const int* __restrict__ ids, int n, int topk, int H,
                                                int I, int E, typename Mid<T>::elem* __restrict__ hi,
                                                typename Mid<T>::elem* __restrict__ lo) {
  typedef typename Num<T>::acc R;
  __shared__ unsigned bits[MAX_E / 32];
  __shared__ int list[64], total;
  __shared__ R red[8][16 * GM][17];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, q = lane >> 4, c16 = lane & 15;
  mark_experts<512>(bits, ids, n, E);
  int used;
  const int e = nth_expert(bits, blockIdx.y, used);
  if (e < 0) return;
  const int i0 = blockIdx.x * 16;
  const T* wg = W1 + ((long long)e * 2 * I + min(i0 + c16, I - 1)) * ld1 + q * Op<T>::E;
  const T* wu = wg + (long long)I * ld1;
  const int steps = (H + Op<T>::KS - 1) / Op<T>::KS, each = (steps + 7) / 8;
  const int s0 = min(steps, w * each), s1 = min(steps, s0 + each);
  for (int skip = 0;; skip += 64) {
    if (w == 0) {
      const int have = slots_of(list, ids, n, e, skip);
      if (lane == 0) total = have;
    }
    __syncthreads();
    const int m = min(64, total - skip);
    auto go = [&](auto width) {
      constexpr int G = decltype(width)::value;
      typename Op<T>::out acc[2][G];
      up_product<T, G>(acc, x, ldx, wg, wu, list, m, topk, H, s0, s1);
      R gate[(16 * 16 * G + 511) / 512];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int v = 0; v < 4; ++v) red[w][16 * g + c16][out_row<T>(lane, v)] = acc[half][g][v];
        __syncthreads();
#pragma unroll
        for (int p = 0; p < (256 * G + 511) / 512; ++p) {
          const int k = tid + 512 * p, i = k & 15, sl = k >> 4;
          if (sl < m) {
            R v = 0;
#pragma unroll
            for (int r = 0; r < 8; ++r) v += red[r][sl][i];
            if (half == 0) {
              gate[p] = v;
            } else if (i0 + i < I) {
              const long long at = (long long)list[sl] * I + i0 + i;
              Mid<T>::put(hi + at, lo + at, v * (gate[p] / (R(1) + exp(-gate[p]))));
            }
          }
        }
        __syncthreads();
      }
    };
    if (m <= 16) go(std::integral_constant<int, 1>());
    else if (GM == 2 || (GM > 2 && m <= 32)) go(std::integral_constant<int, (GM < 2 ? 1 : 2)>());
    else if (GM > 2) go(std::integral_constant<int, GM>());
    if (skip + 64 >= total) return;
    __syncthreads();
  }
}

// ---------------------------------------------------------------- second product
// D[16 h][slots] of one expert over the steps [s0, s1) of I, for m <= 16 G slots
template <typename T, int G>
__device__ inline void down_product(typename Op<T>::out (&acc)[G], const typename Mid<T>::elem* hi,
                                    const typename Mid<T>::elem* lo, const T* pw, const int* list, int m, int I, int s0,
                                    int s1) {
  typedef typename Num<T>::acc R;
  typedef typename Mid<T>::elem M;
  typedef typename Op<T>::vec V;
  typedef typename Op<M>::vec MV;
  constexpr int E = Op<T>::E, KS = Op<T>::KS, U = G == 1 ? 4 : G == 2 ? 2 : 1;
  const int lane = threadIdx.x & 63, q = lane >> 4, c16 = lane & 15;
  long long at[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    acc[g] = typename Op<T>::out{R(0), R(0), R(0), R(0)};
    at[g] = (long long)list[min(16 * g + c16, m - 1)] * I + q * E;
  }
  const int whole = min(s1, I / KS);
  int s = s0;
  for (; s + U <= whole; s += U) {
    V a[U];
    MV h[U][G], l[U][G];
#pragma unroll
    for (int u = 0; u < U; ++u) a[u] = load_vec(pw + (long long)(s + u) * KS);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int g = 0; g < G; ++g) {
        h[u][g] = load_vec(hi + at[g] + (s + u) * KS);
        l[u][g] = Mid<T>::PARTS == 2 ? load_vec(lo + at[g] + (s + u) * KS) : h[u][g];
      }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      MidOp<T> f;
      f.set(a[u]);
#pragma unroll
      for (int g = 0; g < G; ++g) acc[g] = f.mma(h[u][g], l[u][g], acc[g]);
    }
  }
  for (; s < s1; ++s) {
    const int left = I - s * KS - q * E;
    MidOp<T> f;
    f.set(load_part(pw + (long long)s * KS, left));
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const MV h = load_part(hi + at[g] + s * KS, left);
      acc[g] = f.mma(h, Mid<T>::PARTS == 2 ? load_part(lo + at[g] + s * KS, left) : h, acc[g]);
    }
  }
}

// y for 16 h and a batch of tokens: the (expert, split of I) pairs go round the 16 waves, every pair leaves its slots' 16
// values in LDS, and each output adds its slots' and splits' in a fixed order.
template <typename T>
__global__ __launch_bounds__(1024) void k_moe_down(const typename Mid<T>::elem* __restrict__ hi0,
                                                   const typename Mid<T>::elem* __restrict__ lo0,
                                                   const T* __restrict__ W2, long long ld2,
                                                   const int* __restrict__ ids0,
                                                   const typename Num<T>::acc* __restrict__ wt0, int T_, int batch,
                                                   int topk, int H, int I, int E, typename Num<T>::acc alpha,
                                                   typename Num<T>::acc beta, T* __restrict__ y, long long ldy) {
  typedef typename Num<T>::acc R;
  __shared__ unsigned bits[MAX_E / 32];
  __shared__ int list[16][64];
  __shared__ short rank[PARTS];
  __shared__ R part[PARTS][17];
  __shared__ int begin[PARTS + 1];
  const int tid = threadIdx.x, lane = tid & 63, q = lane >> 4, c16 = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int t0 = blockIdx.y * batch, nt = min(batch, T_ - t0), n = nt * topk;
  const int* ids = ids0 + (long long)t0 * topk;
  const typename Mid<T>::elem *hi = hi0 + (long long)t0 * topk * I, *lo = lo0 + (long long)t0 * topk * I;
  const int h0 = blockIdx.x * 16;
  mark_experts<1024>(bits, ids, n, E);
  int used;
  nth_expert(bits, 0, used);
  for (int a = w; a < used; a += 16) {  // slots of each expert in use
    const int m = slots_of(list[w], ids, n, nth_expert(bits, a, used), 0);
    if (lane == 0) begin[a + 1] = m;
  }
  __syncthreads();
  if (w == 0) {  // counts to beginnings, 16 in a lane
    int mine = 0, v[PARTS / 64];
#pragma unroll
    for (int k = 0; k < PARTS / 64; ++k) {
      const int a = lane * (PARTS / 64) + k;
      v[k] = mine += a < used ? begin[a + 1] : 0;
    }
    int upto = mine;
    for (int o = 1; o < 64; o <<= 1) {
      const int b = __shfl_up(upto, o);
      if (lane >= o) upto += b;
    }
    if (lane == 0) begin[0] = 0;
#pragma unroll
    for (int k = 0; k < PARTS / 64; ++k) {
      const int a = lane * (PARTS / 64) + k;
      if (a < used) begin[a + 1] = upto - mine + v[k];
    }
  }
  __syncthreads();
  const int splits = max(1, min(16 / used, PARTS / n));
  const int steps = (I + Op<T>::KS - 1) / Op<T>::KS, each = (steps + splits - 1) / splits;
  for (int unit = w; unit < used * splits; unit += 16) {
    const int a = unit / splits, sp = unit % splits;
    const int e = nth_expert(bits, a, used), b0 = begin[a], m = begin[a + 1] - b0;
    slots_of(list[w], ids, n, e, 0);
    __builtin_amdgcn_wave_barrier();
    const int s0 = min(steps, sp * each), s1 = min(steps, s0 + each);
    const T* pw = W2 + ((long long)e * H + min(h0 + c16, H - 1)) * ld2 + q * Op<T>::E;
    if (sp == 0 && lane < m) rank[list[w][lane]] = (short)(b0 + lane);
    auto go = [&](auto width) {
      constexpr int G = decltype(width)::value;
      typename Op<T>::out acc[G];
      down_product<T, G>(acc, hi, lo, pw, list[w], m, I, s0, s1);
#pragma unroll
      for (int g = 0; g < G; ++g)
        if (16 * g + c16 < m)
#pragma unroll
          for (int v = 0; v < 4; ++v) part[sp * n + b0 + 16 * g + c16][out_row<T>(lane, v)] = acc[g][v];
    };
    if (m <= 16) go(std::integral_constant<int, 1>());
    else if (m <= 32) go(std::integral_constant<int, 2>());
    else go(std::integral_constant<int, 4>());
  }
  __syncthreads();
  for (int k = tid; k < nt * 16; k += 1024) {
    const int h = h0 + (k & 15), t = k >> 4;
    if (h >= H) continue;
    R v = 0;
    for (int j = 0; j < topk; ++j) {
      R s = 0;
      for (int sp = 0; sp < splits; ++sp) s += part[sp * n + rank[t * topk + j]][k & 15];
      v += wt0[(long long)(t0 + t) * topk + j] * s;
    }
    T* o = &y[(long long)(t0 + t) * ldy + h];
    R u = alpha == R(0) ? R(0) : alpha * v;
    if (beta != R(0)) u += beta * widen(*o);
    *o = (T)u;
  }
}

template <typename T> int run(const MoeArgs& g, hipStream_t st) {
  typedef typename Num<T>::acc R;
  MoeWs<T> w(g, g.ws);
  if ((size_t)g.ws_bytes < w.bytes) return -2;
  const T *X = (const T*)g.X, *W1 = (const T*)g.W1, *W2 = (const T*)g.W2;
  const int n = g.T * g.topk;
  k_moe_route<T><<<dim3(cdiv(g.E, 16), g.T), 256, 0, st>>>(X, g.ldx, (const T*)g.G, g.ldg, g.H, g.E, g.topk, g.norm, w.zs, w.arrived, w.ids, w.wt);
  if (g.I > 0) {
    const dim3 grid(cdiv(g.I, 16), min(g.E, n));
    auto up = [&](auto kernel) { kernel<<<grid, 512, 0, st>>>(X, g.ldx, W1, g.ld1, w.ids, n, g.topk, g.H, g.I, g.E, w.hi, w.lo); };
    if (g.T <= 16) up(k_moe_up<T, 1>);
    else if (g.T <= 32) up(k_moe_up<T, 2>);
    else up(k_moe_up<T, 4>);
  }
  const int batch = max(1, min(64, PARTS / g.topk));
  k_moe_down<T><<<dim3(cdiv(g.H, 16), cdiv(g.T, batch)), 1024, 0, st>>>(w.hi, w.lo, W2, g.ld2, w.ids, w.wt, g.T, batch, g.topk, g.H, g.I, g.E,
                                                                      (R)g.alpha, (R)g.beta, (T*)g.Y, g.ldy);
  return (int)hipGetLastError();
}

}  // namespace

DPL_API int dpl_moe_args_bytes() { return (int)sizeof(MoeArgs); }

DPL_API long long dpl_moe_ws_bytes(const MoeArgs* g) {
  switch (g->prec) {
    case DPL_S: return (long long)MoeWs<float>(*g, nullptr).bytes;
    case DPL_D: return (long long)MoeWs<double>(*g, nullptr).bytes;
  }
  return (long long)MoeWs<__bf16>(*g, nullptr).bytes;
}

DPL_API int dpl_moe(const MoeArgs* g, hipStream_t st) {
  if (g->T == 0 || g->H == 0) return 0;
  if (g->E < 1 || g->E > MAX_E || g->topk < 1 || g->topk > g->E || g->topk > MAX_K) return -1;
  switch (g->prec) {
    case DPL_S: return run<float>(*g, st);
    case DPL_D: return run<double>(*g, st);
    case DPL_H: return run<_Float16>(*g, st);
    case DPL_B: return run<__bf16>(*g, st);
  }
  return -1;
}
