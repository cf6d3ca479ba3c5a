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
#include "indexed.h"

namespace {

template <int N> struct Int {
  static constexpr int value = N;
};

constexpr int MAX_E = 4096;  // logits of one token in LDS, in 64 bits
constexpr int MAX_K = 256;
constexpr int MAX_SHARES = 8;
constexpr int ROUTE_WG = 8;  // experts of a router workgroup
constexpr int SLOTS = 512;   // slots of a batch of tokens, and slots times splits that the second product joins in LDS

// Tokens go in batches of at most 64 whose slots fit SLOTS; an expert has at most 64 slots of a batch.
static inline int batch_of(int topk) { return max(1, min(64, SLOTS / topk)); }

// The experts in use in a batch: expert ex[a] has the slots slot[begin[a] .. begin[a + 1]) of tokens token[..]; at[s] is
// slot s's place in `slot`, of[s] its a.  Slots are counted from the batch's first.  (In which order an expert's slots stand is up to
// atomics; nothing depends on it, every slot is a column of its own.)
struct Used {
  int count, ex[SLOTS], begin[SLOTS + 1], slot[SLOTS], token[SLOTS], at[SLOTS], of[SLOTS];
};

// ---------------------------------------------------------------- router
// Two experts per wave; the last workgroup of a token to arrive chooses.  The choice lies next to a border where two
// logits nearly agree, so they are summed in 64 bits: two orders of summation then give the same experts unless the
// logits agree to ~1e-16.  A logit that is NaN counts as the largest (its token's output is NaN either way), so the
// chosen experts are always valid and distinct.
//
// All experts' places at once: an expert's is the number of those before it (larger, or equal with a lower index), the
// comparisons of a group of 64 experts spread over the 4 waves.  (One after the other -- a wave's search for each of k
// places, 64-bit shuffles and exponentials in a chain -- the choice of 8 from 64 took 8 us, the whole router 20.)
// place: E ints of LDS; eid, picked: the chosen experts and their exp(z - top), in order.
template <typename R>
__device__ inline void choose(const double* z, int* place, double* picked, int* eid, double* sums, int E, int topk,
                              int norm, int* ids, R* wt) {
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  auto key = [](double v) { return v != v ? (double)INFINITY : v; };
  for (int e = tid; e < E; e += 256) place[e] = 0;
  __syncthreads();
  const int o0 = E * w / 4, o1 = E * (w + 1) / 4;
  for (int e = lane; e < E; e += 64) {
    const double v = key(z[e]);
    int before = 0;
#pragma unroll 8
    for (int o = o0; o < o1; ++o) {
      const double u = key(z[o]);
      before += u > v || (u == v && o < e);
    }
    if (before) atomicAdd(&place[e], before);
  }
  __syncthreads();
  for (int e = tid; e < E; e += 256)
    if (place[e] < topk) eid[place[e]] = e;
  __syncthreads();
  const double top = z[eid[0]];  // NaN if there is one: every weight of this token is NaN then
  double all = 0;
  for (int j = tid; j < topk; j += 256) picked[j] = exp(z[eid[j]] - top);
  if (!norm) {
    for (int e = tid; e < E; e += 256) all += exp(z[e] - top);
    for (int o = 32; o; o >>= 1) all += __shfl_xor(all, o);
    if (lane == 0) sums[w] = all;
  }
  __syncthreads();
  double part = 0;
  if (norm) {
#pragma unroll 8
    for (int j = 0; j < topk; ++j) part += picked[j];
  } else {
    part = sums[0] + sums[1] + sums[2] + sums[3];
  }
  for (int j = tid; j < topk; j += 256) {
    __hip_atomic_store(&ids[j], eid[j], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the batch's last token
    wt[j] = (R)(picked[j] / part);
  }
}

// Fills a batch's Used from the experts of its n slots.  count, from: E ints of LDS, sums: 4.
__device__ inline void gather(int* count, int* from, int* sums, const int* ids, int n, int topk, int E, Used* u) {
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  for (int e = tid; e < E; e += 256) count[e] = 0;
  __syncthreads();
  int mine[(SLOTS + 255) / 256], place[(SLOTS + 255) / 256];
#pragma unroll
  for (int k = 0; k < (SLOTS + 255) / 256; ++k) {
    const int s = tid + 256 * k;
    if (s >= n) continue;
    mine[k] = __hip_atomic_load(&ids[s], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    place[k] = atomicAdd(&count[mine[k]], 1);
  }
  __syncthreads();
  // experts in use and slots before each expert, one 16-bit half each of a sum over the experts (E / 256 per thread)
  const int per = (E + 255) / 256, e0 = tid * per, e1 = min(E, e0 + per);
  int sum = 0;
  for (int e = e0; e < e1; ++e) sum += count[e] | (count[e] > 0) << 16;
  int upto = sum;
  for (int o = 1; o < 64; o <<= 1) {
    const int b = __shfl_up(upto, o);
    if (lane >= o) upto += b;
  }
  if (lane == 63) sums[w] = upto;
  __syncthreads();
  upto -= sum;
  for (int k = 0; k < w; ++k) upto += sums[k];
  for (int e = e0; e < e1; ++e) {
    from[e] = upto;
    if (count[e]) {
      u->ex[upto >> 16] = e;
      u->begin[upto >> 16] = upto & 0xffff;
    }
    upto += count[e] | (count[e] > 0) << 16;
  }
  if (tid == 255) {
    u->count = upto >> 16;
    u->begin[upto >> 16] = n;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < (SLOTS + 255) / 256; ++k) {
    const int s = tid + 256 * k;
    if (s >= n) continue;
    const int at = (from[mine[k]] & 0xffff) + place[k];
    u->slot[at] = s;
    u->token[at] = s / topk;
    u->at[s] = at;
    u->of[s] = from[mine[k]] >> 16;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void k_moe_route(const T* __restrict__ x, long long ldx, const T* __restrict__ G,
                                                   long long ldg, int H, int E, int topk, int norm, double* zs,
                                                   int* arrived, int* done, int batch, int* __restrict__ ids,
                                                   typename Num<T>::acc* __restrict__ wt, Used* used) {
  constexpr int V = Op<T>::E, P = ROUTE_WG / 4;  // experts per wave
  __shared__ double z[MAX_E], picked[MAX_K], sums[4];
  __shared__ int last, eid[MAX_K], place[MAX_E];
  const int t = blockIdx.y, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int e0 = (blockIdx.x * 4 + w) * P, ne = min(P, E - e0);
  const T* px = x + (long long)t * ldx;
  double s[P] = {};
  if (ne > 0) {
    const T* g[P];
#pragma unroll
    for (int k = 0; k < P; ++k) g[k] = G + (long long)min(e0 + k, E - 1) * ldg;
    auto add = [&](typename Op<T>::vec a, typename Op<T>::vec b, double& sum) {
#pragma unroll
      for (int i = 0; i < V; ++i) sum = fma((double)widen(a[i]), (double)widen(b[i]), sum);
    };
    int h = lane * V;
    for (; h + 3 * 64 * V + V <= H; h += 4 * 64 * V) {
      typename Op<T>::vec a[4], b[4][P];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        a[u] = load_vec(px + h + u * 64 * V);
#pragma unroll
        for (int k = 0; k < P; ++k) b[u][k] = load_vec(g[k] + h + u * 64 * V);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int k = 0; k < P; ++k) add(a[u], b[u][k], s[k]);
    }
    for (; h < H; h += 64 * V) {
      const typename Op<T>::vec a = load_part(px + h, H - h);
#pragma unroll
      for (int k = 0; k < P; ++k) add(a, load_part(g[k] + h, H - h), s[k]);
    }
#pragma unroll
    for (int k = 0; k < P; ++k)
      for (int o = 32; o; o >>= 1) s[k] += __shfl_xor(s[k], o);
  }
  if (gridDim.x > 1) {  // the others' logits come through memory
#pragma unroll
    for (int k = 0; k < P; ++k)
      if (lane == k && k < ne) __hip_atomic_store(&zs[(long long)t * E + e0 + k], s[k], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
      last = __hip_atomic_fetch_add(&arrived[t], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (int)gridDim.x - 1;
      if (last) __hip_atomic_store(&arrived[t], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next run
    }
    __syncthreads();
    if (!last) return;
    for (int e = threadIdx.x; e < E; e += 256) z[e] = __hip_atomic_load(&zs[(long long)t * E + e], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  } else {
#pragma unroll
    for (int k = 0; k < P; ++k)
      if (lane == k && k < ne) z[e0 + k] = s[k];
  }
  __syncthreads();
  choose(z, place, picked, eid, sums, E, topk, norm, ids + (long long)t * topk, wt + (long long)t * topk);
  const int b = t / batch, nt = min(batch, (int)gridDim.y - b * batch);
  if (nt > 1) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
      last = __hip_atomic_fetch_add(&done[b], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == nt - 1;
      if (last) __hip_atomic_store(&done[b], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!last) return;
  } else {  // one token: a slot for each expert
    Used* u = used + b;
    for (int j = threadIdx.x; j <= topk; j += 256) {
      u->begin[j] = j;
      if (j == topk) {
        u->count = topk;
        break;
      }
      u->ex[j] = eid[j];
      u->slot[j] = u->at[j] = u->of[j] = j;
      u->token[j] = 0;
    }
    return;
  }
  gather(place, (int*)z, (int*)sums, ids + (long long)b * batch * topk, nt * topk, topk, E, used + b);
}

template <typename T> struct MoeWs {
  typedef typename Num<T>::acc R;
  int *arrived, *done, *joined, *ids;
  R *wt, *part, *act;
  double* zs;
  Used* used;
  int batch, batches, tiles, shares;
  size_t zero, bytes;
  MoeWs(const MoeArgs& g, void* ws) {
    batch = batch_of(g.topk);
    batches = cdiv(g.T, batch);
    tiles = cdiv(g.H, 16);
    // workgroups that share the second product of 16 rows: about 512 of 8 waves in all
    shares = (int)max(1ll, min((long long)MAX_SHARES, 512 / max(1ll, (long long)tiles * batches)));
    Carve c{(char*)ws};
    const size_t n = (size_t)g.T * g.topk;
    arrived = c.take<int>(g.T);  // counters first: zero before the first run, and left so by every run
    done = c.take<int>(batches);
    joined = c.take<int>((size_t)tiles * batches);
    zero = c.used;
    ids = c.take<int>(n);
    wt = c.take<R>(n);
    zs = c.take<double>((size_t)g.T * g.E);
    used = c.take<Used>(batches);
    part = c.take<R>(shares > 1 ? (size_t)shares * g.T * tiles * 16 : 0);
    act = c.take<R>(n * g.I);
    bytes = c.used;
  }
};

// ---------------------------------------------------------------- first product
// act(slot, i) = silu(g_i) u_i for 16 i of one expert in use: 16 gate and 16 up rows, H split over the waves and joined in
// LDS; G groups of 16 slots at a time (an expert's weights are read again for more than that).
template <typename T, int G, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void k_moe_up(const T* __restrict__ x, long long ldx, const T* __restrict__ W1,
                                                long long ld1, const Used* __restrict__ used, int batch, int topk, int H,
                                                int I, typename Num<T>::acc* __restrict__ act) {
  typedef typename Num<T>::acc R;
  typedef typename Op<T>::vec V;
  constexpr int E = Op<T>::E, KS = Op<T>::KS;
  constexpr int DONE = (4 * G + WAVES - 1) / WAVES;  // results per thread
  __shared__ R red[WAVES][16 * G][17];
  const Used* u = used + blockIdx.z;
  const int a = blockIdx.y, count = u->count, e = u->ex[a], b0 = u->begin[a], total = u->begin[a + 1] - b0;
  asm volatile("" ::"s"(e), "s"(total));  // asked for beside the count, not after its test
  if (a >= count) return;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, q = lane >> 4, c16 = lane & 15;
  const int t0 = blockIdx.z * batch, i0 = blockIdx.x * 16;
  const T* wg = W1 + ((long long)e * 2 * I + min(i0 + c16, I - 1)) * ld1 + q * E;
  const T* wu = wg + (long long)I * ld1;
  const int steps = (H + KS - 1) / KS, s0 = steps * w / WAVES, s1 = steps * (w + 1) / WAVES, whole = min(s1, H / KS);
  for (int skip = 0; skip < total; skip += 16 * G) {
    const int m = min(16 * G, total - skip);
    typename Op<T>::out acc[2][G];
    int token[G], out[DONE];  // out: the slots that this thread finishes
#pragma unroll
    for (int g = 0; g < G; ++g) {
      acc[0][g] = acc[1][g] = typename Op<T>::out{R(0), R(0), R(0), R(0)};
      token[g] = u->token[b0 + skip + min(16 * g + c16, m - 1)];
    }
#pragma unroll
    for (int p = 0; p < DONE; ++p) out[p] = u->slot[b0 + skip + min((tid >> 4) + 4 * WAVES * p, m - 1)];
    // (the tokens' addresses after the weights' loads, which need not wait for them)
    auto px = [&](int g) { return x + (long long)(t0 + token[g]) * ldx + q * E; };
    int s = s0;
    auto run = [&](auto width) {
      constexpr int U = decltype(width)::value;
      V a[U], b[U], v[U][G];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        a[u] = load_vec(wg + (long long)(s + u) * KS);
        b[u] = load_vec(wu + (long long)(s + u) * KS);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int g = 0; g < G; ++g) v[u][g] = load_vec(px(g) + (long long)(s + u) * KS);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int g = 0; g < G; ++g) {
          acc[0][g] = Op<T>::mma(a[u], v[u][g], acc[0][g]);
          acc[1][g] = Op<T>::mma(b[u], v[u][g], acc[1][g]);
        }
      s += U;
    };
    if constexpr (G == 1)
      while (s + 8 <= whole) run(Int<8>());
    if constexpr (G <= 2)
      while (s + 4 <= whole) run(Int<4>());
    while (s + 2 <= whole) run(Int<2>());
    if (s < whole) run(Int<1>());
    for (; s < s1; ++s) {
      const int left = H - s * KS - q * E;
      const V a = load_part(wg + (long long)s * KS, left), b = load_part(wu + (long long)s * KS, left);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const V v = load_part(px(g) + (long long)s * KS, left);
        acc[0][g] = Op<T>::mma(a, v, acc[0][g]);
        acc[1][g] = Op<T>::mma(b, v, acc[1][g]);
      }
    }
    R gate[DONE];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      __syncthreads();
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int v = 0; v < 4; ++v) red[w][16 * g + c16][out_row<T>(lane, v)] = acc[half][g][v];
      __syncthreads();
#pragma unroll
      for (int p = 0; p < DONE; ++p) {
        const int k = tid + 64 * WAVES * p, i = k & 15, sl = k >> 4;
        if (sl >= m) continue;
        R v = 0;
#pragma unroll
        for (int r = 0; r < WAVES; ++r) v += red[r][sl][i];
        if (half == 0) {
          gate[p] = v;
        } else if (i0 + i < I) {
          const long long at = ((long long)t0 * topk + out[p]) * I + i0 + i;
          act[at] = v * (gate[p] / (R(1) + exp(-gate[p])));
        }
      }
    }
  }
}

// `left` steps in batches of MOST and one of what remains (in powers of two that would be up to three ways to memory: fp16,
// 30 experts of 1000 x 728, 24 tokens: 48.7 us with those, 44.7 in one; nothing gained in the first product, whose
// batches fill the registers)
template <int MOST, class F> __device__ inline void in_batches(int left, F run) {
  for (; left >= MOST; left -= MOST) run(Int<MOST>());
  if constexpr (MOST > 4) {
    if (left == 7) run(Int<7>());
    if (left == 6) run(Int<6>());
    if (left == 5) run(Int<5>());
    if (left == 4) run(Int<4>());
  }
  if constexpr (MOST > 2) {
    if (left == 3) run(Int<3>());
    if (left == 2) run(Int<2>());
  }
  if (left == 1) run(Int<1>());
}

// ---------------------------------------------------------------- second product
// y for 16 h and a batch of tokens.  A unit is one (expert in use, split of I); the units are divided evenly over the
// workgroups that share these rows (blockIdx.z) and go round their 8 waves.  A unit leaves its slots' 16 values in LDS,
// each output adds its slots' splits in a fixed order, and the last workgroup of a row tile to arrive adds the shares in
// theirs: which one that is does not change the sum.
template <typename T, int G>
__global__ __launch_bounds__(512, 4) void k_moe_down(const typename Num<T>::acc* __restrict__ act,
                                                  const T* __restrict__ W2, long long ld2,
                                                  const Used* __restrict__ used,
                                                  const typename Num<T>::acc* __restrict__ wt0, int T_, int batch,
                                                  int topk, int H, int I, typename Num<T>::acc alpha,
                                                  typename Num<T>::acc beta, T* __restrict__ y, long long ldy,
                                                  typename Num<T>::acc* share, int* joined) {
  typedef typename Num<T>::acc R;
  typedef typename Op<T>::vec V;
  constexpr int E = Op<T>::E, KS = Op<T>::KS;
  __shared__ R part[SLOTS][17], weight[SLOTS];
  __shared__ short at_of[SLOTS][2];  // a slot's place and expert in use
  __shared__ int last;
  const int tid = threadIdx.x, lane = tid & 63, q = lane >> 4, c16 = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int t0 = blockIdx.y * batch, nt = min(batch, T_ - t0), n = nt * topk, h0 = blockIdx.x * 16;
  const Used* us = used + blockIdx.y;
  const int count = us->count, shares = gridDim.z;
  // splits: a wave for every unit at least; up to 8 while a split keeps 8 steps, so that the waves read neighbouring parts
  // of the same rows at a time (148 -> 135 us for 16 experts of 4096 x 4096)
  const int steps = (I + KS - 1) / KS;
  const int splits = max(1, min(SLOTS / n, max(8 * shares / count, min(8, steps / 8)))), units = count * splits;
  const int u0 = units * (int)blockIdx.z / shares, u1 = units * ((int)blockIdx.z + 1) / shares;
  if (tid < n) {  // for the end, where each would be waited for
    at_of[tid][0] = (short)us->at[tid];
    at_of[tid][1] = (short)us->of[tid];
    weight[tid] = wt0[(long long)t0 * topk + tid];
  }
  for (int unit = u0 + w; unit < u1; unit += 8) {
    const int a = unit / splits, sp = unit % splits;
    const int e = us->ex[a], b0 = us->begin[a], total = us->begin[a + 1] - b0;
    const int s0 = steps * sp / splits, s1 = steps * (sp + 1) / splits, whole = min(s1, I / KS);
    const T* pw = W2 + ((long long)e * H + min(h0 + c16, H - 1)) * ld2 + q * E;
    for (int skip = 0; skip < total; skip += 16 * G) {
      const int m = min(16 * G, total - skip);
      typename Op<T>::out acc[G];
      const R* pa[G];  // a lane's slot's intermediates
#pragma unroll
      for (int g = 0; g < G; ++g) {
        acc[g] = typename Op<T>::out{R(0), R(0), R(0), R(0)};
        pa[g] = act + ((long long)t0 * topk + us->slot[b0 + skip + min(16 * g + c16, m - 1)]) * I + q * E;
      }
      int s = s0;
      auto run = [&](auto width) {  // all loads of a batch before its products: loads are waited for in their order
        constexpr int U = decltype(width)::value;
        V wv[U];
        Mem<T> h[U][G];
#pragma unroll
        for (int u = 0; u < U; ++u) wv[u] = load_vec(pw + (long long)(s + u) * KS);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int g = 0; g < G; ++g) h[u][g].load(pa[g] + (s + u) * KS);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          MidOp<T> f;
          f.set(wv[u]);
#pragma unroll
          for (int g = 0; g < G; ++g) {
            if (g && 16 * g >= m) continue;  // no slot of this unit (48 tokens, 2 of 8 experts of 2048 x 2048: 85 us without, 75)
            Mid<T> p;
            p.set(h[u][g]);
#pragma unroll
            for (int k = 0; k < MidOp<T>::N; ++k) acc[g] = f.product(k, p, acc[g]);
          }
        }
        s += U;
      };
      in_batches<G == 1 ? 8 : G == 2 ? 4 : 2>(whole - s, run);
      for (; s < s1; ++s) {
        const int left = I - s * KS - q * E;
        MidOp<T> f;
        f.set(load_part(pw + (long long)s * KS, left));
#pragma unroll
        for (int g = 0; g < G; ++g) {
          Mem<T> h;
          h.load_to(pa[g] + s * KS, left);
          Mid<T> p;
          p.set(h);
#pragma unroll
          for (int k = 0; k < MidOp<T>::N; ++k) acc[g] = f.product(k, p, acc[g]);
        }
      }
#pragma unroll
      for (int g = 0; g < G; ++g)
        if (16 * g + c16 < m)
#pragma unroll
          for (int v = 0; v < 4; ++v) part[sp * n + b0 + skip + 16 * g + c16][out_row<T>(lane, v)] = acc[g][v];
    }
  }
  __syncthreads();
  auto finish = [&](int t, int h, R v) {
    T* o = &y[(long long)(t0 + t) * ldy + h];
    R r = alpha == R(0) ? R(0) : alpha * v;
    if (beta != R(0)) r += beta * widen(*o);
    *o = (T)r;
  };
  const long long pitch = gridDim.x * 16ll;
  for (int k = tid; k < nt * 16; k += 512) {
    const int h = h0 + (k & 15), t = k >> 4;
    R v = 0;
    for (int j = 0; j < topk; ++j) {
      const int s = t * topk + j, a = at_of[s][1], at = at_of[s][0];
      R sum = 0;
      for (int sp = max(0, u0 - a * splits); sp < min(splits, u1 - a * splits); ++sp) sum += part[sp * n + at][k & 15];
      v += weight[s] * sum;
    }
    if (shares == 1) {
      if (h < H) finish(t, h, v);
    } else {
      __hip_atomic_store(&share[((long long)blockIdx.z * T_ + t0 + t) * pitch + h], v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  if (shares == 1) return;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    int* mine = &joined[blockIdx.y * gridDim.x + blockIdx.x];
    last = __hip_atomic_fetch_add(mine, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == shares - 1;
    if (last) __hip_atomic_store(mine, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!last) return;
  for (int k = tid; k < nt * 16; k += 512) {
    const int h = h0 + (k & 15), t = k >> 4;
    R each[MAX_SHARES], v = 0;
#pragma unroll
    for (int z = 0; z < MAX_SHARES; ++z)  // all asked for before the first is waited for
      each[z] = z < shares ? __hip_atomic_load(&share[((long long)z * T_ + t0 + t) * pitch + h], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : R(0);
#pragma unroll
    for (int z = 0; z < MAX_SHARES; ++z) v += each[z];
    if (h < H) finish(t, h, v);
  }
}

template <typename T> int run(const MoeArgs& g, hipStream_t st) {
  typedef typename Num<T>::acc R;
  MoeWs<T> w(g, g.ws);
  if ((size_t)g.ws_bytes < w.bytes) return -2;
  const T *X = (const T*)g.X, *W1 = (const T*)g.W1, *W2 = (const T*)g.W2;
  const int nb = min(g.T, w.batch) * g.topk, most = min(g.E, nb);
  k_moe_route<T><<<dim3(cdiv(g.E, ROUTE_WG), g.T), 256, 0, st>>>(X, g.ldx, (const T*)g.G, g.ldg, g.H, g.E, g.topk, g.norm, w.zs, w.arrived,
                                                                w.done, w.batch, w.ids, w.wt, w.used);
  // slots of an expert in use, on average: groups of 16 at a time
  const int slots = cdiv(nb, most), groups = slots <= 8 ? 1 : slots <= 24 ? 2 : 4;
  // 8 waves while each has 8 steps (30 experts of 1000 x 728 in fp16: 27.3 us with 8 waves, 27.1 with 4)
  const int waves = g.H >= 64 * Op<T>::KS ? 8 : 4;
  auto up = [&](auto kernel) {
    kernel<<<dim3(cdiv(g.I, 16), most, w.batches), 64 * waves, 0, st>>>(X, g.ldx, W1, g.ld1, w.used, w.batch, g.topk, g.H, g.I, w.act);
  };
  auto down = [&](auto kernel) {
    kernel<<<dim3(w.tiles, w.batches, w.shares), 512, 0, st>>>(w.act, W2, g.ld2, w.used, w.wt, g.T, w.batch, g.topk, g.H, g.I, (R)g.alpha,
                                                             (R)g.beta, (T*)g.Y, g.ldy, w.part, w.joined);
  };
  if (g.I > 0 && waves == 8) groups == 1 ? up(k_moe_up<T, 1, 8>) : groups == 2 ? up(k_moe_up<T, 2, 8>) : up(k_moe_up<T, 4, 8>);
  if (g.I > 0 && waves == 4) groups == 1 ? up(k_moe_up<T, 1, 4>) : groups == 2 ? up(k_moe_up<T, 2, 4>) : up(k_moe_up<T, 4, 4>);
  groups == 1 ? down(k_moe_down<T, 1>) : groups == 2 ? down(k_moe_down<T, 2>) : down(k_moe_down<T, 4>);
  return (int)hipGetLastError();
}

}  // namespace

DPL_API int dpl_moe_args_bytes() { return (int)sizeof(MoeArgs); }

// zero: bytes at its beginning that are zero before the first run
DPL_API long long dpl_moe_ws_bytes(const MoeArgs* g, long long* zero) {
  auto get = [&](auto w) {
    *zero = (long long)w.zero;
    return (long long)w.bytes;
  };
  switch (g->prec) {
    case DPL_S: return get(MoeWs<float>(*g, nullptr));
    case DPL_D: return get(MoeWs<double>(*g, nullptr));
  }
  return get(MoeWs<__bf16>(*g, nullptr));
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
