// Gradient of gemm_lora.
//
//   P = s B dy, S = s A^T x per token (lora_low);  dX by the shared product with A's part added (lora_tile);
//   dA_l = alpha sum_t x_t p_t^T and dB_l = alpha sum_t s_t dy_t^T by k_outer, over an adapter's tokens in order.
//
// The factors are transposed into the workspace first (L r (K + N) elements, read twice at most afterwards), so that
// every fragment of them is 16 contiguous bytes along its contraction.
#include "lora.h"

namespace {

// ---------------------------------------------------------------- tokens in the order of their adapters; factors turned
// off[l] tokens have a smaller adapter; adapter l's tokens take the places begin_of(l) .. in their own order: perm lists
// them by place, pos is its inverse.  Places begin at multiples of 8 (16 bytes of the low-rank vectors) without any
// workgroup having to know the others' counts: ceil8(off[l]) + 8 l leaves room for every rounding before.
__device__ inline int begin_of(const int* off, int l) { return (off[l] + 7 & ~7) + 8 * l; }

struct PrepareArgs {
  const int* ids;
  int *off, *perm, *pos;
  int4* zero;
  void* low[2];  // places after an adapter's last token, up to a multiple of 8, are zeroed here (null: not in use)
  long long tp;
  int nt, L, r;
  struct Turn {
    const void* src;
    void* dst;
    long long lds;
    int ldd, R, C, wgs;  // per adapter
  } turn[2];
};

// dst[l][c][r] = src[l][r][c], rows of dst padded with zeros to ldd; 64 x 64 elements per workgroup
template <typename T> __device__ inline void turn_tile(const PrepareArgs::Turn& a, long long block) {
  __shared__ T s[64][66];
  const int tr = (a.ldd + 63) / 64;
  const long long m = block / a.wgs;
  const int in = (int)(block % a.wgs), r0 = in % tr * 64, c0 = in / tr * 64, tid = threadIdx.x;
  const T* src = (const T*)a.src;
  T v[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const int r = r0 + (tid >> 6) + 4 * k, c = c0 + (tid & 63);
    v[k] = r < a.R && c < a.C ? src[(m * a.R + r) * a.lds + c] : (T)0;
  }
#pragma unroll
  for (int k = 0; k < 16; ++k) s[(tid >> 6) + 4 * k][tid & 63] = v[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const int c = (tid >> 6) + 4 * k, r = tid & 63;
    if (c0 + c < a.C && r0 + r < a.ldd) ((T*)a.dst)[(m * a.C + c0 + c) * a.ldd + r0 + r] = s[r][c];
  }
}

// One workgroup per adapter reads all ids, each wave a run of them, so the order never depends on timing.  64 ids at a time,
// 16 times that under way (the launch with 13416 ids: 23 us with a run for each thread, 12 so).
template <typename R> __device__ inline void sort_one(const PrepareArgs& a, int l) {
  __shared__ int sums[2][4];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (l == 0 && tid == 0) *a.zero = int4{0, 0, 0, 0};
  const int each = ((a.nt + 3) / 4 + 63) / 64 * 64, t0 = min(a.nt, w * each), t1 = min(a.nt, t0 + each);
  constexpr int U = 16;
  auto scan = [&](auto f) {
    for (int t = t0 + lane; t - lane < t1; t += 64 * U) {
      int id[U];
#pragma unroll
      for (int u = 0; u < U; ++u) id[u] = t + 64 * u < t1 ? a.ids[t + 64 * u] : -1;
#pragma unroll
      for (int u = 0; u < U; ++u) f(id[u], t + 64 * u);
    }
  };
  int below = 0, mine = 0;
  scan([&](int id, int) {
    below += __popcll(__ballot(id >= 0 && id < l));
    mine += __popcll(__ballot(id == l));
  });
  if (lane == 0) {
    sums[0][w] = mine;
    sums[1][w] = below;
  }
  __syncthreads();
  const int first = sums[1][0] + sums[1][1] + sums[1][2] + sums[1][3];
  const int count = sums[0][0] + sums[0][1] + sums[0][2] + sums[0][3];
  if (tid == 0) {
    a.off[l] = first;
    if (l == a.L - 1) a.off[l + 1] = first + count;
  }
  const int begin = (first + 7 & ~7) + 8 * l;
  int at = begin;
  for (int k = 0; k < w; ++k) at += sums[0][k];
  if (mine)
    scan([&](int id, int t) {
      const unsigned long long m = __ballot(id == l);
      if (id == l) {
        const int place = at + __popcll(m & ((1ull << lane) - 1));
        a.perm[place] = t;
        a.pos[t] = place;
      }
      at += __popcll(m);
    });
  const int end = begin + count, pad = (8 - count % 8) % 8;
  for (int k = 0; k < 2; ++k)
    if (a.low[k])
      for (int i = tid; i < a.r * pad; i += 256) ((R*)a.low[k])[(i / pad) * a.tp + end + i % pad] = R(0);
}

template <typename T> __global__ __launch_bounds__(256) void k_prepare(PrepareArgs a) {
  const long long first = (long long)a.turn[0].wgs * a.L, all = a.L + first + (long long)a.turn[1].wgs * a.L;
  for (long long b = blockIdx.x; b < all; b += gridDim.x) {
    if (b < a.L) sort_one<typename Num<T>::acc>(a, (int)b);
    else if (b - a.L < first) turn_tile<T>(a.turn[0], b - a.L);
    else turn_tile<T>(a.turn[1], b - a.L - first);
    __syncthreads();
  }
}

// ---------------------------------------------------------------- gradients of the factors
// g_l(j, c) = alpha sum_{t of l} low(t, j) z[t*ldz + c].  An item is the part of one adapter's places that lies in one
// window of `win`; the items of windows and adapters are counted through (window + adapter).  An adapter inside one window
// is finished here (one without tokens gets its zeros), others leave 32-bit parts that k_join adds in the order of the
// windows: slot 2 w for the adapter that came in from window w - 1, 2 w + 1 for one that begins in w and goes on.
// COLS columns per workgroup, 16 JF rows j.  Steps of 128 bytes of tokens go through a ring of LDS buffers: z as
// [token][column], read across as W is in k_tile, low as [j][token] (both laid out as there; a step of h and b holds twice
// 128 bytes of low, one such block for each of its two products).
struct OuterSet {
  const void *z, *low;  // low: by adapter
  void *out, *part;
  long long ldz, ldo;
  int C, win, items, jc;  // jc: g is stored [j][c] (dA), else [c][j] (dB)
};
struct OuterArgs {
  OuterSet set[2];
  const int *off, *perm;
  const int4* zero;
  long long tp;
  double alpha;
  int r, L, wgs0;  // workgroups of the first set
};

constexpr int COLS = 256, WIN_MAX = 2048;

template <typename T, int JF, bool DMA> __global__ __launch_bounds__(256, 1) void k_outer(OuterArgs a) {
  typedef typename Num<T>::acc R;
  typedef typename Op<T>::vec V;
  constexpr int E = Op<T>::E, STEP = 2 * Op<T>::KS;  // tokens of a step
  constexpr int EL = 16 / (int)sizeof(R);            // tokens of a chunk of low
  constexpr int CH = COLS / E, J = STEP * CH / 256;  // chunks of a row of z; of them per thread
  // WJ x 4 / WJ waves of 16 JW rows j x 16 FN columns.  Every wave takes the numbers of low that it uses apart for itself,
  // which with all of 64 rows is the longest part of a step in b: there two waves along j halve it (the whole gradient of
  // 8192 tokens, 4096 and 16384 features, 8 adapters: 1103 us with one, 1083 with two).  In h z's numbers are taken apart
  // too, and no division saves anything
  constexpr int WJ = JF == 4 && __is_same(T, __bf16) ? 2 : 1, JW = JF / WJ, FN = COLS / 64 * WJ;
  constexpr int BLOCKS = STEP / (8 * EL), PARTS = JF == 1 ? 2 : BLOCKS;  // (one of 16 rows is half a load of the workgroup: taken twice)
  constexpr int ZB = STEP * COLS * (int)sizeof(T), PB = JF * 16 * 128, STAGE = ZB + PARTS * PB, RING = DMA ? (JF == 1 ? 4 : 3) : 2;
  constexpr int PJ = PARTS * PB / 4096, LOADS = J + PJ;
  __shared__ __attribute__((aligned(1024))) char sm[RING * STAGE + WIN_MAX * sizeof(int)];
  int* rows = (int*)(sm + RING * STAGE);
  const bool second = (int)blockIdx.x >= a.wgs0;
  const OuterSet& g = a.set[second];
  const int block = second ? blockIdx.x - a.wgs0 : blockIdx.x;
  const int ct = (g.C + COLS - 1) / COLS, item = block / ct;
  const int c0 = block % ct * COLS, j0 = blockIdx.y * 16 * JF;
  const int tid = threadIdx.x, lane = tid & 63, q = lane >> 4, c16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wj = WJ > 1 ? wave & 1 : 0, wc = WJ > 1 ? wave >> 1 : wave;
  int l = 0;
  for (int hi = a.L - 1; l < hi;) {  // the largest adapter whose first item is not past this one
    const int mid = (l + hi + 1) >> 1;
    if (begin_of(a.off, mid) / g.win + mid <= item) l = mid;
    else hi = mid - 1;
  }
  const int w = item - l, lo = begin_of(a.off, l), count = a.off[l + 1] - a.off[l], end = lo + count;
  T* out = (T*)g.out;
  // (copies: a pointer chosen per lane from the arguments would be loaded again, and waited for, in every step)
  const T* z = (const T*)g.z;
  const R* low = (const R*)g.low;
  const void* zero = a.zero;
  const long long ldz = g.ldz, tp = a.tp;
  const int C = g.C, r = a.r;
  auto where = [&](int j, int c) { return g.jc ? ((long long)l * a.r + j) * g.ldo + c : ((long long)l * g.C + c) * g.ldo + j; };
  if (count == 0) {
    if (w == lo / g.win)
      for (int i = tid; i < 16 * JF * COLS; i += 256) {
        const int j = j0 + (g.jc ? i / COLS : i % (16 * JF)), c = c0 + (g.jc ? i % COLS : i / (16 * JF));
        if (j < a.r && c < g.C) out[where(j, c)] = (T)0;
      }
    return;
  }
  const int p0 = max(lo, w * g.win), p1 = min(end, (w + 1) * g.win), n = p1 - p0;
  if (n <= 0) return;
  for (int k = tid; k < n; k += 256) rows[k] = a.perm[p0 + k];
  __syncthreads();
  auto chunk = [](int row, int pc) {
    const int turn = (row & 3) + 4 * ((row >> 3) & 1);
    return sizeof(T) == 2 ? 2 * ((pc >> 1) ^ turn) + (pc & 1) : pc ^ (16 / E * (row / E & 3));
  };
  const int sr = tid / CH, pc = tid % CH;
  V v[DMA ? 1 : J];
  auto stage_low = [&](char* b, int s) {
#pragma unroll
    for (int k = 0; k < PJ; ++k) {
      const int id = tid + 256 * k, pt = BLOCKS > 1 ? id / (PB / 16) : 0, row = id % (PB / 16) >> 3;
      const int at = s + 8 * EL * pt + EL * ((id & 7) ^ (row & 7));
      const R* src = low + min(j0 + row, r - 1) * tp + p0 + at;
      dma_global(at < n ? (const void*)src : zero, b + ZB + wave * 1024 + k * 4096);
    }
  };
  int token[J];  // of the next step's rows
  auto look = [&](int s) {
#pragma unroll
    for (int k = 0; k < J; ++k) token[k] = rows[min(s + sr + k * (256 / CH), n - 1)];
  };
  look(0);
  auto stage = [&](int s) {
    char* b = &sm[s / STEP % RING * STAGE];
#pragma unroll
    for (int k = 0; k < J; ++k) {
      const int row = sr + k * (256 / CH), t = s + row;
      const int c = c0 + chunk(row, pc) * E;
      if constexpr (DMA) {
        const void* p = t < n && c < C ? (const void*)(z + (long long)token[k] * ldz + c) : zero;
        dma_global(p, b + wave * 1024 + k * 4096);
      } else {
        v[k] = load_part(z + (t < n ? (long long)token[k] * ldz + c : 0), t < n ? C - c : 0);
      }
    }
    stage_low(b, s);
    look(s + STEP);
  };
  auto put = [&](int s) {
    char* b = &sm[s / STEP % RING * STAGE];
#pragma unroll
    for (int k = 0; k < J; ++k) *(V*)(b + (tid + 256 * k) * 16) = v[k];
  };
  typename Op<T>::out acc[JW][FN];
#pragma unroll
  for (int i = 0; i < JW; ++i)
#pragma unroll
    for (int f = 0; f < FN; ++f) acc[i][f] = typename Op<T>::out{R(0), R(0), R(0), R(0)};
  const int ftr = (8 * q + (c16 >> 2)) * (COLS * 2) + (c16 & 3) * 8;
  const int tw = (c16 >> 2) + 4 * (q & 1);
  const int fp = ZB + wj * JW * 2048 + c16 * 128 + (((BLOCKS > 1 ? 2 * q : q) ^ (c16 & 7)) << 4);
  auto multiply = [&](int s) {
    const char* b = &sm[s / STEP % RING * STAGE];
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      Mid<T> part[JW];
#pragma unroll
      for (int i = 0; i < JW; ++i) {
        Mem<T> mem;
        if constexpr (BLOCKS > 1) {
          mem.v[0] = *(const f4_t*)(b + fp + kk * PB + i * 2048);
          mem.v[1] = *(const f4_t*)(b + (fp ^ 16) + kk * PB + i * 2048);
        } else {
          mem.v = *(const V*)(b + (fp ^ (64 * kk)) + i * 2048);
        }
        part[i].set(mem);
      }
      MidOp<T> x[FN];
#pragma unroll
      for (int f = 0; f < FN; ++f) {
        V across;
        if constexpr (sizeof(T) == 2) {
          typedef short s8_t __attribute__((ext_vector_type(8)));
          const char* p = b + ftr + (((wc * FN + f) ^ tw) << 5) + kk * 32 * COLS * 2;
          const s4_t v0 = read_turned(p), v1 = read_turned(p + 4 * COLS * 2);
          const s8_t both = __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
          across = __builtin_bit_cast(V, both);
        } else {
#pragma unroll
          for (int e = 0; e < E; ++e)
            across[e] = *(const T*)(b + ((kk * Op<T>::KS + q * E + e) * COLS + ((wc * FN + f) ^ q) * 16 + c16) * (int)sizeof(T));
        }
        x[f].set(across);
      }
#pragma unroll
      for (int k = 0; k < MidOp<T>::N; ++k)
#pragma unroll
        for (int f = 0; f < FN; ++f)
#pragma unroll
          for (int i = 0; i < JW; ++i) acc[i][f] = x[f].product_first(k, part[i], acc[i][f]);
    }
  };
  auto meet = [&]() {
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  if constexpr (DMA) {
#pragma unroll
    for (int k = 0; k < RING - 1; ++k) stage(STEP * k);  // past the last token: zeros
    for (int s = 0; s < n; s += STEP) {
      // this step has arrived, and every wave has read the one before, whose buffer is filled next
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LOADS * (RING - 2)) : "memory");
      meet();
      stage(s + STEP * (RING - 1));
      multiply(s);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // nothing is on its way to LDS when the workgroup ends
  } else {
    stage(0);
    put(0);
    for (int s = 0; s < n; s += STEP) {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      meet();
      if (s + STEP < n) stage(s + STEP);
      multiply(s);
      if (s + STEP < n) put(s + STEP);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }
  const bool whole = lo / g.win == (end - 1) / g.win;
  const R alpha = (R)a.alpha;
  R* part = (R*)g.part + (long long)(2 * w + (lo >= w * g.win)) * a.r * g.C;
#pragma unroll
  for (int f = 0; f < FN; ++f) {
    const int c = c0 + (wc * FN + f) * 16 + c16;
    if (c >= g.C) continue;
#pragma unroll
    for (int i = 0; i < JW; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int j = j0 + 16 * (wj * JW + i) + out_row<T>(lane, k);
        if (j >= a.r) continue;
        if (whole) out[where(j, c)] = (T)(alpha == R(0) ? R(0) : alpha * acc[i][f][k]);
        else part[g.jc ? (long long)j * g.C + c : (long long)c * a.r + j] = acc[i][f][k];
      }
  }
}

// Parts of the adapters that go over several windows, added in the windows' order.
template <typename T> __global__ __launch_bounds__(256) void k_join(OuterArgs a) {
  typedef typename Num<T>::acc R;
  const OuterSet& g = a.set[blockIdx.z];
  const int l = blockIdx.y, lo = begin_of(a.off, l), count = a.off[l + 1] - a.off[l];
  if (!g.out || count == 0) return;
  const int w0 = lo / g.win, w1 = (lo + count - 1) / g.win;
  if (w0 == w1) return;
  const long long n = (long long)a.r * g.C;
  const int width = g.jc ? g.C : a.r;
  const R alpha = (R)a.alpha;
  for (long long e = blockIdx.x * 256ll + threadIdx.x; e < n; e += gridDim.x * 256ll) {
    R v = 0;
#pragma unroll 4
    for (int w = w0; w <= w1; ++w) v += ((const R*)g.part)[(2 * w + (w == w0)) * n + e];
    ((T*)g.out)[((long long)l * (n / width) + e / width) * g.ldo + e % width] = (T)(alpha == R(0) ? R(0) : alpha * v);
  }
}

// places in all, and a window's length: both factors have (windows + adapters) workgroups for each of their tiles of columns
// and ranks, one to a CU (the buffers take most of its LDS).  The windows alone are to make about 192 of them, in whole
// steps, as far as WIN_MAX allows, whose tokens lie in LDS: with few adapters one round of the CUs and few parts to join
// (4096 tokens, 4096 features, r 16, one adapter: 192 workgroups).  With many it is more: 8192 tokens, 4096 and 16384 features,
// 8 adapters are 4 windows of 2048 and 12 items for 80 tiles, 960 workgroups in nearly four rounds.  Few tokens stay in one
// window, which needs no join.  (us of the whole gradient so, and with 1024 in the place of 192: 8192 tokens, r 64, as above
// 1073, 1099; 4096 tokens, 4096 features, r 16 156, 161; 2048 tokens, 2048 features, r 32, 4 adapters 61, 60.)
long long places(const LoraArgs& g) { return cdiv(g.T, 8) * 8ll + 8ll * (g.L + 1); }
int window(const LoraArgs& g) {
  if (places(g) <= 512) return 512;
  const long long tiles = (long long)(cdiv(g.K, COLS) + cdiv(g.N, COLS)) * cdiv(g.r, 64);
  return (int)min((long long)WIN_MAX, max(256ll, (g.T * tiles / 192 + 63) / 64 * 64));
}

template <typename T> struct GradWs {
  int *off, *perm, *pos;
  typedef typename Num<T>::acc R;
  R *p = nullptr, *pt = nullptr, *st = nullptr;  // P by token, P and S by adapter
  T *At = nullptr, *Bt = nullptr;
  int4* zeros;
  R *pa = nullptr, *pb = nullptr;
  bool dx, da, db;
  int rp, ldb, win;
  long long tp;
  size_t bytes;
  GradWs(const LoraArgs& g, void* ws) {
    dx = g.dX && g.K > 0 && g.T > 0;
    da = g.dA && g.K > 0 && g.L > 0;
    db = g.dB && g.N > 0 && g.L > 0;
    rp = low_pitch(g.prec, g.r);
    ldb = cdiv(g.N, 8) * 8;
    tp = (places(g) + 63) / 64 * 64 + 64;
    win = window(g);
    Carve c{(char*)ws};
    zeros = c.take<int4>(1);
    off = c.take<int>(g.L + 1);
    perm = c.take<int>(places(g));
    pos = c.take<int>(g.T);
    if (dx) {
      p = c.take<R>((size_t)g.T * rp);
      At = c.take<T>((size_t)g.L * g.K * rp);
    }
    if (dx || da) Bt = c.take<T>((size_t)g.L * g.r * ldb);
    if (da) {
      pt = c.take<R>(g.r * tp);
      pa = c.take<R>((size_t)2 * (places(g) / win + 1) * g.r * g.K);
    }
    if (db) {
      st = c.take<R>(g.r * tp);
      pb = c.take<R>((size_t)2 * (places(g) / win + 1) * g.r * g.N);
    }
    bytes = c.used;
  }
};

template <typename T> int run(const LoraArgs& g, hipStream_t st) {
  GradWs<T> w(g, g.ws);
  if ((size_t)g.ws_bytes < w.bytes) return -2;
  const int* ids = (const int*)g.ids;
  const bool low = g.L > 0 && g.T > 0, p = low && (w.dx || w.da), s = low && w.db;
  if (g.L > 0) {
    PrepareArgs a{ids, w.off, w.perm, w.pos, w.zeros, {w.pt, w.st}, w.tp, g.T, g.L, g.r, {}};
    if (p && g.N > 0) a.turn[0] = {g.B, w.Bt, g.ldb, w.ldb, g.N, g.r, cdiv(w.ldb, 64) * cdiv(g.r, 64)};
    if (low && w.dx) a.turn[1] = {g.A, w.At, g.lda, w.rp, g.r, g.K, cdiv(w.rp, 64) * cdiv(g.K, 64)};
    k_prepare<T><<<(unsigned)min(1ll << 20, g.L * (1ll + a.turn[0].wgs + a.turn[1].wgs)), 256, 0, st>>>(a);
  }
  int rc = 0;
  if (p || s) {
    LowArgs a[2];
    int n = 0;
    if (p)
      a[n++] = {g.dY, w.Bt, g.scale, ids, g.ldy, w.ldb, g.prec, g.T, g.N, g.r, g.L,
                {w.p, w.pt, w.pos, w.tp, w.rp}};
    if (s)
      a[n++] = {g.X, g.A, g.scale, ids, g.ldx, g.lda, g.prec, g.T, g.K, g.r, g.L,
                {nullptr, w.st, w.pos, w.tp, g.r}};
    rc = lora_low(a, n, st);
  }
  if (!rc && w.dx)
    rc = lora_tile({g.dY, g.W, w.At, w.p, ids, g.dX, g.ldy, g.ldw, w.rp, g.lddx, g.alpha, 0.0, g.prec, g.T, g.N, g.K, g.r, w.rp, g.L}, false, st);
  if (rc || !(w.da || w.db)) return rc;
  OuterArgs a{{}, w.off, w.perm, w.zeros, w.tp, g.alpha, g.r, g.L, 0};
  auto wgs = [&](const OuterSet& o) { return o.out ? cdiv(o.C, COLS) * o.items : 0; };
  if (w.da) a.set[0] = {g.X, w.pt, g.dA, w.pa, g.ldx, g.ldda, g.K, w.win, (int)(places(g) / w.win) + g.L, 1};
  if (w.db) a.set[1] = {g.dY, w.st, g.dB, w.pb, g.ldy, g.lddb, g.N, w.win, (int)(places(g) / w.win) + g.L, 0};
  a.wgs0 = wgs(a.set[0]);
  auto aligned = [&](const OuterSet& o) { return !o.out || (((uintptr_t)o.z | (uintptr_t)(o.ldz * sizeof(T))) % 16 == 0 && o.C % Op<T>::E == 0); };
  const bool dma = aligned(a.set[0]) && aligned(a.set[1]);
  const int jf = g.r <= 16 ? 1 : g.r <= 32 ? 2 : 4;
  const dim3 grid((unsigned)(a.wgs0 + wgs(a.set[1])), cdiv(g.r, 16 * jf));
  auto go = [&](auto kernel) { kernel<<<grid, 256, 0, st>>>(a); };
  if (jf == 1) dma ? go(k_outer<T, 1, true>) : go(k_outer<T, 1, false>);
  else if (jf == 2) dma ? go(k_outer<T, 2, true>) : go(k_outer<T, 2, false>);
  else dma ? go(k_outer<T, 4, true>) : go(k_outer<T, 4, false>);
  if (places(g) > w.win) {
    const long long most = (long long)g.r * max(w.da ? g.K : 0, w.db ? g.N : 0);
    k_join<T><<<dim3((unsigned)min(512ll, (most + 255) / 256), g.L, 2), 256, 0, st>>>(a);
  }
  return (int)hipGetLastError();
}

}  // namespace

size_t lora_grad_ws(const LoraArgs& g) {
  switch (g.prec) {
    case DPL_S: return GradWs<float>(g, nullptr).bytes;
    case DPL_D: return GradWs<double>(g, nullptr).bytes;
  }
  return GradWs<__bf16>(g, nullptr).bytes;
}

int lora_grad(const LoraArgs& g, hipStream_t st) {
  switch (g.prec) {
    case DPL_S: return run<float>(g, st);
    case DPL_D: return run<double>(g, st);
    case DPL_H: return run<_Float16>(g, st);
    case DPL_B: return run<__bf16>(g, st);
  }
  return -1;
}
