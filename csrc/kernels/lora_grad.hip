// Gradient of gemm_lora in the half precisions.
//
//   P = s B dy, S = s A^T x per token (lora_low);  dX by the shared product with A's part added (lora_tile);
//   dA_l = alpha sum_t x_t p_t^T and dB_l = alpha sum_t s_t dy_t^T by k_outer, over an adapter's tokens in order.
//
// The factors are transposed into the workspace first (L r (K + N) elements, read twice at most afterwards), so that
// every fragment of them is 16 contiguous bytes along its contraction.
#include "lora.h"

namespace {

// ---------------------------------------------------------------- tokens in the order of their adapters
// off[l] tokens have a smaller adapter, perm[off[l] ..] lists adapter l's tokens in their own order, pos is its inverse.
// One workgroup per adapter reads all ids, so the order never depends on timing.
__global__ __launch_bounds__(256) void k_sort(const int* __restrict__ ids, int nt, int L, int* __restrict__ off,
                                              int* __restrict__ perm, int* __restrict__ pos, int4* __restrict__ zero) {
  __shared__ int part[4], base;
  const int l = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  if (l == 0 && tid == 0) *zero = int4{0, 0, 0, 0};
  int below = 0;
  for (int t = tid; t < nt; t += 256) {
    const int id = ids[t];
    below += id >= 0 && id < l;
  }
  for (int o = 32; o; o >>= 1) below += __shfl_xor(below, o);
  if (lane == 0) part[w] = below;
  __syncthreads();
  if (tid == 0) base = part[0] + part[1] + part[2] + part[3];
  __syncthreads();
  int at0 = base;
  if (tid == 0) off[l] = at0;
  for (int t0 = 0; t0 < nt; t0 += 256) {
    const bool mine = t0 + tid < nt && ids[t0 + tid] == l;
    const unsigned long long m = __ballot(mine);
    __syncthreads();
    if (lane == 0) part[w] = __popcll(m);
    __syncthreads();
    int at = at0;
    for (int v = 0; v < w; ++v) at += part[v];
    at += __popcll(m & ((1ull << lane) - 1));
    if (mine) {
      perm[at] = t0 + tid;
      pos[t0 + tid] = at;
    }
    at0 += part[0] + part[1] + part[2] + part[3];
  }
  if (tid == 0 && l == L - 1) off[L] = at0;
}

// dst[m][c][r] = src[m][r][c], rows of dst padded with zeros to ldd; 64 x 64 elements per workgroup
template <typename T>
__global__ __launch_bounds__(256) void k_turn(const T* __restrict__ src, long long lds, T* __restrict__ dst, int ldd,
                                              int R, int C) {
  __shared__ T s[64][66];
  const long long m = blockIdx.z;
  const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;
  for (int k = threadIdx.x; k < 4096; k += 256) {
    const int r = k >> 6, c = k & 63;
    s[r][c] = r0 + r < R && c0 + c < C ? src[(m * R + r0 + r) * lds + c0 + c] : (T)0;
  }
  __syncthreads();
  for (int k = threadIdx.x; k < 4096; k += 256) {
    const int c = k >> 6, r = k & 63;
    if (c0 + c < C && r0 + r < ldd) dst[(m * C + c0 + c) * ldd + r0 + r] = s[r][c];
  }
}

// ---------------------------------------------------------------- gradients of the factors
// g_l(j, c) = alpha sum_{t of l} low(t, j) z[t*ldz + c].  An item is the part of one adapter's (sorted) tokens that lies
// in one window of `win` positions; the items of windows and adapters are counted through (window + adapter).  An
// adapter inside one window is finished here, others leave 32-bit parts that k_join adds in the order of the windows:
// slot 2 w for the adapter that came in from window w - 1, 2 w + 1 for one that begins in w and goes on.
// COLS columns per workgroup, 16 JF rows j; z goes through LDS in steps of 64 tokens as [token][column] and is read by
// the transposing LDS read, low comes from memory as it is (both are laid out as in k_tile).
struct OuterArgs {
  const void *z, *thi, *tlo;
  const int *off, *perm;
  const int4* zero;
  void* out;
  float* part;
  long long ldz, ldo, tp;
  double alpha;
  int C, r, L, win, items;
};

__device__ inline int find_item(const OuterArgs& a, int item, int& w) {
  int lo = 0, hi = a.L - 1;  // the largest l whose first item is not past this one
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.off[mid] / a.win + mid <= item) lo = mid;
    else hi = mid - 1;
  }
  w = item - lo;
  return lo;
}

constexpr int COLS = 256, WIN_MAX = 2048;

// JC: g is stored [j][c] (dA), else [c][j] (dB)
template <typename T, int JF, bool JC, bool DMA> __global__ __launch_bounds__(256, 2) void k_outer(OuterArgs a) {
  typedef typename Op<T>::vec V;
  typedef __bf16 M;
  constexpr int FN = COLS / 64, CH = COLS / 8, J = 64 * CH / 256;  // 4 waves of 64 columns; chunks of a row; per thread
  __shared__ __attribute__((aligned(1024))) char sm[2][64 * COLS * 2];
  __shared__ int rows[WIN_MAX];
  const int ct = (a.C + COLS - 1) / COLS;
  const int c0 = blockIdx.x % ct * COLS, j0 = blockIdx.y * 16 * JF;
  int w;
  const int l = find_item(a, blockIdx.x / ct, w);
  const int lo = a.off[l], end = a.off[l + 1];
  const int p0 = max(lo, w * a.win), p1 = min(end, (w + 1) * a.win);
  if (p0 >= p1) return;
  const int tid = threadIdx.x, lane = tid & 63, q = lane >> 4, c16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  for (int k = tid; k < p1 - p0; k += 256) rows[k] = a.perm[p0 + k];
  __syncthreads();
  const T* z = (const T*)a.z;
  auto turn = [](int step) { return (step & 3) + 4 * ((step >> 3) & 1); };
  const int sr = tid / CH, pc = tid % CH;  // chunk tid + 256 j: row sr + 8 j, whose turn only depends on sr and j's parity
  V g[DMA ? 1 : J];
  auto stage = [&](int b, int s) {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int row = sr + j * (256 / CH), k = s + row;
      const int c = c0 + (2 * ((pc >> 1) ^ turn(row)) + (pc & 1)) * 8;
      if constexpr (DMA) {
        const void* p = k < p1 - p0 && c < a.C ? (const void*)(z + (long long)rows[k] * a.ldz + c) : (const void*)a.zero;
        dma_global(p, &sm[b][wave * 1024 + j * 4096]);
      } else {
        g[j] = load_part(z + (k < p1 - p0 ? (long long)rows[k] * a.ldz + c : 0), k < p1 - p0 ? a.C - c : 0);
      }
    }
  };
  typename Op<T>::out acc[JF][FN];
#pragma unroll
  for (int i = 0; i < JF; ++i)
#pragma unroll
    for (int f = 0; f < FN; ++f) acc[i][f] = f4_t{0, 0, 0, 0};
  const int ftr = (8 * q + (c16 >> 2)) * (COLS * 2) + (c16 & 3) * 8;
  const int tw = (c16 >> 2) + 4 * (q & 1);
  const int n = p1 - p0;
  stage(0, 0);
  for (int s = 0, b = 0; s < n; s += 64, b ^= 1) {
    // low's fragments of this step; zeros past the adapter's last token
    b8_t hi[2][JF], lw[2][JF];
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int i = 0; i < JF; ++i) {
        const int j = min(j0 + 16 * i + c16, a.r - 1), k = s + kk * 32 + q * 8;
        const long long at = j * a.tp + p0 + k;
        hi[kk][i] = load_vec((const M*)a.thi + at);
        lw[kk][i] = load_vec((const M*)a.tlo + at);
        if (s + 64 > n) {
#pragma unroll
          for (int v = 0; v < 8; ++v) {
            hi[kk][i][v] = k + v < n ? hi[kk][i][v] : (M)0.f;
            lw[kk][i][v] = k + v < n ? lw[kk][i][v] : (M)0.f;
          }
        }
      }
    if constexpr (!DMA) {
#pragma unroll
      for (int j = 0; j < J; ++j) *(V*)&sm[b][(tid + 256 * j) * 16] = g[j];
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    if (s + 64 < n) stage(b ^ 1, s + 64);
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int f = 0; f < FN; ++f) {
        typedef short s4_t __attribute__((ext_vector_type(4)));
        typedef short s8_t __attribute__((ext_vector_type(8)));
        typedef __attribute__((address_space(3))) s4_t* lp;
        const char* p = &sm[b][ftr + (((wave * FN + f) ^ tw) << 5) + kk * 32 * COLS * 2];
        const s4_t v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(p));
        const s4_t v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(p + 4 * COLS * 2));
        const s8_t both = __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
        MidOp<T> x;
        x.set(__builtin_bit_cast(V, both));
#pragma unroll
        for (int i = 0; i < JF; ++i) acc[i][f] = x.mma_first(hi[kk][i], lw[kk][i], acc[i][f]);
      }
  }
  const bool whole = lo / a.win == (end - 1) / a.win;
  const float alpha = (float)a.alpha;
  float* part = a.part + (long long)(2 * w + (lo >= w * a.win)) * a.r * a.C;
  T* out = (T*)a.out;
#pragma unroll
  for (int f = 0; f < FN; ++f) {
    const int c = c0 + (wave * FN + f) * 16 + c16;
    if (c >= a.C) continue;
#pragma unroll
    for (int i = 0; i < JF; ++i)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int j = j0 + 16 * i + 4 * q + v;
        if (j >= a.r) continue;
        if (whole) {
          const T o = (T)(alpha == 0.f ? 0.f : alpha * acc[i][f][v]);
          out[JC ? ((long long)l * a.r + j) * a.ldo + c : ((long long)l * a.C + c) * a.ldo + j] = o;
        } else {
          part[JC ? (long long)j * a.C + c : (long long)c * a.r + j] = acc[i][f][v];
        }
      }
  }
}

// Parts of an adapter's windows added in order; zeros for an adapter without tokens.
template <typename T, bool JC> __global__ __launch_bounds__(256) void k_join(OuterArgs a) {
  const int l = blockIdx.y, lo = a.off[l], end = a.off[l + 1];
  const int w0 = lo / a.win, w1 = lo < end ? (end - 1) / a.win : w0 - 1;
  if (w0 == w1) return;
  const long long n = (long long)a.r * a.C;
  const int width = JC ? a.C : a.r;
  const float alpha = (float)a.alpha;
  for (long long e = blockIdx.x * 256ll + threadIdx.x; e < n; e += gridDim.x * 256ll) {
    float v = 0;
    for (int w = w0; w <= w1; ++w) v += a.part[(2 * w + (w == w0)) * n + e];
    ((T*)a.out)[((long long)l * (n / width) + e / width) * a.ldo + e % width] = (T)(alpha == 0.f ? 0.f : alpha * v);
  }
}

// Window length: about 512 workgroups (2 per CU), in whole steps, the ids of a window in LDS.
int window(int T, int C, int r) {
  const int tiles = cdiv(C, COLS) * cdiv(r, 64), parts = max(1, 512 / max(1, tiles));
  return min(WIN_MAX, max(64, cdiv(cdiv(T, parts), 64) * 64));
}

template <typename T> struct GradWs {
  __bf16 *hi = nullptr, *lo = nullptr, *pthi = nullptr, *ptlo = nullptr, *sthi = nullptr, *stlo = nullptr;
  T *At = nullptr, *Bt = nullptr;
  int *off, *perm, *pos;
  int4* zero;
  float *pa = nullptr, *pb = nullptr;
  int rp, ldb, wa, wb;
  long long tp;
  size_t bytes;
  GradWs(const LoraArgs& g, void* ws) {
    rp = low_pitch(g.prec, g.r);
    ldb = cdiv(g.N, 8) * 8;
    tp = cdiv(g.T, 64) * 64 + 64;  // fragments past the last token stay inside
    wa = window(g.T, g.K, g.r);
    wb = window(g.T, g.N, g.r);
    const bool fac = g.dA || g.dB;
    Carve c{(char*)ws};
    zero = c.take<int4>(1);
    off = c.take<int>(g.L + 1);
    perm = c.take<int>(g.T);
    pos = c.take<int>(g.T);
    if (g.dX) {
      hi = c.take<__bf16>((size_t)g.T * rp);
      lo = c.take<__bf16>((size_t)g.T * rp);
      At = c.take<T>((size_t)g.L * g.K * rp);
    }
    if (g.dX || g.dA) Bt = c.take<T>((size_t)g.L * g.r * ldb);
    if (fac) {
      if (g.dA) pthi = c.take<__bf16>(g.r * tp), ptlo = c.take<__bf16>(g.r * tp);
      if (g.dB) sthi = c.take<__bf16>(g.r * tp), stlo = c.take<__bf16>(g.r * tp);
      if (g.dA) pa = c.take<float>((size_t)2 * (g.T / wa + 1) * g.r * g.K);
      if (g.dB) pb = c.take<float>((size_t)2 * (g.T / wb + 1) * g.r * g.N);
    }
    bytes = c.used;
  }
};

template <typename T, bool JC> void run_outer(OuterArgs a, int nt, hipStream_t st) {
  const bool dma = ((uintptr_t)a.z | (uintptr_t)(a.ldz * sizeof(T))) % 16 == 0 && a.C % 8 == 0;
  a.items = nt / a.win + a.L;
  const int jf = a.r <= 16 ? 1 : a.r <= 32 ? 2 : 4;
  const dim3 grid((unsigned)(cdiv(a.C, COLS) * a.items), cdiv(a.r, 16 * jf));
  auto go = [&](auto kernel) { kernel<<<grid, 256, 0, st>>>(a); };
  if (nt > 0) {
    if (jf == 1) dma ? go(k_outer<T, 1, JC, true>) : go(k_outer<T, 1, JC, false>);
    else if (jf == 2) dma ? go(k_outer<T, 2, JC, true>) : go(k_outer<T, 2, JC, false>);
    else dma ? go(k_outer<T, 4, JC, true>) : go(k_outer<T, 4, JC, false>);
  }
  k_join<T, JC><<<dim3(min(512, cdiv(a.r, 1) * cdiv(a.C, 256)), a.L), 256, 0, st>>>(a);
}

template <typename T> int run(const LoraArgs& g, hipStream_t st) {
  GradWs<T> w(g, g.ws);
  if ((size_t)g.ws_bytes < w.bytes) return -2;
  const int* ids = (const int*)g.ids;
  const bool dx = g.dX && g.K > 0 && g.T > 0, da = g.dA && g.K > 0 && g.L > 0, db = g.dB && g.N > 0 && g.L > 0;
  if (g.L > 0) k_sort<<<g.L, 256, 0, st>>>(ids, g.T, g.L, w.off, w.perm, w.pos, w.zero);
  if (g.L > 0 && g.T > 0 && (dx || da) && g.N > 0)
    k_turn<T><<<dim3(cdiv(g.r, 64), cdiv(w.ldb, 64), g.L), 256, 0, st>>>((const T*)g.B, g.ldb, w.Bt, w.ldb, g.N, g.r);
  if (g.L > 0 && dx)
    k_turn<T><<<dim3(cdiv(g.K, 64), cdiv(w.rp, 64), g.L), 256, 0, st>>>((const T*)g.A, g.lda, w.At, w.rp, g.r, g.K);
  int rc = 0;
  if (g.L > 0 && g.T > 0 && (dx || da)) {
    LowArgs a{g.dY, w.Bt, g.scale, ids, g.ldy, w.ldb, g.prec, g.T, g.N, g.r, g.L,
              {dx ? w.hi : nullptr, w.lo, da ? w.pthi : nullptr, w.ptlo, w.pos, w.tp, w.rp}};
    rc = lora_low(a, st);
  }
  if (!rc && db && g.T > 0) {
    LowArgs a{g.X, g.A, g.scale, ids, g.ldx, g.lda, g.prec, g.T, g.K, g.r, g.L, {nullptr, nullptr, w.sthi, w.stlo, w.pos, w.tp, g.r}};
    rc = lora_low(a, st);
  }
  if (!rc && dx) {
    TileArgs a{g.dY, g.W, w.At, w.hi, w.lo, ids, g.dX, g.ldy, g.ldw, w.rp, g.lddx, g.alpha, 0.0, g.prec, g.T, g.N, g.K, g.r, w.rp, g.L};
    rc = lora_tile(a, false, st);
  }
  if (rc) return rc;
  if (da) run_outer<T, true>({g.X, w.pthi, w.ptlo, w.off, w.perm, w.zero, g.dA, w.pa, g.ldx, g.ldda, w.tp, g.alpha, g.K, g.r, g.L, w.wa, 0}, g.T, st);
  if (db) run_outer<T, false>({g.dY, w.sthi, w.stlo, w.off, w.perm, w.zero, g.dB, w.pb, g.ldy, g.lddb, w.tp, g.alpha, g.N, g.r, g.L, w.wb, 0}, g.T, st);
  return (int)hipGetLastError();
}

}  // namespace

size_t lora_grad_ws(const LoraArgs& g) { return g.prec == DPL_H ? GradWs<_Float16>(g, nullptr).bytes : GradWs<__bf16>(g, nullptr).bytes; }

int lora_grad_half(const LoraArgs& g, hipStream_t st) {
  return g.prec == DPL_H ? run<_Float16>(g, st) : run<__bf16>(g, st);
}
