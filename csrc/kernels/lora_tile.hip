// The shared product of many tokens with the adapters' parts added to the same accumulators, and the low-rank vectors
// that those parts start from.
#include "lora.h"

namespace {

// ---------------------------------------------------------------- low-rank vectors
// One or two sets of them (the gradient's P and S) in a launch.
struct LowSets {
  LowArgs set[2];
  int sets;
};

// One wave per (token, j): for few tokens, where the tokens of a workgroup's rows would mostly have adapters of their own.
template <typename T> __global__ __launch_bounds__(256) void k_low_dot(LowSets sets) {
  typedef typename Num<T>::acc R;
  const LowArgs& a = sets.set[blockIdx.z];
  const int t = blockIdx.x, j = blockIdx.y * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int l = a.ids[t];
  if (j >= a.r || (unsigned)l >= (unsigned)a.L) return;
  if (j == 0 && lane < a.out.rp - a.r) pad_low<T>(a.out, t, a.r + lane);
  R s;
  const T* f = (const T*)a.F + ((long long)l * a.r + j) * a.ldf;
  wave_dots<1>(&f, (const T*)a.x + (long long)t * a.ldx, a.C, &s);
  s *= a.scale ? ((const R*)a.scale)[l] : R(1);
  if (lane == 0) put_low<T>(a.out, t, j, s);
}

// 16 TF tokens and 16 JF rows of the factors per workgroup, the contraction split over the waves and joined in LDS, one adapter
// of these tokens at a time.
//   DMA (rows begin at multiples of 16 bytes): each wave has a ring of LDS buffers of its own for steps of 128 bytes, laid
//     out as in k_tile and filled straight from memory; no barrier before the join.  (Fragments read where they are used,
//     16 rows x 64 bytes a load, come out of the L2 at 37 GB/s per CU, whole lines at 130.)
//   else: the same lines from any address through registers, two steps ahead (16 JF = 64, 3648 x 2015: 53.6 us with
//     fragments straight from memory, 24 so).
template <typename T, int JF, int TF, bool DMA>
__global__ __launch_bounds__(DMA && JF * TF >= 4 ? 256 : 512) void k_low_tile(LowSets sets) {
  typedef typename Num<T>::acc R;
  typedef typename Op<T>::vec V;
  constexpr int WAVES = DMA && JF * TF >= 4 ? 4 : 8, E = Op<T>::E, KS = Op<T>::KS;
  constexpr int RING = JF == 4 || JF + TF == 3 ? 3 : 4, LOADS = 2 * TF + 2 * JF, STAGE = LOADS * 1024;
  constexpr int JOIN = WAVES * 16 * (16 * TF + 1) * (int)sizeof(R);
  constexpr int BUFS = WAVES * (DMA ? RING : 1) * STAGE, MAIN = BUFS > JOIN ? BUFS : JOIN;
  __shared__ __attribute__((aligned(1024))) char sm[MAIN + 16 * TF * sizeof(int)];
  int* sid = (int*)(sm + MAIN);
  const LowArgs& a = sets.set[blockIdx.z];
  const int tid = threadIdx.x, lane = tid & 63, q = lane >> 4, c = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int t0 = blockIdx.x * 16 * TF, j0 = blockIdx.y * 16 * JF;
  R(*red)[16][16 * TF + 1] = (R(*)[16][16 * TF + 1])sm;
  int mine = -1;
  if (lane < 16 * TF && t0 + lane < a.nt) mine = a.ids[t0 + lane];
  if ((unsigned)mine >= (unsigned)a.L) mine = -1;
  if (tid < 16 * TF) {
    sid[tid] = mine;
    if (mine >= 0 && blockIdx.y == 0)
      for (int j = a.r; j < a.out.rp; ++j) pad_low<T>(a.out, t0 + tid, j);
  }
  unsigned long long todo = __ballot(mine >= 0);
  while (todo) {
    const int l = __builtin_amdgcn_readlane(mine, __builtin_ctzll(todo));
    todo &= ~__ballot(mine == l);
    const T *x = (const T*)a.x + (long long)t0 * a.ldx, *f = (const T*)a.F + ((long long)l * a.r + j0) * a.ldf;
    const int rt = min(16 * TF, a.nt - t0), rj = min(16 * JF, a.r - j0);
    typename Op<T>::out acc[JF][TF];
#pragma unroll
    for (int i = 0; i < JF; ++i)
#pragma unroll
      for (int k = 0; k < TF; ++k) acc[i][k] = typename Op<T>::out{R(0), R(0), R(0), R(0)};
    if constexpr (DMA) {
      constexpr int BK = 2 * KS;
      constexpr unsigned NOWHERE = 0x80000000u;
      const int steps = (a.C + BK - 1) / BK, s0 = steps * w / WAVES, s1 = steps * (w + 1) / WAVES;
      const int row = lane >> 3, chunk = (lane & 7) ^ row;
      const unsigned xbytes = (unsigned)(((rt - 1) * a.ldx + a.C) * (long long)sizeof(T));
      const unsigned fbytes = (unsigned)(((rj - 1) * a.ldf + a.C) * (long long)sizeof(T));
      unsigned ox[2 * TF], of[2 * JF];
#pragma unroll
      for (int k = 0; k < 2 * TF; ++k) ox[k] = (unsigned)(min(row + 8 * k, rt - 1) * (int)a.ldx + chunk * E) * sizeof(T);
#pragma unroll
      for (int k = 0; k < 2 * JF; ++k) of[k] = (unsigned)(min(row + 8 * k, rj - 1) * (int)a.ldf + chunk * E) * sizeof(T);
      char* ring = sm + w * RING * STAGE;
      auto stage = [&](int s) {
        char* b = ring + (s - s0) % RING * STAGE;
        const bool in = s < s1 && s * BK + chunk * E < a.C;
        const int at = s < s1 ? s * BK * (int)sizeof(T) : 0;
#pragma unroll
        for (int k = 0; k < 2 * TF; ++k) dma_buffer(x, xbytes, b + k * 1024, in ? ox[k] : NOWHERE, at);
#pragma unroll
        for (int k = 0; k < 2 * JF; ++k) dma_buffer(f, fbytes, b + TF * 2048 + k * 1024, in ? of[k] : NOWHERE, at);
      };
#pragma unroll
      for (int k = 0; k < RING - 1; ++k) stage(s0 + k);
      const int fr = c * 128 + ((q ^ (c & 7)) << 4);
      for (int s = s0; s < s1; ++s) {
        // this step has arrived, and the one before has been read: its buffer is filled next
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LOADS * (RING - 2)) : "memory");
        __builtin_amdgcn_sched_barrier(0);
        stage(s + RING - 1);
        const char* b = ring + (s - s0) % RING * STAGE;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          V v[TF];
#pragma unroll
          for (int k = 0; k < TF; ++k) v[k] = *(const V*)(b + (fr ^ (64 * half)) + k * 2048);
#pragma unroll
          for (int i = 0; i < JF; ++i) {
            const V fv = *(const V*)(b + TF * 2048 + (fr ^ (64 * half)) + i * 2048);
#pragma unroll
            for (int k = 0; k < TF; ++k) acc[i][k] = Op<T>::mma(fv, v[k], acc[i][k]);
          }
        }
      }
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    } else {
      static_assert(TF == 1, "one fragment of tokens");
      constexpr int BK = 2 * KS;
      const int steps = (a.C + BK - 1) / BK, s0 = steps * w / WAVES, s1 = steps * (w + 1) / WAVES;
      const int row = lane >> 3, chunk = (lane & 7) ^ row, fr = c * 128 + ((q ^ (c & 7)) << 4);
      const T* p[LOADS];
#pragma unroll
      for (int k = 0; k < LOADS; ++k)
        p[k] = (k < 2 ? x + min(row + 8 * k, rt - 1) * a.ldx : f + min(row + 8 * (k - 2), rj - 1) * a.ldf) + chunk * E;
      V g[2][LOADS];
      auto fetch = [&](V* v, int s) {
        if (s >= s1) return;
        const long long k0 = (long long)s * BK;
        if (k0 + BK <= a.C) {
#pragma unroll
          for (int k = 0; k < LOADS; ++k) v[k] = load_vec(p[k] + k0);
        } else {
#pragma unroll
          for (int k = 0; k < LOADS; ++k) v[k] = load_part(p[k] + k0, a.C - (int)k0 - chunk * E);
        }
      };
      char* b = sm + w * STAGE;
      auto use = [&](const V* v) {
#pragma unroll
        for (int k = 0; k < LOADS; ++k) *(V*)(b + k * 1024 + lane * 16) = v[k];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const V xv = *(const V*)(b + (fr ^ (64 * half)));
#pragma unroll
          for (int i = 0; i < JF; ++i) acc[i][0] = Op<T>::mma(*(const V*)(b + 2048 + (fr ^ (64 * half)) + i * 2048), xv, acc[i][0]);
        }
      };
      fetch(g[0], s0);
      for (int s = s0; s < s1; s += 2) {
        fetch(g[1], s + 1);
        use(g[0]);
        if (s + 1 >= s1) break;
        fetch(g[0], s + 2);
        use(g[1]);
      }
    }
    const R scale = a.scale ? ((const R*)a.scale)[l] : R(1);
#pragma unroll
    for (int i = 0; i < JF; ++i) {
      __syncthreads();  // the waves are through with their buffers, or with the join before
#pragma unroll
      for (int k = 0; k < TF; ++k)
#pragma unroll
        for (int v = 0; v < 4; ++v) red[w][out_row<T>(lane, v)][16 * k + c] = acc[i][k][v];
      __syncthreads();
      for (int p = tid; p < 256 * TF; p += 64 * WAVES) {
        const int j = j0 + 16 * i + p % 16, t = p / 16;
        if (sid[t] != l || j >= a.r) continue;
        R v = 0;
#pragma unroll
        for (int k = 0; k < WAVES; ++k) v += red[k][p % 16][t];
        put_low<T>(a.out, t0 + t, j, scale * v);
      }
    }
    __syncthreads();
  }
}

template <typename T> int run_low(const LowSets& sets, hipStream_t st) {
  const LowArgs& a = sets.set[0];
  // one wave per (token, j) for few tokens, and up to 512 where a tile's tokens would go through several adapters one after
  // the other.  Tokens x K x N, us of the whole product by tiles and so (bf16 unless said):
  //   65 x 4096 x 1024, one adapter: r 8 24.8, 22.6, r 64 29.9, 25.5; 32 adapters in any order: r 16 95.6, 47.1
  //   256 x 4096 x 1024, one adapter: r 16 25.3, 24.2, r 64 30.7, 31.4; 4 in runs, r 64: 42.1, 33.1; 32: r 16 91.9, 45.9
  //   256 tokens, one adapter: fp16 2015 x 1001 r 16 30.6, 29.9, r 64 38.2, 41.7; fp32 2048 x 1024 r 64 59.3, 54.5
  //   300 x 4096 x 1024, r 32, 16 adapters: in runs 41.5, 30.0, in any order 91.5, 39.4
  //   413 x 2040 x 5001, fp16, r 12, 9 adapters in runs: 40.5, 34.2
  //   512 x 4096 x 1024, r 32: one adapter 26.6, 29.7, 4 in runs 31.7, 30.6; 500, r 64, one adapter 30.5, 38.4
  // (500 x 4096 x 1024, r 64, 16 adapters would be better so too: in runs 48.4, 43.2, in any order 135.5, 60.4.)
  if (a.nt <= 256 || (a.nt <= 512 && a.r <= 32 && a.L > 1)) {
    k_low_dot<T><<<dim3(a.nt, cdiv(a.r, 4), sets.sets), 256, 0, st>>>(sets);
    return (int)hipGetLastError();
  }
  bool dma = true;
  for (int k = 0; k < sets.sets; ++k) {
    const LowArgs& s = sets.set[k];
    auto wide = [](const void* q, long long ld) { return ((uintptr_t)q | (uintptr_t)(ld * sizeof(T))) % 16 == 0 && ld * (long long)sizeof(T) * 64 < (1ll << 30); };
    dma = dma && wide(s.x, s.ldx) && wide(s.F, s.ldf) && s.C % Op<T>::E == 0;
  }
  const int jf = a.r <= 16 ? 1 : a.r <= 32 || (!dma && sizeof(T) > 2) ? 2 : 4;  // (4 through registers spills in s and d)
  // two fragments of tokens, which halves the factors' traffic, where that leaves a workgroup for every CU
  const int tf = dma && sizeof(T) == 2 && a.nt >= 8192 ? 2 : 1;
  const dim3 grid(cdiv(a.nt, 16 * tf), cdiv(a.r, 16 * jf), sets.sets);
  auto go = [&](auto kernel, int threads) { kernel<<<grid, threads, 0, st>>>(sets); };
  if constexpr (sizeof(T) == 2)
    if (tf == 2) {
      jf == 1 ? go(k_low_tile<T, 1, 2, true>, 512) : jf == 2 ? go(k_low_tile<T, 2, 2, true>, 256) : go(k_low_tile<T, 4, 2, true>, 256);
      return (int)hipGetLastError();
    }
  if (dma) jf == 1 ? go(k_low_tile<T, 1, 1, true>, 512) : jf == 2 ? go(k_low_tile<T, 2, 1, true>, 512) : go(k_low_tile<T, 4, 1, true>, 256);
  else if (jf == 1) go(k_low_tile<T, 1, 1, false>, 512);
  else if (jf == 2) go(k_low_tile<T, 2, 1, false>, 512);
  else if constexpr (sizeof(T) == 2) go(k_low_tile<T, 4, 1, false>, 512);
  return (int)hipGetLastError();
}

// ---------------------------------------------------------------- shared product
// A workgroup owns B tokens x B features, WT x WN waves of (B / WT) x (B / WN).  The contraction goes in steps of 128
// bytes of a row (whole cache lines: with 64-byte steps, which ask for the same lines twice, an earlier form of this kernel
// took 1 % longer at 16384 x 4096 x 16384, and 10 % where all of it lies in the L2) through LDS buffers, each step in two
// halves of one fragment.  While a half is multiplied from registers the fragments of the next one are read from LDS;
// when a step's second half is in registers its buffers take a later step.  So neither latency is waited for, and a step
// has one barrier.  SLOTS buffers, each of one operand's part of a step, X and W in turn: 4 (a step ahead) where several
// workgroups share a CU, 8 where few share the chip and a step's products are much shorter than the way from memory, and
// 5, all of the LDS, with the largest tile: X then has two steps to arrive (16384 x 4096 x 16384, r 64: 1899 us with 4, 1796
// with 5; a gradient with dX of 8192 x 16384 x 4096, W's features contiguous: 1193, 1071; W two steps instead of X: the same).
// What bounds the largest tile: power.  At 16384 x 4096 x 16384 (1.76 ms) the matrix pipes are busy 65 % of the time (8192 x
// 16384 x 4096, W's features contiguous: 72 %) at the 1.9 GHz that the card's limit leaves; the library's product runs at
// 85 % and 1.50 GHz, 1.64 to 1.70 ms.  (4 waves of 128 x 128 would read a third less from LDS, but with 256 accumulators a lane the
// compiler moves them about: 1.04 PFLOP/s.)
//   DMA: rows begin at multiples of 16 bytes and the tile's rows lie within 2^30 bytes: memory to LDS directly.
//        A chunk past the rows' end is fetched from past the buffer descriptor's end, which reads as zero.
//   else: through registers, 16 bytes from any address, with zeros past the rows' end, one step ahead of the buffers on a
//     128 tile and two on a 64 tile (bf16, 184 x 4429 x 704: 38.3 us with 4, 36.5 with 2; 4097^3: 302 with 2, 292 with 1).
// LDS rows are 8 chunks of 16 bytes; chunk c of row i lies at c ^ (i & 7), so that the rows that a fragment read takes
// the same chunk of lie in different banks: the counter's 6144 cycles of conflicts a tile are the same with K = 4096 as
// with 8192, so they are the output's and not the steps'.  W stored with its features contiguous (NT false) is kept as it comes,
// [step][features], and read through the transposing LDS read: a group of 16 lanes takes 4 steps x 16 features; the
// 32-byte pair of such a read is displaced by the step's place in the instruction (16 steps of one instruction: 8 pairs).
// s and d read element by element there, a lane group q its own E steps, with the 16 features of a fragment displaced by q
// (their matrix instructions take 4 and 8 times as long per byte, which hides the reads).
// The result has the tokens in its columns: a lane holds one token and 4 neighbouring features.
template <typename T, int B, int WT, int WN, int SLOTS, bool NT, bool DMA>
__global__ __launch_bounds__(64 * WT * WN, 2) void k_tile(TileArgs a) {
  typedef typename Num<T>::acc R;
  typedef typename Op<T>::vec V;
  constexpr int THREADS = 64 * WT * WN, E = Op<T>::E, BK = 2 * Op<T>::KS, SLOT = B * 128;
  constexpr int FT = B / WT / 16, FN = B / WN / 16;
  constexpr int J = B * 8 / THREADS, CH = B / E;  // CH: chunks of a [step][features] row
  static_assert(SLOTS >= 4 && (DMA || SLOTS == 4), "without DMA the steps after next are in registers");
  constexpr int SETS = DMA || B == 128 ? 1 : 2;  // of registers, a step each
  __shared__ __attribute__((aligned(1024))) char sm[SLOTS * SLOT];
  const int tid = threadIdx.x, lane = tid & 63, q = lane >> 4, c16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wt = wave / WN, wn = wave % WN;
  // tiles of one XCD's workgroups: 4 tile rows of tokens at a time, tokens fastest, so that they share rows in its L2
  // (4 / 8 / 16 rows: 1796 / 1803 / 1835 us at 16384 x 4096 x 16384, 801 / 812 / 836 at 8192^3)
  const int tt = (a.T + B - 1) / B, tn = (a.N + B - 1) / B;
  const int id = xcd_remap(blockIdx.x, tt * tn);
  const int group = id / (4 * tn), in = id % (4 * tn), gs = min(4, tt - group * 4);
  const int t0 = (group * 4 + in % gs) * B, n0 = in / gs * B;
  const T* x = (const T*)a.x + (long long)t0 * a.ldx;
  const T* W = (const T*)a.W + (NT ? (long long)n0 * a.ldw : n0);
  const int rt = min(B, a.T - t0), rn = min(B, a.N - n0);

  // staging: chunk id tid + j * THREADS of either operand
  const int xr = tid >> 3, xc = (tid & 7) ^ (xr & 7);
  const int wr = NT ? xr : tid / CH;
  const int wmask = CH / 2 - 1;
  auto turn = [&](int step) { return ((step & 3) + 4 * ((step >> 3) & 1)) & wmask; };
  auto wchunk = [&](int row, int pc) { return sizeof(T) == 2 ? 2 * ((pc >> 1) ^ turn(row)) + (pc & 1) : pc ^ (16 / E * (row / E & 3)); };
  V gx[SETS][J], gw[SETS][J];  // (not in use with DMA)
  unsigned ox[DMA ? J : 1], ow[DMA ? J : 1];
  constexpr unsigned NOWHERE = 0x80000000u;
  if constexpr (DMA) {
#pragma unroll
    for (int j = 0; j < J; ++j) ox[j] = (unsigned)(min(xr + j * (THREADS / 8), rt - 1) * (int)a.ldx + xc * E) * sizeof(T);
#pragma unroll
    for (int j = 0; j < J; ++j) {
      if (NT) {
        ow[j] = (unsigned)(min(wr + j * (THREADS / 8), rn - 1) * (int)a.ldw + xc * E) * sizeof(T);
      } else {
        const int row = wr + j * (THREADS / CH);
        ow[j] = (unsigned)(row * (int)a.ldw + wchunk(row, tid % CH) * E) * sizeof(T);
      }
    }
  }
  const int xbytes = DMA ? (int)(((rt - 1) * a.ldx + a.C) * (long long)sizeof(T)) : 0;
  const unsigned pitch = (unsigned)a.ldw * sizeof(T);
  const unsigned wbytes = DMA ? (unsigned)((NT ? (rn - 1) * a.ldw + a.C : (a.C - 1) * a.ldw + rn) * (long long)sizeof(T)) : 0;
  const int steps = (a.C + BK - 1) / BK;
  // each XCD begins at another eighth of the contraction: beginning together they all ask for the same rows of W at
  // once (1888 us, so 1796 at 16384 x 4096 x 16384; 850, 801 at 8192^3)
  const int turned = steps / 8 * (blockIdx.x & 7);
  auto place = [&](int s) { return (s >= steps ? s : s + turned >= steps ? s + turned - steps : s + turned) * BK; };
  auto stage_x = [&](int s, char* slot) {  // steps past the last one read as zero
    const int k0 = place(s);
    const bool in = k0 + xc * E < a.C;
#pragma unroll
    for (int j = 0; j < J; ++j) dma_buffer(x, xbytes, slot + j * THREADS * 16, in ? ox[j] : NOWHERE, k0 * (int)sizeof(T));
  };
  auto stage_w = [&](int s, char* slot) {
    const int k0 = place(s);
    if (NT) {
      const bool in = k0 + xc * E < a.C;
#pragma unroll
      for (int j = 0; j < J; ++j) dma_buffer(W, wbytes, slot + j * THREADS * 16, in ? ow[j] : NOWHERE, k0 * (int)sizeof(T));
    } else {
      // the descriptor ends with W's last row
#pragma unroll
      for (int j = 0; j < J; ++j) dma_buffer(W, wbytes, slot + j * THREADS * 16, ow[j] + (unsigned)k0 * pitch, 0);
    }
  };
  auto fetch = [&](V* vx, V* vw, int s) {
    const int k0 = place(s), left = a.C - k0 - xc * E;
    auto px = [&](int j) { return x + (long long)min(xr + j * (THREADS / 8), rt - 1) * a.ldx + k0 + xc * E; };
    auto pw = [&](int j) { return W + (long long)min(wr + j * (THREADS / 8), rn - 1) * a.ldw + k0 + xc * E; };
    // inside the rows without a test per lane.  W's features past the tile are not used, but have to be there: what
    // follows in the same row, or the row after it
    if (NT ? k0 + BK <= a.C : k0 + BK < a.C && a.N >= E) {
#pragma unroll
      for (int j = 0; j < J; ++j) vx[j] = load_vec(px(j));
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int row = wr + j * (THREADS / CH);
        vw[j] = load_vec(NT ? pw(j) : W + (long long)(k0 + row) * a.ldw + min(wchunk(row, tid % CH), (rn - 1) / E) * E);
      }
    } else {
#pragma unroll
      for (int j = 0; j < J; ++j) vx[j] = load_part(px(j), left);
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int row = wr + j * (THREADS / CH), n = wchunk(row, tid % CH) * E;
        vw[j] = NT ? load_part(pw(j), left) : load_part(W + (long long)(k0 + row) * a.ldw + n, k0 + row < a.C ? rn - n : 0);
      }
      __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): lets the compiler count the loads under way where the paths meet
    }
  };
  auto put = [&](const V* vx, const V* vw, char* sx, char* sw) {
#pragma unroll
    for (int j = 0; j < J; ++j) *(V*)(sx + tid * 16 + j * THREADS * 16) = vx[j];
#pragma unroll
    for (int j = 0; j < J; ++j) *(V*)(sw + tid * 16 + j * THREADS * 16) = vw[j];
  };

  typename Op<T>::out acc[FN][FT];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int f = 0; f < FT; ++f) acc[i][f] = typename Op<T>::out{R(0), R(0), R(0), R(0)};
  const int fx = (wt * FT * 16 + c16) * 128 + ((q ^ (c16 & 7)) << 4);  // ^ 64: the second half of the step
  const int fw = (wn * FN * 16 + c16) * 128 + ((q ^ (c16 & 7)) << 4);
  const int ftr = (8 * q + (c16 >> 2)) * (B * 2) + (c16 & 3) * 8;  // + pair * 32
  const int tw = ((c16 >> 2) + 4 * (q & 1)) & wmask;
  struct Frag {
    V x[FT], w[FN];
  };
  auto read = [&](Frag& r, const char* sx, const char* sw, int half) {
#pragma unroll
    for (int i = 0; i < FN; ++i) {
      if constexpr (NT) {
        r.w[i] = *(const V*)(sw + (fw ^ (64 * half)) + i * 2048);
      } else if constexpr (sizeof(T) > 2) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          r.w[i][e] = *(const T*)(sw + ((half * Op<T>::KS + q * E + e) * B + ((wn * FN + i) ^ q) * 16 + c16) * (int)sizeof(T));
      } else {
        typedef short s8_t __attribute__((ext_vector_type(8)));
        const char* p = sw + ftr + (((wn * FN + i) ^ tw) << 5) + half * 32 * B * 2;
        const s4_t lo = read_turned(p);
        const s4_t hi = read_turned(p + 4 * B * 2);
        const s8_t both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        r.w[i] = __builtin_bit_cast(V, both);
      }
    }
#pragma unroll
    for (int f = 0; f < FT; ++f) r.x[f] = *(const V*)(sx + (fx ^ (64 * half)) + f * 2048);
  };
  auto multiply = [&](const Frag& r) {
#pragma unroll
    for (int f = 0; f < FT; ++f)
#pragma unroll
      for (int i = 0; i < FN; ++i) acc[i][f] = Op<T>::mma(r.w[i], r.x[f], acc[i][f]);
  };
  auto meet = [&]() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  constexpr int LOADS = 2 * J, READS = FT + (NT ? FN : 2 * FN), PRODUCTS = FT * FN, EARLY = READS / 2;
  static_assert(J * (SLOTS - 2) < 64, "the wait counts 6 bits");
  auto pace = [&](int loads) {
    // the reads early among the products, then the loads: left alone, the compiler puts the reads where the next half
    // waits for them
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int k = 0; k < EARLY; ++k) {
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, PRODUCTS / 2 / EARLY, 0);
      }
      if (loads) {
#pragma unroll
        for (int k = 0; k < LOADS; ++k) {
          __builtin_amdgcn_sched_group_barrier(0x010, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x008, PRODUCTS / 2 / LOADS, 0);
        }
      }
    }
  };
  if (steps > 0) {
    Frag one, two;
    int sx = 0, sw = SLOT;  // where this step's parts are
    auto next = [&](int slot) { return slot + 2 * SLOT >= SLOTS * SLOT ? slot + (2 - SLOTS) * SLOT : slot + 2 * SLOT; };
    char* own = sm + wave * 1024;  // where this wave's loads go within a buffer
    if constexpr (DMA) {
#pragma unroll
      for (int k = 0; k < SLOTS; ++k) k & 1 ? stage_w(k / 2, own + k * SLOT) : stage_x(k / 2, own + k * SLOT);
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(J * (SLOTS - 2)) : "memory");
    } else {
      fetch(gx[0], gw[0], 0);
      if (SETS == 1) put(gx[0], gw[0], sm, sm + SLOT);
      fetch(gx[SETS - 1], gw[SETS - 1], 1);
      if (SETS > 1) put(gx[0], gw[0], sm, sm + SLOT);
      put(gx[SETS - 1], gw[SETS - 1], sm + 2 * SLOT, sm + 3 * SLOT);
#pragma unroll
      for (int u = 0; u < SETS; ++u) fetch(gx[u], gw[u], u + 2);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    meet();
    read(one, sm + sx, sm + sw, 0);
    for (int s0 = 0; s0 < steps; s0 += SETS)
#pragma unroll
      for (int u = 0; u < SETS; ++u) {
        const int s = s0 + u;
        if (SETS > 1 && s >= steps) break;
        read(two, sm + sx, sm + sw, 1);
        multiply(one);
        pace(0);
        // step s + 1 has arrived, and this step is in registers: its buffers are free
        if constexpr (DMA) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(J * (SLOTS - 4)) : "memory");
        else asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        meet();
        const int fx0 = sx, fw0 = sw;
        sx = next(sx);
        sw = next(sw);
        read(one, sm + sx, sm + sw, 0);
        if constexpr (!DMA) {
          put(gx[u], gw[u], sm + fx0, sm + fw0);
          fetch(gx[u], gw[u], s + 2 + SETS);
        } else if constexpr (SLOTS & 1) {  // an odd number: the operands change places
          stage_w(s + SLOTS / 2, own + fx0);
          stage_x(s + SLOTS / 2 + 1, own + fw0);
        } else {
          stage_x(s + SLOTS / 2, own + fx0);
          stage_w(s + SLOTS / 2, own + fw0);
        }
        multiply(two);
        pace(1);
      }
    // nothing is on its way to LDS when the workgroup ends
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  }

  // the adapters' parts: one adapter of this wave's tokens at a time, fragments straight from memory (r is short).  The
  // product is formed apart and added by a select: what it holds for tokens of other adapters may be anything.
  int lid[FT];
#pragma unroll
  for (int f = 0; f < FT; ++f) {
    const int t = t0 + (wt * FT + f) * 16 + c16;
    int l = a.L > 0 && t < a.T ? a.ids[t] : -1;
    if ((unsigned)l >= (unsigned)a.L) l = -1;
    lid[f] = l;
  }
  constexpr int NONE = 0x7fffffff;
  auto after = [&](int l) {  // the next larger adapter of this wave's tokens
    int next = NONE;
#pragma unroll
    for (int f = 0; f < FT; ++f) next = lid[f] > l ? min(next, lid[f]) : next;
#pragma unroll
    for (int o = 8; o; o >>= 1) next = min(next, __shfl_xor(next, o));
    return __builtin_amdgcn_readfirstlane(next);
  };
  // (one loop over adapters and steps of r together: two nested ones cost a second copy of the accumulators)
  int l = after(-1), j0 = 0;
  while (l != NONE) {
    {
      const int j = j0 + q * E;
      MidOp<T> F[FN];
#pragma unroll
      for (int i = 0; i < FN; ++i) {
        const int n = min(n0 + (wn * FN + i) * 16 + c16, a.N - 1);
        F[i].set(load_part((const T*)a.F + ((long long)l * a.N + n) * a.ldf + j, a.r - j));
      }
#pragma unroll
      for (int f = 0; f < FT; ++f) {
        const unsigned long long m = __ballot(lid[f] == l);
        __builtin_amdgcn_sched_barrier(0);
        if (m == 0) continue;
        const long long at = (long long)min(t0 + (wt * FT + f) * 16 + c16, a.T - 1) * a.rp + j;
        Mem<T> mem;
        mem.load((const R*)a.low + at);
        Mid<T> low;
        low.set(mem);
        const typename Op<T>::out none = {R(0), R(0), R(0), R(0)};
        typename Op<T>::out d[FN];
#pragma unroll
        for (int k = 0; k < MidOp<T>::N; ++k)
#pragma unroll
          for (int i = 0; i < FN; ++i) d[i] = F[i].product(k, low, k ? d[i] : none);
#pragma unroll
        for (int i = 0; i < FN; ++i) acc[i][f] += lid[f] == l ? d[i] : none;
      }
    }
    j0 += Op<T>::KS;
    if (j0 >= a.r) {
      l = after(l);
      j0 = 0;
    }
  }

  // Out through LDS, 16 tokens of a wave at a time, so that memory gets whole rows of the wave's features (from the
  // accumulators a store would write 32 bytes of each of 16 rows)
  const R alpha = (R)a.alpha, beta = (R)a.beta;
  constexpr int ROW = FN * 16, PITCH = ROW + 16 / sizeof(R), OW = 16 / sizeof(T), LANES = ROW / OW;  // lanes of a row
  static_assert(WT * WN * 16 * PITCH * sizeof(R) <= SLOTS * SLOT && 64 % LANES == 0, "staging");
  __syncthreads();
  R* mine = (R*)sm + wave * 16 * PITCH;
  const int col = lane % LANES * OW, n = n0 + wn * ROW + col;
#pragma unroll
  for (int f = 0; f < FT; ++f) {
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < FN; ++i) {
      if constexpr (sizeof(T) == 8) {
#pragma unroll
        for (int v = 0; v < 4; ++v) mine[c16 * PITCH + i * 16 + out_row<T>(lane, v)] = acc[i][f][v];
      } else {
        *(typename Op<T>::out*)&mine[c16 * PITCH + i * 16 + 4 * q] = acc[i][f];
      }
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int r0 = 0; r0 < 16; r0 += 64 / LANES) {
      const int r = r0 + lane / LANES, t = t0 + (wt * FT + f) * 16 + r;
      if (r >= 16 || t >= a.T || n >= a.N) continue;
      T* p = (T*)a.y + (long long)t * a.ldy + n;
      R u[OW];
#pragma unroll
      for (int v = 0; v < OW; ++v) u[v] = alpha == R(0) ? R(0) : alpha * mine[r * PITCH + col + v];
      if (n + OW <= a.N) {
        V o;
        if (beta != R(0)) {
          o = load_vec(p);
#pragma unroll
          for (int v = 0; v < OW; ++v) u[v] += beta * (R)o[v];
        }
#pragma unroll
        for (int v = 0; v < OW; ++v) o[v] = (T)u[v];
        __builtin_memcpy(p, &o, 16);
      } else {
#pragma unroll
        for (int v = 0; v < OW; ++v)
          if (n + v < a.N) p[v] = (T)(beta != R(0) ? u[v] + beta * widen(p[v]) : u[v]);
      }
    }
  }
}

template <typename T, int B, int WT, int WN, int SLOTS, bool NT, bool DMA> void launch(const TileArgs& a, hipStream_t st) {
  k_tile<T, B, WT, WN, SLOTS, NT, DMA><<<cdiv(a.T, B) * cdiv(a.N, B), 64 * WT * WN, 0, st>>>(a);
}

template <typename T, bool NT> int run_tile(const TileArgs& a, hipStream_t st) {
  const long long size = sizeof(T), span = 1ll << 30;
  auto wide = [&](const void* p, long long ld, int rows) {
    return ((uintptr_t)p | (uintptr_t)(ld * size)) % 16 == 0 && ld * size * rows < span;
  };
  // W with its features contiguous also needs whole chunks of them within a row, and offsets in 32 bits over all of it
  const bool dma = wide(a.x, a.ldx, 256) && wide(a.W, a.ldw, 256) && a.C % Op<T>::E == 0 &&
                   (NT || (a.N % Op<T>::E == 0 && (a.C + 1024ll) * a.ldw * size < (1ll << 32)));
  auto tiles = [&](int b) { return (long long)cdiv(a.T, b) * cdiv(a.N, b); };
  if constexpr (sizeof(T) == 2)
    if (dma && tiles(256) >= 160) {
      launch<T, 256, 2, 4, 5, NT, true>(a, st);
      return (int)hipGetLastError();
    }
  // 128 tiles where they reach most CUs (fp64, 1000 x 1000 x 2000: 148 us with 128 of them, 93 with 512 of 64; 300 x 1000
  // x 2000: 150, 59).  8 buffers where they leave every workgroup a CU or two, and 8 waves on a 128 tile (T x K x N, us
  // with 4 and 8 buffers: bf16 100 x 4096 x 4096 38.0, 21.3; 512 x 4096 x 4096 39.7, 31.5; 1024 x 4096 x 4096 51.5, 39.8,
  // with W's features contiguous 55.8, 43.5)
  if (tiles(128) >= 160) {
    if (!dma) launch<T, 128, 2, sizeof(T) == 8 ? 4 : 2, 4, NT, false>(a, st);  // (fp64 spills with 4 waves)
    else if (tiles(128) <= 256) launch<T, 128, 2, 4, 8, NT, true>(a, st);
    else launch<T, 128, 2, 4, 4, NT, true>(a, st);
  } else {
    if (!dma) launch<T, 64, 2, 2, 4, NT, false>(a, st);
    else if (tiles(64) <= 512) launch<T, 64, 2, 2, 8, NT, true>(a, st);
    else launch<T, 64, 2, 2, 4, NT, true>(a, st);
  }
  return (int)hipGetLastError();
}

}  // namespace

int lora_low(const LowArgs* sets, int n, hipStream_t st) {
  LowSets s{};
  s.sets = n;
  for (int k = 0; k < n; ++k) s.set[k] = sets[k];
  switch (sets[0].prec) {
    case DPL_S: return run_low<float>(s, st);
    case DPL_D: return run_low<double>(s, st);
    case DPL_H: return run_low<_Float16>(s, st);
    case DPL_B: return run_low<__bf16>(s, st);
  }
  return -1;
}

int lora_tile(const TileArgs& a, bool nt, hipStream_t st) {
  switch (a.prec) {
    case DPL_S: return nt ? run_tile<float, true>(a, st) : run_tile<float, false>(a, st);
    case DPL_D: return nt ? run_tile<double, true>(a, st) : run_tile<double, false>(a, st);
    case DPL_H: return nt ? run_tile<_Float16, true>(a, st) : run_tile<_Float16, false>(a, st);
    case DPL_B: return nt ? run_tile<__bf16, true>(a, st) : run_tile<__bf16, false>(a, st);
  }
  return -1;
}
