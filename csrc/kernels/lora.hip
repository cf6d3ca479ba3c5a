// Projection with low-rank adapters of many requests, and its gradient.
//
//   y_t  = alpha (W^T x_t + s_l B_l^T A_l^T x_t) + beta y_t            l = ids[t]; outside 0..L-1: no adapter
//   dx_t = alpha (W dy_t + s_l A_l B_l dy_t)
//   dA_l = alpha s_l sum_{t: ids[t]=l} x_t (B_l dy_t)^T                dB_l = alpha s_l sum_t (A_l^T x_t) dy_t^T
//
// Layouts (element offsets): W[n*ldw + k], X[t*ldx + k], Y[t*ldy + n], A_l[(l*r + j)*lda + k], B_l[(l*N + n)*ldb + j].
//
// Here: the entry points.  The forward product of few tokens is in lora_few.hip, that of many and the low-rank vectors in
// lora_tile.hip, the gradient in lora_grad.hip.
//
// Steps: the low-rank vectors S = s_l A_l^T x (and P = s_l B_l dy) of every token into the workspace, then the shared
// product with the adapter's part added to the same accumulators.  Nothing of one adapter ever meets another's token:
// where the rows of a tile use several adapters, each adapter's part is formed apart and kept by a select, so an
// infinity or NaN in one adapter stays with its own tokens.
#include "lora.h"

namespace {

// T > 64: the low-rank vectors, then the shared product that adds the adapters' parts
struct ForwardWs {
  char* low;
  int rp;
  size_t bytes;
  ForwardWs(const LoraArgs& g, void* ws) {
    rp = low_pitch(g.prec, g.r);
    const size_t n = (size_t)g.T * rp * mid_bytes(g.prec);
    Carve c{(char*)ws};
    low = c.take<char>(n);
    bytes = c.used;
  }
};

int forward(const LoraArgs& g, hipStream_t st) {
  if (g.T <= 64) return (size_t)g.ws_bytes < lora_few_ws(g) ? -2 : lora_few(g, st);
  ForwardWs w(g, g.ws);
  if ((size_t)g.ws_bytes < w.bytes) return -2;
  const int* ids = (const int*)g.ids;
  if (g.L > 0) {
    const LowArgs a{g.X, g.A, g.scale, ids, g.ldx, g.lda, g.prec, g.T, g.K, g.r, g.L, {w.low, nullptr, nullptr, 0, w.rp}};
    const int rc = lora_low(&a, 1, st);
    if (rc) return rc;
  }
  return lora_tile({g.X, g.W, g.B, w.low, ids, g.Y, g.ldx, g.ldw, g.ldb, g.ldy, g.alpha, g.beta, g.prec, g.T, g.K, g.N, g.r, w.rp, g.L}, true, st);
}

}  // namespace

DPL_API int dpl_lora_args_bytes() { return (int)sizeof(LoraArgs); }

DPL_API long long dpl_lora_ws_bytes(const LoraArgs* g, int grad) {
  return (long long)(grad ? lora_grad_ws(*g) : g->T <= 64 ? lora_few_ws(*g) : ForwardWs(*g, nullptr).bytes);
}

DPL_API int dpl_lora(const LoraArgs* g, hipStream_t st) { return g->T == 0 || g->N == 0 ? 0 : forward(*g, st); }

DPL_API int dpl_lora_grad(const LoraArgs* g, hipStream_t st) { return lora_grad(*g, st); }
