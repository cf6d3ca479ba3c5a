"""Products whose matrix depends on the column: projections with low-rank adapters, and mixtures of experts.

Beside GEMM, where every column of X meets the same matrix, these pick a column's matrices by an index.  A family of
matrices is a block row of tiles: ``A`` of K x (L r) with tile width r holds A_0 .. A_{L-1}.  Matrices are column-major
with one token per column (a row-major torch tensor [tokens, features] is that as it stands), in LAPACK storage or in
tiles that span all rows, on one process: on a process grid each process runs them on ``ctx.local()`` with the columns
that it holds.

``gemm_lora``       Y(:,t) := alpha (W^T x_t + s_l B_l^T A_l^T x_t) + beta Y(:,t),  l = ids[t]
``gemm_lora_grad``  the gradients of alpha (...) with respect to X, A and B (W, ids and the scales are held fixed)
``moe``             Y(:,t) := alpha sum_j w_j W2_e^T (silu(g) * u) + beta Y(:,t),  [g; u] = W1_e^T x_t, over the k
                    experts e whose logits G^T x_t are largest

Precisions: s and d, and the half precisions h (fp16) and b (bf16), which the other operations do not take.  h and b
are multiplied by the 16-bit matrix instructions and summed in 32 bits; each result is rounded once.

A taskpool runs on the stream that is current when it is run, takes the operands' and indices' values of that moment,
makes no allocation and no host synchronisation, and may be captured into a HIP graph (moe's is built before the
capture).  Its operands are the storages that the descriptors have when it is built, and it holds on to them: a tensor
that is bound to a descriptor later is another matrix's.  It owns its workspace, so one taskpool (and every graph that
captured it) has one run in flight at a time, and it lives as long as those graphs.  Building one takes tens of
microseconds and waits for the current stream; the number of tokens is fixed in it.
Outputs must not overlap inputs.  An infinity or NaN in one adapter, expert, token or output's weights makes what it meets
infinite or NaN (in h and b an infinity of a factor may come out as NaN) and nothing else.
"""
from __future__ import annotations

import copy

import torch

from ..constants import DTYPE_PREC, STORAGE_LAPACK
from ..ops import indexed_ops as ops
from ..runtime import Taskpool

_LIMIT = 4194240      # tokens or features: 65535 tiles of 64 along one grid axis
_FAMILY = 65535       # adapters: one grid axis
_RANK = 262140        # 65535 groups of 4 along one grid axis
# a launch holds less than 2^32 threads:
_FACTORS = 2 ** 23 - 1         # adapters and windows of tokens, times tiles of 256 features: workgroups of 256 threads of
                               # one factor's gradient, both in one launch
_EXPERT = 16 * (2 ** 23 - 1)   # features of tokens and experts: a workgroup of 512 threads for 16 of them


def _matrix(op, ctx, name, M, m, n, dtype):
    """A descriptor that is an m x n column-major matrix (n None: any) on the context's device."""
    if M.dtype != dtype:
        raise TypeError(f"{op}: {name} is {DTYPE_PREC.get(M.dtype, M.dtype)}, the product is {DTYPE_PREC[dtype]}")
    if M.m != m or (n is not None and M.n != n):
        raise ValueError(f"{op}: {name} is {M.m}x{M.n}, expected {m}x{'any' if n is None else n}")
    if M.P * M.Q != 1:
        raise ValueError(f"{op}: {name} is distributed over {M.P}x{M.Q} processes; use a descriptor of ctx.local()")
    if M.storage != STORAGE_LAPACK and M.lmt > 1:
        raise ValueError(f"{op}: {name} needs LAPACK storage, or tiles that span all {M.lm} rows")
    if M.data is None:
        raise ValueError(f"{op}: {name} has no storage")
    if M.data.device != ctx.device:
        raise ValueError(f"{op}: {name} is on {M.data.device}, the context on {ctx.device}")
    if not M.data.is_contiguous():
        raise ValueError(f"{op}: {name}'s storage is not contiguous")
    if M.m and M.n:
        last = M.offset(0, 0) + (M.n - 1) * M.ld + M.m
        if M.ld < M.m or M.data.numel() < last:
            raise ValueError(f"{op}: {name}'s storage holds {M.data.numel()} elements, {last} are needed")
    return M


def _bound(*matrices):
    """Descriptors of the taskpool's own, with the storages of this moment (None stays None)."""
    return [copy.copy(M) for M in matrices]


def _vector(op, ctx, name, v, n, dtype):
    if not isinstance(v, torch.Tensor) or v.dtype != dtype or v.dim() != 1 or v.numel() != n:
        raise ValueError(f"{op}: {name} must be a vector of {n} {dtype}")
    if v.device != ctx.device:
        raise ValueError(f"{op}: {name} is on {v.device}, the context on {ctx.device}")
    if not v.is_contiguous():
        raise ValueError(f"{op}: {name} is not contiguous")
    return v


def _span(M):
    """(first, past the last) byte of a matrix, or None without elements."""
    if isinstance(M, torch.Tensor):
        return (M.data_ptr(), M.data_ptr() + M.numel() * M.element_size()) if M.numel() else None
    if M is None or not (M.m and M.n):
        return None
    at = ops.pointer(M)
    return at, at + ((M.n - 1) * M.ld + M.m) * M.data.element_size()


def _disjoint(op, outputs, inputs):
    """Outputs overlap neither inputs nor each other (matrices side by side in the columns of one buffer may interleave)."""
    for i, (name, out) in enumerate(outputs):
        a = _span(out)
        for other, M in list(inputs) + outputs[i + 1:]:
            b = _span(M)
            if a is None or b is None or a[0] >= b[1] or b[0] >= a[1]:
                continue
            if not isinstance(M, torch.Tensor) and M.ld == out.ld and M.dtype == out.dtype:
                gap = (b[0] - a[0]) // out.data.element_size() % out.ld  # rows from out's first to M's first
                if gap >= out.m and gap + M.m <= out.ld:
                    continue
            raise ValueError(f"{op}: {name} overlaps {other}")


def _precision(op, M):
    if M.dtype not in ops.CODE:
        raise TypeError(f"{op}: precision {DTYPE_PREC.get(M.dtype, M.dtype)} is not supported (s, d, h or b)")
    return M.dtype


def _family(op, name, M, width=None):
    """Number of matrices in a block row of tiles."""
    nb = M.nb if width is None else width
    if M.nb != nb:
        raise ValueError(f"{op}: {name}'s tiles are {M.nb} columns wide, expected {nb}")
    if M.n % nb:
        raise ValueError(f"{op}: {name}'s {M.n} columns are not whole tiles of {nb}")
    return M.n // nb


def _extent(op, **sizes):
    for n, v in sizes.items():
        if v > 2 ** 31 - 65:
            raise ValueError(f"{op}: {n} = {v} is past 32 bits")


def _lora_checks(op, ctx, W, X, A, B, ids, scale, N, outputs, others):
    dtype = _precision(op, X)
    K, T, r = X.m, X.n, A.nb
    _matrix(op, ctx, "X", X, K, T, dtype)
    _matrix(op, ctx, "W", W, K, N, dtype)
    L = _family(op, "A", A)
    _matrix(op, ctx, "A", A, K, L * r, dtype)
    if N and _family(op, "B", B, N) != L:
        raise ValueError(f"{op}: A holds {L} adapters, B {B.n // N}")
    _matrix(op, ctx, "B", B, r, L * N, dtype)
    if max(T, K, N, r) > _LIMIT or L > _FAMILY:
        raise ValueError(f"{op}: at most {_LIMIT} tokens or features and {_FAMILY} adapters, got T = {T}, K = {K}, "
                         f"N = {N}, r = {r}, L = {L}")
    if r > _RANK:
        raise ValueError(f"{op}: at most rank {_RANK}, got {r}")
    _vector(op, ctx, "ids", ids, T, torch.int32)
    if scale is not None:
        _vector(op, ctx, "scale", scale, L, torch.float64 if dtype is torch.float64 else torch.float32)
    _disjoint(op, outputs, [("W", W), ("X", X), ("A", A), ("B", B), ("ids", ids)] + others
              + ([("scale", scale)] if scale is not None else []))


def _pool(ctx, name, gpu, cpu, flops):
    tp = Taskpool(name, ctx)
    tp.flops = float(flops)
    if ctx.is_gpu:
        with torch.cuda.device(ctx.device):
            fn = gpu()
    else:
        fn = cpu
    tp.task(name.upper(), "caller", fn, comm=False)
    return tp.finish_build()


def gemm_lora_New(ctx, alpha, W, X, A, B, ids, scale, beta, Y) -> Taskpool:
    """Taskpool of Y(:,t) := alpha (W^T x_t + s_l B_l^T A_l^T x_t) + beta Y(:,t) with l = ids[t].

    W: K x N, the projection all tokens share.  X: K x T, one token per column.  A: K x (L r) in tiles of r columns
    and B: r x (L N) in tiles of N columns, adapter l's factors.  ids: T int32 on the device, read when the taskpool
    runs; a value outside 0..L-1 (-1, say) means no adapter.  scale: L numbers (float32; float64 in d), or None for
    ones.  Y: N x T; with beta = 0 its old values are not read.
    """
    op = "gemm_lora"
    N = Y.m
    _matrix(op, ctx, "Y", Y, N, X.n, _precision(op, X))
    _lora_checks(op, ctx, W, X, A, B, ids, scale, N, [("Y", Y)], [])
    W, X, A, B, Y = _bound(W, X, A, B, Y)
    return _pool(ctx, op, lambda: ops.lora_call(ctx.device, float(alpha), W, X, A, B, ids, scale, float(beta), Y),
                 lambda: ops.lora_cpu(float(alpha), W, X, A, B, ids, scale, float(beta), Y),
                 2 * X.n * (X.m * N + A.nb * (X.m + N)))


def gemm_lora(ctx, alpha, W, X, A, B, ids, scale, beta, Y):
    """Blocking :func:`gemm_lora_New`."""
    return gemm_lora_New(ctx, alpha, W, X, A, B, ids, scale, beta, Y).execute(ctx)


def gemm_lora_grad_New(ctx, alpha, W, X, A, B, ids, scale, dY, dX, dA, dB) -> Taskpool:
    """Taskpool of the gradient of gemm_lora's alpha (...) term, given dY (N x T) of its result.

    dX: K x T, dA: like A, dB: like B; each may be None.  They are written, not accumulated: an adapter that no token
    names gets zeros.  Sums run over an adapter's tokens in an order that only ids decide, so a run repeats bit by bit.
    """
    op = "gemm_lora_grad"
    dtype, N, K, T, r = _precision(op, X), dY.m, X.m, X.n, A.nb
    _matrix(op, ctx, "dY", dY, N, T, dtype)
    outputs = [("dX", dX, (K, T), None), ("dA", dA, (K, A.n), r), ("dB", dB, (r, B.n), N)]
    for name, M, (m, n), nb in outputs:
        if M is not None:
            _matrix(op, ctx, name, M, m, n, dtype)
            if nb:
                _family(op, name, M, nb)
    _lora_checks(op, ctx, W, X, A, B, ids, scale, N, [o[:2] for o in outputs if o[1] is not None], [("dY", dY)])
    windows = (T + 8 * (A.n // r) + 16) // 256 + 1
    if (A.n // r + windows) * -(-max(K, N) // 256) > _FACTORS:
        raise ValueError(f"{op}: {A.n // r} adapters of {max(K, N)} features and {T} tokens are more than {_FACTORS} "
                         f"tiles of 256")
    W, X, A, B, dY, dX, dA, dB = _bound(W, X, A, B, dY, dX, dA, dB)
    return _pool(ctx, op,
                 lambda: ops.lora_call(ctx.device, float(alpha), W, X, A, B, ids, scale, dY=dY, dX=dX, dA=dA, dB=dB),
                 lambda: ops.lora_grad_cpu(float(alpha), W, X, A, B, ids, scale, dY, dX, dA, dB),
                 2 * T * (N * r * ((dX is not None or dA is not None) + (dB is not None))
                          + (dX is not None) * K * (N + r) + (dA is not None) * K * r + (dB is not None) * K * r))


def gemm_lora_grad(ctx, alpha, W, X, A, B, ids, scale, dY, dX, dA, dB):
    """Blocking :func:`gemm_lora_grad_New`."""
    return gemm_lora_grad_New(ctx, alpha, W, X, A, B, ids, scale, dY, dX, dA, dB).execute(ctx)


def moe_New(ctx, topk, norm, G, W1, W2, alpha, X, beta, Y) -> Taskpool:
    """Taskpool of a mixture-of-experts layer: Y(:,t) := alpha sum_j w_j W2_e^T (silu(g) * u) + beta Y(:,t).

    G: H x E, the router.  W1: H x (E 2I) in tiles of 2I columns, expert e's gate (the first I) and up projections.
    W2: I x (E H) in tiles of H columns, its down projections.  X, Y: H x T.  The logits z = G^T x_t are summed in 64
    bits and the topk largest taken, ties by the lowest index; w is the softmax over all E logits at the chosen ones,
    divided by its sum over them where ``norm`` is true.  Meant for a few tokens: they go in batches of 64 (of 512 / topk
    with more than 8 experts a token), and every batch reads the weights of the experts that it uses.
    """
    op = "moe"
    dtype, H, T, E, width = _precision(op, X), X.m, X.n, G.n, W2.m
    _matrix(op, ctx, "X", X, H, T, dtype)
    _matrix(op, ctx, "Y", Y, H, T, dtype)
    _matrix(op, ctx, "G", G, H, E, dtype)
    most = 4096  # a token's logits stay in LDS
    if not 1 <= E <= most:
        raise ValueError(f"{op}: 1 to {most} experts, got {E}")
    if not 1 <= topk <= min(E, 256) or int(topk) != topk:
        raise ValueError(f"{op}: topk = {topk} of {E} experts (at most 256)")
    if H and (_family(op, "W2", W2, H) != E or width and _family(op, "W1", W1, 2 * width) != E):
        raise ValueError(f"{op}: G has {E} experts, W1 {W1.n} columns and W2 {W2.n}")
    _matrix(op, ctx, "W1", W1, H, E * 2 * width, dtype)
    _matrix(op, ctx, "W2", W2, width, E * H, dtype)
    if T > 65535:
        raise ValueError(f"{op}: at most 65535 tokens, got {T}")
    if max(H, width) > _EXPERT:
        raise ValueError(f"{op}: at most {_EXPERT} features, got {H} and {width} of an expert")
    _extent(op, E=E * 2 * width)
    _disjoint(op, [("Y", Y)], [("G", G), ("W1", W1), ("W2", W2), ("X", X)])
    G, W1, W2, X, Y = _bound(G, W1, W2, X, Y)
    return _pool(ctx, op, lambda: ops.moe_call(ctx.device, int(topk), bool(norm), G, W1, W2, float(alpha), X,
                                               float(beta), Y),
                 lambda: ops.moe_cpu(int(topk), bool(norm), G, W1, W2, float(alpha), X, float(beta), Y),
                 2 * T * H * (E + 3 * topk * width))


def moe(ctx, topk, norm, G, W1, W2, alpha, X, beta, Y):
    """Blocking :func:`moe_New`."""
    return moe_New(ctx, topk, norm, G, W1, W2, alpha, X, beta, Y).execute(ctx)
