"""Bindings and CPU path of the products whose matrix depends on the column.

The GPU side is ``csrc/kernels/lora*.hip`` and ``csrc/kernels/moe*.hip``: one C call per product, given a record of
pointers and extents that is filled once (:class:`LoraCall`, :class:`MoeCall`) and a stream.  The CPU side computes the
same definitions in torch, in 64 bits for d and 32 bits (the choice of experts in 64) for s, h and b.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib

#: precision codes of these kernels (csrc/kernels/indexed.h)
CODE = {torch.float32: 2, torch.float64: 3, torch.float16: 6, torch.bfloat16: 7}

_ll, _vp, _i, _d = ctypes.c_longlong, ctypes.c_void_p, ctypes.c_int, ctypes.c_double


class LoraArgs(ctypes.Structure):
    _fields_ = ([(n, _ll) for n in ("ldw", "ldx", "lda", "ldb", "ldy", "lddx", "ldda", "lddb")]
                + [(n, _vp) for n in ("W", "X", "A", "B", "ids", "scale", "dY", "Y", "dX", "dA", "dB", "ws")]
                + [("alpha", _d), ("beta", _d), ("ws_bytes", _ll)]
                + [(n, _i) for n in ("prec", "T", "K", "N", "r", "L")])


class MoeArgs(ctypes.Structure):
    _fields_ = ([(n, _ll) for n in ("ldg", "ld1", "ld2", "ldx", "ldy")]
                + [(n, _vp) for n in ("G", "W1", "W2", "X", "Y", "ws")]
                + [("alpha", _d), ("beta", _d), ("ws_bytes", _ll)]
                + [(n, _i) for n in ("prec", "T", "H", "I", "E", "topk", "norm", "pad")])


def pointer(M):
    """Device address of element (0, 0) of a descriptor (None: not asked for)."""
    if M is None:
        return None
    return M.data.data_ptr() + M.offset(0, 0) * M.data.element_size() if M.m and M.n else M.data.data_ptr()


def _storages(*matrices):
    """What the addresses of a record belong to: the tensors, as the descriptors can be given others."""
    return [M.data for M in matrices if M is not None]


class _Call:
    """A kernel call with its argument record and workspace; ``__call__`` enqueues it on the current stream."""

    def __init__(self, device, name, args, ws_bytes, keep, zero=0):
        """zero: bytes at the workspace's beginning that start as zeros (every run leaves them so)."""
        self.name, self.args = name, args
        self.index = torch.cuda.current_device() if device.index is None else device.index
        self.keep = keep  # the storages whose addresses the record holds
        if zero and torch.cuda.is_current_stream_capturing():
            # the zeros would be written by the graph's replays, and a run before the first one would read what was there
            raise RuntimeError(f"{name[4:]}: build the taskpool before the capture that runs it")
        self.ws = torch.empty(max(256, ws_bytes), dtype=torch.uint8, device=device)
        self.ws[:zero].zero_()
        self.home = torch.cuda.current_stream(device).cuda_stream
        if not torch.cuda.is_current_stream_capturing():
            # the allocator may have handed out memory that work queued on this stream still uses; the taskpool may
            # run on another stream first
            torch.cuda.current_stream(device).synchronize()
        args.ws, args.ws_bytes = self.ws.data_ptr(), self.ws.numel()
        self.fn, self.ref = getattr(_lib.load(), name), ctypes.byref(args)

    def __call__(self):
        s = torch.cuda.current_stream(self.index)
        stream = s.cuda_stream
        if stream != self.home and not torch.cuda.is_current_stream_capturing():
            self.ws.record_stream(s)
        rc = self.fn(self.ref, stream)
        if rc:
            _lib.check(rc, self.name)


def _checked(lib, name, record):
    if getattr(lib, name)() != ctypes.sizeof(record):
        raise RuntimeError(f"{name}: the kernel library and its binding disagree; rebuild with tools/build.py")
    return lib


def lora_call(device, alpha, W, X, A, B, ids, scale, beta=0.0, Y=None, dY=None, dX=None, dA=None, dB=None):
    lib = _checked(_lib.load(), "dpl_lora_args_bytes", LoraArgs)
    grad = dY is not None
    y = dY if grad else Y
    a = LoraArgs(W=pointer(W), X=pointer(X), A=pointer(A), B=pointer(B), ids=ids.data_ptr(),
                 scale=None if scale is None else scale.data_ptr(), ldw=W.ld, ldx=X.ld, lda=A.ld, ldb=B.ld, ldy=y.ld,
                 alpha=alpha, beta=beta, prec=CODE[X.dtype], T=X.n, K=X.m, N=y.m, r=A.nb, L=A.n // A.nb)
    if grad:
        a.dY, a.dX, a.dA, a.dB = pointer(dY), pointer(dX), pointer(dA), pointer(dB)
        a.lddx, a.ldda, a.lddb = (0 if M is None else M.ld for M in (dX, dA, dB))
    else:
        a.Y = pointer(Y)
    keep = _storages(W, X, A, B, Y, dY, dX, dA, dB) + [ids, scale]
    return _Call(device, "dpl_lora_grad" if grad else "dpl_lora", a, lib.dpl_lora_ws_bytes(ctypes.byref(a), int(grad)),
                 keep)


def moe_call(device, topk, norm, G, W1, W2, alpha, X, beta, Y):
    lib = _checked(_lib.load(), "dpl_moe_args_bytes", MoeArgs)
    a = MoeArgs(G=pointer(G), W1=pointer(W1), W2=pointer(W2), X=pointer(X), Y=pointer(Y), ldg=G.ld, ld1=W1.ld,
                ld2=W2.ld, ldx=X.ld, ldy=Y.ld, alpha=alpha, beta=beta, prec=CODE[X.dtype], T=X.n, H=X.m, I=W2.m,
                E=G.n, topk=topk, norm=int(norm))
    zero = _ll()
    size = lib.dpl_moe_ws_bytes(ctypes.byref(a), ctypes.byref(zero))
    return _Call(device, "dpl_moe", a, size, _storages(G, W1, W2, X, Y), zero.value)


# ----------------------------------------------------------------------------- CPU path
def rows(M):
    """The descriptor's columns as the rows of a torch view."""
    if not (M.m and M.n):
        return M.data.new_zeros(M.n, M.m)
    return torch.as_strided(M.data, (M.n, M.m), (M.ld, 1), M.data.storage_offset() + M.offset(0, 0))


def _wide(M):
    v = rows(M)
    return v if v.dtype is torch.float64 else v.float()


def _finish(out, alpha, value, beta):
    value = alpha * value if alpha != 0 else torch.zeros_like(value)
    if beta != 0:
        value = value + beta * _wide(out)
    rows(out).copy_(value)


def _groups(ids, scale, L):
    """(adapter, its tokens, its scale) for every adapter."""
    for l in range(L):
        yield l, torch.nonzero(ids == l).flatten(), 1.0 if scale is None else scale[l]


def lora_cpu(alpha, W, X, A, B, ids, scale, beta, Y):
    x, r, L, N = _wide(X), A.nb, A.n // A.nb, Y.m
    a, b = _wide(A).view(L, r, X.m), _wide(B).view(L, N, r)
    y = x @ _wide(W).t()
    for l, t, s in _groups(ids, scale, L):
        y[t] += s * (x[t] @ a[l].t()) @ b[l].t()
    _finish(Y, alpha, y, beta)


def lora_grad_cpu(alpha, W, X, A, B, ids, scale, dY, dX, dA, dB):
    x, dy, r, L, N, K = _wide(X), _wide(dY), A.nb, A.n // A.nb, dY.m, X.m
    a, b = _wide(A).view(L, r, K), _wide(B).view(L, N, r)
    dx = dy @ _wide(W) if dX is not None else None
    da, db = torch.zeros_like(a), torch.zeros_like(b)
    for l, t, s in _groups(ids, scale, L):
        p = s * (dy[t] @ b[l])
        if dX is not None:
            dx[t] += p @ a[l]
        da[l] = p.t() @ x[t]
        db[l] = dy[t].t() @ (s * (x[t] @ a[l].t()))
    for out, value in ((dX, dx), (dA, da.view(L * r, K)), (dB, db.view(L * N, r))):
        if out is not None:
            _finish(out, alpha, value, 0.0)


def moe_cpu(topk, norm, G, W1, W2, alpha, X, beta, Y):
    x, E, width = _wide(X), G.n, W2.m
    z = rows(X).double() @ rows(G).double().t()
    p = torch.softmax(z, 1)
    # a logit that is NaN counts as the largest; ties: the lowest index
    order = torch.sort(torch.nan_to_num(z, nan=float("inf"), posinf=float("inf"), neginf=float("-inf")), dim=1,
                       descending=True, stable=True).indices[:, :topk]
    w = torch.gather(p, 1, order)
    if norm:
        w = w / w.sum(1, keepdim=True)
    w = w.to(x.dtype)
    w1, w2 = _wide(W1).view(E, 2 * width, X.m), _wide(W2).view(E, X.m, width)
    y = torch.zeros_like(x)
    for j in range(topk):
        for e in torch.unique(order[:, j]).tolist():
            t = torch.nonzero(order[:, j] == e).flatten()
            h = x[t] @ w1[e].t()
            g, u = h[:, :width], h[:, width:]
            y[t] += w[t, j, None] * (((g / (1 + torch.exp(-g))) * u) @ w2[e].t())
    _finish(Y, alpha, y, beta)
