"""Plain 64-bit forms of the products whose matrix depends on the column, with bounds on what a kernel may be off by.

The bounds hold element by element.  u is the result type's half step; a sum of n products in 32 bits (64 for d) is off
by at most n e times the sum of the products' magnitudes, e = 2^-24 (2^-53).  For h and b there is room
for an intermediate that is kept to 2^-16 of itself (the kernels keep all of its 32 bits).
"""
import torch

import dplasma_amd as dp

HALF = (torch.float16, torch.bfloat16)
U = {t: torch.finfo(t).eps / 2 for t in (torch.float16, torch.bfloat16, torch.float32, torch.float64)}


def matrix(t, nb=None, cols=None):
    """Descriptor of a row-major tensor's rows as columns; cols: how many leading entries of each row are the matrix's."""
    ld = max(1, t.shape[-1])
    n = t.shape[:-1].numel()
    m = t.shape[-1] if cols is None else cols
    return dp.TiledMatrix(t.dtype, max(1, m), max(1, nb or n), m, n, device=t.device, storage="lapack", lld=ld,
                          data=t if t.numel() else None)


def work_eps(dtype):
    return 2.0 ** -53 if dtype is torch.float64 else 2.0 ** -24


def split_eps(dtype):
    return 2.0 ** -16 if dtype in HALF else 0.0


def make_ids(kind, T, L, gen):
    if kind == "none":
        ids = torch.full((T,), -1)
    elif kind == "one":
        ids = torch.full((T,), max(0, L - 1))
    elif kind == "runs":
        ids = torch.sort(torch.randint(-1, L, (T,), generator=gen)).values
    else:  # every token its own, with ids outside the adapters among them
        ids = torch.randint(-2, L + 2, (T,), generator=gen)
    return ids.to(torch.int32)


class Lora:
    """Inputs of one case, and its plain form with bounds, on a device."""

    def __init__(self, dtype, T, K, N, r, L, kind="tokens", pad=0, seed=0, device="cpu"):
        gen = torch.Generator().manual_seed(seed + T + 3 * K + 5 * N + 7 * r + 11 * L)
        self.dtype, self.T, self.K, self.N, self.r, self.L, self.pad = dtype, T, K, N, r, L, pad
        wide = torch.float64 if dtype is torch.float64 else torch.float32

        def normal(*shape, std=1.0):
            return (torch.randn(*shape, generator=gen, dtype=torch.float64) * std).to(dtype).to(device)

        self.x, self.w = normal(T, K + pad), normal(N, K, std=max(K, 1) ** -0.5)
        self.a, self.b = normal(L, r, K, std=max(K, 1) ** -0.5), normal(L, N, r, std=r ** -0.5)
        self.y, self.dy = normal(T, N + pad), normal(T, N + pad, std=0.1)
        self.ids = make_ids(kind, T, L, gen).to(device)
        self.scale = (torch.rand(L, generator=gen, dtype=torch.float64) + 0.5).to(wide).to(device)

    def descriptors(self):
        return (matrix(self.w), matrix(self.x, cols=self.K), matrix(self.a, self.r),
                matrix(self.b, self.N))

    def forward(self, ctx, alpha=1.0, beta=0.0, scale=True):
        """The framework's result (the whole buffer, padding too)."""
        y = self.y.clone()
        W, X, A, B = self.descriptors()
        dp.gemm_lora(ctx, alpha, W, X, A, B, self.ids, self.scale if scale else None, beta, matrix(y, cols=self.N))
        return y

    def plain(self, alpha=1.0, beta=0.0, scale=True):
        """(result, bound) in 64 bits."""
        x, w, a, b = self.x[:, :self.K].double(), self.w.double(), self.a.double(), self.b.double()
        y, ys = x @ w.t(), x.abs() @ w.abs().t()
        ls = torch.zeros_like(y)
        for l in range(self.L):
            t = torch.nonzero(self.ids == l).flatten()
            s = float(self.scale[l]) if scale else 1.0
            y[t] += s * (x[t] @ a[l].t()) @ b[l].t()
            ls[t] = s * (x[t].abs() @ a[l].abs().t()) @ b[l].abs().t()
        old = self.y[:, :self.N].double()
        out = alpha * y + (beta * old if beta else 0.0)
        e = work_eps(self.dtype)
        off = abs(alpha) * ((self.K + self.r + 8) * e * ys + ((self.K + self.r + 16) * e + split_eps(self.dtype)) * ls)
        off += abs(beta) * 4 * e * old.abs() if beta else 0.0
        return out, off + U[self.dtype] * (out.abs() + off) + tiny(self.dtype)

    def backward(self, ctx, alpha=1.0, scale=True, want="xab"):
        W, X, A, B = self.descriptors()
        dx = torch.full_like(self.x, 7.0)
        da, db = torch.full_like(self.a, 7.0), torch.full_like(self.b, 7.0)
        dp.gemm_lora_grad(ctx, alpha, W, X, A, B, self.ids, self.scale if scale else None, matrix(self.dy, cols=self.N),
                          matrix(dx, cols=self.K) if "x" in want else None,
                          matrix(da, self.r) if "a" in want else None,
                          matrix(db, self.N) if "b" in want else None)
        return dx, da, db

    def plain_backward(self, alpha=1.0, scale=True):
        """((dx, bound), (da, bound), (db, bound)) from the formulas in 64 bits."""
        x, w, a, b = self.x[:, :self.K].double(), self.w.double(), self.a.double(), self.b.double()
        dy = self.dy[:, :self.N].double()
        dx, dxs = dy @ w, dy.abs() @ w.abs()
        dxl = torch.zeros_like(dx)
        da, das, db, dbs = (torch.zeros_like(v) for v in (a, a, b, b))
        for l in range(self.L):
            t = torch.nonzero(self.ids == l).flatten()
            s = float(self.scale[l]) if scale else 1.0
            p, ps = s * (dy[t] @ b[l]), s * (dy[t].abs() @ b[l].abs())
            q, qs = s * (x[t] @ a[l].t()), s * (x[t].abs() @ a[l].abs().t())
            dx[t] += p @ a[l]
            dxl[t] = ps @ a[l].abs()
            da[l], das[l] = p.t() @ x[t], ps.t() @ x[t].abs()
            db[l], dbs[l] = dy[t].t() @ q, dy[t].t().abs() @ qs
        e, c = work_eps(self.dtype), split_eps(self.dtype)
        got = []
        for v, off in ((dx, (self.N + self.r + 8) * e * dxs + ((self.N + self.r + 16) * e + c) * dxl),
                       (da, ((self.N + self.T + 16) * e + c) * das), (db, ((self.K + self.T + 16) * e + c) * dbs)):
            v, off = alpha * v, abs(alpha) * off
            got.append((v, off + U[self.dtype] * (v.abs() + off) + tiny(self.dtype)))
        return got


def tiny(dtype):
    """Half a step below the smallest normal number: what gradual underflow may lose."""
    f = torch.finfo(dtype)
    return f.tiny * f.eps


class Moe:
    def __init__(self, dtype, T, H, I, E, k, seed=0, device="cpu"):
        gen = torch.Generator().manual_seed(seed + T + 3 * H + 5 * I + 7 * E + 11 * k)
        self.dtype, self.T, self.H, self.I, self.E, self.k = dtype, T, H, I, E, k

        def normal(*shape, std=1.0):
            return (torch.randn(*shape, generator=gen, dtype=torch.float64) * std).to(dtype).to(device)

        self.x, self.y = normal(T, H), normal(T, H)
        self.g = normal(E, H, std=max(H, 1) ** -0.5)
        self.w1, self.w2 = normal(E, 2 * I, H, std=max(H, 1) ** -0.5), normal(E, H, I, std=max(I, 1) ** -0.5)

    def descriptors(self):
        return (matrix(self.g), matrix(self.w1, 2 * self.I), matrix(self.w2, self.H),
                matrix(self.x))

    def forward(self, ctx, norm=True, alpha=1.0, beta=0.0):
        y = self.y.clone()
        G, W1, W2, X = self.descriptors()
        dp.moe(ctx, self.k, norm, G, W1, W2, alpha, X, beta, matrix(y))
        return y

    def plain(self, norm=True, alpha=1.0, beta=0.0):
        x, g, w1, w2 = (v.double() for v in (self.x, self.g, self.w1, self.w2))
        z = x @ g.t()
        p = torch.softmax(z, 1)
        order = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :self.k]
        w = torch.gather(p, 1, order)
        if norm:
            w = w / w.sum(1, keepdim=True)
        e, c, I = work_eps(self.dtype), split_eps(self.dtype), self.I
        y, off = torch.zeros_like(x), torch.zeros_like(x)
        for j in range(self.k):
            for q in range(self.E):
                t = torch.nonzero(order[:, j] == q).flatten()
                if not t.numel():
                    continue
                h, hs = x[t] @ w1[q].t(), (x[t].abs() @ w1[q].abs().t()) * (self.H + 4) * e
                gate, up = h[:, :I], h[:, I:]
                silu = gate / (1 + torch.exp(-gate))
                act = silu * up
                # |silu'| < 1.1; exp, quotient and product each a few steps
                d = 1.1 * hs[:, :I] * (up.abs() + hs[:, I:]) + silu.abs() * hs[:, I:] + (16 * e + c) * act.abs()
                y[t] += w[t, j, None] * (act @ w2[q].t())
                off[t] += w[t, j, None] * ((d + (I + 32 + self.k) * e * act.abs()) @ w2[q].abs().t())
        old = self.y.double()
        out = alpha * y + (beta * old if beta else 0.0)
        off = abs(alpha) * off + (abs(beta) * 4 * e * old.abs() if beta else 0.0)
        return out, off + U[self.dtype] * (out.abs() + off) + tiny(self.dtype)


def within(got, want, bound, what=""):
    got = got.double()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    bad = (got - want).abs() > bound
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst "
                           f"{float(((got - want).abs() / bound).max()):.3g} times the bound")
