"""Measured cases of the operators whose matrix depends on the column: adapted products and mixtures of experts.

``gemm_lora`` (a projection shared by all tokens plus the low-rank adapter of each token's request), its gradient
``gemm_lora_grad`` and ``moe`` (router, experts' gated products and their weighted sum for a few tokens).  With
``own`` false :func:`run` computes them in elementary torch operations, with ``own`` true through ``dplasma_amd``.
Tensors are row-major with one token per row, which is the column-major one-token-per-column matrix that the
framework's descriptors hold.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "fp64": torch.float64}


def listed():
    return [
        # one token of one request through a square projection: a chat answer being written
        {"name": "lora_one_token", "op": "lora", "dtype": "bf16", "T": 1, "K": 2048, "N": 2048, "r": 16, "L": 8,
         "mix": "tokens", "bare": 0.0, "pad": 0},
        # a serving step: 48 requests, one token each, adapters picked per request, some requests without one
        {"name": "lora_serving_step", "op": "lora", "dtype": "bf16", "T": 48, "K": 4096, "N": 8192, "r": 16, "L": 32,
         "mix": "tokens", "bare": 0.2, "pad": 0},
        # a mixed step of odd sizes in half precision: prompts' pieces and single tokens in one batch
        {"name": "lora_mixed_odd", "op": "lora", "dtype": "fp16", "T": 413, "K": 2040, "N": 5001, "r": 12, "L": 9,
         "mix": "runs", "bare": 0.1, "pad": 24},
        # prompts of several requests one after the other, activations inside a wider buffer
        {"name": "lora_prompts", "op": "lora", "dtype": "bf16", "T": 4096, "K": 4096, "N": 4096, "r": 32, "L": 6,
         "mix": "runs", "bare": 0.1, "pad": 64},
        # the largest: a batch of long prompts through a widening projection
        {"name": "lora_long_prompts", "op": "lora", "dtype": "bf16", "T": 16384, "K": 4096, "N": 16384, "r": 64,
         "L": 4, "mix": "runs", "bare": 0.0, "pad": 0},
        # single precision, as the rest of a single-precision program has it
        {"name": "lora_single", "op": "lora", "dtype": "fp32", "T": 1000, "K": 1024, "N": 2048, "r": 8, "L": 3,
         "mix": "runs", "bare": 0.2, "pad": 0},
        # training on a small batch in half precision, odd sizes, several adapters in one batch
        {"name": "grad_small_odd", "op": "grad", "dtype": "fp16", "T": 190, "K": 1000, "N": 1544, "r": 8, "L": 5,
         "mix": "runs", "bare": 0.1, "pad": 8},
        # the ordinary training step: one adapter, a square projection
        {"name": "grad_one_adapter", "op": "grad", "dtype": "bf16", "T": 4096, "K": 4096, "N": 4096, "r": 16, "L": 1,
         "mix": "runs", "bare": 0.0, "pad": 0},
        # several adapters trained side by side on long sequences
        {"name": "grad_many_adapters", "op": "grad", "dtype": "bf16", "T": 8192, "K": 4096, "N": 16384, "r": 64,
         "L": 8, "mix": "runs", "bare": 0.0, "pad": 0},
        # one token through a layer of many small experts
        {"name": "moe_one_token", "op": "moe", "dtype": "bf16", "T": 1, "H": 2048, "I": 1024, "E": 64, "k": 8,
         "norm": True, "beta": 0.0},
        # a serving step: two dozen tokens, few large experts, added onto the residual
        {"name": "moe_serving_step", "op": "moe", "dtype": "bf16", "T": 24, "H": 4096, "I": 4096, "E": 16, "k": 2,
         "norm": True, "beta": 1.0},
        # odd sizes in half precision, weights not renormalised
        {"name": "moe_odd", "op": "moe", "dtype": "fp16", "T": 37, "H": 1000, "I": 728, "E": 30, "k": 3,
         "norm": False, "beta": 0.0},
    ]


def _size(rng, low, high):
    """A size spread over the logarithm of low..high: round, half-round or odd."""
    n = int(math.exp(rng.uniform(math.log(low), math.log(high))))
    step = rng.choice([1, 8, 64, 64])
    return min(high, max(low, n // step * step))


def draw(rng):
    op = rng.choice(["lora", "lora", "grad", "moe", "moe"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp16", "fp32", "fp64"])
    if op == "moe":
        E = rng.randint(4, 64)
        H, width = _size(rng, 256, 4096), _size(rng, 128, 4096)
        while E * H * width > 16 * 4096 * 4096:
            width = max(128, width // 2)
            H = max(256, H * 3 // 4)
        return {"op": op, "dtype": dtype, "T": _size(rng, 1, 64), "H": H, "I": width, "E": E,
                "k": rng.randint(1, min(8, E)), "norm": rng.random() < 0.5, "beta": rng.choice([0.0, 1.0])}
    big = dtype in ("bf16", "fp16")
    T = _size(rng, 1 if op == "lora" else 64, 16384 if big else 2048)
    K, N = _size(rng, 256, 8192 if big else 2048), _size(rng, 256, 8192 if big else 2048)
    r = rng.choice([4, 8, 12, 16, 32, 64])
    mix = "tokens" if T <= 256 and rng.random() < 0.6 else "runs"
    return {"op": op, "dtype": dtype, "T": T, "K": K, "N": N, "r": r, "L": rng.randint(1, 32 if mix == "tokens" else 8),
            "mix": mix, "bare": rng.choice([0.0, 0.1, 0.5]), "pad": rng.choice([0, 0, 8, 40])}


def work(case):
    size = torch.empty(0, dtype=DTYPES[case["dtype"]]).element_size()
    if case["op"] == "moe":
        T, H, width, E, k = (case[n] for n in ("T", "H", "I", "E", "k"))
        used = E * (1 - (1 - k / E) ** T)  # experts that T tokens reach, on average
        values = H * E + used * 3 * H * width + (2 + bool(case["beta"])) * T * H
        return {"bytes": size * values, "flops": 2.0 * T * (H * E + 3 * k * H * width)}
    T, K, N, r, L = (case[n] for n in ("T", "K", "N", "r", "L"))
    used = min(T, L) * r * (K + N)
    if case["op"] == "lora":
        return {"bytes": size * (T * K + K * N + used + T * N) + 4 * T,
                "flops": 2.0 * T * (K * N + r * (K + N))}
    return {"bytes": size * (2 * T * K + T * N + K * N + used + L * r * (K + N)) + 4 * T,
            "flops": 2.0 * T * (K * N + r * (3 * K + 2 * N))}


def _ids(case, gen):
    """One adapter for each token, -1 for none: runs of tokens of one request, or each token its own request's."""
    T, L = case["T"], case["L"]
    if case["mix"] == "tokens":
        ids = torch.randint(0, L, (T,), generator=gen, device="cuda")
        bare = torch.rand(T, generator=gen, device="cuda") < case["bare"]
    else:
        runs = L + 2
        cuts = torch.randint(0, T + 1, (runs - 1,), generator=gen, device="cuda")
        run = (torch.arange(T, device="cuda")[:, None] >= cuts[None, :]).sum(1)
        ids = torch.randint(0, L, (runs,), generator=gen, device="cuda")[run]
        bare = (torch.rand(runs, generator=gen, device="cuda") < case["bare"])[run]
    return torch.where(bare, -1, ids).to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)
    dtype = DTYPES[case["dtype"]]
    wide = torch.float64 if dtype is torch.float64 else torch.float32

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=wide).mul_(std).to(dtype)

    def activations(T, n, pad=0):
        # channels of unequal size, as activations have them
        channel = torch.randn(n, generator=gen, device="cuda", dtype=wide).mul_(0.5).exp_()
        x = torch.randn(T, n, generator=gen, device="cuda", dtype=wide).mul_(channel)
        buffer = torch.zeros(T, n + pad, device="cuda", dtype=dtype)
        buffer[:, :n] = x
        return buffer

    s = {"case": case, "T": case["T"]}
    if case["op"] == "moe":
        T, H, width, E = (case[n] for n in ("T", "H", "I", "E"))
        s["x"] = activations(T, H)
        s["router"] = normal(E, H, std=H ** -0.5)
        s["w1"] = normal(E, 2 * width, H, std=H ** -0.5)
        s["w2"] = normal(E, H, width, std=width ** -0.5)
        s["residual"] = normal(T, H)
        s["y"] = torch.empty(T, H, device="cuda", dtype=dtype)
    else:
        T, K, N, r, L = (case[n] for n in ("T", "K", "N", "r", "L"))
        s["ids"] = _ids(case, gen)
        s["scale"] = torch.rand(L, generator=gen, device="cuda", dtype=wide) + 0.5
        s["x"] = activations(T, K, case["pad"])
        s["w"] = normal(N, K, std=K ** -0.5)
        s["a"] = normal(L, r, K, std=K ** -0.5)
        s["b"] = normal(L, N, r, std=r ** -0.5)
        if case["op"] == "lora":
            s["y"] = torch.empty(T, N, device="cuda", dtype=dtype)
        else:
            s["dy"] = normal(T, N, std=0.01)
            s["dx"] = torch.empty(T, K, device="cuda", dtype=dtype)
            s["da"], s["db"] = torch.empty_like(s["a"]), torch.empty_like(s["b"])
    if own:
        s["plan"] = _plan(s)
    return s


_ctx = None


def _plan(s):
    """The taskpool that a program keeps and runs for every batch in the same buffers."""
    global _ctx
    import dplasma_amd as dp
    if _ctx is None:
        _ctx = dp.init(device="cuda:0")
    case = s["case"]

    def matrix(t, rows, nb):
        """Rows of ``t`` as columns of a descriptor; blocks of nb columns are its tiles."""
        t2 = t.view(-1, t.shape[-1])
        return dp.TiledMatrix(t.dtype, rows, nb, rows, t2.shape[0], device=t.device, storage="lapack",
                              lld=t2.shape[1], data=t)

    T = case["T"]
    if case["op"] == "moe":
        H, width, E = case["H"], case["I"], case["E"]
        return dp.moe_New(_ctx, case["k"], case["norm"], matrix(s["router"], H, E), matrix(s["w1"], H, 2 * width),
                          matrix(s["w2"], width, H), 1.0, matrix(s["x"], H, T), case["beta"], matrix(s["y"], H, T))
    K, N, r = case["K"], case["N"], case["r"]
    w, x = matrix(s["w"], K, N), matrix(s["x"], K, T)
    a, b = matrix(s["a"], K, r), matrix(s["b"], r, N)
    if case["op"] == "lora":
        return dp.gemm_lora_New(_ctx, 1.0, w, x, a, b, s["ids"], s["scale"], 0.0, matrix(s["y"], N, T))
    return dp.gemm_lora_grad_New(_ctx, 1.0, w, x, a, b, s["ids"], s["scale"], matrix(s["dy"], N, T),
                                 matrix(s["dx"], K, T), matrix(s["da"], K, r), matrix(s["db"], r, N))


def run(s):
    op = s["case"]["op"]
    if own:
        if op == "moe" and s["case"]["beta"]:
            s["y"].copy_(s["residual"])
        s["plan"].run(_ctx)
        return {"lora": lambda: s["y"], "moe": lambda: s["y"],
                "grad": lambda: {"dx": s["dx"], "da": s["da"], "db": s["db"]}}[op]()
    return {"lora": _plain_lora, "grad": _plain_grad, "moe": _plain_moe}[op](s)


def _wide(t):
    return t if t.dtype is torch.float64 else t.float()


def _chosen(s):
    """[T, L] in the working precision: the scale of each token's adapter in its column, zero elsewhere."""
    hot = s["ids"][:, None] == torch.arange(s["a"].shape[0], device="cuda", dtype=torch.int32)[None, :]
    return torch.where(hot, s["scale"][None, :], torch.zeros((), device="cuda", dtype=s["scale"].dtype))


def _plain_lora(s):
    L, r, K = s["a"].shape
    T, N = s["T"], s["w"].shape[0]
    x, chosen = _wide(s["x"][:, :K]), _chosen(s)
    low = (x @ _wide(s["a"]).view(L * r, K).t()).view(T, L, r) * chosen[:, :, None]
    b = _wide(s["b"]).transpose(1, 2).reshape(L * r, N)
    return (x @ _wide(s["w"]).t() + low.view(T, L * r) @ b).to(s["w"].dtype)


def _plain_grad(s):
    L, r, K = s["a"].shape
    T, N = s["T"], s["w"].shape[0]
    x, dy, chosen = _wide(s["x"][:, :K]), _wide(s["dy"]), _chosen(s)
    a = _wide(s["a"]).view(L * r, K)
    b = _wide(s["b"]).transpose(1, 2).reshape(L * r, N)
    low = ((x @ a.t()).view(T, L, r) * chosen[:, :, None]).view(T, L * r)
    back = ((dy @ b.t()).view(T, L, r) * chosen[:, :, None]).view(T, L * r)
    dx = dy @ _wide(s["w"]) + back @ a
    da = (back.t() @ x).view(L, r, K)
    db = (low.t() @ dy).view(L, r, N).transpose(1, 2).contiguous()
    dtype = s["w"].dtype
    return {"dx": dx.to(dtype), "da": da.to(dtype), "db": db.to(dtype)}


def _plain_moe(s):
    case = s["case"]
    T, k, width, E = case["T"], case["k"], case["I"], case["E"]
    # the choice of experts lies next to a border where two logits nearly agree: 64 bits
    logits = s["x"].double() @ s["router"].double().t()
    p = torch.exp(logits - logits.amax(1, keepdim=True))
    p = p / p.sum(1, keepdim=True)
    order = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k]
    weight = torch.gather(p, 1, order)
    if case["norm"]:
        weight = weight / weight.sum(1, keepdim=True)
    x = _wide(s["x"])
    route = torch.zeros(T, E, device="cuda", dtype=torch.float64).scatter_(1, order, weight).to(x.dtype)
    both = (x @ _wide(s["w1"]).view(E * 2 * width, -1).t()).view(T, E, 2, width)
    gate, up = both[:, :, 0], both[:, :, 1]
    act = gate / (1 + torch.exp(-gate)) * up * route[:, :, None]
    y = torch.bmm(_wide(s["w2"]), act.permute(1, 2, 0).contiguous()).sum(0).t()
    if case["beta"]:
        y = y + case["beta"] * _wide(s["residual"])
    return y.to(s["x"].dtype).contiguous()


def exact(case, seed):
    s = prepare(case, seed)
    d = {n: v.double() for n, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    if case["op"] == "moe":
        return _exact_moe(case, d)
    K, L = case["K"], case["L"]
    x = d["x"][:, :K]
    groups = [(l, torch.nonzero(s["ids"] == l).flatten()) for l in range(L)]
    if case["op"] == "lora":
        y = x.matmul(d["w"].t())
        for l, rows in groups:
            y[rows] += d["scale"][l] * x[rows].matmul(d["a"][l].t()).matmul(d["b"][l].t())
        return y
    dx = d["dy"].matmul(d["w"])
    da, db = torch.zeros_like(d["a"]), torch.zeros_like(d["b"])
    for l, rows in groups:
        back = d["scale"][l] * d["dy"][rows].matmul(d["b"][l])
        dx[rows] += back.matmul(d["a"][l])
        da[l] = back.t().matmul(x[rows])
        db[l] = d["scale"][l] * d["dy"][rows].t().matmul(x[rows].matmul(d["a"][l].t()))
    return {"dx": dx, "da": da, "db": db}


def _exact_moe(case, d):
    k, width = case["k"], case["I"]
    x = d["x"]
    p = torch.softmax(x.matmul(d["router"].t()), 1)
    y = case["beta"] * d["residual"]
    left, total = p.clone(), torch.zeros_like(p[:, 0])
    picks = []
    for _ in range(k):
        best = left.max(1).values
        e = (left == best[:, None]).to(torch.int8).argmax(1)  # the lowest index of the largest
        picks.append((e, best))
        total += best
        left.scatter_(1, e[:, None], -1.0)
    for e, weight in picks:
        if case["norm"]:
            weight = weight / total
        for one in torch.unique(e).tolist():
            rows = torch.nonzero(e == one).flatten()
            both = x[rows].matmul(d["w1"][one].t())
            gate, up = both[:, :width], both[:, width:]
            act = gate * torch.sigmoid(gate) * up
            y[rows] += weight[rows, None] * act.matmul(d["w2"][one].t())
    return y
