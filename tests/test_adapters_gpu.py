"""Products whose matrix depends on the column, on the GPU, against plain 64-bit forms (indexed_cases.py has the bounds)."""
import pytest
import torch

import dplasma_amd as dp
from indexed_cases import Lora, Moe, matrix, within

pytestmark = pytest.mark.gpu

S, D, H, B = torch.float32, torch.float64, torch.float16, torch.bfloat16
INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module")
def ctx():
    return dp.init(device="cuda:0")


def lora(*case, **kw):
    return Lora(*case, device="cuda:0", **kw)


def moe(*case, **kw):
    return Moe(*case, device="cuda:0", **kw)


# dtype, tokens, in, out, rank, adapters, ids, padding of the activations' rows
SMALL = [
    (B, 1, 64, 64, 16, 2, "one", 0), (B, 1, 2048, 512, 16, 4, "tokens", 0), (H, 1, 33, 5, 3, 1, "one", 0),
    (B, 2, 256, 256, 8, 3, "tokens", 8), (B, 15, 520, 264, 12, 7, "tokens", 0), (H, 16, 512, 1000, 16, 16, "tokens", 0),
    (H, 17, 1001, 333, 5, 6, "tokens", 3), (B, 31, 768, 130, 64, 4, "runs", 2), (B, 48, 1024, 2048, 16, 32, "tokens", 0),
    (H, 64, 640, 640, 32, 64, "tokens", 0), (B, 64, 256, 256, 100, 3, "runs", 0), (S, 1, 65, 67, 4, 2, "one", 0),
    (S, 30, 100, 90, 8, 3, "tokens", 1), (D, 12, 70, 66, 5, 4, "tokens", 0), (D, 1, 31, 30, 2, 2, "one", 0),
]
LARGE = [
    (B, 65, 512, 512, 16, 5, "runs", 0), (B, 128, 1000, 776, 8, 20, "tokens", 8), (H, 200, 1001, 515, 12, 9, "tokens", 5),
    (H, 257, 64, 257, 16, 4, "runs", 0), (B, 300, 2048, 1024, 64, 8, "runs", 64), (B, 512, 4096, 256, 32, 3, "runs", 0),
    (H, 511, 130, 1030, 7, 3, "tokens", 0), (B, 1024, 1024, 2048, 16, 6, "runs", 0), (B, 333, 256, 256, 200, 2, "runs", 0),
    (B, 2048, 520, 520, 16, 1, "one", 0), (S, 200, 256, 300, 16, 4, "runs", 0), (D, 130, 100, 200, 9, 5, "tokens", 4),
    (B, 300, 8, 16, 4, 3, "tokens", 0), (H, 90, 1, 1, 1, 2, "tokens", 0), (B, 100, 300, 200, 16, 4, "none", 0),
    (S, 1000, 64, 130, 8, 3, "runs", 0),
]


@pytest.mark.parametrize("case", SMALL + LARGE, ids=str)
def test_lora(ctx, case):
    c = lora(*case)
    for alpha, beta, scale in ((1.0, 0.0, True), (-0.5, 2.0, False)):
        y = c.forward(ctx, alpha, beta, scale)
        within(y[:, :c.N], *c.plain(alpha, beta, scale), f"alpha={alpha}")
        assert torch.equal(y[:, c.N:], c.y[:, c.N:])
        assert torch.equal(y, c.forward(ctx, alpha, beta, scale))


@pytest.mark.parametrize("case", SMALL + LARGE, ids=str)
def test_lora_grad(ctx, case):
    c = lora(*case)
    first = c.backward(ctx, 0.75)
    for got, (want, bound), what in zip((first[0][:, :c.K], *first[1:]), c.plain_backward(0.75), ("dx", "da", "db")):
        within(got, want, bound, what)
    assert (first[0][:, c.K:] == 7).all()
    for one, two in zip(first, c.backward(ctx, 0.75)):
        assert torch.equal(one, two)


# sizes on both sides of every choice between the kernels' variants: features per workgroup and launches of one token, two
# fragments of features for few tokens, tiles of 64, 128 and 256 with each number of buffers, through registers and
# directly to LDS, one and two fragments of tokens of the low-rank vectors
VARIANTS = [
    (B, 1, 300, 2500, 20, 2, "one", 0), (H, 1, 256, 4097, 8, 2, "one", 0), (D, 1, 130, 2100, 32, 2, "one", 0),
    (S, 1, 64, 40, 33, 2, "one", 0), (B, 20, 72, 8200, 16, 3, "tokens", 0), (H, 40, 40, 8193, 70, 4, "tokens", 0),
    (B, 64, 64, 8192, 8, 9, "tokens", 0), (S, 50, 72, 8200, 8, 3, "tokens", 0), (D, 64, 40, 520, 8, 3, "tokens", 0),
    (B, 1536, 72, 1664, 16, 4, "runs", 0), (H, 1536, 1664, 72, 8, 5, "tokens", 8), (B, 1700, 1704, 1704, 16, 3, "runs", 0),
    (H, 2100, 72, 2100, 32, 6, "tokens", 0), (B, 2100, 2104, 72, 16, 2, "runs", 0), (S, 1700, 136, 1704, 8, 3, "runs", 0),
    (S, 2100, 68, 2100, 16, 3, "tokens", 0), (B, 1700, 201, 1703, 12, 5, "runs", 0), (H, 1700, 1703, 201, 12, 5, "tokens", 1),
    (D, 130, 101, 201, 9, 5, "tokens", 0), (D, 300, 256, 512, 16, 2, "runs", 0), (B, 4100, 200, 2600, 16, 5, "runs", 0),
    (H, 4100, 2600, 136, 24, 7, "tokens", 8), (B, 8200, 136, 1304, 64, 9, "tokens", 0), (H, 8200, 1304, 136, 20, 4, "runs", 0),
    (B, 8200, 264, 72, 8, 300, "tokens", 0), (H, 8200, 64, 64, 130, 1, "one", 0),
]


@pytest.mark.parametrize("case", VARIANTS, ids=str)
def test_lora_variants(ctx, case):
    c = lora(*case)
    y = c.forward(ctx, -0.5, 2.0)
    within(y[:, :c.N], *c.plain(-0.5, 2.0), "y")
    assert torch.equal(y[:, c.N:], c.y[:, c.N:]) and torch.equal(y, c.forward(ctx, -0.5, 2.0))
    first = c.backward(ctx)
    for got, (want, bound), what in zip((first[0][:, :c.K], *first[1:]), c.plain_backward(), ("dx", "da", "db")):
        within(got, want, bound, what)
    assert (first[0][:, c.K:] == 7).all()
    for one, two in zip(first, c.backward(ctx)):
        assert torch.equal(one, two)


@pytest.mark.parametrize("case", [(B, 300, 512, 256, 16, 3, "runs", 0), (H, 40, 256, 300, 8, 5, "tokens", 0)], ids=str)
def test_lora_grad_parts_alone(ctx, case):
    c = lora(*case)
    whole = c.backward(ctx)
    for want in ("x", "a", "b", "ab", "xb"):
        for n, one, all_ in zip("xab", c.backward(ctx, want=want), whole):
            assert torch.equal(one, all_ if n in want else torch.full_like(one, 7.0)), (want, n)


@pytest.mark.parametrize("case", [(B, 40, 256, 320, 8, 4, "tokens", 0), (B, 260, 512, 512, 16, 3, "runs", 0)], ids=str)
def test_lora_grad_is_the_differences(ctx, case):
    """The gradient along a direction against central differences of the plain 64-bit forward product.  The gradient's
    own bound, summed over the direction, is what the sum may be off by; the differences add their third order."""
    c = lora(*case)
    c.dy = c.dy.abs()
    dx, da, db = c.backward(ctx)
    (_, bx), (_, ba), (_, bb) = c.plain_backward()
    gen = torch.Generator().manual_seed(3)
    step = {n: torch.randn(getattr(c, n).shape, generator=gen, dtype=D).cuda() for n in "xab"}
    got = sum(float((g.double() * step[n]).sum()) for g, n in ((dx, "x"), (da, "a"), (db, "b")))
    room = sum(float((g * step[n].abs()).sum()) for g, n in ((bx, "x"), (ba, "a"), (bb, "b")))
    base = {n: getattr(c, n).double() for n in "xab"}
    dtype, value = c.dtype, []
    for sign in (1, -1):
        for n in "xab":
            setattr(c, n, base[n] + sign * 1e-4 * step[n])
        value.append(float((c.plain()[0] * c.dy.double()).sum()))
    c.dtype = dtype
    slope = (value[0] - value[1]) / 2e-4
    assert abs(slope - got) < room + 1e-6 * (1 + abs(slope))


@pytest.mark.parametrize("T,dtype", [(1, B), (20, H), (64, B), (150, B), (600, H), (150, S)])
def test_lora_keeps_one_adapters_infinities(ctx, T, dtype):
    """Infinities and NaN in one adapter, one token or one output's weights stay there."""
    c = lora(dtype, T, 256, 264, 8, 4, "tokens")
    want, bound = c.plain()
    c.a[1], c.b[1, ::2] = INF, NAN
    c.x[T // 2, 5] = NAN
    c.w[7] = INF
    y = c.forward(ctx)
    ok = (c.ids != 1)[:, None].expand(T, 264).clone()
    ok[T // 2], ok[:, 7] = False, False
    within(torch.where(ok, y.double(), want), want, bound)
    assert not torch.isfinite(y[:, 7]).any() and torch.isnan(y[T // 2]).all()
    if (c.ids == 1).any():
        assert not torch.isfinite(y[c.ids == 1]).any()


@pytest.mark.parametrize("T,dtype", [(20, H), (150, B), (600, B), (150, S)])
def test_lora_grad_keeps_one_adapters_infinities(ctx, T, dtype):
    c = lora(dtype, T, 256, 264, 8, 4, "tokens")
    (dx, bx), (da, ba), (db, bb) = c.plain_backward()
    c.a[1], c.b[1] = INF, NAN
    mine = c.ids == 1
    c.dy[mine] = NAN
    gx, ga, gb = c.backward(ctx)
    ok = ~mine
    within(gx[ok], dx[ok], bx[ok], "dx")
    keep = [0, 2, 3]
    within(ga[keep], da[keep], ba[keep], "da")
    within(gb[keep], db[keep], bb[keep], "db")


@pytest.mark.parametrize("dtype", [H, B])
def test_lora_low_rank_vectors_past_half_range(ctx, dtype):
    """A^T x beyond fp16's largest number, with a B small enough that the result is ordinary."""
    for T in (3, 150):
        c = lora(dtype, T, 512, 320, 8, 2, "one")
        c.x *= 100
        c.a *= 2000
        c.b *= 2.0 ** -14
        within(c.forward(ctx), *c.plain())
        for got, (want, bound) in zip(c.backward(ctx), c.plain_backward()):
            ok = want.abs() + bound < torch.finfo(dtype).max
            within(torch.where(ok, got.double(), want), want, bound)


def test_lora_rows_far_into_a_long_buffer(ctx):
    """Activations whose offsets pass 2^31 elements."""
    T, K, N, ld = 70, 64, 72, 2 ** 25
    c = lora(B, T, K, N, 8, 3, "tokens")
    far = torch.empty(T * ld, dtype=B, device="cuda:0")
    far.view(T, ld)[:, :K] = c.x
    W, X, A, Bd = c.descriptors()
    X = dp.TiledMatrix(B, K, T, K, T, device="cuda:0", storage="lapack", lld=ld, data=far)
    y = torch.empty(T, N, dtype=B, device="cuda:0")
    dp.gemm_lora(ctx, 1.0, W, X, A, Bd, c.ids, c.scale, 0.0, matrix(y))
    want, bound = c.plain()
    within(y, want, bound)
    for t in (0, 30, 69):  # one token at the far end, by a view of the columns
        dp.gemm_lora(ctx, 1.0, W, dp.TiledMatrix(B, K, 1, K, T, device="cuda:0", storage="lapack", lld=ld, data=far)
                     .submatrix(0, t, K, 1), A, Bd, c.ids[t:t + 1], c.scale, 0.0, matrix(y[t:t + 1]))
    within(y, want, bound)


@pytest.mark.parametrize("off", [1, 3, 8])
def test_lora_unaligned_storage(ctx, off):
    """Matrices that begin at any element of their buffers."""
    for T in (5, 100):
        c = lora(B, T, 128, 96, 8, 3, "tokens")

        def moved(t):
            buf = torch.zeros(t.numel() + off, dtype=t.dtype, device="cuda:0")
            buf[off:] = t.reshape(-1)
            return buf[off:].view(t.shape)

        want, bound = c.plain()
        back = c.plain_backward()
        c.x, c.w, c.a, c.b, c.y, c.dy = (moved(t) for t in (c.x, c.w, c.a, c.b, c.y, c.dy))
        y = moved(torch.zeros_like(c.y))
        W, X, A, Bd = c.descriptors()
        dp.gemm_lora(ctx, 1.0, W, X, A, Bd, c.ids, c.scale, 0.0, matrix(y))
        within(y, want, bound)
        dx, da, db = (moved(torch.zeros_like(t)) for t in (c.x, c.a, c.b))
        dp.gemm_lora_grad(ctx, 1.0, W, X, A, Bd, c.ids, c.scale, matrix(c.dy), matrix(dx), matrix(da.view(-1, 128), 8),
                          matrix(db.view(-1, 8), 96))
        for got, (v, e) in zip((dx, da, db), back):
            within(got, v, e)


def test_lora_nothing_to_do(ctx):
    for case in ((B, 0, 64, 64, 8, 2, "none"), (B, 5, 64, 64, 8, 0, "none"), (B, 5, 0, 64, 8, 2, "one"),
                 (B, 100, 64, 0, 8, 2, "none")):
        c = lora(*case)
        y = c.forward(ctx, 1.0, 1.0)
        within(y[:, :c.N], *c.plain(1.0, 1.0))
        dx, da, db = c.backward(ctx)
        for got, (want, bound) in zip((dx, da, db), c.plain_backward()):
            within(got, want, bound)


MOE = [(B, 1, 64, 32, 4, 1), (B, 1, 2048, 1024, 64, 8), (B, 2, 512, 256, 8, 2), (H, 5, 333, 77, 5, 3), (B, 16, 256, 264, 16, 4),
       (H, 24, 1000, 728, 30, 3), (B, 37, 520, 136, 10, 10), (B, 64, 512, 128, 64, 8), (B, 64, 256, 64, 2, 2),
       (H, 64, 130, 50, 3, 1), (B, 100, 264, 72, 7, 2), (B, 200, 128, 64, 2, 1), (S, 3, 100, 60, 6, 2), (S, 20, 256, 130, 9, 3),
       (D, 9, 65, 33, 5, 2), (D, 1, 128, 64, 8, 8), (B, 7, 1, 1, 3, 2), (B, 4, 64, 32, 300, 5), (H, 2, 4096, 40, 4, 2),
       # the most experts of a token, the most experts, groups of 32 and 64 tokens of an expert on 4 and 8 waves, several
       # batches, shares of the second product
       (B, 1, 64, 32, 300, 256), (B, 5, 40, 16, 256, 256), (H, 3, 64, 16, 4096, 2), (B, 24, 2048, 64, 4, 2),
       (B, 64, 2048, 40, 2, 2), (S, 64, 300, 40, 2, 2), (S, 40, 1100, 24, 5, 2), (D, 40, 128, 40, 2, 2), (D, 30, 600, 24, 4, 2),
       (B, 150, 64, 300, 6, 6), (H, 129, 24, 1000, 12, 5)]


@pytest.mark.parametrize("case", MOE, ids=str)
def test_moe(ctx, case):
    c = moe(*case)
    for norm, alpha, beta in ((True, 1.0, 0.0), (False, -0.5, 2.0)):
        y = c.forward(ctx, norm, alpha, beta)
        within(y, *c.plain(norm, alpha, beta), f"norm={norm}")
        assert torch.equal(y, c.forward(ctx, norm, alpha, beta))


def test_moe_nothing_to_do(ctx):
    for case in ((B, 0, 64, 32, 4, 2), (B, 3, 64, 0, 4, 2)):
        c = moe(*case)
        within(c.forward(ctx, True, 1.0, 1.0), *c.plain(True, 1.0, 1.0))


def test_moe_ties_and_one_expert_for_all(ctx):
    c = moe(B, 20, 128, 64, 9, 3)
    c.g[:] = c.g[0]  # every logit equal: experts 0, 1, 2
    within(c.forward(ctx), *c.plain())
    c = moe(B, 64, 128, 64, 9, 1)
    c.x.abs_()
    c.g[:], c.g[5] = -1.0, 1.0  # every token the same expert
    within(c.forward(ctx), *c.plain())


def test_moe_close_logits_are_told_apart(ctx):
    """Two logits that agree to 2^-30 of their size: a sum in 32 bits would not see which is larger."""
    c = moe(S, 8, 512, 64, 4, 1)
    c.x[:], c.g[:] = 1.0, 0.0
    c.g[:, :256], c.g[:, 256:511] = 4.0, -4.0
    c.g[2, 511] = 2.0 ** -20
    c.g[3, 511] = 2.0 ** -20 * (1 + 2.0 ** -20)
    want, bound = c.plain()
    within(c.forward(ctx), want, bound)


def test_moe_keeps_infinities_apart(ctx):
    c = moe(B, 30, 256, 96, 8, 2)
    z = c.x.double() @ c.g.double().t()
    order = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :2]
    want, bound = c.plain()
    c.w1[3], c.w2[3] = INF, NAN
    hit = (order == 3).any(1)
    c.x[4] = NAN
    hit[4] = True
    y = c.forward(ctx)
    within(y[~hit], want[~hit], bound[~hit])
    assert not torch.isfinite(y[hit]).any()


@pytest.mark.parametrize("dtype", [H, B])
def test_moe_activations_past_half_range(ctx, dtype):
    c = moe(dtype, 6, 256, 96, 4, 2)
    c.w1 *= 100
    c.x *= 10
    c.w2 *= 2.0 ** -12
    want, bound = c.plain()
    assert want.abs().max() < 60000
    within(c.forward(ctx), want, bound)


def _layer(ctx, c, m, y, out):
    """An adapted projection, a mixture of experts added onto its result."""
    W, X, A, Bd = c.descriptors()
    G, W1, W2, _ = m.descriptors()
    one = dp.gemm_lora_New(ctx, 1.0, W, X, A, Bd, c.ids, c.scale, 0.0, matrix(y))
    two = dp.moe_New(ctx, m.k, True, G, W1, W2, 1.0, matrix(y), 0.0, matrix(out))
    return one, two


def _layer_plain(c, m):
    m.x = c.plain()[0].to(c.dtype)
    return m.plain()


def test_layers_together(ctx):
    """An adapted projection feeds a mixture of experts, through taskpools queued before one wait, and then again with
    other tokens and ids in the same buffers."""
    c, m = lora(B, 9, 256, 128, 8, 3, "tokens"), moe(B, 9, 128, 64, 6, 2)
    y, out = torch.empty(9, 128, dtype=B, device="cuda:0"), torch.empty(9, 128, dtype=B, device="cuda:0")
    pools = _layer(ctx, c, m, y, out)
    for _ in range(3):
        for tp in pools:
            ctx.add_taskpool(tp)
        ctx.start()
        ctx.wait()
        within(y, *c.plain())
        m.x = y
        within(out, *m.plain())
        c.x.copy_(torch.randn_like(c.x))
        c.ids.copy_(torch.flip(c.ids, [0]))
    for tp in pools:
        tp.destruct()


def test_training_step(ctx):
    """Forward, gradients and an update of the adapters: the gradients are those of the updated adapters each time."""
    c = lora(B, 200, 256, 192, 16, 3, "runs")
    W, X, A, Bd = c.descriptors()
    y = torch.empty(200, 192, dtype=B, device="cuda:0")
    dx, da, db = torch.empty_like(c.x), torch.empty_like(c.a), torch.empty_like(c.b)
    fwd = dp.bgemm_lora_New(ctx, 1.0, W, X, A, Bd, c.ids, c.scale, 0.0, matrix(y))
    bwd = dp.bgemm_lora_grad_New(ctx, 1.0, W, X, A, Bd, c.ids, c.scale, matrix(c.dy), matrix(dx),
                                 matrix(da.view(-1, 256), 16), matrix(db.view(-1, 16), 192))
    for _ in range(3):
        fwd.run(ctx)
        c.dy.copy_(y * 0.01)
        bwd.run(ctx)
        within(y, *c.plain())
        for got, (want, bound) in zip((dx, da, db), c.plain_backward()):
            within(got, want, bound)
        c.a.sub_(da * 0.1)
        c.b.sub_(db * 0.1)


def test_captured_and_replayed(ctx):
    """The products captured into a graph give each replay's inputs their eager result, with eager work between."""
    c, m = lora(B, 33, 512, 256, 16, 4, "tokens"), moe(B, 33, 256, 96, 8, 2)
    y, out = torch.empty(33, 256, dtype=B, device="cuda:0"), torch.empty(33, 256, dtype=B, device="cuda:0")
    dx, da, db = torch.empty_like(c.x), torch.empty_like(c.a), torch.empty_like(c.b)
    W, X, A, Bd = c.descriptors()
    pools = list(_layer(ctx, c, m, y, out))
    pools.append(dp.gemm_lora_grad_New(ctx, 1.0, W, X, A, Bd, c.ids, c.scale, matrix(c.dy), matrix(dx),
                                       matrix(da.view(-1, 512), 16), matrix(db.view(-1, 16), 256)))
    for tp in pools:
        tp.run(ctx)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for tp in pools:
            tp.run(ctx)
    gen = torch.Generator(device="cuda:0").manual_seed(5)
    for k in range(4):
        c.x.copy_(torch.randn(c.x.shape, generator=gen, device="cuda:0"))
        c.dy.copy_(torch.randn(c.dy.shape, generator=gen, device="cuda:0"))
        c.ids.copy_(torch.randint(-1, 4, c.ids.shape, generator=gen, device="cuda:0", dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in (y, out, dx, da, db)]
        within(y, *c.plain())
        m.x = y
        within(out, *m.plain())
        for tp in pools:
            tp.run(ctx)
        torch.cuda.synchronize()
        for one, two in zip(replayed, (y, out, dx, da, db)):
            assert torch.equal(one, two)


def test_two_at_once_on_two_streams(ctx):
    """Taskpools of their own on two streams, each on a stream that is not the one it was built on."""
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    work = []
    for k in range(2):
        c, m = lora(B, 40 + k, 512, 512, 16, 4, "tokens", seed=k), moe(B, 40 + k, 512, 128, 8, 2, seed=k)
        y, out = (torch.empty(40 + k, 512, dtype=B, device="cuda:0") for _ in range(2))
        work.append((c, m, y, out, _layer(ctx, c, m, y, out)))
    torch.cuda.synchronize()
    for _ in range(5):
        for s, (_, _, _, _, pools) in zip(streams, work):
            with torch.cuda.stream(s):
                for tp in pools:
                    tp.run(ctx)
    torch.cuda.synchronize()
    for c, m, y, out, _ in work:
        within(y, *c.plain())
        m.x = y
        within(out, *m.plain())


def test_storage_on_another_device_is_refused(ctx):
    c = lora(B, 4, 64, 64, 8, 2)
    W, X, A, Bd = c.descriptors()
    Y = matrix(c.y)
    with pytest.raises(ValueError):
        dp.gemm_lora(ctx, 1.0, matrix(c.w.cpu()), X, A, Bd, c.ids, None, 0.0, Y)
    with pytest.raises(ValueError):
        dp.gemm_lora(ctx, 1.0, W, X, A, Bd, c.ids.cpu(), None, 0.0, Y)


@pytest.mark.parametrize("args", ["bgemm_lora -N 2048 -M 300 -K 1024 -x", "hgemm_lora_grad -N 512 -M 700 -K 640 -x",
                                  "sgemm_lora_grad -N 300 -M 200 -x", "dgemm_lora -N 200 -M 20 -x", "bmoe -N 512 -K 256 -x --nruns 2"])
def test_testing_driver(args, capsys):
    from dplasma_amd import testing
    assert testing.main(args.split()) == 0
    out = capsys.readouterr().out
    assert "[****] TIME(s)" in out and "CORRECT" in out and "SUSPICIOUS" not in out


def test_traced_run(ctx, tmp_path):
    """A lone task's run with tracing on: the same result, and its span in the trace."""
    c = lora(B, 9, 256, 128, 8, 3, "tokens")
    plain = c.forward(ctx)
    dp.profiling_start(ctx)
    try:
        assert torch.equal(plain, c.forward(ctx))
    finally:
        dp.profiling_stop(ctx, str(tmp_path / "t.json"))
    assert "GEMM_LORA" in (tmp_path / "t.json").read_text()


def test_lora_grad_of_many_adapters(ctx):
    """More than 2^20 pieces of preparation, so that a workgroup takes several."""
    c = lora(B, 70, 1024, 8, 1, 60000, "tokens")
    c.ids[:] = torch.randint(0, 60000, (70,), generator=torch.Generator().manual_seed(2)).to(torch.int32)
    c.ids[:3] = torch.tensor([59999, 0, 59999], dtype=torch.int32)
    x, w, a, b, dy = (v.double() for v in (c.x, c.w, c.a, c.b, c.dy))
    dx, da, db = c.backward(ctx, 0.5)
    lid = c.ids.long()
    s = c.scale.double()[lid, None, None]
    p, q = s * dy[:, None, :] @ b[lid], s * x[:, None, :] @ a[lid].transpose(1, 2)
    # one rounding of the result, and within 2^-13 of the magnitudes: sums of at most 1024 + 70 + 8 + 16 products
    # in 32 bits (1118 2^-24 < 2^-13.8), the split intermediate (2^-16) and the rounding of these errors with the result
    want = 0.5 * (dy @ w + (p @ a[lid])[:, 0])
    room = 0.5 * (dy.abs() @ w.abs() + (p.abs() @ a[lid].abs())[:, 0])
    assert ((dx.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -13 * room).all()
    da_, db_ = torch.zeros_like(a), torch.zeros_like(b)
    da_.index_add_(0, lid, 0.5 * p.transpose(1, 2) * x[:, None, :])
    db_.index_add_(0, lid, 0.5 * dy[:, :, None] * q)
    room_a, room_b = torch.zeros_like(a), torch.zeros_like(b)
    room_a.index_add_(0, lid, 0.5 * (s * dy[:, None, :].abs() @ b[lid].abs()).transpose(1, 2) * x[:, None, :].abs())
    room_b.index_add_(0, lid, 0.5 * dy[:, :, None].abs() * (s * x[:, None, :].abs() @ a[lid].abs().transpose(1, 2)))
    assert ((da.double() - da_).abs() <= 2.0 ** -8 * da_.abs() + 2.0 ** -13 * room_a).all()
    assert ((db.double() - db_).abs() <= 2.0 ** -8 * db_.abs() + 2.0 ** -13 * room_b).all()


def test_moe_is_built_before_a_capture(ctx, monkeypatch):
    m = moe(B, 3, 64, 32, 4, 2)
    G, W1, W2, X = m.descriptors()
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="before the capture"):
        dp.moe_New(ctx, 2, True, G, W1, W2, 1.0, X, 0.0, matrix(m.y))


def _third(n, *lead):
    """Rows [1, 2^-5, 2^-9, 0 ..] and [1, 2^-5, 0 ..] of n: against [1, 2^-4, 2^-8, 0 ..] they give 1 + 2^-9 + 2^-17, which
    takes 18 bits, and 1 + 2^-9."""
    rows = torch.zeros(2, n, dtype=D)
    rows[:, :3] = torch.tensor([[1, 2.0 ** -5, 2.0 ** -9], [1, 2.0 ** -5, 0]], dtype=D)
    one = torch.tensor([1, 2.0 ** -4, 2.0 ** -8] + [0] * (n - 3), dtype=D)
    return rows, one


@pytest.mark.parametrize("T", [70, 600])
@pytest.mark.parametrize("dtype,b", [(B, 1.0), (H, 1.0), (H, 1 + 2.0 ** -10), (S, 1.0)])
def test_low_rank_vectors_keep_32_bits(ctx, T, dtype, b):
    """Two low-rank numbers that differ in their 18th bit, subtracted by the second product."""
    c = lora(dtype, T, 24, 72, 2, 1, "one")
    rows, one = _third(24)
    c.w.zero_()
    c.x[:], c.a[0] = one.to(c.x), rows.to(c.a)
    c.b[0, :, 0], c.b[0, :, 1] = b, -b
    # S is exact.  Its product with B is a sum of at most 12 numbers whose partial sums stay below 1.01, each rounded by
    # 2^-24 at most: 12 2^-24 1.01, times alpha, below 2^-10
    y = c.forward(ctx, 1024.0, scale=False).double()
    want = b * 2.0 ** -7
    assert ((y - want).abs() <= 2.0 ** -10 + 2.0 ** -8 * want).all(), float((y - want).abs().max())
    # dX = alpha (p_0 - p_1), the same numbers
    rows, one = _third(72)
    c.dy[:], c.b[0] = one.to(c.dy), rows.t().to(c.b)
    c.a[0, 0], c.a[0, 1] = b, -b
    dx = c.backward(ctx, 1024.0, scale=False)[0].double()
    assert ((dx - want).abs() <= 2.0 ** -10 + 2.0 ** -8 * want).all(), float((dx - want).abs().max())


@pytest.mark.parametrize("T", [70, 600, 5000])
@pytest.mark.parametrize("dtype,z", [(B, 1.0), (H, 1.0), (H, 1 + 2.0 ** -10), (S, 1.0)])
@pytest.mark.parametrize("r", [2, 20, 40])
def test_gradients_of_the_factors_keep_32_bits(ctx, T, dtype, z, r):
    """The low-rank numbers of even tokens are those of odd ones plus 2^-17, and the two meet opposite signs."""
    c = lora(dtype, T, 24, 72, r, 1, "one")
    sign = torch.where(torch.arange(T) % 2 == 0, z, -z)[:, None]
    # Every product of parts is a multiple of 2^-19, and no more than 16 tokens of one sign come one after the other (an
    # instruction adds 32), so partial sums below 2^4.1 are exact in 32 bits in any order, but for the products of the last
    # parts, 2^-10 of 2^-17 each; the result is rounded once.  Ranks past the first are not looked at
    room = 2.0 ** -8 + 2.0 ** -10
    for n, what in ((72, "a"), (24, "b")):
        rows, one = _third(n)
        every = one.repeat(T, 1)
        every[1::2, 2] = 0
        if what == "a":
            c.dy[:], c.b[0, :, 0] = every.to(c.dy), rows[0].to(c.b)
            c.x[:] = sign.to(c.x)
            got = c.backward(ctx, 1.0, scale=False, want="a")[1][0, 0]
        else:
            c.x[:], c.a[0, 0] = every.to(c.x), rows[0].to(c.a)
            c.dy[:] = sign.to(c.dy)
            got = c.backward(ctx, 1.0, scale=False, want="b")[2][0, :, 0]
        want = z * (T // 2) * 2.0 ** -17
        assert ((got.double() - want).abs() <= room * want).all(), (what, got[:4].tolist(), want)


@pytest.mark.parametrize("T,I", [(3, 2), (3, 256), (20, 2), (20, 256), (60, 2), (60, 256)])
@pytest.mark.parametrize("dtype,b", [(B, 1.0), (H, 1.0), (H, 1 + 2.0 ** -10), (S, 1.0)])
def test_moe_activations_keep_32_bits(ctx, T, I, dtype, b):
    """Two activations, 32 + 2^-4 + 2^-12 and 32 + 2^-4, subtracted by the down projection (silu(32) is 32 in 32 bits)."""
    c = moe(dtype, T, 40, I, 1, 1)
    rows, one = _third(40)
    c.x[:] = one.to(c.x)
    c.w1.zero_()
    c.w1[0, :I, 0] = 32
    c.w1[0, I:I + 2] = rows.to(c.w1)
    c.w2.zero_()
    c.w2[0, :, 0], c.w2[0, :, 1] = b, -b
    # as for the low-rank vectors, with partial sums below 33: 12 2^-24 33 1024 < 2^-5
    y = c.forward(ctx, True, 1024.0).double()
    want = b * 2.0 ** -2
    assert ((y - want).abs() <= 2.0 ** -5 + 2.0 ** -8 * want).all(), float((y - want).abs().max())


@pytest.mark.parametrize("case", [(H, 300, 520, 264, 24, 3, "runs", 0), (B, 300, 520, 264, 24, 3, "runs", 0),
                                  (B, 700, 264, 520, 64, 5, "runs", 0), (H, 900, 201, 333, 40, 4, "tokens", 1)], ids=str)
def test_lora_without_room_for_short_intermediates(ctx, case, monkeypatch):
    """The bounds of sums in 32 bits alone, nothing for an intermediate of fewer bits."""
    import indexed_cases
    monkeypatch.setattr(indexed_cases, "split_eps", lambda dtype: 0.0)
    c = lora(*case)
    within(c.forward(ctx)[:, :c.N], *c.plain(), "y")
    got = c.backward(ctx)
    for one, (want, bound), what in zip((got[0][:, :c.K], *got[1:]), c.plain_backward(), ("dx", "da", "db")):
        within(one, want, bound, what)


def test_a_taskpool_keeps_its_storages(ctx):
    """A taskpool's operands stay in memory when the descriptors are given other tensors and nobody else holds the old ones."""
    c, m = lora(B, 40, 512, 320, 16, 4, "tokens"), moe(B, 12, 256, 96, 8, 2)
    want, (back, _, _), mixed = c.plain(), c.plain_backward(), m.plain()
    ops = list(c.descriptors())
    Y, dY, dX = (matrix(v.clone()) for v in (c.y, c.dy, c.x))
    G, W1, W2, X = m.descriptors()
    Z = matrix(m.y.clone())
    one = dp.gemm_lora_New(ctx, 1.0, *ops, c.ids, c.scale, 0.0, Y)
    two = dp.gemm_lora_grad_New(ctx, 1.0, *ops, c.ids, c.scale, dY, dX, None, None)
    three = dp.moe_New(ctx, 2, True, G, W1, W2, 1.0, X, 0.0, Z)
    outs = [M.data for M in (Y, dX, Z)]
    # no tensor of the program's own: what only the descriptors held would return to the allocator here ...
    for name in ("x", "w", "a", "b", "dy"):
        setattr(c, name, None)
    for name in ("x", "g", "w1", "w2"):
        setattr(m, name, None)
    every = [*ops, Y, dY, dX, G, W1, W2, X, Z]
    sizes = [M.data.numel() for M in every]
    for M in every:
        M.data = None
    others = [torch.full((n,), NAN, dtype=B, device="cuda:0") for n in sizes for _ in range(2)]  # ... and be theirs
    for tp in (one, two, three):
        tp.execute(ctx)
    for got, (value, bound), what in zip(outs, (want, back, mixed), ("y", "dx", "moe")):
        within(got, value, bound, what)
    assert all(torch.isnan(o).all() for o in others)


# x of few tokens in whole lines: every number of fragments of tokens and of features that these kernels are made for, in 16
# and 32 bits, with waves that have no step, four, and one to four rounds of four more, and a last step that K ends inside
LINES = [
    (B, 1, 4096, 4200, 16, 4, "tokens", 0), (H, 1, 8192, 264, 40, 3, "one", 0), (B, 16, 4104, 264, 8, 5, "tokens", 8),
    (H, 9, 2048, 136, 70, 3, "tokens", 0), (S, 1, 2048, 130, 33, 2, "one", 0), (S, 16, 4100, 72, 8, 3, "tokens", 4),
    (S, 7, 1024, 264, 8, 3, "runs", 0), (B, 17, 4096, 264, 16, 4, "tokens", 0), (H, 32, 520, 136, 33, 6, "tokens", 0),
    (S, 20, 4100, 264, 8, 3, "tokens", 0), (S, 32, 256, 72, 8, 3, "tokens", 0), (H, 32, 4104, 8200, 12, 7, "tokens", 8),
    (B, 20, 8192, 8192, 16, 3, "runs", 0), (B, 18, 512, 8192, 8, 3, "tokens", 0), (S, 32, 2048, 8192, 8, 3, "tokens", 0),
    (S, 17, 260, 8196, 70, 2, "tokens", 0), (H, 48, 8192, 264, 16, 5, "tokens", 0), (B, 33, 2056, 520, 64, 4, "tokens", 8),
    (S, 40, 2048, 136, 8, 3, "tokens", 0), (B, 48, 4096, 8192, 16, 32, "tokens", 0), (H, 40, 1024, 8264, 24, 4, "tokens", 0),
    (S, 33, 1028, 8200, 8, 3, "tokens", 0), (S, 48, 4100, 8192, 8, 3, "runs", 4), (B, 64, 8192, 520, 16, 64, "tokens", 0),
    (H, 50, 4104, 264, 100, 3, "tokens", 8), (S, 64, 2052, 264, 8, 3, "tokens", 0), (H, 64, 4104, 8264, 16, 9, "tokens", 0),
    (B, 50, 1024, 8192, 8, 3, "tokens", 0), (S, 64, 4100, 8192, 8, 3, "tokens", 0),
]


@pytest.mark.parametrize("case", LINES, ids=str)
def test_lora_of_few_tokens_in_whole_lines(ctx, case):
    c = lora(*case)
    y = c.forward(ctx, -0.5, 2.0)
    within(y[:, :c.N], *c.plain(-0.5, 2.0), "y")
    assert torch.equal(y[:, c.N:], c.y[:, c.N:])
    for _ in range(3):
        assert torch.equal(y, c.forward(ctx, -0.5, 2.0))


def test_built_inside_a_capture(ctx):
    """gemm_lora and its gradient built and run while a graph is captured, with other work between the replays."""
    c = lora(B, 100, 256, 320, 16, 4, "tokens")
    y, dx = torch.empty(100, 320, dtype=B, device="cuda:0"), torch.empty_like(c.x)
    da, db = torch.empty_like(c.a), torch.empty_like(c.b)
    W, X, A, Bd = c.descriptors()

    def build():
        return (dp.gemm_lora_New(ctx, 1.0, W, X, A, Bd, c.ids, c.scale, 0.0, matrix(y)),
                dp.gemm_lora_grad_New(ctx, 1.0, W, X, A, Bd, c.ids, c.scale, matrix(c.dy), matrix(dx),
                                      matrix(da.view(-1, 256), 16), matrix(db.view(-1, 16), 320)))
    for tp in build():
        tp.execute(ctx)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pools = build()
        for tp in pools:
            tp.run(ctx)
    gen = torch.Generator(device="cuda:0").manual_seed(5)
    for _ in range(3):
        c.x.copy_(torch.randn(c.x.shape, generator=gen, device="cuda:0"))
        c.ids.copy_(torch.randint(-1, 4, c.ids.shape, generator=gen, device="cuda:0", dtype=torch.int32))
        other = [torch.full((1 << 20,), NAN, device="cuda:0") for _ in range(4)]
        graph.replay()
        torch.cuda.synchronize()
        within(y, *c.plain(), "y")
        for got, (want, bound), what in zip((dx, da, db), c.plain_backward(), ("dx", "da", "db")):
            within(got, want, bound, what)
        assert all(torch.isnan(o).all() for o in other)
    for tp in pools:
        tp.destruct()


@pytest.mark.parametrize("T", [70, 600])
def test_products_of_half_precision_keep_every_part(ctx, T):
    """The last 8 of a low-rank number's 24 bits against the last 3 of a half precision number's 11."""
    last, z = 255 * 2.0 ** -23, 1 + 7 * 2.0 ** -10
    c = lora(H, T, 24, 72, 2, 1, "one")
    c.w.zero_()
    first = torch.zeros(2, 72, dtype=D)  # against [1, 2^-4, 0 ..]: 1 + 2^-8 + last, and 1 + 2^-8
    first[:, 0], first[0, 1] = 1 + 2.0 ** -8, 16 * last
    one = torch.tensor([1, 2.0 ** -4] + [0] * 70, dtype=D)
    c.x[:], c.a[0] = one[:24].to(c.x), first[:, :24].to(c.a)
    c.b[0, :, 0], c.b[0, :, 1] = z, -z
    # all but the last parts cancel, each of a product's parts has at most 16 bits: sums are exact, the result is rounded once
    y = c.forward(ctx, 1024.0, scale=False).double()
    want = 1024 * z * last
    assert ((y - want).abs() <= 2.0 ** -11 * want).all(), float((y - want).abs().max() / want)
    c.dy[:], c.b[0] = one.to(c.dy), first.t().to(c.b)
    c.a[0, 0], c.a[0, 1] = z, -z
    dx = c.backward(ctx, 1024.0, scale=False, want="x")[0].double()
    assert ((dx - want).abs() <= 2.0 ** -11 * want).all(), float((dx - want).abs().max() / want)
    # even tokens have the last bits; T / 2 of these terms are summed, in 32 bits
    c.dy[1::2, 1] = 0
    c.x[:] = torch.where(torch.arange(T) % 2 == 0, z, -z)[:, None].to(c.x)
    da = c.backward(ctx, 1024.0, scale=False, want="a")[1][0, 0].double()
    want *= T // 2
    assert ((da - want).abs() <= (2.0 ** -11 + T * 2.0 ** -24) * want).all(), float((da - want).abs().max() / want)


@pytest.mark.parametrize("T", [3, 20, 60])
def test_experts_of_half_precision_keep_every_part(ctx, T):
    last, z = 255 * 2.0 ** -23, 1 + 7 * 2.0 ** -10
    c = moe(H, T, 40, 16, 1, 1)
    c.x.zero_(), c.w1.zero_(), c.w2.zero_()
    c.x[:, 0], c.x[:, 1] = 1, 2.0 ** -4
    c.w1[0, :16, 0] = 32  # silu(32) is 32 in 32 bits
    c.w1[0, 16:18, 0], c.w1[0, 16, 1] = 1 + 2.0 ** -8, 16 * last
    c.w2[0, :, 0], c.w2[0, :, 1] = z, -z
    y = c.forward(ctx, True, 1024.0).double()
    want = 1024 * 32 * z * last
    assert ((y - want).abs() <= 2.0 ** -11 * want).all(), float((y - want).abs().max() / want)
