"""Products whose matrix depends on the column on the CPU: definitions, gradients, refusals, the testing driver."""
import pytest
import torch

import dplasma_amd as dp
from indexed_cases import HALF, Lora, Moe, matrix, within

S, D, H, B = torch.float32, torch.float64, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def ctx():
    return dp.init(device="cpu")


LORA = [(D, 7, 12, 9, 3, 4, "tokens", 0), (S, 33, 40, 21, 5, 3, "runs", 4), (B, 5, 64, 32, 8, 2, "tokens", 8),
        (H, 1, 17, 19, 1, 1, "one", 0), (D, 6, 8, 8, 4, 3, "none", 0), (D, 0, 8, 8, 4, 2, "none", 0),
        (D, 5, 8, 8, 4, 0, "none", 0), (D, 5, 0, 8, 4, 2, "one", 0), (D, 5, 8, 0, 4, 2, "one", 0)]


@pytest.mark.parametrize("case", LORA, ids=str)
@pytest.mark.parametrize("alpha,beta,scale", [(1.0, 0.0, True), (0.5, -2.0, True), (0.0, 1.5, False)])
def test_lora_cpu(ctx, case, alpha, beta, scale):
    c = Lora(*case)
    y = c.forward(ctx, alpha, beta, scale)
    within(y[:, :c.N], *c.plain(alpha, beta, scale), "y")
    assert torch.equal(y[:, c.N:], c.y[:, c.N:])


@pytest.mark.parametrize("case", LORA, ids=str)
def test_lora_grad_cpu(ctx, case):
    c = Lora(*case)
    dx, da, db = c.backward(ctx, 0.75)
    for got, (want, bound), what in zip((dx[:, :c.K], da, db), c.plain_backward(0.75), ("dx", "da", "db")):
        within(got, want, bound, what)
    assert (dx[:, c.K:] == 7).all()


def test_lora_grad_is_the_differences(ctx):
    """Directional differences of the forward product: it is quadratic along (x, a, b), so the central difference is
    exact up to the third order term, which is below 1e-9 at this step."""
    c = Lora(D, 9, 11, 7, 3, 3)
    dx, da, db = c.backward(ctx, 1.25)
    gen = torch.Generator().manual_seed(1)
    step = {n: torch.randn(getattr(c, n).shape, generator=gen, dtype=D) for n in "xab"}
    eps, value = 1e-4, []
    base = {n: getattr(c, n).clone() for n in "xab"}
    for sign in (1, -1):
        for n in "xab":
            setattr(c, n, base[n] + sign * eps * step[n])
        value.append(float((c.forward(ctx, 1.25) * c.dy).sum()))
    slope = (value[0] - value[1]) / (2 * eps)
    exact = sum(float((g * step[n]).sum()) for g, n in ((dx, "x"), (da, "a"), (db, "b")))
    assert abs(slope - exact) < 1e-6 * (1 + abs(exact))


def test_lora_grad_parts_alone(ctx):
    c = Lora(D, 9, 11, 7, 3, 3)
    whole = c.backward(ctx)
    for want in ("x", "a", "b", "ab"):
        for n, one, all_ in zip("xab", c.backward(ctx, want=want), whole):
            assert torch.equal(one, all_ if n in want else torch.full_like(one, 7.0))


@pytest.mark.parametrize("case", [(D, 5, 12, 9, 6, 2), (S, 11, 32, 24, 8, 3), (B, 3, 64, 16, 5, 5), (H, 1, 24, 16, 4, 1),
                                  (D, 0, 8, 8, 4, 2), (D, 3, 8, 0, 4, 2)], ids=str)
@pytest.mark.parametrize("norm,alpha,beta", [(True, 1.0, 0.0), (False, 0.5, 1.0)])
def test_moe_cpu(ctx, case, norm, alpha, beta):
    c = Moe(*case)
    within(c.forward(ctx, norm, alpha, beta), *c.plain(norm, alpha, beta), "y")


def test_moe_ties_go_to_the_lowest_index(ctx):
    c = Moe(D, 4, 8, 6, 5, 2)
    c.g[:] = c.g[0]  # every logit equal
    within(c.forward(ctx), *c.plain())


def test_old_values_are_not_read_without_beta(ctx):
    c = Lora(D, 5, 8, 6, 2, 2)
    c.y.fill_(float("nan"))
    assert torch.isfinite(c.forward(ctx)).all()
    m = Moe(D, 5, 8, 6, 4, 2)
    m.y.fill_(float("nan"))
    assert torch.isfinite(m.forward(ctx)).all()


def test_tile_storage_and_views(ctx):
    """Tiles that span all rows, and column views of a larger block row, are the same matrices."""
    c = Lora(D, 6, 8, 5, 2, 4, "one")
    W, X, A, Bd = c.descriptors()
    At = dp.block_cyclic(ctx, D, 8, 2, 8, 8)
    At.from_dense(c.a.view(-1, 8).t())
    y1, y2 = c.y.clone(), c.y.clone()
    dp.dgemm_lora(ctx, 1.0, W, X, A, Bd, c.ids, None, 0.0, matrix(y1))
    dp.dgemm_lora(ctx, 1.0, W, X, At, Bd, c.ids, None, 0.0, matrix(y2))
    assert torch.equal(y1, y2)
    last = c.ids - 2  # adapters 2 and 3 alone
    dp.gemm_lora(ctx, 1.0, W, X, At.submatrix(0, 4, 8, 4), Bd.submatrix(0, 10, 2, 10), last, None, 0.0, matrix(y2))
    assert torch.equal(y1, y2)


def test_precision_aliases(ctx):
    c = Lora(B, 3, 8, 8, 2, 2)
    W, X, A, Bd = c.descriptors()
    dp.bgemm_lora(ctx, 1.0, W, X, A, Bd, c.ids, None, 0.0, matrix(c.y))
    for fn in (dp.dgemm_lora, dp.hgemm_lora, dp.sgemm_lora_New):
        with pytest.raises(TypeError):
            fn(ctx, 1.0, W, X, A, Bd, c.ids, None, 0.0, matrix(c.y))
    for name in ("dmoe", "hmoe_New", "bgemm_lora_grad", "sgemm_lora_grad_New", "gemm_lora_Destruct", "moe_Destruct"):
        assert hasattr(dp, name)
    assert not hasattr(dp, "zmoe")


def _lora_args(c):
    W, X, A, Bd = c.descriptors()
    return dict(W=W, X=X, A=A, B=Bd, ids=c.ids, scale=c.scale, Y=matrix(c.y))


def _shared(c):
    return matrix(c.x.view(-1)[:c.T * c.N].view(c.T, c.N))


@pytest.mark.parametrize("change,error", [
    (lambda c, a: a.update(W=matrix(c.w[:, 1:].contiguous())), ValueError),                    # K differs
    (lambda c, a: a.update(Y=matrix(c.y[1:])), ValueError),                                    # T differs
    (lambda c, a: a.update(X=matrix(c.x.float())), TypeError),                                 # precision differs
    (lambda c, a: a.update(X=matrix(c.x.to(torch.complex128))), TypeError),
    (lambda c, a: a.update(A=matrix(c.a.view(-1, c.K)[:-1], c.r)), ValueError),                # a torn tile
    (lambda c, a: a.update(B=matrix(c.b[1:].reshape(-1, c.r), c.N)), ValueError),              # fewer adapters in B
    (lambda c, a: a.update(B=matrix(c.b.view(-1, c.r), c.r)), ValueError),                     # B's tile width
    (lambda c, a: a.update(ids=c.ids.long()), ValueError),
    (lambda c, a: a.update(ids=c.ids[1:]), ValueError),
    (lambda c, a: a.update(ids=torch.stack([c.ids, c.ids], 1)[:, 0]), ValueError),             # strided
    (lambda c, a: a.update(ids=list(range(c.T))), ValueError),
    (lambda c, a: a.update(scale=c.scale[1:]), ValueError),
    (lambda c, a: a.update(scale=c.scale.float()), ValueError),
    (lambda c, a: a.update(Y=_shared(c)), ValueError),                                         # Y inside X
    (lambda c, a: a.update(W=dp.TiledMatrix(D, 4, c.N, c.K, c.N)), ValueError),                # tiles that cut the rows
    (lambda c, a: a.update(W=dp.TiledMatrix(D, c.K, c.N, c.K, c.N, P=2)), ValueError),         # distributed
    (lambda c, a: a.update(W=dp.TiledMatrix(D, c.K, c.N, c.K, c.N, alloc=False)), ValueError),
    (lambda c, a: a.update(W=dp.TiledMatrix(D, c.K, c.N, c.K, c.N, storage="lapack",
                                            data=torch.zeros(c.N, c.K, dtype=D).t())), ValueError),  # not contiguous
])
def test_lora_refusals(ctx, change, error):
    c = Lora(D, 6, 10, 7, 3, 4)
    a = _lora_args(c)
    change(c, a)
    before = c.y.clone()
    with pytest.raises(error):
        dp.gemm_lora(ctx, 1.0, a["W"], a["X"], a["A"], a["B"], a["ids"], a["scale"], 0.0, a["Y"])
    assert torch.equal(c.y, before)


def test_lora_grad_refusals(ctx):
    c = Lora(D, 6, 10, 7, 3, 4)
    W, X, A, Bd = c.descriptors()
    dY, dX = matrix(c.dy), matrix(torch.zeros_like(c.x))
    dA, dB = matrix(torch.zeros_like(c.a).view(-1, c.K), c.r), matrix(torch.zeros_like(c.b).view(-1, c.r), c.N)
    for bad in (dict(dX=X), dict(dA=A), dict(dB=Bd), dict(dX=dY), dict(dA=matrix(torch.zeros(12, 10, dtype=D))),
                dict(dB=dA), dict(dY=matrix(c.dy[1:]))):
        args = dict(dY=dY, dX=dX, dA=dA, dB=dB)
        args.update(bad)
        with pytest.raises(ValueError):
            dp.gemm_lora_grad(ctx, 1.0, W, X, A, Bd, c.ids, c.scale, **args)


@pytest.mark.parametrize("change,error", [
    (lambda c, a: a.update(topk=0), ValueError), (lambda c, a: a.update(topk=c.E + 1), ValueError),
    (lambda c, a: a.update(G=matrix(c.g[1:])), ValueError),
    (lambda c, a: a.update(W1=matrix(c.w1.view(-1, c.H), c.I)), ValueError),
    (lambda c, a: a.update(W2=matrix(c.w2.view(-1, c.I), c.I)), ValueError),
    (lambda c, a: a.update(W2=matrix(c.w2[1:].reshape(-1, c.I), c.H)), ValueError),
    (lambda c, a: a.update(Y=matrix(c.x)), ValueError), (lambda c, a: a.update(Y=matrix(c.y[1:])), ValueError),
    (lambda c, a: a.update(G=matrix(c.g.float())), TypeError),
    (lambda c, a: a.update(G=matrix(torch.zeros(5000, c.H, dtype=D))), ValueError),
])
def test_moe_refusals(ctx, change, error):
    c = Moe(D, 4, 8, 6, 5, 2)
    G, W1, W2, X = c.descriptors()
    a = dict(topk=2, G=G, W1=W1, W2=W2, X=X, Y=matrix(c.y))
    change(c, a)
    with pytest.raises(error):
        dp.moe(ctx, a["topk"], True, a["G"], a["W1"], a["W2"], 1.0, a["X"], 0.0, a["Y"])


def test_columns_side_by_side_in_one_buffer(ctx):
    """An output whose columns lie between an input's columns in one buffer does not overlap it."""
    c = Lora(D, 5, 8, 6, 2, 2)
    both = torch.zeros(6, 14, dtype=D)
    both[:5, :8] = c.x
    W, _, A, Bd = c.descriptors()
    X = matrix(both[:5], cols=8)
    Y = dp.TiledMatrix(D, 6, 5, 6, 5, storage="lapack", lld=14, data=both.view(-1)[8:])
    dp.gemm_lora(ctx, 1.0, W, X, A, Bd, c.ids, c.scale, 0.0, Y)
    within(both[:5, 8:], *c.plain())
    assert torch.equal(both[:5, :8], c.x) and not both[5].any()


DRIVER = ["bgemm_lora -N 96 -M 70 -K 64 -i 8 -x", "dgemm_lora -N 50 -M 9 -x --nruns 2", "hgemm_lora_grad -N 96 -M 70 -K 64 -x",
          "sgemm_lora_grad -N 40 -M 30 -K 64 -x -a 0.5", "bmoe -N 64 -K 48 -x", "dmoe -N 40 -M 5 -x"]


@pytest.mark.parametrize("args", DRIVER)
def test_testing_driver(args, capsys):
    from dplasma_amd import testing
    assert testing.main(args.split() + ["-g", "0"]) == 0
    out = capsys.readouterr().out
    assert "[****] TIME(s)" in out and "CORRECT" in out and "SUSPICIOUS" not in out


@pytest.mark.parametrize("args", ["bpotrf -N 40", "hgemm -N 40", "zmoe -N 40", "cgemm_lora -N 40"])
def test_testing_driver_refuses_other_precisions(args):
    from dplasma_amd import testing
    with pytest.raises(SystemExit):
        testing.main(args.split() + ["-g", "0"])


def test_run_of_a_lone_task_is_traced(ctx, tmp_path):
    """A taskpool of one task leaves its spans where tracing is on."""
    c = Lora(D, 5, 8, 8, 4, 2)
    tr = dp.profiling_start(ctx)
    try:
        c.forward(ctx)
    finally:
        dp.profiling_stop(ctx, str(tmp_path / "t.json"))
    assert "GEMM_LORA" in (tmp_path / "t.json").read_text()


def test_extents_past_a_launch_are_refused(ctx):
    """Ranks and families that no grid holds (storage that is never touched)."""
    r = 262144
    W, X, Y = matrix(torch.zeros(1, 1)), matrix(torch.zeros(2, 1)), matrix(torch.zeros(2, 1))
    A, Bd, ids = matrix(torch.empty(r, 1), r), matrix(torch.empty(1, r), 1), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="rank"):
        dp.gemm_lora(ctx, 1.0, W, X, A, Bd, ids, None, 0.0, Y)
    L, K = 65535, 33000
    W, X, Y = matrix(torch.empty(1, K, dtype=H)), matrix(torch.empty(2, K, dtype=H)), matrix(torch.empty(2, 1, dtype=H))
    A, Bd = matrix(torch.empty(L, K, dtype=H), 1), matrix(torch.empty(L, 1, dtype=H), 1)
    with pytest.raises(ValueError, match="tiles of 256"):
        dp.gemm_lora_grad(ctx, 1.0, W, X, A, Bd, ids, None, Y, matrix(torch.empty(2, K, dtype=H)), None, None)


def _rebind(descriptors):
    """Another tensor in the place of every descriptor's storage."""
    for M in descriptors:
        M.data = torch.full_like(M.data, float("nan"))


def test_a_taskpool_keeps_its_storages(ctx):
    """Tensors bound to the descriptors after a taskpool was built are not its operands."""
    c, m = Lora(D, 6, 10, 7, 3, 4), Moe(D, 4, 8, 6, 5, 2)
    ops, y = list(c.descriptors()), torch.zeros_like(c.y)
    dY, outs = matrix(c.dy), [torch.zeros_like(v) for v in (c.x, c.a, c.b)]
    dX, dA, dB = matrix(outs[0]), matrix(outs[1].view(-1, c.K), c.r), matrix(outs[2].view(-1, c.r), c.N)
    Y = matrix(y)
    one = dp.gemm_lora_New(ctx, 1.0, *ops, c.ids, c.scale, 0.0, Y)
    two = dp.gemm_lora_grad_New(ctx, 1.0, *ops, c.ids, c.scale, dY, dX, dA, dB)
    G, W1, W2, X = m.descriptors()
    out = torch.zeros_like(m.y)
    Z = matrix(out)
    three = dp.moe_New(ctx, 2, True, G, W1, W2, 1.0, X, 0.0, Z)
    _rebind([*ops, dY, dX, dA, dB, Y, G, W1, W2, X, Z])
    for tp in (one, two, three):
        tp.execute(ctx)
    within(y, *c.plain(), "y")
    for got, (want, bound), what in zip(outs, c.plain_backward(), ("dx", "da", "db")):
        within(got, want, bound, what)
    within(out, *m.plain(), "moe")


def test_workgroups_past_a_launch_are_refused(ctx):
    """Extents that fit a grid's axes and have more threads than a launch holds (storage that is never touched)."""
    L, K = 65535, 32640  # 65535 x 128 tiles of 256 features are below 2^23, with the windows of the tokens they are not
    W, X, dY = matrix(torch.empty(K, K, dtype=H)), matrix(torch.empty(2, K, dtype=H)), matrix(torch.empty(2, K, dtype=H))
    A, Bd = matrix(torch.empty(L, K, dtype=H), 1), matrix(torch.empty(L * K, 1, dtype=H), K)
    dA, dB = matrix(torch.empty(L, K, dtype=H), 1), matrix(torch.empty(L * K, 1, dtype=H), K)
    with pytest.raises(ValueError, match="tiles of 256"):
        dp.gemm_lora_grad_New(ctx, 1.0, W, X, A, Bd, torch.zeros(2, dtype=torch.int32), None, dY, None, dA, dB)
    wide = 16 * (2 ** 23 - 1) + 1  # 2^23 workgroups of 512 threads
    for h, i in ((wide, 1), (1, wide)):
        x, y, g = (matrix(torch.empty(1, h, dtype=H)) for _ in range(3))
        w1, w2 = matrix(torch.empty(2 * i, h, dtype=H), 2 * i), matrix(torch.empty(h, i, dtype=H), h)
        with pytest.raises(ValueError, match="features"):
            dp.moe_New(ctx, 1, True, g, w1, w2, 1.0, x, 0.0, y)
