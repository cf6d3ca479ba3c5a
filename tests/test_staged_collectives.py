"""Collectives on a program's tensors go through parallel.comm, which takes device tensors through host memory under gloo."""
import ast
from pathlib import Path

import torch

from helpers import run_distributed

COLLECTIVES = {"all_reduce", "all_gather", "all_gather_into_tensor", "all_to_all", "all_to_all_single", "broadcast", "reduce",
               "reduce_scatter", "reduce_scatter_tensor", "gather", "scatter"}
# calls of their own: what they move, under which condition
OWN = {"context.py": "RCCL alone (its communicators are brought up)",
       "models/gemm_ooc.py": "device tensors under RCCL, host buffers otherwise",
       "models/potrf_dtr_dist.py": "copied to host memory unless under RCCL"}


def test_no_collective_of_its_own():
    root = Path(__file__).resolve().parents[1] / "dplasma_amd"
    found = {}
    for f in sorted(root.rglob("*.py")):
        name = str(f.relative_to(root))
        if name == "parallel/comm.py":
            continue
        for node in ast.walk(ast.parse(f.read_text())):
            if isinstance(node, ast.Call) and isinstance(node.func, ast.Attribute) and node.func.attr in COLLECTIVES \
                    and isinstance(node.func.value, ast.Name) and node.func.value.id == "dist":
                found.setdefault(name, []).append(node.lineno)
    assert set(found) <= set(OWN), {n: v for n, v in found.items() if n not in OWN}


def _worker(rank, world, P):
    import torch.distributed as dist

    import dplasma_amd as dp
    from dplasma_amd import scalapack, testing
    from dplasma_amd.parallel import comm
    ctx = dp.init(device="cpu", P=P)
    inside, calls, plain, through = [0], [0], dist.all_reduce, comm.allreduce

    def allreduce(*a, **kw):
        inside[0] += 1
        calls[0] += 1
        try:
            return through(*a, **kw)
        finally:
            inside[0] -= 1

    def all_reduce(*a, **kw):
        assert inside[0], "a reduction of its own"
        return plain(*a, **kw)
    comm.allreduce, dist.all_reduce = allreduce, all_reduce
    comm._staged = lambda t: True  # as a device tensor under gloo
    counts, out = [], []

    def step(value):
        counts.append(calls[0])
        out.append(value)
    # tiles of another size: element by element
    A, C = dp.block_cyclic(ctx, torch.float64, 8, 8, 20, 20), dp.block_cyclic(ctx, torch.float64, 5, 5, 20, 20)
    dp.plrnt(ctx, A, 3)
    dp.redistribute(ctx, A, C, 10, 9, 3, 2, 4, 6)
    step((A.to_dense_local(), C.to_dense_local()))
    S = dp.block_cyclic(ctx, torch.float64, 8, 8, 24, 24)
    dp.plghe(ctx, 24.0, dp.dplasmaLower, S, 5)
    step(dp.potrf_dtd(ctx, dp.dplasmaLower, S))
    step(testing._dense(type("H", (), {"ctx": ctx}), A))
    W, tau = dp.block_cyclic(ctx, torch.float64, 8, 8, 80, 16), torch.zeros(16, dtype=torch.float64)
    gen = torch.Generator().manual_seed(1)
    W.from_dense(torch.randn(80, 16, generator=gen, dtype=torch.float64))
    desc = scalapack.descinit(80, 16, 8, 8, 0, 0, scalapack.blacs_gridinit(ctx), max(1, W.llmt * 8))
    local = torch.cat([torch.cat([W.tile(i, j) for i in W.rows], 0) for j in W.cols], 1).t().contiguous().view(-1)
    scalapack.pdlatsqr_(80, 16, local, 1, 1, desc, tau)
    step(tau)
    return counts, out


def test_reductions_of_device_tensors_under_gloo():
    got = run_distributed(_worker, 2, 2)
    (counts, one), (_, two) = got[0], got[1]
    assert all(b > a for a, b in zip([0] + list(counts), counts)), counts
    src, dst = one[0][0] + two[0][0], one[0][1] + two[0][1]
    want = torch.zeros(20, 20, dtype=torch.float64)
    want[4:14, 6:15] = src[3:13, 2:11]
    assert torch.equal(dst, want)
    assert one[1] == two[1] == 0
    assert torch.equal(one[2], src) and torch.equal(two[2], src)
    assert torch.equal(one[3], two[3]) and bool((one[3] != 0).any())
