"""Bias gradients behind an activation: column sums of the gradient before it is rounded.

Whole numbers: the derivative of ReLU and of none is 0 or 1, so sums of small whole numbers are exact in fp32 in any order.

Against fp64: a slope of the kernels is b = (8 + 7 |x|) 2^-24 of its two terms off at most (test_linear_tails_gpu.py derives it).  dy is drawn
independently of it with either sign alike, so the error of a column's sum has the variance sum dy^2 b^2 at most, and the norm over all
columns sqrt(sum over everything dy^2 b^2), to 10 % for the hundreds of columns here: 1.2 times that; additions in fp32 of up to 16 numbers a
thread at these sizes, 2^-24 of a running sum each: 4 2^-24 sqrt(sum dpre^2) covers them.  The sums of rounded high and low parts are two to three
times that bound off."""
import math

import pytest
import torch

from test_linear_gpu import BF16, F32, Framed, near, rnd, slope, value
from test_linear_tails_gpu import relative, slope_terms

pytestmark = pytest.mark.gpu

SIZES = [(1, 8), (3, 24), (33, 8), (70, 520), (257, 136), (1000, 1032), (1023, 2736), (2050, 72), (4097, 504), (9001, 4096), (100_003, 16), (5, 66_000)]


def whole(*shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + sum(shape))
    return torch.randint(-2, 3, shape, generator=g, device="cuda").to(dtype)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("M,N", SIZES)
def test_whole_numbers(ctx, M, N, dtype):
    from sirius_amd import ops
    dy, pre = whole(M, N, dtype=dtype, seed=1), whole(M, 2 * N, dtype=dtype, seed=2)
    g, up = pre[:, :N].double(), pre[:, N:].double()
    d = dy.double()
    for i, (act, split) in enumerate((("relu", True), ("none", True), ("relu", False))):
        wide, accumulate = i != 1, i == 1
        s = (g > 0).double() if act == "relu" else torch.ones_like(g)
        value_ = g.clamp(min=0) if act == "relu" else g
        src, z, dz = Framed(M, N, dtype, wide, dy), Framed(M, 2 * N, dtype, wide, pre), Framed(M, N, dtype, wide)
        db = Framed(1, N, F32, False)
        db.view.fill_(5.0)
        need = ops.act_bwd_workspace_bytes(dy)
        ws = torch.full((need + 64,), 99, dtype=torch.uint8, device="cuda")
        low = Framed(M, N, dtype, wide) if dtype == BF16 else None
        ops.act_bwd(ctx, src.view, z.view[:, :N], dz.view, act, dz_low=low.view if low else None, dbias=db.view, accumulate=accumulate,
                    workspace=ws[:need] if split else None)
        assert torch.equal(dz.view.double(), d * s), act
        assert torch.equal(db.view.double(), (d * s).sum(0, keepdim=True) + 5 * accumulate), act
        for f in (dz, db, low):
            if f:
                f.check(act)
        assert bool((ws[need:] == 99).all()) and (low is None or not bool(low.view.any()))
        # gated, dpre over pre
        want = torch.cat([d * up * s, d * value_], 1)
        h, db = Framed(M, N, dtype, wide), Framed(1, 2 * N, F32, False)
        db.view.fill_(5.0)
        need = ops.act_bwd_workspace_bytes(dy, gated=True)
        ws = torch.full((need + 64,), 99, dtype=torch.uint8, device="cuda")
        ops.gated_act_bwd(ctx, src.view, z.view, z.view, act, h=h.view, dbias=db.view, accumulate=accumulate, workspace=ws[:need] if split else None)
        assert torch.equal(z.view.double(), want) and torch.equal(h.view.double(), value_ * up), act
        assert torch.equal(db.view.double(), want.sum(0, keepdim=True) + 5 * accumulate), act
        z.check(act)
        db.check(act)
        assert bool((ws[need:] == 99).all())


@pytest.mark.parametrize("with_low", [True, False], ids=["low", "rounded"])
@pytest.mark.parametrize("M,K,N", [(1023, 64, 2736), (2000, 72, 520), (4096, 64, 1024)])
def test_backward_passes(ctx, M, K, N, with_low):
    """linear_bwd and gated_linear_bwd in bf16, with a workspace: dbias is that of the unrounded gradient, whether dw is or not."""
    from sirius_amd import ops
    x, w = rnd(M, K, dtype=BF16, seed=1), rnd(2 * N, K, dtype=BF16, seed=2, std=1 / math.sqrt(K))
    dy, pre = rnd(M, N, dtype=BF16, seed=3), rnd(M, 2 * N, dtype=BF16, seed=4, std=0.5)
    z, up = pre[:, :N].double(), pre[:, N:].double()
    d = dy.double()
    cdf, rest = slope_terms(z, "silu")
    off = d * (relative(z, "silu", BF16) + 4 * 2.0 ** -24) * (cdf.abs() + rest.abs())

    def check(db, exact, off):
        bound = 1.2 * float((off ** 2).sum().sqrt()) + 4 * 2.0 ** -24 * float((exact ** 2).sum().sqrt())
        err = float((db.double() - exact.sum(0)).norm())
        assert err <= bound, (err, bound)

    def new(*shape, dtype=BF16):
        return torch.empty(shape, dtype=dtype, device="cuda")
    dx, dpre = new(M, K), new(M, N)
    dw, db = new(N, K, dtype=F32), new(N, dtype=F32)
    ws = new(ops.linear_bwd_workspace_bytes(x, N), dtype=torch.uint8)
    ops.linear_bwd(ctx, dy, x, w[:N].t().contiguous(), dx, dw, dbias=db, act="silu", pre=pre[:, :N].contiguous(), dpre=dpre, workspace=ws,
                   dpre_low=new(M, N) if with_low else None)
    check(db, d * (cdf + rest), off)
    again = torch.full_like(db, 3.0)
    ops.linear_bwd(ctx, dy, x, None, None, dw, dbias=again, act="silu", pre=pre[:, :N].contiguous(), dpre=dpre, workspace=ws, accumulate=True)
    near(again, db.double() + 3, 2.0 ** -23 * (db.double().abs() + 3), "accumulated")
    dpre, dw, db = new(M, 2 * N), new(2 * N, K, dtype=F32), new(2 * N, dtype=F32)
    ws = new(ops.linear_bwd_workspace_bytes(x, 2 * N), dtype=torch.uint8)
    ops.gated_linear_bwd(ctx, dy, x, w.t().contiguous(), dx, dw, pre, dpre, dbias=db, workspace=ws, dpre_low=new(M, 2 * N) if with_low else None)
    check(db[:N], d * up * (cdf + rest), off * up)
    check(db[N:], d * value(z, "silu"), d * relative(z, "silu", BF16) * value(z, "silu").abs())


def test_refusals(ctx):
    from sirius_amd import ops
    from sirius_amd._lib import TorchColHipError
    dy, pre = rnd(9000, 4096, dtype=BF16, seed=1), rnd(9000, 4096, dtype=BF16, seed=2)
    dz, db = torch.empty_like(dy), torch.empty(4096, device="cuda")
    need = ops.act_bwd_workspace_bytes(dy)
    assert need > 4096
    for kind, call in [
            (AssertionError, lambda: ops.act_bwd(ctx, dy, pre, dz, "silu", dbias=db[:8])),
            (AssertionError, lambda: ops.act_bwd(ctx, dy, pre, dz, "silu", dbias=db.to(BF16))),
            (AssertionError, lambda: ops.gated_act_bwd(ctx, dy[:, :2048], pre, dz, dbias=db[:2048])),
            (AssertionError, lambda: ops.act_bwd(ctx, dy, pre, dz, "silu", dbias=db, workspace=torch.empty(need, dtype=torch.uint8))),
            (TorchColHipError, lambda: ops.act_bwd(ctx, dy, pre, dz, "silu", dbias=db, workspace=torch.empty(need // 2, dtype=torch.uint8, device="cuda"))),
            (TorchColHipError, lambda: ops.act_bwd(ctx, dy, pre, dz, "silu", dbias=dz.view(torch.float32).view(-1)[:4096])),
            (TorchColHipError, lambda: ops.act_bwd(ctx, dy, pre, dz, "silu", dbias=db, workspace=pre.view(torch.uint8).view(-1)[:need]))]:
        with pytest.raises(kind):
            call()


def test_no_rows(ctx):
    from sirius_amd import ops
    none, db = torch.empty(0, 64, dtype=BF16, device="cuda"), torch.full((64,), 5.0, device="cuda")
    ops.act_bwd(ctx, none, none, none, "silu", dbias=db, accumulate=True)
    assert bool((db == 5).all())
    ops.act_bwd(ctx, none, none, none, "silu", dbias=db)
    assert bool((db == 0).all())


def test_captured_graph(ctx):
    """A backward pass with its bias gradient as a graph: every replay on new inputs has the eager result's bits."""
    from sirius_amd import ops
    M, K, N = 1023, 264, 520
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        c = ops.Context(stream)
        x, w = rnd(M, K, dtype=BF16, seed=1), rnd(N, K, dtype=BF16, seed=2, std=0.06)
        wt, dy, pre = w.t().contiguous(), rnd(M, N, dtype=BF16, seed=3), rnd(M, N, dtype=BF16, seed=4)
        dx, dpre, low = torch.empty_like(x), torch.empty_like(dy), torch.empty_like(dy)
        dw, db = torch.empty(N, K, device="cuda"), torch.empty(N, device="cuda")
        ws = torch.empty(ops.linear_bwd_workspace_bytes(x, N), dtype=torch.uint8, device="cuda")

        def step():
            ops.linear_bwd(c, dy, x, wt, dx, dw, dbias=db, act="gelu", pre=pre, dpre=dpre, dpre_low=low, workspace=ws)
        step()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
        for i in range(3):
            dy.copy_(rnd(M, N, dtype=BF16, seed=50 + i))
            graph.replay()
            stream.synchronize()
            got = [t.clone() for t in (dx, dw, db)]
            for t in (dx, dw, db):
                t.fill_(-3.0)
            step()
            stream.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, (dx, dw, db))), i
