"""The linear layers and the gradient clip where they can go wrong: values that are not finite in and around the operands, activations
far out, in-place forms, no rows at all, tensors beyond 2 GiB, captured graphs, several streams at once, and refused calls."""
import math

import pytest
import torch

from test_linear_gpu import ACTS, BF16, F32, half_step, near, product, rnd, slope, value

pytestmark = pytest.mark.gpu

# among them every kernel's: 16 x 16, dealt-out reductions of 32 and 64 rows, 128 x 64, 128 x 128, 256 x 128, 256 x 256 tiles
SHAPES = [(3, 4104, 4096), (5, 72, 40), (70, 264, 136), (520, 72, 520), (1000, 136, 1032), (2040, 264, 1544), (4090, 520, 2056)]


def poisoned(rows, cols, dtype, seed):
    """rows x cols values in the upper left of a larger matrix of NaN, its rows cols + 16 apart."""
    full = torch.full((rows + 40, cols + 16), float("nan"), dtype=dtype, device="cuda")
    full[:rows, :cols] = rnd(rows, cols, dtype=dtype, seed=seed)
    return full[:rows, :cols]


def behind(*shape, dtype, seed, std=1.0):
    """A dense tensor with NaN right behind it."""
    n = math.prod(shape)
    full = torch.full((n + 70_000,), float("nan"), dtype=dtype, device="cuda")
    full[:n] = rnd(*shape, dtype=dtype, seed=seed, std=std).reshape(-1)
    return full[:n].view(shape)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_what_lies_around_the_operands_does_not_count(ctx, M, K, N, dtype):
    from sirius_amd import ops
    F = N // 16 * 8
    x, pre = poisoned(M, K, dtype, 1), poisoned(M, 2 * N, dtype, 4)
    w, wg = behind(N, K, dtype=dtype, seed=2, std=0.1), behind(2 * F, K, dtype=dtype, seed=3, std=0.1)
    bias, res = behind(N, dtype=F32, seed=5), poisoned(M, N, dtype, 6)
    y, kept = torch.empty(M, N, dtype=dtype, device="cuda"), torch.empty(M, N, dtype=dtype, device="cuda")
    ops.linear_fwd(ctx, x, w, y, bias=bias, act="silu", residual=res, pre=kept)
    h, kept2 = torch.empty(M, F, dtype=dtype, device="cuda"), torch.empty(M, 2 * F, dtype=dtype, device="cuda")
    ops.gated_linear_fwd(ctx, x, wg, h, act="gelu", pre=kept2)
    dx, dpre, again = torch.empty_like(y), torch.empty(M, 2 * N, dtype=dtype, device="cuda"), torch.empty_like(y)
    ops.linear_dgrad(ctx, x, w, dx, act="gelu_tanh", pre=pre[:, :N], residual=res)
    ops.linear_dgrad_gated(ctx, x, w, pre, dpre, act="silu", h=again)
    for t in (y, kept, h, kept2, dx, dpre, again):
        assert bool(t.isfinite().all())
    xd, dyd = behind(M, K, dtype=dtype, seed=7), behind(M, N, dtype=dtype, seed=8)
    low = behind(M, N, dtype=dtype, seed=9) if dtype == BF16 else None
    dw, db = torch.empty(N, K, device="cuda"), torch.empty(N, device="cuda")
    ws = torch.full((ops.linear_bwd_workspace_bytes(xd, N) // 4 + 1,), float("nan"), device="cuda")
    ops.linear_wgrad(ctx, xd, dyd, dw, dbias=db, workspace=ws, dy_low=low)
    assert bool(dw.isfinite().all()) and bool(db.isfinite().all())


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_a_row_that_is_not_finite_stays_by_itself(ctx, M, K, N, dtype):
    from sirius_amd import ops
    x, w = rnd(M, K, dtype=dtype, seed=1), rnd(N, K, dtype=dtype, seed=2, std=0.1)
    bad = M // 2
    x[bad, K - 1] = float("nan")
    x[M - 1, 0] = float("inf")
    y, z = (torch.empty(M, N, dtype=dtype, device="cuda") for _ in range(2))
    ops.linear_fwd(ctx, x, w, y, act="gelu_tanh", pre=z)
    fine = torch.ones(M, dtype=torch.bool, device="cuda")
    fine[bad] = fine[M - 1] = False
    assert bool(y[fine].isfinite().all()) and bool(z[fine].isfinite().all())
    assert bool(y[bad].isnan().all()) and bool(z[bad].isnan().all())
    assert not bool(z[M - 1].isfinite().any())
    v = rnd(M, N, dtype=dtype, seed=3)
    pre = rnd(M, 2 * N, dtype=dtype, seed=4)
    pre[0, :] = float("nan")
    dpre = torch.empty_like(pre)
    ops.gated_act_bwd(ctx, v, pre, dpre, "silu")
    assert bool(dpre[0].isnan().all()) and bool(dpre[1:].isfinite().all())


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("act", ACTS)
def test_activations_far_out(ctx, act, dtype):
    """Values and slopes from the middle to the ends of the type: against fp64 where that is a number, and against the limits, 0 and 1,
    behind; an infinite pre-activation has the limit's slope, one that is not a number gives none."""
    from sirius_amd import ops
    mags = torch.tensor([0.0, 1e-30, 1e-8, 1e-3, 0.1, 0.5, 1, 2, 3, 4, 4.9, 5.2, 6, 8, 11, 15.9, 16.1, 20, 60, 103, 105, 1e3, 1e9, 1e19, 1e25, 3e38])
    z = torch.cat([mags, -mags, torch.tensor([math.inf, -math.inf, math.nan])]).to(dtype)
    z = torch.cat([z, z.new_zeros(64 - z.numel())]).cuda()
    u, e = half_step(dtype), torch.eye(8, dtype=dtype, device="cuda")
    # a layer that hands its bias on: products with zero weights
    x, w = torch.ones(3, 8, dtype=dtype, device="cuda"), torch.zeros(64, 8, dtype=dtype, device="cuda")
    y = torch.empty(3, 64, dtype=dtype, device="cuda")
    ops.linear_fwd(ctx, x, w, y, bias=z.float(), act=act)
    zd = z.double()
    finite = zd.isfinite()
    ref = value(zd, act)
    ref = torch.where(zd < -300, ref * 0 if act != "none" else ref, ref)     # fp64 reference without its own overflow
    for row in y:
        near(row[finite], ref[finite], 2.0 ** -20 * zd[finite].abs() * (zd[finite] > -104 if act not in ("none",) else 1) + u * ref[finite].abs() + 1e-37,
             "value")
    assert bool(y[:, z.isnan()].isnan().all())
    assert bool((y[:, z == math.inf] == math.inf).all())
    # slopes: the derivative times one
    one, dz = torch.ones(1, 64, dtype=dtype, device="cuda"), torch.empty(1, 64, dtype=dtype, device="cuda")
    ops.act_bwd(ctx, one, z.view(1, 64), dz, act)
    held = zd.clamp(-200, 200)
    ref = slope(held, act)
    ok = ~zd.isnan()
    near(dz[0][ok], ref[ok], 2.0 ** -19 + u * ref[ok].abs(), "slope")
    assert act == "none" or bool(dz[0][zd.isnan()].isnan().all())
    # the same slopes in the epilogues: one row, and enough rows for tiles
    for rows in (1, 300):
        dx = torch.empty(rows, 64, dtype=dtype, device="cuda")
        ops.linear_dgrad(ctx, e[:1].expand(rows, 8).contiguous(), torch.ones(64, 8, dtype=dtype, device="cuda"), dx, act=act,
                         pre=z.expand(rows, 64).contiguous())
        for row in (dx[0], dx[-1]):
            near(row[ok], ref[ok], 2.0 ** -19 + u * ref[ok].abs(), "slope in an epilogue")


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_in_place(ctx, M, K, N, dtype):
    """A residual that is the output, gradients written over what they are made of: the bits of the forms with places of their own."""
    from sirius_amd import ops
    x, w, res = rnd(M, K, dtype=dtype, seed=1), rnd(N, K, dtype=dtype, seed=2, std=0.1), rnd(M, N, dtype=dtype, seed=3)
    pre = rnd(M, 2 * N, dtype=dtype, seed=4)
    y, y2 = torch.empty_like(res), res.clone()
    ops.linear_fwd(ctx, x, w, y, act="silu", residual=res)
    ops.linear_fwd(ctx, x, w, y2, act="silu", residual=y2)
    assert torch.equal(y, y2)
    ops.linear_dgrad(ctx, x, w, y, residual=res)
    y2 = res.clone()
    ops.linear_dgrad(ctx, x, w, y2, residual=y2)
    assert torch.equal(y, y2)
    d, d2 = torch.empty_like(pre), pre.clone()
    ops.linear_dgrad_gated(ctx, x, w, pre, d, act="gelu")
    ops.linear_dgrad_gated(ctx, x, w, d2, d2, act="gelu")
    assert torch.equal(d, d2)
    ops.gated_act_bwd(ctx, res, pre, d, "gelu")
    d2 = pre.clone()
    ops.gated_act_bwd(ctx, res, d2, d2, "gelu")
    assert torch.equal(d, d2)
    ops.act_bwd(ctx, res, y, z := torch.empty_like(y), "silu")
    z2, z3 = res.clone(), y.clone()
    ops.act_bwd(ctx, z2, y, z2, "silu")
    ops.act_bwd(ctx, res, z3, z3, "silu")
    assert torch.equal(z, z2) and torch.equal(z, z3)


def test_no_rows(ctx):
    from sirius_amd import ops
    x, w = torch.empty(0, 64, dtype=BF16, device="cuda"), rnd(32, 64, dtype=BF16, seed=1)
    y, pre = torch.empty(0, 32, dtype=BF16, device="cuda"), torch.empty(0, 64, dtype=BF16, device="cuda")
    ops.linear_fwd(ctx, x, w, y, act="gelu", pre=torch.empty_like(y))
    ops.gated_linear_fwd(ctx, x, rnd(64, 64, dtype=BF16, seed=1), y, pre=pre)
    ops.linear_dgrad_gated(ctx, x, w, pre, torch.empty_like(pre))
    for dtype in (BF16, F32):
        dw, db = torch.full((32, 64), 5.0, device="cuda"), torch.full((32,), 5.0, device="cuda")
        xs, ys = x.to(dtype), y.to(dtype)
        wt = w.t().contiguous().to(dtype)
        ws = torch.empty(ops.linear_bwd_workspace_bytes(xs, 32), dtype=torch.uint8, device="cuda")
        ops.linear_bwd(ctx, ys, xs, wt, torch.empty_like(xs), dw, dbias=db, act="silu", pre=ys, dpre=torch.empty_like(ys), accumulate=True, workspace=ws)
        assert bool((dw == 5).all()) and bool((db == 5).all())
        ops.linear_bwd(ctx, ys, xs, wt, torch.empty_like(xs), dw, dbias=db, workspace=ws)
        assert bool((dw == 0).all()) and bool((db == 0).all())


def test_more_than_two_gigabytes(ctx):
    """Rows far behind 2 GiB and 4 GiB of an operand, an output and a gradient."""
    from sirius_amd import ops
    M, K, N = 2_200_000, 1024, 64       # x 4.5 GB
    x = torch.empty(M, K, dtype=BF16, device="cuda")
    pattern = rnd(5000, K, dtype=BF16, seed=1)
    for at in range(0, M, 5000):
        x[at:at + 5000] = pattern
    w = rnd(N, K, dtype=BF16, seed=2, std=1 / 32)
    y = torch.empty(M, N, dtype=BF16, device="cuda")
    ops.linear_fwd(ctx, x, w, y, act="silu")
    z, e = product(pattern, w)
    ref = value(z, "silu")
    tol = 1.2 * e + 2.0 ** -20 * z.abs()
    for at in (0, 1_045_000, 2_095_000, 2_195_000):     # about 2^31 and 2^32 bytes, and the end
        near(y[at:at + 5000], ref, tol + half_step(BF16) * (ref.abs() + tol), f"rows from {at}")
    # the gradient of the weights over all of these rows, and a data gradient as wide as x
    dw, db = torch.empty(N, K, device="cuda"), torch.empty(N, device="cuda")
    ws = torch.empty(ops.linear_bwd_workspace_bytes(x, N), dtype=torch.uint8, device="cuda")
    ops.linear_wgrad(ctx, x, y, dw, dbias=db, workspace=ws)
    ref = 440 * (y[:5000].double().t() @ pattern.double())
    sums = 440 * (y[:5000].double().abs().t() @ pattern.double().abs())
    # runs of at most 2^16 rows are added up one by one, their sums by the hundreds: 2^17 2^-24 of the magnitudes
    near(dw, ref, 2.0 ** -7 * sums, "dw")
    near(db, 440 * y[:5000].double().sum(0), 2.0 ** -7 * 440 * y[:5000].double().abs().sum(0), "db")
    dx = x
    wt = w.t().contiguous()
    ops.linear_dgrad(ctx, y, wt, dx)
    v, e = product(y[:5000], wt)
    for at in (0, 1_045_000, 2_095_000, 2_195_000):
        near(dx[at:at + 5000], v, e + half_step(BF16) * (v.abs() + e), f"dx from {at}")
    ops.act_bwd(ctx, x, x, x, "relu")
    assert bool((x[2_195_000:] == torch.where(v > 0, dx[:5000].double() * 0 + x[:5000].double(), torch.zeros_like(v)).to(BF16)).all())


def _graph_case(ctx, ops):
    M, C, F = 300, 264, 520
    x, w, wd = rnd(M, C, dtype=BF16, seed=1), rnd(2 * F, C, dtype=BF16, seed=2, std=0.06), rnd(C, F, dtype=BF16, seed=3, std=0.04)
    t = dict(x=x, dy=rnd(M, C, dtype=BF16, seed=4))
    wt, wdt = w.t().contiguous(), wd.t().contiguous()

    def new(*shape, dtype=BF16):
        return torch.zeros(shape, dtype=dtype, device="cuda")
    h, pre, y, dpre, low, h2, h2_low, dx = new(M, F), new(M, 2 * F), new(M, C), new(M, 2 * F), new(M, 2 * F), new(M, F), new(M, F), new(M, C)
    dw, dwd, db, norm = new(2 * F, C, dtype=F32), new(C, F, dtype=F32), new(2 * F, dtype=F32), new(1, dtype=F32)
    ws, wsd = new(ops.linear_bwd_workspace_bytes(x, 2 * F), dtype=torch.uint8), new(ops.linear_bwd_workspace_bytes(h, C), dtype=torch.uint8)
    table = ops.GradTable([dw, dwd, db])
    scratch = new(ops.grad_norm_workspace_bytes(table), dtype=torch.uint8)

    def step(c):
        ops.gated_linear_fwd(c, x, w, h, act="silu", pre=pre)
        ops.linear_fwd(c, h, wd, y, residual=x)
        ops.linear_dgrad_gated(c, t["dy"], wdt, pre, dpre, act="silu", h=h2, dpre_low=low, h_low=h2_low)
        ops.linear_wgrad(c, h2, t["dy"], dwd, workspace=wsd, x_low=h2_low)
        ops.linear_bwd(c, dpre, x, wt, dx, dw, dbias=db, workspace=ws, dy_low=low)
        ops.clip_grad_norm(c, table, 0.5, norm, scratch)
    return t, step, (y, dx, dw, dwd, db, norm, h2, pre)


def test_captured_graph(ctx):
    """A block forward and back and the clip as one captured graph: several replays on changing inputs, eager work in between, each
    the eager result's bits."""
    from sirius_amd import ops
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        c = ops.Context(stream)
        t, step, outs = _graph_case(c, ops)
        step(c)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step(c)
        for i in range(4):
            t["x"].copy_(rnd(*t["x"].shape, dtype=BF16, seed=50 + i))
            t["dy"].copy_(rnd(*t["dy"].shape, dtype=BF16, seed=60 + i))
            for o in outs:
                o.fill_(3.0)
            graph.replay()
            stream.synchronize()
            got = [o.clone() for o in outs]
            for o in outs:
                o.fill_(-3.0)
            step(c)
            stream.synchronize()
            for a, b in zip(got, outs):
                assert torch.equal(a, b), i


def test_two_streams_at_once(ctx):
    """Two programs of the same calls on two streams, each with its own tensors and workspaces: each gets what it gets alone."""
    from sirius_amd import ops
    cases = []
    for _ in range(2):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            c = ops.Context(stream)
            t, step, outs = _graph_case(c, ops)
            prog = ops.Program()
            c.begin_record(prog)
            step(c)
            c.end_record()
            c.run(prog)
            stream.synchronize()
            cases.append((c, prog, outs, [o.clone() for o in outs], stream, t))
    for _ in range(20):
        for c, prog, *_ in cases:
            c.run(prog)
    torch.cuda.synchronize()
    for _, _, outs, alone, *_ in cases:
        assert all(torch.equal(a, b) for a, b in zip(outs, alone))


def test_refusals(ctx):
    from sirius_amd import ops
    from sirius_amd._lib import TorchColHipError
    x, w, y = rnd(4, 64, dtype=BF16, seed=1), rnd(32, 64, dtype=BF16, seed=2), torch.empty(4, 32, dtype=BF16, device="cuda")
    ops.linear_fwd(ctx, x, w, y)
    bad = [
        (ValueError, lambda: ops.linear_fwd(ctx, x, w, y, act="tanh")),
        (AssertionError, lambda: ops.linear_fwd(ctx, x[:, :56], w, y)),                    # rows shorter than the layer
        (AssertionError, lambda: ops.linear_fwd(ctx, x, w, y[:3])),
        (AssertionError, lambda: ops.linear_fwd(ctx, x, w.float(), y)),
        (AssertionError, lambda: ops.linear_fwd(ctx, x, w, y.float())),
        (AssertionError, lambda: ops.linear_fwd(ctx, x, w, y, bias=torch.zeros(32, dtype=BF16, device="cuda"))),
        (AssertionError, lambda: ops.linear_fwd(ctx, x, w, y, bias=torch.zeros(31, device="cuda"))),
        (TypeError, lambda: ops.linear_fwd(ctx, x.half(), w.half(), y.half())),
        (ValueError, lambda: ops.linear_fwd(ctx, x.cpu(), w, y)),
        (ValueError, lambda: ops.linear_fwd(ctx, x, w.t().contiguous().t(), y)),           # weights that are not dense
        (ValueError, lambda: ops.linear_fwd(ctx, rnd(64, 4, dtype=BF16, seed=1).t(), w, y)),   # a row's elements apart
        (ValueError, lambda: ops.linear_fwd(ctx, x[:1].expand(4, 64), w, y)),              # rows on top of each other
        (TorchColHipError, lambda: ops.linear_fwd(ctx, torch.zeros(4, 68, dtype=BF16, device="cuda")[:, :64], w, y)),   # rows off the 16-byte grid
        (TorchColHipError, lambda: ops.linear_fwd(ctx, torch.zeros(4, 72, dtype=BF16, device="cuda")[:, 4:68], w, y)),
        (TorchColHipError, lambda: ops.linear_fwd(ctx, rnd(4, 60, dtype=BF16, seed=1), rnd(32, 60, dtype=BF16, seed=1), y)),
        (TorchColHipError, lambda: ops.linear_dgrad(ctx, x, w, y, act="silu")),            # a derivative without its pre-activations
        (AssertionError, lambda: ops.gated_linear_fwd(ctx, x, w[:31], y)),
        (AssertionError, lambda: ops.gated_linear_fwd(ctx, x, w, y)),                      # h is half as wide
        (AssertionError, lambda: ops.linear_bwd(ctx, y, x, None, None, torch.empty(32, 64, device="cuda"), act="silu", pre=y)),
        (AssertionError, lambda: ops.linear_bwd(ctx, y, x, None, None, torch.empty(64, 32, device="cuda"))),
        (AssertionError, lambda: ops.linear_bwd(ctx, y, x, None, None, None, dbias=torch.empty(32, device="cuda"))),
        (AssertionError, lambda: ops.linear_wgrad(ctx, x[:3], y, torch.empty(32, 64, device="cuda"))),
        (AssertionError, lambda: ops.linear_wgrad(ctx, x, y, torch.empty(32, 64, device="cuda"), dy_low=y.clone(), x_low=x.clone())),
        (AssertionError, lambda: ops.linear_wgrad(ctx, x, y, torch.empty(32, 64, device="cuda"), dy_low=y.t().contiguous().t())),
        (AssertionError, lambda: ops.linear_wgrad(ctx, x.float(), y.float(), torch.empty(32, 64, device="cuda"), dy_low=y.float())),
        (AssertionError, lambda: ops.linear_wgrad(ctx, torch.zeros(4, 128, dtype=BF16, device="cuda")[:, :64], y, torch.empty(32, 64, device="cuda"))),
    ]
    for i, (kind, call) in enumerate(bad):
        with pytest.raises(kind):
            call()
            print("not refused:", i)
    big = rnd(4096, 1024, dtype=BF16, seed=1)
    dy = rnd(4096, 4096, dtype=BF16, seed=1)
    need = ops.linear_bwd_workspace_bytes(big, 4096)
    assert need > 4
    with pytest.raises(TorchColHipError):       # a workspace that is too small is no invitation to write behind it
        ops.linear_wgrad(ctx, big, dy, torch.empty(4096, 1024, device="cuda"), workspace=torch.empty(need // 2, dtype=torch.uint8, device="cuda"))


def test_outputs_that_overlap_are_refused(ctx):
    from sirius_amd import ops
    from sirius_amd._lib import TorchColHipError

    def new(*shape, dtype=BF16):
        return torch.zeros(*shape, dtype=dtype, device="cuda")
    M, N = 40, 64
    wide, w, pre = new(M, 4 * N), rnd(N, N, dtype=BF16, seed=1, std=0.1), rnd(M, 2 * N, dtype=BF16, seed=2)
    wide.copy_(rnd(M, 4 * N, dtype=BF16, seed=3))
    col = [wide[:, i * N:(i + 1) * N] for i in range(4)]
    want = new(M, N)
    ops.linear_fwd(ctx, col[0], w, want, residual=col[2])
    ops.linear_fwd(ctx, col[0], w, col[1], residual=col[2], pre=col[3])      # columns of one matrix side by side are apart
    assert torch.equal(want, col[1])
    flat = new(M * N + 8)
    shifted = flat[8:].view(M, N)
    flat = flat[:M * N].view(M, N)
    square = new(M, M)
    for call in [
            lambda: ops.linear_fwd(ctx, col[0], w, col[0]),
            lambda: ops.linear_fwd(ctx, col[0], w, wide[:, 8:8 + N]),
            lambda: ops.linear_fwd(ctx, col[0], w, flat, residual=shifted),
            lambda: ops.linear_fwd(ctx, col[0], w, flat, pre=flat),
            lambda: ops.linear_fwd(ctx, col[0], w, flat, residual=col[2], pre=shifted),
            lambda: ops.linear_fwd(ctx, square, wide.view(-1)[:M * M].view(M, M), wide[:, :M]),       # over the weights
            lambda: ops.linear_fwd(ctx, col[0], w, flat, residual=wide[:M // 4].view(M, N), pre=col[0]),
            lambda: ops.linear_dgrad(ctx, flat, w, flat),
            lambda: ops.linear_dgrad(ctx, flat, w, col[1], act="silu", pre=wide[:, N + 8:2 * N + 8]),
            lambda: ops.linear_dgrad_gated(ctx, flat, w, pre, pre, h=pre[:, :N]),
            lambda: ops.linear_dgrad_gated(ctx, flat, w, pre, wide[:, :2 * N], dpre_low=wide[:, N:3 * N]),
            lambda: ops.linear_dgrad_gated(ctx, flat, w, pre, wide[:, :2 * N], dpre_low=pre),
            lambda: ops.act_bwd(ctx, col[0], flat, wide[:, 8:8 + N], "silu"),
            lambda: ops.act_bwd(ctx, col[0], flat, col[1], "silu", dz_low=col[1]),
            lambda: ops.gated_act_bwd(ctx, pre[:, :N], wide[:, :2 * N], pre),
            lambda: ops.linear_wgrad(ctx, flat, flat, wide.view(torch.float32).view(-1)[:N * N].view(N, N), x_low=wide.view(-1)[:M * N].view(M, N))]:
        with pytest.raises((TorchColHipError, AssertionError)):
            call()


@pytest.mark.parametrize("act", ACTS[2:])
@pytest.mark.parametrize("gated", [False, True], ids=["linear", "gated"])
def test_gradients_against_differences(ctx, act, gated):
    """The directional derivative of sum(c * output) along the computed gradient, against central differences of the forward operator
    (fp32).  Off by the additions of the outputs, (K + 8) 2^-23 sum |x w| each (1.2 times that behind an activation, and times the
    other factor of a gated layer), over the step, and by the third derivative, for which the difference of two step sizes stands:
    D(2 h) - D(h) is three times D(h)'s own error to leading order."""
    from sirius_amd import ops
    M, K, N = 20, 64, 24
    wide = 2 * N if gated else N
    x, w, b = rnd(M, K, dtype=F32, seed=1), rnd(wide, K, dtype=F32, seed=2, std=1 / 8), rnd(wide, dtype=F32, seed=3, std=0.3)
    c = rnd(M, N, dtype=F32, seed=4)

    def forward(x, w, b, pre=None):
        y = torch.empty(M, N, device="cuda")
        if gated:
            ops.gated_linear_fwd(ctx, x, w, y, bias=b, act=act, pre=pre)
        else:
            ops.linear_fwd(ctx, x, w, y, bias=b, act=act, pre=pre)
        return float((y.double() * c.double()).sum())
    pre, dpre = torch.empty(M, wide, device="cuda"), torch.empty(M, wide, device="cuda")
    forward(x, w, b, pre)
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    if gated:
        ops.gated_linear_bwd(ctx, c, x, w.t().contiguous(), dx, dw, pre, dpre, dbias=db, act=act)
    else:
        ops.linear_bwd(ctx, c, x, w.t().contiguous(), dx, dw, dbias=db, act=act, pre=pre, dpre=dpre)
    grads = (dx, dw, db)
    largest = max(float(g.abs().max()) for g in grads)
    d = [g / largest for g in grads]
    predicted = sum(float((g.double() * e.double()).sum()) for g, e in zip(grads, d))

    def difference(h):
        return (forward(x + h * d[0], w + h * d[1], b + h * d[2]) - forward(x - h * d[0], w - h * d[1], b - h * d[2])) / (2 * h)
    h = 2.0 ** -6
    one, two = difference(h), difference(2 * h)
    z, e = product(x, w)
    e = 1.2 * 1.5 * e           # the operands move by up to 2 h
    if gated:
        e = e[:, :N] * (z[:, N:].abs() + 1) + e[:, N:] * (z[:, :N].abs() + 1)
    rounding = float((c.double().abs() * e).sum()) / h
    assert abs(one - predicted) <= abs(two - one) + rounding, (one, two, predicted, rounding)
    assert rounding + abs(two - one) < 0.1 * abs(predicted)       # the bound says something
