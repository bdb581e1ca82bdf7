"""Linear layers with bias, activation and residual in one launch, gated feed-forward layers and their backward passes, against
fp64 on the same inputs.

Bounds, element by element (u = half a step of the type, torch.finfo(t).eps / 2: bf16 2^-8, fp32 2^-24):
* a product of K terms added up in fp32: (K + 8) 2^-23 sum |a b| (each addition is off by 2^-24 of the running sum at most;
  doubled, since the matrix instructions add groups of terms in an order of their own);
* an activation: 2^-20 |z| + 1.2 times its argument's error (no slope exceeds 1.13); a slope 2^-19 (the bf16 kernels' exponential and
  reciprocal are good to 2^-21, their error function to 1.5e-7);
* a stored value: u |value| on top; a stored gradient that is multiplied again (dz, dpre): u |dz| per term of the sum.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu")


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def value(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "gelu":
        return 0.5 * z * torch.special.erfc(-z / math.sqrt(2))
    if act == "gelu_tanh":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    if act == "silu":
        return z * torch.sigmoid(z)
    return z.clone()


def slope(z, act):
    if act == "relu":
        return (z > 0).double()
    if act == "gelu":
        return 0.5 * torch.special.erfc(-z / math.sqrt(2)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        a, b = 2 * math.sqrt(2 / math.pi), 0.044715
        s = torch.sigmoid(a * (z + b * z ** 3))
        return s + z * s * torch.sigmoid(-a * (z + b * z ** 3)) * a * (1 + 3 * b * z * z)
    if act == "silu":
        return torch.sigmoid(z) + z * torch.sigmoid(z) * torch.sigmoid(-z)
    return torch.ones_like(z)


def rnd(*shape, dtype, seed, std=1.0):
    g = torch.Generator().manual_seed(seed * 7919 + sum(shape))
    return (torch.randn(*shape, generator=g) * std).to(dtype).cuda()


def product(a, b):
    """fp64 a b^T and what fp32 additions may be off."""
    a, b = a.double(), b.double()
    return a @ b.t(), (a.shape[1] + 8) * 2.0 ** -23 * (a.abs() @ b.abs().t())


def near(got, ref, tol, what):
    err = (got.double() - ref).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}, "
                           f"worst {float((err / tol).nan_to_num(9e9).max()):.3g} of the bound")


SENTINEL = 777.0


class Framed:
    """A matrix inside a wider and longer one full of a sentinel: `view` is what the operator gets (columns of the wider one when
    `wide`), and nothing around it may change."""

    def __init__(self, rows, cols, dtype, wide, init=None):
        pad = 16 if wide else 0
        self.full = torch.full((rows + 3, cols + pad), SENTINEL, dtype=dtype, device="cuda")
        self.view = self.full[:rows, pad // 2:pad // 2 + cols]
        self.rows, self.lo, self.hi = rows, pad // 2, pad // 2 + cols
        if init is not None:
            self.view.copy_(init)

    def check(self, what):
        rest = self.full.clone()
        rest[:self.rows, self.lo:self.hi] = SENTINEL
        assert bool((rest == SENTINEL).all()), f"{what}: wrote outside its output"


# rows of every kernel: up to 16 tokens; reductions dealt to wavefronts; tiles of 128 x 64 to 256 x 256.  Sizes that end inside
# tiles, reductions shorter than a step, one step long, a chunk longer
SHAPES = [(1, 8, 8), (1, 64, 24), (1, 4096, 104), (6, 4096, 4096), (2, 72, 2056), (7, 1000, 64), (15, 520, 136), (16, 136, 1032),
          (17, 8, 16), (31, 64, 64), (33, 72, 40), (65, 1000, 200), (128, 256, 512), (130, 2056, 96), (333, 200, 1032),
          (700, 40, 2056), (2050, 24, 1544), (1800, 200, 1928), (2049, 328, 1664), (1536, 1024, 2048),
          (100, 776, 4104), (4100, 8, 2056), (4097, 72, 2104), (4096, 256, 2048), (130, 96, 66000)]


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_linear_fwd(ctx, M, K, N, dtype):
    from sirius_amd import ops
    u = half_step(dtype)
    x, w = rnd(M, K, dtype=dtype, seed=1), rnd(N, K, dtype=dtype, seed=2, std=1 / math.sqrt(K))
    bias, res = rnd(N, dtype=F32, seed=3), rnd(M, N, dtype=dtype, seed=4)
    z0, e0 = product(x, w)
    for i, act in enumerate(ACTS):
        with_bias, with_res, with_pre, wide = i % 2 == 0, i in (1, 2), i in (0, 2, 3), i in (2, 4)
        xs = Framed(M, K, dtype, wide, x)
        y, pre = Framed(M, N, dtype, wide), Framed(M, N, dtype, wide)
        r = Framed(M, N, dtype, wide, res)
        ops.linear_fwd(ctx, xs.view, w, y.view, bias=bias if with_bias else None, act=act, residual=r.view if with_res else None,
                       pre=pre.view if with_pre else None)
        z, e = (z0 + bias.double(), e0 + 2.0 ** -23 * (z0.abs() + bias.abs().double())) if with_bias else (z0, e0)
        ref = value(z, act)
        tol = 1.2 * e + 2.0 ** -20 * z.abs()
        if with_res:
            ref = ref + res.double()
            tol = tol + 2.0 ** -23 * ref.abs()
        near(y.view, ref, tol + u * (ref.abs() + tol), f"{act} y")
        y.check(act)
        pre.check(act)
        if with_pre:
            near(pre.view, z, e + u * (z.abs() + e), f"{act} pre")


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("M,K,N", SHAPES[:-1])
def test_gated_linear_fwd(ctx, M, K, N, dtype):
    from sirius_amd import ops
    u, F = half_step(dtype), N // 16 * 8 if N >= 16 else 8
    x, w = rnd(M, K, dtype=dtype, seed=1), rnd(2 * F, K, dtype=dtype, seed=2, std=1 / math.sqrt(K))
    bias = rnd(2 * F, dtype=F32, seed=3)
    z0, e0 = product(x, w)
    for i, act in enumerate(ACTS):
        with_bias, with_pre, wide = i % 2 == 0, i in (0, 2, 3), i in (2, 4)
        xs, h, pre = Framed(M, K, dtype, wide, x), Framed(M, F, dtype, wide), Framed(M, 2 * F, dtype, wide)
        ops.gated_linear_fwd(ctx, xs.view, w, h.view, bias=bias if with_bias else None, act=act, pre=pre.view if with_pre else None)
        z, e = (z0 + bias.double(), e0 + 2.0 ** -23 * (z0.abs() + bias.abs().double())) if with_bias else (z0, e0)
        g, up, eg, eu = z[:, :F], z[:, F:], e[:, :F], e[:, F:]
        a = value(g, act)
        ea = 1.2 * eg + 2.0 ** -20 * g.abs()
        ref, tol = a * up, ea * (up.abs() + eu) + a.abs() * eu + 2.0 ** -23 * (a * up).abs()
        near(h.view, ref, tol + u * (ref.abs() + tol), f"{act} h")
        h.check(act)
        pre.check(act)
        if with_pre:
            near(pre.view, z, e + u * (z.abs() + e), f"{act} pre")


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("M,K,N", SHAPES[:-1])
def test_data_gradients(ctx, M, K, N, dtype):
    """linear_dgrad through an activation and linear_dgrad_gated: reductions over K, outputs N (F) wide."""
    from sirius_amd import ops
    u = half_step(dtype)
    dy, w = rnd(M, K, dtype=dtype, seed=1), rnd(N, K, dtype=dtype, seed=2, std=1 / math.sqrt(K))   # w: the layer's weight transposed
    pre, res = rnd(M, 2 * N, dtype=dtype, seed=5, std=2.0), rnd(M, N, dtype=dtype, seed=4)
    v, e = product(dy, w)
    g, up = pre[:, :N].double(), pre[:, N:].double()
    for i, act in enumerate(ACTS):
        with_res, wide = i in (0, 2, 3), i in (1, 2)
        dys, r = Framed(M, K, dtype, wide, dy), Framed(M, N, dtype, wide, res)
        z = Framed(M, 2 * N, dtype, wide, pre)
        dx = Framed(M, N, dtype, wide)
        ops.linear_dgrad(ctx, dys.view, w, dx.view, act=act, pre=z.view[:, :N] if act != "none" else None,
                         residual=r.view if with_res else None)
        s = slope(g, act)
        ref, tol = v * s, (e + 2.0 ** -23 * v.abs()) * s.abs() + 2.0 ** -19 * (v.abs() + e)
        if with_res:
            ref = ref + res.double()
            tol = tol + 2.0 ** -23 * ref.abs()
        near(dx.view, ref, tol + u * (ref.abs() + tol), f"{act} dx")
        dx.check(act)
        dpre, h = Framed(M, 2 * N, dtype, wide), Framed(M, N, dtype, wide)
        ops.linear_dgrad_gated(ctx, dys.view, w, z.view, dpre.view, act=act, h=h.view if with_res else None)
        a = value(g, act)
        ea = 2.0 ** -20 * g.abs()
        for got, ref, tol in ((dpre.view[:, :N], v * up * s, (e * s.abs() + 2.0 ** -19 * (v.abs() + e)) * up.abs()),
                              (dpre.view[:, N:], v * a, e * a.abs() + ea * (v.abs() + e))):
            tol = tol + 2.0 ** -22 * ref.abs()
            near(got, ref, tol + u * (ref.abs() + tol), f"{act} dpre")
        dpre.check(act)
        h.check(act)
        if with_res:
            ref, tol = a * up, ea * up.abs() + 2.0 ** -23 * (a * up).abs()
            near(h.view, ref, tol + u * (ref.abs() + tol), f"{act} h")


def check_backward(got, dpre, x, w, u, extra, residual=None, dw0=None, db0=None, low=False):
    """dx, dw, db against fp64; dpre [M, N] in fp64 with `extra`, what it may be off before it is rounded to the type.  low: the
    weight gradient had its low part, which leaves 2^-8 of what rounding took off (2^-8): 2^-16."""
    dx, dw, db = got
    M, N = dpre.shape
    edp = extra + u * (dpre.abs() + extra)
    edw = extra + 2.0 ** -16 * (dpre.abs() + extra) if low else edp
    wd, xd = w.double(), x.double()
    ref = dpre @ wd
    tol = edp @ wd.abs() + (N + 8) * 2.0 ** -23 * (dpre.abs() @ wd.abs())
    if residual is not None:
        ref = ref + residual.double()
        tol = tol + 2.0 ** -23 * ref.abs()
    near(dx, ref, tol + u * (ref.abs() + tol), "dx")
    sums = ((2 if low else 1) * M + 64) * 2.0 ** -23      # the split reduction adds partial sums on top
    ref, tol = dpre.t() @ xd, edw.t() @ xd.abs() + sums * (dpre.abs().t() @ xd.abs())
    if dw0 is not None:
        ref = ref + dw0.double()
        tol = tol + 2.0 ** -23 * ref.abs()
    near(dw, ref, tol + 2.0 ** -23 * ref.abs() + 1e-30, "dw")
    ref, tol = dpre.sum(0), edw.sum(0) + sums * dpre.abs().sum(0)
    if db0 is not None:
        ref = ref + db0.double()
        tol = tol + 2.0 ** -23 * ref.abs()
    near(db, ref, tol + 1e-30, "db")


BWD_SHAPES = [(1, 64, 72), (8, 136, 24), (33, 72, 200), (392, 512, 264), (1023, 264, 520), (2050, 1544, 136), (300, 8, 8)]


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("M,K,N", BWD_SHAPES)
def test_linear_bwd(ctx, M, K, N, dtype):
    from sirius_amd import ops
    u = half_step(dtype)
    x, w = rnd(M, K, dtype=dtype, seed=1), rnd(N, K, dtype=dtype, seed=2, std=1 / math.sqrt(K))
    dy, pre, res = rnd(M, N, dtype=dtype, seed=3), rnd(M, N, dtype=dtype, seed=4, std=2.0), rnd(M, K, dtype=dtype, seed=5)
    wt = w.t().contiguous()
    for i, act in enumerate(ACTS):
        accumulate, with_res, split = i in (1, 3), i in (1, 2), i != 2
        low = torch.empty_like(dy) if dtype == BF16 and i in (1, 2, 4) else None
        dx, dpre = torch.empty_like(x), torch.empty_like(dy)
        dw, db = rnd(N, K, dtype=F32, seed=6), rnd(N, dtype=F32, seed=7)
        dw0, db0 = (dw.clone(), db.clone()) if accumulate else (None, None)
        ws = torch.empty(ops.linear_bwd_workspace_bytes(x, N), dtype=torch.uint8, device="cuda") if split else None
        ops.linear_bwd(ctx, dy, x, wt, dx, dw, dbias=db, act=act, pre=pre, dpre=dpre, residual=res if with_res else None,
                       accumulate=accumulate, workspace=ws, dpre_low=low)
        s = slope(pre.double(), act)
        ref = dy.double() * s
        extra = torch.zeros_like(ref) if act == "none" else 2.0 ** -19 * dy.double().abs()
        check_backward((dx, dw, db), ref, x, w, u, extra, res if with_res else None, dw0, db0, low is not None)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("M,K,F", BWD_SHAPES)
def test_gated_linear_bwd(ctx, M, K, F, dtype):
    from sirius_amd import ops
    u = half_step(dtype)
    x, w = rnd(M, K, dtype=dtype, seed=1), rnd(2 * F, K, dtype=dtype, seed=2, std=1 / math.sqrt(K))
    dh, pre = rnd(M, F, dtype=dtype, seed=3), rnd(M, 2 * F, dtype=dtype, seed=4, std=2.0)
    wt = w.t().contiguous()
    for i, act in enumerate(ACTS):
        low = torch.empty_like(pre) if dtype == BF16 and i in (0, 2, 4) else None
        dx, dpre = torch.empty_like(x), torch.empty_like(pre)
        dw, db = torch.empty(2 * F, K, device="cuda"), torch.empty(2 * F, device="cuda")
        ws = torch.empty(ops.linear_bwd_workspace_bytes(x, 2 * F), dtype=torch.uint8, device="cuda")
        ops.gated_linear_bwd(ctx, dh, x, wt, dx, dw, pre, dpre, dbias=db, act=act, workspace=ws, dpre_low=low)
        d, g, up = dh.double(), pre[:, :F].double(), pre[:, F:].double()
        ref = torch.cat([d * up * slope(g, act), d * value(g, act)], 1)
        extra = torch.cat([2.0 ** -19 * (d * up).abs(), 2.0 ** -20 * (d * g).abs()], 1) + 2.0 ** -22 * ref.abs()
        check_backward((dx, dw, db), ref, x, w, u, extra, low=low is not None)


@pytest.mark.parametrize("M,C,F", [(5, 72, 40), (130, 264, 520), (1100, 512, 1544), (2100, 520, 2056)])
def test_feed_forward_block(ctx, M, C, F):
    """A whole gated block as a training step runs it: gated layer, down projection with the block's residual, and back through
    linear_dgrad_gated with low parts; the inner results are the program's own rounded ones, everything against fp64."""
    from sirius_amd import ops
    u = half_step(BF16)
    x, res = rnd(M, C, dtype=BF16, seed=1), rnd(M, C, dtype=BF16, seed=2)
    w, wd = rnd(2 * F, C, dtype=BF16, seed=3, std=1 / math.sqrt(C)), rnd(C, F, dtype=BF16, seed=4, std=1 / math.sqrt(F))
    bias, dy = rnd(2 * F, dtype=F32, seed=5), rnd(M, C, dtype=BF16, seed=6)
    wt, wdt = w.t().contiguous(), wd.t().contiguous()

    def new(*shape, dtype=BF16):
        return torch.empty(shape, dtype=dtype, device="cuda")
    h, pre, y = new(M, F), new(M, 2 * F), new(M, C)
    dpre, dpre_low, h2, h2_low, dx = new(M, 2 * F), new(M, 2 * F), new(M, F), new(M, F), new(M, C)
    dw, db, dwd = new(2 * F, C, dtype=F32), new(2 * F, dtype=F32), new(C, F, dtype=F32)
    ws, wsd = (new(ops.linear_bwd_workspace_bytes(*a), dtype=torch.uint8) for a in ((x, 2 * F), (h, C)))
    ops.gated_linear_fwd(ctx, x, w, h, bias=bias, act="silu", pre=pre)
    ops.linear_fwd(ctx, h, wd, y, residual=res)
    ops.linear_dgrad_gated(ctx, dy, wdt, pre, dpre, act="silu", h=h2, dpre_low=dpre_low, h_low=h2_low)
    ops.linear_wgrad(ctx, h2, dy, dwd, workspace=wsd, x_low=h2_low)
    ops.linear_bwd(ctx, dpre, x, wt, dx, dw, dbias=db, residual=dy, workspace=ws, dy_low=dpre_low)

    z, e = product(x, w)
    z, e = z + bias.double(), e + 2.0 ** -23 * (z.abs() + bias.abs().double())
    near(pre, z, e + u * (z.abs() + e), "pre")
    g, up = z[:, :F], z[:, F:]
    a, ea = value(g, "silu"), 1.2 * e[:, :F] + 2.0 ** -20 * g.abs()
    ref, tol = a * up, ea * (up.abs() + e[:, F:]) + a.abs() * e[:, F:] + 2.0 ** -23 * (a * up).abs()
    near(h, ref, tol + u * (ref.abs() + tol), "h")
    v, ev = product(h, wd)
    ref = v + res.double()
    near(y, ref, ev + u * (ref.abs() + ev) + 2.0 ** -23 * ref.abs(), "y")

    dh, edh = product(dy, wdt)
    g, up = pre[:, :F].double(), pre[:, F:].double()
    a, s = value(g, "silu"), slope(g, "silu")
    exact = torch.cat([dh * up * s, dh * a], 1)
    edp = torch.cat([(edh * s.abs() + 2.0 ** -19 * (dh.abs() + edh)) * up.abs(), edh * a.abs() + 2.0 ** -20 * g.abs() * (dh.abs() + edh)], 1)
    edp = edp + 2.0 ** -22 * exact.abs()
    both = dpre.double() + dpre_low.double()
    near(both, exact, edp + 2.0 ** -16 * (exact.abs() + edp), "dpre and its low part")
    eh = 2.0 ** -20 * (g * up).abs() + 2.0 ** -16 * (a * up).abs()
    near(h2.double() + h2_low.double(), a * up, eh, "h and its low part")
    ref = dy.double().t() @ (a * up)
    near(dwd, ref, dy.abs().double().t() @ eh + (2 * M + 64) * 2.0 ** -23 * (dy.abs().double().t() @ (a * up).abs()) + 2.0 ** -23 * ref.abs(), "dw_down")
    check_backward((dx, dw, db), exact, x, w, u, edp, residual=dy, low=True)


@pytest.mark.parametrize("low", ["none", "dy", "x"])
@pytest.mark.parametrize("M,K,N", [(1, 8, 8), (31, 264, 72), (33, 8, 520), (64, 136, 136), (1000, 256, 256), (3001, 776, 1288), (4100, 1032, 2056),
                                   (9000, 264, 264), (70, 2056, 2312),
                                   # whole rounds of tiles and a rest that fewer workgroups share; two rounds and a rest
                                   (1803, 5120, 3312), (2319, 3976, 8736)])
def test_linear_wgrad(ctx, M, K, N, low):
    """bf16 weight gradients with and without a low part, rows split and not, added to what is there and not."""
    from sirius_amd import ops
    x, dy = rnd(M, K, dtype=BF16, seed=1), rnd(M, N, dtype=BF16, seed=2)
    dy_low = rnd(M, N, dtype=BF16, seed=3, std=2.0 ** -9) if low == "dy" else None
    x_low = rnd(M, K, dtype=BF16, seed=4, std=2.0 ** -9) if low == "x" else None
    a = dy.double() + (0 if dy_low is None else dy_low.double())
    b = x.double() + (0 if x_low is None else x_low.double())
    for split, accumulate, with_bias in ((True, False, True), (False, True, True), (True, True, False)):
        dw, db = Framed(N, K, F32, False), Framed(1, N, F32, False)
        dw.view.copy_(rnd(N, K, dtype=F32, seed=5))
        db.view.copy_(rnd(1, N, dtype=F32, seed=6))
        dw0, db0 = dw.view.double(), db.view.double()
        need = ops.linear_bwd_workspace_bytes(x, N)
        ws = torch.full((need + 64,), 99, dtype=torch.uint8, device="cuda")
        ops.linear_wgrad(ctx, x, dy, dw.view, dbias=db.view if with_bias else None, accumulate=accumulate,
                         workspace=ws[:need] if split else None, dy_low=dy_low, x_low=x_low)
        ref, tol = a.t() @ b, (2 * M + 64) * 2.0 ** -23 * (a.abs().t() @ b.abs())
        if accumulate:
            ref = ref + dw0
        near(dw.view, ref, tol + 2.0 ** -22 * ref.abs() + 1e-30, "dw")
        ref, tol = a.sum(0, keepdim=True), (2 * M + 64) * 2.0 ** -23 * a.abs().sum(0, keepdim=True)
        if accumulate:
            ref = ref + db0
        if with_bias:
            near(db.view, ref, tol + 2.0 ** -22 * ref.abs() + 1e-30, "db")
        else:
            assert torch.equal(db.view.double(), db0)
        dw.check("dw")
        db.check("db")
        assert bool((ws[need:] == 99).all())
