"""The backward pass from activations kept in 8 bits: derivatives and weight gradients of what is kept, against the formulas in 64
bits and, where the arithmetic is the same, bit for bit against the calls that take the unpacked tensors."""
import pytest
import torch

from oracle import block_ops as O

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def normal(*shape, dtype=torch.float32, std=1.0, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=g)


def keep(ctx, x, fmt):
    from sirius_amd import ops
    packed = ops.Packed8.empty(*x.shape, fmt)
    ops.pack8(ctx, x, packed)
    back = torch.empty_like(x)
    ops.unpack8(ctx, packed, back)
    return packed, back


def value_and_slope(z, act):
    z = z.clone().requires_grad_(True)
    y = {"relu": lambda: torch.relu(z), "gelu": lambda: z * 0.5 * torch.special.erfc(-z / 2 ** 0.5), "none": lambda: z * 1.0,
         "gelu_tanh": lambda: z * torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (z + 0.044715 * z ** 3)), "silu": lambda: z * torch.sigmoid(z)}[act]()
    return y.detach(), torch.autograd.grad(y.sum(), z)[0]


def sums_close(a, b, terms):
    """Column sums of the same terms by two kernels: where one adds a product in a fused multiply-add and the other after it is rounded,
    a term is off by 2^-24 of its size, and each of the additions by 2^-24 of the sum of magnitudes, on either side."""
    size = terms.double().abs().sum(0)
    assert ((a.double() - b.double()).abs() <= 2 * (terms.shape[0] + 4) * O.U * (size + b.double().abs())).all()


def close(got, ref, size, dtype, at_most=2.0 ** -17):
    """Half a step of the type, and at_most of the terms' size: slopes are exact to 2^-17 next to 1 (bf16: an exponential, a reciprocal
    and a polynomial of some 2^-21 each; fp32: of some 2^-22)."""
    assert ((got.double() - ref).abs() <= torch.finfo(dtype).eps / 2 * ref.abs() + at_most * size + 2.0 ** -120).all(), \
        float(((got.double() - ref).abs() / (ref.abs() + size + 1e-30)).max())


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh", "silu", "none"])
@pytest.mark.parametrize("M,N", [(1, 8), (5, 40), (130, 264), (517, 1000), (1024, 2048)], ids=str)
def test_derivatives(ctx, dtype, fmt, act, M, N):
    from sirius_amd import ops
    dt = TYPES[dtype]
    pre, dy = normal(M, N, dtype=dt, std=2.0), normal(M, N, dtype=dt, seed=1)
    packed, kept = keep(ctx, pre, fmt)
    dz, h, db = torch.empty_like(dy), torch.empty_like(dy), torch.empty(N, device="cuda")
    low = torch.empty_like(dy) if dtype == "bf16" else None
    ws = torch.empty(max(ops.act_bwd_workspace_bytes(dy), 4), dtype=torch.uint8, device="cuda")
    ops.act_bwd_packed(ctx, dy, packed, dz, act, h=h, dz_low=low, dbias=db, workspace=ws)
    value, slope = value_and_slope(kept.double(), act)
    close(dz, dy.double() * slope, dy.double().abs(), dt)
    close(h, value, kept.double().abs(), dt)
    # the same as from the tensor that was kept, to the last bit
    dz2, db2, low2 = torch.empty_like(dy), torch.empty(N, device="cuda"), None if low is None else torch.empty_like(dy)
    ops.act_bwd(ctx, dy, kept, dz2, act, dz_low=low2, dbias=db2, workspace=ws)
    sums_close(db, db2, dy.double() * slope)
    assert torch.equal(dz, dz2) and (low is None or torch.equal(low, low2))
    # without anything beside it, in place; and without a workspace
    alone = dy.clone()
    ops.act_bwd_packed(ctx, alone, packed, alone, act)
    assert torch.equal(alone, dz)
    db.fill_(1.0), db2.fill_(1.0)
    ops.act_bwd_packed(ctx, dy, packed, dz2, act, dbias=db, accumulate=True)
    ops.act_bwd(ctx, dy, kept, dz2, act, dbias=db2, accumulate=True)
    sums_close(db, db2, dy.double() * slope)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("M,F", [(1, 8), (5, 40), (130, 264), (517, 1000)], ids=str)
def test_gated_derivatives(ctx, dtype, fmt, act, M, F):
    """The up half of a row begins inside a group of 32 where F is no multiple of it."""
    from sirius_amd import ops
    dt = TYPES[dtype]
    pre, dh = normal(M, 2 * F, dtype=dt, std=2.0), normal(M, F, dtype=dt, seed=1)
    packed, kept = keep(ctx, pre, fmt)
    dpre, h, db = torch.empty_like(pre), torch.empty_like(dh), torch.empty(2 * F, device="cuda")
    low = torch.empty_like(pre) if dtype == "bf16" else None
    ws = torch.empty(max(ops.act_bwd_workspace_bytes(dh, gated=True), 4), dtype=torch.uint8, device="cuda")
    ops.gated_act_bwd_packed(ctx, dh, packed, dpre, act, h=h, dpre_low=low, dbias=db, workspace=ws)
    g, u, d = kept[:, :F].double(), kept[:, F:].double(), dh.double()
    value, slope = value_and_slope(g, act)
    close(dpre, torch.cat([d * u * slope, d * value], 1), torch.cat([(d * u).abs(), (d * g).abs()], 1), dt)
    close(h, value * u, (g * u).abs(), dt)
    dpre2, h2, db2, low2 = torch.empty_like(pre), torch.empty_like(dh), torch.empty_like(db), None if low is None else torch.empty_like(pre)
    ops.gated_act_bwd(ctx, dh, kept, dpre2, act, h=h2, dpre_low=low2, dbias=db2, workspace=ws)
    sums_close(db, db2, torch.cat([d * u * slope, d * value], 1))
    assert torch.equal(dpre, dpre2) and torch.equal(h, h2) and (low is None or torch.equal(low, low2))


def test_derivative_by_columns_and_of_not_a_number(ctx):
    from sirius_amd import ops
    M, N = 19, 72
    pre = normal(M, N, dtype=torch.bfloat16)
    pre[3, 40] = float("nan")
    packed, kept = keep(ctx, pre, "int8")
    wide = normal(M, N + 32, dtype=torch.bfloat16, seed=2)
    out = torch.full((M + 2, N + 32), 3.0, dtype=torch.bfloat16, device="cuda")
    ops.act_bwd_packed(ctx, wide[:, 8:8 + N], packed, out[1:-1, 16:16 + N], "silu")
    want = torch.empty(M, N, dtype=torch.bfloat16, device="cuda")
    ops.act_bwd(ctx, wide[:, 8:8 + N], kept, want, "silu")
    got = out[1:-1, 16:16 + N]
    assert torch.equal(got.nan_to_num(99.0), want.nan_to_num(99.0))
    nan = torch.isnan(got)
    assert nan[3, 32:64].all() and nan.sum() == 32
    out[1:-1, 16:16 + N] = 3.0
    assert (out == 3.0).all()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("M,K,N", [(1, 8, 8), (7, 40, 24), (33, 136, 64), (257, 264, 520), (1000, 1000, 776), (4115, 176, 272), (2048, 1024, 512), (300, 2056, 2600)], ids=str)
def test_weight_gradients(ctx, dtype, fmt, M, K, N):
    """Whole numbers: every product and every sum below 2^24 is exact, whatever the order; then numbers of all sizes, each of the M
    additions of a sum within 2^-24 of the sum of magnitudes (fp32 operands in three parts of 8 bits: 2^-22 more of a product)."""
    from sirius_amd import ops
    dt = TYPES[dtype]
    x = torch.randint(-3, 4, (M, K), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(dt)
    dy = torch.randint(-3, 4, (M, N), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).to(dt)
    packed, kept = keep(ctx, x, fmt)
    assert torch.equal(kept, x)
    dw, db = torch.full((N, K), 7.0, device="cuda"), torch.full((N,), 7.0, device="cuda")
    ws = torch.empty(ops.linear_wgrad_packed_workspace_bytes(packed, dy), dtype=torch.uint8, device="cuda").fill_(255)
    ops.linear_wgrad_packed(ctx, packed, dy, dw, dbias=db, workspace=ws)
    assert torch.equal(dw.double(), dy.double().t() @ x.double()) and torch.equal(db.double(), dy.double().sum(0))
    ops.linear_wgrad_packed(ctx, packed, dy, dw, dbias=db, accumulate=True, workspace=ws)
    assert torch.equal(dw.double(), 2 * (dy.double().t() @ x.double()))
    x, dy = normal(M, K, dtype=dt), normal(M, N, dtype=dt, seed=1)
    x[:, 5::97] *= 16.0
    packed, kept = keep(ctx, x, fmt)
    ops.linear_wgrad_packed(ctx, packed, dy, dw, dbias=db, workspace=ws)
    ref, size = dy.double().t() @ kept.double(), dy.double().abs().t() @ kept.double().abs()
    assert ((dw.double() - ref).abs() <= ((M + 4) * O.U + (2.0 ** -21 if dtype == "f32" else 0.0)) * size).all()
    assert ((db.double() - dy.double().sum(0)).abs() <= (M + 4) * O.U * dy.double().abs().sum(0)).all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("M,K,N", [(31, 8, 8), (33, 24, 520), (95, 1032, 136), (2319, 3976, 8736), (4100, 520, 264), (65, 256, 256)], ids=str)
def test_weight_gradients_are_those_of_the_fetched_input(ctx, fmt, M, K, N):
    """Numbers of all sizes in groups of all sizes, rows and columns that end inside a tile or a group of 32: the same products in the
    same order as from the fetched input in bf16, bit for bit, with and without a low part; nothing is written beside dw."""
    from sirius_amd import ops
    x, exact = normal(M, K, dtype=torch.bfloat16), normal(M, N, seed=1)
    x *= 2.0 ** torch.randint(-30, 30, (M, 1), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).float()
    x = x.bfloat16()
    dy = exact.bfloat16()
    low = (exact - dy.float()).bfloat16()
    packed, kept = keep(ctx, x, fmt)
    room = torch.full((N + 2, K), 7.0, device="cuda")
    want, db, db2 = torch.empty(N, K, device="cuda"), torch.empty(N, device="cuda"), torch.empty(N, device="cuda")
    ws = torch.empty(ops.linear_wgrad_packed_workspace_bytes(packed, dy), dtype=torch.uint8, device="cuda").fill_(255)
    dense = torch.empty(ops.linear_bwd_workspace_bytes(kept, N), dtype=torch.uint8, device="cuda")
    for part in (None, low):
        ops.linear_wgrad_packed(ctx, packed, dy, room[1:-1], dbias=db, workspace=ws, dy_low=part)
        ops.linear_wgrad(ctx, kept, dy, want, dbias=db2, workspace=dense, dy_low=part)
        assert torch.equal(room[1:-1], want) and torch.equal(db, db2)
        assert (room[0] == 7.0).all() and (room[-1] == 7.0).all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("M,K,N", [(70, 72, 136), (900, 264, 392)], ids=str)
def test_weight_gradients_of_an_unrounded_gradient(ctx, fmt, M, K, N):
    from sirius_amd import ops
    x, exact = normal(M, K, dtype=torch.bfloat16), normal(M, N, seed=1)
    dy = exact.bfloat16()
    low = (exact - dy.float()).bfloat16()
    packed, kept = keep(ctx, x, fmt)
    dw, db = torch.empty(N, K, device="cuda"), torch.empty(N, device="cuda")
    ws = torch.empty(ops.linear_wgrad_packed_workspace_bytes(packed, dy), dtype=torch.uint8, device="cuda")
    ops.linear_wgrad_packed(ctx, packed, dy, dw, dbias=db, workspace=ws, dy_low=low)
    both = dy.double() + low.double()
    size = (dy.double().abs() + low.double().abs()).t() @ kept.double().abs()
    assert ((dw.double() - both.t() @ kept.double()).abs() <= (2 * M + 4) * O.U * size).all()
    assert ((db.double() - both.sum(0)).abs() <= (2 * M + 4) * O.U * both.abs().sum(0)).all()


def test_groups_that_are_marked(ctx):
    """A NaN among the kept inputs: the columns of its group, and no others."""
    from sirius_amd import ops
    x, dy = normal(64, 96, dtype=torch.bfloat16), normal(64, 40, dtype=torch.bfloat16, seed=1)
    x[9, 70] = float("nan")
    packed, _ = keep(ctx, x, "e4m3")
    dw = torch.empty(40, 96, device="cuda")
    ws = torch.empty(ops.linear_wgrad_packed_workspace_bytes(packed, dy), dtype=torch.uint8, device="cuda")
    ops.linear_wgrad_packed(ctx, packed, dy, dw, workspace=ws)
    assert torch.isnan(dw[:, 64:]).all() and torch.isfinite(dw[:, :64]).all()


def test_no_rows(ctx):
    from sirius_amd import ops
    nothing, dy = ops.Packed8.empty(0, 64), torch.empty(0, 32, dtype=torch.bfloat16, device="cuda")
    dw, db = torch.full((32, 64), 2.0, device="cuda"), torch.full((32,), 2.0, device="cuda")
    ws = torch.empty(max(ops.linear_wgrad_packed_workspace_bytes(nothing, dy), 4), dtype=torch.uint8, device="cuda")
    ops.linear_wgrad_packed(ctx, nothing, dy, dw, dbias=db, accumulate=True, workspace=ws)
    assert (dw == 2.0).all() and (db == 2.0).all()
    ops.linear_wgrad_packed(ctx, nothing, dy, dw, dbias=db, workspace=ws)
    assert (dw == 0.0).all() and (db == 0.0).all()
    ops.act_bwd_packed(ctx, dy, ops.Packed8.empty(0, 32), dy, "silu")
    ops.gated_act_bwd_packed(ctx, dy, nothing, torch.empty(0, 64, dtype=torch.bfloat16, device="cuda"))


def test_recorded_and_replayed(ctx):
    from sirius_amd import ops
    c, prog = ops.Context(), ops.Program()
    M, K, N = 900, 136, 264
    x, pre, dy = normal(M, K, dtype=torch.bfloat16), normal(M, N, dtype=torch.bfloat16), normal(M, N, dtype=torch.bfloat16)
    px, pp = ops.Packed8.empty(M, K, "e4m3"), ops.Packed8.empty(M, N)
    h, dz, low = torch.empty_like(pre), torch.empty_like(dy), torch.empty_like(dy)
    dw, db = torch.empty(N, K, device="cuda"), torch.empty(N, device="cuda")
    ws = torch.empty(ops.linear_wgrad_packed_workspace_bytes(px, dy) + ops.act_bwd_workspace_bytes(dy), dtype=torch.uint8, device="cuda")

    def calls(context):
        ops.pack8(context, x, px)
        ops.act_fwd_pack8(context, pre, h, pp, "gelu")
        ops.act_bwd_packed(context, dy, pp, dz, "gelu", dz_low=low, dbias=db, workspace=ws)
        ops.linear_wgrad_packed(context, px, dz, dw, workspace=ws, dy_low=low)
    c.begin_record(prog)
    calls(c)
    c.end_record()
    for step in range(3):
        x.copy_(normal(M, K, dtype=torch.bfloat16, seed=10 + step))
        pre.copy_(normal(M, N, dtype=torch.bfloat16, seed=20 + step))
        ws.fill_(255)
        c.run(prog)
        c.synchronize()
        got = [t.clone() for t in (h, dz, low, dw, db)]
        calls(ctx)
        ctx.synchronize()
        for a, b in zip(got, (h, dz, low, dw, db)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_more_than_the_cache_holds(ctx, fmt):
    """The kernels that stream past the cache: the bits of those that do not, on a part of the rows."""
    from sirius_amd import ops
    M, F, few = 8192, 5632, 300
    pre, dh = normal(M, 2 * F, dtype=torch.bfloat16), normal(M, F, dtype=torch.bfloat16, seed=1)
    packed, kept = keep(ctx, pre, fmt)
    part, kept_part = keep(ctx, pre[:few].contiguous(), fmt)
    assert torch.equal(packed.data[:few], part.data) and torch.equal(packed.scales[:few], part.scales) and torch.equal(kept[:few], kept_part)
    out, h, low = torch.empty_like(pre), torch.empty_like(dh), torch.empty_like(pre)
    ops.gated_act_bwd_packed(ctx, dh, packed, out, "silu", h=h, dpre_low=low)
    out2, h2, low2 = torch.empty_like(pre[:few]), torch.empty_like(dh[:few]), torch.empty_like(pre[:few])
    ops.gated_act_bwd_packed(ctx, dh[:few], part, out2, "silu", h=h2, dpre_low=low2)
    assert torch.equal(out[:few], out2) and torch.equal(h[:few], h2) and torch.equal(low[:few], low2)
    big, dz, z = normal(M, 2 * F, dtype=torch.bfloat16, seed=2), torch.empty_like(pre), torch.empty_like(pre)
    ops.act_fwd_pack8(ctx, pre, z, packed, "gelu")
    ops.act_bwd_packed(ctx, big, packed, dz, "gelu")
    z2, dz2 = torch.empty_like(pre[:few]), torch.empty_like(pre[:few])
    ops.act_fwd_pack8(ctx, pre[:few], z2, part, "gelu")
    ops.act_bwd_packed(ctx, big[:few], part, dz2, "gelu")
    assert torch.equal(z[:few], z2) and torch.equal(dz[:few], dz2)


def test_two_streams_at_once(ctx):
    """Two contexts on streams of their own, each with its own buffers and workspace, submitted in turn."""
    from sirius_amd import ops
    M, K, N = 2048, 512, 768
    sides = []
    for seed in (1, 2):
        s = torch.cuda.Stream()
        x, dy = normal(M, K, dtype=torch.bfloat16, seed=seed), normal(M, N, dtype=torch.bfloat16, seed=seed + 5)
        packed = ops.Packed8.empty(M, K, "e4m3")
        stats, y = torch.empty(M, 4, device="cuda"), torch.empty_like(x)
        w, dwn = torch.rand(K, device="cuda"), torch.empty(K, device="cuda")
        dw, dx = torch.empty(N, K, device="cuda"), torch.empty_like(x)
        ws = torch.empty(ops.linear_wgrad_packed_workspace_bytes(packed, dy), dtype=torch.uint8, device="cuda")
        ws2 = torch.empty(ops.residual_norm_bwd_workspace_bytes(x), dtype=torch.uint8, device="cuda")
        sides.append((s, x, dy, packed, stats, y, w, dwn, dw, dx, ws, ws2))
    torch.cuda.synchronize()

    def go(c, side):
        _, x, dy, packed, stats, y, w, dwn, dw, dx, ws, ws2 = side
        ops.residual_norm_fwd(c, x, None, None, y, stats, weight=w, packed=packed)
        ops.linear_wgrad_packed(c, packed, dy, dw, workspace=ws)
        ops.residual_norm_bwd(c, y, None, x, None, dx, None, stats, weight=w, dweight=dwn, workspace=ws2)
    contexts = [ops.Context(side[0]) for side in sides]
    for _ in range(5):
        for c, side in zip(contexts, sides):
            go(c, side)
    for c in contexts:
        c.synchronize()
    both = [[t.clone() for t in (side[5], side[7], side[8], side[9])] for side in sides]
    for side, got in zip(sides, both):
        go(ctx, side)
        ctx.synchronize()
        for a, b in zip(got, (side[5], side[7], side[8], side[9])):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("gated", [False, True])
def test_every_row_and_the_sums_of_more_than_the_cache_holds(ctx, dtype, fmt, gated):
    """Kept, fetched and taken derivatives of with column sums, streaming past the cache: every row as launches over an eighth of the rows
    have it, which do not stream, and the sums as the dense call adds them up."""
    from sirius_amd import ops
    dt, M, N = TYPES[dtype], 8200 if dtype == "bf16" else 4616, 5640
    wide = N * (2 if gated else 1)
    M = M if gated else 2 * M
    pre, dy = normal(M, wide, dtype=dt, std=2.0), normal(M, N, dtype=dt, seed=1)
    h, dz, again = torch.empty_like(pre), torch.empty_like(pre), torch.empty_like(dy)
    packed, back = ops.Packed8.empty(M, wide, fmt), torch.empty_like(pre)
    low = torch.empty_like(pre) if dtype == "bf16" else None
    db = torch.empty(wide, device="cuda")
    ws = torch.empty(max(ops.act_bwd_workspace_bytes(dy, gated=gated), 4), dtype=torch.uint8, device="cuda").fill_(255)

    def bwd(*args, low=None, **more):
        (ops.gated_act_bwd_packed if gated else ops.act_bwd_packed)(*args, **{"dpre_low" if gated else "dz_low": low}, **more)
    ops.act_fwd_pack8(ctx, pre, h, packed, "gelu")
    ops.unpack8(ctx, packed, back)
    bwd(ctx, dy, packed, dz, "silu", h=again, low=low, dbias=db, workspace=ws)
    each = M // 8
    for r0 in range(0, M, each):
        rows = slice(r0, r0 + each)
        part = ops.Packed8.empty(each, wide, fmt)
        h2, back2, dz2, again2 = torch.empty_like(h[rows]), torch.empty_like(h[rows]), torch.empty_like(h[rows]), torch.empty_like(dy[rows])
        low2 = None if low is None else torch.empty_like(dz2)
        ops.act_fwd_pack8(ctx, pre[rows], h2, part, "gelu")
        ops.unpack8(ctx, part, back2)
        bwd(ctx, dy[rows], part, dz2, "silu", h=again2, low=low2)
        for a, b in ((h, h2), (packed.data, part.data), (packed.scales, part.scales), (back, back2), (dz, dz2), (again, again2)):
            assert torch.equal(a[rows], b), r0
        assert low is None or torch.equal(low[rows], low2), r0
    dz2, db2 = torch.empty_like(dz), torch.empty_like(db)
    (ops.gated_act_bwd if gated else ops.act_bwd)(ctx, dy, back, dz2, "silu", dbias=db2, workspace=ws)
    assert torch.equal(dz, dz2)
    sums_close(db, db2, dz)
