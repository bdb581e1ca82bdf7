"""The global gradient norm over many tensors, clipping by it, and optimizer steps that take its coefficient, against fp64.

Bounds: squares of fp32 (bf16) numbers are exact in fp64 and their sum is off by 2^-30 of itself at the very most (n 2^-53, n < 2^23
here), so the norm is the fp32 number next to the exact one: 2^-24 of itself, and 2^-23 leaves room for the sum.  The coefficient
is rounded to fp32 once (2^-24), a gradient times it rounded once more to its type (u): 2^-23 + u of the value."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def make(sizes, dtypes, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=g) * std).to(dtypes[i % len(dtypes)]).cuda() for i, n in enumerate(sizes)]


def workspace(table):
    from sirius_amd import ops
    return torch.empty(ops.grad_norm_workspace_bytes(table), dtype=torch.uint8, device="cuda")


def exact_norm(tensors):
    return math.sqrt(math.fsum(float((t.double() ** 2).sum()) for t in tensors))


LISTS = [[1], [0, 5, 0], [3], [4], [8192], [8193], [64, 1, 33, 7, 100, 4096], [100_003, 2, 8191], [1] * 300,
         [50_000 * i % 70_001 + 1 for i in range(60)], [3_000_000, 5, 17_000_001]]


@pytest.mark.parametrize("dtypes", [(F32,), (BF16,), (F32, BF16)], ids=["f32", "bf16", "mixed"])
@pytest.mark.parametrize("sizes", LISTS, ids=lambda s: f"{len(s)}of{max(s)}")
def test_clip(ctx, sizes, dtypes):
    from sirius_amd import ops
    for place, limit in (("in", 0.5), ("out", 0.25), ("other", 0.125), ("in", 1e9)):
        grads = make(sizes, dtypes, len(sizes))
        before = [g.clone() for g in grads]
        if place == "other":    # into the other type
            out = [torch.full((g.numel(),), 7.0, dtype=BF16 if g.dtype == F32 else F32, device="cuda") for g in grads]
        else:
            out = [torch.full_like(g, 7.0) for g in grads] if place == "out" else None
        table = ops.GradTable(grads, out=out)
        norm, ws = torch.full((1,), -1.0, device="cuda"), workspace(table)
        ops.clip_grad_norm(ctx, table, limit, norm, ws)
        ref = exact_norm(before)
        assert abs(norm.item() - ref) <= 2.0 ** -23 * ref
        coef = min(1.0, limit / (ref + 1e-6))
        for g, b, o in zip(grads, before, out or grads):
            if out is not None:
                assert torch.equal(g, b), "a gradient changed although the result went elsewhere"
            want = b.double() * coef
            u = torch.finfo(o.dtype).eps / 2
            assert ((o.double() - want).abs() <= (2.0 ** -23 + u) * want.abs()).all()
            if coef == 1.0 and place == "in":
                assert torch.equal(o, b)


@pytest.mark.parametrize("shift", [1, 2, 3])
def test_unaligned_views_of_one_buffer(ctx, shift):
    """Tensors that start anywhere in a bucket, source and destination differently; what lies between them stays as it was."""
    from sirius_amd import ops
    sizes = [5, 1, 8192, 20_000, 3]
    src, dst = torch.full((40_000,), 3.0, device="cuda"), torch.full((40_000,), 9.0, device="cuda")
    at, views, outs = shift, [], []
    for i, n in enumerate(sizes):
        views.append(src[at:at + n])
        outs.append(dst[at + i:at + i + n])
        at += n + 5
    table = ops.GradTable(views, out=outs)
    norm, ws = torch.empty(1, device="cuda"), workspace(table)
    ops.clip_grad_norm(ctx, table, 1.0, norm, ws)
    ref = exact_norm(views)
    assert abs(norm.item() - ref) <= 2.0 ** -23 * ref
    for o in outs:
        assert ((o.double() - 3.0 / (ref + 1e-6)).abs() <= 2.0 ** -22 * 3.0 / ref).all()
    assert int((dst == 9.0).sum()) == dst.numel() - sum(sizes) and bool((src == 3.0).all())


def test_large_and_small_values(ctx):
    """Squares beyond fp32's range on both sides."""
    from sirius_amd import ops
    for scale in (1e30, 1e-30):
        grads = make([5000, 77], (F32,), 3, std=scale)
        before = [g.clone() for g in grads]
        table = ops.GradTable(grads)
        norm, ws = torch.empty(1, device="cuda"), workspace(table)
        ops.clip_grad_norm(ctx, table, 2.0, norm, ws)
        ref = exact_norm(before)
        assert abs(norm.item() - ref) <= 2.0 ** -23 * ref
        coef = min(1.0, 2.0 / (ref + 1e-6))
        for g, b in zip(grads, before):
            want = b.double() * coef
            assert ((g.double() - want).abs() <= 2.0 ** -22 * want.abs()).all()


def test_norms_that_are_not_finite(ctx):
    from sirius_amd import ops
    grads = make([100, 9000], (F32,), 1)
    grads[1][8999] = float("inf")
    table = ops.GradTable(grads)
    norm, ws = torch.empty(1, device="cuda"), workspace(table)
    ops.clip_grad_norm(ctx, table, 1.0, norm, ws)
    assert norm.item() == math.inf
    assert bool((grads[0] == 0).all()) and bool(grads[1][8999].isnan()) and bool((grads[1][:8999] == 0).all())
    grads = make([100, 9000], (F32,), 1)
    grads[0][3] = float("nan")
    table = ops.GradTable(grads)
    coef = torch.empty(1, device="cuda")
    ops.grad_norm(ctx, table, norm, ws, max_norm=1.0, coef=coef)
    assert math.isnan(norm.item()) and math.isnan(coef.item())
    ops.clip_grad_norm(ctx, table, 1.0, norm, ws)
    assert all(bool(g.isnan().all()) for g in grads)


def test_nothing_to_clip(ctx):
    from sirius_amd import ops
    grads = make([0, 0], (F32,), 1)
    table = ops.GradTable(grads)
    norm, ws, coef = torch.full((1,), 5.0, device="cuda"), workspace(table), torch.empty(1, device="cuda")
    ops.clip_grad_norm(ctx, table, 1.0, norm, ws)
    assert norm.item() == 0.0
    zeros = [torch.zeros(4097, device="cuda")]
    table = ops.GradTable(zeros)
    ops.grad_norm(ctx, table, norm, workspace(table), max_norm=0.0, coef=coef)
    assert norm.item() == 0.0 and coef.item() == 0.0


def test_same_bits_every_time(ctx):
    from sirius_amd import ops
    grads = make([3_000_000, 5, 17_000_001], (F32,), 2)
    table = ops.GradTable(grads)
    ws, got = workspace(table), []
    for _ in range(5):
        norm = torch.empty(1, device="cuda")
        ops.grad_norm(ctx, table, norm, ws)
        got.append(norm.item())
    assert len(set(got)) == 1


@pytest.mark.parametrize("optimizer", ["adamw", "sgd"])
def test_step_with_a_factor_is_the_step_on_scaled_gradients(ctx, optimizer):
    """grad_scale multiplies the gradient before anything else: bit for bit the step on gradients scaled ahead."""
    from sirius_amd import ops
    for n in (1, 1000, 4099):
        p, g, m, v = make([n, n, n, n], (F32,), 5)
        v = v.abs()
        scale = torch.full((1,), 0.37, device="cuda")
        states = []
        for scaled in (False, True):
            w, a, b = p.clone(), m.clone(), v.clone()
            shadow = torch.empty(n, dtype=BF16, device="cuda")
            grad, extra = (g, dict(grad_scale=scale)) if scaled else (g * scale, {})
            if optimizer == "adamw":
                step, scalars = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(2, device="cuda")
                ops.adamw_step(ctx, w, grad, a, b, step, scalars, lr=1e-2, shadow=shadow, **extra)
            else:
                ops.sgd_momentum_step(ctx, w, grad, a, 1e-2, 0.9, 1e-2, shadow=shadow, **extra)
            states.append((w, a, b, shadow))
        for x, y in zip(*states):
            assert torch.equal(x, y)


def test_refusals(ctx):
    from sirius_amd import ops
    from sirius_amd._lib import TorchColHipError
    buf = torch.zeros(1000, device="cuda")
    with pytest.raises(AssertionError):
        ops.GradTable([buf[:500], buf[:500]])                      # the same twice, in place
    with pytest.raises(AssertionError):
        ops.GradTable([buf[:500], buf[499:]])                      # overlapping views
    with pytest.raises(AssertionError):
        ops.GradTable([buf[:100], buf[200:300]], out=[buf[100:200], buf[250:350]])   # an output over another gradient
    with pytest.raises(AssertionError):
        ops.GradTable([buf[:100]], out=[buf[50:150]])              # shifted over itself
    with pytest.raises(AssertionError):
        ops.GradTable([buf[:100]], out=[buf[100:201]])             # another size
    with pytest.raises(AssertionError):
        ops.GradTable([])
    with pytest.raises(TypeError):
        ops.GradTable([buf.half()])
    with pytest.raises(ValueError):
        ops.GradTable([torch.zeros(4)])
    with pytest.raises(ValueError):
        ops.GradTable([buf[::2]])
    ops.GradTable([buf[:500], buf[:500]], out=[torch.empty(500, device="cuda") for _ in range(2)])   # read twice: allowed
    table = ops.GradTable([buf])
    norm, ws = torch.empty(1, device="cuda"), workspace(table)
    for bad in (-1.0, float("nan")):
        with pytest.raises(TorchColHipError):
            ops.clip_grad_norm(ctx, table, bad, norm, ws)
        with pytest.raises(TorchColHipError):
            ops.grad_norm(ctx, table, norm, ws, max_norm=bad, coef=norm.clone())
    with pytest.raises(AssertionError):
        ops.clip_grad_norm(ctx, table, 1.0, norm.double(), ws)
    with pytest.raises(AssertionError):
        ops.grad_norm(ctx, table, norm, ws, max_norm=1.0)
    with pytest.raises(AssertionError):
        ops.clip_grad_norm(ctx, table, 1.0, norm, ws[:4])
    with pytest.raises(AssertionError):
        ops.sgd_momentum_step(ctx, buf, buf.clone(), buf.clone(), 0.1, 0.9, 0.0, grad_scale=torch.ones(2, device="cuda"))
