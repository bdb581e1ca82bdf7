"""Rotary positions and the rotation back against the formula in 64 bits.

Tolerance of an element y = s (a cos t - b sin t): half a step of its type, and in fp32 the factors s cos t and s sin t (the library's
sine and cosine within 2^-22, the product with s and the fused multiply-adds within 2^-23 together) on |a| + |b|.  The angle is taken
in 64 bits on both sides, each within 2^-52 of |p f| radians (and no nearer than 2^-50 of a turn)."""
import math

import pytest
import torch

gpu = pytest.mark.gpu
pytestmark = gpu
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def oracle(x, freqs, head_dim, layout, positions, scale, back=False):
    """x [rows, width] -> (y, the tolerance but for the type's own rounding), in 64 bits on the CPU."""
    x, freqs = x.detach().double().cpu(), freqs.double().cpu()
    rows, width = x.shape
    h = x.view(rows, width // head_dim, head_dim)
    r = 2 * freqs.numel()
    angle = (positions.double().cpu()[:, None] * freqs)[:, None, :]
    c, s = torch.cos(angle) * scale, torch.sin(angle) * scale * (-1 if back else 1)
    a, b = (h[..., :r // 2], h[..., r // 2:r]) if layout == "half" else (h[..., 0:r:2], h[..., 1:r:2])
    y, tol = h.clone(), torch.zeros_like(h)
    off = (a.abs() + b.abs()) * abs(scale) * (2.0 ** -22 + 2.0 ** -23 + 2 * angle.abs() * 2.0 ** -52 + 2.0 ** -47)
    u, v = a * c - b * s, b * c + a * s
    if layout == "half":
        y[..., :r // 2], y[..., r // 2:r] = u, v
        tol[..., :r // 2], tol[..., r // 2:r] = off, off
    else:
        y[..., 0:r:2], y[..., 1:r:2] = u, v
        tol[..., 0:r:2], tol[..., 1:r:2] = off, off
    return y.view(rows, width), tol.view(rows, width)


def close(got, ref, tol, dtype):
    got = got.double().cpu()
    bad = ~((got - ref).abs() <= tol + ref.abs() * (torch.finfo(dtype).eps / 2) + torch.finfo(dtype).tiny)
    assert not bad.any(), (int(bad.sum()), float((got - ref).abs().max()))


def make(shape, dtype, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=g)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("heads,head_dim,rot", [(1, 2, 2), (3, 16, 16), (12, 64, 64), (5, 80, 20), (7, 40, 10), (3, 9, 6), (2, 7, 2), (40, 128, 128),
                                                (64, 256, 64), (1, 4096, 4096), (300, 8, 8)], ids=str)
@pytest.mark.parametrize("rows,back", [(1, False), (37, True)], ids=str)
def test_against_the_formula(ctx, dtype, layout, heads, head_dim, rot, rows, back):
    from sirius_amd import ops
    dt = TYPES[dtype]
    x, freqs = make((rows, heads * head_dim), dt), ops.rotary_freqs(rot).cuda()
    y = torch.empty_like(x)
    at = torch.arange(rows, dtype=torch.int64, device="cuda") * 4001 + 17
    (ops.rotary_bwd if back else ops.rotary_fwd)(ctx, x, y, freqs, head_dim, layout=layout, positions=at, scale=1.25)
    ref, tol = oracle(x, freqs, head_dim, layout, at, 1.25, back)
    close(y, ref, tol, dt)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_sequences_are_counted_and_given_alike(ctx, dtype):
    from sirius_amd import ops
    B, T, heads, D = 3, 129, 6, 64
    x, freqs = make((B, T, heads * D), TYPES[dtype]), ops.rotary_freqs(D, base=500.0).cuda()
    counted, narrow, wide = (torch.empty_like(x) for _ in range(3))
    at = (torch.arange(T, device="cuda") + 11).expand(B, T).contiguous()
    ops.rotary_fwd(ctx, x, counted, freqs, D, start=11)
    ops.rotary_fwd(ctx, x, narrow, freqs, D, positions=at.int())
    ops.rotary_fwd(ctx, x, wide, freqs, D, positions=at)
    assert torch.equal(counted, narrow) and torch.equal(counted, wide)
    ref, tol = oracle(x.view(B * T, -1), freqs, D, "half", at.view(-1), 1.0)
    close(counted.view(B * T, -1), ref, tol, TYPES[dtype])


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("first,gap", [(0, 0), (1, 3), (2, 2), (8, 64)], ids=str)
def test_columns_of_a_wider_tensor_and_in_place(ctx, dtype, layout, first, gap):
    """Queries and keys of a packed projection, off any boundary; what lies beside them stays."""
    from sirius_amd import ops
    rows, heads, D = 33, 4, 24
    dt, width = TYPES[dtype], heads * D
    wide = make((rows, first + width + gap), dt)
    before, x = wide.clone(), wide[:, first:first + width]
    freqs = ops.rotary_freqs(16).cuda()
    at = torch.arange(rows, device="cuda")
    ref, tol = oracle(x, freqs, D, layout, at, 1.0)
    out = torch.full((rows + 2, first + width + gap), 7.0, dtype=dt, device="cuda")
    ops.rotary_fwd(ctx, x, out[1:-1, first:first + width], freqs, D, layout=layout, start=0, seq=rows)
    assert torch.equal(wide, before)
    close(out[1:-1, first:first + width], ref, tol, dt)
    out[1:-1, first:first + width] = 7.0
    assert (out == 7.0).all()
    ops.rotary_fwd(ctx, x, x, freqs, D, layout=layout, start=0, seq=rows)
    close(x, ref, tol, dt)
    keep = torch.ones_like(wide, dtype=torch.bool)
    keep[:, first:first + width] = False
    assert torch.equal(wide[keep], before[keep])


def test_far_and_negative_positions(ctx):
    from sirius_amd import ops
    at = torch.tensor([0, -1, -123456, 2 ** 20 + 1, 2 ** 24 - 1, 2 ** 31 - 1, 2 ** 31 + 5, 2 ** 33 + 3], device="cuda")
    x, freqs = make((at.numel(), 128), torch.float32), ops.rotary_freqs(128, factor=8.0, trained=4096).cuda()
    y = torch.empty_like(x)
    ops.rotary_fwd(ctx, x, y, freqs, 128, positions=at)
    ref, tol = oracle(x, freqs, 128, "half", at, 1.0)
    close(y, ref, tol, torch.float32)
    far = at[at >= 2 ** 31 - 1].tolist()
    ops.rotary_fwd(ctx, x, y, freqs, 128, start=far[1] - 6, seq=8)       # counted from beyond 2^31
    ref, tol = oracle(x, freqs, 128, "half", torch.arange(8) + far[1] - 6, 1.0)
    close(y, ref, tol, torch.float32)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_the_gradient_is_the_transpose(ctx, layout):
    """<dy, R x> = <R' dy, x> for unit vectors x: the columns of R against the rows of what rotary_bwd does (fp32: R is made of the same
    factors, so the two agree but for the signs' order of additions: to the last bit, there are no sums)."""
    from sirius_amd import ops
    D, rot = 12, 8
    freqs, at = ops.rotary_freqs(rot).cuda(), torch.full((D,), 5, device="cuda")
    eye = torch.eye(D, device="cuda")
    fwd, bwd = torch.empty_like(eye), torch.empty_like(eye)
    ops.rotary_fwd(ctx, eye, fwd, freqs, D, layout=layout, positions=at, scale=1.5)
    ops.rotary_bwd(ctx, eye, bwd, freqs, D, layout=layout, positions=at, scale=1.5)
    assert torch.equal(fwd, bwd.t())


def test_not_a_number_stays_in_its_pair(ctx):
    from sirius_amd import ops
    x, freqs = make((4, 64), torch.bfloat16), ops.rotary_freqs(32).cuda()
    x[1, 3], x[2, 40] = float("nan"), float("inf")
    y = torch.empty_like(x)
    ops.rotary_fwd(ctx, x, y, freqs, 64, start=1, seq=4)
    bad = ~torch.isfinite(y)
    want = torch.zeros_like(bad)
    want[1, 3] = want[1, 19] = want[2, 40] = True
    assert torch.equal(bad, want) and y[2, 40] == float("inf")


def test_no_rows(ctx):
    from sirius_amd import ops
    x = torch.empty(0, 64, device="cuda")
    ops.rotary_fwd(ctx, x, x, ops.rotary_freqs(64).cuda(), 64)


def test_recorded_and_replayed(ctx):
    from sirius_amd import ops
    c, prog = ops.Context(), ops.Program()
    x, freqs = make((64, 256), torch.bfloat16), ops.rotary_freqs(64).cuda()
    at, y, z = torch.arange(64, device="cuda"), torch.empty_like(x), torch.empty_like(x)
    c.begin_record(prog)
    ops.rotary_fwd(c, x, y, freqs, 64, positions=at)
    c.end_record()
    for step in range(3):       # new positions and values in the same buffers
        x.copy_(make((64, 256), torch.bfloat16, seed=step))
        at.add_(1000)
        c.run(prog)
        ops.rotary_fwd(c, x, z, freqs, 64, positions=at)
        c.synchronize()
        assert torch.equal(y, z)
        close(y, *oracle(x, freqs, 64, "half", at, 1.0), torch.bfloat16)


def test_rows_beyond_four_gib(ctx):
    """4.3 billion elements behind the first row: 64-bit offsets of rows."""
    from sirius_amd import ops
    rows, ld, D = 5, 2 ** 30 + 64, 64
    flat = torch.empty(rows * ld, dtype=torch.bfloat16, device="cuda")
    x = flat.view(rows, ld)[:, :2 * D]
    x.copy_(make((rows, 2 * D), torch.bfloat16))
    freqs, y = ops.rotary_freqs(D).cuda(), torch.empty(rows, 2 * D, dtype=torch.bfloat16, device="cuda")
    ops.rotary_fwd(ctx, x, y, freqs, D, start=math.floor(1e6), seq=rows)
    close(y, *oracle(x, freqs, D, "half", torch.arange(rows) + 1_000_000, 1.0), torch.bfloat16)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_more_than_the_cache_holds(ctx, dtype, layout):
    """The kernel that streams past the cache: the bits of the one that does not, on a part of the rows."""
    from sirius_amd import ops
    rows = 14_000 if dtype == "bf16" else 7_000
    x, freqs = make((rows, 40 * 128), TYPES[dtype]), ops.rotary_freqs(128).cuda()
    y, few = torch.empty_like(x), torch.empty_like(x[:300])
    ops.rotary_fwd(ctx, x, y, freqs, 128, layout=layout, start=0, seq=rows)
    ops.rotary_fwd(ctx, x[:300], few, freqs, 128, layout=layout, start=0, seq=rows)
    assert torch.equal(y[:300], few)
    close(y[-50:], *oracle(x[-50:], freqs, 128, layout, torch.arange(rows - 50, rows), 1.0), TYPES[dtype])
