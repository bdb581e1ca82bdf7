"""The norms at a block's boundary and their gradients against the formulas in 64 bits; tolerances count the roundings on the way
(oracle/block_ops.py) and half a step of the type that a result is stored in."""
import pytest
import torch

from oracle import block_ops as O

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
GRADS = ("dweight", "dbias", "dpost_weight", "dpost_bias", "dgate")


def normal(gen, *shape, dtype=torch.float32, std=1.0, mean=0.0):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(mean, std, generator=gen)


def make(rows, C, dtype, kind, pre=True, branch=True, post=True, gates=1, gate="f32", biases=True, seed=0, mean=0.3):
    """The tensors of a call, in the types that it takes them in."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt = TYPES[dtype]
    vector = lambda m: normal(gen, C, std=0.3, mean=m)  # noqa: E731
    s = dict(x=normal(gen, rows, C, dtype=dt, std=2.0, mean=mean), branch=normal(gen, rows, C, dtype=dt, mean=mean) if branch else None)
    s["weight"], s["bias"] = (vector(1.0), vector(0.0) if biases else None) if pre else (None, None)
    s["post_weight"], s["post_bias"] = (vector(1.0), vector(0.1) if biases else None) if branch and post else (None, None)
    s["gate"] = None
    if branch and gates:
        s["gate"] = normal(gen, gates, C, dtype=torch.float32 if gate == "f32" else dt, mean=0.5, std=0.5)
    s["dy"] = normal(gen, rows, C, dtype=dt) if pre else None
    s["dtotal"] = normal(gen, rows, C, dtype=dt)
    return s


def wide(t):
    return None if t is None else t.double()


def close(name, got, ref, err, stored=None):
    got = got.double()
    step = 0.0 if stored is None else torch.finfo(stored).eps / 2
    tol = err + step * ref.abs() + 1e-37
    bad = ~((got - ref.view_as(got)).abs() <= tol.view_as(got))
    assert not bad.any(), (name, int(bad.sum()), float(((got - ref.view_as(got)).abs() / tol.view_as(got)).max()))


def forward(ctx, s, kind, scale, eps=1e-5, **more):
    from sirius_amd import ops
    rows, C = s["x"].shape
    out = dict(total=torch.empty_like(s["x"]) if s["branch"] is not None else None, y=torch.empty_like(s["x"]) if s["weight"] is not None else None,
               stats=torch.full((rows, 4), 9.0, device="cuda"))
    out.update(more)
    ops.residual_norm_fwd(ctx, s["x"], s["branch"], out["total"], out["y"], out["stats"], kind=kind, weight=s["weight"], bias=s["bias"],
                          post_weight=s["post_weight"], post_bias=s["post_bias"], gate=s["gate"], scale=scale, eps=eps, packed=out.get("packed"))
    return out


def check_forward(s, out, kind, scale, eps=1e-5, x=None, branch=None):
    dt = s["x"].dtype
    x = wide(s["x"] if x is None else x)
    branch = wide(s["branch"] if branch is None else branch)
    total = x
    if branch is not None:
        ref, err = O.boundary(x, branch, kind, wide(s["post_weight"]), wide(s["post_bias"]), wide(s["gate"]), scale, eps)
        close("total", out["total"], ref, err, dt)
        total = wide(out["total"])
    if s["weight"] is not None:
        ref, err = O.norm(total, kind, wide(s["weight"]), wide(s["bias"]), eps)
        close("y", out["y"], ref, err, dt)


def backward(ctx, s, total, stats, kind, scale, accumulate=False, dx=None, dbranch=None, grads=None):
    from sirius_amd import ops
    rows, C = s["x"].shape
    out = dict(dx=torch.empty_like(s["x"]) if dx is None else dx, dbranch=None)
    if s["branch"] is not None:
        out["dbranch"] = torch.empty_like(s["x"]) if dbranch is None else dbranch
    have = dict(dweight="weight", dbias="bias", dpost_weight="post_weight", dpost_bias="post_bias", dgate="gate")
    for name, of in have.items():
        out[name] = None if s[of] is None else torch.full(s[of].shape, 0.5, device="cuda")
    if grads is not None:
        out = {k: v if not k in have or k in grads else None for k, v in out.items()}
    ws = torch.empty(ops.residual_norm_bwd_workspace_bytes(total, gate=s["gate"]), dtype=torch.uint8, device="cuda").fill_(255)
    ops.residual_norm_bwd(ctx, s["dy"], s["dtotal"], total, s["branch"], out["dx"], out["dbranch"], stats, kind=kind, weight=s["weight"],
                          post_weight=s["post_weight"], post_bias=s["post_bias"], gate=s["gate"], scale=scale,
                          **{k: out[k] for k in GRADS}, accumulate=accumulate, workspace=ws)
    return out


def check_backward(s, out, total, kind, scale, eps=1e-5, accumulate=False, stat_err=None, inputs=None):
    # statistics as the forward pass leaves them: within hat_error of v^ (the mean as large as the deviation here, at most)
    stat_err = 100 * O.U if stat_err is None else stat_err
    v = {k: wide(t) for k, t in (inputs or s).items()}
    ref = O.boundary_grads(v["dy"], v["dtotal"], wide(total), v["branch"], kind, v["weight"], v["post_weight"], v["post_bias"], v["gate"], scale, eps, stat_err)
    for name, got in out.items():
        if got is None:
            continue
        value, err = ref[name]
        if name in GRADS:
            value = value + (0.5 if accumulate else 0.0)
            close(name, got, value, err + 2 * O.U * value.abs() + (2 * O.U if accumulate else 0.0))
        else:
            close(name, got, value, err, s["x"].dtype)


SHAPES = [(1, 8), (5, 128), (37, 200), (16, 256), (3, 264), (33, 512), (9, 520), (70, 1000), (11, 1536), (4, 2304), (6, 4096), (3, 8192), (300, 768)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("rows,C", SHAPES, ids=str)
def test_all_of_it(ctx, dtype, kind, rows, C):
    s = make(rows, C, dtype, kind)
    out = forward(ctx, s, kind, 1.25)
    check_forward(s, out, kind, 1.25)
    check_backward(s, backward(ctx, s, out["total"], out["stats"], kind, 1.25), out["total"], kind, 1.25)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("parts", [dict(post=False), dict(post=False, gates=0), dict(gates=0), dict(pre=False), dict(pre=False, post=False),
                                   dict(branch=False), dict(biases=False), dict(gate="own"), dict(pre=False, gates=0, biases=False)], ids=str)
@pytest.mark.parametrize("rows,C", [(1, 64), (29, 712), (12, 2048)], ids=str)
def test_parts_of_it(ctx, dtype, kind, parts, rows, C):
    s = make(rows, C, dtype, kind, **parts)
    scale = 0.5 if s["branch"] is not None else 1.0
    out = forward(ctx, s, kind, scale)
    check_forward(s, out, kind, scale)
    total = out["total"] if s["branch"] is not None else s["x"]
    check_backward(s, backward(ctx, s, total, out["stats"], kind, scale), total, kind, scale)
    if s["weight"] is not None:
        s["dtotal"] = None       # the last boundary: nothing else reads the sum
        check_backward(s, backward(ctx, s, total, out["stats"], kind, scale), total, kind, scale)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("gate", ["f32", "own"])
@pytest.mark.parametrize("rows,C,gates", [(6, 128, 3), (24, 96, 24), (390, 256, 6), (400, 520, 2), (500, 64, 100), (77, 1024, 7), (64, 8, 8), (9, 4096, 3),
                                          (6144, 40, 3), (5000, 72, 1250), (20000, 16, 4)], ids=str)
@pytest.mark.parametrize("post", [True, False])
def test_gates_of_samples(ctx, dtype, gate, rows, C, gates, post):
    """Samples of many rows over several workgroups, and several samples in one."""
    s = make(rows, C, dtype, "layer", gates=gates, gate=gate, post=post)
    out = forward(ctx, s, "layer", 1.0)
    check_forward(s, out, "layer", 1.0)
    check_backward(s, backward(ctx, s, out["total"], out["stats"], "layer", 1.0), out["total"], "layer", 1.0)
    check_backward(s, backward(ctx, s, out["total"], out["stats"], "layer", 1.0, accumulate=True), out["total"], "layer", 1.0, accumulate=True)


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_the_same_bits_every_run_and_single_gradients(ctx, kind):
    s = make(700, 520, "bf16", kind, gates=4)
    out = forward(ctx, s, kind, 1.0)
    first = backward(ctx, s, out["total"], out["stats"], kind, 1.0)
    again = backward(ctx, s, out["total"], out["stats"], kind, 1.0)
    for k, v in first.items():
        assert torch.equal(v, again[k]), k
    for name in GRADS:
        alone = backward(ctx, s, out["total"], out["stats"], kind, 1.0, grads=(name,))
        assert torch.equal(alone[name], first[name]) and torch.equal(alone["dbranch"], first["dbranch"])
    none = backward(ctx, s, out["total"], out["stats"], kind, 1.0, grads=())
    assert torch.equal(none["dx"], first["dx"])


def test_rows_of_zeros_and_of_one_value(ctx):
    """Padding rows: a deviation of 0, held off it by eps."""
    s = make(6, 136, "f32", "layer")
    s["x"][1:3], s["branch"][1:4] = 0.0, 0.0
    s["branch"][4] = 3.0
    out = forward(ctx, s, "layer", 1.0)
    assert all(torch.isfinite(t).all() for t in out.values())
    check_forward(s, out, "layer", 1.0)
    # (a row of one value c: what the mean is off, up to 30 u c, is magnified by 1 / sqrt(eps) = 316; hat_error has that factor)
    got = backward(ctx, s, out["total"], out["stats"], "layer", 1.0)
    assert all(torch.isfinite(t).all() for t in got.values())
    check_backward(s, got, out["total"], "layer", 1.0, stat_err=30 * O.U * 3.0 * 317)


def test_large_means(ctx):
    """A mean of a thousand deviations: what a plain sum of squares would lose."""
    s = make(8, 1544, "f32", "layer", mean=1000.0)
    out = forward(ctx, s, "layer", 1.0)
    check_forward(s, out, "layer", 1.0)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_not_a_number_stays_in_its_row(ctx, bad):
    s = make(20, 256, "bf16", "rms")
    s["branch"][7, 3] = bad
    out = forward(ctx, s, "rms", 1.0)
    rows = torch.isfinite(out["y"]).all(1)
    assert not rows[7] and rows.sum() == 19
    got = backward(ctx, s, out["total"], out["stats"], "rms", 1.0)
    rows = torch.isfinite(got["dbranch"]).all(1)
    assert not rows[7] and rows.sum() == 19


@pytest.mark.parametrize("dtype", list(TYPES))
def test_columns_of_wider_tensors(ctx, dtype):
    from sirius_amd import ops
    rows, C, kind = 21, 264, "layer"
    s = make(rows, C, dtype, kind)
    spread = {k: torch.full((rows + 2, C + 16 * (i + 1)), 5.0, dtype=TYPES[dtype], device="cuda")
              for i, k in enumerate(("x", "branch", "total", "y", "dy", "dtotal", "dx", "dbranch"))}
    view = {k: v[1:-1, 8:8 + C] for k, v in spread.items()}
    dense = forward(ctx, s, kind, 1.5)
    for k in ("x", "branch", "dy", "dtotal"):
        view[k].copy_(s[k])
    strided = dict(s, **{k: view[k] for k in ("x", "branch", "dy", "dtotal")})
    out = forward(ctx, strided, kind, 1.5, total=view["total"], y=view["y"])
    assert torch.equal(out["total"], dense["total"]) and torch.equal(out["y"], dense["y"]) and torch.equal(out["stats"], dense["stats"])
    a = backward(ctx, s, dense["total"], dense["stats"], kind, 1.5)
    b = backward(ctx, strided, view["total"], dense["stats"], kind, 1.5, dx=view["dx"], dbranch=view["dbranch"])
    for k in a:
        assert torch.equal(a[k], b[k]), k
    for k, v in spread.items():
        view[k].fill_(5.0)
        assert (v == 5.0).all(), k
    assert ops.NORMS["layer"] == 1


@pytest.mark.parametrize("rows,C", [(50, 128), (40, 2304)], ids=str)
def test_in_place(ctx, rows, C):
    s = make(rows, C, "bf16", "rms")
    want = forward(ctx, s, "rms", 1.0)
    grads = backward(ctx, s, want["total"], want["stats"], "rms", 1.0)
    t = dict(s, x=s["x"].clone(), branch=s["branch"].clone())
    out = forward(ctx, t, "rms", 1.0, total=t["x"], y=t["branch"])
    assert torch.equal(out["total"], want["total"]) and torch.equal(out["y"], want["y"])
    t = dict(s, dy=s["dy"].clone(), dtotal=s["dtotal"].clone(), branch=s["branch"].clone())
    got = backward(ctx, t, want["total"], want["stats"], "rms", 1.0, dx=t["dtotal"], dbranch=t["dy"])
    for k in grads:
        assert torch.equal(got[k], grads[k]), k


def test_no_rows(ctx):
    s = make(0, 64, "f32", "rms")
    out = forward(ctx, s, "rms", 1.0)
    got = backward(ctx, s, out["total"], out["stats"], "rms", 1.0)
    assert all((got[k] == 0).all() for k in GRADS if got[k] is not None)
    got = backward(ctx, s, out["total"], out["stats"], "rms", 1.0, accumulate=True)
    assert all((got[k] == 0.5).all() for k in GRADS if got[k] is not None)


@pytest.mark.parametrize("format", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,C", [(1, 8), (9, 128), (31, 200), (7, 520), (5, 1000), (3, 4096)], ids=str)
def test_kept_in_8_bits(ctx, dtype, format, rows, C):
    """What is kept is y as it is stored, by the definition."""
    from sirius_amd import ops
    s = make(rows, C, dtype, "layer")
    s["branch"][0, C // 2] = 40.0
    packed = ops.Packed8.empty(rows, C, format)
    out = forward(ctx, s, "layer", 1.0, packed=packed)
    assert torch.equal(out["y"], forward(ctx, s, "layer", 1.0)["y"])
    kept, codes = O.packed(out["y"], format)
    assert torch.equal(packed.scales, codes)
    back = torch.empty_like(out["y"])
    ops.unpack8(ctx, packed, back)
    assert torch.equal(back.double(), kept)


def test_recorded_and_replayed(ctx):
    """Forward and backward as one program, several times, over new values in the same buffers, with eager calls in between."""
    from sirius_amd import ops
    c, prog = ops.Context(), ops.Program()
    s = make(130, 1032, "bf16", "layer", gates=5)
    keep = {}

    def calls(context):
        out = forward(context, s, "layer", 1.0, **{k: keep[k] for k in ("total", "y", "stats") if k in keep})
        g = dict(dx=keep.get("dx"), dbranch=keep.get("dbranch"))
        return out, g
    total, y, stats = torch.empty_like(s["x"]), torch.empty_like(s["x"]), torch.empty(130, 4, device="cuda")
    dx, db = torch.empty_like(s["x"]), torch.empty_like(s["x"])
    grads = {k: torch.empty(s[k[1:]].shape, device="cuda") for k in GRADS}
    ws = torch.empty(ops.residual_norm_bwd_workspace_bytes(s["x"], gate=s["gate"]), dtype=torch.uint8, device="cuda")
    args = dict(kind="layer", weight=s["weight"], post_weight=s["post_weight"], post_bias=s["post_bias"], gate=s["gate"], scale=1.0)
    c.begin_record(prog)
    ops.residual_norm_fwd(c, s["x"], s["branch"], total, y, stats, bias=s["bias"], **args)
    ops.residual_norm_bwd(c, s["dy"], s["dtotal"], total, s["branch"], dx, db, stats, workspace=ws, **args, **grads)
    c.end_record()
    for step in range(3):
        fresh = make(130, 1032, "bf16", "layer", gates=5, seed=step + 1)
        for k, v in fresh.items():
            s[k].copy_(v)
        ws.fill_(255)
        c.run(prog)
        out, _ = calls(ctx)
        want = backward(ctx, s, out["total"], out["stats"], "layer", 1.0)
        c.synchronize()
        assert torch.equal(total, out["total"]) and torch.equal(y, out["y"])
        for k, v in dict(grads, dx=dx, dbranch=db).items():
            assert torch.equal(v, want[k]), (step, k)


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_against_differences(ctx, kind):
    """The kernel's gradients along a direction against differences of the formula in 64 bits: h = 2^-12, an error of h^2 times the third
    derivative (below 100 here: a few factors of size one each) and of the gradients' own bounds."""
    s = make(10, 72, "f32", kind, gates=2)
    out = forward(ctx, s, kind, 1.25)
    # the sum as a leaf of its own: dx and the branch's side from dtotal' = dtotal + (gradient through y), as the kernel takes it
    got = backward(ctx, s, out["total"], out["stats"], kind, 1.25)
    v = {k: wide(t) for k, t in s.items()}
    gen = torch.Generator(device="cuda")
    gen.manual_seed(3)
    names = ("x", "branch", "weight", "bias", "post_weight", "post_bias", "gate")
    along = {k: normal(gen, *s[k].shape).double() for k in names}

    def loss(h):
        a = {k: v[k] + h * along[k] for k in names}
        total = O.boundary(a["x"], a["branch"], kind, a["post_weight"], a["post_bias"], a["gate"], 1.25)[0]
        return (O.norm(total, kind, a["weight"], a["bias"])[0] * v["dy"]).sum() + (total * v["dtotal"]).sum()
    h = 2.0 ** -12
    slope = ((loss(h) - loss(-h)) / (2 * h)).item()
    mine = sum((got["d" + k].double() * along[k]).sum() for k in names).item()
    ref = O.boundary_grads(v["dy"], v["dtotal"], wide(out["total"]), v["branch"], kind, v["weight"], v["post_weight"], v["post_bias"], v["gate"], 1.25, stat_err=100 * O.U)
    tol = sum((ref["d" + k][1].abs() * along[k].view_as(ref["d" + k][0]).abs()).sum() for k in names).item()
    size = sum((ref["d" + k][0].abs() * along[k].view_as(ref["d" + k][0]).abs()).sum() for k in names).item()
    # (total is stored in fp32: the gradients are taken half a step beside the formula's place)
    assert abs(slope - mine) <= tol + 100 * h * h * size + 2.0 ** -20 * size, (slope, mine, tol, size)


def test_rows_beyond_four_gib(ctx):
    """Rows 2^31 bytes apart: 64-bit offsets, forward and back."""
    rows, C, ld = 4, 520, 2 ** 30 + 64
    s = make(rows, C, "bf16", "layer")
    want = forward(ctx, s, "layer", 1.0)
    grads = backward(ctx, s, want["total"], want["stats"], "layer", 1.0)
    far = {k: torch.empty(rows * ld, dtype=torch.bfloat16, device="cuda").view(rows, ld)[:, :C] for k in ("x", "branch", "dy", "dtotal", "total", "y", "dx", "dbranch")}
    for k in ("x", "branch", "dy", "dtotal"):
        far[k].copy_(s[k])
    t = dict(s, **{k: far[k] for k in ("x", "branch", "dy", "dtotal")})
    out = forward(ctx, t, "layer", 1.0, total=far["total"], y=far["y"])
    assert torch.equal(out["total"], want["total"]) and torch.equal(out["y"], want["y"])
    got = backward(ctx, t, far["total"], out["stats"], "layer", 1.0, dx=far["dx"], dbranch=far["dbranch"])
    for k in grads:
        assert torch.equal(got[k], grads[k]), k


@pytest.mark.parametrize("dtype", list(TYPES))
def test_more_than_the_cache_holds(ctx, dtype):
    """The kernels that stream past the cache give the same bits as those that do not: a part of the rows alone."""
    rows, C = (6000, 8192) if dtype == "bf16" else (9000, 4096)
    for kind in ("rms", "layer"):
        s = make(rows, C, dtype, kind, gates=1)
        out = forward(ctx, s, kind, 1.0)
        got = backward(ctx, s, out["total"], out["stats"], kind, 1.0)
        part = {k: t[:200].contiguous() if k in ("x", "branch", "dy", "dtotal") and t is not None else t for k, t in s.items()}
        few = forward(ctx, part, kind, 1.0)
        back = backward(ctx, part, few["total"], few["stats"], kind, 1.0)
        for k in ("total", "y", "stats"):
            assert torch.equal(out[k][:200], few[k]), k
        for k in ("dx", "dbranch"):
            assert torch.equal(got[k][:200], back[k]), k
        check_backward(s, {k: t for k, t in got.items() if k in GRADS}, out["total"], kind, 1.0)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("rows,C,gates", [(600, 4608, 300), (772, 8192, 193), (258, 6152, 258), (40, 8184, 5)], ids=str)
@pytest.mark.parametrize("post", [True, False])
def test_gates_of_long_rows(ctx, dtype, kind, rows, C, gates, post):
    """Rows of more than eight wavefronts: a workgroup has one gate, several, or a part of one's rows."""
    s = make(rows, C, dtype, kind, gates=gates, post=post)
    out = forward(ctx, s, kind, 1.25)
    check_forward(s, out, kind, 1.25)
    check_backward(s, backward(ctx, s, out["total"], out["stats"], kind, 1.25), out["total"], kind, 1.25)
    check_backward(s, backward(ctx, s, out["total"], out["stats"], kind, 1.25, accumulate=True), out["total"], kind, 1.25, accumulate=True)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("parts", [dict(post=False, gates=0), dict(gates=0), dict(pre=False), dict(pre=False, post=False), dict(branch=False), dict(biases=False)], ids=str)
@pytest.mark.parametrize("rows,C", [(300, 4104), (7, 5128), (513, 6144), (260, 7168)], ids=str)
def test_parts_of_long_rows(ctx, dtype, kind, parts, rows, C):
    s = make(rows, C, dtype, kind, **parts)
    scale = 0.5 if s["branch"] is not None else 1.0
    out = forward(ctx, s, kind, scale)
    check_forward(s, out, kind, scale)
    total = out["total"] if s["branch"] is not None else s["x"]
    check_backward(s, backward(ctx, s, total, out["stats"], kind, scale), total, kind, scale)
    if s["weight"] is not None:
        s["dtotal"] = None
        check_backward(s, backward(ctx, s, total, out["stats"], kind, scale), total, kind, scale)


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("rows,C", [(37, 200), (70, 1000), (300, 8192)], ids=str)
def test_nobody_wants_the_gradient_of_x(ctx, kind, rows, C):
    """dx None (the first block): everything else as with it, to the last bit."""
    from sirius_amd import ops
    s = make(rows, C, "bf16", kind)
    out = forward(ctx, s, kind, 1.0)
    want = backward(ctx, s, out["total"], out["stats"], kind, 1.0)
    got = {k: None if v is None else torch.empty_like(v) for k, v in want.items()}
    ws = torch.empty(ops.residual_norm_bwd_workspace_bytes(s["x"], s["gate"]), dtype=torch.uint8, device="cuda")
    ops.residual_norm_bwd(ctx, s["dy"], s["dtotal"], out["total"], s["branch"], None, got["dbranch"], out["stats"], kind=kind, weight=s["weight"],
                          post_weight=s["post_weight"], post_bias=s["post_bias"], gate=s["gate"], scale=1.0, workspace=ws, **{k: got[k] for k in GRADS})
    torch.cuda.synchronize()
    for k, v in want.items():
        assert k == "dx" or v is None or torch.equal(got[k], v), k


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("gates", [1, 4])
def test_every_row_of_more_than_the_cache_holds(ctx, dtype, kind, gates):
    """A workgroup of a streaming launch goes round many times: what it stores in each, and in the last one, which not all of them have, is
    to the last bit what launches over a sixth of the rows store, which do not stream.  (With a gate a sample too.)"""
    rows, C = (6008, 8192) if dtype == "bf16" else (9004, 4096)
    s = make(rows, C, dtype, kind, gates=gates)
    out = forward(ctx, s, kind, 1.25)
    got = backward(ctx, s, out["total"], out["stats"], kind, 1.25)
    each = rows // 4
    for gate in range(4):
        for r0, r1 in ((gate * each, gate * each + each // 2 + 1), (gate * each + each // 2 + 1, (gate + 1) * each)):
            part = {k: t[r0:r1].contiguous() if k in ("x", "branch", "dy", "dtotal") else t for k, t in s.items()}
            part["gate"] = s["gate"][gate % gates:gate % gates + 1].contiguous()
            few = forward(ctx, part, kind, 1.25)
            back = backward(ctx, part, few["total"], few["stats"], kind, 1.25)
            for k in ("total", "y", "stats"):
                assert torch.equal(out[k][r0:r1], few[k]), (k, r0)
            for k in ("dx", "dbranch"):
                assert torch.equal(got[k][r0:r1], back[k]), (k, r0)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("rows,C", [(40000, 128), (20001, 256), (9001, 512), (3001, 2304), (1030, 8192)], ids=str)
def test_in_place_over_many_rounds(ctx, dtype, kind, rows, C):
    """The next rows are on their way when a row's results go over what it was read from: all of them, in every place that may be shared."""
    s = make(rows, C, dtype, kind)
    want = forward(ctx, s, kind, 1.25)
    grads = backward(ctx, s, want["total"], want["stats"], kind, 1.25)
    for total, y in (("x", "branch"), ("branch", "x")):
        t = dict(s, x=s["x"].clone(), branch=s["branch"].clone())
        out = forward(ctx, t, kind, 1.25, total=t[total], y=t[y])
        for k in ("total", "y", "stats"):
            assert torch.equal(out[k], want[k]), (k, total, y)
    for dx, dbranch in (("dtotal", "dy"), ("dy", "dtotal"), ("total", "branch"), ("branch", "total")):
        t = dict(s, **{k: s[k].clone() for k in ("dy", "dtotal", "branch")})
        t["total"] = want["total"].clone()
        got = backward(ctx, t, t["total"], want["stats"], kind, 1.25, dx=t[dx], dbranch=t[dbranch])
        for k in grads:
            assert torch.equal(got[k], grads[k]), (k, dx, dbranch)
