"""What the norms at a block's boundary refuse at the C ABI and in the wrapper, without a GPU; and the oracle's gradients against
differences of its forward form."""
import ctypes

import pytest
import torch

from oracle import block_ops as O

BF16, F32 = 1, 0
P = [ctypes.c_void_p(0x1000000 * i) for i in range(1, 24)]
ODD = ctypes.c_void_p(0x1000008)


def last():
    from sirius_amd._lib import lib
    return (lib().tch_last_error() or b"").decode()


def fwd(dtype=BF16, layer=0, x=P[0], ldx=64, branch=P[1], ldb=64, total=P[2], ldt=64, y=P[3], ldy=64, stats=P[4], weight=P[5], bias=None, pw=P[6],
        pb=None, gate=P[7], gate_f32=1, gates=1, scale=1.0, eps=1e-5, packed=None, codes=None, format=0, rows=4, C=64):
    from sirius_amd._lib import lib
    return lib().tch_residual_norm_fwd(None, dtype, layer, x, ldx, branch, ldb, total, ldt, y, ldy, stats, weight, bias, pw, pb, gate, gate_f32, gates,
                                       scale, eps, packed, codes, format, rows, C)


def bwd(dtype=BF16, layer=0, dy=P[0], lddy=64, dtotal=P[1], lddt=64, total=P[2], ldt=64, branch=P[3], ldb=64, dx=P[8], lddx=64, dbranch=P[9], lddb=64,
        stats=P[4], weight=P[5], pw=P[6], pb=None, gate=P[7], gate_f32=1, gates=1, scale=1.0, dw=P[10], db=None, dpw=P[11], dpb=None, dgate=P[12],
        accumulate=0, rows=4, C=64, ws=P[13], ws_bytes=1 << 20):
    from sirius_amd._lib import lib
    return lib().tch_residual_norm_bwd(None, dtype, layer, dy, lddy, dtotal, lddt, total, ldt, branch, ldb, dx, lddx, dbranch, lddb, stats, weight, pw,
                                       pb, gate, gate_f32, gates, scale, dw, db, dpw, dpb, dgate, accumulate, rows, C, ws, ws_bytes)


@pytest.mark.parametrize("change", [
    dict(dtype=2), dict(rows=-1), dict(rows=1 << 31), dict(C=0), dict(C=60), dict(C=8200, ldx=8200, ldb=8200, ldt=8200, ldy=8200), dict(dtype=F32, C=62),
    dict(gates=0), dict(gates=3), dict(gates=8), dict(x=None), dict(stats=None), dict(total=None), dict(branch=None), dict(y=None), dict(weight=None),
    dict(branch=None, total=None), dict(branch=None, total=None, pw=None), dict(branch=None, total=None, pw=None, gate=None, scale=2.0),
    dict(branch=None, total=None, pw=None, gate=None, weight=None, y=None), dict(pw=None, pb=P[14]), dict(weight=None, y=None, bias=P[14]), dict(gate=None, gates=2),
    dict(eps=-1.0), dict(x=ODD), dict(branch=ODD), dict(total=ODD), dict(y=ODD), dict(ldx=56), dict(ldx=68), dict(ldy=0), dict(weight=ODD), dict(gate=ODD),
    dict(stats=ODD), dict(packed=P[15]), dict(codes=P[15]), dict(packed=P[15], codes=P[16], format=2), dict(packed=ODD, codes=P[16]),
    dict(weight=None, y=None, packed=P[15], codes=P[16]), dict(y=P[2]), dict(total=P[5]), dict(stats=P[0]), dict(y=P[7]), dict(packed=P[0], codes=P[16]),
    dict(total=ctypes.c_void_p(0x1000010))], ids=str)
def test_forward(change):
    assert fwd(**change) == -22 and "residual_norm_fwd" in last()


@pytest.mark.parametrize("change", [
    dict(dtype=2), dict(rows=-1), dict(C=60), dict(C=8200), dict(gates=3), dict(stats=None), dict(dy=None), dict(total=None), dict(weight=None, dw=None, dy=None, dtotal=None),
    dict(branch=None), dict(dbranch=None), dict(branch=None, dbranch=None), dict(branch=None, dbranch=None, pw=None, gate=None, dpw=None, dgate=None, dx=None),
    dict(branch=None, dbranch=None, pw=None, gate=None, dpw=None, dgate=None, scale=2.0), dict(gate=None, dgate=None, gates=2), dict(weight=None, dy=None),
    dict(pw=None), dict(gate=None), dict(pw=None, dpw=None, pb=P[14]), dict(dy=ODD), dict(dx=ODD), dict(lddx=60), dict(dw=ODD), dict(ws=ODD), dict(ws=None),
    dict(ws_bytes=100), dict(dx=P[9]), dict(dx=P[5]), dict(dw=P[11]), dict(dw=P[0]), dict(ws=P[0]), dict(dgate=P[7])], ids=str)
def test_backward(change):
    assert bwd(**change) == -22 and "residual_norm_bwd" in last()


def test_no_rows_is_no_error():
    assert fwd(rows=0, x=None, stats=None) == 0
    assert bwd(rows=0, dy=None, accumulate=1) == 0


def test_workspace_bytes():
    from sirius_amd._lib import lib
    need = lib().tch_residual_norm_bwd_workspace_bytes
    assert need(0, 64, 1) == need(4, 0, 1) == need(4, 64, 0) == need(4, 64, 3) == need(4, 16384, 1) == 0
    assert need(8192, 1024, 1) > 0 and need(8192, 1024, 8) > 0 and need(8192, 1024, 8192) > 0
    assert "workspace" in (last() if bwd(ws_bytes=need(4, 64, 1) // 4) else "")


def test_wrapper():
    from sirius_amd import ops

    class Here:
        handle = None

        class stream:
            device = torch.device("cpu")
    with pytest.raises(ValueError, match="norm"):
        ops._norm_args(Here, "batch", 8, 4, torch.float32, None)
    for gate, rows in ((torch.zeros(3, 8), 4), (torch.zeros(1, 4), 4), (torch.zeros(2, 8, dtype=torch.float64), 4), (torch.zeros(8, 2).t(), 4)):
        with pytest.raises(AssertionError, match="gate"):
            ops._norm_args(Here, "rms", 8, rows, torch.float32, gate)
    with pytest.raises(ValueError, match="GPU"):
        ops.residual_norm_fwd(Here, torch.zeros(2, 8), None, None, None, None)


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("post,gates,pre", [(True, 2, True), (True, 1, False), (False, 2, True), (False, 0, True)])
def test_the_oracles_gradients_against_differences(kind, post, gates, pre):
    g = torch.Generator()
    g.manual_seed(1)
    rows, C = 4, 12
    new = lambda *shape: torch.randn(*shape, generator=g, dtype=torch.float64)  # noqa: E731
    v = dict(x=new(rows, C), branch=new(rows, C), weight=new(C) if pre else None, bias=new(C) if pre else None, post_weight=new(C) if post else None,
             post_bias=new(C) if post else None, gate=new(gates, C) if gates else None)
    dy, dtotal = new(rows, C), new(rows, C)

    def loss(**change):
        a = dict(v, **change)
        total = O.boundary(a["x"], a["branch"], kind, a["post_weight"], a["post_bias"], a["gate"], 1.5)[0]
        out = (total * dtotal).sum()
        return out + (O.norm(total, kind, a["weight"], a["bias"])[0] * dy).sum() if pre else out
    total = O.boundary(v["x"], v["branch"], kind, v["post_weight"], v["post_bias"], v["gate"], 1.5)[0]
    grads = O.boundary_grads(dy if pre else None, dtotal, total, v["branch"], kind, v["weight"], v["post_weight"], v["post_bias"], v["gate"], 1.5)
    for name, value in v.items():
        if value is None:
            continue
        along, h = new(*value.shape), 1e-5
        slope = (loss(**{name: value + h * along}) - loss(**{name: value - h * along})) / (2 * h)
        mine = (grads["d" + name][0].view_as(value) * along).sum()
        assert abs(slope - mine) <= 1e-7 * (1 + abs(slope)), name


def test_no_gradient_at_all():
    """Refused as such: a StopIteration would quietly end the generator that the call is made in."""
    from sirius_amd import ops
    with pytest.raises(AssertionError, match="no gradient"):
        ops.residual_norm_bwd(None, None, None, None, None, None, None, None)
