"""What the linear layers, their weight gradients and the gradient norm refuse at the C ABI, without a GPU: every call here is turned
away by its arguments (the addresses are never read), with a message, and none aborts."""
import ctypes

import pytest

BF16, F32 = 1, 0
A, B, C, D = (ctypes.c_void_p(0x10000 * i) for i in range(1, 5))
ODD = ctypes.c_void_p(0x10008)


def refused(fn, *args):
    from sirius_amd._lib import lib
    rc = getattr(lib(), fn)(*args)
    message = lib().tch_last_error()
    assert rc == -22 and message, (fn, rc, message)
    return message.decode()


def fwd(dtype=BF16, x=A, ldx=64, w=B, y=C, ldy=32, bias=None, act=0, res=None, ldr=0, pre=None, ldp=0, M=4, K=64, N=32):
    return (None, dtype, x, ldx, w, y, ldy, bias, act, res, ldr, pre, ldp, M, K, N)


@pytest.mark.parametrize("change", [
    dict(dtype=2), dict(act=5), dict(act=-1), dict(M=-1), dict(K=0), dict(N=0), dict(N=-8), dict(K=60, ldx=64), dict(N=30), dict(dtype=F32, K=62),
    dict(x=None), dict(w=None), dict(y=None), dict(x=ODD), dict(w=ODD), dict(y=ODD), dict(bias=ODD), dict(res=ODD, ldr=32), dict(pre=ODD, ldp=32),
    dict(ldx=56), dict(ldx=68), dict(ldy=24), dict(res=D, ldr=0), dict(pre=D, ldp=36), dict(ldx=1 << 21), dict(M=1 << 31),
    dict(K=1 << 15, ldx=1 << 15, N=1 << 15), dict(K=1 << 22, ldx=1 << 22)], ids=str)
def test_linear_fwd(change):
    refused("tch_linear_fwd", *fwd(**change))


def test_messages_name_the_operator():
    assert "linear_fwd" in refused("tch_linear_fwd", *fwd(K=60))
    assert "gated_linear_fwd" in refused("tch_gated_linear_fwd", None, BF16, A, 64, B, C, 28, None, 4, None, 0, 4, 64, 28)
    assert "linear_dgrad" in refused("tch_linear_dgrad", None, BF16, A, 64, B, C, 32, 9, D, 32, None, 0, 4, 64, 32)


def test_no_rows_is_no_error():
    from sirius_amd._lib import lib
    assert lib().tch_linear_fwd(*fwd(M=0, x=None, y=None)) == 0
    assert lib().tch_act_bwd(None, BF16, None, 32, None, 32, None, None, 32, 1, 0, 32) == 0


def test_data_gradients():
    refused("tch_linear_dgrad", None, BF16, A, 64, B, C, 32, 4, None, 0, None, 0, 4, 64, 32)          # an activation without pre
    refused("tch_linear_dgrad_gated", None, BF16, A, 64, B, None, 0, C, None, 64, None, None, 0, 4, 4, 64, 32)
    refused("tch_linear_dgrad_gated", None, BF16, A, 64, B, D, 32, C, None, 64, None, None, 0, 4, 4, 64, 32)   # pre is 2 F wide
    refused("tch_linear_dgrad_gated", None, BF16, A, 64, B, D, 64, C, None, 32, None, None, 0, 4, 4, 64, 32)   # dpre too
    refused("tch_linear_dgrad_gated", None, F32, A, 64, B, D, 64, C, C, 64, None, None, 0, 4, 4, 64, 32)       # fp32 has no low part
    refused("tch_linear_dgrad_gated", None, BF16, A, 64, B, D, 64, C, None, 64, None, C, 32, 4, 4, 64, 32)     # h's low part without h
    refused("tch_linear_dgrad_gated", None, BF16, A, 64, B, D, 64, C, ODD, 64, None, None, 0, 4, 4, 64, 32)


def test_derivatives():
    refused("tch_act_bwd", None, BF16, A, 32, B, 32, C, None, 32, 7, 4, 32)
    refused("tch_act_bwd", None, BF16, A, 32, None, 32, C, None, 32, 1, 4, 32)
    refused("tch_act_bwd", None, F32, A, 32, B, 32, C, D, 32, 1, 4, 32)
    refused("tch_act_bwd", None, BF16, A, 24, B, 32, C, None, 32, 1, 4, 32)
    refused("tch_act_bwd", None, BF16, A, 1024, B, 1024, C, None, 1024, 1, 1 << 30, 1024)
    refused("tch_gated_act_bwd", None, BF16, A, 32, B, 32, C, None, 64, None, 0, 4, 4, 32)


@pytest.mark.parametrize("change", [
    dict(x=None), dict(dy=None), dict(dw=None), dict(K=60), dict(N=4), dict(M=-1), dict(K=1 << 21), dict(M=1 << 31), dict(x=ODD), dict(dy=ODD), dict(dw=ODD),
    dict(dbias=ODD), dict(x_low=ODD), dict(dy_low=D, x_low=D)], ids=str)
def test_weight_gradient(change):
    a = dict(x=A, x_low=None, dy=B, dy_low=None, dw=C, dbias=None, M=64, K=64, N=64)
    a.update(change)
    refused("tch_linear_wgrad", None, a["x"], a["x_low"], a["dy"], a["dy_low"], a["dw"], a["dbias"], 0, a["M"], a["K"], a["N"], None, 0)


def test_weight_gradient_workspace():
    from sirius_amd._lib import lib
    need = lib().tch_linear_wgrad_workspace_bytes(8192, 1024, 4096)
    assert need > 0 and lib().tch_linear_wgrad_workspace_bytes(0, 64, 64) == 0
    assert "workspace" in refused("tch_linear_wgrad", None, A, None, B, C, D, None, 0, 8192, 1024, 4096, A, need // 4)


def test_gradient_norm():
    refused("tch_grad_norm", None, None, 1, 4, -1.0, A, None, B)
    refused("tch_grad_norm", None, A, 1, 4, -1.0, None, None, B)
    refused("tch_grad_norm", None, A, 1, 4, -1.0, B, None, None)
    refused("tch_grad_norm", None, A, -1, 4, -1.0, B, None, C)
    refused("tch_grad_norm", None, A, 1, 4, -1.0, B, C, D)                  # a coefficient of a negative limit
    refused("tch_grad_norm", None, A, 1, 4, float("nan"), B, C, D)
    refused("tch_clip_grad_norm", None, A, 1, 4, 4, -0.5, B, C)
    refused("tch_clip_grad_norm", None, A, 1, 4, 4, float("nan"), B, C)
    refused("tch_clip_grad_norm", None, A, 1, 4, 4, 1.0, B, ctypes.c_void_p(0x10004))
    refused("tch_adamw_step_scaled", None, A, A, A, A, None, 4, 0.1, 0.9, 0.99, 1e-8, 0.0, B, C, None)
    refused("tch_sgd_momentum_step_scaled", None, A, A, A, None, 4, 0.1, 0.9, 0.0, None)


def test_outputs_that_overlap():
    def at(byte):
        return ctypes.c_void_p(0x100000 + byte)
    assert "overlaps" in refused("tch_linear_fwd", *fwd(x=at(0), y=at(16), ldx=64, ldy=64))
    assert "overlaps" in refused("tch_linear_fwd", *fwd(y=at(0), ldy=96, res=at(32), ldr=96))
    assert "overlaps" in refused("tch_linear_fwd", *fwd(y=at(0), ldy=32, pre=at(0), ldp=32))
    assert "overlaps" in refused("tch_linear_fwd", *fwd(y=at(0), ldy=32, bias=at(64)))
    assert "overlaps" in refused("tch_linear_fwd", *fwd(w=at(0), y=at(32 * 64 * 2 - 16), ldy=32))
    assert "overlaps" in refused("tch_linear_dgrad_gated", None, BF16, A, 64, B, at(0), 64, at(0), at(0), 64, None, None, 0, 4, 4, 64, 32)
    assert "overlaps" in refused("tch_act_bwd", None, BF16, at(0), 32, B, 32, at(64), None, 32, 1, 4, 32)
    assert "overlaps" in refused("tch_linear_wgrad", None, at(0), None, B, None, at(64 * 64 * 2 - 16), None, 0, 64, 64, 64, None, 0)
    assert "overlaps" in refused("tch_linear_wgrad", None, A, None, B, None, at(0), at(16), 0, 64, 64, 64, None, 0)
