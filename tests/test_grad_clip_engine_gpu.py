"""Gradient clipping and the fused MLP through the engines: an optimizer step with clipping is the step on gradients scaled by the
norm's coefficient, bit for bit; the fused MLP's loss and gradients are the oracle's within the bounds of the unfused engine."""
import math

import pytest
import torch

from oracle import gpt2 as G
from test_gpt2_gpu import CFG, T, _engine, _ids, _rel, _state

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("optimizer", ["adamw", "sgd"])
@pytest.mark.parametrize("use_global", [False, True], ids=["own", "accumulated"])
def test_clipped_step(optimizer, use_global):
    sd, limit = _state(3), 0.05
    hp = dict(lr=1e-2, weight_decay=0.01)

    def engine():
        eng = _engine(torch.bfloat16, optimizer=optimizer, **hp)
        eng.load_state_dict(sd)
        return eng
    clipped, plain = engine(), engine()
    assert math.isnan(clipped.last_grad_norm())
    clipped.set_grad_clip(limit)
    for step in range(3):
        for eng in (clipped, plain):
            eng.forward_backward(_ids(2, 20 + step).cuda())
            if use_global:
                eng.accumulate()
        plain.synchronize()
        grads = plain.global_grads if use_global else plain.grads
        norm = math.sqrt(float((grads.double() ** 2).sum()))
        coef = min(1.0, limit / (norm + 1e-6))
        assert coef < 1.0
        # the coefficient as the kernel rounds it: the norm in fp64, the quotient once to fp32
        grads *= torch.tensor(coef, dtype=torch.float64).to(torch.float32).cuda()
        torch.cuda.synchronize()
        for eng in (clipped, plain):
            eng.optimizer_step(use_global=use_global)
        assert abs(clipped.last_grad_norm() - norm) <= 2.0 ** -23 * norm
        a, b = clipped.state_dict(), plain.state_dict()
        for k in a:
            assert torch.equal(a[k], b[k]), (step, k)
    # a limit above the norm changes nothing; without a limit there is no norm
    clipped.set_grad_clip(1e9)
    for eng in (clipped, plain):
        eng.forward_backward(_ids(2, 40).cuda())
        if use_global:
            eng.accumulate()
        eng.optimizer_step(use_global=use_global)
    a, b = clipped.state_dict(), plain.state_dict()
    assert all(torch.equal(a[k], b[k]) for k in a) and clipped.last_grad_norm() > 0
    clipped.set_grad_clip(None)
    clipped.forward_backward(_ids(2, 41).cuda())
    clipped.optimizer_step()
    assert math.isnan(clipped.last_grad_norm())
    with pytest.raises(ValueError):
        clipped.set_grad_clip(-1.0)
    with pytest.raises(ValueError):
        clipped.set_grad_clip(float("nan"))


@pytest.mark.parametrize("name", ["resnet", "swin"])
def test_other_engines_clip(name):
    """After a clipped step the weights are those of a step on gradients scaled ahead."""
    if name == "resnet":
        from oracle import resnet as R
        from sirius_amd.resnet import ResNetEngine
        model = R.make_model((1, 1, 1, 1), 16, 16, seed=0)
        x, y = R.make_batch(4, 64, 16, seed=0)

        def engine():
            eng = ResNetEngine((1, 1, 1, 1), 16, 16, dtype=torch.float32, image_size=64)
            eng.load_state_dict(model.state_dict())
            return eng
    else:
        from test_swin_gpu import CFGS
        from sirius_amd.swin import SwinEngine
        cfg = CFGS["shifted"]
        g = torch.Generator().manual_seed(0)
        x, y = torch.randn(2, 3, cfg["image"], cfg["image"], generator=g), torch.randint(0, cfg["classes"], (2,), generator=g)

        def engine():
            eng = SwinEngine(embed=cfg["embed"], depths=cfg["depths"], heads=cfg["heads"], window=cfg["window"], patch=cfg["patch"],
                             image_size=cfg["image"], num_classes=cfg["classes"], dtype=torch.float32)
            eng.init_normal(0)
            return eng
    clipped, plain = engine(), engine()
    clipped.set_grad_clip(1e-3)
    for eng in (clipped, plain):
        eng.forward_backward(x.cuda(), y.cuda())
        eng.synchronize()
    plain.grads.copy_(clipped.grads)
    norm = math.sqrt(float((plain.grads.double() ** 2).sum()))
    plain.grads *= torch.tensor(min(1.0, 1e-3 / (norm + 1e-6)), dtype=torch.float64).to(torch.float32).cuda()
    torch.cuda.synchronize()
    for eng in (clipped, plain):
        eng.optimizer_step()
    assert abs(clipped.last_grad_norm() - norm) <= 2.0 ** -23 * norm and torch.equal(clipped.params, plain.params)


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-3), (torch.bfloat16, 2e-2)])
@pytest.mark.parametrize("B", [1, 3])
def test_fused_mlp(dtype, tol, B):
    sd = _state()
    if dtype == torch.bfloat16:
        sd = {k: v.to(torch.bfloat16).float() for k, v in sd.items()}
    ids = _ids(B, 1)
    loss_ref, grads_ref = G.loss_and_grads(sd, ids, CFG["n_head"], CFG["n_layer"], loss_scale=0.5)
    eng = _engine(dtype, fused_mlp=True)
    eng.load_state_dict(sd)
    for _ in range(2):    # the recorded program, replayed
        p, cut = eng.forward_backward(ids.cuda(), loss_scale=0.5)
        assert not cut
        assert abs(eng.last_loss() - loss_ref.item()) <= tol * abs(loss_ref.item())
        logits_ref = G.forward(sd, ids, CFG["n_head"], CFG["n_layer"]).reshape(B * T, -1)
        assert _rel(p.logits[:, :CFG["vocab"]].cpu(), logits_ref) <= tol
        grads = eng.grads_dict()
        for k, ref in grads_ref.items():
            assert _rel(grads[k], ref) <= tol, (k, _rel(grads[k], ref))
