"""What an engine's gradient norm counts, and what it says of a step whose launches were rejected."""
import math

import pytest
import torch

from test_gpt2_gpu import _engine, _ids, _state

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["gpt2", "resnet", "swin"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_the_norm_is_over_the_parameters(name, dtype):
    """The flat buffer has room between the parameters and rows that stand for no class or channel: none of it counts.  Every
    gradient of the state dict does, in fp64: off by the sum's roundings and the norm's own, 2^-23 as in test_grad_norm_gpu.py."""
    if name == "gpt2":
        eng = _engine(dtype, optimizer="adamw")
        eng.load_state_dict(_state(3))
        inputs = (_ids(2, 20).cuda(),)
    elif name == "resnet":
        from oracle import resnet as R
        from sirius_amd.resnet import ResNetEngine
        eng = ResNetEngine((1, 1, 1, 1), 16, 16, dtype=dtype, image_size=64)
        eng.load_state_dict(R.make_model((1, 1, 1, 1), 16, 16, seed=0).state_dict())
        inputs = tuple(t.cuda() for t in R.make_batch(4, 64, 16, seed=0))
    else:
        from test_swin_gpu import CFGS
        from sirius_amd.swin import SwinEngine
        cfg = CFGS["shifted"]
        eng = SwinEngine(embed=cfg["embed"], depths=cfg["depths"], heads=cfg["heads"], window=cfg["window"], patch=cfg["patch"],
                         image_size=cfg["image"], num_classes=cfg["classes"], dtype=dtype)
        eng.init_normal(0)
        g = torch.Generator().manual_seed(0)
        inputs = (torch.randn(2, 3, cfg["image"], cfg["image"], generator=g).cuda(), torch.randint(0, cfg["classes"], (2,), generator=g).cuda())
    eng.set_grad_clip(1.0)
    for _ in range(2):
        eng.forward_backward(*inputs)
        eng.synchronize()
        norm = math.sqrt(math.fsum(float((t.double() ** 2).sum()) for t in eng.grads_dict().values()))
        eng.optimizer_step()
        assert norm > 0 and abs(eng.last_grad_norm() - norm) <= 2.0 ** -23 * norm


def test_a_rejected_step_has_no_norm():
    """A step whose launches were rejected consumed nothing: the norm stays that of the step before."""
    from sirius_amd._lib import lib
    eng = _engine(torch.bfloat16, optimizer="adamw")
    eng.load_state_dict(_state(3))
    eng.set_grad_clip(1.0)
    eng.forward_backward(_ids(2, 20).cuda())
    eng.synchronize()
    lib().tch_SetRejectCudaCalls(1)
    try:
        assert eng.optimizer_step()
    finally:
        lib().tch_SetRejectCudaCalls(0)
    assert math.isnan(eng.last_grad_norm())
    assert not eng.optimizer_step()
    norm = eng.last_grad_norm()
    assert norm > 0
    for use_global in (False, True):
        eng.forward_backward(_ids(2, 21).cuda())
        if use_global:
            eng.accumulate()
        lib().tch_SetRejectCudaCalls(1)
        try:
            assert eng.optimizer_step(use_global=use_global)
        finally:
            lib().tch_SetRejectCudaCalls(0)
        assert eng.last_grad_norm() == norm
