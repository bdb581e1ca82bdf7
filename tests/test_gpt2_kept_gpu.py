"""GPT-2's step with the projections' inputs and the MLP's pre-activations kept in 8 bits, against a CPU oracle in 64 bits: the forward
pass is that of oracle/gpt2.py, the weight gradients are those of what the step kept, GELU's derivative is taken of what it kept, and the
MLP's hidden values are computed from that again.  (What is kept of an activation next to the middle between two 8-bit numbers is the one
or the other by its last bits: the oracle takes the step's own numbers, and checks that they are next to its activations.)

Tolerances: fp32 rtol 1e-3, bf16 rtol 2e-2 of the largest magnitude of the oracle's tensor, as for the step that keeps everything."""
import math

import pytest
import torch
import torch.nn.functional as F

from oracle import block_ops as O
from oracle import gpt2 as G

pytestmark = pytest.mark.gpu


class Kept(torch.autograd.Function):
    """x w + b whose weight gradient is taken of `kept`"""

    @staticmethod
    def forward(ctx, x, kept, w, b):
        ctx.save_for_backward(kept, w)
        return x @ w + b

    @staticmethod
    def backward(ctx, dy):
        kept, w = ctx.saved_tensors
        return dy @ w.t(), None, kept.reshape(-1, kept.shape[-1]).t() @ dy.reshape(-1, dy.shape[-1]), dy.reshape(-1, dy.shape[-1]).sum(0)


class KeptGelu(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, kept):
        ctx.save_for_backward(kept)
        return F.gelu(z, approximate="tanh")

    @staticmethod
    def backward(ctx, dy):
        kept, = ctx.saved_tensors
        with torch.enable_grad():
            z = kept.clone().requires_grad_(True)
            return dy * torch.autograd.grad(F.gelu(z, approximate="tanh").sum(), z)[0], None


def loss_and_grads(sd, ids, n_head, n_layer, fmt, loss_scale, held, tol):
    """held: what the step kept, per layer"""
    sd = {k: v.detach().double().requires_grad_(True) for k, v in sd.items()}
    held = iter([t for layer in held for t in layer])

    def keep(x):
        kept = next(held).view_as(x)
        best, codes = O.packed(x.detach().reshape(-1, x.shape[-1]), fmt)
        # a step at most beside what the definition keeps of this activation (of a group's whole range in fp8, 448 / 8), and the
        # activation's own error; a group whose largest number is at the edge may have the next power of two
        unit = 2 * O.two_to(codes.long() - 127).repeat_interleave(32, 1)[:, :x.shape[-1]].reshape(x.shape)
        step = unit if fmt == "int8" else torch.maximum(x.detach().abs() / 8, unit * 2.0 ** -9) * 1.25
        assert ((kept - best.view_as(x)).abs() <= step + tol * x.detach().abs().max()).all()
        return kept
    B, T = ids.shape
    wte = sd["transformer.wte.weight"]
    C = wte.shape[1]
    D = C // n_head
    h = F.embedding(ids, wte) + sd["transformer.wpe.weight"][:T].unsqueeze(0)
    causal = torch.tril(torch.ones(T, T, dtype=torch.bool))
    for i in range(n_layer):
        p = f"transformer.h.{i}."
        linear = lambda x, kept, name: Kept.apply(x, kept, sd[p + name + ".weight"], sd[p + name + ".bias"])  # noqa: E731
        a = F.layer_norm(h, (C,), sd[p + "ln_1.weight"], sd[p + "ln_1.bias"], 1e-5)
        q, k, v = (t.view(B, T, n_head, D).transpose(1, 2) for t in linear(a, keep(a), "attn.c_attn").split(C, dim=2))
        att = torch.softmax(((q @ k.transpose(-1, -2)) / math.sqrt(D)).masked_fill(~causal, float("-inf")), dim=-1)
        o = (att @ v).transpose(1, 2).reshape(B, T, C)
        h = h + linear(o, o.detach(), "attn.c_proj")
        m = F.layer_norm(h, (C,), sd[p + "ln_2.weight"], sd[p + "ln_2.bias"], 1e-5)
        z = linear(m, keep(m), "mlp.c_fc")
        kept_z = keep(z)
        f = KeptGelu.apply(z, kept_z)
        h = h + linear(f, F.gelu(kept_z, approximate="tanh"), "mlp.c_proj")
    h = F.layer_norm(h, (C,), sd["transformer.ln_f.weight"], sd["transformer.ln_f.bias"], 1e-5)
    loss = G.loss_of(h @ wte.t(), ids)
    (loss * loss_scale).backward()
    return loss.detach().item(), {k: v.grad for k, v in sd.items()}


def state(cfg, seed=0):
    sd = G.make_state_dict(cfg["vocab"], cfg["n_pos"], cfg["n_embd"], cfg["n_layer"], seed=seed)
    g = torch.Generator()
    g.manual_seed(seed + 100)
    for v in sd.values():
        if v.dim() == 1:
            v.add_(torch.randn(v.shape, generator=g) * 0.1)
    return {k: v.to(torch.bfloat16).float() for k, v in sd.items()}


def tokens(cfg, B, T, seed=1):
    g = torch.Generator()
    g.manual_seed(seed)
    return torch.randint(0, cfg["vocab"], (B, T), generator=g)


SMALL = dict(vocab=97, n_pos=40, n_embd=64, n_layer=2, n_head=4)
DEEP = dict(vocab=200, n_pos=128, n_embd=128, n_layer=5, n_head=2)     # heads of 64: fused attention in bf16; five layers through three sets


def run(cfg, T, dtype, sd, ids, **kw):
    from sirius_amd.gpt2 import GPT2Engine
    eng = GPT2Engine(seq_len=T, dtype=dtype, **cfg, **kw)
    eng.load_state_dict(sd)
    plan, cut = eng.forward_backward(ids.cuda(), loss_scale=0.5)
    assert not cut
    return eng, eng.last_loss(), eng.grads_dict()


def fetched(eng):
    """What the step kept, in 64 bits on the CPU."""
    from sirius_amd import ops
    eng.synchronize()
    out = []
    for layer in eng._last_plan.kept:
        out.append([])
        for packed in layer:
            x = torch.empty(packed.shape, device="cuda")
            ops.unpack8(eng.ctx, packed, x)
            eng.synchronize()
            out[-1].append(x.double().cpu())
    return out


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-3), (torch.bfloat16, 2e-2)], ids=["f32", "bf16"])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("cfg,T,B", [(SMALL, 32, 1), (SMALL, 32, 3), (DEEP, 128, 2)], ids=["small1", "small3", "deep"])
def test_loss_and_gradients(dtype, tol, fmt, cfg, T, B):
    print("case", dtype, fmt, T, B, flush=True)
    sd, ids = state(cfg), tokens(cfg, B, T)
    eng, loss, grads = run(cfg, T, dtype, sd, ids, kept=fmt)
    want, ref = loss_and_grads(sd, ids, cfg["n_head"], cfg["n_layer"], fmt, 0.5, fetched(eng), tol)
    assert abs(loss - want) <= tol * abs(want)
    for k, r in ref.items():
        off = (grads[k].double() - r).abs().max().item() / (r.abs().max().item() + 1e-12)
        assert off <= tol, (k, off)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_lanes_change_no_bit(dtype):
    """Weight gradients beside the data gradients, a layer behind them, or in line: the same bits, step after step."""
    sd = state(DEEP)
    results = []
    for kw in (dict(), dict(overlap_wgrad=False), dict(trailing_wgrad=False), dict(trailing_reduce=False)):
        eng, loss, grads = run(DEEP, 128, dtype, sd, tokens(DEEP, 2, 128), kept="int8", **kw)
        for step in range(3):
            eng.forward_backward(tokens(DEEP, 2, 128, seed=step).cuda())
            eng.optimizer_step()
        results.append((loss, grads, eng.state_dict()))
    for loss, grads, sd2 in results[1:]:
        assert loss == results[0][0]
        for k in grads:
            assert torch.equal(grads[k], results[0][1][k]), k
            assert torch.equal(sd2[k], results[0][2][k]), k


def test_what_a_plan_holds():
    """18 C bytes a token and layer instead of 32 C in bf16; what the layers share does not grow with them."""
    from sirius_amd.gpt2 import GPT2Engine
    cfg, T, B = dict(vocab=97, n_pos=128, n_embd=256, n_head=4), 128, 4
    size = {}
    for layers in (4, 8):
        for kept in ("full", "int8"):
            eng = GPT2Engine(seq_len=T, n_layer=layers, kept=kept, **cfg)
            size[layers, kept] = eng.plan(B).bytes
    a_layer = {k: (size[8, k] - size[4, k]) / 4 / (B * T * cfg["n_embd"]) for k in ("full", "int8")}
    assert 32 <= a_layer["full"] <= 32.2 and 18 <= a_layer["int8"] <= 18.6, a_layer
    assert size[8, "int8"] < size[8, "full"]


def test_refusals():
    from sirius_amd.gpt2 import GPT2Engine
    with pytest.raises(ValueError, match="kept"):
        GPT2Engine(seq_len=32, kept="int4", **SMALL)
    with pytest.raises(ValueError, match="fused_mlp"):
        GPT2Engine(seq_len=32, kept="int8", fused_mlp=True, **SMALL)


def test_a_step_on_other_batches_and_clipping():
    """Another batch size takes another plan; the clip, the optimizer and the released activations work as with everything kept."""
    sd = state(SMALL)
    eng, _, _ = run(SMALL, 32, torch.bfloat16, sd, tokens(SMALL, 2, 32), kept="int8")
    eng.set_grad_clip(1.0)
    for B in (3, 1, 3):
        eng.forward_backward(tokens(SMALL, B, 32, seed=B).cuda())
        eng.optimizer_step()
        assert math.isfinite(eng.last_loss()) and math.isfinite(eng.last_grad_norm())
    assert eng.release_activations() > 0
    eng.forward_backward(tokens(SMALL, 2, 32).cuda())
    assert math.isfinite(eng.last_loss())


from test_colocate_gpu import clean_runtime  # noqa: E402,F401


def test_handover_with_8_bits_kept(clean_runtime, monkeypatch, tmp_path):  # noqa: F811
    """The train script under the colocation protocol with the activations in the shared pool: the peer asks for memory, a micro-batch is
    killed between its launches and trained again, and every sequence counts once."""
    from sirius_amd.train import gpt2 as script
    env = {"COLTRAIN_MODE": "colocate-l1", "COLTRAIN_HOOK_MODE": "xsched-sync", "COLTRAIN_USE_XSCHED": "1", "COLTRAIN_HAS_INFER_SERVER": "1",
           "COLTRAIN_USE_SHARED_TENSOR": "1", "COLTRAIN_SHARED_TENSOR_POOL_GB": "2", "COLTRAIN_PROFILE_LOG_PATH": str(tmp_path / "train-profile.csv")}
    for k, v in env.items():
        monkeypatch.setenv(k, v)
    peer = script.PeerScript({3: ("l1", 2), 10: ("exit", 8)}, delay_ms=1.0)
    try:
        out = script.train(1, 8, dataset_size=8 * 8, seq_len=64, dtype=torch.bfloat16, optimizer="adamw", peer=peer, num_distinct_samples=16,
                           n_embd=64, n_layer=2, n_head=4, n_pos=64, kept="int8")
    finally:
        peer.stop()
    assert out["trainer"].get_last_epoch_stat().finished_sample == 8 * 8
    assert [k for _, k, _ in peer.sent] == ["l1", "exit"]
    assert all(torch.isfinite(v).all() for v in out["model"].state_dict().values())
