"""A transformer block's training step of the operators as they are used together: boundary norms that keep their outputs in 8 bits,
a packed projection whose queries and keys are rotated in place, fused attention, a gated feed-forward layer whose pre-activations are
kept in 8 bits, and the way back, recorded once and replayed over new values; against autograd of the formulas in 64 bits, where weight
gradients and derivatives take what the step kept.

Tolerance: bf16, 2e-2 of the largest magnitude of the oracle's tensor, as for the training steps."""
import math

import pytest
import torch

from oracle import block_ops as O
from test_gpt2_kept_gpu import Kept

pytestmark = pytest.mark.gpu
H, D, F = 4, 64, 384
C = H * D


class KeptGated(torch.autograd.Function):
    """silu(g) u whose derivative is taken of what is kept of (g | u)"""

    @staticmethod
    def forward(ctx, pre, kept):
        ctx.save_for_backward(kept)
        g, u = pre.split(F, -1)
        return g * torch.sigmoid(g) * u

    @staticmethod
    def backward(ctx, dh):
        g, u = ctx.saved_tensors[0].split(F, -1)
        s = torch.sigmoid(g)
        return torch.cat([dh * u * s * (1 + g * (1 - s)), dh * g * s], -1), None


def new(gen, *shape, std=1.0, mean=0.0, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(mean, std, generator=gen)


class Step:
    def __init__(self, ctx, B, T, kind, fmt):
        from sirius_amd import ops
        self.ops, self.ctx, self.B, self.T, self.kind = ops, ctx, B, T, kind
        R = B * T
        gen = torch.Generator(device="cuda").manual_seed(0)
        e = lambda *s, dtype=torch.bfloat16: torch.empty(s, dtype=dtype, device="cuda")  # noqa: E731
        f32 = torch.float32
        self.w = dict(qkv=new(gen, 3 * C, C, std=C ** -0.5), o=new(gen, C, C, std=C ** -0.5), up=new(gen, 2 * F, C, std=C ** -0.5), down=new(gen, C, F, std=F ** -0.5))
        self.wt = {k: v.t().contiguous() for k, v in self.w.items()}
        vec = lambda m, *s: new(gen, *s, std=0.2, mean=m, dtype=f32)  # noqa: E731
        bias = kind == "layer"
        self.v = {k: vec(1.0, C) for k in ("w0", "w1", "w2", "pw1", "pw2")}
        self.v.update({k: vec(0.0, C) if bias else None for k in ("b0", "b1", "b2", "pb1", "pb2")})
        self.v["g1"], self.v["g2"] = vec(0.7, B, C), vec(0.7, C)      # a gate a sample, and one for all
        self.x, self.dy2, self.dt2 = e(R, C), e(R, C), e(R, C)
        self.freqs = ops.rotary_freqs(D, factor=2.0, trained=64).cuda()
        self.p0, self.p1, self.pp = ops.Packed8.empty(R, C, fmt), ops.Packed8.empty(R, C, fmt), ops.Packed8.empty(R, 2 * F, fmt)
        self.y0, self.o, self.a, self.t1, self.y1, self.f, self.t2, self.y2 = (e(R, C) for _ in range(8))
        self.qkv, self.lse, self.delta = e(R, 3 * C), e(B * H, T, dtype=f32), e(B * H, T, dtype=f32)
        self.pre, self.h = e(R, 2 * F), e(R, F)
        self.s0, self.s1, self.s2 = (e(R, 4, dtype=f32) for _ in range(3))
        self.dt1, self.df, self.dy1, self.dxa, self.da, self.do, self.dy0, self.dx = (e(R, C) for _ in range(8))
        self.dh, self.h2, self.dpre, self.dqkv = e(R, F), e(R, F), e(R, 2 * F), e(R, 3 * C)
        self.dw = {k: e(*v.shape, dtype=f32) for k, v in self.w.items()}
        self.dv = {k: None if v is None else e(*v.shape, dtype=f32) for k, v in self.v.items()}
        need = [ops.linear_bwd_workspace_bytes(self.h, C), ops.linear_bwd_workspace_bytes(self.o, C), ops.linear_wgrad_packed_workspace_bytes(self.p1, self.dpre),
                ops.linear_wgrad_packed_workspace_bytes(self.p0, self.dqkv), ops.residual_norm_bwd_workspace_bytes(self.x, gate=self.v["g1"])]
        self.ws = e(max(need), dtype=torch.uint8)

    def forward(self):
        o, c, v = self.ops, self.ctx, self.v
        o.residual_norm_fwd(c, self.x, None, None, self.y0, self.s0, kind=self.kind, weight=v["w0"], bias=v["b0"], packed=self.p0)
        o.linear_fwd(c, self.y0, self.w["qkv"], self.qkv)
        both = self.qkv.view(self.B, self.T, 3 * C)[..., :2 * C]
        o.rotary_fwd(c, both, both, self.freqs, D)
        flat, rs = self.qkv.view(-1), (3 * C, self.T * 3 * C)
        o.flash_attn_fwd(c, flat, flat[C:], flat[2 * C:], self.o.view(-1), self.lse, self.B, H, self.T, rs, (C, self.T * C), D ** -0.5, any_length=True)
        o.linear_fwd(c, self.o, self.w["o"], self.a)
        o.residual_norm_fwd(c, self.x, self.a, self.t1, self.y1, self.s1, kind=self.kind, weight=v["w1"], bias=v["b1"], post_weight=v["pw1"], post_bias=v["pb1"],
                            gate=v["g1"], scale=0.8, packed=self.p1)
        o.gated_linear_fwd(c, self.y1, self.w["up"], self.h, pre=self.pre)
        o.pack8(c, self.pre, self.pp)
        o.linear_fwd(c, self.h, self.w["down"], self.f)
        o.residual_norm_fwd(c, self.t1, self.f, self.t2, self.y2, self.s2, kind=self.kind, weight=v["w2"], bias=v["b2"], post_weight=v["pw2"], post_bias=v["pb2"], gate=v["g2"])

    def backward(self):
        o, c, v, dv, ws = self.ops, self.ctx, self.v, self.dv, self.ws
        o.residual_norm_bwd(c, self.dy2, self.dt2, self.t2, self.f, self.dt1, self.df, self.s2, kind=self.kind, weight=v["w2"], post_weight=v["pw2"],
                            post_bias=v["pb2"], gate=v["g2"], dweight=dv["w2"], dbias=dv["b2"], dpost_weight=dv["pw2"], dpost_bias=dv["pb2"], dgate=dv["g2"], workspace=ws)
        o.linear_dgrad(c, self.df, self.wt["down"], self.dh)
        o.gated_act_bwd_packed(c, self.dh, self.pp, self.dpre, h=self.h2)
        o.linear_wgrad(c, self.h2, self.df, self.dw["down"], workspace=ws)
        o.linear_wgrad_packed(c, self.p1, self.dpre, self.dw["up"], workspace=ws)
        o.linear_dgrad(c, self.dpre, self.wt["up"], self.dy1)
        o.residual_norm_bwd(c, self.dy1, self.dt1, self.t1, self.a, self.dxa, self.da, self.s1, kind=self.kind, weight=v["w1"], post_weight=v["pw1"],
                            post_bias=v["pb1"], gate=v["g1"], scale=0.8, dweight=dv["w1"], dbias=dv["b1"], dpost_weight=dv["pw1"], dpost_bias=dv["pb1"], dgate=dv["g1"], workspace=ws)
        o.linear_wgrad(c, self.o, self.da, self.dw["o"], workspace=ws)
        o.linear_dgrad(c, self.da, self.wt["o"], self.do)
        flat, g, rs = self.qkv.view(-1), self.dqkv.view(-1), (3 * C, self.T * 3 * C)
        o.flash_attn_bwd(c, flat, flat[C:], flat[2 * C:], self.o.view(-1), self.do.view(-1), self.lse, self.delta, g, g[C:], g[2 * C:], self.B, H, self.T, rs,
                         (C, self.T * C), D ** -0.5, any_length=True)
        both = self.dqkv.view(self.B, self.T, 3 * C)[..., :2 * C]
        o.rotary_bwd(c, both, both, self.freqs, D)
        o.linear_wgrad_packed(c, self.p0, self.dqkv, self.dw["qkv"], workspace=ws)
        o.linear_dgrad(c, self.dqkv, self.wt["qkv"], self.dy0)
        o.residual_norm_bwd(c, self.dy0, self.dxa, self.x, None, self.dx, None, self.s0, kind=self.kind, weight=v["w0"], dweight=dv["w0"], dbias=dv["b0"], workspace=ws)

    def fill(self, seed):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.x.copy_(new(gen, *self.x.shape)), self.dy2.copy_(new(gen, *self.x.shape)), self.dt2.copy_(new(gen, *self.x.shape))
        self.ws.fill_(255)

    def results(self):
        out = dict(y2=self.y2, t2=self.t2, dx=self.dx)
        out.update({"d" + k: t for k, t in self.dw.items()})
        out.update({"d" + k: t for k, t in self.dv.items() if t is not None})
        return {k: t.clone() for k, t in out.items()}

    def fetched(self, packed):
        x = torch.empty(packed.shape, device="cuda")
        self.ops.unpack8(self.ctx, packed, x)
        return x.double()

    def oracle(self):
        w = {k: t.double().requires_grad_(True) for k, t in self.w.items()}
        v = {k: None if t is None else t.double().requires_grad_(True) for k, t in self.v.items()}
        x = self.x.double().requires_grad_(True)
        B, T, R = self.B, self.T, self.B * self.T
        linear = lambda t, kept, name: Kept.apply(t, kept, w[name].t(), 0.0 * w[name][:, 0])  # noqa: E731
        norm = lambda t, i: O.norm(t, self.kind, v["w%d" % i], v["b%d" % i])[0]  # noqa: E731
        qkv = linear(norm(x, 0), self.fetched(self.p0), "qkv").view(B, T, 3, H, D)
        turn = torch.polar(torch.ones(T, D // 2, dtype=torch.float64, device="cuda"), torch.arange(T, device="cuda").double()[:, None] * self.freqs)

        def rotated(t):
            z = torch.complex(t[..., :D // 2], t[..., D // 2:]) * turn[None, :, None]
            return torch.cat([z.real, z.imag], -1)
        q, k, val = (t.transpose(1, 2) for t in (rotated(qkv[:, :, 0]), rotated(qkv[:, :, 1]), qkv[:, :, 2]))
        scores = (q @ k.transpose(-1, -2)) * D ** -0.5
        causal = torch.ones(T, T, dtype=torch.bool, device="cuda").tril()
        att = torch.softmax(scores.masked_fill(~causal, -math.inf), -1) @ val
        o = att.transpose(1, 2).reshape(R, C)
        a = linear(o, o.detach(), "o")
        t1 = O.boundary(x, a, self.kind, v["pw1"], v["pb1"], v["g1"], 0.8)[0]
        pre = linear(norm(t1, 1), self.fetched(self.p1), "up")
        kept = self.fetched(self.pp)
        h = KeptGated.apply(pre, kept)
        g, u = kept.split(F, -1)
        f = linear(h, g * torch.sigmoid(g) * u, "down")
        t2 = O.boundary(t1, f, self.kind, v["pw2"], v["pb2"], v["g2"])[0]
        y2 = norm(t2, 2)
        torch.autograd.backward([y2, t2], [self.dy2.double(), self.dt2.double()])
        out = dict(y2=y2.detach(), t2=t2.detach(), dx=x.grad)
        out.update({"d" + n: t.grad for n, t in w.items()})
        out.update({"d" + n: t.grad for n, t in v.items() if t is not None})
        return out


@pytest.mark.parametrize("kind,fmt,B,T", [("rms", "e4m3", 2, 128), ("layer", "int8", 3, 77), ("rms", "int8", 1, 1), ("layer", "e4m3", 2, 300)], ids=str)
def test_a_block_forward_and_back(kind, fmt, B, T):
    from sirius_amd import ops
    step = Step(ops.Context(), B, T, kind, fmt)
    prog = ops.Program()
    step.fill(1)
    step.ctx.begin_record(prog)
    step.forward()
    step.backward()
    step.ctx.end_record()
    for seed in (1, 2, 3):
        step.fill(seed)
        step.ctx.run(prog)
        step.ctx.synchronize()
        got = step.results()
        step.ws.fill_(1)
        step.forward()      # eager, between the replays
        step.backward()
        step.ctx.synchronize()
        for k, t in step.results().items():
            assert torch.equal(got[k], t), (seed, k)
        for k, ref in step.oracle().items():
            off = (got[k].double().view_as(ref) - ref).abs().max().item() / (ref.abs().max().item() + 1e-12)
            assert off <= 2e-2, (seed, k, off)
