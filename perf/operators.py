"""The feed-forward operators and the gradient clip, case by case: linear layers with bias, activation and residual in one
launch, gated feed-forward layers, their backward passes, and the global gradient norm with clipping.

``own = False`` computes every case in elementary torch operations in 32 bits, rounded once at the end; ``own = True`` makes the
calls of this package.  As the training engines do, a program records its calls once, on buffers that it keeps, and a pass
replays them.
"""
import math
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f32": 4}
ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu")


def _sizes(case):
    """Element counts of a clip case's tensors: those of GPT-2 small's 148 parameters (the configuration that this repository
    trains; a projection and its transpose count alike), or `count` numbers up to `largest`, evenly over the logarithm."""
    if case["tensors"] == "gpt2":
        C, out = 768, [50257 * 768, 1024 * 768]
        for _ in range(12):
            out += [C, C, 3 * C * C, 3 * C, C * C, C, C, C, 4 * C * C, 4 * C, 4 * C * C, C]
        return out + [C, C]
    rng, left, out = random.Random(case["layout"]), 150_000_000, []
    for _ in range(case["count"]):
        n = min(_log(rng, 1, case["largest"]), max(left, 1))
        out.append(n)
        left -= n
    return out


def listed():
    return [
        # one token of a server: the weights are read once for a single row, latency is what counts
        dict(name="linear_fwd_token", op="linear_fwd", dtype="bf16", rows=1, cin=4096, cout=4096, act="gelu_tanh", bias=True,
             residual=False, pre=False),
        # a ragged evaluation batch: no size is a multiple of a tile, the block's residual added
        dict(name="linear_fwd_ragged", op="linear_fwd", dtype="bf16", rows=777, cin=1000, cout=2056, act="silu", bias=True,
             residual=True, pre=False),
        # the first MLP layer of a training step, 8 sequences of 1024 tokens; the pre-activation is kept for the backward pass
        dict(name="linear_fwd_train", op="linear_fwd", dtype="bf16", rows=8192, cin=1024, cout=4096, act="gelu_tanh", bias=True,
             residual=False, pre=True),
        # Swin-B's last stage in fp32, 32 images of 49 tokens
        dict(name="linear_fwd_f32", op="linear_fwd", dtype="f32", rows=1568, cin=1024, cout=4096, act="gelu", bias=True,
             residual=False, pre=True),
        # the gradients of linear_fwd_train's layer
        dict(name="linear_bwd_train", op="linear_bwd", dtype="bf16", rows=8192, cin=1024, cout=4096, act="gelu_tanh"),
        # Swin-B's third stage in fp32, two images of 196 tokens
        dict(name="linear_bwd_f32", op="linear_bwd", dtype="f32", rows=392, cin=512, cout=2048, act="gelu"),
        # seven sequences that decode together
        dict(name="gated_fwd_tokens", op="gated_fwd", dtype="bf16", rows=7, cin=2048, cout=5632, act="silu", bias=False,
             pre=False),
        # a long prompt or a large evaluation batch through a wide model: the largest product
        dict(name="gated_fwd_large", op="gated_fwd", dtype="bf16", rows=16384, cin=4096, cout=11008, act="silu", bias=False,
             pre=False),
        # a small training batch with odd sizes, biases too
        dict(name="gated_bwd_ragged", op="gated_bwd", dtype="bf16", rows=1023, cin=1024, cout=2736, act="silu"),
        # the whole feed-forward block of a training step, from the gradient behind its down projection
        dict(name="block_bwd_train", op="block_bwd", dtype="bf16", rows=8192, cin=2048, cout=5632, act="silu"),
        # a small model's or an adapter's gradients: many short tensors, latency is what counts
        dict(name="clip_short", op="clip", dtype="f32", tensors="drawn", count=48, largest=12288, layout=1),
        # all gradients of GPT-2 small, ahead of the optimizer step
        dict(name="clip_gpt2", op="clip", dtype="f32", tensors="gpt2"),
    ]


def _log(rng, low, high, step=1):
    """Between low and high, evenly over the logarithm, a multiple of step."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(low, min(high, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(["linear_fwd", "linear_fwd", "linear_bwd", "gated_fwd", "gated_fwd", "gated_bwd", "block_bwd", "clip"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op == "clip":
        return dict(op=op, dtype=dtype, tensors="drawn", count=_log(rng, 1, 400), largest=_log(rng, 1000, 40_000_000),
                    layout=rng.randrange(1 << 30))
    step = 8 if dtype == "bf16" else 4
    while True:
        case = dict(op=op, dtype=dtype, rows=_log(rng, 1 if op.endswith("fwd") else 8, 16384), cin=_log(rng, 64, 8192, step),
                    cout=_log(rng, 64, 11008, step), act=rng.choice(ACTS))
        if op.endswith("fwd"):
            case["bias"], case["pre"] = rng.random() < 0.5, rng.random() < 0.5
        if op == "linear_fwd":
            case["residual"] = rng.random() < 0.5
        # no dearer than the largest listed case; fp32 products take about ten times as long
        if work(case)["flops"] <= (2.5e12 if dtype == "bf16" else 2.0e11):
            return case


def work(case):
    op, e = case["op"], _SIZE[case["dtype"]]
    if op == "clip":
        n = sum(_sizes(case))
        return {"bytes": 2 * e * n + 4, "flops": 4 * n}
    M, K, N = case["rows"], case["cin"], case["cout"]
    if op == "linear_fwd":
        return {"bytes": e * (M * K + N * K + M * N * (1 + case["residual"] + case["pre"])) + 4 * N * case["bias"],
                "flops": 2 * M * N * K}
    if op == "linear_bwd":
        return {"bytes": e * (2 * M * N + 2 * M * K + N * K) + 4 * (N * K + N), "flops": 4 * M * N * K}
    if op == "gated_fwd":
        return {"bytes": e * (M * K + 2 * N * K + M * N * (1 + 2 * case["pre"])) + 8 * N * case["bias"], "flops": 4 * M * N * K}
    if op == "gated_bwd":
        return {"bytes": e * (3 * M * N + 2 * M * K + 2 * N * K) + 8 * (N * K + N), "flops": 8 * M * N * K}
    return {"bytes": e * (2 * M * N + 3 * M * K + 3 * N * K) + 12 * N * K, "flops": 12 * M * N * K}   # block_bwd


def _views(case, dtype=None):
    """The tensors of a clip case inside one buffer of zeros, each from a multiple of eight elements on, as the engines keep
    their gradients; and the buffer."""
    sizes = _sizes(case)
    flat = torch.zeros(sum((n + 7) // 8 * 8 for n in sizes), dtype=dtype or _TYPES[case["dtype"]], device="cuda")
    views, at = [], 0
    for n in sizes:
        views.append(flat[at:at + n])
        at += (n + 7) // 8 * 8
    return views, flat


def _inputs(case, seed):
    """The tensors that both forms and the exact one start from."""
    dt = _TYPES[case["dtype"]]
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def normal(*shape, std=1.0, dtype=dt):
        return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=gen)
    op = case["op"]
    if op == "clip":
        # the layers of a model have gradients of different sizes; their norm together is far above the limit of 1
        grads, flat = _views(case)
        for i, g in enumerate(grads):
            g.normal_(0.0, 0.3 / (1 + i % 5), generator=gen)
        return dict(grads=grads, flat=flat)
    M, K, N = case["rows"], case["cin"], case["cout"]
    width = 1 if op.startswith("linear") else 2     # a gated layer has two projections, gate rows first
    s = dict(x=normal(M, K), w=normal(width * N, K, std=1 / math.sqrt(K)))
    if op.endswith("fwd"):
        s["bias"] = normal(width * N, std=0.3, dtype=torch.float32) if case["bias"] else None
        s["residual"] = normal(M, N) if case.get("residual") else None
    else:
        s["pre"] = normal(M, width * N)
        s["dy"] = normal(M, K if op == "block_bwd" else N, std=0.02)
        if op == "block_bwd":
            s["w_down"] = normal(K, N, std=1 / math.sqrt(N))
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        _record(s, case)
    return s


def _record(s, case):
    """What a program of this package keeps: a context, output buffers, the transposed weights that data gradients read, and
    the recorded calls."""
    from sirius_amd import ops
    op, act = case["op"], case.get("act")
    ctx = ops.Context()

    def new(*shape, dtype=_TYPES[case["dtype"]]):
        return torch.empty(shape, dtype=dtype, device="cuda")
    if op == "clip":
        out, flat = _views(case)
        norm = new(1, dtype=torch.float32)
        table = ops.GradTable(s["grads"], out=out)
        scratch = new(ops.grad_norm_workspace_bytes(table), dtype=torch.uint8)
        s["keep"], s["out"] = (table, scratch), [norm, flat]
        calls = [lambda: ops.clip_grad_norm(ctx, table, 1.0, norm, scratch)]
    else:
        M, K, N = case["rows"], case["cin"], case["cout"]
        if op.endswith("fwd"):
            y = new(M, N)
            pre = new(M, s["w"].shape[0]) if case["pre"] else None
            s["out"] = [y] if pre is None else [y, pre]
            if op == "linear_fwd":
                calls = [lambda: ops.linear_fwd(ctx, s["x"], s["w"], y, bias=s["bias"], act=act, residual=s["residual"], pre=pre)]
            else:
                calls = [lambda: ops.gated_linear_fwd(ctx, s["x"], s["w"], y, bias=s["bias"], act=act, pre=pre)]
        else:
            wide = s["w"].shape[0]
            wt = s["w"].t().contiguous()
            dx, dpre = new(M, K), new(M, wide)
            dw, db = new(wide, K, dtype=torch.float32), new(wide, dtype=torch.float32)
            # weight gradients are fp32: those of bf16 gradients take the gradients' low parts as well
            dpre_low = new(M, wide) if case["dtype"] == "bf16" else None
            scratch = new(ops.linear_bwd_workspace_bytes(s["x"], wide), dtype=torch.uint8)
            s["keep"], s["out"] = (wt, dpre, dpre_low, scratch), [dx, dw, db]
            if op == "linear_bwd":
                calls = [lambda: ops.linear_bwd(ctx, s["dy"], s["x"], wt, dx, dw, dbias=db, act=act, pre=s["pre"], dpre=dpre,
                                                workspace=scratch, dpre_low=dpre_low)]
            elif op == "gated_bwd":
                calls = [lambda: ops.gated_linear_bwd(ctx, s["dy"], s["x"], wt, dx, dw, s["pre"], dpre, dbias=db, act=act,
                                                      workspace=scratch, dpre_low=dpre_low)]
            else:
                wt_down = s["w_down"].t().contiguous()
                h, dw_down = new(M, N), new(K, N, dtype=torch.float32)
                h_low = new(M, N) if case["dtype"] == "bf16" else None
                scratch_down = new(ops.linear_bwd_workspace_bytes(h, K), dtype=torch.uint8)
                s["keep"], s["out"] = (wt, wt_down, dpre, dpre_low, h, h_low, scratch, scratch_down), [dx, dw, dw_down]
                calls = [lambda: ops.linear_dgrad_gated(ctx, s["dy"], wt_down, s["pre"], dpre, act=act, h=h, dpre_low=dpre_low,
                                                        h_low=h_low),
                         lambda: ops.linear_bwd(ctx, s["dy"], h, None, None, dw_down, workspace=scratch_down, x_low=h_low),
                         lambda: ops.linear_bwd(ctx, dpre, s["x"], wt, dx, dw, workspace=scratch, dy_low=dpre_low)]
    prog = ops.Program()
    ctx.begin_record(prog)
    try:
        for call in calls:
            call()
    finally:
        ctx.end_record()
    s["ctx"], s["prog"] = ctx, prog


def run(state):
    if own:
        state["ctx"].run(state["prog"])
        return state["out"]
    return _plain(state, state["case"])


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------

_TANH_A, _TANH_B = math.sqrt(2.0 / math.pi), 0.044715


def _act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(_TANH_A * (z + _TANH_B * z * z * z)))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    if act == "gelu_tanh":
        t = torch.tanh(_TANH_A * (z + _TANH_B * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * _TANH_A * (1.0 + 3.0 * _TANH_B * z * z)
    if act == "silu":
        sig = 1.0 / (1.0 + torch.exp(-z))
        return sig * (1.0 + z * (1.0 - sig))
    return torch.ones_like(z)


def _plain(s, case):
    op, dt, act = case["op"], _TYPES[case["dtype"]], case.get("act")
    if op == "clip":
        total = s["grads"][0].new_zeros((), dtype=torch.float64)
        for g in s["grads"]:
            g = g.double()
            total = total + (g * g).sum()
        norm = torch.sqrt(total)
        coef = torch.clamp(1.0 / (norm + 1e-6), max=1.0).float()
        out, flat = _views(case)
        for g, o in zip(s["grads"], out):
            o.copy_(g.float() * coef)
        return [norm.float().reshape(1), flat]
    x, w, N = s["x"].float(), s["w"].float(), case["cout"]
    if op.endswith("fwd"):
        z = x @ w.t()
        if s["bias"] is not None:
            z = z + s["bias"]
        if op == "linear_fwd":
            y = _act(z, act)
            if s["residual"] is not None:
                y = y + s["residual"].float()
        else:
            y = _act(z[:, :N], act) * z[:, N:]
        return [y.to(dt), z.to(dt)] if case["pre"] else [y.to(dt)]
    pre, dy = s["pre"].float(), s["dy"].float()
    if op == "linear_bwd":
        dpre = dy * _slope(pre, act)
    else:
        dh = dy @ s["w_down"].float() if op == "block_bwd" else dy
        g, u = pre[:, :N], pre[:, N:]
        value = _act(g, act)
        dpre = torch.cat([dh * u * _slope(g, act), dh * value], 1)
    dx, dw = dpre @ w, dpre.t() @ x
    if op == "block_bwd":
        return [dx.to(dt), dw, dy.t() @ (value * u)]
    return [dx.to(dt), dw, dpre.sum(0)]


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "clip":
        flat = s["flat"].double()       # the elements between two tensors are zeros
        norm = float(torch.linalg.vector_norm(flat))
        return [torch.full((1,), norm, dtype=torch.float64, device="cuda"), flat * min(1.0, 1.0 / (norm + 1e-6))]
    op, act, N = case["op"], case["act"], case["cout"]
    d = {k: v.double() if torch.is_tensor(v) else v for k, v in s.items()}

    def value(z):
        if act == "gelu":       # z times the normal distribution's integral, without cancellation on the left
            return z * 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
        if act == "gelu_tanh":
            return z * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z.pow(3)))
        return {"none": lambda: z, "relu": lambda: z.clamp(min=0), "silu": lambda: z * torch.sigmoid(z)}[act]()

    def derivative(z):
        z = z.clone().requires_grad_(True)
        return torch.autograd.grad(value(z).sum(), z)[0]
    if op.endswith("fwd"):
        pre = torch.matmul(d["x"], d["w"].t())
        if d["bias"] is not None:
            pre += d["bias"]
        if op == "linear_fwd":
            y = value(pre) + (0 if d["residual"] is None else d["residual"])
        else:
            y = value(pre[:, :N]) * pre[:, N:]
        return [y, pre] if case["pre"] else [y]
    if op == "linear_bwd":
        dpre = d["dy"] * derivative(d["pre"])
    else:
        gate, up = d["pre"].split(N, 1)
        dh = torch.matmul(d["dy"], d["w_down"]) if op == "block_bwd" else d["dy"]
        dpre = torch.cat((dh * up * derivative(gate), dh * value(gate)), 1)
    dx, dw = torch.matmul(dpre, d["w"]), torch.matmul(dpre.t(), d["x"])
    if op == "block_bwd":
        return [dx, dw, torch.matmul(d["dy"].t(), value(gate) * up)]
    return [dx, dw, dpre.sum(0)]
