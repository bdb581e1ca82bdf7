"""What a transformer's training step has between its matrix products, case by case: rotary positions, the norms at a block's
boundary with its gate and residual scale, and activations kept in 8 bits for the backward pass.

``own = False`` computes every case in elementary torch operations in 32 bits (angles in 64), rounded once at the end; ``own = True``
makes the calls of this package.  As the training engines do, a program records its calls once, on buffers that it keeps, and a pass
replays them.
"""
import math
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f32": 4}
ACTS = ("relu", "gelu", "gelu_tanh", "silu")
_LARGEST = {"int8": 127.0, "e4m3": 448.0}
_GROUP = 32        # neighbours of a row that share a scale


def listed():
    return [
        # a server's next token, far into a long context: 32 query and 8 key heads, latency is what counts
        dict(name="rotary_token", op="rotary", dtype="bf16", batch=1, tokens=1, heads=40, head_dim=128, rot=128, layout="half",
             at="given", factor=8.0, back=False, wide=5120),
        # GPT-2 small's queries and keys, 8 sequences of 1024 tokens, columns of the packed projection
        dict(name="rotary_train", op="rotary", dtype="bf16", batch=8, tokens=1024, heads=24, head_dim=64, rot=64, layout="half",
             at="counted", factor=1.0, back=False, wide=2304),
        # sequences of any length packed together, a quarter of each head rotated, no size a multiple of a chunk
        dict(name="rotary_ragged", op="rotary", dtype="f32", batch=1, tokens=777, heads=14, head_dim=80, rot=20, layout="interleaved",
             at="given", factor=1.0, back=False, wide=1680),
        # the gradients of one long sequence's queries and keys
        dict(name="rotary_bwd_long", op="rotary", dtype="bf16", batch=1, tokens=131072, heads=40, head_dim=128, rot=128,
             layout="interleaved", at="counted", factor=4.0, back=True, wide=5120),
        # the boundary of a block for one token: both norms and a gate
        dict(name="norm_fwd_token", op="norm_fwd", dtype="bf16", samples=1, rows=1, width=4096, kind="rms", post=True, gate="vector",
             scale=1.0),
        # a training step's boundary, 8 sequences of 1024 tokens, with a scaled residual
        dict(name="norm_fwd_train", op="norm_fwd", dtype="bf16", samples=8, rows=1024, width=1024, kind="layer", post=False,
             gate="vector", scale=1.25),
        # 16 images of 196 tokens in fp32, each with a gate of its own
        dict(name="norm_bwd_samples", op="norm_bwd", dtype="f32", samples=16, rows=196, width=1024, kind="layer", post=True,
             gate="sample", scale=1.0),
        # a wide model's boundary, the largest batch
        dict(name="norm_bwd_large", op="norm_bwd", dtype="bf16", samples=16, rows=1024, width=8192, kind="rms", post=True,
             gate="vector", scale=1.0),
        # a small layer's input kept and fetched again; the last group of a row is short
        dict(name="pack_ragged", op="pack", dtype="f32", rows=1568, width=1000, format="e4m3"),
        # the activation of a training step's MLP: its input is kept in 8 bits, its gradient taken from that
        dict(name="act_train", op="act", dtype="bf16", rows=8192, width=4096, act="gelu_tanh", format="int8"),
        # the gated layer's derivative from its kept pre-activations, the hidden values computed again
        dict(name="gated_bwd_train", op="gated", dtype="bf16", rows=8192, width=5632, act="silu", format="int8"),
        # the weight gradient of a training step's projection from its kept input
        dict(name="wgrad_train", op="wgrad", dtype="bf16", rows=8192, cin=1024, cout=4096, format="e4m3"),
    ]


def _log(rng, low, high, step=1):
    """Between low and high, evenly over the logarithm, a multiple of step."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(low, min(high, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(["rotary", "rotary", "norm_fwd", "norm_bwd", "norm_bwd", "pack", "act", "gated", "wgrad"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    step = 8 if dtype == "bf16" else 4
    while True:
        case = dict(op=op, dtype=dtype)
        if op == "rotary":
            batch, tokens, heads = _log(rng, 1, 16), _log(rng, 1, 131072), _log(rng, 1, 64)
            head_dim = rng.choice([16, 32, 40, 64, 80, 96, 128, 256])
            case.update(batch=batch, tokens=tokens, heads=heads, head_dim=head_dim, rot=max(2, head_dim // rng.choice([1, 1, 2, 4])),
                        layout=rng.choice(["half", "interleaved"]), at=rng.choice(["given", "counted"]),
                        factor=rng.choice([1.0, 1.0, 4.0, 32.0]), back=rng.random() < 0.5,
                        wide=heads * head_dim + rng.choice([0, 0, head_dim * step, heads * head_dim]))
        elif op.startswith("norm"):
            case.update(samples=_log(rng, 1, 32), rows=_log(rng, 1, 4096), width=_log(rng, 64, 8192, step),
                        kind=rng.choice(["rms", "layer"]), post=rng.random() < 0.6, gate=rng.choice(["none", "vector", "sample"]),
                        scale=rng.choice([1.0, 1.0, 0.5, 2.5]))
        else:
            case.update(rows=_log(rng, 1, 16384), format=rng.choice(["int8", "e4m3"]))
            if op == "wgrad":
                case.update(cin=_log(rng, 64, 8192, step), cout=_log(rng, 64, 8192, step))
            else:
                case["width"] = _log(rng, 64, 11008, step)
                if op != "pack":
                    case["act"] = rng.choice(ACTS)
        w = work(case)
        # no dearer than the largest listed case; fp32 products take about ten times as long
        if w["bytes"] <= 2.6e9 and w["flops"] <= (4e11 if dtype == "bf16" else 4e10):
            return case


def work(case):
    op, e = case["op"], _SIZE[case["dtype"]]
    if op == "rotary":
        rows, n = case["batch"] * case["tokens"], case["heads"] * case["head_dim"]
        return {"bytes": 2 * e * rows * n + (8 * rows if case["at"] == "given" else 0) + 4 * case["rot"],
                "flops": 3 * rows * case["heads"] * case["rot"]}
    if op.startswith("norm"):
        n, C = case["samples"] * case["rows"], case["width"]
        vectors = 4 * C * (2 + 2 * case["post"]) + 4 * C * {"none": 0, "vector": 1, "sample": case["samples"]}[case["gate"]]
        if op == "norm_fwd":
            return {"bytes": 4 * e * n * C + 16 * n + vectors, "flops": 16 * n * C}
        return {"bytes": 6 * e * n * C + 16 * n + 2 * vectors, "flops": 30 * n * C}
    M = case["rows"]
    if op == "wgrad":
        K, N = case["cin"], case["cout"]
        return {"bytes": M * K * 33 / 32 + e * M * N + 4 * (K + 1) * N, "flops": 2 * M * K * N}
    n = M * case["width"]
    if op == "pack":        # read, kept, fetched, written
        return {"bytes": n * (2 * e + 2 * 33 / 32), "flops": 4 * n}
    if op == "act":         # forward: read, written, kept; backward: two read, one written
        return {"bytes": n * (4 * e + 2 * 33 / 32) + 4 * case["width"], "flops": 40 * n}
    return {"bytes": n * (4 * e + 2 * 33 / 32), "flops": 40 * n}   # gated: dh and the kept pair read, the pair's gradient and h written


def _inputs(case, seed):
    """The tensors that both forms and the exact one start from."""
    dt, op = _TYPES[case["dtype"]], case["op"]
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def normal(*shape, std=1.0, mean=0.0, dtype=dt):
        return torch.empty(shape, dtype=dtype, device="cuda").normal_(mean, std, generator=gen)

    def vector(n, mean):
        return normal(n, std=0.2, mean=mean, dtype=torch.float32)
    if op == "rotary":
        B, T, n = case["batch"], case["tokens"], case["heads"] * case["head_dim"]
        s = dict(x=normal(B, T, case["wide"])[..., :n], freqs=_frequencies(case).cuda())
        s["positions"] = None
        if case["at"] == "given":
            s["positions"] = torch.randint(0, 200_000, (B * T,), generator=gen, device="cuda")
        return s
    if op.startswith("norm"):
        n, C = case["samples"] * case["rows"], case["width"]
        layer = case["kind"] == "layer"
        s = dict(weight=vector(C, 1.0), bias=vector(C, 0.0) if layer else None, post_weight=None, post_bias=None, gate=None)
        if case["post"]:
            s["post_weight"], s["post_bias"] = vector(C, 1.0), vector(C, 0.0) if layer else None
        if case["gate"] != "none":
            s["gate"] = vector(case["samples"] * C, 0.5).view(-1, C) if case["gate"] == "sample" else vector(C, 0.5)
        if op == "norm_fwd":
            s["x"], s["branch"] = normal(n, C, std=2.0, mean=0.25), normal(n, C)
            return s
        # behind the forward pass: the sum and the branch, their statistics, and the gradients of both outputs
        s["total"], s["branch"] = normal(n, C, std=2.0, mean=0.25), normal(n, C)
        s["dy"], s["dtotal"] = normal(n, C, std=0.02), normal(n, C, std=0.02)
        s["stats"] = torch.cat([_statistics(s["branch"], layer, case["post"]), _statistics(s["total"], layer, True)], 1)
        return s
    M = case["rows"]
    if op == "wgrad":
        x = _outlying(normal(M, case["cin"]))
        data, scales = _pack(x.float(), case["format"])
        return dict(data=data, scales=scales, dy=normal(M, case["cout"], std=0.02))
    C = case["width"]
    if op == "pack":
        return dict(x=_outlying(normal(M, C)))
    if op == "act":
        return dict(pre=_outlying(normal(M, C)), dy=normal(M, C, std=0.02))
    data, scales = _pack(_outlying(normal(M, 2 * C)).float(), case["format"])
    return dict(data=data, scales=scales, dh=normal(M, C, std=0.02))


def _outlying(x):
    """A few channels of a trained model's activations are much larger than the others."""
    x[:, 5::97] *= 16.0
    return x


def _frequencies(case):
    """Radians a position of every pair.  A longer context than the 4096 tokens trained on: pairs that turn over 32 times within
    those stay, those that turn over less than once are slowed down by the factor, and in between the one goes over into the other."""
    i = torch.arange(case["rot"] // 2, dtype=torch.float64)
    f = torch.pow(torch.tensor(10000.0, dtype=torch.float64), -2.0 * i / case["rot"])
    kept = ((4096.0 * f / (2.0 * math.pi) - 1.0) / 31.0).clamp(0.0, 1.0)
    return f * (kept + (1.0 - kept) / case["factor"])


def _statistics(v, layer, wanted):
    """[rows, 2] fp32: mean (RMS: 0) and one over the deviation."""
    v = v.float()
    if not wanted:
        return v.new_zeros(v.shape[0], 2)
    mean = v.mean(1, keepdim=True) if layer else v.new_zeros(v.shape[0], 1)
    d = v - mean
    return torch.cat([mean, 1.0 / torch.sqrt((d * d).mean(1, keepdim=True) + 1e-5)], 1)


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        _record(s, case)
    return s


def _record(s, case):
    """What a program of this package keeps: a context, output buffers, workspaces and the recorded calls."""
    from sirius_amd import ops
    op, ctx = case["op"], ops.Context()

    def new(*shape, dtype=_TYPES[case["dtype"]]):
        return torch.empty(shape, dtype=dtype, device="cuda")

    def vector(name):
        return None if s[name] is None else torch.empty_like(s[name])
    if op == "rotary":
        y = new(*s["x"].shape)
        rotary = ops.rotary_bwd if case["back"] else ops.rotary_fwd
        calls = [lambda: rotary(ctx, s["x"], y, s["freqs"], case["head_dim"], layout=case["layout"], positions=s["positions"],
                                seq=case["tokens"], scale=_rotary_scale(case))]
        s["out"] = [y]
    elif op == "norm_fwd":
        total, y, stats = new(*s["x"].shape), new(*s["x"].shape), new(s["x"].shape[0], 4, dtype=torch.float32)
        calls = [lambda: ops.residual_norm_fwd(ctx, s["x"], s["branch"], total, y, stats, kind=case["kind"], weight=s["weight"],
                                               bias=s["bias"], post_weight=s["post_weight"], post_bias=s["post_bias"],
                                               gate=s["gate"], scale=case["scale"])]
        s["out"] = [total, y]
    elif op == "norm_bwd":
        dx, dbranch = new(*s["total"].shape), new(*s["total"].shape)
        grads = {k: vector(k) for k in ("weight", "bias", "post_weight", "post_bias", "gate")}
        scratch = new(ops.residual_norm_bwd_workspace_bytes(s["total"], gate=s["gate"]), dtype=torch.uint8)
        calls = [lambda: ops.residual_norm_bwd(ctx, s["dy"], s["dtotal"], s["total"], s["branch"], dx, dbranch, s["stats"],
                                               kind=case["kind"], weight=s["weight"], post_weight=s["post_weight"],
                                               post_bias=s["post_bias"], gate=s["gate"], scale=case["scale"],
                                               dweight=grads["weight"], dbias=grads["bias"], dpost_weight=grads["post_weight"],
                                               dpost_bias=grads["post_bias"], dgate=grads["gate"], workspace=scratch)]
        s["keep"], s["out"] = scratch, [dx, dbranch] + [g for g in grads.values() if g is not None]
    elif op in ("pack", "act"):
        C = case["width"]
        packed = ops.Packed8(new(case["rows"], C, dtype=torch.uint8), new(case["rows"], -(-C // _GROUP), dtype=torch.uint8),
                             case["format"])
        if op == "pack":
            back = new(case["rows"], C)
            calls = [lambda: ops.pack8(ctx, s["x"], packed), lambda: ops.unpack8(ctx, packed, back)]
            s["keep"], s["out"] = packed, [back]
        else:
            h, dz, db = new(case["rows"], C), new(case["rows"], C), new(C, dtype=torch.float32)
            scratch = new(ops.act_bwd_workspace_bytes(s["dy"]), dtype=torch.uint8)
            calls = [lambda: ops.act_fwd_pack8(ctx, s["pre"], h, packed, case["act"]),
                     lambda: ops.act_bwd_packed(ctx, s["dy"], packed, dz, case["act"], dbias=db, workspace=scratch)]
            s["keep"], s["out"] = (packed, scratch), [h, dz, db]
    elif op == "gated":
        packed = ops.Packed8(s["data"], s["scales"], case["format"])
        dpre, h = new(case["rows"], 2 * case["width"]), new(case["rows"], case["width"])
        calls = [lambda: ops.gated_act_bwd_packed(ctx, s["dh"], packed, dpre, case["act"], h=h)]
        s["keep"], s["out"] = packed, [dpre, h]
    else:
        packed = ops.Packed8(s["data"], s["scales"], case["format"])
        dw, db = new(case["cout"], case["cin"], dtype=torch.float32), new(case["cout"], dtype=torch.float32)
        scratch = new(ops.linear_wgrad_packed_workspace_bytes(packed, s["dy"]), dtype=torch.uint8)
        calls = [lambda: ops.linear_wgrad_packed(ctx, packed, s["dy"], dw, dbias=db, workspace=scratch)]
        s["keep"], s["out"] = (packed, scratch), [dw, db]
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
    return z / (1.0 + torch.exp(-z))


def _slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    if act == "gelu_tanh":
        t = torch.tanh(_TANH_A * (z + _TANH_B * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * _TANH_A * (1.0 + 3.0 * _TANH_B * z * z)
    sig = 1.0 / (1.0 + torch.exp(-z))
    return sig * (1.0 + z * (1.0 - sig))


def _rotary_scale(case):
    """The factor on queries and keys that goes with a longer context."""
    return 1.0 + 0.1 * math.log(case["factor"])


def _grouped(x):
    """[rows, groups, 32], the last group filled up with zeros."""
    M, C = x.shape
    groups = -(-C // _GROUP)
    full = x.new_zeros(M, groups * _GROUP)
    full[:, :C] = x
    return full.view(M, groups, _GROUP)


def _power(e):
    """2^e in fp32, from its bits."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _pack(x, fmt):
    """fp32 [rows, C] -> the 8-bit numbers [rows, C] as bytes, and a byte for the power of two of every 32 neighbours: 127 + e, e the
    smallest (down to -117) with which none of them is beyond the type's largest number."""
    most = _LARGEST[fmt]
    g = _grouped(x)
    m, e = torch.frexp(g.abs().amax(2))
    m0, e0 = math.frexp(most)
    e = (e - e0 + (m > m0)).clamp(min=-117)
    v = (g * _power(-e)[..., None]).clamp(-most, most).view(x.shape[0], -1)[:, :x.shape[1]]
    q = torch.round(v).to(torch.int8) if fmt == "int8" else v.to(torch.float8_e4m3fn)
    return q.contiguous().view(torch.uint8), (e + 127).to(torch.uint8)


def _values(data, scales, fmt):
    """fp32 [rows, C] that the bytes stand for."""
    M, C = data.shape
    q = data.view(torch.int8 if fmt == "int8" else torch.float8_e4m3fn).float()
    return (_grouped(q) * _power(scales.int() - 127)[..., None]).view(M, -1)[:, :C]


def _rotate(x, cos, sin, case):
    rot, half = case["rot"], case["rot"] // 2
    if case["layout"] == "half":
        a, b = x[..., :half], x[..., half:rot]
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
    y = x.clone()
    u, v = a * cos - b * sin, b * cos + a * sin
    if case["layout"] == "half":
        y[..., :half], y[..., half:rot] = u, v
    else:
        y[..., 0:rot:2], y[..., 1:rot:2] = u, v
    return y


def _normed(v, stats, weight, bias):
    h = (v - stats[:, :1]) * stats[:, 1:]
    y = h * weight
    return y if bias is None else y + bias


def _rowwise(gate, rows):
    """The gate of every row."""
    if gate.dim() == 1:
        return gate
    return gate.repeat_interleave(rows // gate.shape[0], 0)


def _plain(s, case):
    op, dt = case["op"], _TYPES[case["dtype"]]
    if op == "rotary":
        B, T = case["batch"], case["tokens"]
        at = s["positions"].view(B, T) if s["positions"] is not None else torch.arange(T, device="cuda").expand(B, T)
        angle = at.double()[..., None, None] * s["freqs"]
        if case["back"]:
            angle = -angle
        scale = _rotary_scale(case)
        x = s["x"].float().reshape(B, T, case["heads"], case["head_dim"])
        y = _rotate(x, (torch.cos(angle) * scale).float(), (torch.sin(angle) * scale).float(), case)
        return [y.view(B, T, -1).to(dt)]
    if op == "norm_fwd":
        layer, n = case["kind"] == "layer", case["samples"] * case["rows"]
        v = s["branch"].float()
        if case["post"]:
            v = _normed(v, _statistics(v, layer, True), s["post_weight"], s["post_bias"])
        if s["gate"] is not None:
            v = v * _rowwise(s["gate"], n)
        total = (s["x"].float() * case["scale"] + v).to(dt)
        t = total.float()
        return [total, _normed(t, _statistics(t, layer, True), s["weight"], s["bias"]).to(dt)]
    if op == "norm_bwd":
        return _norm_bwd(s, case, dt)
    if op == "pack":
        data, scales = _pack(s["x"].float(), case["format"])
        return [_values(data, scales, case["format"]).to(dt)]
    if op == "act":
        pre = s["pre"].float()
        kept = _values(*_pack(pre, case["format"]), case["format"])
        dz = s["dy"].float() * _slope(kept, case["act"])
        return [_act(pre, case["act"]).to(dt), dz.to(dt), dz.sum(0)]
    kept = _values(s["data"], s["scales"], case["format"])
    if op == "gated":
        g, u = kept[:, :case["width"]], kept[:, case["width"]:]
        dh, value = s["dh"].float(), _act(g, case["act"])
        return [torch.cat([dh * u * _slope(g, case["act"]), dh * value], 1).to(dt), (value * u).to(dt)]
    dy = s["dy"].float()
    return [dy.t() @ kept, dy.sum(0)]


def _through(d, h, rstd, weight, layer):
    """The gradient of a normalised tensor's input from that of its output."""
    d = d * weight
    r = d - h * (d * h).mean(1, keepdim=True)
    if layer:
        r = r - d.mean(1, keepdim=True)
    return r * rstd


def _norm_bwd(s, case, dt):
    layer, n = case["kind"] == "layer", case["samples"] * case["rows"]
    st, dy, b = s["stats"], s["dy"].float(), s["branch"].float()
    h = (s["total"].float() - st[:, 2:3]) * st[:, 3:]
    dt_all = s["dtotal"].float() + _through(dy, h, st[:, 3:], s["weight"], layer)
    grads = [(dy * h).sum(0)] + ([dy.sum(0)] if layer else [])
    dn = dt_all if s["gate"] is None else dt_all * _rowwise(s["gate"], n)
    out, db = b, dn
    if case["post"]:
        h = (b - st[:, :1]) * st[:, 1:2]
        out = h * s["post_weight"] if s["post_bias"] is None else h * s["post_weight"] + s["post_bias"]
        db = _through(dn, h, st[:, 1:2], s["post_weight"], layer)
        grads += [(dn * h).sum(0)] + ([dn.sum(0)] if layer else [])
    if s["gate"] is not None:
        dg = dt_all * out
        grads.append(dg.sum(0) if s["gate"].dim() == 1 else dg.view(case["samples"], case["rows"], -1).sum(1))
    return [(dt_all * case["scale"]).to(dt), db.to(dt)] + grads


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def _two_to(power):
    """2^power in 64 bits, exactly: a power function's last bit would decide between two neighbours of a value half way."""
    return ((power.long() + 1023) << 52).view(torch.float64)


def _kept(x, fmt):
    """What 8 bits keep of x, by the definition: multiples of a step within each group of 32."""
    most = _LARGEST[fmt]
    blocks = torch.nn.functional.pad(x, (0, -x.shape[1] % _GROUP)).unflatten(1, (-1, _GROUP))
    top = blocks.abs().amax(2, keepdim=True)
    power = torch.ceil(torch.log2(torch.where(top > 0, top, 1.0) / most))
    power = torch.where(top > most * _two_to(power), power + 1, power)       # (a logarithm next to a whole number)
    power = torch.where(top <= most * _two_to(power - 1), power - 1, power).clamp(min=-117)
    unit = _two_to(power)
    if fmt == "int8":
        step = unit
    else:
        ratio = blocks.abs() / unit
        step = unit * _two_to(torch.frexp(ratio.clamp(min=2.0 ** -6))[1] - 4)
    return (torch.round(blocks / step) * step).flatten(1)[:, :x.shape[1]]


def _decoded(data, scales, fmt):
    """The numbers behind the bytes, from their bits."""
    b = data.long()
    if fmt == "int8":
        v = torch.where(b > 127, b - 256, b).double()
    else:
        power, part = (b >> 3) & 15, (b & 7).double()
        v = torch.where(power > 0, (8.0 + part) * _two_to(power - 10), part * 2.0 ** -9) * torch.where(b > 127, -1.0, 1.0)
    return v * _two_to(scales.long() - 127).repeat_interleave(_GROUP, 1)[:, :data.shape[1]]


def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    d = {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in s.items()}
    if op == "rotary":
        B, T, r = case["batch"], case["tokens"], case["rot"]
        at = d["positions"].double().view(B, T, 1, 1) if d["positions"] is not None else \
            torch.arange(T, dtype=torch.float64, device="cuda").view(1, T, 1, 1)
        turn = torch.polar(torch.full_like(d["freqs"], 1.0 + 0.1 * math.log(case["factor"])).expand(*at.shape[:3], -1),
                           (-at if case["back"] else at) * d["freqs"])
        x = d["x"].reshape(B, T, case["heads"], case["head_dim"])
        part = x[..., :r]
        pairs = part.unflatten(-1, (2, r // 2)).transpose(-1, -2) if case["layout"] == "half" else part.unflatten(-1, (r // 2, 2))
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        z = z.transpose(-1, -2).flatten(-2) if case["layout"] == "half" else z.flatten(-2)
        return [torch.cat([z, x[..., r:]], -1).reshape(B, T, -1)]
    if op.startswith("norm"):
        def norm(v, weight, bias):
            if case["kind"] == "layer":
                v = v - v.mean(1, keepdim=True)
            v = v / torch.sqrt(v.square().mean(1, keepdim=True) + 1e-5) * weight
            return v if bias is None else v + bias

        def boundary(x, t=None):
            v = norm(d["branch"], d["post_weight"], d["post_bias"]) if case["post"] else d["branch"]
            if d["gate"] is not None:
                v = (v.view(case["samples"], case["rows"], -1) * d["gate"].view(-1, 1, case["width"])).flatten(0, 1)
            return x * case["scale"] + v
        if op == "norm_fwd":
            total = boundary(d["x"])
            # the second norm is that of the sum as it is stored
            return [total, norm(total.to(_TYPES[case["dtype"]]).double(), d["weight"], d["bias"])]
        names = [k for k in ("weight", "bias", "post_weight", "post_bias", "gate") if d[k] is not None]
        x = torch.zeros_like(d["total"])
        leaves = [x, d["branch"]] + [d[k] for k in names]
        for v in leaves + [d["total"]]:
            v.requires_grad_(True)
        # the gradient of the sum, from its norm; then through the sum
        y = norm(d["total"], d["weight"], d["bias"])
        first = [d["total"]] + [d[k] for k in names if k in ("weight", "bias")]
        g = torch.autograd.grad(y, first, d["dy"])
        rest = [x, d["branch"]] + [d[k] for k in names if k not in ("weight", "bias")]
        h = torch.autograd.grad(boundary(x), rest, d["dtotal"] + g[0])
        return list(h[:2]) + list(g[1:]) + list(h[2:])
    fmt = case["format"]
    if op == "pack":
        return [_kept(d["x"], fmt)]

    def value(z):
        if case["act"] == "gelu":       # z times the normal distribution's integral, without cancellation on the left
            return z * 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
        if case["act"] == "gelu_tanh":
            return z * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z.pow(3)))
        return {"relu": lambda: z.clamp(min=0), "silu": lambda: z * torch.sigmoid(z)}[case["act"]]()

    def derivative(z):
        z = z.clone().requires_grad_(True)
        return torch.autograd.grad(value(z).sum(), z)[0]
    if op == "act":
        dz = d["dy"] * derivative(_kept(d["pre"], fmt))
        return [value(d["pre"]), dz, dz.sum(0)]
    kept = _decoded(s["data"], s["scales"], fmt)
    if op == "gated":
        gate, up = kept.split(case["width"], 1)
        return [torch.cat((d["dh"] * up * derivative(gate), d["dh"] * value(gate)), 1), value(gate) * up]
    return [torch.matmul(d["dy"].t(), kept), d["dy"].sum(0)]
