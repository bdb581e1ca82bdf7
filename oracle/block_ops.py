"""The norms at a block's boundary and the 8-bit activations in 64 bits (torch on any device), and how far a kernel that computes in
fp32 may be off: bounds by the number of roundings on the way, in units of u = 2^-24."""
import torch

U = 2.0 ** -24


def hat(v, kind, eps):
    """(v^, mean, 1 / deviation) of the rows of v."""
    mean = v.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(v[:, :1])
    r = 1.0 / torch.sqrt((v - mean).square().mean(1, keepdim=True) + eps)
    return (v - mean) * r, mean, r


def hat_error(v, h, r):
    """Of v^ from a mean and a deviation that are added up in fp32: eight numbers a lane, six steps over a wavefront and sixteen wavefronts
    are at most 30 additions."""
    return U * (30.0 * v.square().mean(1, keepdim=True).sqrt() * r + 22.0 * h.abs())


def gate_rows(gate, rows):
    """The gate of every row, [rows or 1, C]."""
    if gate is None:
        return 1.0
    gate = gate.view(-1, gate.shape[-1])
    return gate.repeat_interleave(rows // gate.shape[0], 0)


def boundary(x, branch, kind, post_weight=None, post_bias=None, gate=None, scale=1.0, eps=1e-5):
    """(total, its error) before it is rounded to its type."""
    n, err = branch, torch.zeros_like(branch)
    if post_weight is not None:
        h, _, r = hat(branch, kind, eps)
        n = h * post_weight + (0.0 if post_bias is None else post_bias)
        err = post_weight.abs() * hat_error(branch, h, r) + 2 * U * n.abs()
    g = gate_rows(gate, x.shape[0])
    total = scale * x + g * n
    g = abs(g) if gate is None else g.abs()
    return total, g * err + 3 * U * ((scale * x).abs() + g * n.abs())


def norm(total, kind, weight, bias=None, eps=1e-5):
    h, _, r = hat(total, kind, eps)
    y = h * weight + (0.0 if bias is None else bias)
    return y, weight.abs() * hat_error(total, h, r) + 2 * U * ((h * weight).abs() + y.abs())


def through(k, h, r, kind, k_err, stat_err):
    """The gradient of a norm's input from k, that of v^, and its error."""
    mean = (lambda t: t.mean(1, keepdim=True)) if kind == "layer" else (lambda t: 0.0)
    q = (k * h).mean(1, keepdim=True)
    d = r * (k - mean(k) - h * q)
    abs_q = (k * h).abs().mean(1, keepdim=True)
    err = k_err + mean(k_err) + h.abs() * (k_err * h.abs()).mean(1, keepdim=True)
    err = err + U * (4 * k.abs() + 40 * mean(k.abs()) + 44 * h.abs() * abs_q)
    # where mean and deviation are off by stat_err themselves: one factor r, and v^ twice
    err = err + stat_err * (k.abs() + mean(k.abs()) + 3 * h.abs() * abs_q + abs_q)
    return d, r * err


def boundary_grads(dy, dtotal, total, branch, kind, weight=None, post_weight=None, post_bias=None, gate=None, scale=1.0, eps=1e-5, stat_err=0.0):
    """{name: (gradient, error)} of dx, dbranch, dweight, dbias, dpost_weight, dpost_bias, dgate; the errors without the rounding of dx
    and dbranch to their type.  Sums over rows: a lane's rows one by one, sixteen row groups, then fp64: at most 60 roundings here."""
    out = {}
    like = total if total is not None else dtotal
    rows = like.shape[0]
    d = torch.zeros_like(like) if dtotal is None else dtotal.clone()
    err = 2 * U * d.abs()
    many = 60 * U
    if weight is not None:
        h, _, r = hat(total, kind, eps)
        k = dy * weight
        more, e = through(k, h, r, kind, U * k.abs(), stat_err)
        d, err = d + more, err + e + 2 * U * (d + more).abs()
        out["dweight"] = ((dy * h).sum(0), (many + stat_err) * (dy * h).abs().sum(0) + stat_err * dy.abs().sum(0))
        out["dbias"] = (dy.sum(0), many * dy.abs().sum(0))
    out["dx"] = (scale * d, abs(scale) * err + U * (scale * d).abs())
    if branch is None:
        return out
    g = gate_rows(gate, rows)
    ga = abs(g) if gate is None else g.abs()
    dn, dn_err = g * d, ga * err + U * (g * d).abs()
    h, r = branch, 1.0
    if post_weight is not None:
        h, _, r = hat(branch, kind, eps)
        k = dn * post_weight
        out["dbranch"] = through(k, h, r, kind, dn_err * post_weight.abs() + U * k.abs(), stat_err)
        out["dpost_weight"] = ((dn * h).sum(0), (dn_err * h.abs() + (many + stat_err) * (dn * h).abs() + stat_err * dn.abs()).sum(0))
        out["dpost_bias"] = (dn.sum(0), (dn_err + many * dn.abs()).sum(0))
    else:
        out["dbranch"] = (dn, dn_err)
    if gate is not None:
        gates = gate.numel() // gate.shape[-1]
        w = 1.0 if post_weight is None else post_weight
        n = h * w + (0.0 if post_bias is None else post_bias)
        size = (h * w).abs() + (0.0 if post_bias is None else post_bias.abs())
        part = lambda t: t.view(gates, rows // gates, -1).sum(1)  # noqa: E731
        out["dgate"] = (part(d * n), part(err * size + (many + stat_err) * d.abs() * size + stat_err * d.abs() * abs(w)))
    return out


def two_to(power):
    """2^power, exactly (a power function may be off by its last bit, which then decides about values half way between two)."""
    return ((power.long() + 1023) << 52).view(torch.float64)


LARGEST = {"int8": 127.0, "e4m3": 448.0}


def packed(x, fmt):
    """(what 8 bits keep of x [rows, C], the scales' bytes): multiples of a step within every 32 neighbours, to nearest even."""
    x = x.double()
    rows, C = x.shape
    most, groups = LARGEST[fmt], -(-C // 32)
    blocks = torch.nn.functional.pad(x, (0, 32 * groups - C)).view(rows, groups, 32)
    top = blocks.abs().amax(2)
    power = torch.full_like(top, -117.0)
    last = {"int8": 121.0, "e4m3": 119.0}[fmt]
    good = torch.isfinite(top)
    for _ in range(260):       # one by one: the definition, not a formula for it
        power = torch.where(good & (top > most * two_to(power)) & (power < last), power + 1, power)
    unit = two_to(power)[..., None]
    v = (blocks / unit).clamp(-most, most)
    if fmt == "int8":
        kept = torch.round(v)
    else:
        step = torch.full_like(v, 2.0 ** -9)
        for e in range(-5, 9):
            step = torch.where(v.abs() >= 2.0 ** e, 2.0 ** (e - 3), step)
        kept = torch.round(v / step) * step
    kept = torch.where(good[..., None], kept * unit, float("nan"))
    codes = torch.where(good, power + 127, 255.0).to(torch.uint8)
    return kept.view(rows, -1)[:, :C], codes
