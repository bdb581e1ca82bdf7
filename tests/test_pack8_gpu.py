"""Activations in 8 bits: bit for bit what the definition keeps (oracle/block_ops.py, a search over powers of two and multiples of steps
in 64 bits), where nothing but powers of two is multiplied; activations on the way within their own tolerance."""
import pytest
import torch

from oracle import block_ops as O

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
ACTS = ("relu", "gelu", "gelu_tanh", "silu", "none")


def make(rows, C, dtype, seed=0):
    """Numbers of all sizes: groups from 2^-130 to 2^120, ties, signed zeros, a few channels much larger than the rest."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.empty(rows, C, device="cuda").normal_(generator=g)
    x[:, 5::97] *= 16.0
    if rows > 4:
        x[1] *= 2.0 ** torch.randint(-130, 120, (C,), generator=g, device="cuda").float()
        x[2] = torch.randint(-300, 300, (C,), generator=g, device="cuda").float() * 0.5      # many halves of steps
        x[3] = 0.0
        x[4] = -0.0
    return x.to(TYPES[dtype])


def kept_of(x, fmt):
    kept, codes = O.packed(x.cpu(), fmt)
    return kept.cuda(), codes.cuda()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("rows,C", [(1, 8), (1, 32), (7, 40), (5, 96), (33, 200), (6, 1000), (129, 264), (3, 4096), (1000, 128), (2, 20000)], ids=str)
def test_by_the_definition(ctx, dtype, fmt, rows, C):
    from sirius_amd import ops
    x = make(rows, C, dtype)
    packed = ops.Packed8.empty(rows, C, fmt)
    packed.data.fill_(0x5a), packed.scales.fill_(0x5a)
    ops.pack8(ctx, x, packed)
    kept, codes = kept_of(x, fmt)
    assert torch.equal(packed.scales, codes)
    for out in TYPES.values():
        if out == torch.bfloat16 and C % 8:
            continue
        back = torch.empty(rows, C, dtype=out, device="cuda")
        ops.unpack8(ctx, packed, back)
        assert torch.equal(back.double(), kept)       # exact in either type
    # the bound that the format has
    unit = O.two_to(codes.long() - 127).repeat_interleave(32, 1)[:, :C]
    off = (x.double() - kept).abs()
    assert (off <= (unit / 2 if fmt == "int8" else torch.maximum(x.double().abs() / 16, unit * 2.0 ** -10))).all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_f32_rows_of_four(ctx, fmt):
    """Rows that are no multiple of eight elements (fp32)."""
    from sirius_amd import ops
    for C in (4, 12, 36, 60, 1004):
        x = make(9, C, "f32")
        packed = ops.Packed8.empty(9, C, fmt)
        ops.pack8(ctx, x, packed)
        back = torch.empty_like(x)
        ops.unpack8(ctx, packed, back)
        kept, codes = kept_of(x, fmt)
        assert torch.equal(packed.scales, codes) and torch.equal(back.double(), kept)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_the_ends_of_the_range(ctx, dtype, fmt):
    """The largest finite numbers saturate, the smallest go to zero; an infinity or a NaN takes its group with it and no other."""
    from sirius_amd import ops
    x = torch.zeros(6, 96, dtype=TYPES[dtype], device="cuda")
    x[0, 0], x[0, 40], x[0, 70] = torch.finfo(TYPES[dtype]).max, -torch.finfo(TYPES[dtype]).max, 2.0 ** 126
    x[1, 0], x[1, 40], x[1, 70] = 2.0 ** -117, 2.0 ** -126, -(2.0 ** -118)
    x[2, 33], x[3, 95], x[4, 2] = float("inf"), float("nan"), float("-inf")
    x[2:5, 1::7] = 1.5
    x[2, 33] = float("inf")
    x[5] = 127.0
    packed = ops.Packed8.empty(6, 96, fmt)
    ops.pack8(ctx, x, packed)
    back = torch.empty_like(x)
    ops.unpack8(ctx, packed, back)
    kept, codes = kept_of(x, fmt)
    assert torch.equal(packed.scales, codes)
    assert torch.equal(torch.isnan(back), torch.isnan(kept))
    assert torch.equal(back.double().nan_to_num(), kept.nan_to_num())
    assert torch.isfinite(back[:2]).all() and torch.isnan(back[2, 32:64]).all() and torch.isfinite(back[2, :32]).all()
    assert sorted(set(codes[2:5].view(-1).tolist()))[-1] == 255


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("rows,C", [(1, 8), (37, 200), (300, 1024)], ids=str)
def test_activations_on_the_way(ctx, dtype, act, rows, C):
    """h is that of linear_fwd's epilogue: its formulas within the tolerances of that (2^-21 of a value in fp32, 2^-17 before it is
    rounded in bf16: an exponential and a reciprocal of 2^-23 each, and 7.7e-6 at the far left end of GELU), of x as it came."""
    from sirius_amd import ops
    x = make(rows, C, dtype)
    if rows > 4:
        x[1].clamp_(-30, 30)
    packed, alone = ops.Packed8.empty(rows, C), ops.Packed8.empty(rows, C)
    h = torch.empty_like(x)
    ops.act_fwd_pack8(ctx, x, h, packed, act)
    ops.pack8(ctx, x, alone)
    assert torch.equal(packed.data, alone.data) and torch.equal(packed.scales, alone.scales)
    z = x.double()
    ref = {"relu": lambda: z.clamp(min=0), "gelu": lambda: z * 0.5 * torch.special.erfc(-z / 2 ** 0.5), "none": lambda: z,
           "gelu_tanh": lambda: z * torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (z + 0.044715 * z ** 3)), "silu": lambda: z * torch.sigmoid(z)}[act]()
    # the exponent's argument is rounded: up to 1.5 z^2 roundings of 2^-24 for GELU, |x| for the others
    far = {"gelu": 1.5 * z * z, "gelu_tanh": 4 * (z.abs() + z.abs() ** 3), "silu": 2 * z.abs()}.get(act, torch.zeros_like(z))
    rel = (40 + far) * 2.0 ** -24 + torch.finfo(TYPES[dtype]).eps / 2
    # a sigmoid or an integral below 2^-126 (x = -88 in SiLU: 6e-39) is subnormal, and the hardware's reciprocal and exponential leave 0
    # of it: up to 2^-126 of a factor |x| is lost there, and as much of a stored subnormal
    assert ((h.double() - ref).abs() <= rel * ref.abs() + (z.abs() + 1) * 2.0 ** -126).all()
    inplace = x.clone()
    ops.act_fwd_pack8(ctx, inplace, inplace, packed, act)
    assert torch.equal(inplace, h) and torch.equal(packed.data, alone.data)


def test_columns_of_wider_tensors(ctx):
    from sirius_amd import ops
    rows, C = 21, 104
    wide = make(rows, C + 64, "bf16")
    x = wide[:, 16:16 + C]
    packed, dense = ops.Packed8.empty(rows, C), ops.Packed8.empty(rows, C)
    ops.pack8(ctx, x, packed)
    ops.pack8(ctx, x.contiguous(), dense)
    assert torch.equal(packed.data, dense.data) and torch.equal(packed.scales, dense.scales)
    out = torch.full((rows + 2, C + 64), 3.0, dtype=torch.bfloat16, device="cuda")
    ops.unpack8(ctx, packed, out[1:-1, 8:8 + C])
    want = torch.empty(rows, C, dtype=torch.bfloat16, device="cuda")
    ops.unpack8(ctx, packed, want)
    assert torch.equal(out[1:-1, 8:8 + C], want)
    out[1:-1, 8:8 + C] = 3.0
    assert (out == 3.0).all()


def test_no_rows_and_replays(ctx):
    from sirius_amd import ops
    empty = torch.empty(0, 64, device="cuda")
    nothing = ops.Packed8.empty(0, 64)
    ops.pack8(ctx, empty, nothing)
    ops.unpack8(ctx, nothing, empty)
    c, prog = ops.Context(), ops.Program()
    x, back, packed = make(70, 136, "bf16"), torch.empty(70, 136, device="cuda"), ops.Packed8.empty(70, 136, "e4m3")
    c.begin_record(prog)
    ops.pack8(c, x, packed)
    ops.unpack8(c, packed, back)
    c.end_record()
    for step in range(3):
        x.copy_(make(70, 136, "bf16", seed=step))
        c.run(prog)
        c.synchronize()
        assert torch.equal(back.double(), kept_of(x, "e4m3")[0])


def test_offsets_beyond_four_gib(ctx):
    """Rows of x 2^31 bytes apart, and kept numbers behind 2^31 of their own."""
    from sirius_amd import ops
    ld, C = 2 ** 30 + 64, 96
    x = torch.empty(4 * ld, dtype=torch.bfloat16, device="cuda").view(4, ld)[:, :C]
    x.copy_(make(4, C, "bf16"))
    packed = ops.Packed8.empty(4, C)
    ops.pack8(ctx, x, packed)
    kept, codes = kept_of(x.contiguous(), "int8")
    assert torch.equal(packed.scales, codes)
    x.zero_()
    ops.unpack8(ctx, packed, x)
    assert torch.equal(x.double(), kept)
    del x
    rows, C = 270_000, 8192
    x = torch.zeros(rows, C, dtype=torch.bfloat16, device="cuda")
    x[-5:] = make(5, C, "bf16")
    packed = ops.Packed8.empty(rows, C, "e4m3")
    ops.pack8(ctx, x, packed)
    kept, codes = kept_of(x[-5:], "e4m3")
    assert torch.equal(packed.scales[-5:], codes) and int(packed.data[:-5].max()) == 0
    x.fill_(7.0)
    ops.unpack8(ctx, packed, x)
    assert torch.equal(x[-5:].double(), kept) and x[:-5].abs().max().item() == 0
