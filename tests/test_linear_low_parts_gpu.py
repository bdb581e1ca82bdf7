"""Low parts of bf16 gradients where a lost, shifted or repeated one shows: drawn as large as the high part, so that the result without
them is off by as much as there is of it.

Bounds: as in test_linear_gpu.py; both parts' products are added up separately, so a sum over n terms has 2 n of them, of
|high| + |low| in size."""
import pytest
import torch

from test_linear_gpu import BF16, F32, Framed, near, rnd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("low", ["dy", "x"])
@pytest.mark.parametrize("M,K,N", [(1, 8, 8), (31, 264, 72), (64, 136, 136), (1000, 256, 256), (3001, 776, 1288), (9000, 264, 264), (70, 2056, 2312),
                                   # 256 x 256 tiles: whole rounds and a rest that fewer workgroups share; two rounds and a rest
                                   (1803, 5120, 3312), (2319, 3976, 8736)])
def test_weight_gradients(ctx, M, K, N, low):
    from sirius_amd import ops
    x, dy = rnd(M, K, dtype=BF16, seed=1), rnd(M, N, dtype=BF16, seed=2)
    part = rnd(M, N if low == "dy" else K, dtype=BF16, seed=3)
    a, b, a_size, b_size = dy.double(), x.double(), dy.double().abs(), x.double().abs()
    if low == "dy":
        a, a_size = a + part.double(), a_size + part.double().abs()
    else:
        b, b_size = b + part.double(), b_size + part.double().abs()
    for split in (True, False):
        dw, db = Framed(N, K, F32, False), Framed(1, N, F32, False)
        ws = torch.empty(ops.linear_bwd_workspace_bytes(x, N), dtype=torch.uint8, device="cuda") if split else None
        ops.linear_wgrad(ctx, x, dy, dw.view, dbias=db.view, workspace=ws, **{low + "_low": part})
        sums = (2 * M + 64) * 2.0 ** -23
        near(dw.view, a.t() @ b, sums * (a_size.t() @ b_size) + 1e-30, "dw")
        near(db.view, a.sum(0, keepdim=True), sums * a_size.sum(0, keepdim=True) + 1e-30, "db")
        dw.check("dw")
        db.check("db")
