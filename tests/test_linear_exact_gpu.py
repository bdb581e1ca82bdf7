"""Products whose sums are whole numbers below 2^24, which fp32 adds up without a rounding whatever the order: every bit has to be
right, so that no row may be left out or counted twice."""
import pytest
import torch

from test_linear_gpu import BF16, F32

pytestmark = pytest.mark.gpu


def signs(*shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-1, 2, shape, generator=g, device="cuda", dtype=torch.int8).to(dtype)


@pytest.mark.parametrize("dtype,M,K,N", [(BF16, 2_200_123, 1024, 64), (BF16, 1_050_011, 136, 1032), (F32, 600_011, 1024, 64)], ids=str)
def test_weight_gradients_beyond_two_gigabytes(ctx, dtype, M, K, N):
    """2.2 million rows: operands and their pieces far behind 2^31 and 2^32 bytes."""
    from sirius_amd import ops
    assert M < 2 ** 24 and M * max(K, N) * torch.finfo(dtype).bits // 8 > 2 ** 31
    x, dy = signs(M, K, dtype=dtype, seed=1), signs(M, N, dtype=dtype, seed=2)
    want, want_db = torch.zeros(N, K, dtype=torch.float64, device="cuda"), torch.zeros(N, dtype=torch.float64, device="cuda")
    for at in range(0, M, 100_000):
        part = dy[at:at + 100_000].double()
        want += part.t() @ x[at:at + 100_000].double()
        want_db += part.sum(0)
    need = ops.linear_bwd_workspace_bytes(x, N)
    for ws in (torch.empty(need, dtype=torch.uint8, device="cuda"), None):
        dw, db = torch.full((N, K), 3.0, device="cuda"), torch.full((N,), 3.0, device="cuda")
        ops.linear_wgrad(ctx, x, dy, dw, dbias=db, workspace=ws)
        assert torch.equal(dw.double(), want) and torch.equal(db.double(), want_db), "with" if ws is not None else "without"
        ops.linear_wgrad(ctx, x, dy, dw, dbias=db, workspace=ws, accumulate=True)
        assert torch.equal(dw.double(), 2 * want) and torch.equal(db.double(), 2 * want_db)
