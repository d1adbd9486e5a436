"""What the sums of linear_8bit hold where large products cancel: float32 results and 16-bit results of up
to 32 rows come from float32 sums; 16-bit results of more rows lose what the documentation says."""
import pytest
import torch

import kalman_vae_amd as kv

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
UNIT = 2.0 ** -24
ROWS = [1, 2, 15, 16, 17, 31, 32]


def cancelling(M, N, K, seed):
    """Rows whose products in columns 8 i and 8 i + 5 are large and cancel; the others are small."""
    g = torch.Generator("cuda").manual_seed(seed)
    x, w = (torch.randn(n, K, generator=g, device="cuda").mul(2.0 ** -4) for n in (M, N))
    big = torch.arange(0, K - 5, 8, device="cuda")
    x[:, big] = torch.rand(M, big.numel(), generator=g, device="cuda") * 200 + 200
    x[:, big + 5] = x[:, big]
    w[:, big] = torch.rand(N, big.numel(), generator=g, device="cuda") * 200 + 200
    w[:, big + 5] = -w[:, big]
    one = lambda n: torch.ones(n, device="cuda")  # noqa: E731
    return x.to(E4M3), one(M), w.to(E4M3), one(N)


def float_bound(a, b, want, dtype):
    """K exact terms added in float32 in some order, one rounding to the type; below its normal range a
    fixed step."""
    size = a.abs() @ b.abs().t().contiguous()
    err = a.shape[1] * UNIT * size
    half = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    return err + half * (want.abs() + err) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


@pytest.mark.parametrize("M", ROWS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,K", [(40, 8), (33, 24), (384, 128), (100, 250)])
def test_float_sums(M, dtype, N, K):
    x, sx, w, sw = cancelling(M, N, K, M + K)
    a, b = x.double(), w.double()
    want = a @ b.t().contiguous()
    y = kv.linear_8bit(x, sx, w, sw, dtype=dtype).double()
    assert ((y - want).abs() <= float_bound(a, b, want, dtype)).all()


@pytest.mark.parametrize("M", ROWS + [33, 64, 65, 300])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_one_beside_two_that_cancel(M, dtype):
    """448 * 448 - 448 * 448 + 1: 1 from a float sum; the 8-bit instructions lose the 1 (2^-17.6 of the largest)."""
    x, w = torch.zeros(M, 8, device="cuda"), torch.zeros(3, 8, device="cuda")
    x[:, 0], x[:, 3], x[:, 6] = 448, 448, 1
    w[:, 0], w[:, 3], w[:, 6] = 448, -448, 1
    y = kv.linear_8bit(x.to(E4M3), torch.ones(M, device="cuda"), w.to(E4M3), torch.ones(3, device="cuda"), dtype=dtype)
    if dtype == torch.float32 or M <= 32:
        assert (y == 1).all()
    else:
        assert ((y.double() - 1).abs() <= 7 * 2.0 ** -13 * 448 ** 2).all()


@pytest.mark.parametrize("M", [33, 64, 200, 4096])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_documented_loss(M, dtype):
    """More rows, 16 bits: within 2^-13 of the largest product for each of the other seven of every eight."""
    N, K = (4096, 1024) if M == 4096 else (384, 128)
    x, sx, w, sw = cancelling(M, N, K, M)
    rows = torch.arange(0, M, max(1, M // 50), device="cuda")
    a, b = x.double(), w.double()
    want = a[rows] @ b.t().contiguous()
    largest = sum((a[rows, None, k:k + 8] * b[None, :, k:k + 8]).abs().amax(-1) for k in range(0, K, 8))
    y = kv.linear_8bit(x, sx, w, sw, dtype=dtype)[rows].double()
    err = float_bound(a[rows], b, want, dtype) + 7 * 2.0 ** -13 * largest * (1 + torch.finfo(dtype).eps)
    assert ((y - want).abs() <= err).all()
