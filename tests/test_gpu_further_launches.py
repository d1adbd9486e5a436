"""More rows than one launch takes: the rows behind go in further launches of the norm (a row of two
elements has four lanes, a launch fewer than 2^31 of these) and of the product (65535 blocks of rows)."""
import pytest
import torch

import kalman_vae_amd as kv

pytestmark = pytest.mark.gpu

UNIT = 2.0 ** -24


def around(seam, rows):
    """Slices that cover the first rows, the rows on either side of the seam, and the last ones."""
    return [slice(0, 5000), slice(seam - 5000, min(seam + 5000, rows)), slice(rows - 5000, rows)]


def test_norm():
    seam = 1 << 29
    rows, D = seam + 100_003, 2
    x = torch.empty(rows, D, dtype=torch.float16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(1))
    res = torch.empty(rows, D, dtype=torch.float16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(2))
    w = torch.tensor([0.5, -2.0], device="cuda")
    exact = {}
    for i, part in enumerate(around(seam, rows)):
        r = x[part].double() + res[part].double()
        exact[i] = r, r * (r.square().mean(1, keepdim=True) + 1e-6).rsqrt() * w.double()
    with torch.no_grad():
        y, total = kv.rms_norm(x, w, residual=res)
    for i, part in enumerate(around(seam, rows)):
        r, want = exact[i]
        assert torch.equal(total[part], x[part] + res[part])
        # float16's rounding and a few of float32's; below its normal range a fixed step
        assert ((y[part].double() - want).abs() <= (2.0 ** -11 + 40 * UNIT) * want.abs() + 2.0 ** -25).all()
    del y, total
    with torch.no_grad():
        q, scale, total = kv.rms_norm_quantized(x, w, residual=res)
    for i, part in enumerate(around(seam, rows)):
        r, want = exact[i]
        assert torch.equal(total[part], x[part] + res[part])
        s = (want.abs().amax(1) / 448).clamp(min=2.0 ** -126)
        assert ((scale[part].double() - s).abs() <= 40 * UNIT * s).all()
        t = want / s[:, None]
        assert ((q[part].double() - t).abs() <= (2.0 ** -4 + 80 * UNIT) * t.abs() + 2.0 ** -10 * (1 + 80 * UNIT)).all()
    del q, scale, total
    q, scale = kv.quantize_rows(x)
    for part in around(seam, rows):
        s = (x[part].double().abs().amax(1) / 448).clamp(min=2.0 ** -126)
        assert ((scale[part].double() - s).abs() <= 4 * UNIT * s).all()
        t = x[part].double() / s[:, None]
        assert ((q[part].double() - t).abs() <= (2.0 ** -4 + 8 * UNIT) * t.abs() + 2.0 ** -10 * (1 + 8 * UNIT)).all()


def test_norm_training_and_single_columns():
    """The backward pass walks over its rows in one launch; rstd comes from both of the forward pass's."""
    seam = 1 << 29
    rows = seam + 1003
    x = torch.empty(rows, 1, dtype=torch.float16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(3))
    x.abs_().requires_grad_(True)
    w = torch.tensor([1.5], device="cuda", requires_grad=True)
    y = kv.rms_norm(x, w)
    dy = torch.ones_like(y)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    total = 0.0
    for first in range(0, rows, 1 << 26):
        r = x.detach()[first:first + (1 << 26)].double()
        total += float((r / (r.square() + 1e-6).sqrt()).sum())
    # each of 1024 workgroups takes 64 rows at a time, so a lane adds some 2^13 terms between 0 and 1 in float32: at
    # most 2^13 roundings of 2^-24 of at most 2^13; the sums of lanes and workgroups add a few units of the whole
    assert abs(float(dw) - total) <= rows * 2.0 ** -11 + total * 64 * UNIT
    for part in around(seam, rows)[:2] + [slice(rows - 1003, rows)]:
        r = x.detach()[part].double()
        s = (r.square() + 1e-6).rsqrt()
        want = 1.5 * s * (1 - r * r * s * s)                       # = 1.5 s^3 1e-6, what the two terms leave
        # float32's roundings of the two terms, whose difference this is, and float16's of the result
        assert ((dx[part].double() - want).abs() <= 16 * UNIT * 1.5 * s + 2.0 ** -11 * want.abs() + 2.0 ** -25).all()


def rows_of(M, K, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.randint(-3, 4, (M, K), generator=g, device="cuda", dtype=torch.int8)


@pytest.mark.parametrize("seam,N,K", [(65535 * 128, 16, 16), (65535 * 64, 16, 9)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_product(seam, N, K, dtype):
    """Small whole numbers: every sum is exact, and rounded once."""
    M = seam + 1077
    a, b = rows_of(M, K, 1), rows_of(N, K, 2)
    codes = lambda t: t.to(torch.float16).to(torch.float8_e4m3fn)  # noqa: E731
    sx = torch.ones(M, device="cuda")
    sx[seam:] = 2.0
    bias = torch.arange(N, device="cuda", dtype=torch.float32)
    y = kv.linear_8bit(codes(a), sx, codes(b), torch.ones(N, device="cuda"), bias=bias, dtype=dtype)
    for first in range(0, M, 1 << 21):
        part = slice(first, first + (1 << 21))
        want = (a[part].float() @ b.float().t().contiguous()) * sx[part, None] + bias
        assert torch.equal(y[part], want.to(dtype)), first
