"""The root-mean-square norm with the residual's addition (rms_norm, rms_norm_quantized,
quantize_rows) against its formulas in float64."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
UNIT = 2.0 ** -24
EPS = 1e-6
E4M3_MAX = 448.0


def half_step(dtype):
    return 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2


def tiny(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def roundings(D):
    # a row's sum: a lane adds at most 32 terms, then at most 6 exchanges and 16 wavefronts;
    # the mean, the root and the products a few more; every rounding is half an ulp = one unit
    return (min(D, 32) + 6 + 16 + 12) * UNIT


def check(got, want, err, what):
    bad = (got.double() - want).abs() > err + half_step(got.dtype) * (want.abs() + err) + tiny(got.dtype)
    assert not bad.any(), (what, int(bad.sum()), float(((got.double() - want).abs() / (err + tiny(got.dtype))).max()))


def make(rows, D, dtype, wdtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    return (n(rows, D).to(dtype), (2 * n(rows, D)).to(dtype), (1 + 0.3 * n(D)).to(wdtype), n(rows, D).to(dtype),
            n(rows, D).to(dtype))


def oracle(x, residual, w):
    r = x.double() + (residual.double() if residual is not None else 0.0)
    s = (r.square().mean(1, keepdim=True) + EPS).rsqrt()
    return r, s, r * s * w.double()


def run(x, residual, w, dy, dsum):
    import kalman_vae_amd as kv
    leaves = [t.detach().requires_grad_(True) for t in (x, w) + ((residual,) if residual is not None else ())]
    out = kv.rms_norm(leaves[0], leaves[1], residual=leaves[2] if residual is not None else None, eps=EPS)
    if residual is None:
        return (out.detach(), None) + torch.autograd.grad(out, leaves, dy) + (None,)
    return tuple(o.detach() for o in out) + torch.autograd.grad(out, leaves, (dy, dsum))


WIDTHS = [1, 2, 7, 63, 64, 65, 127, 128, 256, 257, 500, 513, 1000, 1025, 2048, 2049, 4099, 8192, 9001, 16384]


@pytest.mark.parametrize("D", WIDTHS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("wide_weight", [True, False])
@pytest.mark.parametrize("with_residual", [True, False])
def test_forward_and_backward(D, dtype, wide_weight, with_residual):
    """Widths around every change of lanes per row, odd ones among them."""
    rows = 37 if D < 3000 else 5
    x, residual, w, dy, dsum = make(rows, D, dtype, torch.float32 if wide_weight else dtype)
    residual, dsum = (residual, dsum) if with_residual else (None, None)
    y, total, dx, dw, dres = run(x, residual, w, dy, dsum)
    r, s, want = oracle(x, residual, w)
    k = roundings(D)
    check(y, want, k * want.abs(), "y")
    if with_residual:
        check(total, r, UNIT * r.abs(), "sum")
    # gradients (of the unrounded sum whatever the types)
    n, d = r * s, dy.double() * w.double()
    along, size = (d * n).mean(1, keepdim=True), (d * n).abs().mean(1, keepdim=True)
    grad = s * (d - n * along) + (dsum.double() if dsum is not None else 0.0)
    err = k * s * (d.abs() + 2 * n.abs() * size) + UNIT * grad.abs()
    check(dx, grad, err, "dx")
    if with_residual:
        assert torch.equal(dx, dres)
    terms = dy.double() * n
    check(dw, terms.sum(0), (k + rows * UNIT) * terms.abs().sum(0), "dw")
    again = run(x, residual, w, dy, dsum)
    assert all(a is None or torch.equal(a, b) for a, b in zip((y, total, dx, dw, dres), again))


@pytest.mark.parametrize("rows", [1, 15, 16, 17, 255, 5000, 40000])
def test_many_rows(rows):
    """The weight gradient's sum over workgroups, from one row to many."""
    D = 128
    x, residual, w, dy, dsum = make(rows, D, torch.float32, torch.float32)
    y, total, dx, dw, dres = run(x, residual, w, dy, dsum)
    r, s, want = oracle(x, residual, w)
    check(y, want, roundings(D) * want.abs(), "y")
    terms = dy.double() * r * s
    # every partial sum adds at most rows terms in order
    check(dw, terms.sum(0), (roundings(D) + min(rows, 64 + rows // 16) * UNIT) * terms.abs().sum(0), "dw")


@pytest.mark.parametrize("rows", [1, 63, 64, 65, 1000, 70001])
@pytest.mark.parametrize("D", [3, 16, 17, 20, 40, 64])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_narrow_rows(rows, D, dtype):
    """Several rows in a quarter wavefront: outputs, and the weight gradient's sum over them."""
    x, residual, w, dy, dsum = make(rows, D, dtype, torch.float32)
    y, total, dx, dw, dres = run(x, residual, w, dy, dsum)
    r, s, want = oracle(x, residual, w)
    k = roundings(D)
    check(y, want, k * want.abs(), "y")
    n, d = r * s, dy.double() * w.double()
    along, size = (d * n).mean(1, keepdim=True), (d * n).abs().mean(1, keepdim=True)
    grad = s * (d - n * along) + dsum.double()
    check(dx, grad, k * s * (d.abs() + 2 * n.abs() * size) + UNIT * grad.abs(), "dx")
    terms = dy.double() * n
    check(dw, terms.sum(0), (k + min(rows, 64 + rows // 16) * UNIT) * terms.abs().sum(0), "dw")


def test_directional_derivative():
    x, residual, w, dy, dsum = make(9, 50, torch.float32, torch.float32)
    _, _, dx, dw, dres = run(x, residual, w, dy, dsum)
    g = torch.Generator(device="cuda").manual_seed(4)
    dirs = [torch.randn(t.shape, generator=g, device="cuda").double() for t in (x, residual, w)]
    h = 1e-5

    def loss(sign):
        a, b, c = (t.double() + sign * h * d for t, d in zip((x, residual, w), dirs))
        r, _, y = oracle(a, b, c)
        return (y * dy.double()).sum() + (r * dsum.double()).sum()

    diff = (loss(1) - loss(-1)) / (2 * h)
    terms = [(g_.double() * d) for g_, d in zip((dx, dres, dw), dirs)]
    assert abs(float(diff - sum(t.sum() for t in terms))) < 1e-5 * float(sum(t.abs().sum() for t in terms))


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_shapes(dtype):
    """Three axes, rows of a wider tensor at an odd offset, leading axes that do not merge, a
    broadcast row, expanded cotangents."""
    import kalman_vae_amd as kv
    x, residual, w, dy, dsum = make(24, 33, dtype, dtype)
    want = run(x, residual, w, dy, dsum)
    pad = lambda t: torch.cat([torch.full((24, 1), 7.0, device="cuda", dtype=dtype), t, t[:, :2]], 1)[:, 1:34]  # noqa: E731
    got = run(pad(x), pad(residual), w, pad(dy), pad(dsum))
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    x3, r3 = (t.view(4, 6, 33).transpose(0, 1).contiguous().transpose(0, 1) for t in (x, residual))
    y, total = kv.rms_norm(x3, w, residual=r3, eps=EPS)
    assert y.shape == (4, 6, 33) and torch.equal(y.reshape(24, 33), want[0])
    assert torch.equal(total.reshape(24, 33), want[1])
    one = kv.rms_norm(x[3], w, eps=EPS)
    assert torch.equal(one, kv.rms_norm(x[3:4].expand(5, 33), w, eps=EPS)[2])
    v = x.clone().requires_grad_(True)
    a = torch.autograd.grad(kv.rms_norm(v, w, eps=EPS).sum(), v)[0]
    b = torch.autograd.grad(kv.rms_norm(v, w, eps=EPS), v, torch.ones_like(v))[0]
    assert torch.equal(a, b)
    # only the sum's cotangent: it passes through
    y, total = kv.rms_norm(v, w, residual=residual, eps=EPS)
    assert torch.equal(torch.autograd.grad(total, v, dsum)[0], dsum)


def test_zero_and_non_finite_rows():
    import kalman_vae_amd as kv
    x = torch.randn(4, 40, device="cuda")
    w = torch.ones(40, device="cuda")
    x[1] = 0
    x[2, 5] = float("nan")
    x[3] = 1e-30
    y = kv.rms_norm(x, w, eps=EPS)
    assert not y[1].any() and torch.isnan(y[2]).all() and torch.isfinite(y[[0, 1, 3]]).all()
    q, scale = kv.rms_norm_quantized(x, w, eps=EPS)
    assert torch.isfinite(scale).all() and not q[1].float().any() and torch.isnan(q[2].float()).all()
    assert float(scale[1]) == 2.0 ** -126
    x[2] = 1
    x[2, 5] = float("nan")
    q, scale = kv.quantize_rows(x)              # the row's other values keep their scale
    assert torch.isnan(q[2, 5].float()) and abs(float(scale[2]) * 448 - 1) < 1e-6
    assert (q[2].float() == 448).sum() == 39


def nearest_e4m3(t):
    """t (float64, |t| <= 448) to the nearest e4m3 value, ties to even."""
    power = torch.floor(torch.log2(t.abs().clamp_min(2.0 ** -30))).clamp_min(-6)
    quantum = torch.exp2(power - 3)
    return torch.round(t / quantum) * quantum


@pytest.mark.parametrize("D", [1, 2, 7, 16, 64, 65, 128, 300, 513, 1025, 2048, 4099, 9001, 16384])
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantized(D, dtype):
    import kalman_vae_amd as kv
    rows = 19
    x, residual, w, _, _ = make(rows, D, dtype, torch.float32)
    q, scale, total = kv.rms_norm_quantized(x, w, residual=residual, eps=EPS)
    r, s, y = oracle(x, residual, w)
    k = roundings(D)
    amax = y.abs().amax(1)
    assert ((scale.double() - amax / E4M3_MAX).abs() <= (k + 4 * UNIT) * amax / E4M3_MAX).all()
    check(total, r, UNIT * r.abs(), "sum")
    # the code is the nearest to y / scale, up to the error of that quotient
    t, got = y / scale.double()[:, None], q.double()
    slack = (2 * k + 4 * UNIT) * t.abs()
    low, high = nearest_e4m3((t - slack).clamp(-E4M3_MAX, E4M3_MAX)), nearest_e4m3((t + slack).clamp(-E4M3_MAX, E4M3_MAX))
    assert ((got >= low) & (got <= high)).all()
    q2, s2 = kv.quantize_rows(x)
    amax = x.double().abs().amax(1)
    assert ((s2.double() - amax / E4M3_MAX).abs() <= 4 * UNIT * amax / E4M3_MAX).all()
    t, slack = x.double() / s2.double()[:, None], 4 * UNIT * (x.double() / s2.double()[:, None]).abs()
    low, high = nearest_e4m3((t - slack).clamp(-E4M3_MAX, E4M3_MAX)), nearest_e4m3((t + slack).clamp(-E4M3_MAX, E4M3_MAX))
    assert ((q2.double() >= low) & (q2.double() <= high)).all()


@pytest.mark.parametrize("D", [24, 256, 1500])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_codes_are_those_of_the_quotient(D, dtype):
    """y / scale = 448 r w / max |r w|: the codes are this quotient's, rounded to float and then to e4m3,
    every one of them, as the kernel carries products to twice float's digits.  (Inputs on a grid on which
    x + residual is exact, and r w is exact in float64.)"""
    import kalman_vae_amd as kv
    rows = 2_000_000 // D
    x, residual, w, _, _ = make(rows, D, dtype, torch.float32, seed=D)
    x, residual = ((t.float() * 32).round().div(32).to(dtype) for t in (x, residual))
    q = kv.rms_norm_quantized(x, w, residual=residual, eps=EPS)[0]
    p = (x.double() + residual.double()) * w.double()
    t = p * (E4M3_MAX / p.abs().amax(1, keepdim=True))
    assert torch.equal(q.double(), nearest_e4m3(t.float().double()))


def test_empty():
    import kalman_vae_amd as kv
    w = torch.ones(5, device="cuda", requires_grad=True)
    x = torch.zeros(0, 5, device="cuda", requires_grad=True)
    y, r = kv.rms_norm(x, w, residual=x.detach())
    y.sum().backward()
    assert y.shape == r.shape == x.grad.shape == (0, 5) and not w.grad.any()
    with torch.no_grad():
        q, s = kv.rms_norm_quantized(x, w)
        assert q.shape == (0, 5) and s.shape == (0,)
        q, s = kv.quantize_rows(torch.zeros(3, 0, device="cuda"))
        assert q.shape == (3, 0) and s.shape == (3,)


def test_captured_step_equals_the_eager_one():
    import kalman_vae_amd as kv
    x, residual, w, dy, dsum = make(1000, 65, torch.float32, torch.float32)
    static = [t.clone().requires_grad_(True) for t in (x, residual, w)]

    def step():
        y, r = kv.rms_norm(static[0], static[2], residual=static[1], eps=EPS)
        dx, dres, dw = torch.autograd.grad((y, r), static, (dy, dsum))
        with torch.no_grad():
            q, s, _ = kv.rms_norm_quantized(static[0], static[2], residual=static[1], eps=EPS)
        return y, r, dx, dw, dres, q, s

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step()
    for k in range(4):
        v, res, ww, _, _ = make(1000, 65, torch.float32, torch.float32, seed=k)
        with torch.no_grad():
            for s, t in zip(static, (v, res, ww)):
                s.copy_(t)
        graph.replay()
        want = run(v, res, ww, dy, dsum)
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k
        with torch.no_grad():
            q, s, _ = kv.rms_norm_quantized(v, ww, residual=res, eps=EPS)
        assert torch.equal(out[5].view(torch.uint8), q.view(torch.uint8)) and torch.equal(out[6], s)
