"""The gated linear recurrence (gated_scan, gated_scan_step) against its definition, step by step in
float64, with error bounds that follow the recurrence: every step adds a few roundings and passes
the error before it on with the gate's weight.  The kernels also compose stretches of steps (P, S)
and apply them to a start state, so a rounding is charged with the size of the terms in the state,
sum of |f ... f keep x|, and not with the state, in which they may cancel: for any grouping of the
steps each term passes at most one product and one sum per step."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
UNIT = 2.0 ** -24
# float32 roundings charged to each step: products, sum, reciprocal (1 ulp = 2 units), exponential
# (2 ulp; its argument, |z| <= 10, is rounded once: up to 10 units of the exponential)
STEP = 32 * UNIT


def half_step(dtype):
    return 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2


def oracle(u, h0, mask, gated, dy=None, dlast=None):
    """Values and error bounds in float64: dicts with y, last (and du, dh0)."""
    T, B, W = u.shape
    H = W // (3 if gated else 2)
    dtype, u = u.dtype, u.double()
    x, z = u[..., :H], u[..., H:2 * H]
    f, keep = torch.sigmoid(z), torch.sigmoid(-z)
    o = u[..., 2 * H:] if gated else None
    silu = o * torch.sigmoid(o) if gated else torch.ones_like(x)
    live = torch.ones(T, B, dtype=torch.bool, device=u.device) if mask is None else mask != 0
    c = torch.zeros(B, H, dtype=torch.float64, device=u.device) if h0 is None else h0.double()
    e, size = torch.zeros_like(c), c.abs()
    before, after, eafter, ebefore = [], [], [], []
    for t in range(T):
        on = live[t][:, None]
        before.append(c)
        ebefore.append(e)
        new, grown = f[t] * c + keep[t] * x[t], f[t] * size + (keep[t] * x[t]).abs()
        c, e = torch.where(on, new, c), torch.where(on, f[t] * e + STEP * grown, e)
        size = torch.where(on, grown, size)
        after.append(c)
        eafter.append(e)
    on = live[..., None]
    after, eafter, before, ebefore = (torch.stack(v) for v in (after, eafter, before, ebefore))
    y = torch.where(on, after * silu, 0.0)
    ey = torch.where(on, eafter * silu.abs() + STEP * y.abs(), 0.0)
    out, err = {"y": y, "last": c}, {"y": ey + half_step(dtype) * (y.abs() + ey), "last": e}
    if dy is None:
        return out, err
    dy = torch.where(on, dy.double(), 0.0)
    G = torch.zeros_like(c) if dlast is None else dlast.double()
    eG, sG = torch.zeros_like(G), G.abs()
    du, edu = torch.zeros_like(u), torch.zeros_like(u)
    for t in reversed(range(T)):
        add = dy[t] * silu[t]
        sG = sG + add.abs()
        tot, etot = G + add, eG + STEP * sG
        m = live[t][:, None]
        du[t, :, :H] = torch.where(m, keep[t] * tot, 0.0)
        edu[t, :, :H] = torch.where(m, keep[t] * etot + STEP * (keep[t] * tot).abs(), 0.0)
        w, diff = f[t] * keep[t], before[t] - x[t]
        du[t, :, H:2 * H] = torch.where(m, w * diff * tot, 0.0)
        size = before[t].abs() + x[t].abs()
        edu[t, :, H:2 * H] = torch.where(
            m, w * (diff.abs() * etot + ebefore[t] * (tot.abs() + etot) + STEP * size * tot.abs()), 0.0)
        if gated:
            s = torch.sigmoid(o[t])
            slope = s * (1 + o[t] * torch.sigmoid(-o[t]))
            rough = s * (1 + o[t].abs() * torch.sigmoid(-o[t]))
            du[t, :, 2 * H:] = dy[t] * after[t] * slope
            edu[t, :, 2 * H:] = dy[t].abs() * (eafter[t] * slope.abs() + STEP * after[t].abs() * rough)
        G = torch.where(m, f[t] * tot, G)
        eG = torch.where(m, f[t] * etot + STEP * f[t] * sG, eG)
        sG = torch.where(m, f[t] * sG, sG)
    out.update(du=du, dh0=G)
    err.update(du=edu + half_step(dtype) * (du.abs() + edu), dh0=eG)
    return out, err


def smallest(dtype):
    # results below the type's smallest normal number are rounded to a fixed step
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def compare(got, want, err, what):
    tiny = smallest(got.dtype)
    assert torch.isfinite(got.float()).all(), what
    bad = (got.double() - want).abs() > err + tiny
    assert not bad.any(), (what, int(bad.sum()), float(((got.double() - want).abs() / (err + tiny)).max()))


def make(T, B, H, dtype, gated, seed=0, masked=False, with_h0=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    u = torch.randn(T, B, (3 if gated else 2) * H, generator=g, device="cuda")
    u[..., H:2 * H] = 2 * u[..., H:2 * H] + 1
    mask = None
    if masked:
        mask = torch.rand(T, B, generator=g, device="cuda") < 0.7
        mask[:, 0] = False                       # a sequence without any step
    h0 = torch.randn(B, H, generator=g, device="cuda") if with_h0 else None
    dy = torch.randn(T, B, H, generator=g, device="cuda").to(dtype)
    dlast = torch.randn(B, H, generator=g, device="cuda")
    return u.to(dtype).clamp(-10, 10), h0, mask, dy, dlast


def run(u, h0, mask, gated, dy, dlast):
    import kalman_vae_amd as kv
    u = u.detach().requires_grad_(True)
    h0 = h0.detach().requires_grad_(True) if h0 is not None else None
    y, last = kv.gated_scan(u, h0, mask=mask, output_gate=gated)
    leaves = [u] if h0 is None else [u, h0]
    grads = torch.autograd.grad((y, last), leaves, (dy, dlast))
    return {"y": y.detach(), "last": last.detach(), "du": grads[0], "dh0": grads[1] if h0 is not None else None}


@pytest.mark.parametrize("T,B,H", [(1, 1, 1), (1, 5, 7), (2, 3, 2), (15, 2, 3), (16, 2, 64), (17, 3, 65),
                                   (20, 33, 128), (33, 1, 129), (64, 2, 5), (100, 3, 31), (1000, 2, 16),
                                   (4097, 1, 3), (300, 40, 128), (5000, 1, 70)])
@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("dtype", DTYPES)
def test_forward_and_backward(T, B, H, gated, dtype):
    """Lengths around the chunks of 8 and 16 steps and the workgroup's 64 and 128, odd widths, and
    lengths that are cut into segments."""
    u, h0, mask, dy, dlast = make(T, B, H, dtype, gated, masked=B > 1, with_h0=T % 2 == 1)
    got = run(u, h0, mask, gated, dy, dlast)
    want, err = oracle(u, h0, mask, gated, dy, dlast)
    for k, v in got.items():
        if v is not None:
            compare(v, want[k], err[k], k)
    import kalman_vae_amd as kv
    with torch.no_grad():                        # without a gradient: the same bits
        y, last = kv.gated_scan(u, h0, mask=mask, output_gate=gated)
    assert torch.equal(y, got["y"]) and torch.equal(last, got["last"])
    again = run(u, h0, mask, gated, dy, dlast)
    assert all(v is None or torch.equal(v, again[k]) for k, v in got.items())


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_sequences(dtype):
    """Enough channels that the time axis stays whole."""
    u, h0, mask, dy, dlast = make(20, 2100, 129, dtype, True, masked=True, with_h0=True)
    got = run(u, h0, mask, True, dy, dlast)
    want, err = oracle(u, h0, mask, True, dy, dlast)
    for k, v in got.items():
        compare(v, want[k], err[k], k)


def test_directional_derivative():
    """du and dh0 against central differences of the definition in float64."""
    u, h0, mask, dy, dlast = make(40, 3, 20, torch.float32, True, masked=True, with_h0=True)
    got = run(u, h0, mask, True, dy, dlast)
    g = torch.Generator(device="cuda").manual_seed(9)
    ud = torch.randn(u.shape, generator=g, device="cuda").double()
    hd = torch.randn(h0.shape, generator=g, device="cuda").double()
    step = 1e-5

    def loss(sign):
        out, _ = oracle(u.double() + sign * step * ud, h0.double() + sign * step * hd, mask, True)
        return (out["y"] * dy.double()).sum() + (out["last"] * dlast.double()).sum()

    # the float64 oracle's own type: bounds are not used here
    diff = (loss(1) - loss(-1)) / (2 * step)
    along = (got["du"].double() * ud).sum() + (got["dh0"].double() * hd).sum()
    size = (got["du"].double() * ud).abs().sum() + (got["dh0"].double() * hd).abs().sum()
    # float32 gradients: a few hundred roundings of each term; the differences' own error is step^2
    assert abs(float(diff - along)) < 1e-5 * float(size)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(dtype):
    """A batch-first tensor transposed, a slice of a wider tensor at an odd offset, a reversed mask's
    transpose, expanded cotangents: the same bits as from contiguous tensors."""
    T, B, H = 37, 4, 33
    u, h0, mask, dy, dlast = make(T, B, H, dtype, True, masked=True, with_h0=True)
    want = run(u, h0, mask, True, dy, dlast)
    wide = torch.full((B, T, 3 * H + 5), float("nan"), dtype=dtype, device="cuda")
    view = wide[:, :, 1:3 * H + 1].transpose(0, 1)
    view.copy_(u)
    mview = mask.t().contiguous().t()
    dview = dy.transpose(0, 1).contiguous().transpose(0, 1)
    got = run(view, h0.t().contiguous().t(), mview, True, dview, dlast.t().contiguous().t())
    assert all(torch.equal(v, got[k]) for k, v in want.items())
    one = torch.ones((), dtype=dtype, device="cuda").expand(T, B, H)
    a, b = (run(u, h0, mask, True, d, torch.ones_like(dlast)) for d in (one, one.contiguous()))
    assert all(torch.equal(v, b[k]) for k, v in a.items())
    same = u[:1].expand(T, B, 3 * H)              # one step's input broadcast over time
    a, b = (run(v, h0, mask, True, dy, dlast) for v in (same, same.contiguous()))
    assert all(torch.equal(v, b[k]) for k, v in a.items())


def test_masked_places_are_not_read_as_numbers():
    """NaN and infinities where the mask is zero change nothing; masks of any type."""
    u, h0, mask, dy, dlast = make(50, 6, 17, torch.float32, True, masked=True, with_h0=True)
    want = run(u, h0, mask, True, dy, dlast)
    dirty, ddirty = u.clone(), dy.clone()
    dirty[~mask] = float("nan")
    dirty[3][~mask[3]] = float("inf")
    ddirty[~mask] = float("nan")
    for m in (mask, mask.to(torch.uint8) * 3, mask.float() * 0.5, mask.double(), mask.long()):
        got = run(dirty, h0, m, True, ddirty, dlast)
        assert all(torch.equal(v, got[k]) for k, v in want.items())
    assert torch.equal(got["last"][0], h0[0]) and torch.equal(got["dh0"][0], dlast[0])
    assert not got["y"][:, 0].any() and not got["du"][:, 0].any()


def test_saturated_gates():
    """Gates far outside the exponential's range: the state is kept or replaced, without NaN."""
    H = 8
    u = torch.zeros(3, 1, 3 * H, device="cuda")
    u[..., :H] = 2.0
    u[..., H:2 * H] = torch.tensor([200.0, -200.0, 3e38, -3e38, 88.0, -88.0, 0.0, 1.0], device="cuda")
    u[..., 2 * H:] = 300.0
    h0 = torch.ones(1, H, device="cuda")
    got = run(u, h0, None, True, torch.ones(3, 1, H, device="cuda"), torch.ones(1, H, device="cuda"))
    assert all(torch.isfinite(v).all() for v in got.values())
    assert torch.equal(got["last"][0, :4].cpu(), torch.tensor([1.0, 2.0, 1.0, 2.0]))


def test_only_one_cotangent_and_partial_needs():
    import kalman_vae_amd as kv
    u, h0, mask, dy, dlast = make(33, 2, 9, torch.float32, True, with_h0=True)
    zero_y, zero_l = torch.zeros_like(dy), torch.zeros_like(dlast)
    v = u.clone().requires_grad_(True)
    y, last = kv.gated_scan(v, h0)
    assert torch.equal(torch.autograd.grad(y, v, dy)[0], run(u, h0, None, True, dy, zero_l)["du"])
    y, last = kv.gated_scan(v, h0)
    assert torch.equal(torch.autograd.grad(last, v, dlast)[0], run(u, h0, None, True, zero_y, dlast)["du"])
    w = h0.clone().requires_grad_(True)
    y, last = kv.gated_scan(u, w)
    assert torch.equal(torch.autograd.grad((y, last), w, (dy, dlast))[0], run(u, h0, None, True, dy, dlast)["dh0"])
    # an initial state shared by all sequences: the gradient of the broadcast input is the sum
    shared = h0[:1].clone().requires_grad_(True)
    y, last = kv.gated_scan(u, shared.expand(2, 9))
    got = torch.autograd.grad((y, last), shared, (dy, dlast))[0]
    full = run(u, h0[:1].expand(2, 9).contiguous(), None, True, dy, dlast)["dh0"]
    assert torch.equal(got, full.sum(0, keepdim=True))


def test_pieces_equal_the_whole():
    """A sequence fed in pieces, the state carried on, and one step at a time: each within the bound
    of the definition, so within twice that of each other (the steps are grouped differently)."""
    import kalman_vae_amd as kv
    u, h0, mask, _, _ = make(50, 5, 33, torch.float32, True, masked=True, with_h0=True)
    want, err = oracle(u, h0, mask, True)
    with torch.no_grad():
        a, s = kv.gated_scan(u[:21], h0, mask=mask[:21])
        b, s = kv.gated_scan(u[21:], s, mask=mask[21:])
        compare(torch.cat([a, b]), want["y"], err["y"], "pieces")
        compare(s, want["last"], err["last"], "pieces' state")
        s = h0.clone()
        steps = torch.stack([kv.gated_scan_step(u[t], s, mask=mask[t]) for t in range(50)])
    compare(steps, want["y"], err["y"], "steps")
    compare(s, want["last"], err["last"], "steps' state")


@pytest.mark.parametrize("B,H", [(1, 1), (3, 2), (5, 7), (64, 128), (1000, 33)])
@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("dtype", DTYPES)
def test_step(B, H, gated, dtype):
    import kalman_vae_amd as kv
    u, h0, mask, _, _ = make(1, B, H, dtype, gated, masked=True, with_h0=True)
    want, err = oracle(u, h0, mask, gated)
    wide = torch.zeros(B, u.shape[2] + 3, dtype=dtype, device="cuda")
    wide[:, 1:-2] = u[0]
    for v in (u[0], wide[:, 1:-2]):
        s = h0.clone()
        y = kv.gated_scan_step(v, s, mask=mask[0], output_gate=gated)
        compare(y, want["y"][0], err["y"][0], "y")
        compare(s, want["last"], err["last"], "state")


def test_empty():
    import kalman_vae_amd as kv
    h0 = torch.randn(3, 4, device="cuda")
    for shape, first in (((0, 3, 12), h0), ((0, 3, 12), None), ((5, 0, 12), None), ((5, 3, 0), None)):
        u = torch.zeros(shape, device="cuda", requires_grad=True)
        y, last = kv.gated_scan(u, first)
        assert y.shape == (shape[0], shape[1], shape[2] // 3) and last.shape == (shape[1], shape[2] // 3)
        assert torch.equal(last, first if first is not None else torch.zeros_like(last))
        y.sum().backward()
        assert u.grad.shape == u.shape
    with torch.no_grad():
        assert kv.gated_scan_step(torch.zeros(0, 12, device="cuda"), torch.zeros(0, 4, device="cuda")).shape == (0, 4)


def test_captured_step_equals_the_eager_one():
    """Forward and backward in a captured graph (segmented time axis: workspaces included), replayed
    several times with eager calls between, on new inputs each time."""
    import kalman_vae_amd as kv
    u, h0, mask, dy, dlast = make(200, 2, 65, torch.bfloat16, True, masked=True, with_h0=True)
    static = [t.clone() for t in (u, h0)]
    static[0].requires_grad_(True)
    static[1].requires_grad_(True)

    def step():
        y, last = kv.gated_scan(static[0], static[1], mask=mask)
        return (y, last) + torch.autograd.grad((y, last), static, (dy, dlast))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step()
        graphs.append((graph, out))
    for k in range(4):
        v, h = make(200, 2, 65, torch.bfloat16, True, seed=k, with_h0=True)[:2]
        with torch.no_grad():
            static[0].copy_(v)
            static[1].copy_(h)
        for graph, _ in graphs:
            graph.replay()
        want = run(v, h, mask, True, dy, dlast)
        for _, out in graphs:
            for got, key in zip(out, ("y", "last", "du", "dh0")):
                assert torch.equal(got, want[key]), (k, key)


def test_another_stream():
    u, h0, mask, dy, dlast = make(300, 3, 40, torch.float32, True, with_h0=True)
    want = run(u, h0, None, True, dy, dlast)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(u, h0, None, True, dy, dlast)
    side.synchronize()
    assert all(torch.equal(v, got[k]) for k, v in want.items())


def test_offsets_beyond_32_bits():
    """u of more than 2^32 bytes reached through a stride: a few steps far apart in one tensor."""
    import kalman_vae_amd as kv
    T, B, H = 3, 2, 16
    big = torch.empty(1_200_000_000, dtype=torch.bfloat16, device="cuda")
    stride = 1_199_990_000 // 2                  # elements between steps: over 2^31 bytes each
    u, h0, _, _, _ = make(T, B, H, torch.bfloat16, True, with_h0=True)
    view = big.as_strided((T, B, 3 * H), (stride, 3 * H, 1))
    view.copy_(u)
    with torch.no_grad():
        a, b = kv.gated_scan(view, h0), kv.gated_scan(u, h0)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
