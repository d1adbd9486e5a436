"""The sequence-network operators and the optimiser where a launch's own limits lie (threads of one
launch, 32-bit lane offsets), on two streams at once, and differentiated twice."""
import pytest
import torch

import kalman_vae_amd as kv
from kalman_vae_amd.optim import adamw_step, state_blocks

pytestmark = pytest.mark.gpu

UNIT = 2.0 ** -24


def randn(*shape, seed, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


@pytest.mark.parametrize("wide", ["u", "mask", "dy"])
def test_batch_strides_of_gigabytes(wide):
    """Sequences whose places in a tensor span more than 32-bit lane offsets reach (float32: 2^29
    elements, mask: 2^31 bytes): the same bits as from dense tensors."""
    T, B, H = 40, 3, 4
    u, dy, h0 = randn(T, B, 3 * H, seed=1), randn(T, B, H, seed=2), randn(B, H, seed=3)
    mask = (torch.arange(T * B, device="cuda").view(T, B) % 5 != 0).to(torch.uint8)

    def run(u, mask, dy):
        u = u.detach().requires_grad_(True)
        h = h0.clone().requires_grad_(True)
        y, last = kv.gated_scan(u, h, mask=mask)
        return (y.detach(), last.detach()) + torch.autograd.grad((y, last), (u, h), (dy, torch.ones_like(last)))

    want = run(u, mask, dy)
    spread = {"u": u, "mask": mask, "dy": dy}
    t = spread[wide]
    apart = ((1 << 31) // t.element_size()) // 2 + 7      # two strides: more than 2^31 bytes
    memory = torch.empty(apart * (B - 1) + T * t.shape[-1], dtype=t.dtype, device="cuda")
    spread[wide] = memory.as_strided(t.shape, (t.shape[-1], apart) + ((1,) if t.dim() == 3 else ()))
    if t.dim() == 2:
        spread[wide] = memory.as_strided(t.shape, (1, apart))
    spread[wide].copy_(t)
    got = run(**spread)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_norm_of_more_rows_than_a_launch_has_threads():
    """2^27 rows fill the threads of one launch (16 lanes each); the rows behind go in another."""
    rows, D = (1 << 27) + 100_003, 2
    x = torch.empty(rows, D, dtype=torch.float16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(4))
    w = torch.tensor([0.5, -2.0], device="cuda")
    with torch.no_grad():
        y, total = kv.rms_norm(x, w, residual=x)
        q, scale = kv.quantize_rows(x)
    for first in [*range(0, rows, 1 << 24), (1 << 27) - 500]:
        part = slice(first, first + (1 << 24))
        r = 2 * x[part].double()
        want = r * (r.square().mean(1, keepdim=True) + 1e-6).rsqrt() * w.double()
        # float16's rounding and a few of float32's; below its normal range a fixed step
        assert ((y[part].double() - want).abs() <= (2.0 ** -11 + 40 * UNIT) * want.abs() + 2.0 ** -25).all()
        assert torch.equal(total[part], x[part] + x[part])
        amax = x[part].double().abs().amax(1)
        assert ((scale[part].double() - (amax / 448).clamp(min=2.0 ** -126)).abs() <= 4 * UNIT * amax / 448).all()
        # half a step of three mantissa bits (and the quotient's roundings); below 2^-6 half of 2^-9
        back, t = q[part].double(), x[part].double() / scale[part].double()[:, None]
        assert ((back - t).abs() <= (2.0 ** -4 + 8 * UNIT) * t.abs() + 2.0 ** -10 * (1 + 8 * UNIT)).all()


def test_two_streams_at_once():
    """Every operator on two streams without a wait between them, each on its own tensors: what the
    calls give one after the other."""
    def work(seed, steps):
        u = randn(300, 5, 3 * 64, seed=seed, dtype=torch.bfloat16).requires_grad_(True)
        x, w = randn(2000, 256, seed=seed + 1).requires_grad_(True), randn(256, seed=seed + 2).requires_grad_(True)
        rows, weight = randn(500, 256, seed=seed + 3), randn(384, 256, seed=seed + 4)
        p, g = randn(30_000, seed=seed + 5), randn(30_000, seed=seed + 6)
        m = [(torch.zeros(30_000, device="cuda", dtype=torch.float8_e4m3fn), torch.zeros(state_blocks(30_000), device="cuda"))
             for _ in range(2)]
        state = torch.zeros(5, 64, device="cuda")

        def go():
            out = []
            for k in range(steps):
                y, last = kv.gated_scan(u)
                out += [y, last, *torch.autograd.grad((y, last), u, (torch.ones_like(y), torch.ones_like(last)))]
                n = kv.rms_norm(x, w)
                out += [n, *torch.autograd.grad(n, (x, w), torch.ones_like(n))]
                with torch.no_grad():
                    q, wq = kv.rms_norm_quantized(rows, w), kv.quantize_rows(weight)
                    out += [kv.linear_8bit(*q, *wq, dtype=d) for d in (torch.float32, torch.bfloat16)]
                    out.append(kv.gated_scan_step(u[k], state))
                    adamw_step([p], [g], [m[0]], [m[1]], k + 1, lr=1e-2)
            return [t.detach() for t in out] + [p, state, m[0][0].view(torch.uint8), m[1][0].view(torch.uint8)]
        return go

    want = [[t.clone() for t in work(seed, 3)()] for seed in (10, 20)]
    torch.cuda.synchronize()
    calls = [work(seed, 3) for seed in (10, 20)]
    streams = [torch.cuda.Stream() for _ in calls]
    got = []
    for call, stream in zip(calls, streams):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            got.append(call())
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert len(a) == len(b) and all(torch.equal(s, t) for s, t in zip(a, b))


def test_second_derivatives_are_refused():
    """The first derivative may be asked for with create_graph; going on from it raises."""
    u = randn(5, 2, 12, seed=1).requires_grad_(True)
    x, w, r = (randn(*s, seed=2).requires_grad_(True) for s in ((4, 8), (8,), (4, 8)))
    for out, leaves in ((kv.gated_scan(u), [u]), (kv.rms_norm(x, w, residual=r), [x, w, r])):
        plain = torch.autograd.grad(sum(o.square().sum() for o in out), leaves, retain_graph=True)
        grads = torch.autograd.grad(sum(o.square().sum() for o in out), leaves, create_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(plain, grads))
        again = sum(g.sum() for g in grads)
        for ask in (lambda: torch.autograd.grad(again, leaves, retain_graph=True),
                    lambda: torch.autograd.grad(again, leaves, retain_graph=True, allow_unused=True), again.backward):
            with pytest.raises(RuntimeError, match="differentiable once"):
                ask()


def test_backward_twice_through_one_graph():
    u = randn(50, 3, 12, seed=1).requires_grad_(True)
    y, last = kv.gated_scan(u)
    first, second = (torch.autograd.grad(y.sum() + last.sum(), u, retain_graph=True)[0] for _ in range(2))
    assert torch.equal(first, second)
    with torch.no_grad():
        u.add_(1.0)                                # what was saved is stale: autograd says so
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_gradients_that_one_leaf_shares():
    """x as its own residual, and the sum going into two consumers: both gradients arrive, apart."""
    x, w = randn(6, 16, seed=1).requires_grad_(True), randn(16, seed=2).requires_grad_(True)
    y, r = kv.rms_norm(x, w, residual=x)
    (y.sum() + r.sum()).backward()
    a, b = x.detach().clone().requires_grad_(True), x.detach().clone().requires_grad_(True)
    y2, r2 = kv.rms_norm(a, w.detach(), residual=b)
    (y2.sum() + r2.sum()).backward()
    assert torch.equal(a.grad, b.grad) and a.grad.data_ptr() != b.grad.data_ptr()
    assert torch.equal(x.grad, a.grad + b.grad)
