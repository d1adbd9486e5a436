"""Tensors that carry a tangent of torch.autograd.forward_ad: the operators have no forward-mode
derivative, and a call that went through would answer without one."""
import pytest
import torch
import torch.autograd.forward_ad as fw

import kalman_vae_amd as kv

E4M3 = torch.float8_e4m3fn


def calls(device, dual):
    """Every operator with a tangent on each of its inputs in turn: (name, call)."""
    z = lambda *s: torch.ones(s, device=device)  # noqa: E731
    e = lambda *s: torch.ones(s, device=device).to(E4M3)  # noqa: E731
    d = lambda *s: dual(z(*s))  # noqa: E731
    state = lambda: [[z(4)], [z(4)]]  # noqa: E731
    return [
        ("scan u", lambda: kv.gated_scan(d(3, 2, 12))), ("scan h0", lambda: kv.gated_scan(z(3, 2, 12), d(2, 4))),
        ("step u", lambda: kv.gated_scan_step(d(2, 12), z(2, 4))), ("step state", lambda: kv.gated_scan_step(z(2, 12), d(2, 4))),
        ("norm x", lambda: kv.rms_norm(d(3, 4), z(4))), ("norm weight", lambda: kv.rms_norm(z(3, 4), d(4))),
        ("norm residual", lambda: kv.rms_norm(z(3, 4), z(4), residual=d(3, 4))),
        ("norm to 8 bits x", lambda: kv.rms_norm_quantized(d(3, 4), z(4))),
        ("norm to 8 bits weight", lambda: kv.rms_norm_quantized(z(3, 4), d(4))),
        ("norm to 8 bits residual", lambda: kv.rms_norm_quantized(z(3, 4), z(4), residual=d(3, 4))),
        ("rows", lambda: kv.quantize_rows(d(3, 4))),
        ("product x_scale", lambda: kv.linear_8bit(e(3, 4), d(3), e(5, 4), z(5))),
        ("product weight_scale", lambda: kv.linear_8bit(e(3, 4), z(3), e(5, 4), d(5))),
        ("product bias", lambda: kv.linear_8bit(e(3, 4), z(3), e(5, 4), z(5), bias=d(5))),
        ("update parameter", lambda: kv.adamw_step([d(4)], [z(4)], *state(), 1)),
        ("update gradient", lambda: kv.adamw_step([z(4)], [d(4)], *state(), 1)),
    ]


NAMES = [name for name, _ in calls("meta", lambda t: t)]


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_tangents_are_refused(name, device, monkeypatch):
    if device == "cpu":                      # (the refusal comes before anything that needs a GPU)
        from kalman_vae_amd import sequence_ops
        monkeypatch.setattr(sequence_ops, "_device_of", lambda *t: torch.device("cpu"))
    with fw.dual_level():
        for grad_mode in (True, False):
            with torch.set_grad_enabled(grad_mode):
                call = dict(calls(device, lambda t: fw.make_dual(t, torch.ones_like(t))))[name]
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call()


@pytest.mark.gpu
def test_tangent_of_an_incoming_gradient():
    """Forward over reverse: the tangent sits in what the backward pass receives."""
    u = torch.randn(3, 2, 12, device="cuda", requires_grad=True)
    x, w = (torch.randn(s, device="cuda", requires_grad=True) for s in ((3, 4), (4,)))
    for out, leaf in ((kv.gated_scan(u)[0], u), (kv.gated_scan(u)[1], u), (kv.rms_norm(x, w), x), (kv.rms_norm(x, w, residual=x)[1], x)):
        with fw.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
            g = fw.make_dual(torch.ones_like(out), torch.ones_like(out))
            torch.autograd.grad(out, leaf, g)


@pytest.mark.gpu
def test_functional_transforms_do_not_pass():
    u, v = (torch.randn(3, 2, 12, device="cuda") for _ in range(2))
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: kv.gated_scan(t)[0], (u,), (v,))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: kv.rms_norm(t, torch.ones(12, device="cuda")))(u)


@pytest.mark.gpu
def test_without_a_tangent_nothing_is_refused():
    """Inside a dual level, tensors without a tangent, and any under a switched-off forward mode, pass."""
    u = torch.randn(3, 2, 12, device="cuda")
    want = kv.gated_scan(u)[0]
    with fw.dual_level():
        assert torch.equal(kv.gated_scan(u)[0], want)
        dual = fw.make_dual(u, torch.ones_like(u))
        with fw._set_fwd_grad_enabled(False):
            assert torch.equal(kv.gated_scan(dual)[0], want)
