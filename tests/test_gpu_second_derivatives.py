"""A gradient of a gradient raises whatever it is asked for with respect to, also where the incoming
gradient carries no graph and where the tensor is one that the first gradient was not asked for."""
import pytest
import torch

import kalman_vae_amd as kv

pytestmark = pytest.mark.gpu


def leaf(*shape, seed):
    return torch.randn(shape, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)).requires_grad_(True)


def scan():
    leaves = {"u": leaf(5, 2, 12, seed=1), "h0": leaf(2, 4, seed=2)}
    return leaves, list(kv.gated_scan(leaves["u"], leaves["h0"]))


def norm(residual, dtype):
    def make():
        leaves = {"x": leaf(4, 8, seed=1), "weight": leaf(8, seed=2)}
        if residual:
            leaves["residual"] = leaf(4, 8, seed=3)
        out = kv.rms_norm(leaves["x"].to(dtype), leaves["weight"], residual=leaves["residual"].to(dtype) if residual else None)
        return leaves, list(out) if residual else [out]
    return make


CASES = [scan] + [norm(r, d) for r in (False, True) for d in (torch.float32, torch.bfloat16)]


@pytest.mark.parametrize("square", [False, True])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_every_pair_of_tensors(case, square):
    names = list(CASES[case]()[0])
    for first in names:
        for second in names:
            leaves, out = CASES[case]()
            total = sum((o.square() if square else o).sum() for o in out)
            g, = torch.autograd.grad(total, leaves[first], create_graph=True)
            with pytest.raises(RuntimeError, match="differentiable once"):
                torch.autograd.grad(g.sum(), leaves[second], allow_unused=True)


def test_start_state_may_change_before_the_backward_pass():
    """The backward pass does not read h0: a state that is stepped on in place is no obstacle."""
    leaves, (y, last) = scan()
    want = torch.autograd.grad((y.sum(), last.sum()), list(leaves.values()), retain_graph=True)
    with torch.no_grad():
        leaves["h0"].add_(1.0)
    got = torch.autograd.grad((y.sum(), last.sum()), list(leaves.values()))
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("square", [False, True])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_backward_pass_called_by_hand(case, square):
    """The operator's node called outside a backward pass: the same gradients, and the same refusal."""
    leaves, out = CASES[case]()
    total = sum((o.square() if square else o).sum() for o in out)
    want = torch.autograd.grad(total, list(leaves.values()), retain_graph=True)
    incoming = torch.autograd.grad(total, out, retain_graph=True, create_graph=square)
    got = [g for g in out[0].grad_fn(*incoming) if g is not None]
    assert len(got) == len(want)
    # (the norm's node has x, weight and residual in this order; between it and a leaf a conversion may stand)
    assert all(torch.equal(g.float(), w) for g, w in zip(got, want))
    for second in leaves.values():
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(got[0].sum(), second, retain_graph=True, allow_unused=True)
