"""The "gated" dynamics-parameter network on the CPU (plain torch): its place among the networks,
the state carried between calls, checkpoint keys."""
import pytest
import torch

from kalman_vae_amd import GatedModel, KalmanVariationalAutoencoder, StateSpaceModel


def test_kind_and_parameters():
    ssm = StateSpaceModel(2, 4, 3, "gated", hidden_dim=16, num_layers=3)
    assert isinstance(ssm.weight_model, GatedModel) and len(ssm.weight_model.blocks) == 3
    names = set(ssm.weight_model.state_dict())
    assert {"embed.weight", "blocks.0.norm", "blocks.2.proj.bias", "blocks.1.out.weight", "norm", "linear.bias"} <= names
    KalmanVariationalAutoencoder((16, 16), 1, 2, 4, 3, 0.9, 0.9, True, 0.7, "gated")
    with pytest.raises(ValueError, match="Invalid"):
        StateSpaceModel(2, 4, 3, "gatedd")
    with pytest.raises(ValueError, match="num_layers"):
        GatedModel(2, 3, 8, 0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_steps_equal_the_whole_sequence(dtype):
    torch.manual_seed(0)
    net = GatedModel(2, 3, 16, 2).to(dtype)
    x = torch.randn(7, 4, 2, dtype=dtype)
    whole = net(x, lead=True)
    assert whole.shape == (8, 4, 3) and torch.allclose(whole.sum(-1), torch.ones(8, 4, dtype=dtype))
    assert torch.equal(whole[0], torch.full((4, 3), 1 / 3, dtype=dtype)) and net.hidden.shape == (2, 4, 16)
    end = net.hidden
    net.clear_hidden_state()
    assert net.hidden is None
    steps = torch.cat([net(x[t:t + 1]) for t in range(7)])
    tol = 1e-12 if dtype == torch.float64 else 1e-6
    assert (steps - whole[1:]).abs().max() < tol and (net.hidden - end).abs().max() < 10 * tol
    net.reset_hidden_state(4, x.device, dtype)
    assert not net.hidden.any()
    assert (net(x) - whole[1:]).abs().max() < tol


def test_gradient_through_the_carried_state():
    """Step by step under autograd (the masked filter's use) equals the whole sequence's gradient."""
    torch.manual_seed(1)
    net = GatedModel(2, 3, 8, 2).double()
    x = torch.randn(5, 3, 2, dtype=torch.float64)
    g = torch.randn(5, 3, 3, dtype=torch.float64)
    grads = []
    for pieces in ([x], list(x.split(1))):
        net.clear_hidden_state()
        net.zero_grad()
        (torch.cat([net(p) for p in pieces]) * g).sum().backward()
        grads.append([p.grad.clone() for p in net.parameters()])
    assert all((a - b).abs().max() < 1e-12 for a, b in zip(*grads))


def test_eight_bit_needs_a_gpu():
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        GatedModel(2, 3, 8, 1).eight_bit()
