"""The gated network as a torch.nn.Module: initialisation deferred on the meta device."""
import torch

from kalman_vae_amd import GatedModel, StateSpaceModel


def test_deferred_initialisation():
    torch.manual_seed(0)
    want = GatedModel(2, 3, 8, 2)
    with torch.device("meta"):
        net = GatedModel(2, 3, 8, 2)
    assert net.to_empty(device="cpu") is net
    net.load_state_dict(want.state_dict())
    x = torch.randn(4, 3, 2)
    assert torch.equal(net(x), want(x))


def test_only_the_module_itself():
    net = GatedModel(2, 3, 8, 1)
    moved = net.to_empty(device="meta", recurse=False)                  # its own parameter, not its children's
    assert moved.norm.is_meta and not moved.embed.weight.is_meta
    ssm = StateSpaceModel(2, 4, 3, "gated", hidden_dim=8).to_empty(device="meta")
    assert all(p.is_meta for p in ssm.parameters())
