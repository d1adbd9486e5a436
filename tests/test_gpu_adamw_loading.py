"""A capturable optimiser's state dict, loaded on the CPU as checkpoints often are."""
import pytest
import torch

from kalman_vae_amd import AdamW

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("where", ["cpu", "cuda"])
@pytest.mark.parametrize("bits", [32, 8])
def test_rate_and_count_as_tensors(where, bits, tmp_path):
    def go(ps, opt, steps):
        for k in steps:
            for i, p in enumerate(ps):
                p.grad = torch.randn(p.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(10 * k + i))
            opt.step()

    ps = [torch.nn.Parameter(torch.ones(s, device="cuda")) for s in (300, 7)]
    opt = AdamW(ps, lr=torch.tensor([0.01], device="cuda"), state_bits=bits, capturable=True)
    go(ps, opt, range(3))
    torch.save({"p": [p.detach() for p in ps], "opt": opt.state_dict()}, tmp_path / "s.pth")
    go(ps, opt, range(3, 6))
    saved = torch.load(tmp_path / "s.pth", weights_only=True, map_location=where)
    qs = [torch.nn.Parameter(p.cuda()) for p in saved["p"]]
    again = AdamW(qs, lr=torch.ones(1, device="cuda"), state_bits=bits, capturable=True)
    again.load_state_dict(saved["opt"])
    again.param_groups[0]["lr"].mul_(1.0)                           # its own: not the loaded dict's
    assert again.param_groups[0]["lr"].data_ptr() != saved["opt"]["param_groups"][0]["lr"].data_ptr()
    go(qs, again, range(3, 6))
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))
