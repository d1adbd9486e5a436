"""The gated network on tensors of another device than the current one: its launches on the current
device's stream are made with the tensors' device current."""
import pytest
import torch

from kalman_vae_amd import GatedModel
from kalman_vae_amd import _capi as capi

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("other", [False, True])
def test_launches_on_the_tensors_device(monkeypatch, other):
    """(with one GPU: the current device is said to be another one)"""
    torch.manual_seed(0)
    net = GatedModel(2, 3, 32, 1).cuda()
    x = torch.randn(4, 5, 2, device="cuda")
    inside, launches = [], []

    class Device(torch.cuda.device):
        def __enter__(self):
            inside.append(self.idx)
            return super().__enter__()

        def __exit__(self, *args):
            inside.pop()
            return super().__exit__(*args)

    stream = capi.current_stream_ptr()

    def recorded():
        launches.append(list(inside))
        return stream

    want = net(x).detach()
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(capi, "current_stream_ptr", recorded)
    if other:
        monkeypatch.setattr(torch.cuda, "current_device", lambda: x.device.index + 1)
    net.clear_hidden_state()
    out = net(x)
    with torch.no_grad():
        net.clear_hidden_state()
        stepper, steps = net.inference_stepper(x[0]), torch.empty_like(want)
        for t in range(4):
            stepper.step(x[t], steps[t])
    assert torch.equal(out, want) and float((steps - want).abs().max()) < 1e-5
    assert len(launches) == 5 and all(at == ([x.device.index] if other else []) for at in launches)
