"""A step of the optimiser that is refused counts as none: what follows is what would have followed."""
import pytest
import torch

from kalman_vae_amd import AdamW

pytestmark = pytest.mark.gpu


def run(bits, capturable, refuse):
    g = torch.Generator("cuda").manual_seed(1)
    ps = [torch.nn.Parameter(torch.randn(s, s, generator=g, device="cuda")) for s in (20, 33)]
    opt = AdamW(ps, lr=1e-2, state_bits=bits, seed=2, capturable=capturable)
    for k in range(4):
        for p in ps:
            p.grad = torch.randn(p.shape, generator=g, device="cuda")
        refuse(k, ps, opt)
        opt.step()
    return [p.detach() for p in ps] + [opt.state[p][name].view(torch.uint8) for p in ps for name in ("exp_avg", "exp_avg_sq")]


def turned(k, ps, opt):
    if k in (0, 2):
        ps[1].data = ps[1].data.t()
        with pytest.raises(ValueError, match="contiguous"):
            opt.step()
        ps[1].data = ps[1].data.t()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("capturable", [False, True])
def test_refused_steps_are_not_counted(bits, capturable):
    want = run(bits, capturable, lambda *a: None)
    got = run(bits, capturable, turned)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_counts_of_refused_groups():
    ps = [torch.nn.Parameter(torch.ones(5, device="cuda")) for _ in range(2)]
    opt = AdamW(ps, capturable=True)
    for p in ps:
        p.grad = torch.ones_like(p)
    opt.step()
    ps[0].grad = None
    opt.step()                                                     # its count stays behind from here on
    ps[0].grad = torch.ones_like(ps[0])
    before = [p.detach().clone() for p in ps]
    for _ in range(3):
        with pytest.raises(RuntimeError, match="share one step count"):
            opt.step()
        assert [opt.state[p]["step"] for p in ps] + [int(opt.param_groups[0]["step"])] == [1, 2, 2]
    assert all(torch.equal(p, b) for p, b in zip(ps, before))
