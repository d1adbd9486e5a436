"""``capturable`` switched in the middle of a run: the step count goes on."""
import copy

import pytest
import torch

from kalman_vae_amd import AdamW

pytestmark = pytest.mark.gpu


def parameters():
    return [torch.nn.Parameter(torch.linspace(-1, 1, n, device="cuda")) for n in (300, 7)]


def grad(k, p):
    return torch.randn(p.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(31 * k + p.numel()))


def go(ps, opt, steps):
    for k in steps:
        for p in ps:
            p.grad = grad(k, p)
        opt.step()


def same(ps, qs):
    # (lr / (1 - b^t) is formed on the device in one run and on the host in the other: some units of an update)
    return all(float((p - q).detach().abs().max()) < 2e-6 for p, q in zip(ps, qs))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("before,after", [(False, True), (True, False)])
def test_the_count_goes_on(bits, before, after):
    kw = dict(lr=1e-2, state_bits=bits, seed=4)
    ps, qs = parameters(), parameters()
    opt, plain = AdamW(ps, capturable=before, **kw), AdamW(qs, **kw)
    go(ps, opt, range(3))
    opt.param_groups[0]["capturable"] = after
    go(ps, opt, range(3, 6))
    go(qs, plain, range(6))
    assert same(ps, qs)
    if bits == 8:                                # the random bits follow the count
        assert all(torch.equal(opt.state[p]["exp_avg"].view(torch.uint8), plain.state[q]["exp_avg"].view(torch.uint8))
                   for p, q in zip(ps, qs))


def test_after_replays():
    ps, qs = parameters(), parameters()
    opt, plain = AdamW(ps, lr=1e-2, capturable=True), AdamW(qs, lr=1e-2)
    for p in ps:
        p.grad = torch.zeros_like(p)
    held = [p.grad for p in ps]

    def fill(k):
        for p, h in zip(ps, held):
            h.copy_(grad(k, p))

    fill(0)
    opt.step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        opt.step()
    for k in range(1, 5):
        fill(k)
        graph.replay()
    opt.param_groups[0]["capturable"] = False
    go(ps, opt, range(5, 8))
    go(qs, plain, range(8))
    assert same(ps, qs) and all(opt.state[p]["step"] == 8 for p in ps)


def test_counts_of_former_graphs_stay_allocated():
    """A graph that was captured before the switch still writes its count: nothing else gets that memory."""
    ps = parameters()
    opt = AdamW(ps, capturable=True)
    go(ps, opt, range(2))
    place = opt.param_groups[0]["step"].data_ptr()
    opt.param_groups[0]["capturable"] = False
    go(ps, opt, range(2, 4))
    others = [torch.empty(1, dtype=torch.int64, device="cuda") for _ in range(1000)]
    assert place not in {t.data_ptr() for t in others}
    opt.param_groups[0]["capturable"] = True
    go(ps, opt, range(4, 5))
    assert int(opt.param_groups[0]["step"]) == 5 and opt.param_groups[0]["step"].data_ptr() != place
    again = copy.deepcopy(opt)                   # (what a copy lacks is not missed)
    again.param_groups[0]["capturable"] = False
    go(again.param_groups[0]["params"], again, range(5, 6))
