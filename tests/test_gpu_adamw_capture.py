"""The optimiser's step where a capture would record something that a replay repeats wrongly."""
import pytest
import torch

from kalman_vae_amd import AdamW

pytestmark = pytest.mark.gpu


def parameters(dtype=torch.float32):
    ps = [torch.nn.Parameter(torch.ones(s, device="cuda", dtype=dtype)) for s in ((300,), (5, 7))]
    for p in ps:
        p.grad = torch.full_like(p, 0.5)
    return ps


def capture(opt):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        opt.step()
    return graph


@pytest.mark.parametrize("bits", [32, 8])
def test_a_count_on_the_host_is_refused(bits):
    ps = parameters()
    opt = AdamW(ps, state_bits=bits)
    opt.step()
    with pytest.raises(RuntimeError, match="capturable=True"):
        capture(opt)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("known", [0, 1])
def test_states_made_in_the_capture_are_refused(bits, known):
    """No step before the capture, or one in which a parameter had no gradient."""
    ps = parameters()
    opt = AdamW(ps, state_bits=bits, capturable=True)
    if known:
        grad, ps[1].grad = ps[1].grad, None
        opt.step()
        ps[1].grad = grad
    before = [p.detach().clone() for p in ps]
    with pytest.raises(RuntimeError, match="before the capture"):
        capture(opt)
    torch.cuda.synchronize()
    assert all(torch.equal(p, b) for p, b in zip(ps, before)) and ps[1] not in opt.state


def test_refused_once_it_goes_on():
    """What a refusal leaves is a whole optimiser: step, capture and replays as if it had not been asked."""
    ps, qs = parameters(), parameters()
    opt, plain = AdamW(ps, capturable=True), AdamW(qs)
    with pytest.raises(RuntimeError, match="before the capture"):
        capture(opt)
    opt.step()
    graph = capture(opt)
    for _ in range(3):
        graph.replay()
    for _ in range(4):
        plain.step()
    for p, q in zip(ps, qs):
        assert float((p - q).abs().max()) < 1e-6              # lr / (1 - b^t) is rounded at another place
