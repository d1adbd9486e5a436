"""The gated network's 8-bit form after its parameters have changed, by every way in which they can: a
call either raises or answers from the parameters that the model has."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def networks():
    import kalman_vae_amd as kv
    torch.manual_seed(0)
    net, other = (kv.GatedModel(2, 3, 64, 2).cuda() for _ in range(2))
    return net, other, torch.randn(12, 50, 2, device="cuda")


@torch.no_grad()
def answer(net, x, stepped=False):
    net.clear_hidden_state()
    if not stepped:
        return net(x)
    stepper = net.inference_stepper(x[0])
    out = torch.empty(*x.shape[:2], 3, device="cuda")
    for t in range(x.shape[0]):
        stepper.step(x[t], out[t])
    return out


def fresh(net, x, stepped):
    """What a new model with net's parameters answers in 8 bits."""
    import kalman_vae_amd as kv
    new = kv.GatedModel(2, 3, 64, 2).cuda()
    new.load_state_dict(net.state_dict(), assign=True)             # (the same addresses: library products alike)
    return answer(new.eight_bit(), x, stepped)


def scale_data(net, other):
    for p in net.blocks.parameters():
        p.data.mul_(1.5)


def replace_data(net, other):
    for p, q in zip(net.parameters(), other.parameters()):
        p.data = q.data.clone()


def from_vector(net, other):
    torch.nn.utils.vector_to_parameters(torch.nn.utils.parameters_to_vector(other.parameters()), net.parameters())


def replace_layer(net, other):
    net.blocks[0].proj = other.blocks[0].proj


@pytest.mark.parametrize("stepped", [False, True])
@pytest.mark.parametrize("change", [scale_data, replace_data, from_vector, replace_layer])
def test_changes_that_autograd_does_not_see(change, stepped):
    net, other, x = networks()
    old = answer(net.eight_bit(), x, stepped)
    with torch.no_grad():
        change(net, other)
    try:
        got = answer(net, x, stepped)
    except RuntimeError as e:
        assert "eight_bit" in str(e)
        got = answer(net.eight_bit(), x, stepped)
    assert torch.equal(got, fresh(net, x, stepped)) and not torch.equal(got, old)


def load_assign(net, other):
    # (versions of the two models' parameters agree)
    net.load_state_dict(other.state_dict(), assign=True)


def replace_parameter(net, other):
    for a, b in zip(net.blocks, other.blocks):
        a.out.weight = torch.nn.Parameter(b.out.weight.detach().clone())


def load_in_place(net, other):
    net.load_state_dict(other.state_dict())


@pytest.mark.parametrize("change", [load_assign, replace_parameter, load_in_place])
def test_changes_that_autograd_sees(change):
    net, other, x = networks()
    old = answer(net.eight_bit(), x)
    stepper = None
    with torch.no_grad():
        net.clear_hidden_state()
        stepper = net.inference_stepper(x[0])
    change(net, other)
    for stepped in (False, True):
        with pytest.raises(RuntimeError, match="eight_bit"):
            answer(net, x, stepped)
    with pytest.raises(RuntimeError, match="eight_bit"):           # one that was made before the change
        stepper.step(x[0], torch.empty(50, 3, device="cuda"))
    got = answer(net.eight_bit(), x)
    assert torch.equal(got, fresh(net, x, False)) and not torch.equal(got, old)


def test_replays_of_a_captured_optimiser_step():
    """A replay runs no Python, so nothing notes its changes."""
    from kalman_vae_amd import AdamW
    net, _, x = networks()
    opt = AdamW(net.parameters(), lr=1e-2, capturable=True)
    for p in net.parameters():
        p.grad = torch.randn_like(p)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        opt.step()
    answers = [answer(net.eight_bit(), x)]
    for _ in range(3):
        graph.replay()
        answers.append(answer(net, x))
        assert torch.equal(answers[-1], fresh(net, x, False)) and not torch.equal(answers[-1], answers[-2])


def test_off_and_refusals():
    import kalman_vae_amd as kv
    net, _, x = networks()
    full = answer(net, x)
    assert not torch.equal(answer(net.eight_bit(), x), full)
    assert torch.equal(answer(net.eight_bit(False), x), full)
    assert torch.equal(answer(net.eight_bit().cuda(), x), full)    # moved: off
    with pytest.raises(TypeError, match="float64"):
        kv.GatedModel(2, 3, 64, 1).double().cuda().eight_bit()
