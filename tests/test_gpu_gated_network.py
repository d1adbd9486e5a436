"""The "gated" dynamics-parameter network on its kernels: against itself in float64, inside the
Kalman objective and the masked filter, trained with AdamW, served in 8 bits, captured."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu


def rel(a, b):
    return float((a.detach().cpu().double() - b.detach().cpu().double()).norm() / b.detach().cpu().double().norm())


@pytest.mark.parametrize("hidden,layers,T,B", [(32, 1, 9, 5), (128, 2, 20, 33), (48, 3, 130, 2)])
def test_against_float64(hidden, layers, T, B):
    from kalman_vae_amd import GatedModel
    torch.manual_seed(0)
    net = GatedModel(2, 3, hidden, layers).cuda()
    ref = copy.deepcopy(net).cpu().double()
    x = torch.randn(T, B, 2, device="cuda", requires_grad=True)
    x64 = x.detach().cpu().double().requires_grad_(True)
    g = torch.randn(T + 1, B, 3, device="cuda")
    out, want = net(x, lead=True), ref(x64, lead=True)
    (out * g).sum().backward()
    (want * g.cpu().double()).sum().backward()
    # float32 against float64 through a few matrix products and norms per layer (each some 1e-6)
    assert rel(out, want) < 1e-5 and rel(x.grad, x64.grad) < 1e-4 and rel(net.hidden, ref.hidden) < 1e-5
    for (k, p), q in zip(net.named_parameters(), ref.parameters()):
        assert rel(p.grad, q.grad) < 1e-4, k


def test_steps_and_state():
    """Whole sequence, pieces and the one-step form agree; the state is carried on."""
    from kalman_vae_amd import GatedModel
    torch.manual_seed(0)
    net = GatedModel(2, 3, 64, 2).cuda()
    x = torch.randn(30, 17, 2, device="cuda")
    with torch.no_grad():
        whole = net(x)
        end = net.hidden
        net.clear_hidden_state()
        pieces = torch.cat([net(p) for p in x.split(7)])
        assert rel(pieces, whole) < 1e-5 and rel(net.hidden, end) < 1e-5
        net.clear_hidden_state()
        stepper = net.inference_stepper(x[0])
        out = torch.empty(30, 17, 3, device="cuda")
        for t in range(30):
            stepper.step(x[t], out[t])
        net.finish_steps(stepper, 30)
        assert rel(out, whole) < 1e-5 and rel(net.hidden, end) < 1e-5
    assert net.inference_stepper(x[0]) is None                   # a gradient is recorded


def objective_pair(net_kind="gated"):
    import kalman_vae_amd.elbo as ke
    from kalman_vae_amd import SampleControl, StateSpaceModel, kalman_elbo
    from oracle import kalman_oracle as O
    torch.manual_seed(0)
    T, B = 20, 64
    ssm = StateSpaceModel(2, 4, 3, net_kind, hidden_dim=32).cuda().train()
    ssm.rng_parity = False
    a = (0.7 * torch.randn(T, B, 2, device="cuda")).requires_grad_(True)
    orig, draws = ke._standard_normal, []

    def recording(shape, dtype, device):
        draws.append(orig(shape, dtype=dtype, device=device))
        return draws[-1]

    ke._standard_normal = recording
    try:
        obj, _ = kalman_elbo(ssm, a, SampleControl(), burn_in=3)
        obj.backward()
    finally:
        ke._standard_normal = orig
    eps = draws[0][-T * B * 4:].view(T, B, 4)
    ref = StateSpaceModel(2, 4, 3, net_kind, hidden_dim=32)
    ref.load_state_dict({k: v.cpu() for k, v in ssm.state_dict().items()})
    ref = ref.double()
    a64 = a.detach().cpu().double().requires_grad_(True)
    obj64, _ = O.kalman_objective(a64, ref._mat_A_K, ref._mat_C_K, ref.mat_Q, ref.mat_R, ref.initial_state_mean,
                                  ref.initial_state_covariance, ref.weight_model, eps.cpu().double(), burn_in=3)
    obj64.backward()
    return ssm, ref, a, a64, obj, obj64


def test_kalman_objective():
    """The training objective with this network against the float64 oracle: value, gradients of the
    observations, the bases and every parameter of the network."""
    ssm, ref, a, a64, obj, obj64 = objective_pair()
    assert rel(obj, obj64) < 1e-4 and rel(a.grad, a64.grad) < 1e-4
    for (k, p), q in zip(ssm.named_parameters(), ref.parameters()):
        if q.grad is not None and q.grad.any():
            assert rel(p.grad, q.grad) < 2e-4, k


def masked_case():
    from kalman_vae_amd import SampleControl, StateSpaceModel
    torch.manual_seed(3)
    ssm = StateSpaceModel(2, 4, 3, "gated", hidden_dim=32).cuda()
    a = 0.7 * torch.randn(15, 40, 2, device="cuda")
    mask = (torch.rand(15, 40, device="cuda") < 0.6).float()
    mask[0] = 1
    return ssm, a, mask, SampleControl(encoder="mean", decoder="mean", state_transition="mean", observation="mean")


def test_masked_filter_takes_the_stepper():
    """The masked filter without a gradient: the in-place one-step form against the module called
    step by step in plain torch."""
    ssm, a, mask, sc = masked_case()
    ssm.eval()
    with torch.no_grad():
        got = ssm.kalman_filter(a, sc, observation_mask=mask)
        assert ssm.weight_model.count == 15
        ssm.weight_model.use_hip_kernels = False
        want = ssm.kalman_filter(a, sc, observation_mask=mask)
    for g, w in zip(got, want):
        assert rel(g, w) < 2e-5
    ssm.weight_model.use_hip_kernels = True
    filled, regenerated = ssm.impute(a, sc, observation_mask=mask)
    assert torch.isfinite(filled).all() and torch.isfinite(regenerated).all()


def test_masked_filter_under_autograd():
    ssm, a, mask, _ = masked_case()
    from kalman_vae_amd import SampleControl, kalman_elbo
    ssm.train()
    grads = []
    for kernels in (True, False):
        ssm.weight_model.use_hip_kernels = kernels
        ssm.zero_grad(set_to_none=True)
        torch.manual_seed(5)
        obj, _ = kalman_elbo(ssm, a, SampleControl(), observation_mask=mask)
        obj.backward()
        grads.append([obj.detach()] + [p.grad for p in ssm.parameters() if p.grad is not None])
    assert len(grads[0]) == len(grads[1]) > 10
    for g, w in zip(*grads):
        # float32 both sides, a 15-step recursion through filter and network
        assert rel(g, w) < 1e-3


def test_captured_step_equals_the_eager_one():
    """GraphedElboStep with this network: replays on new observations equal eager steps."""
    from kalman_vae_amd import SampleControl, StateSpaceModel, kalman_elbo
    from kalman_vae_amd.graphed import GraphedElboStep
    torch.manual_seed(0)
    ssm = StateSpaceModel(2, 4, 3, "gated", hidden_dim=64).cuda().train()
    ssm.rng_parity = False
    ssm.fused_loss = True
    a = 0.7 * torch.randn(20, 64, 2, device="cuda")
    step = GraphedElboStep(ssm, a, SampleControl(), burn_in=3)
    state = torch.cuda.get_rng_state()
    for k in range(3):
        b = 0.7 * torch.randn(20, 64, 2, device="cuda", generator=torch.Generator("cuda").manual_seed(k))
        torch.cuda.set_rng_state(state)
        objective = step(b).clone()
        got = {n: p.grad.clone() for n, p in ssm.named_parameters() if p.grad is not None}
        ssm.zero_grad(set_to_none=True)
        torch.cuda.set_rng_state(state)
        want, _ = kalman_elbo(ssm, b.requires_grad_(True), SampleControl(), burn_in=3)
        (-want).backward()
        assert torch.allclose(objective, want, rtol=1e-6)
        for n, p in ssm.named_parameters():
            if p.grad is not None:
                assert rel(got[n], p.grad) < 1e-5, n


def test_eight_bit_form():
    """The 8-bit form is the chain of its operators, in the whole-sequence and the one-step form; it
    notices changed parameters and does not run where a gradient is recorded."""
    import kalman_vae_amd as kv
    torch.manual_seed(0)
    net = kv.GatedModel(2, 3, 64, 2).cuda()
    x = torch.randn(12, 50, 2, device="cuda")
    full = net(x).detach()
    net.clear_hidden_state()
    assert net.eight_bit() is net
    with torch.no_grad():
        got = net(x)
        h, branch = net.embed(x), None
        for block in net.blocks:
            if branch is None:
                q, s = kv.rms_norm_quantized(h, block.norm, eps=net.eps)
            else:
                q, s, h = kv.rms_norm_quantized(branch, block.norm, residual=h, eps=net.eps)
            u = kv.linear_8bit(q, s, *kv.quantize_rows(block.proj.weight), bias=block.proj.bias, dtype=torch.bfloat16)
            y, _ = kv.gated_scan(u)
            branch = kv.linear_8bit(*kv.quantize_rows(y), *kv.quantize_rows(block.out.weight), bias=block.out.bias)
        n, _ = kv.rms_norm(branch, net.norm, residual=h, eps=net.eps)
        want = torch.softmax(net.linear(n), -1)
        assert rel(got, want) < 1e-5 and not torch.equal(got, full)
        net.clear_hidden_state()
        stepper = net.inference_stepper(x[0])
        out = torch.empty_like(got)
        for t in range(12):
            stepper.step(x[t], out[t])
        # one step at a time the recurrence rounds differently, which can move a state's 8-bit code
        # by one step (1/16 of it at most) and a weight by a small part of that
        assert float((out - got).abs().max()) < 1 / 16
    net.clear_hidden_state()
    assert torch.equal(net(x).detach(), full)                    # with a gradient: the full form
    with torch.no_grad():
        net.clear_hidden_state()
        net.blocks[1].out.weight.mul_(1.01)
        with pytest.raises(RuntimeError, match="eight_bit"):
            net(x)
        net.clear_hidden_state()
        net.eight_bit()(x)
        net.clear_hidden_state()
        net.eight_bit(False)
        assert rel(net(x), full) < 0.1


def test_train_then_serve():
    """All of it together, as a program uses it: a few data-parallel training steps with 8-bit
    AdamW states, the optimiser noticing nothing of the layout; then masked imputation in 8 bits."""
    from kalman_vae_amd import AdamW, SampleControl, kalman_elbo
    from kalman_vae_amd.parallel import DataParallelStep
    ssm, a, mask, sc = masked_case()
    ssm.train()
    before = {k: v.clone() for k, v in ssm.state_dict().items()}
    ssm.weight_model.eight_bit()
    opt = AdamW(ssm.parameters(), lr=1e-3, state_bits=8)
    step = DataParallelStep(ssm, opt)
    for k in range(3):
        objective = step(lambda: kalman_elbo(ssm, a, SampleControl(), burn_in=2)[0])
        assert torch.isfinite(objective)
    for k, p in ssm.named_parameters():
        if p.grad is not None and p.grad.any():
            # an element moves by at most lr (1 + weight decay) a step, times sqrt(v)'s coarseness
            # (codes 1/8 apart, bias-corrected from the same step's gradient)
            assert 0 < float((p.detach() - before[k]).abs().max()) < 3 * 1e-3 * 2, k
    ssm.eval()
    with torch.no_grad(), pytest.raises(RuntimeError, match="eight_bit"):
        ssm.impute(a, sc, observation_mask=mask)
    ssm.weight_model.eight_bit()
    with torch.no_grad():
        filled, regenerated = ssm.impute(a, sc, observation_mask=mask)
        assert torch.isfinite(filled).all() and torch.isfinite(regenerated).all()
        assert torch.equal(filled[mask == 1], a[mask == 1])


def test_bfloat16_module():
    from kalman_vae_amd import GatedModel
    torch.manual_seed(0)
    net = GatedModel(2, 3, 64, 2).cuda()
    low = copy.deepcopy(net).bfloat16()
    ref = copy.deepcopy(low).float()
    x = torch.randn(10, 8, 2, device="cuda").bfloat16()
    out = low(x)
    out.float().square().sum().backward()
    want = ref(x.float())
    assert out.dtype == torch.bfloat16 and all(p.grad is not None for p in low.parameters())
    # bfloat16 activations through a dozen roundings of 2^-8 each
    assert float((out.float() - want).abs().max()) < 12 * 2.0 ** -8
