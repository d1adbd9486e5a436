"""adamw_step and the AdamW optimiser against the update's formulas in float64; the 8-bit states'
codes against the rounding rule written out one float32 operation at a time."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
UNIT = 2.0 ** -24
LR, B1, B2, EPS, WD = 1e-2, 0.9, 0.999, 1e-8, 0.1
SIZES = [1, 2, 15, 16, 17, 255, 256, 257, 4095, 4096, 4097, 70001]


def half_step(dtype):
    return 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2


def make(sizes, dtype, bits, seed=0, offset=0):
    """Lists of parameters, gradients and states; offset: elements that shift every view off alignment."""
    from kalman_vae_amd.optim import state_blocks
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda k: torch.randn(k, generator=g, device="cuda")  # noqa: E731

    def placed(t):
        flat = torch.zeros(t.numel() + offset, dtype=t.dtype, device="cuda")
        flat[offset:].copy_(t) if t.dtype != torch.float8_e4m3fn else flat.view(torch.uint8)[offset:].copy_(t.view(torch.uint8))
        return flat[offset:]

    params = [placed(n(k).to(dtype)) for k in sizes]
    grads = [placed((n(k) * math.exp(float(n(1)))).to(dtype)) for k in sizes]
    masters = [p.float() * (1 + 1e-4) for p in params] if dtype != torch.float32 else None
    m, v = [n(k) * 0.3 for k in sizes], [0.05 * n(k).abs() + 0.01 for k in sizes]
    if bits == 32:
        return params, grads, [placed(t) for t in m], [placed(t * t) for t in v], masters
    pairs = []
    for ts in (m, v):
        row = []
        for t in ts:
            blocks = torch.nn.functional.pad(t, (0, -t.numel() % 256)).view(-1, 256)
            scale = (blocks.abs().amax(1) / 448).clamp_min(2.0 ** -126)
            codes = (blocks / scale[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(-1)[:t.numel()]
            assert scale.numel() == state_blocks(t.numel())
            row.append((placed(codes.contiguous()), scale))
        pairs.append(row)
    return params, grads, pairs[0], pairs[1], masters


def value(state):
    """float64 values of a state: a float32 tensor, or 8-bit codes and scales."""
    if isinstance(state, torch.Tensor):
        return state.double()
    codes, scale = state
    return codes.double() * scale.double().repeat_interleave(256)[:codes.numel()]


def oracle(p, g, m, v, t):
    """(p, m, v) in float64 and the size of the parameter's update."""
    m, v = B1 * m + (1 - B1) * g, B2 * v + (1 - B2) * g * g
    move = LR / (1 - B1 ** t) * m / (v.sqrt() / math.sqrt(1 - B2 ** t) + EPS)
    return p * (1 - LR * WD) - move, m, v, move


def step(lists, t, **kw):
    import kalman_vae_amd as kv
    params, grads, m, v, masters = lists
    kv.adamw_step(params, grads, m, v, t, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, masters=masters, **kw)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("offset", [0, 1])
def test_one_step(dtype, bits, offset):
    lists = make(SIZES, dtype, bits, offset=offset)
    params, grads, m, v, masters = lists
    start = masters if masters is not None else params
    before = [(p.double(), g.double(), value(a), value(b) if bits == 32 else value(b) ** 2)
              for p, g, a, b in zip(start, grads, m, v)]
    step(lists, 7)
    for i, (p0, g0, m0, v0) in enumerate(before):
        p, m1, v1, move = oracle(p0, g0, m0, v0, 7)
        # float32: a dozen roundings of the update's relative value (its m may cancel: charged with
        # the terms' sizes), two of the decayed parameter
        rough = (B1 * m0.abs() + (1 - B1) * g0.abs()) / m1.abs().clamp_min(1e-30)
        err = 4 * UNIT * p0.abs() + 16 * UNIT * move.abs() * (1 + rough)
        got = (masters if masters is not None else params)[i].double()
        assert ((got - p).abs() <= err).all(), i
        if masters is not None:
            assert torch.equal(params[i], masters[i].to(dtype))
        if bits == 32:
            assert ((m[i].double() - m1).abs() <= 4 * UNIT * (B1 * m0.abs() + (1 - B1) * g0.abs())).all()
            assert ((v[i].double() - v1).abs() <= 5 * UNIT * v1).all()


def test_16_bit_parameters_without_masters():
    params, grads, m, v, _ = lists = make(SIZES, torch.bfloat16, 32)
    before = [(p.double(), g.double(), value(a), value(b)) for p, g, a, b in zip(params, grads, m, v)]
    step(lists[:4] + (None,), 3)
    for i, args in enumerate(before):
        p, _, _, move = oracle(*args, 3)
        assert ((params[i].double() - p).abs() <= half_step(torch.bfloat16) * p.abs() * 1.01 + 1e-5 * move.abs() + 1e-9).all()


def hashed(index, seed, t):
    low = 0xFFFFFFFF
    h = (index * 0x9E3779B1 + ((seed + t * 0x9E3779B9) & low)) & low
    h = ((h ^ (h >> 16)) * 0x7FEB352D) & low
    h = ((h ^ (h >> 15)) * 0x846CA68B) & low
    return h ^ (h >> 16)


def codes_of(x, bits16, positive):
    """The rounding rule, one float32 operation at a time: (codes, scales) of x, padded to blocks."""
    x = torch.nn.functional.pad(x, (0, -x.numel() % 256)).view(-1, 256)
    scale = (x.abs().amax(1) * (1.0 / 448)).clamp_min(2.0 ** -126)
    t = (x * (1.0 / scale)[:, None]).view(-1)
    size = t.abs().clamp_max(448.0)
    up = ((size.view(torch.int32) + (bits16 * 16 + 8).int()) & ~0xFFFFF).view(torch.float32).clamp_max(448.0)
    small = torch.floor(size * 512 + (bits16.float() + 0.5) * (1.0 / 65536))
    if positive:
        small = torch.where(size > 0, small.clamp_min(1.0), 0.0)
    r = torch.where(size < 0.015625, small / 512, up)
    return torch.copysign(r, t).to(torch.float8_e4m3fn), scale


@pytest.mark.parametrize("count", [1, 5, 48, 49, 130])
def test_codes_follow_the_rounding_rule(count):
    """Bit for bit, the hash index running on over the tensors of the list and its launches."""
    sizes = [(37 * i * i + 1) % 3001 + 1 for i in range(count)]
    lists = make(sizes, torch.float32, 8, seed=1)
    params, grads, m, v, _ = lists
    f = lambda s: s[0].float() * s[1].repeat_interleave(256)[:s[0].numel()]  # noqa: E731
    before = [(f(a), f(b), g) for a, b, g in zip(m, v, grads)]
    step(lists, 12, seed=99)
    first = 0
    for i, (m0, r0, g) in enumerate(before):
        m1 = m0 * B1 + g * (1 - B1)
        root = torch.sqrt((r0 * r0) * B2 + (g * g) * (1 - B2))
        n = sizes[i]
        blocks = -(-n // 256)
        h = hashed(first + torch.arange(256 * blocks, device="cuda"), 99, 12)
        for got, want in ((m[i], codes_of(m1, h & 0xFFFF, False)), (v[i], codes_of(root, h >> 16, True))):
            assert torch.equal(got[1], want[1]), i
            assert torch.equal(got[0].view(torch.uint8), want[0].view(torch.uint8)[:n]), i
        first += 256 * blocks


def known_block(n):
    """States whose codes are 448 at each block's head and 8 behind it, scales 1/448."""
    lists = make([n], torch.float32, 8)
    for s in (lists[2][0], lists[3][0]):
        s[0].view(torch.uint8).fill_(0x50)
        s[0].view(torch.uint8)[::256] = 0x7E
        s[1].fill_(1.0 / 448)
    lists[1][0].zero_()
    return lists


def test_block_that_decays_as_a_whole():
    """Without a gradient everything shrinks alike: the scales move and the codes stay."""
    n = 1 << 18
    lists = known_block(n)
    params, grads, m, v, _ = lists
    step(lists, 1)
    body = torch.arange(n, device="cuda") % 256 != 0
    for s, factor in ((m[0], B1), (v[0], math.sqrt(B2))):
        assert ((s[1].double() * 448 - factor).abs() < 8 * UNIT).all()
        assert (s[0].float()[body] == 8).all() and (s[0].float()[~body] == 448).all()


def test_rounding_keeps_the_mean():
    """A state between two codes stays there on average; to the nearest it would be stuck."""
    n = 1 << 18
    lists = known_block(n)
    params, grads, m, v, _ = lists
    grads[0][::256] = 1.0                                        # keeps the heads, so the scales, at 1
    step(lists, 1)
    body = torch.arange(n, device="cuda") % 256 != 0
    for s, factor, low in ((m[0], B1, 7.0), (v[0], math.sqrt(B2), 7.5)):
        t = 8 * factor                                           # between the codes low and low + 0.5
        share = (t - low) / 0.5
        got = s[0].double()[body]
        assert set(got.tolist()) == {low, low + 0.5}
        # six standard deviations of the share; 2^-16 is the step of the random bits
        sigma = math.sqrt(share * (1 - share) / got.numel())
        assert abs(float((got == low + 0.5).double().mean()) - share) < 6 * sigma + 2.0 ** -16 + 1e-5


def test_zero_small_and_non_finite_blocks():
    lists = make([256 * 6], torch.float32, 8)
    params, grads, m, v, _ = lists
    for s in (m[0], v[0]):
        s[0].view(torch.uint8).zero_()
        s[1].fill_(2.0 ** -126)
    g = grads[0].view(6, 256)
    g[0] = 0                                                     # nothing has happened yet
    g[1] = 1e-30                                                 # g^2 underflows, m does not
    g[2, 1:] *= 1e-6                                             # one element dwarfs the block
    g[2, 0] = 100.0
    g[3, 5] = float("nan")
    g[4, 5] = float("inf")
    p0 = params[0].clone().view(6, 256)
    for t in range(1, 4):
        step(lists, t)
    p = params[0].view(6, 256)
    moved = (p - p0 * (1 - LR * WD) ** 3).abs()
    assert torch.equal(moved[0] < 1e-6, torch.ones(256, dtype=torch.bool, device="cuda"))
    assert torch.isfinite(p[:3]).all() and torch.isfinite(p[5]).all()
    # no element moves by more than a few learning rates: sqrt(v) never has the code 0 under a
    # positive value (|m| / sqrt(v) is at most about 1 here; a factor for the codes' coarseness)
    assert float(moved[2].max()) < 3 * 4 * LR
    assert torch.isnan(p[3, 5]) and int(torch.isnan(p[3]).sum()) == 1
    assert float(m[0][1][0]) == 2.0 ** -126 and not m[0][0].view(6, 256)[0].float().any()


def test_neighbours_are_left_alone():
    """Tensors that are slices of one buffer: nothing is written outside them."""
    buf = torch.full((5000,), 7.0, device="cuda")
    g = torch.full((5000,), 1.0, device="cuda")
    codes = [torch.full((5000,), 3.0, device="cuda").to(torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.full((30,), 5.0, device="cuda") for _ in range(2)]
    cut = slice(1001, 3333)
    n = 3333 - 1001
    step(([buf[cut]], [g[cut]], [(codes[0][cut], scales[0][3:13])], [(codes[1][cut], scales[1][3:13])], None), 1)
    keep = torch.ones(5000, dtype=torch.bool, device="cuda")
    keep[cut] = False
    assert (buf[keep] == 7).all() and (buf[~keep] != 7).all() and n > 0
    for c, s in zip(codes, scales):
        assert (c.float()[keep] == 3).all() and (s[:3] == 5).all() and (s[13:] == 5).all() and (s[3:13] != 5).all()


def model_and_data(dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    shapes = [(3, 5), (128,), (64, 65), (7,), (1,), (300, 11), (0, 4)]
    ps = [torch.nn.Parameter(torch.randn(s, generator=g, device="cuda").to(dtype)) for s in shapes]
    return ps, lambda k: [torch.randn(s, generator=torch.Generator(device="cuda").manual_seed(1000 * k + i), device="cuda").to(dtype)
                          for i, s in enumerate(shapes)]


def test_optimiser_follows_torch():
    """Thirty steps of the 32-bit optimiser against torch.optim.AdamW in float64, a parameter without a gradient in some steps."""
    from kalman_vae_amd import AdamW
    ps, grads = model_and_data(torch.float32)
    qs = [torch.nn.Parameter(p.detach().double()) for p in ps]
    a = AdamW(ps, lr=LR, weight_decay=WD)
    b = torch.optim.AdamW(qs, lr=LR, weight_decay=WD, foreach=False)
    for k in range(30):
        for i, (p, q, g) in enumerate(zip(ps, qs, grads(k))):
            p.grad, q.grad = (None, None) if i == 1 and k % 3 else (g.clone(), g.double())
        a.step()
        b.step()
    for p, q in zip(ps, qs):
        # per step: 4 units of the parameter, and of an update of at most 10 lr (1e-2) 40 units
        assert ((p.double() - q).abs() <= 30 * UNIT * (4 * (q.abs() + 3) + 40 * 10 * LR)).all()


@pytest.mark.parametrize("dtype,bits", [(torch.float32, 32), (torch.float32, 8), (torch.bfloat16, 32), (torch.float16, 8)])
def test_state_dict_round_trip(dtype, bits, tmp_path):
    """A checkpoint in the middle: the continued run equals the uninterrupted one bit for bit."""
    from kalman_vae_amd import AdamW
    ps, grads = model_and_data(dtype)
    opt = AdamW(ps, lr=LR, state_bits=bits, seed=5)

    def go(ps, opt, steps):
        for k in steps:
            for p, g in zip(ps, grads(k)):
                p.grad = g
            opt.step()

    go(ps, opt, range(3))
    torch.save({"p": [p.detach() for p in ps], "opt": opt.state_dict()}, tmp_path / "s.pth")
    go(ps, opt, range(3, 6))
    saved = torch.load(tmp_path / "s.pth", weights_only=True)
    rs = [torch.nn.Parameter(p) for p in saved["p"]]
    again = AdamW(rs, lr=1.0, state_bits=bits)
    again.load_state_dict(saved["opt"])
    go(rs, again, range(3, 6))
    assert all(torch.equal(p, r) for p, r in zip(ps, rs))
    if bits == 8:
        assert again.state[rs[0]]["exp_avg"].dtype == torch.float8_e4m3fn


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step(bits):
    """A captured step replayed, the step count and the rate on the device, against eager steps."""
    from kalman_vae_amd import AdamW
    ps, grads = model_and_data(torch.float32)
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    lr = torch.full((1,), LR, device="cuda")
    a = AdamW(ps, lr=lr, state_bits=bits, capturable=True)
    b = AdamW(qs, lr=LR, state_bits=bits)
    static = [torch.zeros_like(p) for p in ps]
    for p, s, g in zip(ps, static, grads(0)):
        s.copy_(g)
        p.grad = s
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a.step()                                   # (states are made outside the capture)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        a.step()
    for k in range(6):
        if k:
            lr.fill_(LR * (1 + k))
            b.param_groups[0]["lr"] = LR * (1 + k)
            for s, g in zip(static, grads(k)):
                s.copy_(g)
            graph.replay()
        for q, g in zip(qs, grads(k)):
            q.grad = g
        b.step()
        for p, q in zip(ps, qs):
            # lr and 1 / (1 - b^t) are rounded at other places: a few units of the update
            assert ((p - q).abs() <= 6 * (16 * UNIT * 10 * LR * 7 + 4 * UNIT * (p.abs() + 1))).all(), k
    if bits == 8:
        assert all(torch.equal(a.state[p]["exp_avg"].view(torch.uint8), b.state[q]["exp_avg"].view(torch.uint8))
                   for p, q in zip(ps, qs))


def test_with_the_data_parallel_step():
    """DataParallelStep: gradients are slices of the flat bucket, at any 4-byte address."""
    from kalman_vae_amd import AdamW, SampleControl, StateSpaceModel, kalman_elbo
    from kalman_vae_amd.parallel import DataParallelStep
    torch.manual_seed(0)
    ssm = StateSpaceModel(2, 4, 3, "lstm", hidden_dim=32).cuda().train()
    ref = {k: v.clone() for k, v in ssm.state_dict().items()}
    a = torch.randn(8, 16, 2, device="cuda")

    def run(make_optimizer):
        ssm.load_state_dict(ref)
        step = DataParallelStep(ssm, make_optimizer(ssm.parameters()))
        for k in range(3):
            torch.manual_seed(k)
            step(lambda: kalman_elbo(ssm, a, SampleControl())[0])
        return {k: v.clone() for k, v in ssm.state_dict().items()}

    got = run(lambda p: AdamW(p, lr=1e-3, weight_decay=0.01))
    want = run(lambda p: torch.optim.AdamW(p, lr=1e-3, weight_decay=0.01))
    eight = run(lambda p: AdamW(p, lr=1e-3, weight_decay=0.01, state_bits=8))
    for k, v in want.items():
        # three steps of 1e-3; an update's relative error (the objective's gradients, float32) stays
        # far below a percent, an 8-bit state's below one of the codes' coarseness, 1/8 per state
        assert ((got[k] - v).abs() <= 3e-5 + 1e-5 * v.abs()).all(), k
        assert ((eight[k] - v).abs() <= 3e-3).all(), k
