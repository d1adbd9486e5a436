"""8-bit states of elements behind the first 2^32 of a step (a model of that size is not needed: the C
call says how many blocks came before): their bits follow the hash, under another key."""
import ctypes as C

import pytest
import torch

from kalman_vae_amd import _capi as capi
from test_gpu_adamw import B1, B2, EPS, LR, WD, codes_of, hashed, make

pytestmark = pytest.mark.gpu

LOW = 0xFFFFFFFF
SEED, STEP = 99, 12


def key_of(high):
    """The step's key for indexes whose high half is `high`."""
    key = (SEED + STEP * 0x9E3779B9) & LOW
    if high:
        h = (key + high * 0x9E3779B1) & LOW
        h = ((h ^ (h >> 16)) * 0x7FEB352D) & LOW
        h = ((h ^ (h >> 15)) * 0x846CA68B) & LOW
        key = h ^ (h >> 16)
    return key


def call(n, first_block):
    """States and gradient before, states behind one step on n elements."""
    params, grads, m, v, _ = make([n], torch.float32, 8, seed=5)
    value = lambda s: s[0].float() * s[1].repeat_interleave(256)[:n]  # noqa: E731
    before = value(m[0]), value(v[0]), grads[0]
    row = (C.c_int64 * 8)(n, params[0].data_ptr(), grads[0].data_ptr(), m[0][0].data_ptr(), v[0][0].data_ptr(),
                          m[0][1].data_ptr(), v[0][1].data_ptr(), 0)
    d = capi.AdamW(count=1, state_bits=8, step=STEP, seed=SEED, lr=LR, beta1=B1, beta2=B2, eps=EPS, weight_decay=WD,
                   first_block=first_block)
    d.tensors = C.addressof(row)
    capi.check(capi.load().kvae_adamw_step(C.byref(d), torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    return before, [m[0], v[0]]


@pytest.mark.parametrize("first_block", [0, 1000, (1 << 24) - 3, 1 << 24, (1 << 24) + 1000, (3 << 24) + 7, 1 << 31])
def test_codes_follow_the_rule(first_block):
    n = 5000                                     # (one case begins three blocks before the border)
    (m0, r0, g), got = call(n, first_block)
    m1 = m0 * B1 + g * (1 - B1)
    root = torch.sqrt((r0 * r0) * B2 + (g * g) * (1 - B2))
    index = 256 * first_block + torch.arange(5120, device="cuda")
    h = torch.zeros_like(index)
    for high in (index >> 32).unique().tolist():
        # hashed() takes the seed and adds the step's share of the key to it
        seed = (key_of(high) - STEP * 0x9E3779B9) & LOW
        h = torch.where(index >> 32 == high, hashed(index & LOW, seed, STEP), h)
    for state, want in ((got[0], codes_of(m1, h & 0xFFFF, False)), (got[1], codes_of(root, h >> 16, True))):
        assert torch.equal(state[1], want[1]) and torch.equal(state[0].view(torch.uint8), want[0].view(torch.uint8)[:n])


def test_elements_apart_draw_different_bits():
    """4096 states between two codes, rounded with the bits of four places 2^32 elements apart: each pair
    agrees about as often as chance has it."""
    codes = [call(4096, k << 24)[1][0][0].view(torch.uint8) for k in range(4)]
    for i in range(4):
        for j in range(i):
            assert 0.01 < float((codes[i] != codes[j]).double().mean()) < 0.6
