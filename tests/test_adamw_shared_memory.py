"""Optimiser lists over memory that several storages share (a buffer or a tensor handed over by another
library): what overlaps is refused, whatever storage it is seen through."""
import pytest
import torch

from kalman_vae_amd import adamw_step


def from_buffer(device):
    memory = bytearray(64 * 4)
    return lambda first, n: torch.frombuffer(memory, dtype=torch.float32, offset=4 * first, count=n)


def from_dlpack(device):
    memory = torch.zeros(64, device=device)
    return lambda first, n: torch.from_dlpack(memory[first:first + n])


def beside_its_owner(device):
    memory = torch.zeros(64, device=device)
    views = []

    def piece(first, n):
        views.append(memory[first:first + n] if len(views) % 2 == 0 else torch.from_dlpack(memory[first:first + n]))
        return views[-1]
    return piece


KINDS = [("cpu", from_buffer), ("cpu", from_dlpack), ("cpu", beside_its_owner)]
KINDS += [pytest.param("cuda", k, marks=pytest.mark.gpu) for k in (from_dlpack, beside_its_owner)]


@pytest.mark.parametrize("device,kind", KINDS)
def test_overlap_across_storages(device, kind):
    z = lambda n: torch.zeros(n, device=device)  # noqa: E731
    piece = kind(device)
    a, b = piece(0, 20), piece(10, 20)
    assert a.untyped_storage().data_ptr() != b.untyped_storage().data_ptr() or kind is not from_buffer
    for params, m in (([a, b], [z(20), z(20)]), ([b, a], [z(20), z(20)]), ([a, z(20)], [z(20), b])):
        with pytest.raises(ValueError, match="share memory"):
            adamw_step(params, [z(20), z(20)], m, [z(20), z(20)], 1)


@pytest.mark.parametrize("device,kind", KINDS)
def test_neighbours_pass(device, kind):
    z = lambda n: torch.zeros(n, device=device)  # noqa: E731
    piece = kind(device)
    a, b = piece(20, 20), piece(0, 20)
    if device == "cpu":                                            # (past the check of the lists)
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            adamw_step([a, b], [z(20), z(20)], [z(20), z(20)], [z(20), z(20)], 1)
        return
    adamw_step([a, b], [z(20) + 1, z(20) + 1], [z(20), z(20)], [z(20), z(20)], 1, lr=0.5, weight_decay=0.0)
    for t in (a, b):                                               # the first step moves by lr (eps apart)
        assert float((t + 0.5).abs().max()) < 1e-6
