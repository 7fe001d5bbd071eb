"""Rows so long that the 32 slices of a row hold more than a workgroup loads at once: which tokens stay, exactly."""
from __future__ import annotations

import pytest
import torch

from compactattention_amd import ops
from tests.test_gpu_evict import masses, want_keep

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["spread", "ties", "equal", "close", "odd"])
@pytest.mark.parametrize("lens,Hkv,budget,sinks,recent", [
    ([262145], 1, 4096, 4, 1024),  # slices of 8256
    ([270001, 9000, 16385], 1, 20001, 64, 5),
    ([600000], 1, 599990, 0, 0),
])
def test_slices_of_several_loads(kind, lens, Hkv, budget, sinks, recent):
    mass = masses(len(lens) * Hkv, max(lens) + 3, kind, seed=budget)
    keep = ops.heavy_tokens(mass, lens, Hkv, budget, sinks, recent)
    assert torch.equal(keep.cpu(), want_keep(mass, lens, Hkv, budget, sinks, recent))


def test_weights_of_zero_in_long_slices():
    g = torch.Generator().manual_seed(3)
    n = 540000
    some = (torch.rand((2, n // 64 + 1), generator=g) < 0.1).repeat_interleave(64, 1)[:, :n]
    mass = (masses(2, n, "spread", 4).cpu() * some).cuda()
    for budget in (5000, 100000):  # within the weights that are not 0, and past them
        keep = ops.heavy_tokens(mass, n, 2, budget, 4, 100)
        assert torch.equal(keep.cpu(), want_keep(mass, [n], 2, budget, 4, 100)), budget
