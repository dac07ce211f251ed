"""Every pair of a stretched table against the definition, in plain numbers."""
import math

import pytest
import torch

from sensenova_u1_amd import RotaryTable

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,base,factor,context,fast,slow", [(128, 1e6, 4.0, 32768, 32.0, 1.0), (64, 10000.0, 8.0, 4096, 32.0, 1.0), (128, 5e6, 16.0, 40960, 24.0, 2.0),
                                                               (64, 10000.0, 0.5, 2048, 32.0, 1.0), (8, 100.0, 2.0, 64, 32.0, 1.0)])
def test_ramp(dev, dim, base, factor, context, fast, slow):
    """A pair i turns context base^(-2 i / dim) / (2 pi) times over the context.  Solved for i, `fast` and `slow` turns are the places between which (the first
    rounded down, the second up) the stretch grows linearly with i from none to `factor`."""
    table = RotaryTable.for_model(dim, base, scaling="yarn", factor=factor, original_context=context, beta_fast=fast, beta_slow=slow, device=dev)
    place = [dim * math.log(context / (2 * math.pi * turns)) / (2 * math.log(base)) for turns in (fast, slow)]
    low, high = max(0, math.floor(place[0])), min(dim - 1, math.ceil(place[1]))
    assert low < high
    between = 0
    for i, got in enumerate(table.turns.tolist()):
        plain = base ** (-2 * i / dim) / (2 * math.pi)
        part = min(1.0, max(0.0, (i - low) / (high - low)))
        between += 0 < part < 1
        assert got == pytest.approx((1 - part) * plain + part * plain / factor, rel=1e-12), i
    assert between > 0
    assert table.magnitude == pytest.approx(0.1 * math.log(factor) + 1 if factor > 1 else 1.0)


def test_magnitude_and_layout_as_given(dev):
    table = RotaryTable.for_model(64, scaling="yarn", factor=4.0, original_context=4096, magnitude=0.75, interleaved=True, device=dev)
    assert table.magnitude == 0.75 and table.interleaved
    plain = RotaryTable.for_model(64, device=dev)
    assert torch.equal(RotaryTable.for_model(64, factor=7.0, device=dev).turns, plain.turns)      # (without a scaling the factor is not used)
