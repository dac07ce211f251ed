"""Rotation of keys alone: queries without heads."""
import pytest
import torch

from sensenova_u1_amd import RotaryTable, rotary

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens", [0, 1, 37])
def test_no_query_heads(dev, tokens, interleaved):
    gen = torch.Generator().manual_seed(tokens)
    table = RotaryTable.for_model(64, interleaved=interleaved, device=dev)
    positions = torch.arange(tokens, device=dev) + 3
    k = torch.randn((tokens, 3, 64), generator=gen).to(torch.bfloat16).to(dev)
    none = k[:, :0]
    want = rotary(k, None, positions, table)[0]
    # (memory of the size that the result takes is given back with other values in it)
    torch.full_like(k, 9.0)
    q2, k2 = rotary(none, k, positions, table)
    assert q2.shape == (tokens, 0, 64) and torch.equal(k2, want)
    q2, k2 = rotary(k, none, positions, table)
    assert torch.equal(q2, want) and k2.shape == (tokens, 0, 64)
    assert rotary(none, None, positions, table)[0].shape == (tokens, 0, 64) and rotary(none, none, positions, table)[1].shape == (tokens, 0, 64)
    own = k.clone()
    q2, k2 = rotary(own[:, :0], own, positions, table, inplace=True)
    assert k2.data_ptr() == own.data_ptr() and torch.equal(own, want)
