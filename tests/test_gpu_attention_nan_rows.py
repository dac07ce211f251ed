"""A model that has gone NaN: all rows are done again, and none takes long."""
import pytest
import torch

from sensenova_u1_amd import prompt_attention

pytestmark = pytest.mark.gpu


def _time(call):
    best = float("inf")
    for _ in range(3):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        call()
        end.record()
        torch.cuda.synchronize()
        best = min(best, start.elapsed_time(end))
    return best


@pytest.mark.parametrize("what", ["queries", "first key", "first value", "everything"])
def test_prompt(dev, what):
    """A row takes one look at 64 keys more; key by key over all it sees, 4096 tokens would take 500 times as long as finite ones."""
    gen = torch.Generator(device=dev).manual_seed(0)
    tokens = 4096
    q, k, v = (torch.randn((tokens, h, 128), generator=gen, device=dev).to(torch.bfloat16) for h in (32, 8, 8))
    ends = torch.tensor([0, tokens], dtype=torch.int32, device=dev)
    assert bool(torch.isfinite(prompt_attention(q, k, v, ends).float()).all())
    usual = _time(lambda: prompt_attention(q, k, v, ends))
    nan = float("nan")
    if what in ("queries", "everything"):
        q[:] = nan
    if what in ("first key", "everything"):
        k[0] = nan
    if what in ("first value", "everything"):
        v[0] = nan
    assert bool(torch.isnan(prompt_attention(q, k, v, ends)).all())
    assert _time(lambda: prompt_attention(q, k, v, ends)) < 100 * usual
