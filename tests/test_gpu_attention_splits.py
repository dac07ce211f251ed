"""Rows whose keys are split over workgroups: queries and keys that are not finite."""
import pytest
import torch

from sensenova_u1_amd import PagedKVCache, ops, paged_attention, prompt_attention

from . import attention_oracle as ao

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")
HEADS, KV, DIM, KEYS, PAGE = 4, 2, 128, 9000, 64


def _values(gen, tokens, heads):
    return torch.randn((tokens, heads, DIM), generator=gen).to(torch.bfloat16)


def _ends(n, dev):
    return torch.tensor([0, n], dtype=torch.int32, device=dev)


def _packed(dev, q, k, v, **options):
    return prompt_attention(q.to(dev), k.to(dev), v.to(dev), _ends(len(q), dev), _ends(len(k), dev), **options)


def _paged(dev, q, k, v, qt=ops.BF16, **options):
    cache = PagedKVCache.empty(-(-len(k) // PAGE), KV, PAGE, DIM, qt, dev)
    for t in (cache.k, cache.v, cache.k_scale, cache.v_scale):
        if t is not None:
            t.zero_()
    cache.write(k.to(dev), v.to(dev), torch.arange(len(k), device=dev))
    pages = torch.arange(cache.pages, dtype=torch.int32, device=dev)[None]
    return paged_attention(q.to(dev), cache, pages, torch.tensor([len(k)], dtype=torch.int32, device=dev), _ends(len(q), dev), max_new=len(q), **options)


@pytest.mark.parametrize("keys", [40, KEYS])
@pytest.mark.parametrize("new", [1, 9, 30, 200])
@pytest.mark.parametrize("what", [NAN, INF])
def test_queries_that_are_not_finite(dev, keys, new, what):
    """Their rows are NaN wherever they see a key (an infinite element meets keys of both signs), however the keys are split; all others as ever."""
    gen = torch.Generator().manual_seed(new)
    q, k, v = _values(gen, new, HEADS), _values(gen, keys, KV), _values(gen, keys, KV)
    k[:, :, 9] = torch.where(torch.arange(keys)[:, None] % 2 == 0, 1.0, -1.0).to(k.dtype)
    bad = q.clone()
    rows = [new - 1] + ([new // 2] if new > 1 and keys >= new else [])
    bad[rows, 1, 9] = what
    for qt in (None, ops.BF16, ops.Q8_0):
        got = (_packed(dev, bad, k, v) if qt is None else _paged(dev, bad, k, v, qt)).double().cpu()
        held = [ao.quantised(x)[2] for x in (k, v)] if qt == ops.Q8_0 else (k, v)
        want, most = ao.attention(q, *held, operand=torch.float16 if qt == ops.Q8_0 else torch.bfloat16)
        odd = torch.zeros((new, HEADS), dtype=torch.bool)
        odd[rows, 1] = True
        assert bool(torch.isnan(got[odd]).all()), (qt, got[odd].unique()[:4])
        assert bool(((got - want).abs() <= most)[~odd].all()), qt


@pytest.mark.parametrize("keys", [40, KEYS])
@pytest.mark.parametrize("new", [1, 30])
def test_keys_that_are_all_nan(dev, keys, new):
    gen = torch.Generator().manual_seed(new)
    q, k, v = _values(gen, new, HEADS), _values(gen, keys, KV), _values(gen, keys, KV)
    k[:, 1] = NAN
    for call in (_packed, _paged):
        got = call(dev, q, k, v).cpu()
        assert bool(torch.isnan(got[:, 2:]).all()) and bool(torch.isfinite(got[:, :2].float()).all())
