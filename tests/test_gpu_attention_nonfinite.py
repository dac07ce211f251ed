"""Infinities and NaN among keys and values reach the queries that see them and no others; values at the end of bf16's range."""
import pytest
import torch

from sensenova_u1_amd import PagedKVCache, ops, paged_attention, prompt_attention

from . import attention_oracle as ao

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


def _values(gen, tokens, heads, dim):
    return torch.randn((tokens, heads, dim), generator=gen).to(torch.bfloat16)


def _ends(lens, dev):
    return torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(dev)


def _check(got, q, k, v, odd_k, odd_v, causal, window, operand=torch.bfloat16):
    """``k``, ``v``: finite, as they are but at the tokens odd_k and odd_v, where one element (8 bits: one run) of each head was not."""
    got = got.double().cpu()
    seen = ao.visible(len(q), len(k), causal, window)
    hit_k = seen[:, odd_k].any(1) if odd_k else torch.zeros(len(q), dtype=torch.bool)
    hit_v = seen[:, odd_v].any(1) if odd_v else torch.zeros(len(q), dtype=torch.bool)
    want, most = ao.attention(q, k, v, causal, window, None, operand)
    clean = ~(hit_k | hit_v)
    assert clean.any() or not (odd_k or odd_v)
    off = (got[clean] - want[clean]).abs()
    assert bool((off <= most[clean]).all()), f"{int((~(off <= most[clean])).sum())} values of rows that see none are off"
    assert bool((~torch.isfinite(got[hit_k])).all())                         # every element of a row with a score that is none
    assert bool((~torch.isfinite(got[hit_v][:, :, 3])).all())
    only = hit_v & ~hit_k
    elements = torch.arange(got.shape[2]) >= 32                              # (elements of other runs)
    off = (got[only] - want[only]).abs()[..., elements]
    assert bool((off <= most[only][..., elements]).all()), "elements beside those of a value that is not finite"


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 50), (False, 0)])
@pytest.mark.parametrize("what", [NAN, INF, -INF])
def test_prompt(dev, dim, causal, window, what):
    gen = torch.Generator().manual_seed(dim)
    for lens_q, lens_k in (([300], [300]), ([40, 20], [60, 400])):
        q, k, v = _values(gen, sum(lens_q), 4, dim), _values(gen, sum(lens_k), 2, dim), _values(gen, sum(lens_k), 2, dim)
        for odd in (lens_k[0] - 1, lens_k[0] - 30, 5):
            if not causal and odd != 5:
                continue
            bad = v.clone()
            bad[odd, :, 3] = what
            got = prompt_attention(q.to(dev), k.to(dev), bad.to(dev), _ends(lens_q, dev), _ends(lens_k, dev), causal=causal, window=window)
            n, m = lens_q[0], lens_k[0]
            if causal:
                hit = ao.visible(n, m, causal, window)[:, odd]
                if not bool((~hit).any()):
                    continue
                _check(got[:n], q[:n], k[:m], v[:m], [], [odd], causal, window)
            else:
                assert bool((~torch.isfinite(got[:n, :, 3])).all())
            if len(lens_q) > 1:
                _check(got[n:], q[n:], k[m:], v[m:], [], [], causal, window)


def test_prompt_keys(dev):
    gen = torch.Generator().manual_seed(1)
    q, k, v = _values(gen, 200, 4, 128), _values(gen, 200, 2, 128), _values(gen, 200, 2, 128)
    bad = k.clone()
    bad[150, :, 3] = NAN
    got = prompt_attention(q.to(dev), bad.to(dev), v.to(dev), _ends([200], dev))
    _check(got, q, k, v, [150], [], True, 0)


@pytest.mark.parametrize("tokens", [1, 30, 200])
def test_prompt_split_over_workgroups(dev, tokens):
    """An infinity that only the last rows see, where a sequence's keys are split."""
    gen = torch.Generator().manual_seed(2)
    q, k, v = _values(gen, tokens, 4, 128), _values(gen, 9000, 2, 128), _values(gen, 9000, 2, 128)
    assert ops.load_library().sngguf_attention_workspace_bytes(tokens, 9000, 1, 4, 2, 128) > 0
    bad = v.clone()
    odd = [8990, 8999] if tokens > 20 else []
    bad[odd, :, 3] = INF
    bad[:1001 - tokens] = NAN
    got = prompt_attention(q.to(dev), k.to(dev), bad.to(dev), _ends([tokens], dev), _ends([9000], dev), window=8000)
    _check(got, q, k, v, [], odd, True, 8000)


@pytest.mark.parametrize("qt", [ops.Q8_0, ops.BF16])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("new,length,window", [(1, 700, 100), (3, 700, 100), (1, 6000, 5000), (7, 90, 0), (150, 400, 0), (150, 400, 60), (60, 9000, 8000)])
def test_paged(dev, qt, dim, new, length, window):
    """NaN in every value in front of the first that any row sees, in every key there, and in the last token."""
    gen = torch.Generator().manual_seed(new + length)
    page, heads, kv_heads = 16, 4, 2
    q, k, v = _values(gen, new, heads, dim), _values(gen, length, kv_heads, dim), _values(gen, length, kv_heads, dim)
    pages = -(-length // page) + 1
    order = torch.randperm(pages - 1, generator=gen) + 1
    table = order[None].int()
    cache = PagedKVCache.empty(pages, kv_heads, page, dim, qt, dev)
    for t in (cache.k, cache.v, cache.k_scale, cache.v_scale):
        if t is not None:
            t.fill_(-128) if t.dtype == torch.int8 else t.fill_(NAN)
    first = max(0, length - new + 1 - window) if window else 0
    odd = [length - 1] if new > 1 else []
    bad_k, bad_v = k.clone(), v.clone()
    bad_k[:first], bad_v[:first] = NAN, NAN
    bad_v[odd, :, 3] = NAN
    t = torch.arange(length)
    cache.write(bad_k.to(dev), bad_v.to(dev), (table[0].long()[t // page] * page + t % page).to(dev))
    table[:, :first // page] = -1                                            # pages given back: read as page 0, which holds NaN
    got = paged_attention(q.to(dev), cache, table.to(dev), torch.tensor([length], dtype=torch.int32, device=dev), _ends([new], dev), max_new=new, window=window)
    if qt == ops.Q8_0:
        k, v = ao.quantised(k)[2], ao.quantised(v)[2]
    _check(got, q, k, v, [], odd, True, window, torch.float16 if qt == ops.Q8_0 else torch.bfloat16)


def test_values_at_the_end_of_the_range(dev):
    """Masked places with the type's lowest value; values whose sum, though not their average, is beyond fp32."""
    gen = torch.Generator().manual_seed(3)
    low = torch.finfo(torch.bfloat16).min
    q, k, v = _values(gen, 130, 4, 128), _values(gen, 130, 2, 128), _values(gen, 130, 2, 128)
    bad_k, bad_v = k.clone(), v.clone()
    bad_k[100:], bad_v[100:] = low, low
    got = prompt_attention(q.to(dev), bad_k.to(dev), bad_v.to(dev), _ends([130], dev))
    want, most = ao.attention(q[:100], k[:100], v[:100])
    assert bool(((got[:100].double().cpu() - want).abs() <= most).all())
    big = (v.clamp(-1, 1).float() * 2.0 ** 127).to(torch.bfloat16)
    got = prompt_attention(q.to(dev), k.to(dev), big.to(dev), _ends([130], dev))
    want, most = ao.attention(q, k, big)
    assert bool(((got.double().cpu() - want).abs() <= most).all())
    cache = PagedKVCache.empty(9, 2, 16, 128, ops.BF16, dev)
    cache.write(k.to(dev), big.to(dev), torch.arange(130, device=dev))
    table = torch.arange(9, dtype=torch.int32, device=dev)[None]
    got = paged_attention(q[129:].to(dev), cache, table, torch.tensor([130], dtype=torch.int32, device=dev))
    want, most = ao.attention(q[129:], k, big)
    assert bool(((got.double().cpu() - want).abs() <= most).all())


@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
def test_many_rows(dev, dim):
    gen = torch.Generator().manual_seed(dim)
    q, k, v = _values(gen, 1300, 16, dim), _values(gen, 1300, 16, dim), _values(gen, 1300, 16, dim)
    bad = v.clone()
    bad[[700, 1290], :, 3] = torch.tensor([INF, NAN], dtype=v.dtype)[:, None]
    got = prompt_attention(q.to(dev), k.to(dev), bad.to(dev), _ends([1300], dev))
    _check(got, q, k, v, [], [700, 1290], True, 0)
