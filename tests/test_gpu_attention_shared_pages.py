"""Sequences whose tables hold the same pages: a common prompt, the same page at other places, a whole table in common."""
import pytest
import torch

from sensenova_u1_amd import PagedKVCache, ops, paged_attention

from . import attention_oracle as ao

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("qt", [ops.Q8_0, ops.BF16])
@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("count,common,new", [(3, 1024, 1), (5, 4096, 3), (70, 64, 1), (2, 0, 1), (4, 320, 40)])
def test_shared_pages(dev, qt, dim, count, common, new):
    gen = torch.Generator().manual_seed(count + common)
    page, heads, kv_heads, pages = 16, 4, 2, common // 16 + 20
    cache = PagedKVCache.empty(pages, kv_heads, page, dim, qt, dev)
    k, v = (torch.randn((pages * page, kv_heads, dim), generator=gen).to(torch.bfloat16) for _ in range(2))
    cache.write(k.to(dev), v.to(dev), torch.arange(pages * page, device=dev))
    if qt == ops.Q8_0:
        k, v = ao.quantised(k)[2], ao.quantised(v)[2]
    order = torch.randperm(pages, generator=gen)
    first = common // page
    # the common prompt, then some of twenty pages in an order of its own: other sequences have them at the same places or at others
    table = torch.stack([torch.cat([order[:first], order[first:][torch.randperm(20, generator=gen)[:5]]]) for _ in range(count)])
    table[-1] = table[0]
    lens = torch.randint(common + new, common + 80, (count,), generator=gen)
    lens[-1] = lens[0]
    q = torch.randn((count, new, heads, dim), generator=gen).to(torch.bfloat16)
    q[-1] = q[0]
    ends = torch.arange(0, count * new + 1, new, dtype=torch.int32, device=dev)
    got = paged_attention(q.flatten(0, 1).to(dev), cache, table.int().to(dev), lens.int().to(dev), ends, max_new=new).view(q.shape).cpu()
    assert torch.equal(got[-1], got[0])
    for i in range(0, count, 1 if count < 10 else 9):
        t = torch.arange(int(lens[i]))
        slots = table[i][t // page] * page + t % page
        want, most = ao.attention(q[i], k[slots], v[slots], operand=torch.float16 if qt == ops.Q8_0 else torch.bfloat16)
        assert bool(((got[i].double() - want).abs() <= most).all()), i
