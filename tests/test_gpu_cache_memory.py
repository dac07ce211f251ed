"""Caches over memory that the caller has: halves that share some, and tokens copied from one place of a cache to another."""
import pytest
import torch

from sensenova_u1_amd import PagedKVCache, RotaryTable, ops, paged_attention

pytestmark = pytest.mark.gpu


def test_keys_and_values_in_one_memory_are_not_written(dev):
    gen = torch.Generator().manual_seed(0)
    x = torch.randn((16, 2, 64), generator=gen).to(torch.bfloat16).to(dev)
    slots, table = torch.arange(16, device=dev), RotaryTable.for_model(64, device=dev)
    room = torch.zeros((5, 2, 16, 64), dtype=torch.bfloat16, device=dev)
    bytes_, scales = torch.zeros((5, 2, 16, 64), dtype=torch.int8, device=dev), torch.zeros((5, 2, 2, 16), dtype=torch.float16, device=dev)
    for cache in (PagedKVCache(room, room), PagedKVCache(room[:4], room[1:]), PagedKVCache(room[2:], room[:3]),
                  PagedKVCache(bytes_, bytes_, scales, scales.clone()), PagedKVCache(bytes_, bytes_.clone(), scales, scales), PagedKVCache(bytes_[:4], bytes_[1:], scales[:4], scales[:4].clone())):
        for call in (lambda: cache.write(x, x, slots), lambda: cache.write_rotary(x, x, x, slots, table, slots)):
            with pytest.raises(ops.SnGgufError, match="share memory"):
                call()
    for cache in (PagedKVCache(room[:2], room[2:4]), PagedKVCache(bytes_[:2], bytes_[2:4], scales[:2], scales[2:4])):
        cache.write(x, x, slots)
        assert torch.equal(cache.read(slots)[0], cache.read(slots)[1])
    # one memory for both is read as it is
    cache = PagedKVCache(room[:1], room[:1])
    out = paged_attention(x[:1], cache, torch.zeros((1, 1), dtype=torch.int32, device=dev), torch.tensor([16], dtype=torch.int32, device=dev))
    k, v = cache.read(slots)
    assert torch.equal(k, v) and torch.equal(out, paged_attention(x[:1], PagedKVCache(room[:1], room[2:3]), torch.zeros((1, 1), dtype=torch.int32, device=dev),
                                                                  torch.tensor([16], dtype=torch.int32, device=dev)))


def test_tokens_from_one_page_to_another(dev):
    gen = torch.Generator().manual_seed(1)
    cache = PagedKVCache.empty(3, 2, 16, 64, ops.BF16, dev)
    k, v = (torch.randn((16, 2, 64), generator=gen).to(torch.bfloat16).to(dev) for _ in range(2))
    cache.write(k, v, torch.arange(16, device=dev))
    cache.write(cache.k[0].transpose(0, 1), cache.v[0].transpose(0, 1), torch.arange(32, 48, device=dev))
    got = cache.read(torch.arange(32, 48, device=dev))
    assert torch.equal(got[0], k) and torch.equal(got[1], v)
