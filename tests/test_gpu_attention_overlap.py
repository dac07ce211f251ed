"""Calls whose output or in-place rows share memory with an input at an offset are refused; interleaved ones that share none are taken."""
import pytest
import torch

from sensenova_u1_amd import PagedKVCache, RotaryTable, ops, paged_attention, prompt_attention, rotary

pytestmark = pytest.mark.gpu


def _values(gen, *shape):
    return torch.randn(shape, generator=gen).to(torch.bfloat16)


def test_overlapping_calls_are_refused(dev):
    x = torch.zeros((8, 12, 64), dtype=torch.bfloat16, device=dev)
    table, positions = RotaryTable.for_model(64, device=dev), torch.arange(8, device=dev)
    ends = torch.tensor([0, 8], dtype=torch.int32, device=dev)
    refused = [lambda: rotary(x[:, :4], x[:, 2:6], positions, table, inplace=True), lambda: rotary(x[:, :4], x[:, 3:4], positions, table, inplace=True),
               lambda: rotary(x[..., :32], x[:, :, 16:48], positions, table, inplace=True)]
    # over the queries, the keys, the values, by one head or by half of one
    for q, k, v, out in ((x[:, :8], x[:, 9:10], x[:, 10:11], x[:, 1:9]), (x[:, :4], x[:, 6:8], x[:, 8:10], x[:, 7:11]), (x[:, :4], x[:, 4:6], x[:, 9:11], x[:, 6:10]),
                         (x[:, :4, :32], x[:, 8:, :32], x[:, 8:, 32:], x[:, :4, 16:48])):
        refused.append(lambda q=q, k=k, v=v, out=out: prompt_attention(q, k, v, ends, out=out))
    for qt in (ops.BF16, ops.Q8_0):
        cache = PagedKVCache.empty(4, 2, 16, 64, qt, dev)
        pages, lens = torch.zeros((1, 4), dtype=torch.int32, device=dev), torch.tensor([8], dtype=torch.int32, device=dev)
        refused.append(lambda c=cache: c.write_rotary(x[:, :4], x[:, 3:5], x[:, 6:8], positions, table, positions, inplace=True))
        refused.append(lambda c=cache: c.write_rotary(x[:, :4], x[:, 6:8], x[:, 2:4], positions, table, positions, inplace=True))
        refused.append(lambda c=cache, p=pages, n=lens: paged_attention(x[:, :4], c, p, n, ends, out=x[:, 2:6]))
        room = cache.v.view(-1).view(torch.bfloat16)
        inside = room[64:64 + 8 * 4 * 64].view(8, 4, 64) if qt == ops.BF16 else room[1024:1024 + 2 * 4 * 64].view(2, 4, 64)
        n = len(inside)
        refused.append(lambda c=cache, p=pages, i=inside, n=n: paged_attention(x[:n, :4], c, p, torch.tensor([n], dtype=torch.int32, device=dev),
                                                                               torch.tensor([0, n], dtype=torch.int32, device=dev), out=i))
    for i, call in enumerate(refused):
        with pytest.raises(ops.SnGgufError, match="overlap|share"):
            call()
            pytest.fail(f"call {i} was taken")


def test_interleaved_views_are_taken(dev):
    gen = torch.Generator().manual_seed(0)
    table, positions = RotaryTable.for_model(64, device=dev), torch.arange(40, device=dev)
    ends = torch.tensor([0, 40], dtype=torch.int32, device=dev)
    for pick in (lambda x: (x[:, :8], x[:, 8:10], x[:, 10:12]), lambda x: (x[:, 0:8:2], x[:, 1:4:2], x[:, 5:8:2]),
                 lambda x: (x[:, 4:8], x[:, 2:4], x[:, 0:2])):
        x = _values(gen, 40, 12, 64).to(dev)
        q, k, v = pick(x)
        want = rotary(q, k, positions, table)
        out = prompt_attention(*want, v, ends)
        cache = PagedKVCache.empty(3, 2, 16, 64, ops.BF16, dev)
        whole = x.clone()
        a, b, c = pick(whole)
        got = cache.write_rotary(a, b, c, positions, table, positions, inplace=True)
        assert torch.equal(got, want[0]) and torch.equal(b, k)
        whole = x.clone()
        a, b, c = pick(whole)
        got = rotary(a, b, positions, table, inplace=True)
        assert torch.equal(a, want[0]) and torch.equal(b, want[1]) and torch.equal(c, v)
        room = torch.empty((40, 2 * q.shape[1], 64), dtype=x.dtype, device=dev)
        room[:, ::2] = want[0]
        prompt_attention(room[:, ::2], want[1], v, ends, out=room[:, 1::2])
        assert torch.equal(room[:, 1::2], out)
