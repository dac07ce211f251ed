"""A captured decoder layer, projections to MLP, replayed over growing sequences: every replay is what the same calls give outside the graph."""
import pytest
import torch

from sensenova_u1_amd import PagedKVCache, ops

from .test_gpu_layer_steps import DIM, HIDDEN, KV, _Layer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("qt", [ops.BF16, ops.Q8_0])
@pytest.mark.parametrize("new", [[1], [1, 1, 1], [1, 40, 3]])
def test_replays_of_a_layer_step(dev, qt, new):
    layer, page, width, n = _Layer(dev), 16, 40, len(new)
    gen = torch.Generator().manual_seed(sum(new))
    tokens = sum(new)
    caches = [PagedKVCache.empty(n * width, KV, page, DIM, qt, dev) for _ in range(2)]
    for c in caches:
        for t in (c.k, c.v, c.k_scale, c.v_scale):
            if t is not None:
                t.zero_()
    x = torch.zeros((tokens, HIDDEN), dtype=torch.bfloat16, device=dev)
    positions, slots = (torch.zeros(tokens, dtype=torch.int64, device=dev) for _ in range(2))
    pages = torch.zeros((n, width), dtype=torch.int32, device=dev)
    lens = torch.ones(n, dtype=torch.int32, device=dev)
    ends = torch.tensor([0] + new).cumsum(0).to(torch.int32).to(dev)

    def step(cache):
        return layer.step(x, cache, positions, slots, pages, lens, ends, max(new))

    step(caches[0])                                                          # (kernels are loaded, stacked weights laid out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(caches[0])
    order = torch.randperm(n * width, generator=gen).view(n, width)
    pages.copy_(order.int())
    have = [0] * n
    for replay in range(5):
        # the sequences' new tokens, and now and then others in between that came another way
        at = []
        for i, m in enumerate(new):
            have[i] += m + (37 * i + 50 if replay in (1, 3) else 0)
            at.append(torch.arange(have[i] - m, have[i]))
        positions.copy_(torch.cat(at))
        slots.copy_(torch.cat([order[i][t // page] * page + t % page for i, t in enumerate(at)]))
        lens.copy_(torch.tensor(have, dtype=torch.int32))
        x.copy_(torch.randn((tokens, HIDDEN), generator=gen).to(torch.bfloat16))
        graph.replay()
        eager = step(caches[1])
        torch.cuda.synchronize()
        assert torch.equal(captured, eager) and bool(torch.isfinite(eager.float()).all()) and bool((eager != x).any()), replay
        for a, b in ((caches[0].k, caches[1].k), (caches[0].v, caches[1].v), (caches[0].k_scale, caches[1].k_scale)):
            assert a is None or torch.equal(a, b), replay
