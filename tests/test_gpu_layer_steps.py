"""A decoder layer on packed weights with everything between its projections from this package: a prompt at once, the same tokens in
chunks and one by one over a paged cache, and the layer in 64 bits."""
import pytest
import torch

from oracle import gguf_oracle as go
from sensenova_u1_amd import FusedProjections, GGUFLinear, GGUFParameter, PagedKVCache, RotaryTable, gated_mlp, ops, paged_attention, prompt_attention, rotary, synthetic

from . import attention_oracle as ao

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, KV, DIM, INTER, EPS = 512, 8, 2, 64, 1024, 1e-6


def _linear(dev, n, k, seed):
    lin = GGUFLinear(k, n, bias=False, compute_dtype=torch.bfloat16, device="meta")
    lin.weight = GGUFParameter(synthetic.make_packed(go.Q8_0, n, k, seed=seed).to(dev), quant_type=go.Q8_0)
    return lin


class _Layer:
    def __init__(self, dev):
        q, k, v = (_linear(dev, n * DIM, HIDDEN, 20 + i) for i, n in enumerate((HEADS, KV, KV)))
        self.plain = [q, k, v]
        self.qkv = FusedProjections([q, k, v])
        self.o = _linear(dev, HIDDEN, HEADS * DIM, 30)
        self.gate, self.up, self.down = _linear(dev, INTER, HIDDEN, 31), _linear(dev, INTER, HIDDEN, 32), _linear(dev, HIDDEN, INTER, 33)
        gen = torch.Generator().manual_seed(34)
        self.norm1, self.norm2 = ((1 + 0.1 * torch.randn(HIDDEN, generator=gen)).to(torch.bfloat16).to(dev) for _ in range(2))
        self.table = RotaryTable.for_model(DIM, 10000.0, device=dev)

    def project(self, x):
        return (y.view(len(x), -1, DIM) for y in self.qkv(x, self.norm1, EPS))

    def finish(self, x, attended):
        x = self.o.forward_residual(attended.reshape(len(x), -1), x)
        return gated_mlp(x, self.gate, self.up, self.down, self.norm2, EPS, residual=x)

    def prompt(self, x, ends, positions):
        q, k, v = self.project(x)
        q, k = rotary(q, k, positions, self.table)
        return self.finish(x, prompt_attention(q, k, v, ends))

    def step(self, x, cache, positions, slots, pages, lens, ends, max_new):
        q, k, v = self.project(x)
        q = cache.write_rotary(q, k, v, positions, self.table, slots)
        return self.finish(x, paged_attention(q, cache, pages, lens, ends, max_new=max_new))

    def exact(self, x, lens):
        """In 64 bits, on the CPU, every sequence from position 0."""
        def weight(m):
            return go.dequantize_gguf_tensor(m.weight.as_tensor().cpu(), go.Q8_0, go.NUM_UPSTREAM_FP16).to(torch.bfloat16).double()

        def norm(x, g):
            return x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * g.double().cpu()

        x = x.double().cpu()
        n = norm(x, self.norm1)
        q, k, v = ((n @ weight(m).T).view(len(x), -1, DIM) for m in self.plain)
        positions = torch.cat([torch.arange(m) for m in lens])
        q, k = (ao.turned(y, positions, self.table.turns) for y in (q, k))
        out, at = [], 0
        for m in lens:
            out.append(ao.attention(q[at:at + m], k[at:at + m], v[at:at + m])[0])
            at += m
        x = x + torch.cat(out).flatten(1) @ weight(self.o).T
        n = norm(x, self.norm2)
        return x + (torch.nn.functional.silu(n @ weight(self.gate).T) * (n @ weight(self.up).T)) @ weight(self.down).T


@pytest.mark.parametrize("qt", [ops.BF16, ops.Q8_0])
def test_prompt_chunks_and_single_tokens_of_a_layer(dev, qt):
    layer, lens, page = _Layer(dev), [37, 5, 90], 16
    x = synthetic.make_activations(sum(lens), HIDDEN, seed=35).to(dev)
    want = layer.exact(x, lens)
    ends = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(dev)
    positions = torch.cat([torch.arange(n) for n in lens]).to(dev)
    whole = layer.prompt(x, ends, positions)
    # the norm, three projections, the turned pair, attention's weights and result, the residual, and the MLP's five values are rounded
    # to bf16, each by 2^-8 of itself at most; an 8-bit cache holds runs to 1 / 254 of their largest element besides
    bound = 12 * 2.0 ** -8
    assert go.rel_l2(whole.cpu().float(), want.float()) <= bound

    cache = PagedKVCache.empty(12, KV, page, DIM, qt, dev)
    order = torch.randperm(12, generator=torch.Generator().manual_seed(36))
    pages = torch.zeros((3, 6), dtype=torch.int64)
    pages[0, :3], pages[1, :1], pages[2, :6] = order[:3], order[3:4], order[4:10]
    done, got = [0, 0, 0], [[], [], []]
    # chunks of all three, then single tokens
    for new in ([20, 3, 1], [1, 1, 33], [14, 0, 40]) + ([1, 1, 1],) * 16:
        new = [min(n, m - d) for n, m, d in zip(new, lens, done)]
        if not any(new):
            continue
        rows, at, slots = [], [], []
        for i, n in enumerate(new):
            t = torch.arange(done[i], done[i] + n)
            rows.append(x[sum(lens[:i]) + done[i]:sum(lens[:i]) + done[i] + n])
            at.append(t)
            slots.append(pages[i][t // page] * page + t % page)
            done[i] += n
        y = layer.step(torch.cat(rows), cache, torch.cat(at).to(dev), torch.cat(slots).to(dev), pages.int().to(dev), torch.tensor(done, dtype=torch.int32, device=dev),
                       torch.tensor([0] + new).cumsum(0).to(torch.int32).to(dev), max(new))
        for i, part in enumerate(y.split(new)):
            got[i].append(part)
    assert done == lens
    stepped = torch.cat([p for parts in got for p in parts])
    if qt == ops.Q8_0:
        bound += 2 / 254
    assert go.rel_l2(stepped.cpu().float(), want.float()) <= bound
