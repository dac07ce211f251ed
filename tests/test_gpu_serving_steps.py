"""Requests that begin with one prompt, served together: tables of the step, heads normed and turned into the cache, attention over what they have in
common and over their own, until they end and others take their pages; every step against 64 bits."""
import pytest
import torch

from sensenova_u1_amd import HeadNorm, PagedKVCache, PageTables, RotaryAxes, ops, paged_attention, rotary, shared_prefix_attention

from . import attention_oracle as ao
from . import head_oracle as ho

pytestmark = pytest.mark.gpu

HEADS, KV, DIM, PAGE, SEQUENCES = 8, 2, 64, 16, 6
WIDTH = -(-(50 << 20) // (SEQUENCES * KV * DIM * PAGE))      # so many keys could there be that the groups count
PARTS, EPS = [(32, 0, 1e5), (16, 1, 1e4), (16, 2, 1e4)], 1e-6


class Service:
    def __init__(self, dev, qt, pages=200):
        self.dev, self.gen = dev, torch.Generator().manual_seed(qt)
        self.tables = PageTables.empty(SEQUENCES, WIDTH, pages, PAGE, dev)
        self.cache = PagedKVCache.empty(pages, KV, PAGE, DIM, qt, dev)
        for t in (self.cache.k, self.cache.v, self.cache.k_scale, self.cache.v_scale):
            if t is not None:
                t.fill_(-128 if t.dtype == torch.int8 else float("nan"))       # what was never written may be anything
        self.table = RotaryAxes.for_model(PARTS, device=dev)
        self.weights = [[(1 + 0.3 * torch.randn(32, generator=self.gen)).to(torch.bfloat16) for _ in range(2)] for _ in range(2)]
        self.q_norm, self.k_norm = (HeadNorm(*(w.to(dev) for w in half), eps=EPS) for half in self.weights)
        self.history = [[] for _ in range(SEQUENCES)]                            # (k, v) of each token, as the cache is to hold them
        self.operand = torch.float16 if qt == ops.Q8_0 else torch.bfloat16

    def ints(self, values):
        return torch.tensor(values, dtype=torch.int32, device=self.dev)

    def tokens(self, count):
        return torch.randn((count, HEADS + 2 * KV, DIM), generator=self.gen).to(torch.bfloat16)

    def three(self, positions):
        """Text: the place in it, and the first row and column."""
        out = torch.zeros((3, positions.shape[0]), dtype=torch.int64, device=self.dev)
        out[0] = positions
        return out

    def device_step(self, qkv, new, groups, shared, tokens, max_new):
        step = self.tables.append(new, tokens)
        q, k, v = qkv.split([HEADS, KV, KV], 1)
        q = self.cache.write_rotary(q, k, v, self.three(step.positions), self.table, step.slots, q_norm=self.q_norm, k_norm=self.k_norm)
        return step, q, shared_prefix_attention(q, self.cache, self.tables.pages, step.lens, groups, shared, step.ends, max_new=max_new)

    def check(self, qkv, new, q, out, step):
        """q, out of a step of `new` tokens of each sequence, whose history grows by them."""
        assert step.missing.item() == 0 and step.ends.tolist() == [sum(new[:i]) for i in range(SEQUENCES + 1)]
        heads, axis = qkv.split([HEADS, KV, KV], 1), self.table.axis.cpu()
        row = 0
        for i, n in enumerate(new):
            rows = slice(row, row + n)
            at = torch.zeros((3, n), dtype=torch.int64)
            at[0] = len(self.history[i]) + torch.arange(n)
            want, most = ho.head(heads[0][rows], at, self.table.turns, axis, self.table.parts, weights=self.weights[0], eps=EPS)
            assert bool(((q[rows].double().cpu() - want).abs() <= most).all()), i
            # what the cache holds of the keys: as the operator gives them, which other tests hold to 64 bits
            turned = rotary(heads[1][rows].to(self.dev), None, at.to(self.dev), self.table, q_norm=self.k_norm)[0].cpu()
            for j in range(n):
                k, v = turned[j:j + 1], heads[2][row + j:row + j + 1]
                self.history[i].append((ao.quantised(k)[2], ao.quantised(v)[2]) if self.operand == torch.float16 else (k.double(), v.double()))
            if n:
                k, v = (torch.cat(x) for x in zip(*self.history[i]))
                want, most = ao.attention(q[rows], k, v, operand=self.operand)
                off = (out[rows].double().cpu() - want).abs()
                assert bool((off <= most).all()), (i, float((off / most).max()))
            row += n
        assert step.lens.tolist() == [len(h) for h in self.history]

    def step(self, new, groups, shared):
        qkv = self.tokens(sum(new))
        step, q, out = self.device_step(qkv.to(self.dev), self.ints(new), self.ints(groups), self.ints(shared), sum(new), max(new))
        self.check(qkv, new, q, out, step)
        return q, step

    def fork(self, parent, common):
        self.tables.fork(self.ints(parent), self.ints(common))
        for i, (p, n) in enumerate(zip(parent, common)):
            if p >= 0:
                self.history[i] = list(self.history[p][:n // PAGE * PAGE])

    def release(self, which):
        done = torch.zeros(SEQUENCES, dtype=torch.bool)
        done[which] = True
        self.tables.release(done.to(self.dev))
        for i in which:
            self.history[i] = []


BOTH = pytest.mark.parametrize("qt", [ops.BF16, ops.Q8_0])


@BOTH
def test_answers_to_one_prompt(dev, qt):
    s = Service(dev, qt)
    sizes = (4, SEQUENCES, 1, 1, WIDTH * PAGE, HEADS, KV, DIM, qt)
    lib = ops.load_library()
    assert lib.sngguf_shared_attention_workspace_bytes(*sizes) > lib.sngguf_paged_attention_workspace_bytes(*sizes[:2], *sizes[3:8])
    # the prompt, in two chunks; then four that answer it and one of another user
    s.step([300, 0, 0, 0, 0, 0], [0, 0], [0])
    s.step([131, 0, 0, 0, 0, 50], [0, 0], [0])
    s.fork([-1, 0, 0, 0, 0, -1], [0, 431, 431, 290, 431, 0])
    assert s.tables.lens.tolist() == [431, 416, 416, 288, 416, 50]
    for turn in range(20):
        new = [0, 1, 1 + turn % 3, 1, int(turn > 5), 1]
        q, step = s.step(new, [1, 5], [416] if turn % 2 else [10 ** 6])           # (what is said beyond what they have counts as far as they have it)
    # the same without groups
    want = paged_attention(q, s.cache, s.tables.pages, step.lens, step.ends)
    got = shared_prefix_attention(q, s.cache, s.tables.pages, step.lens, s.ints([1, 5]), s.ints([416]), step.ends)
    assert float((got.float() - want.float()).abs().max()) < 0.02
    # two end, another user's first prompt takes their pages; a new answer to the old prompt
    before = s.tables.cursor.tolist()
    s.release([1, 2])
    assert s.tables.cursor[1].item() > before[1]
    s.step([0, 90, 0, 1, 1, 1], [2, 5], [288])
    s.fork([-1, -1, 0, -1, -1, -1], [0, 0, 200, 0, 0, 0])
    for _ in range(3):
        s.step([0, 1, 2, 1, 1, 1], [0, 1, 2, 5, 6], [416, 0, 192, 0])
    s.release([2, 3, 4])
    s.release([0, 1, 5])
    assert s.tables.lens.tolist() == [0] * SEQUENCES and s.tables.cursor[1].item() - s.tables.cursor[0].item() == 200
    assert sorted(s.tables.free.tolist()) == list(range(200))
    s.step([40, 41, 42, 43, 44, 45], [0, 6], [0])


@BOTH
def test_captured_steps(dev, qt):
    s = Service(dev, qt)
    s.step([290, 0, 0, 0, 0, 33], [0, 0], [0])
    s.fork([-1, 0, 0, 0, 0, -1], [0, 288, 288, 288, 288, 0])
    rows = 10
    qkv, new = torch.zeros((rows, HEADS + 2 * KV, DIM), dtype=torch.bfloat16, device=dev), s.ints([0] * SEQUENCES)
    groups, shared = s.ints([1, 5]), s.ints([288])
    s.device_step(qkv, new, groups, shared, rows, 0)                             # (no tokens: nothing changes)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step, q, out = s.device_step(qkv, new, groups, shared, rows, 0)
    for turn, count in enumerate(([0, 1, 1, 1, 1, 1], [0, 2, 1, 1, 3, 1], [0, 1, 0, 4, 1, 1], [0, 0, 0, 0, 0, 0], [0, 1, 1, 1, 1, 6], [1, 1, 1, 1, 1, 1])):
        some = s.tokens(sum(count))
        qkv[:sum(count)] = some.to(dev)
        new.copy_(s.ints(count))
        if turn == 5:
            groups.copy_(s.ints([0, 5]))
        graph.replay()
        s.check(some, count, q, out, step)
        Service(dev, qt, 30).step([20, 1, 0, 0, 0, 3], [0, 6], [0])              # (the program's own eager work between)


def test_more_requests_than_pages(dev):
    """A step that does not fit says so, and what did fit is right."""
    s = Service(dev, ops.BF16, 30)
    s.step([300, 100, 0, 0, 0, 0], [0, 2], [0])                                  # 19 + 7 pages
    qkv = s.tokens(80)
    step, q, out = s.device_step(qkv.to(dev), s.ints([0, 0, 80, 0, 0, 0]), s.ints([0, 6]), s.ints([0]), 80, 80)
    assert step.missing.item() == 80 - 4 * PAGE and step.lens.tolist()[2] == 4 * PAGE and step.slots[4 * PAGE:].tolist() == [-1] * 16
    s.release([0])
    s.history[2] = []
    s.release([2])
    s.step([10, 3, 70, 0, 0, 0], [0, 6], [0])
