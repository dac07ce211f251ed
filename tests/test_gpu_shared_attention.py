"""Attention of sequences that begin alike against 64 bits, each sequence by itself."""
import itertools
import random

import pytest
import torch

from sensenova_u1_amd import PagedKVCache, ops, paged_attention, shared_prefix_attention

from . import attention_oracle as ao

pytestmark = pytest.mark.gpu

UNIT = 128          # what is common is taken in multiples of so many tokens
KEYS = 50 << 20     # elements of keys that sequences could have, by the width of their tables, for the groups to count
FEW, MANY = "few", "many"     # which kernel takes the common keys, by rows x keys of a group


def _values(gen, tokens, heads, dim, wide=False):
    x = torch.randn((tokens, heads, dim), generator=gen)
    if wide:
        x *= 1 + 3 * (torch.rand((heads, dim), generator=gen) > 0.95)
    return x.to(torch.bfloat16)


def _ints(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def _close(got, want, most, what):
    off = (got.double().cpu() - want).abs()
    bad = ~(off <= most)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} values, worst {float((off / most)[bad].max()):.3g} times the bound, first at {bad.nonzero()[0].tolist()}"


class Batch:
    """Sequences of some groups in a cache, in tables so wide that the groups count (``kernel``: as wide as that kernel needs; None: as narrow as the
    sequences are); where they do, pages that nobody reads for what is common hold NaN."""

    def __init__(self, dev, counts, shared, new, own, heads, kv_heads, dim, page, qt, seed=0, outside=0, kernel=FEW):
        gen = torch.Generator().manual_seed(seed)
        self.dev, self.new = dev, new
        group = [g for g, n in enumerate(counts) for _ in range(n)] + [None] * outside
        self.lens = [(shared[g] if g is not None else 0) + n for g, n in zip(group, own)]
        assert len(group) == len(new) == len(own)
        prefixes = [(_values(gen, n, kv_heads, dim, True), _values(gen, n, kv_heads, dim)) for n in shared]
        self.kv = []
        for g, n in zip(group, own):
            k, v = _values(gen, n, kv_heads, dim, True), _values(gen, n, kv_heads, dim)
            self.kv.append((k, v) if g is None else (torch.cat([prefixes[g][0], k]), torch.cat([prefixes[g][1], v])))
        total = sum(-(-n // page) for n in self.lens) + sum(n // page for n in shared) + 4
        order = torch.randperm(total, generator=gen).tolist()
        nan_page = order.pop()
        width = max(-(-n // page) for n in self.lens) + 1
        group_rows = sum(new) * (heads // kv_heads) // len(counts)
        if kernel is not None:
            width = max(width, -(-KEYS // (len(new) * kv_heads * dim * page)))
        if kernel == MANY:
            width = max(width, -(-(2 << 20) // (max(group_rows, 1) * page)))
        self.cache = PagedKVCache.empty(total, kv_heads, page, dim, qt, dev)
        for t in (self.cache.k, self.cache.v):
            t.fill_(-128 if qt == ops.Q8_0 else float("nan"))
        for t in (self.cache.k_scale, self.cache.v_scale):
            if t is not None:
                t.fill_(float("nan"))
        rows = [[2 ** 30] * width for _ in self.lens]
        heads_of = [[order.pop() for _ in range(n // page)] for n in shared]
        for i, (g, n) in enumerate(zip(group, self.lens)):
            lead = heads_of[g] if g is not None else []
            mine = lead + [order.pop() for _ in range(-(-n // page) - len(lead))]
            rows[i][:len(mine)] = mine
            slots = torch.tensor(mine, dtype=torch.int64)[torch.arange(n) // page] * page + torch.arange(n) % page
            self.cache.write(self.kv[i][0].to(dev), self.kv[i][1].to(dev), slots.to(dev))
        self.whole = _ints(rows, dev)
        lib = ops.load_library()
        sizes = (sum(new), len(new), len(counts), max(new), width * page, heads, kv_heads, dim, qt)
        self.counts = lib.sngguf_shared_attention_workspace_bytes(*sizes) != lib.sngguf_paged_attention_workspace_bytes(*sizes[:2], *sizes[3:8])
        # what is common, and who need not have it
        hidden = [list(r) for r in rows]
        for g, (a, n) in enumerate(zip(itertools.accumulate([0] + counts), counts)):
            live = [i for i in range(a, a + n) if new[i]]
            common = max(0, min([shared[g]] + [self.lens[i] - new[i] for i in live])) // UNIT * UNIT if len(live) > 1 and self.counts else 0
            for i in range(a, a + n):
                if not live or i == live[0]:
                    continue
                for p in range(common // page):
                    hidden[i][p] = nan_page
        self.pages = _ints(hidden, dev)
        self.q = _values(gen, sum(new), heads, dim)
        self.ends = _ints([0] + list(itertools.accumulate(new)), dev)
        self.groups = _ints([0] + list(itertools.accumulate(counts)), dev)
        self.shared, self.lens_dev = _ints(shared, dev), _ints(self.lens, dev)
        self.operand = torch.float16 if qt == ops.Q8_0 else torch.bfloat16

    def __call__(self, **kw):
        args = dict(ends_q=self.ends, max_new=max(self.new))
        args.update(kw)
        return shared_prefix_attention(self.q.to(self.dev), self.cache, self.pages, self.lens_dev, self.groups, self.shared, **args)

    def check(self, got, scale=None, only=None):
        row = 0
        for i, (n, (k, v)) in enumerate(zip(self.new, self.kv)):
            if only is None or i in only:
                if self.operand == torch.float16:
                    k, v = ao.quantised(k)[2], ao.quantised(v)[2]
                want, most = ao.attention(self.q[row:row + n], k, v, True, 0, scale, self.operand)
                _close(got[row:row + n], want, most, f"sequence {i}: {n} of {len(k)}")
            row += n


BOTH = pytest.mark.parametrize("qt", [ops.BF16, ops.Q8_0])


KERNELS = pytest.mark.parametrize("kernel", [FEW, MANY])


@BOTH
@pytest.mark.parametrize("kernel", [FEW, MANY, None])
@pytest.mark.parametrize("shared", [0, 1, 16, 127, 128, 129, 255, 256, 300, 1000, 2048])
def test_lengths_of_what_is_common(dev, shared, kernel, qt):
    b = Batch(dev, [5], [shared], [1] * 5, [1, 3, 40, 129, 200], 8, 2, 128, 16, qt, shared, kernel=kernel)
    assert b.counts == (kernel is not None)
    b.check(b())
    assert torch.equal(b(), b())


@BOTH
@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 8, 128), (1, 1, 64), (4, 4, 64), (28, 4, 128), (5, 1, 96), (12, 1, 128), (16, 2, 32), (6, 2, 160), (4, 2, 192), (6, 2, 256), (40, 8, 64), (130, 1, 64)])
@pytest.mark.parametrize("count", [2, 9, 40])
@KERNELS
def test_head_layouts_and_row_counts(dev, heads, kv_heads, dim, count, kernel, qt):
    rng = random.Random(count)
    b = Batch(dev, [count], [640], [1] * count, [rng.randint(1, 70) for _ in range(count)], heads, kv_heads, dim, 32, qt, dim + count, kernel=kernel)
    assert b.counts
    b.check(b())


@BOTH
@pytest.mark.parametrize("page", [16, 64, 256, 4096])
@KERNELS
def test_groups_that_differ(dev, page, kernel, qt):
    counts, shared = [3, 1, 0, 6, 2], [300, 700, 5000, 1500, 0]
    new, own = [1] * 12, [5, 1, 100, 30, 1, 2, 3, 400, 5, 6, 77, 1]
    b = Batch(dev, counts, shared, new, own, 8, 2, 64, page, qt, page, kernel=kernel)
    b.check(b())
    b = Batch(dev, counts, shared, new + [1, 1], own + [300, 1], 8, 2, 64, page, qt, page, outside=2, kernel=kernel)      # sequences of no group
    b.check(b())


@BOTH
@pytest.mark.parametrize("new", [[2, 3, 1], [7, 1, 5], [16, 16, 16], [1, 64, 3], [200, 1, 1], [300, 129, 257], [0, 4, 9], [0, 0, 5], [1, 1, 700]])
@pytest.mark.parametrize("known", [True, False])
@KERNELS
def test_runs_of_new_tokens(dev, new, known, kernel, qt):
    own = [n + 20 * i for i, n in enumerate(new)]
    b = Batch(dev, [3], [520], new, own, 8, 2, 128, 32, qt, sum(new), kernel=kernel)
    assert b.counts == (sum(new) * 4 < 256 * 3)
    b.check(b(max_new=max(new) if known else 0))


@BOTH
def test_new_tokens_that_reach_into_what_is_said_to_be_common(dev, qt):
    # the second sequence is a prompt that has just come in: its first tokens are new, so nothing is common, or less is
    for own in ([30, 40, 9], [30, 200, 9]):
        new = [1, 170, 2]
        b = Batch(dev, [3], [500], new, own, 8, 2, 64, 16, qt, own[1])
        b.check(b())


@BOTH
@pytest.mark.parametrize("dim", [64, 128, 256])
@KERNELS
def test_long_common_parts_are_split(dev, dim, kernel, qt):
    for count, shared in ((2, 20000), (20, 6000), (70, 2500)):
        b = Batch(dev, [count], [shared], [1] * count, [1 + i % 50 for i in range(count)], 4, 1, dim, 64, qt, count, kernel=kernel)
        b.check(b(), only={0, 1, count - 1})


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("count", [60, 150])
@KERNELS
def test_joins_of_many_queries(dev, dim, count, kernel):
    """From 1024 and from 4096 queries on (32 a token) fewer lanes have one, and partial results come in turns."""
    own = [1 + i % 20 for i in range(count)]
    own[3] = 3000
    b = Batch(dev, [count], [1300], [1] * count, own, 32, 4, dim, 64, ops.BF16, count + dim, kernel=kernel)
    b.check(b(), only={0, 3, count // 2, count - 1})


@BOTH
def test_long_own_parts_are_split(dev, qt):
    b = Batch(dev, [3], [256], [1, 1, 2], [6000, 5, 3000], 4, 1, 128, 64, qt)
    b.check(b())


@pytest.mark.parametrize("counts", [[127, 127], [200, 150], [3] * 90, [1100, 5], [0] * 300 + [2] * 20])
def test_many_sequences_and_groups(dev, counts):
    """Up to 256 of them are planned in one go, more in turns."""
    n = sum(counts)
    b = Batch(dev, counts, [256 + 16 * (i % 3) for i in range(len(counts))], [1] * n, [1 + i % 40 for i in range(n)], 2, 1, 64, 16, ops.BF16, n)
    b.check(b(), only=set(range(0, n, 7)) | {n - 1})


@BOTH
def test_every_sequence_one_token_without_ends(dev, qt):
    b = Batch(dev, [4, 3], [260, 900], [1] * 7, [1, 2, 3, 4, 5, 6, 700], 8, 2, 128, 16, qt)
    b.check(b(ends_q=None, max_new=0))


def test_the_same_as_attention_without_groups(dev):
    b = Batch(dev, [4, 3], [260, 900], [1, 5, 1, 0, 1, 90, 1], [1, 9, 3, 4, 5, 96, 700], 8, 2, 128, 16, ops.BF16)
    q = b.q.to(dev)
    none = shared_prefix_attention(q, b.cache, b.whole, b.lens_dev, _ints([0], dev), _ints([], dev), b.ends)
    assert torch.equal(none, paged_attention(q, b.cache, b.whole, b.lens_dev, b.ends))
    b.check(none)
    b.check(shared_prefix_attention(q, b.cache, b.whole, b.lens_dev, _ints([0, 0, 7, 7], dev), _ints([3, 0, 5], dev), b.ends))


@BOTH
def test_scales_and_large_scores(dev, qt):
    for scale in (5.0, 1e-6, 0.3):
        b = Batch(dev, [4], [700], [1, 2, 1, 1], [9, 9, 200, 1], 8, 2, 128, 16, qt)
        b.check(b(scale=scale), scale)


@BOTH
def test_what_is_common_outweighs_what_is_not_and_the_other_way_round(dev, qt):
    """Maxima of the two parts far from each other, both ways."""
    for factor in (0.01, 30.0):
        gen = torch.Generator().manual_seed(3)
        b = Batch(dev, [3], [384], [1] * 3, [100] * 3, 4, 1, 64, 16, qt)
        lead = (_values(gen, 384, 1, 64) * factor).to(torch.bfloat16)
        pages = b.whole[0].long()
        slots = pages[torch.arange(384, device=dev) // 16] * 16 + torch.arange(384, device=dev) % 16
        b.cache.write(lead.to(dev), b.kv[0][1][:384].to(dev), slots)
        b.kv = [(torch.cat([lead, k[384:]]), v) for k, v in b.kv]
        b.check(b())


def test_rows_behind_the_last_sequence_are_left_and_outputs_of_any_layout(dev):
    b = Batch(dev, [3], [256], [2, 1, 3], [5, 6, 7], 8, 2, 128, 16, ops.BF16)
    q = torch.cat([b.q, b.q[:4]]).to(dev)
    out = torch.full_like(q, 3.0)
    shared_prefix_attention(q, b.cache, b.pages, b.lens_dev, b.groups, b.shared, b.ends, out=out)
    want = b()
    b.check(want)
    assert torch.equal(out[:6], want) and bool((out[6:] == 3).all())
    room = torch.full((6, 12, 128), 7.0, dtype=torch.bfloat16, device=dev)
    b(out=room[:, 2:10])
    assert torch.equal(room[:, 2:10], want) and bool((room[:, :2] == 7).all()) and bool((room[:, 10:] == 7).all())
    # queries as they lie in a stacked projection
    stacked = torch.randn((6, 20, 128), device=dev).to(torch.bfloat16)
    stacked[:, 3:11] = b.q.to(dev)
    assert torch.equal(shared_prefix_attention(stacked[:, 3:11], b.cache, b.pages, b.lens_dev, b.groups, b.shared, b.ends), want)
    # tables whose rows lie apart
    wide = torch.zeros((3, 40 + b.pages.shape[1]), dtype=torch.int32, device=dev)
    wide[:, 5:5 + b.pages.shape[1]] = b.pages
    assert torch.equal(shared_prefix_attention(b.q.to(dev), b.cache, wide[:, 5:5 + b.pages.shape[1]], b.lens_dev, b.groups, b.shared, b.ends), want)


@BOTH
@KERNELS
def test_values_that_are_not_finite(dev, kernel, qt):
    """An infinity or a NaN in what is common reaches all of the group and no other; one in a sequence's own part that sequence alone."""
    for where in ("common", "own"):
        for bad in (float("inf"), float("nan"), -float("inf")):
            b = Batch(dev, [3, 2], [400, 300], [1, 2, 1, 1, 1], [5, 6, 30, 4, 5], 4, 2, 64, 16, qt, kernel=kernel)
            at = 130 if where == "common" else 400
            slot = b.whole[1].long()[at // 16] * 16 + at % 16
            k, v = b.kv[1][0][at:at + 1].clone(), b.kv[1][1][at:at + 1].clone()
            v[0, 0, 3] = bad
            b.cache.write(k.to(dev), v.to(dev), slot[None])
            got = b().float().cpu()
            hit = range(0, 4) if where == "common" else range(1, 3)
            for row in range(6):
                rows_heads = got[row]
                if row not in hit:
                    assert bool(torch.isfinite(rows_heads).all()), (where, bad, row)
                elif qt == ops.BF16:
                    assert bool((rows_heads[:2, 3] == bad).all()) if bad == bad else bool(torch.isnan(rows_heads[:2, 3]).all()), (where, bad, row)
                    keep = torch.ones(64, dtype=torch.bool)
                    keep[3] = False
                    assert bool(torch.isfinite(rows_heads[:2, keep]).all()) and bool(torch.isfinite(rows_heads[2:]).all())
                else:
                    assert bool(torch.isfinite(rows_heads[2:]).all())
            b.check(got, only={3, 4} if where == "common" else {0, 2, 3, 4})


@KERNELS
def test_sums_beyond_fp32_stay_finite_where_their_average_is(dev, kernel):
    b = Batch(dev, [2], [1024], [1, 1], [3, 5], 2, 1, 64, 16, ops.BF16, kernel=kernel)
    b.cache.v.fill_(3e38)
    got = b().float()
    assert bool(torch.isfinite(got).all()) and float((got / 3e38 - 1).abs().max()) < 0.02


@KERNELS
def test_a_query_that_is_not_a_number(dev, kernel):
    """It gives NaN, and the other queries what they have without it, within the bound of each: a wavefront that meets the NaN sets the maxima of
    all its rows right, so the others' weights exp2(s - m) are rounded to bf16 with another m (u in the bound, either way)."""
    b = Batch(dev, [3], [512], [1, 1, 1], [3, 5, 200], 4, 2, 128, 16, ops.BF16, kernel=kernel)
    clean = b.q.clone()
    b.q[1, 2, 7] = torch.nan
    got = b()
    assert bool(torch.isnan(got[1, 2]).all())
    b.q = clean
    for i, (k, v) in enumerate(b.kv):
        want, most = ao.attention(clean[i:i + 1], k, v)
        keep = [0, 1, 3] if i == 1 else [0, 1, 2, 3]
        _close(got[i:i + 1, keep], want[:, keep], most[:, keep], f"sequence {i}")


@KERNELS
def test_lengths_and_groups_that_are_none_stay_within_the_tensors(dev, kernel):
    b = Batch(dev, [4, 3], [260, 900], [1, 5, 1, 2, 1, 40, 1], [1, 9, 3, 4, 5, 46, 700], 8, 2, 128, 16, ops.BF16, kernel=kernel)
    assert b.counts
    q = b.q.to(dev)
    for groups, shared, ends, lens in (([0, 9000, -5], [10 ** 9, -7], None, None), ([5, 2, 7], [900, 900], None, None), ([0, 7, 3], [128, 256], None, None), ([0, 4, 7], [2 ** 31 - 1, 2 ** 31 - 1], None, None),
                                       ([0, 4, 7], [260, 900], [0, 60, -1, 10, 51, 20, 3, 51], None), ([0, 4, 7], [260, 900], [50, 0, 50, 0, 50, 0, 50, 0], None),
                                       ([0, 4, 7], [260, 900], None, [-5, 10 ** 9, 0, 2 ** 31 - 1, 300, 1, 2]), ([0, 4, 7], [-2 ** 31, 5], None, [0] * 7)):
        out = shared_prefix_attention(q, b.cache, b.whole, _ints(lens, dev) if lens else b.lens_dev, _ints(groups, dev), _ints(shared, dev), _ints(ends, dev) if ends else b.ends)
        assert out.shape == q.shape
    torch.cuda.synchronize()
    wild = torch.full_like(b.whole, -2 ** 31)
    shared_prefix_attention(q, b.cache, wild, b.lens_dev, b.groups, b.shared, b.ends)
    torch.cuda.synchronize()


@BOTH
@KERNELS
def test_captured_steps_see_new_lengths_groups_and_queries(dev, kernel, qt):
    counts, shared = [5, 3], [700, 300]
    b = Batch(dev, counts, shared, [1] * 8, [1, 2, 3, 40, 500, 6, 7, 130], 8, 2, 128, 16, qt, kernel=kernel)
    q = b.q.to(dev)
    args = (b.cache, b.whole, b.lens_dev, b.groups, b.shared)
    shared_prefix_attention(q, *args)
    torch.cuda.synchronize()
    one, two = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(one):
        first = shared_prefix_attention(q, *args)
    with torch.cuda.graph(two):
        second = shared_prefix_attention(q, *args)
    gen = torch.Generator().manual_seed(9)
    whole = list(b.lens)
    for step in range(5):
        lens = [max(1, n - step * 3) for n in whole]
        b.lens_dev.copy_(_ints(lens, dev))
        b.groups.copy_(_ints([[0, 5, 8], [0, 4, 5], [1, 5, 8], [0, 0, 5], [5, 8, 8]][step], dev))
        b.shared.copy_(_ints([[700, 300], [699, 9000], [128, 256], [0, 640], [300, 0]][step], dev))
        q.copy_(_values(gen, 8, 8, 128))
        one.replay()
        two.replay()
        got = first.clone(), second.clone()
        torch.cuda.synchronize()
        eager = shared_prefix_attention(q, *args)
        assert torch.equal(got[0], eager) and torch.equal(got[1], eager), step
        b.q = q.cpu()
        b.kv = [(k[:n], v[:n]) for (k, v), n in zip(b.kv, lens)]
        b.check(eager)


def test_two_streams_at_once(dev):
    b = Batch(dev, [6], [1500], [1] * 6, [30, 2, 3, 400, 5, 6], 8, 2, 128, 16, ops.Q8_0)
    want = b()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append([b() for _ in range(5)])
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(x, want) for o in outs for x in o)


def test_what_is_refused(dev):
    b = Batch(dev, [2], [128], [1, 1], [3, 5], 4, 2, 64, 16, ops.BF16)
    q = b.q.to(dev)
    good = dict(q=q, cache=b.cache, pages=b.pages, lens=b.lens_dev, groups=b.groups, shared=b.shared)
    for bad in (dict(groups=b.groups[:0]), dict(groups=b.groups.long()), dict(groups=b.groups.cpu()), dict(shared=b.shared[:0]), dict(shared=b.shared.long()), dict(shared=b.shared.cpu()),
                dict(lens=b.lens_dev[:1]), dict(pages=b.pages[:1]), dict(pages=b.pages.long()), dict(q=q[:1]), dict(q=q[..., :32]), dict(q=q[:, :3]), dict(q=q.float()), dict(scale=0.0),
                dict(max_new=-1), dict(out=q), dict(out=torch.empty_like(q)[:1]), dict(ends_q=b.ends[:2]), dict(q=q.cpu())):
        with pytest.raises(ops.SnGgufError):
            shared_prefix_attention(**{**good, **bad})
    assert shared_prefix_attention(**good).shape == q.shape
    none = shared_prefix_attention(q[:0], b.cache, b.pages[:0], b.lens_dev[:0], _ints([0, 0], dev), _ints([5], dev))
    assert none.shape == (0, 4, 64)
