"""Rows whose keys are split over workgroups against the same rows in one: sums beyond fp32 whose averages are not, infinities with their
signs, and queries that are not finite."""
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


def _unsplit(dev, q, k, v):
    """Through the C entry point without a workspace."""
    qd, kd, vd, ends_q, ends_k = q.to(dev), k.to(dev), v.to(dev), _ends(len(q), dev), _ends(len(k), dev)
    out = torch.empty_like(qd)
    assert ops.load_library().sngguf_attention(qd.data_ptr(), len(q), HEADS, HEADS * DIM, DIM, kd.data_ptr(), KV * DIM, DIM, vd.data_ptr(), KV * DIM, DIM, len(k), KV, DIM,
                                               ends_q.data_ptr(), ends_k.data_ptr(), 1, DIM ** -0.5, 1, 0, out.data_ptr(), HEADS * DIM, DIM, None, 0,
                                               torch.cuda.current_stream().cuda_stream) == 0
    return out


def _all_split(new):
    lib = ops.load_library()
    assert lib.sngguf_attention_workspace_bytes(new, KEYS, 1, HEADS, KV, DIM) > 0
    assert lib.sngguf_paged_attention_workspace_bytes(new, 1, new, -(-KEYS // PAGE) * PAGE, HEADS, KV, DIM) > 0


@pytest.mark.parametrize("new", [1, 9, 30, 200])
@pytest.mark.parametrize("power", [127, 117])
def test_sums_beyond_fp32(dev, new, power):
    """Weights that are nearly equal: with values near 2^127 a split's own sum leaves fp32, with values near 2^117 only that of all splits does."""
    _all_split(new)
    gen = torch.Generator().manual_seed(new)
    q, k = (_values(gen, new, HEADS).float() * 0.1).to(torch.bfloat16), _values(gen, KEYS, KV)
    v = (_values(gen, KEYS, KV).float().abs().clamp(0.5, 1) * 2.0 ** power).to(torch.bfloat16)
    want, most = ao.attention(q, k, v)
    for name, call in (("unsplit", _unsplit), ("packed", _packed), ("paged", _paged)):
        off = (call(dev, q, k, v).double().cpu() - want).abs()
        assert bool((off <= most).all()), f"{name}: {int((~(off <= most)).sum())} of {off.numel()} values are off"


def _classes(q, k, v):
    """1, -1 and 2 where the result is +infinity, -infinity and NaN: a value's weight is more than nothing wherever it is seen."""
    seen = ao.visible(len(q), len(k), True, 0)
    out = torch.zeros(q.shape, dtype=torch.int64)
    for h in range(HEADS):
        x = v[:, h // (HEADS // KV)]
        up, down, none = ((seen.double() @ hit.double()) > 0 for hit in (x == INF, x == -INF, torch.isnan(x)))
        out[:, h] = torch.where(none | (up & down), 2, up.long() - down.long())
    return out


@pytest.mark.parametrize("new", [1, 9, 30, 200])
def test_infinities_keep_their_signs(dev, new):
    """One in the first split, in a middle one, in the last, and some that only the last rows see."""
    _all_split(new)
    gen = torch.Generator().manual_seed(new)
    q, k, v = _values(gen, new, HEADS), _values(gen, KEYS, KV), _values(gen, KEYS, KV)
    bad = v.clone()
    bad[5, :, 3], bad[4444, :, 4], bad[KEYS - 1, :, 5], bad[KEYS - 1, :, 6] = INF, -INF, INF, -INF
    bad[100, :, 7], bad[8000, :, 7] = INF, -INF
    bad[200, :, 8] = NAN
    want, most = ao.attention(q, k, v)
    classes = _classes(q, k, bad)
    assert {1, -1, 2} <= set(classes.unique().tolist())
    for name, call in (("unsplit", _unsplit), ("packed", _packed), ("paged", _paged)):
        got = call(dev, q, k, bad).double().cpu()
        found = torch.where(torch.isnan(got), 2, (got == INF).long() - (got == -INF).long())
        assert torch.equal(found, classes), f"{name}: elements {(found != classes).any(0).any(0).nonzero().flatten().tolist()}"
        fine = classes == 0
        assert bool(((got - want).abs() <= most)[fine].all()), name


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


@pytest.mark.parametrize("keys", [40, KEYS])
@pytest.mark.parametrize("new", [1, 30])
def test_scores_of_minus_infinity(dev, keys, new):
    """They have no weight: a row with one other key is that key's value, a row without any is zeros."""
    gen = torch.Generator().manual_seed(new)
    q, k, v = _values(gen, new, HEADS), _values(gen, keys, KV), _values(gen, keys, KV)
    q[:, :, 2] = q[:, :, 2].abs() + 1
    k[:, :, 2] = -INF
    for one in (False, True):
        if one:
            k[3, 1] = 0.5
        want = torch.zeros_like(q)
        want[:, 2:] = v[3, 1] if one else 0
        for name, call in (("unsplit", _unsplit), ("packed", _packed), ("paged", _paged)):
            got = call(dev, q, k, v).cpu()
            assert bool(((got.double() - want.double()).abs() <= 2.0 ** -8 * want.double().abs()).all()), (name, one)
