"""What the 8-bit cache holds of runs of small values, whose scales fp16 holds with few bits: every number is equal."""
import pytest
import torch

from sensenova_u1_amd import HeadNorm, PagedKVCache, RotaryAxes, RotaryTable, ops, rotary

from . import attention_oracle as ao

pytestmark = pytest.mark.gpu

HEADS, DIM, PAGE = 8, 128, 64


def _bits(values):
    return torch.tensor(values, dtype=torch.float64).to(torch.bfloat16).view(torch.int16).tolist()


def _runs(first, last, octaves):
    """Runs of 32 whose largest magnitudes are all those of bf16 in [first, last], of either sign, among members of all magnitudes down to 2^-octaves of
    it: [tokens][HEADS][DIM]."""
    first, last = _bits([first, last])
    top = torch.arange(first, last + 1)
    member = (top[:, None] - torch.arange(128 * octaves)).clamp(min=0)
    member = torch.nn.functional.pad(member, (0, -member.shape[1] % 31)).unflatten(1, (-1, 31))
    run = torch.cat([top[:, None, None].expand(-1, member.shape[1], 1), member], 2)
    sign = torch.arange(32) % 2 ^ torch.arange(run.shape[1])[:, None] % 2          # (the largest one's changes from run to run)
    runs = torch.stack([run | sign << 15, run | (1 - sign) << 15]).flatten(0, 2)
    runs = torch.nn.functional.pad(runs.flatten(), (0, -runs.numel() % (HEADS * DIM)))
    return (runs - (runs >> 15 << 16)).to(torch.int16).view(torch.bfloat16).view(-1, HEADS, DIM)


def _held(cache, name, tokens):
    x, scale = getattr(cache, name), getattr(cache, name + "_scale")
    return (x.permute(0, 2, 1, 3).flatten(0, 1)[:tokens].cpu().double(), scale.permute(0, 3, 1, 2).flatten(0, 1)[:tokens].cpu().double())


def _same(cache, name, x):
    q, s, _ = ao.quantised(x)
    held, scale = _held(cache, name, len(x))
    bad = held != q
    assert not bad.any(), (name, int(bad.sum()), x.cpu()[bad][:4].tolist(), held[bad][:4].tolist(), q[bad][:4].tolist())
    assert torch.equal(scale, s)


@pytest.mark.parametrize("first,last,octaves", [(3e-6, 1.1e-2, 10), (0.99, 4.0, 10), (3e4, 2e5, 10), (1e-9, 3.1e-6, 1)])
def test_every_largest_magnitude(dev, first, last, octaves):
    x = _runs(first, last, octaves)
    if first == 3e-6:
        scale = ao.quantised(x)[1]
        off = (x.double().unflatten(-1, (-1, 32)) / scale[..., None]).abs()[scale > 0]
        assert int((off > 127.5).sum()) > 1000 and float(off.max()) > 189      # (numbers beyond 127 are among them)
    tokens = len(x)
    cache = PagedKVCache.empty(-(-tokens // PAGE), HEADS, PAGE, DIM, ops.Q8_0, dev)
    cache.write(x.to(dev), x.flip(0).to(dev), torch.arange(tokens, device=dev))
    _same(cache, "k", x)
    _same(cache, "v", x.flip(0))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_small_runs_beside_the_rotation(dev, interleaved, norm):
    """Values as they are, and keys that the norm's weights make as small."""
    x = _runs(7e-6, 5.2e-4, 2)
    tokens, gen = len(x), torch.Generator().manual_seed(1)
    k = torch.randn((tokens, HEADS, DIM), generator=gen)
    if norm:
        weights = (2.0 ** -torch.arange(12, 20).repeat_interleave(16)).split(64)
        norms, table, positions = dict(k_norm=HeadNorm(*(w.to(dev) for w in weights))), RotaryAxes.for_model([(64, 0, 5e6), (32, 1, 1e4), (32, 2, 1e4)], interleaved, dev), torch.randint(0, 900, (3, tokens), generator=gen)
    else:
        k *= 2.0 ** -(12 + torch.arange(tokens) % 6)[:, None, None]
        norms, table, positions = {}, RotaryTable.for_model(DIM, interleaved=interleaved, device=dev), torch.randint(0, 900, (tokens,), generator=gen)
    k, positions = k.to(torch.bfloat16).to(dev), positions.to(dev)
    cache = PagedKVCache.empty(-(-tokens // PAGE), HEADS, PAGE, DIM, ops.Q8_0, dev)
    cache.write_rotary(k[:, :1], k, x.to(dev), positions, table, torch.arange(tokens, device=dev), **norms)
    _same(cache, "v", x)
    turned = rotary(k[:, :1], k, positions, table, **norms)[1]
    assert bool((turned.float().abs().unflatten(-1, (-1, 32)).amax(-1) < 4.8e-4).any())
    _same(cache, "k", turned)
