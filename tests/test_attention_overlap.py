"""Whether two tensors of rows share memory, against the sets of their bytes (on the CPU)."""
import random

import pytest
import torch

from sensenova_u1_amd.attention import _apart, _places, _rows_share, _share, _whole


def _bytes(x):
    size = x.element_size()
    return {x.data_ptr() + size * (t * x.stride(0) + h * x.stride(1) + e) + i for t in range(x.shape[0]) for h in range(x.shape[1]) for e in range(x.shape[2])
            for i in range(size)}


def _same(a, b):
    want = bool(_bytes(a) & _bytes(b))
    assert _share(_places(a), _places(b)) == want and _share(_places(b), _places(a)) == want, (a.shape, a.stride(), b.shape, b.stride(), b.data_ptr() - a.data_ptr())
    if a.shape[2] == b.shape[2]:
        assert _rows_share(a, b) == want and _rows_share(b, a) == want
    return want


def test_views_of_stacked_rows():
    x = torch.zeros((9, 12, 16), dtype=torch.bfloat16)
    # parts of a projection's output; parts of heads; every other head; heads ahead of tokens
    for a, b in ((x[:, :4], x[:, 4:6]), (x[:, 4:6], x[:, 6:]), (x[..., :8], x[..., 8:]), (x[:, ::2], x[:, 1::2]), (x[::2], x[1::2]), (x[:4], x[4:]),
                 (x[:, :4, :8], x[:, 2:6, 8:]), (x.transpose(0, 1)[:6], x.transpose(0, 1)[6:]), (x[:, :4].transpose(0, 1), x[:, 4:].transpose(0, 1)),
                 (x[:1, :4], x[:, 4:]), (x[:, 3:4], x[:, 4:5]), (x[:5, ::3], x[:5, 1::3])):
        assert not _same(a, b)
    for a, b in ((x, x), (x[:, :4], x[:, 2:6]), (x[:, :8], x[:, 1:9]), (x[..., :8], x[..., 7:]), (x[:, ::2], x[:, ::3]), (x[:5], x[4:]), (x[:, :1], x[3:4]),
                 (x.transpose(0, 1)[:6], x.transpose(0, 1)[5:]), (x[:, :1].expand(9, 3, 16), x[:, :2]), (x[:1].expand(3, 12, 16), x[1:])):
        assert _same(a, b) == bool(_bytes(a) & _bytes(b))
    assert _share(_places(x[:, :8]), _places(x[:, 1:9]))


@pytest.mark.parametrize("seed", range(8))
def test_any_strides(seed):
    rng = random.Random(seed)
    room = torch.zeros((4000,), dtype=torch.bfloat16)
    both = [0, 0]
    for _ in range(300):
        dim = rng.choice([1, 2, 3, 8])
        views = []
        for _ in range(2):
            shape, stride = (rng.randint(1, 6), rng.randint(1, 5), dim), (rng.choice([0, dim, 2 * dim, 24, 25, 40, 97, 120]), rng.choice([dim, 2 * dim, 16, 24, 40, 9]), 1)
            views.append(room.as_strided(shape, stride, rng.randint(0, 400)))
        both[_same(*views)] += 1
    assert min(both) > 20


def test_one_row_of_many_bytes():
    room = torch.zeros((1000,), dtype=torch.int8)
    rows = room.view(torch.bfloat16)[:320].view(10, 4, 8)
    for a, b in ((0, 64), (64, 128), (600, 640), (640, 700), (639, 640), (1, 2)):
        assert _share(_places(rows), _whole(room[a:b])) == (a < 640)
    assert _share(_whole(room[:100]), _whole(room[99:])) and not _share(_whole(room[:100]), _whole(room[100:]))
    gaps = rows[:, ::2]
    assert not _share(_places(gaps), _whole(room[16:32])) and _share(_places(gaps), _whole(room[16:33]))
    assert _apart(gaps)
