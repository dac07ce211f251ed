"""Norms of single heads and rotation by several positions in 64 bits, on the CPU, and how far a kernel's results may be from them."""
import torch

E = 2.0 ** -24


def pairs_of(parts, interleaved):
    """Elements (a, b) of each pair, counted from part to part."""
    ia, ib, start = [], [], 0
    for n in parts:
        at = torch.arange(n // 2)
        ia.append(start + (2 * at if interleaved else at))
        ib.append(start + (2 * at + 1 if interleaved else at + n // 2))
        start += n
    return torch.cat(ia), torch.cat(ib)


def head(x, positions, turns, axis, parts, interleaved=False, magnitude=1.0, weights=(), eps=1e-6):
    """x [tokens][heads][dim], positions [axes][tokens] -> (out, most) float64.

    ``most`` bounds the error of a kernel that norms and turns in 32 bits and rounds once.  With e = 2^-24: a sum of n squares is off by
    n e of itself at most, its mean, root and reciprocal (a step of 2^-23 each at most, the root halves what is before it) and the
    two products with it and the weight by 8 e more: (n / 2 + 8) e of a normed value.  Cosine and sine are rounded (e each), so are
    their products and the sum: 4 e of |a c| + |b s|.  The result is rounded to bf16: 2^-8 of it."""
    x, positions, turns = x.double().cpu(), positions.double().cpu(), turns.double().cpu()
    y, n = x.clone(), 0
    start = 0
    for w in weights:
        w = w.double().cpu()
        part = x[..., start:start + len(w)]
        y[..., start:start + len(w)] = part / torch.sqrt(part.square().mean(-1, keepdim=True) + eps) * w
        start += len(w)
        n = max(n, len(w))
    t = positions[axis.cpu().long().clamp(0, positions.shape[0] - 1)].T * turns
    a = 2 * torch.pi * (t - t.round())
    c, s = magnitude * a.cos()[:, None], magnitude * a.sin()[:, None]
    ia, ib = pairs_of(parts, interleaved)
    out, size = y.clone(), y.abs()
    out[..., ia], out[..., ib] = y[..., ia] * c - y[..., ib] * s, y[..., ib] * c + y[..., ia] * s
    both = (y[..., ia].abs() + y[..., ib].abs()) * abs(magnitude)
    size[..., ia], size[..., ib] = both, both
    most = ((n / 2 + 8 if n else 0) + 4) * E * size
    return out, 1.01 * (2.0 ** -8 * (out.abs() + most) + most) + 1e-40
