"""The operators between the projections in 64 bits, on the CPU, and how far a kernel's results may be from them."""
import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def visible(lq, lk, causal, window):
    """[lq][lk]: which keys a query sees, the last query standing at the last key."""
    place = torch.arange(lq)[:, None] + (lk - lq)
    key = torch.arange(lk)[None]
    seen = torch.ones((lq, lk), dtype=torch.bool)
    if causal:
        seen &= key <= place
    if window:
        seen &= key > place - window
    return seen


def attention(q, k, v, causal=True, window=0, scale=None, operand=torch.bfloat16):
    """One sequence: q [lq][heads][dim], k, v [lk][kv_heads][dim] of any type -> (out, most) float64 [lq][heads][dim].

    ``most`` bounds the error of a kernel that sums in 32 bits, rounds the weights (``operand`` float16: keys and values too) to
    ``operand`` and the result to bf16.  With A = sum_j p_j |v_j|, S = max_j scale sum_d |q_d k_jd| of a row, u = the operand's half
    step, e = 2^-24, n keys:
    * a score is off by d = dim e S from the sum and 4 e S from its scaling (operand float16: u S more from its key).  A weight
      p_j / sum_i p_i becomes p_j exp(d_j) / sum_i p_i exp(d_i), |d_j| <= d, so it changes by a factor between exp(-2 d) and
      exp(2 d): by exp(2 d) - 1 of itself at most (2 d, to first order, where d is small, which it is not for scores of thousands);
    * exp2 is off by 2^-21, n-term sums of weights and products by n e, each weight's rounding by u (float16: the value's too, and
      2^-36 absolute of the largest weight for n weights below its smallest step);
    * the result is rounded to bf16: 2^-8 of its value."""
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    lq, heads, dim = q.shape
    lk, group = k.shape[0], heads // k.shape[1]
    scale = dim ** -0.5 if scale is None else scale
    out, most = torch.zeros_like(q), torch.zeros_like(q)
    if lq == 0 or lk == 0:
        return out, most
    seen = visible(lq, lk, causal, window)
    e, u = 2.0 ** -24, HALF_STEP[operand]
    for h in range(heads):
        kh, vh = k[:, h // group], v[:, h // group]
        s = (q[:, h] @ kh.T * scale).masked_fill(~seen, -torch.inf)
        top = s.amax(1, keepdim=True)
        p = torch.exp(s - torch.where(top == -torch.inf, 0.0, top))
        total = p.sum(1, keepdim=True)
        p = p / torch.where(total == 0, 1.0, total)
        out[:, h] = p @ vh
        spread = p @ vh.abs()
        size = (q[:, h].abs() @ kh.abs().T * scale).masked_fill(~seen, 0.0).amax(1, keepdim=True)
        n = seen.sum(1, keepdim=True)
        d = ((dim + 4) * e + (u if operand == torch.float16 else 0.0)) * size
        most[:, h] = (torch.expm1(2 * d) + 2.0 ** -21 + 2 * n * e + u) * spread
        if operand == torch.float16:
            most[:, h] += u * spread + n * 2.0 ** -36 * vh.abs().amax()
        most[:, h] = 1.01 * (most[:, h] + 2.0 ** -8 * (out[:, h].abs() + most[:, h])) + 1e-37
    return out, most


def quantised(x):
    """(whole numbers, fp16 scales, values) that an 8-bit cache holds of ``x``, [..., dim]."""
    runs = x.double().cpu().unflatten(-1, (-1, 32))
    top = runs.abs().amax(-1, keepdim=True)
    scale = (top / 127).clamp(max=512.0).to(torch.float16).double()
    q = torch.where(scale > 0, torch.round(runs / scale), torch.zeros(())).clamp(-127, 127)
    q = torch.where(torch.isnan(scale), torch.zeros(()), q)
    return q.flatten(-2), scale.squeeze(-1), (q * scale).flatten(-2)


def turned(x, positions, turns, interleaved=False, magnitude=1.0):
    """x [tokens][heads][dim] turned, float64."""
    x, positions, turns = x.double().cpu(), positions.double().cpu(), turns.double().cpu()
    n = turns.numel()
    t = positions[:, None] * turns
    a = 2 * torch.pi * (t - t.round())
    c, s = magnitude * a.cos()[:, None], magnitude * a.sin()[:, None]
    y = x.clone()
    i = torch.arange(n)
    ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
    y[..., ia], y[..., ib] = x[..., ia] * c - x[..., ib] * s, x[..., ib] * c + x[..., ia] * s
    return y
