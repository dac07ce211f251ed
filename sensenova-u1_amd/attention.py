"""What stands between a decoder layer's projections: rotary positions, a paged cache of keys and values, and attention over
whole prompts or over that cache (``modeling_qwen3.py:431-505,583-745``, where the reference runs tensor operations).

All of it takes and gives bf16 ``[tokens][heads][dim]`` on one HIP device, enqueues on the current stream, never synchronises,
and reads every length, position, slot and page number on the device: a captured step replays with new ones.  Views into a
stacked projection's output go in as they are.  Forward only: nothing here records a gradient.

A layer's attention for new tokens of sequences that lie in a cache::

    q, k, v = (y.view(tokens, -1, dim) for y in qkv(hidden, norm_weight, eps))     # FusedProjections
    q = cache.write_rotary(q, k, v, positions, table, slots, q_norm=q_norm, k_norm=k_norm)      # HeadNorm, where the model norms single heads
    out = paged_attention(q, cache, pages, lens, ends)                              # [tokens][heads][dim]
    hidden = o_proj.forward_residual(out.view(tokens, -1), hidden)
"""
from __future__ import annotations

import ctypes
import functools
import math
import operator
import struct
from typing import Optional, Sequence, Union

import torch

from . import ops
from .ops import SnGgufError

_BF16 = torch.bfloat16


class _TableStruct(ctypes.Structure):
    _fields_ = [("turns", ctypes.c_void_p), ("pairs", ctypes.c_int64), ("magnitude", ctypes.c_double), ("interleaved", ctypes.c_int32)]


# sngguf_rotary_axes and sngguf_head_norm as bytes, which ctypes hands on by their address (half the time of a Structure that is made and filled)
_AXES = struct.Struct("PPqd6i")     # turns, axis, pairs, magnitude, interleaved, parts, part[4]
_NORM = struct.Struct("4P6if4x")    # weight[4], elements[4], parts, weight_type, eps


class _CacheStruct(ctypes.Structure):
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("k_scale", ctypes.c_void_p), ("v_scale", ctypes.c_void_p),
                ("pages", ctypes.c_int64), ("page_size", ctypes.c_int64), ("kv_heads", ctypes.c_int64), ("dim", ctypes.c_int64),
                ("qtype", ctypes.c_int32)]


def _new(x: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _field(name: str) -> property:
    """A field that calls have by its address: it can be written into, not replaced."""
    held = operator.attrgetter("_" + name)

    def refuse(self, value):
        if value is not held(self):     # (x.field += 1 ends here with the field itself)
            raise SnGgufError(f"{type(self).__name__}: {name} cannot be replaced (calls use what it was made with)")

    return property(held, refuse)


def _stream(index: int) -> int:
    return ops._raw_stream(index) if ops._raw_stream is not None else torch.cuda.current_stream(index).cuda_stream


def _launch(index: int, name: str, *args) -> None:
    """``lib.<name>(*args, current stream)`` with device ``index`` current."""
    fn = getattr(ops.load_library(), name)
    if index == ops._current_device():
        rc = fn(*args, _stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _stream(index))
    if rc:
        ops._check(rc, name)


@functools.lru_cache(1024)
def _prompt_workspace(*sizes: int) -> int:
    return ops.load_library().sngguf_attention_workspace_bytes(*sizes)


@functools.lru_cache(1024)
def _paged_workspace(*sizes: int) -> int:
    return ops.load_library().sngguf_paged_attention_workspace_bytes(*sizes)


@functools.lru_cache(1024)
def _shared_workspace(*sizes: int) -> int:
    return ops.load_library().sngguf_shared_attention_workspace_bytes(*sizes)


def _launch_with_workspace(index: int, nbytes: int, name: str, *args) -> None:
    if not nbytes:
        return _launch(index, name, *args, None, 0)
    dev = torch.device("cuda", index)
    with ops._on(dev), ops._whole_call(dev):
        _launch(index, name, *args, ops.pooled_workspace(dev, nbytes).data_ptr(), nbytes)


def _same_device(what: str, index: int, *tensors: Optional[torch.Tensor]) -> None:
    for t in tensors:
        if t is not None and t.get_device() != index:
            raise SnGgufError(f"{what}: tensors on different devices (or on the host; there is no CPU implementation)")


def _heads(x: torch.Tensor, what: str, name: str, pieces: bool = False):
    """``x`` as [tokens][heads][dim] rows whose elements are neighbours (``pieces``: each at a 16-byte boundary), copied where it is not,
    and its (token, head) strides; those of an axis of one entry are never stepped over and count as 0."""
    if not x.is_cuda:
        raise SnGgufError(f"sn_gguf ops run on a HIP device only, got {name} on '{x.device}'; there is no CPU implementation")
    shape = x.shape
    if x.dtype != _BF16 or len(shape) != 3:
        raise SnGgufError(f"{what}: {name} must be bf16 [tokens][heads][dim], got {x.dtype} {tuple(shape)}")
    if x.requires_grad and torch.is_grad_enabled():
        raise SnGgufError(f"{what}: forward only, but {name} requires a gradient")
    tokens, heads, dim = shape
    t, h, e = x.stride()
    if tokens < 2:
        t = 0
    if heads < 2:
        h = 0
    if (e != 1 and x.numel()) or (pieces and (t % 8 or h % 8 or x.data_ptr() % 16)):
        return x.clone(memory_format=torch.contiguous_format), heads * dim, dim
    return x, t, h


def _apart(x: torch.Tensor) -> bool:
    """Whether no two rows of ``x`` share an element (as they do in an expanded tensor)."""
    reach = x.shape[2]
    for stride, size in sorted((x.stride(i), x.shape[i]) for i in (0, 1) if x.shape[i] > 1):
        if stride < reach:
            return False
        reach += stride * (size - 1)
    return True


def _places(x: torch.Tensor):
    """Where the rows of ``x`` [tokens][heads][dim] lie: (address, ((count, stride) of each axis), length of a row), in bytes."""
    size = x.element_size()
    return x.data_ptr(), [(x.shape[i], x.stride(i) * size) for i in (0, 1) if x.shape[i] > 1 and x.stride(i)], x.shape[2] * size


def _whole(x: torch.Tensor):
    """The same of a contiguous tensor: one row."""
    return x.data_ptr(), [], x.numel() * x.element_size()


def _share(a, b) -> bool:
    """Whether a row of ``a`` and one of ``b`` (of ``_places``) have a byte in common."""
    (a_at, a_axes, a_row), (b_at, b_axes, b_row) = a, b
    off = b_at - a_at

    def reach(axes, row):
        return sum((n - 1) * s for n, s in axes) + row

    if off >= reach(a_axes, a_row) or -off >= reach(b_axes, b_row):
        return False
    # interleaved, as the parts of a stacked projection are: what lies within some strides repeats at every multiple of what divides the longer ones
    for least in sorted({s for _, s in a_axes + b_axes}):
        every = math.gcd(*(s for _, s in a_axes + b_axes if s >= least))
        a_reach, b_reach = (reach([x for x in axes if x[1] < least], row) for axes, row in ((a_axes, a_row), (b_axes, b_row)))
        if a_reach <= off % every <= every - b_reach:
            return False
    # row by row
    starts = []
    for at, axes in ((0, a_axes), (off, b_axes)):
        rows = torch.tensor([at], dtype=torch.int64)
        for n, s in axes:
            rows = (rows[:, None] + torch.arange(n, dtype=torch.int64) * s).flatten()
        starts.append(rows)
    rows = starts[0].sort().values
    behind = torch.searchsorted(rows, starts[1], right=True)
    before = rows[(behind - 1).clamp(min=0)]
    after = rows[behind.clamp(max=len(rows) - 1)]
    return bool((((behind > 0) & (starts[1] - before < a_row)) | ((behind < len(rows)) & (after - starts[1] < b_row))).any())


def _rows_share(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether rows of two bf16 [tokens][heads][dim] share an element."""
    (n, heads, dim), (t, h, _), (_, b_heads, b_dim), (b_t, b_h, _) = a.shape, a.stride(), b.shape, b.stride()
    if not n or t != b_t or n != b.shape[0]:
        return _share(_places(a), _places(b))
    # the usual case, parts of one projection's output, without the rest (11 us, as much as a call)
    off, reach, b_reach = (b.data_ptr() - a.data_ptr()) // 2, (heads - 1) * h + dim, (b_heads - 1) * b_h + b_dim
    if off >= (n - 1) * t + reach or -off >= (n - 1) * t + b_reach or (t and reach <= off % t <= t - b_reach):
        return False
    return _share(_places(a), _places(b))


def _numbers(x: torch.Tensor, dtype: torch.dtype, count: Optional[int], what: str, name: str) -> torch.Tensor:
    if x.dtype != dtype or x.dim() != 1 or (count is not None and x.shape[0] != count):
        raise SnGgufError(f"{what}: {name} must be {dtype} [{count if count is not None else 'n'}], got {x.dtype} {tuple(x.shape)}")
    return x if x.stride(0) == 1 or x.shape[0] < 2 else x.contiguous()


class RotaryTable:
    """How the pairs of a head turn: pair i by ``turns[i]`` turns (of 2 pi) a position, and the result scaled by ``magnitude``.

    ``turns``: float64 on the device, one for each pair; pairs are elements (i, i + pairs), or (2 i, 2 i + 1) with
    ``interleaved``; elements behind the 2 * pairs first are left as they are.  ``for_model`` makes it of a checkpoint's settings."""

    __slots__ = ("_turns", "_interleaved", "_magnitude", "_struct", "_address", "_axes", "_memory")
    turns, interleaved, magnitude = map(_field, ("turns", "interleaved", "magnitude"))

    def __init__(self, turns: torch.Tensor, interleaved: bool = False, magnitude: float = 1.0) -> None:
        if turns.dtype != torch.float64 or turns.dim() != 1 or turns.shape[0] < 1 or not turns.is_cuda:
            raise SnGgufError(f"RotaryTable: turns must be float64 [pairs] on a HIP device, got {turns.dtype} {tuple(turns.shape)} on '{turns.device}'")
        if not math.isfinite(magnitude):
            raise SnGgufError("RotaryTable: the magnitude is not finite")
        self._turns = turns = turns if turns.is_contiguous() else turns.contiguous()
        self._interleaved, self._magnitude = bool(interleaved), float(magnitude)
        self._struct = _TableStruct(turns.data_ptr(), turns.shape[0], self._magnitude, self._interleaved)
        self._address = ctypes.addressof(self._struct)
        # (the same as a table of one axis and one part, where heads are normed as well)
        self._memory = turns.untyped_storage()      # (a tensor may be given other memory: its .data)
        self._axes = _AXES.pack(turns.data_ptr(), 0, turns.shape[0], self._magnitude, self._interleaved, 1, 2 * turns.shape[0], 0, 0, 0)

    @classmethod
    def for_model(cls, rotary_dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0, original_context: int = 0,
                  beta_fast: float = 32.0, beta_slow: float = 1.0, magnitude: Optional[float] = None, interleaved: bool = False,
                  device="cuda") -> "RotaryTable":
        """The table of ``rotary_dim`` elements with wavelengths from 2 pi to 2 pi ``base`` positions.

        ``scaling`` (a GGUF file's ``rope.scaling.type``): ``"none"``; ``"linear"``: positions count 1 / ``factor``;
        ``"yarn"``: pairs that turn more than ``beta_fast`` times over ``original_context`` positions are left, those that turn
        less than ``beta_slow`` times are stretched by ``factor``, with a ramp between, and the magnitude is 0.1 ln(factor) + 1."""
        if rotary_dim < 2 or rotary_dim % 2:
            raise SnGgufError(f"RotaryTable: {rotary_dim} elements are no pairs")
        if scaling not in ("none", "linear", "yarn") or not factor > 0 or not base > 1:
            raise SnGgufError(f"RotaryTable: scaling '{scaling}' by {factor} on base {base} is not known")
        half = rotary_dim // 2
        pair = torch.arange(half, dtype=torch.float64)
        turns = float(base) ** (-pair / half) / (2 * math.pi)
        size = 1.0
        if scaling == "linear":
            turns = turns / factor
        elif scaling == "yarn":
            if original_context < 1:
                raise SnGgufError("RotaryTable: yarn scaling needs the original context")
            at = [half * math.log(original_context / (beta * 2 * math.pi)) / math.log(base) for beta in (beta_fast, beta_slow)]
            low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rotary_dim - 1)
            keep = 1 - ((pair - low) / max(high - low, 0.001)).clamp(0, 1)
            turns = turns * keep + turns / factor * (1 - keep)
            size = 0.1 * math.log(factor) + 1 if factor > 1 else 1.0
        return cls(turns.to(device), interleaved, size if magnitude is None else magnitude)


class RotaryAxes:
    """How the pairs of a head turn by several positions of their token: pair i by ``turns[i]`` turns (of 2 pi) a position of axis
    ``axis[i]`` (time, row, column of a picture ...), and the result scaled by ``magnitude``.

    ``turns``: float64, ``axis``: int32, both on the device, one entry for each pair.  ``parts``: elements of the stretches, one to four, into
    which the first 2 * pairs elements of a head are cut; the pairs of one of n elements are (i, i + n / 2) of it, and pairs are
    counted from part to part (default: one part).  With ``interleaved`` pairs are (2 i, 2 i + 1) throughout.  Elements behind are
    left as they are.  An axis that positions do not have counts as the nearest that they have.  Fields cannot be replaced."""

    __slots__ = ("_turns", "_axis", "_parts", "_interleaved", "_magnitude", "_axes", "_pairs", "_memory")
    turns, axis, parts, interleaved, magnitude = map(_field, ("turns", "axis", "parts", "interleaved", "magnitude"))

    def __init__(self, turns: torch.Tensor, axis: torch.Tensor, parts: Optional[Sequence[int]] = None, interleaved: bool = False, magnitude: float = 1.0) -> None:
        if turns.dtype != torch.float64 or turns.dim() != 1 or turns.shape[0] < 1 or not turns.is_cuda:
            raise SnGgufError(f"RotaryAxes: turns must be float64 [pairs] on a HIP device, got {turns.dtype} {tuple(turns.shape)} on '{turns.device}'")
        self._pairs = pairs = turns.shape[0]
        axis = _numbers(axis, torch.int32, pairs, "RotaryAxes", "axis")
        _same_device("RotaryAxes", turns.get_device(), axis)
        parts = (2 * pairs,) if parts is None else tuple(parts)
        if not 1 <= len(parts) <= 4 or min(parts) < 2 or [n for n in parts if n % 2] or sum(parts) != 2 * pairs:
            raise SnGgufError(f"RotaryAxes: parts of {parts} elements (one to four, even) do not hold {pairs} pairs")
        if not math.isfinite(magnitude):
            raise SnGgufError("RotaryAxes: the magnitude is not finite")
        self._turns = turns = turns if turns.is_contiguous() else turns.contiguous()
        self._axis, self._parts, self._interleaved, self._magnitude = axis, parts, bool(interleaved), float(magnitude)
        self._memory = turns.untyped_storage(), axis.untyped_storage()
        self._axes = _AXES.pack(turns.data_ptr(), axis.data_ptr(), pairs, magnitude, self._interleaved, len(parts), *parts, *(0, 0, 0)[len(parts) - 1:])

    def __reduce__(self):               # (a copy has the addresses of its own tensors)
        return RotaryAxes, (self._turns, self._axis, self._parts, self._interleaved, self._magnitude)

    @classmethod
    def for_model(cls, parts: Sequence[tuple], interleaved: bool = False, device="cuda") -> "RotaryAxes":
        """The table of a head whose parts turn by an axis each: ``parts`` holds (elements, axis, base) of each part, with wavelengths
        from 2 pi to 2 pi ``base`` positions.  ``[(64, 0, 5e6), (32, 1, 1e4), (32, 2, 1e4)]``: half a head of 128 by the place in the
        text, a quarter each by row and column."""
        if not parts or any(n < 2 or n % 2 or not base > 1 for n, _, base in parts):
            raise SnGgufError(f"RotaryAxes: parts {parts} (elements, axis, base) are not known")
        turns = torch.cat([float(base) ** (-torch.arange(n // 2, dtype=torch.float64) / (n // 2)) / (2 * math.pi) for n, _, base in parts])
        axis = torch.cat([torch.full((n // 2,), int(a), dtype=torch.int32) for n, a, _ in parts])
        return cls(turns.to(device), axis.to(device), [n for n, _, _ in parts], interleaved)


class HeadNorm:
    """The norm of single heads in front of the rotation: y = weight * x / sqrt(mean(x^2) + eps), in 32 bits.

    ``weights``: one to four tensors [elements] on the device, bf16 or fp32, for the consecutive parts of a head that are normed each by
    itself (one: the whole head); their elements, multiples of 8, are a head's together.  Their memory is read at every call: a change in place counts, a tensor
    put in a module's place does not.  (Weights that do not start at a 16-byte boundary, or are not neighbours, are copied, and stay as they are now.)  A part
    whose squares add up to more than 32 bits hold, from magnitudes of 1.8e19 on, becomes zeros; with an ``eps`` of zero, or near it, one of magnitudes below
    1e-19 loses digits, and below 2.6e-23, where squares vanish, it is not finite.  Fields cannot be replaced."""

    __slots__ = ("_weights", "_eps", "_dim", "_norm", "_index", "_memory")
    weights, eps, dim = map(_field, ("weights", "eps", "dim"))

    def __init__(self, *weights: torch.Tensor, eps: float = 1e-6) -> None:
        if not 1 <= len(weights) <= 4:
            raise SnGgufError(f"HeadNorm: {len(weights)} parts (one to four are possible)")
        kind, index, at, sizes, kept, memory = weights[0].dtype, weights[0].get_device(), [], [], [], []
        for w in weights:
            size = w.numel() if w.dim() == 1 else 0
            if w.dtype is not kind or size < 8 or size % 8 or w.get_device() != index or index < 0 or (kind is not _BF16 and kind is not torch.float32):
                raise SnGgufError("HeadNorm: weights must be bf16 or fp32 [a multiple of 8] on a HIP device, of one type, "
                                  f"got {[(str(x.dtype), tuple(x.shape), str(x.device)) for x in weights]}")
            if type(w) is not torch.Tensor or w.requires_grad:
                if w.requires_grad and torch.is_grad_enabled():
                    raise SnGgufError("HeadNorm: forward only, but a weight requires a gradient")
                w = w.detach()          # (a parameter's .data may be set to another tensor, which is not what is read)
            address = w.data_ptr()
            if address % 16 or w.stride(0) != 1:
                w = w.clone(memory_format=torch.contiguous_format)
                address = w.data_ptr()
            kept.append(w)
            memory.append(w.untyped_storage())
            at.append(address)
            sizes.append(size)
        if not 0 <= eps <= 3.4028234663852886e38:       # (the largest number of 32 bits)
            raise SnGgufError(f"HeadNorm: eps is {eps}")
        self._weights, self._eps, self._dim, self._index = tuple(kept), float(eps), sum(sizes), index
        self._memory = memory
        rest = (0, 0, 0)[len(at) - 1:]
        self._norm = _NORM.pack(*at, *rest, *sizes, *rest, len(at), 2 if kind is _BF16 else 0, eps)

    def __reduce__(self):               # (a copy has the addresses of its own tensors)
        return functools.partial(HeadNorm, eps=self._eps), self._weights


def _axes_of(what: str, index: int, tokens: int, dim: int, positions: torch.Tensor, table, q_norm: Optional[HeadNorm], k_norm: Optional[HeadNorm]):
    """(positions, their axes, elements from one axis to the next) where heads are normed or turned by several positions, and the norms' addresses"""
    if isinstance(table, RotaryAxes):
        shape = positions.shape
        if positions.dtype != torch.int64 or len(shape) != 2 or shape[1] != tokens or shape[0] < 1:
            raise SnGgufError(f"{what}: positions must be torch.int64 [axes][{tokens}], got {positions.dtype} {tuple(shape)}")
        if positions.stride(1) != 1 and tokens > 1:
            positions = positions.contiguous()
        axes, stride = shape[0], positions.stride(0)
        if 2 * table._pairs > dim:
            raise SnGgufError(f"{what}: {table._pairs} pairs do not fit heads of {dim} elements")
        _same_device(what, index, table._axis)
    else:
        positions, axes, stride = _numbers(positions, torch.int64, tokens, what, "positions"), 1, 0
    for norm in (q_norm, k_norm):
        if norm is not None and (norm._dim != dim or norm._index != index):
            raise SnGgufError(f"{what}: a norm of {norm._dim} elements on device {norm._index} does not go with heads of {dim} on device {index}")
    if dim > 512:
        raise SnGgufError(f"{what}: heads of {dim} elements (up to 512 are normed or turned by several positions)")
    return positions, (positions.data_ptr(), axes, stride), q_norm and q_norm._norm, k_norm and k_norm._norm


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, table: Union[RotaryTable, RotaryAxes], inplace: bool = False,
           q_norm: Optional[HeadNorm] = None, k_norm: Optional[HeadNorm] = None):
    """Queries and keys turned by their positions: ``(q, k)``, new tensors or with ``inplace`` the given ones.

    q, k: bf16 [tokens][heads][dim], ``dim`` a multiple of 8; ``k`` may be None, either may have no heads.  positions: int64 [tokens], or [axes][tokens] with
    ``RotaryAxes``.  ``q_norm``, ``k_norm``: the norm of each head in front of the rotation, in the same launch; norm and rotation are
    in 32 bits and rounded once.  ``dim`` is up to 1024, up to 512 with a norm or several axes.  In place, no two rows may share an element."""
    q0, k0 = q, k
    q, qt, qh = _heads(q, "rotary", "q")
    tokens, heads, dim = q.shape
    index = q.get_device()
    wide = q_norm is not None or k_norm is not None or isinstance(table, RotaryAxes)
    if wide:
        positions, at, q_at, k_at = _axes_of("rotary", index, tokens, dim, positions, table, q_norm, k_norm)
    else:
        positions = _numbers(positions, torch.int64, tokens, "rotary", "positions")
    _same_device("rotary", index, k, positions, table._turns)
    if k is not None:
        k, kt, kh = _heads(k, "rotary", "k")
        if k.shape[0] != tokens or k.shape[2] != dim:
            raise SnGgufError(f"rotary: k {tuple(k.shape)} does not go with q {tuple(q.shape)}")
    if inplace and (q is not q0 or k is not k0):
        raise SnGgufError("rotary: in place needs the elements of a head next to each other")
    if inplace and not (_apart(q) and (k is None or (_apart(k) and not (q.numel() and k.numel() and _rows_share(q, k))))):
        raise SnGgufError("rotary: in place needs rows that share no element")
    q_out, qot, qoh = (q, qt, qh) if inplace else (_new(q), heads * dim, dim)
    k_out = k if inplace or k is None else _new(k)
    if k is None or not k.shape[1]:
        rest = (None, 0, 0, 0, None, 0, 0)
    else:
        rest = (k.data_ptr(), k.shape[1], kt, kh, k_out.data_ptr(), *((kt, kh) if inplace else (k.shape[1] * dim, dim)))
    first = (q.data_ptr(), heads, qt, qh, q_out.data_ptr(), qot, qoh)
    if not heads:                       # keys alone: in the queries' place
        first, rest, heads = rest, (None, 0, 0, 0, None, 0, 0), rest[1]
        if wide:
            q_at, k_at = k_at, None
    if tokens and heads:
        if wide:
            _launch(index, "sngguf_head_rotary", table._axes, *at, tokens, dim, q_at, *first, k_at, *rest)
        else:
            _launch(index, "sngguf_rotary", table._address, positions.data_ptr(), tokens, dim, *first, *rest)
    return q_out, k_out


class PagedKVCache:
    """Keys and values of ``pages`` * ``page_size`` tokens of one layer.

    bf16: ``k`` and ``v`` are bf16 ``[pages][kv_heads][page_size][dim]``.  8 bits: int8 of that shape, with fp16 ``k_scale`` and
    ``v_scale`` ``[pages][kv_heads][dim / 32][page_size]``; 32 elements of a token share a scale, as in a Q8_0 block (magnitudes
    beyond 65024 saturate, a NaN makes its 32 elements NaN).  ``page_size`` is a power of two from 16 to 4096, ``dim`` a multiple
    of 32 up to 256.  ``PagedKVCache.empty`` allocates one; the constructor takes tensors that are there (keys and values that share memory
    can be read, not written).

    Token t of a sequence lies at slot ``page_of_the_sequence[t // page_size] * page_size + t % page_size``."""

    __slots__ = ("_k", "_v", "_k_scale", "_v_scale", "_quant_type", "_pages", "_kv_heads", "_page_size", "_dim", "_struct", "_address", "_index", "_shared", "_memory")
    k, v, k_scale, v_scale, quant_type, pages, kv_heads, page_size, dim = map(_field, ("k", "v", "k_scale", "v_scale", "quant_type", "pages", "kv_heads", "page_size", "dim"))

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None) -> None:
        if not k.is_cuda:
            raise SnGgufError(f"sn_gguf ops run on a HIP device only, got a cache on '{k.device}'; there is no CPU implementation")
        shape = k.shape
        if len(shape) != 4 or v.shape != shape or v.dtype != k.dtype or k.dtype not in (_BF16, torch.int8) or not k.is_contiguous() or not v.is_contiguous():
            raise SnGgufError("PagedKVCache: k and v must be contiguous bf16 or int8 [pages][kv_heads][page_size][dim]")
        pages, kv_heads, page, dim = shape
        if pages < 1 or kv_heads < 1 or page < 16 or page > 4096 or page & (page - 1) or dim % 32 or not 32 <= dim <= 256:
            raise SnGgufError(f"PagedKVCache: pages of 16 .. 4096 tokens (a power of two) and heads of 32 .. 256 elements (a multiple of 32) are needed, got {tuple(shape)}")
        q8 = k.dtype == torch.int8
        for s in (k_scale, v_scale):
            if (s is not None) != q8 or (q8 and (s.dtype != torch.float16 or s.shape != (pages, kv_heads, dim // 32, page) or not s.is_contiguous())):
                raise SnGgufError("PagedKVCache: an int8 cache has contiguous fp16 scales [pages][kv_heads][dim / 32][page_size], a bf16 cache none")
        index = k.get_device()
        _same_device("PagedKVCache", index, v, k_scale, v_scale)
        self._k, self._v, self._k_scale, self._v_scale = k, v, k_scale, v_scale
        self._memory = k.untyped_storage(), v.untyped_storage(), *((k_scale.untyped_storage(), v_scale.untyped_storage()) if q8 else ())
        self._quant_type = ops.Q8_0 if q8 else ops.BF16
        self._pages, self._kv_heads, self._page_size, self._dim, self._index = pages, kv_heads, page, dim, index
        at = (k.data_ptr(), v.data_ptr(), k_scale.data_ptr() if q8 else None, v_scale.data_ptr() if q8 else None)
        self._struct = _CacheStruct(*at, pages, page, kv_heads, dim, self._quant_type)
        count = pages * kv_heads * page * dim
        self._shared = abs(at[0] - at[1]) < (count if q8 else 2 * count) or (q8 and abs(at[2] - at[3]) < count // 16)
        self._address = ctypes.addressof(self._struct)

    @classmethod
    def empty(cls, pages: int, kv_heads: int, page_size: int, dim: int, quant_type: int = ops.Q8_0, device="cuda") -> "PagedKVCache":
        """A cache of uninitialised pages: ``quant_type`` ``ops.Q8_0`` (8 bits) or ``ops.BF16``."""
        if quant_type not in (ops.Q8_0, ops.BF16):
            raise SnGgufError(f"PagedKVCache: quant type {quant_type} is not implemented (have Q8_0=8, BF16=30)")
        q8 = quant_type == ops.Q8_0
        k, v = (torch.empty((pages, kv_heads, page_size, dim), dtype=torch.int8 if q8 else _BF16, device=device) for _ in range(2))
        scales = [torch.empty((pages, kv_heads, dim // 32, page_size), dtype=torch.float16, device=device) for _ in range(2)] if q8 else [None, None]
        return cls(k, v, *scales)

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self._k, self._v, self._k_scale, self._v_scale) if t is not None)

    def _rows(self, k, v, slots, what):
        if self._shared:
            raise SnGgufError(f"{what}: the cache's keys and values share memory")
        (k, kt, kh), (v, vt, vh) = _heads(k, what, "k"), _heads(v, what, "v")
        if k.shape != v.shape or k.shape[1] != self._kv_heads or k.shape[2] != self._dim:
            raise SnGgufError(f"{what}: k {tuple(k.shape)} and v {tuple(v.shape)} do not go with a cache of {self._kv_heads} heads of {self._dim}")
        slots = _numbers(slots, torch.int64, k.shape[0], what, "slots")
        _same_device(what, self._index, k, v, slots)
        return k, v, slots, (k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, slots.data_ptr(), k.shape[0])

    def write(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """Keys and values [tokens][kv_heads][dim] into ``slots`` (int64 [tokens], different ones; negative ones and those behind
        the last page are passed over).  k and v may be views of the cache itself, of other slots."""
        k, v, slots, rows = self._rows(k, v, slots, "PagedKVCache.write")
        if k.shape[0]:
            _launch(self._index, "sngguf_cache_write", self._address, *rows)

    def write_rotary(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, table: Union[RotaryTable, RotaryAxes],
                     slots: torch.Tensor, inplace: bool = False, q_norm: Optional[HeadNorm] = None, k_norm: Optional[HeadNorm] = None) -> torch.Tensor:
        """``rotary`` of q and k (with their norms, if given), then ``write`` of the turned k and of v, in one launch; returns the turned q
        (with ``inplace`` in q's own memory; k is left as it is)."""
        what = "PagedKVCache.write_rotary"
        q0 = q
        q, qt, qh = _heads(q, what, "q")
        k, v, slots, rows = self._rows(k, v, slots, what)
        tokens, heads, dim = q.shape
        if k.shape[0] != tokens or dim != self._dim:
            raise SnGgufError(f"{what}: q {tuple(q.shape)} does not go with k {tuple(k.shape)}")
        if inplace and (q is not q0 or not _apart(q) or (q.numel() and (_rows_share(q, k) or _rows_share(q, v)))):
            raise SnGgufError(f"{what}: in place needs rows that share no element, the elements of a head next to each other")
        wide = q_norm is not None or k_norm is not None or isinstance(table, RotaryAxes)
        if wide:
            positions, at, q_at, k_at = _axes_of(what, self._index, tokens, dim, positions, table, q_norm, k_norm)
        else:
            positions = _numbers(positions, torch.int64, tokens, what, "positions")
        _same_device(what, self._index, q, positions, table._turns)
        out, ot, oh = (q, qt, qh) if inplace else (_new(q), heads * dim, dim)
        if tokens and wide:
            _launch(self._index, "sngguf_cache_write_head_rotary", self._address, table._axes, *at, q_at, q.data_ptr(), heads, qt, qh, out.data_ptr(),
                    ot, oh, k_at, *rows)
        elif tokens:
            _launch(self._index, "sngguf_cache_write_rotary", self._address, table._address, positions.data_ptr(), q.data_ptr(), heads, qt, qh, out.data_ptr(),
                    ot, oh, *rows)
        return out

    def read(self, slots: torch.Tensor):
        """``(k, v)`` of ``slots`` (int64 [tokens]) as bf16 [tokens][kv_heads][dim]; a slot outside the cache gives zeros."""
        slots = _numbers(slots, torch.int64, None, "PagedKVCache.read", "slots")
        _same_device("PagedKVCache.read", self._index, slots)
        tokens = slots.shape[0]
        k = self._k.new_empty((tokens, self._kv_heads, self._dim), dtype=_BF16)
        v = torch.empty_like(k)
        if tokens:
            _launch(self._index, "sngguf_cache_read", self._address, slots.data_ptr(), tokens, k.data_ptr(), v.data_ptr())
        return k, v


def _output(out: Optional[torch.Tensor], q: torch.Tensor, what: str, k: torch.Tensor, v: torch.Tensor, *scales: Optional[torch.Tensor]):
    """(out, its token and head strides); k, v: packed rows, or the halves of a cache"""
    tokens, heads, dim = q.shape
    if out is None:
        return _new(q), heads * dim, dim
    if out.dtype != _BF16 or out.shape != q.shape or out.get_device() != q.get_device():
        raise SnGgufError(f"{what}: out must be bf16 {tuple(q.shape)} on q's device")
    rows, t, h = _heads(out, what, "out", True)
    if rows is not out:
        raise SnGgufError(f"{what}: out must have rows of whole 16-byte pieces")
    if out.numel():
        if not _apart(out) or any(_rows_share(out, x) if len(x.shape) == 3 else _share(_places(out), _whole(x)) for x in (q, k, v, *scales) if x is not None and x.numel()):
            raise SnGgufError(f"{what}: out must not overlap itself or an input")
    return out, t, h


def _check_options(what: str, heads: int, kv_heads: int, dim: int, scale: Optional[float], window: int) -> float:
    if kv_heads < 1 or heads % kv_heads or heads < 1:
        raise SnGgufError(f"{what}: {heads} query heads cannot share {kv_heads} key / value heads")
    if dim % 32 or not 32 <= dim <= 256:
        raise SnGgufError(f"{what}: heads of {dim} elements (a multiple of 32 up to 256 is needed)")
    if not 0 <= window < 1 << 63:
        raise SnGgufError(f"{what}: a window of {window} tokens")
    scale = dim ** -0.5 if scale is None else float(scale)
    if not 1e-30 <= scale <= 1e30:
        raise SnGgufError(f"{what}: a scale of {scale}")
    return scale


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, ends_q: torch.Tensor, ends_k: Optional[torch.Tensor] = None,
                     causal: bool = True, scale: Optional[float] = None, window: int = 0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of packed sequences: sequence i has the queries ``ends_q[i] : ends_q[i + 1]`` and the keys ``ends_k[i] :
    ends_k[i + 1]`` (int32 [sequences + 1], not decreasing; ``ends_k`` defaults to ``ends_q``).

    q [tokens][heads][dim], k and v [keys][kv_heads][dim], ``heads`` a multiple of ``kv_heads``, ``dim`` a multiple of 32 up to
    256.  Causal: the last query of a sequence stands at its last key, and none sees a key behind its own place; ``window`` > 0: only the last
    ``window`` keys up to it.  A query that sees nothing, or only scores of minus infinity, gives zeros, and keys and values that a query does not see
    have no part in its result, whatever they hold.  ``scale`` defaults to dim ** -0.5.  Rows of ``out`` behind the last sequence are not
    written; ``out`` overlaps no input."""
    what = "prompt_attention"
    (q, qt, qh), (k, kt, kh), (v, vt, vh) = _heads(q, what, "q", True), _heads(k, what, "k", True), _heads(v, what, "v", True)
    tokens, heads, dim = q.shape
    if k.shape != v.shape or k.shape[2] != dim:
        raise SnGgufError(f"{what}: k {tuple(k.shape)} and v {tuple(v.shape)} do not go with q {tuple(q.shape)}")
    keys, kv_heads = k.shape[0], k.shape[1]
    scale = _check_options(what, heads, kv_heads, dim, scale, window)
    if window and not causal:
        raise SnGgufError(f"{what}: a window needs causal attention")
    ends_q = _numbers(ends_q, torch.int32, None, what, "ends_q")
    ends_k = ends_q if ends_k is None else _numbers(ends_k, torch.int32, ends_q.shape[0], what, "ends_k")
    if ends_q.shape[0] < 1:
        raise SnGgufError(f"{what}: ends_q has no entry")
    index = q.get_device()
    _same_device(what, index, k, v, ends_q, ends_k)
    out, ot, oh = _output(out, q, what, k, v)
    sequences = ends_q.shape[0] - 1
    if tokens and sequences:
        nbytes = _prompt_workspace(tokens, keys, sequences, heads, kv_heads, dim)
        _launch_with_workspace(index, nbytes, "sngguf_attention", q.data_ptr(), tokens, heads, qt, qh, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, keys,
                               kv_heads, dim, ends_q.data_ptr(), ends_k.data_ptr(), sequences, scale, int(causal), window, out.data_ptr(), ot, oh)
    return out


def _paged(what: str, q: torch.Tensor, cache: PagedKVCache, pages: torch.Tensor, lens: torch.Tensor, ends_q: Optional[torch.Tensor], max_new: int,
           scale: Optional[float], window: int):
    """The checked arguments of a call over a cache: (q, its token and head strides, pages, lens, ends_q, scale)"""
    q, qt, qh = _heads(q, what, "q", True)
    tokens, heads, dim = q.shape
    if dim != cache._dim:
        raise SnGgufError(f"{what}: q {tuple(q.shape)} does not go with a cache of heads of {cache._dim}")
    scale = _check_options(what, heads, cache._kv_heads, dim, scale, window)
    if not 0 <= max_new < 1 << 63:
        raise SnGgufError(f"{what}: max_new is {max_new}")
    lens = _numbers(lens, torch.int32, None, what, "lens")
    sequences = lens.shape[0]
    if pages.dtype != torch.int32 or pages.dim() != 2 or pages.shape[0] != sequences:
        raise SnGgufError(f"{what}: pages must be int32 [{sequences}][width], got {pages.dtype} {tuple(pages.shape)}")
    width = pages.shape[1]
    if width * cache._page_size > (1 << 31) - 65536:
        raise SnGgufError(f"{what}: {width} pages of {cache._page_size} tokens a sequence are too many")
    if (width > 1 and pages.stride(1) != 1) or (sequences > 1 and pages.stride(0) < width):
        pages = pages.contiguous()
    if ends_q is not None:
        ends_q = _numbers(ends_q, torch.int32, sequences + 1, what, "ends_q")
    elif tokens != sequences:
        raise SnGgufError(f"{what}: {tokens} queries of {sequences} sequences need ends_q")
    _same_device(what, cache._index, q, pages, lens, ends_q)
    return q, qt, qh, pages, lens, ends_q, scale


def paged_attention(q: torch.Tensor, cache: PagedKVCache, pages: torch.Tensor, lens: torch.Tensor, ends_q: Optional[torch.Tensor] = None,
                    max_new: int = 0, scale: Optional[float] = None, window: int = 0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of new tokens over sequences in a paged cache, their own keys and values already written.

    pages: int32 [sequences][width], the pages of each sequence in order.  lens: int32 [sequences], its tokens in all.  The queries
    of sequence i are ``ends_q[i] : ends_q[i + 1]`` (int32 [sequences + 1]) and stand at its last places; without ``ends_q`` every
    sequence has one, in order.  ``max_new``: the most queries of any sequence, where the program knows it (0: unknown); it
    decides which kernels are launched and never what they compute.  With a ``window``, the pages in front of it may be anyone's.
    ``scale``, ``window``, ``out``: as ``prompt_attention``."""
    what = "paged_attention"
    q, qt, qh, pages, lens, ends_q, scale = _paged(what, q, cache, pages, lens, ends_q, max_new, scale, window)
    (tokens, heads, dim), (sequences, width) = q.shape, pages.shape
    out, ot, oh = _output(out, q, what, cache._k, cache._v, cache._k_scale, cache._v_scale)
    if tokens and sequences:
        if ends_q is None:
            max_new = 1
        nbytes = _paged_workspace(tokens, sequences, max_new, width * cache._page_size, heads, cache._kv_heads, dim)
        _launch_with_workspace(cache._index, nbytes, "sngguf_paged_attention", q.data_ptr(), tokens, heads, qt, qh, cache._address, pages.data_ptr(),
                               pages.stride(0), width, lens.data_ptr(), ops._ptr(ends_q), sequences, max_new, scale, window, out.data_ptr(), ot, oh)
    return out


def shared_prefix_attention(q: torch.Tensor, cache: PagedKVCache, pages: torch.Tensor, lens: torch.Tensor, groups: torch.Tensor, shared: torch.Tensor,
                            ends_q: Optional[torch.Tensor] = None, max_new: int = 0, scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``paged_attention`` of sequences that begin alike, as answers to one prompt do: what a group has in common is read once for all of it.

    Group g is the sequences ``groups[g] : groups[g + 1]`` (int32 [groups + 1], not decreasing), whose first ``shared[g]`` tokens (int32 [groups])
    lie in the pages of the first of them that has queries; the other ones' pages hold the same there (``PageTables.fork`` makes them the same pages).
    No more counts as common than every sequence of the group with queries has in front of its new tokens; sequences of no group, or of a group of
    one, have nothing in common.  The result is that of ``paged_attention`` but for the order of its sums; everything else is as there, and where
    nothing would be gained (few keys, by the width of the tables, or many new tokens of each sequence) it is what runs."""
    what = "shared_prefix_attention"
    q, qt, qh, pages, lens, ends_q, scale = _paged(what, q, cache, pages, lens, ends_q, max_new, scale, 0)
    (tokens, heads, dim), (sequences, width) = q.shape, pages.shape
    groups = _numbers(groups, torch.int32, None, what, "groups")
    if groups.shape[0] < 1:
        raise SnGgufError(f"{what}: groups has no entry")
    count = groups.shape[0] - 1
    shared = _numbers(shared, torch.int32, count, what, "shared")
    _same_device(what, cache._index, groups, shared)
    if not count:
        return paged_attention(q, cache, pages, lens, ends_q, max_new, scale, out=out)
    out, ot, oh = _output(out, q, what, cache._k, cache._v, cache._k_scale, cache._v_scale)
    if tokens and sequences:
        if ends_q is None:
            max_new = 1
        nbytes = _shared_workspace(tokens, sequences, count, max_new, width * cache._page_size, heads, cache._kv_heads, dim, cache._quant_type)
        _launch_with_workspace(cache._index, nbytes, "sngguf_shared_attention", q.data_ptr(), tokens, heads, qt, qh, cache._address, pages.data_ptr(),
                               pages.stride(0), width, lens.data_ptr(), ops._ptr(ends_q), sequences, groups.data_ptr(), shared.data_ptr(), count, max_new, scale,
                               out.data_ptr(), ot, oh)
    return out
