"""What is timed of the operators between a decoder layer's projections: rotary positions, the paged cache of keys and
values, and the attention that reads prompts or that cache.

A layer of the 8B backbone has 32 query heads and 8 key / value heads of 128 elements behind its q / k / v projections;
most cases are of that shape, drawn ones of others too.  Kinds of case

* ``rotary``  query and key heads of some tokens turned by their positions;
* ``append``  the step between the projections and attention of a program that keeps an 8-bit (or bf16) paged cache: queries
              and keys turned, keys and values written to the cache; then what was written is read back;
* ``read``    tokens of a cache decoded to bf16, for a program that wants the keys and values themselves;
* ``prompt``  attention over packed sequences of different lengths, each token to those before it or to all;
* ``paged``   new tokens, one a sequence or a chunk of a prompt, over sequences that lie in a paged cache.

An 8-bit cache holds runs of 32 elements as whole numbers from -127 to 127 and one fp16 scale a run (the arithmetic of
the Q8_0 blocks), elements as [page][head][token][element], scales as [page][head][run][token].
"""
import math

import torch

own = False

LAYER = {"heads": 32, "kv_heads": 8, "dim": 128}


def listed():
    return [
        # one token of one sequence: latency
        {"name": "rotary_1token", "kind": "rotary", "tokens": 1, **LAYER, "turned": 128, "interleaved": False, "far": 4096, "scaling": 0},
        # a long prompt, half of each head turned in neighbouring pairs, positions stretched to a longer context
        {"name": "rotary_8192tokens_half_head", "kind": "rotary", "tokens": 8192, **LAYER, "turned": 64, "interleaved": True, "far": 1 << 20, "scaling": 8},
        # batched decode: one new token of each of 24 sequences
        {"name": "append_24tokens_q8", "kind": "append", "tokens": 24, **LAYER, "page": 16, "bits": 8},
        # a prompt of an odd number of tokens goes into the cache
        {"name": "append_5003tokens_q8", "kind": "append", "tokens": 5003, **LAYER, "page": 64, "bits": 8},
        # the keys and values of a long context as tensors
        {"name": "read_40000tokens_q8", "kind": "read", "tokens": 40000, **LAYER, "page": 64, "bits": 8},
        # a short prompt
        {"name": "prompt_77tokens", "kind": "prompt", "lens": "77", "before": 0, "causal": True, "window": 0, **LAYER},
        # prompts of several users in one batch
        {"name": "prompt_ragged", "kind": "prompt", "lens": "1,2047,33,700,1300,512,129", "before": 0, "causal": True, "window": 0, **LAYER},
        # image tokens of a 2048 x 2048 picture after a prompt: each sees the prompt and the whole picture
        {"name": "image_4096_after_512", "kind": "prompt", "lens": "4096", "before": 512, "causal": False, "window": 0, **LAYER},
        # a long document
        {"name": "prompt_16384tokens", "kind": "prompt", "lens": "16384", "before": 0, "causal": True, "window": 0, **LAYER},
        # batched decode over contexts of different lengths
        {"name": "decode_24_ragged_q8", "kind": "paged", "new": "1" + ",1" * 23, "lens": ",".join(str(37 + 433 * ((7 * i) % 24)) for i in range(24)),
         "page": 16, "bits": 8, "window": 0, **LAYER},
        # one sequence with a very long context
        {"name": "decode_1_of_131071_bf16", "kind": "paged", "new": "1", "lens": "131071", "page": 64, "bits": 16, "window": 0, **LAYER},
        # the next chunk of a long prompt, beside short ones that are further on
        {"name": "chunk_1024_of_30000_q8", "kind": "paged", "new": "1024,1,300,1", "lens": "30000,5000,300,900", "page": 32, "bits": 8, "window": 0, **LAYER},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kv_heads, group = rng.choice([(8, 4)] * 3 + [(4, 7), (8, 5), (16, 1), (2, 8), (1, 12)])
    shape = {"heads": kv_heads * group, "kv_heads": kv_heads, "dim": rng.choice([128] * 3 + [64, 96, 256])}
    kind = rng.choice(["rotary", "append", "read", "prompt", "prompt", "paged", "paged", "paged"])
    bits, page = rng.choice([8, 8, 16]), rng.choice([16, 32, 64, 128])
    if kind == "rotary":
        return {"kind": kind, "tokens": _log_int(rng, 1, 8192), **shape, "turned": rng.choice([shape["dim"], shape["dim"] // 2]),
                "interleaved": rng.random() < 0.5, "far": _log_int(rng, 512, 1 << 20), "scaling": rng.choice([0, 0, 4, 8])}
    if kind in ("append", "read"):
        return {"kind": kind, "tokens": _log_int(rng, 1, 5000 if kind == "append" else 40000), **shape, "page": page, "bits": bits}
    window = rng.choice([0, 0, 0, _log_int(rng, 16, 2048)])
    if kind == "prompt":
        count = rng.choice([1, 1, 2, 5, 9])
        # together no more pairs of tokens than the longest listed prompt has
        most = min(8192, int(8192 * math.sqrt(32 / shape["heads"] / count)))
        lens = [_log_int(rng, 1, most) for _ in range(count)]
        causal = rng.random() < 0.7
        return {"kind": kind, "lens": ",".join(map(str, lens)), "before": rng.choice([0, 0, _log_int(rng, 1, 1024)]), "causal": causal,
                "window": window if causal else 0, **shape}
    count = rng.choice([1, 2, 5, 16, 48])
    chunk = rng.choice([1, 1, 1, 3, _log_int(rng, 2, 1024)])
    lens = [_log_int(rng, 1, 120000 // count) for _ in range(count)]
    new = [min(length, chunk if i % 3 == 0 else 1) for i, length in enumerate(lens)]
    return {"kind": kind, "new": ",".join(map(str, new)), "lens": ",".join(map(str, lens)), "page": page, "bits": bits, "window": window, **shape}


def _ints(text):
    return [int(t) for t in text.split(",")]


def _visible(case):
    """(query, key) pairs of a head that take part, over all sequences."""
    lens = _ints(case["lens"])
    new = lens if case["kind"] == "prompt" else _ints(case["new"])
    pairs = 0
    for n, length in zip(new, lens):
        total = length + case["before"] if case["kind"] == "prompt" else length
        if not case.get("causal", True):
            pairs += n * total
            continue
        first, last = total - n + 1, total      # keys that the first and the last query see without a window
        w = case["window"] or total
        full = min(max(w - first, 0), n)        # queries that see fewer keys than the window is wide
        pairs += full * first + full * (full - 1) // 2 + (n - full) * min(w, last)
    return pairs


def work(case):
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    element = 2 if case.get("bits", 16) == 16 else 1 + 2 / 32
    if case["kind"] == "rotary":
        values = case["tokens"] * (heads + kv) * dim
        return {"bytes": 4 * values, "flops": 3 * values}
    if case["kind"] == "append":
        t = case["tokens"]
        # q, k, v in, q out, the cache written, and read back as bf16
        return {"bytes": t * dim * (4 * heads + 4 * kv + 2 * kv * (2 * element + 2)), "flops": t * dim * (3 * heads + 10 * kv)}
    if case["kind"] == "read":
        return {"bytes": 2 * case["tokens"] * kv * dim * (element + 2), "flops": 2 * case["tokens"] * kv * dim}
    lens = _ints(case["lens"])
    new = lens if case["kind"] == "prompt" else _ints(case["new"])
    keys = 0
    for n, length in zip(new, lens):
        total = length + case["before"] if case["kind"] == "prompt" else length
        keys += min(total, case["window"] + n - 1) if case["window"] else total
    return {"bytes": 4 * sum(new) * heads * dim + 2 * keys * kv * dim * element, "flops": 4 * _visible(case) * heads * dim}


# ---- inputs -------------------------------------------------------------------------------------------------------------


def _heads(gen, tokens, heads, dim, wide=False):
    """bf16 values of ``tokens`` tokens; keys have a few wide channels, as trained ones do."""
    x = torch.randn((tokens, heads, dim), generator=gen, device="cuda", dtype=torch.float32)
    if wide:
        x *= 1 + 3 * (torch.rand((heads, dim), generator=gen, device="cuda") > 0.95)
    return x.to(torch.bfloat16)


def _quantised(x):
    """(whole numbers, fp16 scales) of runs of 32 elements."""
    runs = x.float().unflatten(-1, (-1, 32))
    scale = (runs.abs().amax(-1, keepdim=True) / 127).clamp(max=512).to(torch.float16)
    s = scale.float()
    q = torch.where(s > 0, torch.round(runs / s), torch.zeros((), device=x.device)).clamp(-127, 127)
    return q.flatten(-2).to(torch.int8), scale.squeeze(-1)


def _empty_cache(case, pages):
    """The tensors of a cache, by the names that the framework gives them."""
    kv, dim, page = case["kv_heads"], case["dim"], case["page"]
    kind = torch.int8 if case["bits"] == 8 else torch.bfloat16
    cache = {n: torch.zeros((pages, kv, page, dim), dtype=kind, device="cuda") for n in ("k", "v")}
    if case["bits"] == 8:
        cache.update({n: torch.zeros((pages, kv, dim // 32, page), dtype=torch.float16, device="cuda") for n in ("k_scale", "v_scale")})
    return cache


def _write(cache, name, x, slots):
    """Tokens ``x`` [T][heads][dim] to ``slots`` of one half of a cache."""
    page = cache[name].shape[2]
    at, row = slots // page, slots % page
    if cache[name].dtype == torch.int8:
        q, scale = _quantised(x)
        cache[name][at, :, row] = q
        cache[name + "_scale"][at, :, :, row] = scale
    else:
        cache[name][at, :, row] = x


def _read(cache, name, slots):
    """Tokens at ``slots`` in 32 bits: [..., heads, dim]."""
    page = cache[name].shape[2]
    at, row = slots // page, slots % page
    x = cache[name][at, :, row].float()
    if cache[name].dtype == torch.int8:
        x = (x.unflatten(-1, (-1, 32)) * cache[name + "_scale"][at, :, :, row].float().unsqueeze(-1)).flatten(-2)
    return x


def _base(case):
    return 5000000.0 if case["scaling"] else 1000000.0


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    s = {"case": case}
    if case["kind"] in ("rotary", "append"):
        t = case["tokens"]
        # one projection's output holds q, k and v of a token next to each other
        qkv = torch.cat([_heads(gen, t, heads, dim), _heads(gen, t, kv, dim, wide=True), _heads(gen, t, kv, dim)], 1)
        s["q"], s["k"], s["v"] = qkv.split([heads, kv, kv], 1)
        far = case.get("far", 40000)
        start = int(torch.randint(0, max(1, far - t), (1,), generator=gen, device="cuda"))
        s["positions"] = torch.arange(start, start + t, device="cuda")
        s["turns"] = _turns(case if case["kind"] == "rotary" else {**case, "turned": dim, "scaling": 0}).cuda()
        s["table"] = _table(case, s["turns"])
    if case["kind"] in ("append", "read"):
        t, page = case["tokens"], case["page"]
        pages = -(-t // page) + 7
        s["cache"] = _empty_cache(case, pages)
        order = torch.randperm(pages, generator=gen, device="cuda")
        s["slots"] = order[torch.arange(t, device="cuda") // page] * page + torch.arange(t, device="cuda") % page
        if case["kind"] == "read":
            _write(s["cache"], "k", _heads(gen, t, kv, dim, wide=True), s["slots"])
            _write(s["cache"], "v", _heads(gen, t, kv, dim), s["slots"])
    if case["kind"] == "prompt":
        lens = _ints(case["lens"])
        total = [n + case["before"] for n in lens]
        s["q"] = _heads(gen, sum(lens), heads, dim)
        s["k"], s["v"] = _heads(gen, sum(total), kv, dim, wide=True), _heads(gen, sum(total), kv, dim)
        s["new"], s["lens"] = lens, total
        s["ends_k"] = torch.tensor([0] + total, device="cuda").cumsum(0).to(torch.int32)
        s["ends"] = torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)
    if case["kind"] == "paged":
        s["new"], s["lens"], page = _ints(case["new"]), _ints(case["lens"]), case["page"]
        width = -(-max(s["lens"]) // page)
        pages = [-(-n // page) for n in s["lens"]]
        order = torch.randperm(sum(pages), generator=gen, device="cuda").to(torch.int32)
        s["pages"] = torch.zeros((len(pages), width), dtype=torch.int32, device="cuda")
        for i, n in enumerate(pages):
            s["pages"][i, :n] = order[sum(pages[:i]):sum(pages[:i + 1])]
        s["cache"] = _empty_cache(case, sum(pages))
        slots = (order.long()[:, None] * page + torch.arange(page, device="cuda")).flatten()
        _write(s["cache"], "k", _heads(gen, len(slots), kv, dim, wide=True), slots)
        _write(s["cache"], "v", _heads(gen, len(slots), kv, dim), slots)
        s["q"] = _heads(gen, sum(s["new"]), heads, dim)
        s["ends"] = torch.tensor([0] + s["new"], device="cuda").cumsum(0).to(torch.int32)
        s["lens_dev"] = torch.tensor(s["lens"], dtype=torch.int32, device="cuda")
    return s


# ---- the operators in plain form ------------------------------------------------------------------------------------


def _turns(case):
    """Turns (of 2 pi) a position for each pair, in 64 bits; ``scaling`` > 0 stretches the slow pairs that many times and
    leaves the fast ones, with a ramp between the pairs that turn 32 times and once over 32768 positions."""
    half = case["turned"] // 2
    pair = torch.arange(half, dtype=torch.float64)
    turns = _base(case) ** (-pair / half) / (2 * math.pi)
    if case["scaling"]:
        at = [half * math.log(32768 / (rounds * 2 * math.pi)) / math.log(_base(case)) for rounds in (32, 1)]
        low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), 2 * half - 1)
        keep = 1 - ((pair - low) / max(high - low, 0.001)).clamp(0, 1)
        turns = turns * keep + turns / case["scaling"] * (1 - keep)
    return turns


def _table(case, turns):
    """What a program makes once of its model's settings: how pairs turn, and by how much the result is scaled."""
    return {"turns": turns, "interleaved": case.get("interleaved", False),
            "magnitude": 0.1 * math.log(case["scaling"]) + 1 if case.get("scaling") else 1.0}


def _turn(x, positions, table):
    """x [T][heads][dim] turned by its positions: angles in 64 bits, cosines and sines rounded to 32."""
    turned = 2 * table["turns"].numel()
    turns = positions.double()[:, None] * table["turns"]
    angle = 2 * math.pi * (turns - turns.round())
    c = (angle.cos() * table["magnitude"]).float()[:, None]
    s = (angle.sin() * table["magnitude"]).float()[:, None]
    part = x[..., :turned].float()
    if table["interleaved"]:
        a, b = part[..., 0::2], part[..., 1::2]
        y = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = part.chunk(2, -1)
        y = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([y.to(x.dtype), x[..., turned:]], -1)


def _padded(ends, lens, most, device):
    """Row of each (sequence, token) in packed rows, and which of them are there."""
    at = torch.arange(most, device=device)
    there = at < torch.tensor(lens, device=device)[:, None]
    return torch.where(there, ends[:-1, None].long() + at, 0), there


def _attend(q, k, v, new, lens, causal, window):
    """q [n][queries][heads][dim] over k, v [n][keys][kv heads][dim], padded, one key / value head after the other; a query
    that sees nothing gives zero."""
    dev, group = q.device, q.shape[2] // k.shape[2]
    new, lens = torch.tensor(new, device=dev), torch.tensor(lens, device=dev)
    key = torch.arange(k.shape[1], device=dev)
    place = torch.arange(q.shape[1], device=dev) + (lens - new)[:, None]     # where a query stands among the keys
    seen = (key < lens[:, None])[:, None]
    if causal:
        seen = seen & (key <= place[..., None])
    if window:
        seen = seen & (key > place[..., None] - window)
    out = []
    for h in range(k.shape[2]):
        rows = q[:, :, h * group:(h + 1) * group].float().transpose(1, 2)        # [n][group][queries][dim]
        scores = torch.matmul(rows.flatten(1, 2), k[:, :, h].float().transpose(1, 2).contiguous()).unflatten(1, rows.shape[1:3]) / math.sqrt(q.shape[3])
        scores = scores.masked_fill(~seen[:, None], -math.inf)
        top = scores.amax(-1, keepdim=True)
        p = torch.exp(scores - top.masked_fill(top == -math.inf, 0.0))
        total = p.sum(-1, keepdim=True)
        y = torch.matmul(p.flatten(1, 2), v[:, :, h].float().contiguous()).unflatten(1, rows.shape[1:3])
        out.append((y / total.masked_fill(total == 0, 1.0)).to(q.dtype).transpose(1, 2))
    return torch.cat(out, 2)


def _run_plain(s):
    case = s["case"]
    if case["kind"] in ("rotary", "append"):
        q, k, v = _turn(s["q"], s["positions"], s["table"]), _turn(s["k"], s["positions"], s["table"]), s["v"]
        if case["kind"] == "rotary":
            return {"q": q, "k": k}
        _write(s["cache"], "k", k, s["slots"])
        _write(s["cache"], "v", v, s["slots"])
        return {"q": q, "k": _read(s["cache"], "k", s["slots"]).to(q.dtype), "v": _read(s["cache"], "v", s["slots"]).to(q.dtype)}
    if case["kind"] == "read":
        return {"k": _read(s["cache"], "k", s["slots"]).to(torch.bfloat16), "v": _read(s["cache"], "v", s["slots"]).to(torch.bfloat16)}
    rows, there = _padded(s["ends"], s["new"], max(s["new"]), s["q"].device)
    if case["kind"] == "prompt":
        keys, _ = _padded(s["ends_k"], s["lens"], max(s["lens"]), s["q"].device)
        k, v = s["k"][keys], s["v"][keys]
    else:
        page = case["page"]
        at = torch.arange(max(s["lens"]), device=s["q"].device)
        slots = s["pages"].long()[:, at // page] * page + at % page
        k, v = _read(s["cache"], "k", slots), _read(s["cache"], "v", slots)
    out = _attend(s["q"][rows], k, v, s["new"], s["lens"], case.get("causal", True), case["window"])
    return out[there]


# ---- the framework's calls ----------------------------------------------------------------------------------------------


def _run_own(s):
    from sensenova_u1_amd import PagedKVCache, RotaryTable, paged_attention, prompt_attention, rotary

    case = s["case"]
    if case["kind"] in ("rotary", "append"):
        q, k, v = s["q"], s["k"], s["v"]
        table = RotaryTable(s["table"]["turns"], interleaved=s["table"]["interleaved"], magnitude=s["table"]["magnitude"])
        if case["kind"] == "rotary":
            q, k = rotary(q, k, s["positions"], table)
            return {"q": q, "k": k}
        cache = PagedKVCache(**s["cache"])
        q = cache.write_rotary(q, k, v, s["positions"], table, s["slots"])
        k, v = cache.read(s["slots"])
        return {"q": q, "k": k, "v": v}
    if case["kind"] == "read":
        k, v = PagedKVCache(**s["cache"]).read(s["slots"])
        return {"k": k, "v": v}
    if case["kind"] == "prompt":
        return prompt_attention(s["q"], s["k"], s["v"], s["ends"], s["ends_k"], causal=case["causal"], window=case["window"])
    return paged_attention(s["q"], PagedKVCache(**s["cache"]), s["pages"], s["lens_dev"], s["ends"], max_new=max(s["new"]), window=case["window"])


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------------


def _exact_turn(x, positions, case):
    """Pairs as complex numbers, multiplied by e^(i angle)."""
    case = {"scaling": 0, "interleaved": False, "turned": case["dim"], **case}
    half = case["turned"] // 2
    rate = _turns(case).to(x.device) * 2 * math.pi
    size = 0.1 * math.log(case["scaling"]) + 1 if case["scaling"] else 1.0
    w = torch.polar(torch.full((), size, dtype=torch.float64, device=x.device).expand(len(positions), half).contiguous(), positions.double()[:, None] * rate)
    y = x.double().clone()
    ia = torch.arange(half, device=x.device) * (2 if case["interleaved"] else 1)
    ib = ia + (1 if case["interleaved"] else half)
    z = torch.complex(y[..., ia], y[..., ib]) * w[:, None]
    y[..., ia], y[..., ib] = z.real, z.imag
    return y


def _exact_held(x):
    """What an 8-bit cache holds of bf16 values ``x``, as the numbers that it stands for."""
    runs = x.double().reshape(*x.shape[:-1], -1, 32)
    scale = (runs.abs().max(-1, keepdim=True).values / 127).clamp(max=512).half().double()
    q = torch.nan_to_num(runs / scale).round().clamp(-127, 127)
    return (q * scale).reshape(x.shape)


def exact(case, seed):
    s = prepare(case, seed)
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] in ("rotary", "append"):
        q, k, v = _exact_turn(s["q"], s["positions"], case), _exact_turn(s["k"], s["positions"], case), s["v"]
        if case["kind"] == "rotary":
            return {"q": q, "k": k}
        if case["bits"] == 8:
            return {"q": q, "k": _exact_held(k.to(torch.bfloat16)), "v": _exact_held(v)}
        return {"q": q, "k": k, "v": v.double()}
    if case["kind"] == "read" or case["kind"] == "paged":
        full = {}
        for n in ("k", "v"):
            x = s["cache"][n].double()
            if case["bits"] == 8:
                x = x * s["cache"][n + "_scale"].double().transpose(2, 3).repeat_interleave(32, -1)
            full[n] = x.transpose(1, 2).flatten(0, 1)        # [slot][head][dim]
    if case["kind"] == "read":
        return {n: x[s["slots"]] for n, x in full.items()}
    out, group = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"), heads // kv
    row, first = 0, 0
    for i, (n, length) in enumerate(zip(s["new"], s["lens"])):
        if case["kind"] == "prompt":
            k, v = s["k"][first:first + length].double(), s["v"][first:first + length].double()
            first += length
        else:
            at = torch.arange(length, device="cuda")
            slots = s["pages"][i].long()[at // case["page"]] * case["page"] + at % case["page"]
            k, v = full["k"][slots], full["v"][slots]
        for lo in range(0, n, 2048):
            hi = min(n, lo + 2048)
            last = torch.arange(lo, hi, device="cuda")[:, None] + (length - n)
            key = torch.arange(length, device="cuda")[None]
            hidden = torch.zeros((hi - lo, length), dtype=torch.bool, device="cuda")
            if case.get("causal", True):
                hidden |= key > last
            if case["window"]:
                hidden |= key <= last - case["window"]
            for h in range(heads):
                z = (s["q"][row + lo:row + hi, h].double() @ k[:, h // group].T) * dim ** -0.5
                z[hidden] = -math.inf
                weight = torch.nan_to_num(torch.exp(z - torch.logsumexp(z, -1, keepdim=True)))
                out[row + lo:row + hi, h] = weight @ v[:, h // group]
        row += n
    return out
