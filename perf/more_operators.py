"""What is timed of the operators that stand around the paged cache where many requests are served together: norms of single
heads with the rotation by several positions behind them, the tables of a step, and attention of sequences that begin alike.

Kinds of case

* ``axes``    query and key heads turned by several positions of their token (time, row and column of a picture), or by one
              in the order that a model of several has; with or without the norm of each head in front;
* ``append``  the step between the projections and attention: heads normed and turned, keys and values written to a paged
              cache; then what was written is read back;
* ``tables``  what a step of many requests needs besides their tokens: where each sequence's queries end, its new length, the
              position and the slot of each new token, and pages for those that outgrow theirs;
* ``shared``  attention of new tokens over a paged cache in which groups of sequences begin with the same pages.

A layer of the 8B backbone has 32 query heads and 8 key / value heads of 128 elements; half of a head turns by the place in
the text, a quarter each by the row and the column in a picture, and the two halves have norms of their own.
"""
import math

import torch

own = False

LAYER = {"heads": 32, "kv_heads": 8, "dim": 128}
EPS = 1e-6


def listed():
    return [
        # one token of one sequence behind the model's own norms: latency
        {"name": "axes_1token", "kind": "axes", "tokens": 1, **LAYER, "layout": "parts", "norms": 0, "interleaved": False, "image": False},
        # image tokens of a 2048 x 2048 picture, positions alone
        {"name": "axes_4096image_sections", "kind": "axes", "tokens": 4096, **LAYER, "layout": "sections", "norms": 0, "interleaved": False, "image": True},
        # the same tokens as a layer of the backbone has them: two norms a head, three positions
        {"name": "norm_4096image", "kind": "axes", "tokens": 4096, **LAYER, "layout": "parts", "norms": 2, "interleaved": False, "image": True},
        # batched decode: one new token of each of 24 sequences
        {"name": "norm_append_24tokens_q8", "kind": "append", "tokens": 24, **LAYER, "layout": "parts", "norms": 2, "interleaved": False, "image": False, "page": 16, "bits": 8},
        # a prompt of an odd number of tokens goes into the cache of a model with one norm and one position
        {"name": "norm_append_5003tokens_q8", "kind": "append", "tokens": 5003, **LAYER, "layout": "one", "norms": 1, "interleaved": False, "image": False, "page": 64, "bits": 8},
        # a decode step of 200 requests
        {"name": "tables_200decode", "kind": "tables", "sequences": 200, "least": 1, "most": 1, "far": 4000, "page": 16},
        # prompts of 37 requests come in at once, some of them empty
        {"name": "tables_37prompts", "kind": "tables", "sequences": 37, "least": 0, "most": 3000, "far": 1, "page": 64},
        # two answers to one question: latency
        {"name": "shared_2_of_512_bf16", "kind": "shared", "groups": "2", "shared": "512", "new": 1, "every": 1, "own": 40, "page": 16, "bits": 16, **LAYER},
        # a chat service: 32 sequences behind one long instruction
        {"name": "shared_32_of_8192_q8", "kind": "shared", "groups": "32", "shared": "8192", "new": 1, "every": 1, "own": 900, "page": 32, "bits": 8, **LAYER},
        # many questions about one long document
        {"name": "shared_64_of_16384_bf16", "kind": "shared", "groups": "64", "shared": "16384", "new": 1, "every": 1, "own": 400, "page": 64, "bits": 16, **LAYER},
        # several documents at once, and requests that share nothing
        {"name": "shared_4groups_q8", "kind": "shared", "groups": "12,5,3,9", "shared": "2992,20000,0,640", "new": 1, "every": 1, "own": 700, "page": 16, "bits": 8, **LAYER},
        # the next 256 tokens of two prompts behind a common one, beside four that are being answered
        {"name": "shared_chunks_of_6016_bf16", "kind": "shared", "groups": "6", "shared": "6016", "new": 256, "every": 3, "own": 600, "page": 64, "bits": 16, **LAYER},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kv_heads, group = rng.choice([(8, 4)] * 3 + [(4, 7), (8, 5), (16, 1), (2, 8), (1, 12)])
    shape = {"heads": kv_heads * group, "kv_heads": kv_heads, "dim": rng.choice([128] * 3 + [64, 96, 256])}
    kind = rng.choice(["axes", "append", "tables", "shared", "shared"])
    bits, page = rng.choice([8, 8, 16]), rng.choice([16, 32, 64, 128])
    if kind in ("axes", "append"):
        image = rng.random() < 0.4
        layout = rng.choice(["parts", "sections"]) if image else rng.choice(["parts", "sections", "one"])
        norms = rng.choice([0, 1, 2] if layout != "one" else [1, 2])
        case = {"kind": kind, "tokens": _log_int(rng, 1, 8192 if kind == "axes" else 5000), **shape, "layout": layout, "norms": norms,
                "interleaved": rng.random() < 0.3, "image": image}
        return case if kind == "axes" else {**case, "page": page, "bits": bits}
    if kind == "tables":
        decode = rng.random() < 0.5
        sequences = _log_int(rng, 1, 1000 if decode else 60)
        return {"kind": kind, "sequences": sequences, "least": rng.choice([0, 1]), "most": rng.choice([1, 1, 4]) if decode else _log_int(rng, 8, 4000),
                "far": _log_int(rng, 1, 8000), "page": page}
    count = rng.choice([1, 1, 1, 2, 4])
    groups = [_log_int(rng, 1, 64 // count) for _ in range(count)]
    new = rng.choice([1, 1, 1, 2, 5, _log_int(rng, 2, 256)])
    # together no more keys a sequence and no more new tokens than the listed ones have
    most = (min(16384, 1000000 // sum(groups)) if new < 9 else min(6000, 100000 // sum(groups))) * 1024 // max(1024, kv_heads * shape["dim"])
    shared = [rng.choice([1, 1, 1, 0]) * (_log_int(rng, page, most) // page) * page for _ in groups]
    return {"kind": kind, "groups": ",".join(map(str, groups)), "shared": ",".join(map(str, shared)), "new": new, "every": 1 if new < 9 else rng.choice([2, 3, 5]),
            "own": max(_log_int(rng, 8, 1000), 2 * new), "page": page, "bits": bits, **shape}


def _ints(text):
    return [int(t) for t in text.split(",")]


def _sequences(case):
    """Of each sequence of a ``shared`` case: (tokens that its group has in common, tokens in all, new ones)."""
    out = []
    for count, shared in zip(_ints(case["groups"]), _ints(case["shared"])):
        for _ in range(count):
            i = len(out)
            new = case["new"] if i % case["every"] == 0 else 1
            out.append((shared, shared + max(new, 1 + case["own"] * ((7 * i + 3) % 16) // 16), new))
    return out


def work(case):
    if case["kind"] == "tables":
        new = case["sequences"] * (case["least"] + case["most"]) // 2
        pages = case["sequences"] + new // case["page"]
        return {"bytes": 16 * case["sequences"] + 16 * new + 8 * pages, "flops": 10 * (case["sequences"] + new)}
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    element = 2 if case.get("bits", 16) == 16 else 1 + 2 / 32
    if case["kind"] == "axes":
        values = case["tokens"] * (heads + kv) * dim
        return {"bytes": 4 * values, "flops": (3 + 4 * (case["norms"] > 0)) * values}
    if case["kind"] == "append":
        t = case["tokens"]
        return {"bytes": t * dim * (4 * heads + 4 * kv + 2 * kv * (2 * element + 2)), "flops": t * dim * (7 * heads + 14 * kv)}
    of = _sequences(case)
    keys = sum(_ints(case["shared"])) + sum(length - shared for shared, length, _ in of)
    pairs = sum(n * length - n * (n - 1) // 2 for _, length, n in of)
    return {"bytes": 4 * sum(n for *_, n in of) * heads * dim + 2 * keys * kv * dim * element, "flops": 4 * pairs * heads * dim}


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


def _layout(case):
    """(turns of 2 pi a position of each pair in 64 bits, which position turns it, elements of each part of a head).

    ``parts``: a half and two quarters of a head, each with wavelengths and a position of its own, pairs within each;
    ``sections``: pairs over the whole head, one row of wavelengths, a quarter of the pairs by the first position and the rest
    by the two others in turn; ``one``: one position for all."""
    dim, layout = case["dim"], case["layout"]
    half = dim // 2

    def rates(pairs, base):
        return base ** (-torch.arange(pairs, dtype=torch.float64) / pairs) / (2 * math.pi)

    if layout == "parts":
        a, b = half // 2, half // 4
        axis = torch.tensor([0] * a + [1] * b + [2] * b, dtype=torch.int32)
        return torch.cat([rates(a, 5000000.0), rates(b, 10000.0), rates(b, 10000.0)]), axis, [dim // 2, dim // 4, dim // 4]
    pair = torch.arange(half)
    axis = torch.where(pair < half // 4, 0, 1 + pair % 2) if layout == "sections" else torch.zeros_like(pair)
    return rates(half, 1000000.0), axis.to(torch.int32), [dim]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    if case["kind"] == "tables":
        count, page = case["sequences"], case["page"]
        s["lens"] = torch.randint(0, case["far"], (count,), generator=gen, device="cuda", dtype=torch.int32)
        s["new"] = torch.randint(case["least"], case["most"] + 1, (count,), generator=gen, device="cuda", dtype=torch.int32)
        width = -(-(case["far"] + case["most"]) // page)
        s["tokens"] = count * case["most"]                     # what the program makes room for
        # pages in the order in which they came back from sequences that are gone
        order = torch.randperm(count * width, generator=gen, device="cuda").to(torch.int32)
        s["pages"] = torch.full((count, width), -1, dtype=torch.int32, device="cuda")
        has = torch.arange(width, device="cuda") < (-(-s["lens"] // page))[:, None]
        taken = int(has.sum())
        s["pages"][has] = order[:taken]
        s["free"] = order.roll(7)                               # a ring, in use from some place on
        s["cursor"] = torch.tensor([taken + 7, 7 + count * width], dtype=torch.int64, device="cuda")
        return s
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] in ("axes", "append"):
        t = case["tokens"]
        # one projection's output holds q, k and v of a token next to each other
        qkv = torch.cat([_heads(gen, t, heads, dim), _heads(gen, t, kv, dim, wide=True), _heads(gen, t, kv, dim)], 1)
        s["q"], s["k"], s["v"] = qkv.split([heads, kv, kv], 1)
        turns, axis, s["parts"] = _layout(case)
        s["turns"], s["axis"] = turns.cuda(), axis.cuda()
        start = int(torch.randint(0, 40000, (1,), generator=gen, device="cuda"))
        at = torch.arange(t, device="cuda")
        if case["layout"] == "one":
            s["positions"] = start + at
        elif case["image"]:
            # a picture behind a text: its tokens share the place in the text
            side = math.isqrt(t - 1) + 1
            s["positions"] = torch.stack([torch.full_like(at, start), at // side, at % side])
        else:
            s["positions"] = torch.stack([start + at, torch.zeros_like(at), torch.zeros_like(at)])
        widths = [dim // max(case["norms"], 1)] * case["norms"]
        s["q_weights"], s["k_weights"] = ([(1 + 0.3 * torch.randn(w, generator=gen, device="cuda")).to(torch.bfloat16) for w in widths] for _ in range(2))
    if case["kind"] == "append":
        page = case["page"]
        pages = -(-t // page) + 7
        s["cache"] = _empty_cache(case, pages)
        order = torch.randperm(pages, generator=gen, device="cuda")
        s["slots"] = order[at // page] * page + at % page
    if case["kind"] == "shared":
        of, page = _sequences(case), case["page"]
        lens, new = [x[1] for x in of], [x[2] for x in of]
        width = -(-max(lens) // page)
        s["pages"] = torch.zeros((len(of), width), dtype=torch.int32, device="cuda")
        total = sum(_ints(case["shared"])) // page + sum(-(-(length - shared) // page) for shared, length, _ in of)
        order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
        at = i = 0
        for count, shared in zip(_ints(case["groups"]), _ints(case["shared"])):
            common = order[at:at + shared // page]
            at += shared // page
            for _ in range(count):
                mine = -(-(lens[i] - shared) // page)
                s["pages"][i, :shared // page + mine] = torch.cat([common, order[at:at + mine]])
                at += mine
                i += 1
        s["cache"] = _empty_cache(case, total)
        slots = torch.arange(total * page, device="cuda")
        _write(s["cache"], "k", _heads(gen, len(slots), kv, dim, wide=True), slots)
        _write(s["cache"], "v", _heads(gen, len(slots), kv, dim), slots)
        s["q"] = _heads(gen, sum(new), heads, dim)
        s["lens"], s["new"] = lens, new
        s["lens_dev"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        s["ends"] = torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32)
        s["groups"] = torch.tensor([0] + _ints(case["groups"]), device="cuda").cumsum(0).to(torch.int32)
        s["shared"] = torch.tensor(_ints(case["shared"]), dtype=torch.int32, device="cuda")
    return s


# ---- the operators in plain form ------------------------------------------------------------------------------------


def _normed(x, weights):
    """x [T][heads][dim] in 32 bits, each part of a head divided by its root of the mean square and scaled by its weights."""
    x = x.float()
    if not weights:
        return x
    parts = x.unflatten(-1, (len(weights), -1))
    parts = parts * torch.rsqrt(parts.square().mean(-1, keepdim=True) + EPS)
    return (parts * torch.stack(weights).float()).flatten(-2)


def _turned(x, s):
    """x [T][heads][dim] in 32 bits turned by the positions: angles in 64 bits, cosines and sines rounded to 32."""
    positions = s["positions"] if s["positions"].dim() == 2 else s["positions"][None]
    turns = positions.double()[s["axis"].long()].T * s["turns"]
    angle = 2 * math.pi * (turns - turns.round())
    c, r = angle.cos().float()[:, None], angle.sin().float()[:, None]
    element = torch.arange(x.shape[-1], device=x.device)
    if s["case"]["interleaved"]:
        ia, ib = element[0::2], element[1::2]
    else:
        halves = [part.chunk(2) for part in element.split(s["parts"])]
        ia, ib = (torch.cat(side) for side in zip(*halves))
    a, b = x[..., ia], x[..., ib]
    y = torch.empty_like(x)
    y[..., ia], y[..., ib] = a * c - b * r, b * c + a * r
    return y


def _plain_tables(s):
    page, width = s["case"]["page"], s["pages"].shape[1]
    lens, count = s["lens"].long(), s["lens"].shape[0]
    ends = torch.cat([s["new"].new_zeros(1), s["new"]]).long().cumsum(0).clamp(max=s["tokens"])
    new = ends.diff()
    has = -(-lens // page)
    wants = -(-(lens + new).clamp(max=width * page) // page) - has
    before = wants.cumsum(0) - wants
    there = s["cursor"][1] - s["cursor"][0]
    gets = torch.minimum(wants, (there - before).clamp(min=0))
    after = torch.minimum(lens + new, (has + gets) * page)
    column = torch.arange(width, device=lens.device) - has[:, None]
    fresh = (column >= 0) & (column < gets[:, None])
    ring = (s["cursor"][0] + before[:, None] + column) % s["free"].shape[0]
    pages = torch.where(fresh, s["free"][ring], s["pages"])
    row = torch.arange(s["tokens"], device=lens.device)
    of = torch.searchsorted(ends[1:].contiguous(), row, right=True)
    there = of < count
    of = of.clamp(max=count - 1)
    position = lens[of] + row - ends[of]
    slot = pages[of, (position // page).clamp(max=width - 1)].long() * page + position % page
    cursor = torch.stack([s["cursor"][0] + gets.sum(), s["cursor"][1]])
    return {"ends": ends.int(), "lens": after.int(), "positions": torch.where(there, position, 0), "slots": torch.where(there & (position < after[of]), slot, -1),
            "pages": pages, "cursor": cursor, "missing": (lens + new - after).sum().int().reshape(1)}


def _plain_attention(s):
    """Every sequence by itself, in one batch: [sequence][kv head][query, head of the group][...]."""
    q, dev = s["q"], s["q"].device
    kv, page = s["case"]["kv_heads"], s["case"]["page"]
    new, lens = torch.tensor(s["new"], device=dev), s["lens_dev"].long()
    query = torch.arange(max(s["new"]), device=dev)
    there = query < new[:, None]
    rows = torch.where(there, s["ends"][:-1, None].long() + query, 0)
    key = torch.arange(max(s["lens"]), device=dev)
    slots = s["pages"].long()[:, key // page] * page + key % page
    k, v = (_read(s["cache"], n, slots).transpose(1, 2) for n in ("k", "v"))
    x = q[rows].float().unflatten(2, (kv, -1)).transpose(1, 2)                 # [n][kv][query][group][dim]
    scores = torch.matmul(x.flatten(2, 3), k.transpose(2, 3).contiguous()) / math.sqrt(q.shape[2])
    del k
    scores = scores.unflatten(2, x.shape[2:4])
    seen = key <= (query + (lens - new)[:, None])[..., None]                   # a query stands at one of the last places
    scores.masked_fill_(~seen[:, None, :, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    del scores
    total = p.sum(-1, keepdim=True)
    y = torch.matmul(p.flatten(2, 3), v.contiguous()).unflatten(2, x.shape[2:4]) / total
    return y.transpose(1, 2).flatten(2, 3)[there].to(q.dtype)


def _run_plain(s):
    kind = s["case"]["kind"]
    if kind == "tables":
        return _plain_tables(s)
    if kind == "shared":
        return _plain_attention(s)
    q = _turned(_normed(s["q"], s["q_weights"]), s).to(s["q"].dtype)
    k = _turned(_normed(s["k"], s["k_weights"]), s).to(s["k"].dtype)
    if kind == "axes":
        return {"q": q, "k": k}
    _write(s["cache"], "k", k, s["slots"])
    _write(s["cache"], "v", s["v"], s["slots"])
    return {"q": q, "k": _read(s["cache"], "k", s["slots"]).to(q.dtype), "v": _read(s["cache"], "v", s["slots"]).to(q.dtype)}


# ---- the framework's calls ----------------------------------------------------------------------------------------------


def _run_own(s):
    from sensenova_u1_amd import HeadNorm, PagedKVCache, PageTables, RotaryAxes, RotaryTable, rotary, shared_prefix_attention

    case = s["case"]
    if case["kind"] == "tables":
        tables = PageTables(s["pages"], s["lens"], s["free"], s["cursor"], page_size=case["page"])
        step = tables.append(s["new"], s["tokens"], inplace=False)
        return {"ends": step.ends, "lens": step.lens, "positions": step.positions, "slots": step.slots, "pages": tables.pages, "cursor": step.cursor, "missing": step.missing}
    if case["kind"] == "shared":
        return shared_prefix_attention(s["q"], PagedKVCache(**s["cache"]), s["pages"], s["lens_dev"], s["groups"], s["shared"], s["ends"], max_new=max(s["new"]))
    if case["layout"] == "one":
        table = RotaryTable(s["turns"], interleaved=case["interleaved"])
    else:
        table = RotaryAxes(s["turns"], s["axis"], parts=s["parts"], interleaved=case["interleaved"])
    norms = {}
    if case["norms"]:
        norms = {"q_norm": HeadNorm(*s["q_weights"], eps=EPS), "k_norm": HeadNorm(*s["k_weights"], eps=EPS)}
    if case["kind"] == "axes":
        q, k = rotary(s["q"], s["k"], s["positions"], table, **norms)
        return {"q": q, "k": k}
    cache = PagedKVCache(**s["cache"])
    q = cache.write_rotary(s["q"], s["k"], s["v"], s["positions"], table, s["slots"], **norms)
    k, v = cache.read(s["slots"])
    return {"q": q, "k": k, "v": v}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------------


def _exact_head(x, weights, s):
    """Pairs as complex numbers, multiplied by e^(i angle), behind the norm."""
    y = x.double()
    lo = 0
    for w in weights:
        part = y[..., lo:lo + len(w)]
        y[..., lo:lo + len(w)] = w.double() * part / (part.pow(2).sum(-1, keepdim=True) / len(w) + EPS).sqrt()
        lo += len(w)
    positions = s["positions"].double().reshape(-1, x.shape[0])
    ia, ib, lo = [], [], 0
    for n in s["parts"]:
        for i in range(n // 2):
            ia.append(lo + (2 * i if s["case"]["interleaved"] else i))
            ib.append(lo + (2 * i + 1 if s["case"]["interleaved"] else i + n // 2))
        lo += n
    for i, (a, b) in enumerate(zip(ia, ib)):
        angle = positions[int(s["axis"][i])] * (s["turns"][i] * 2 * math.pi)
        z = torch.complex(y[..., a], y[..., b]) * torch.polar(torch.ones_like(angle), angle)[:, None]
        y[..., a], y[..., b] = z.real, z.imag
    return y


def _exact_held(x):
    """What an 8-bit cache holds of bf16 values ``x``, as the numbers that it stands for."""
    runs = x.double().reshape(*x.shape[:-1], -1, 32)
    scale = (runs.abs().max(-1, keepdim=True).values / 127).clamp(max=512).half().double()
    q = torch.nan_to_num(runs / scale).round().clamp(-127, 127)
    return (q * scale).reshape(x.shape)


def _exact_tables(s):
    """One sequence after the other, as a program on the host would do it; whole numbers, compared as such."""
    page, width = s["case"]["page"], s["pages"].shape[1]
    pages, free = s["pages"].tolist(), s["free"].tolist()
    taken, given = s["cursor"].tolist()
    ends, lens, positions, slots, missing = [0], [], [], [], 0
    for i, (length, new) in enumerate(zip(s["lens"].tolist(), s["new"].tolist())):
        new = min(new, s["tokens"] - ends[-1])
        ends.append(ends[-1] + new)
        for position in range(length, length + new):
            if position % page == 0 and position < width * page and taken < given:
                pages[i][position // page] = free[taken % len(free)]
                taken += 1
            positions.append(position)
            there = position < width * page and pages[i][position // page] >= 0
            slots.append(pages[i][position // page] * page + position % page if there else -1)
            missing += not there
        lens.append(length + sum(x >= 0 for x in slots[ends[-2]:ends[-1]]))
    rest = s["tokens"] - len(slots)
    whole = {"ends": ends, "lens": lens, "positions": positions + [0] * rest, "slots": slots + [-1] * rest, "pages": pages, "cursor": [taken, given], "missing": [missing]}
    kinds = {"positions": torch.int64, "slots": torch.int64, "cursor": torch.int64}
    return {n: torch.tensor(x, dtype=kinds.get(n, torch.int32)) for n, x in whole.items()}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "tables":
        return _exact_tables(s)
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] in ("axes", "append"):
        q, k = _exact_head(s["q"], s["q_weights"], s), _exact_head(s["k"], s["k_weights"], s)
        if case["kind"] == "axes":
            return {"q": q, "k": k}
        if case["bits"] == 8:
            return {"q": q, "k": _exact_held(k.to(torch.bfloat16)), "v": _exact_held(s["v"])}
        return {"q": q, "k": k, "v": s["v"].double()}
    full = {}
    for n in ("k", "v"):
        x = s["cache"][n].double()
        if case["bits"] == 8:
            x = x * s["cache"][n + "_scale"].double().transpose(2, 3).repeat_interleave(32, -1)
        full[n] = x.transpose(1, 2).flatten(0, 1)        # [slot][head][dim]
    out, row = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    for i, (n, length) in enumerate(zip(s["new"], s["lens"])):
        at = torch.arange(length, device="cuda")
        slots = s["pages"][i].long()[at // case["page"]] * case["page"] + at % case["page"]
        hidden = at > torch.arange(length - n, length, device="cuda")[:, None]
        for h in range(heads):
            z = (s["q"][row:row + n, h].double() @ full["k"][slots, h * kv // heads].T) * dim ** -0.5
            z[hidden] = -math.inf
            out[row:row + n, h] = torch.softmax(z, -1) @ full["v"][slots, h * kv // heads]
        row += n
    return out
