"""Cases, plain forms and exact values of the paged key/value cache's operators.

Four operators, one cache: ``rotary`` (positions with several axes, forward and backward), ``append``
(rotate and store new rows), ``attend`` (one new token per sequence over its pages, with the attention
weight every row receives) and ``evict`` (keep the rows with the largest accumulated weight).

The cache is ``keys`` / ``values`` [pages, page_size, heads, width] (any strides) and ``weights``
[pages, heads, page_size] in fp32; a sequence is a row of ``page_table`` (int32 page ids) and a length.
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4, "e4m3": 1}
_E4M3_MAX = 448.0


# ---- cases ---------------------------------------------------------------------------------------
def _rotary(name, tokens, q_heads, kv_heads, width, pairs, axes, interleaved, dtype, far):
    return dict(op="rotary", name=name, tokens=tokens, q_heads=q_heads, kv_heads=kv_heads, width=width, pairs=pairs,
                axes=axes, interleaved=interleaved, dtype=dtype, far=far)


def _append(name, sequences, longest, shortest, q_heads, kv_heads, width, pairs, axes, interleaved, dtype, cache, page,
            held, layout):
    return dict(op="append", name=name, sequences=sequences, longest=longest, shortest=shortest, q_heads=q_heads,
                kv_heads=kv_heads, width=width, pairs=pairs, axes=axes, interleaved=interleaved, dtype=dtype,
                cache=cache, page=page, held=held, layout=layout)


def _attend(name, sequences, longest, shortest, q_heads, kv_heads, width, dtype, cache, page, layout):
    return dict(op="attend", name=name, sequences=sequences, longest=longest, shortest=shortest, q_heads=q_heads,
                kv_heads=kv_heads, width=width, dtype=dtype, cache=cache, page=page, layout=layout)


def _evict(name, sequences, longest, shortest, kv_heads, width, cache, page, layout, budget, sinks, recent):
    return dict(op="evict", name=name, sequences=sequences, longest=longest, shortest=shortest, kv_heads=kv_heads,
                width=width, cache=cache, page=page, layout=layout, budget=budget, sinks=sinks, recent=recent)


def listed():
    return [
        # a training step over packed image-and-text sequences: queries and keys turned, gradients turned back
        _rotary("rotary train 3 axes", 16384, 32, 8, 128, 64, 3, False, "bf16", 20000),
        # an image encoder's patches (height, width), odd count, fp32
        _rotary("rotary patches fp32", 1023, 16, 16, 80, 40, 2, True, "f32", 96),
        # the smallest call of a decode step: one token each for a few sequences
        _append("append one token", 4, 1, 1, 32, 8, 128, 64, 1, False, "bf16", "bf16", 16, 5000, "head"),
        # a batch of prompts with images goes in, the cache in eight bits
        _append("append prompts e4m3", 6, 4096, 37, 32, 8, 128, 64, 3, False, "bf16", "e4m3", 64, 900, "head"),
        # one short sequence: latency
        _attend("attend one short", 1, 777, 777, 32, 8, 128, "bf16", "bf16", 16, "head"),
        # a batch being served, lengths mixed
        _attend("attend batch ragged", 64, 6000, 300, 32, 8, 128, "bf16", "bf16", 16, "head"),
        # one long document: the split over the length and its join
        _attend("attend one long", 1, 131072, 131072, 64, 8, 128, "f16", "f16", 32, "head"),
        # a large batch over eight-bit rows
        _attend("attend large e4m3", 128, 12000, 4000, 32, 4, 128, "bf16", "e4m3", 64, "head"),
        # as many key heads as query heads, odd width and page, heads side by side in memory, an empty sequence
        _attend("attend odd own heads", 9, 1531, 0, 20, 20, 80, "f16", "f16", 7, "slot"),
        # prompts pressed to a budget after their prefill
        _evict("evict prompts", 4, 32768, 20000, 8, 128, "bf16", 16, "head", 8192, 4, 512),
        # the periodic trim of a decoding batch
        _evict("evict trim e4m3", 16, 1100, 1000, 8, 128, "e4m3", 16, "head", 1024, 4, 128),
        # one long document pressed to an eighth, odd sizes
        _evict("evict one long", 1, 131071, 131071, 4, 80, "f16", 24, "slot", 16001, 1, 1000),
    ]


def _between(rng, low, high):
    """A whole number in [low, high], spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(max(low, 1)), math.log(high)))))))


def draw(rng):
    op = rng.choice(["rotary", "append", "attend", "attend", "evict"])
    kv_heads = rng.choice([1, 2, 4, 5, 8, 16])
    group = rng.choice([1, 1, 2, 3, 4, 7, 8, 16])
    width = rng.choice([32, 64, 80, 96, 128, 128, 192, 256])
    axes = rng.choice([1, 2, 3, 4])
    pairs = rng.choice([width // 2, width // 2, width // 4])
    interleaved = rng.random() < 0.5
    if op == "rotary":
        heads = kv_heads * group
        most = max(2, 80_000_000 // ((heads + kv_heads) * width))
        return _drawn(_rotary("", _between(rng, 1, min(16384, most)), heads, kv_heads, width, pairs, axes, interleaved,
                              rng.choice(["bf16", "f16", "f32"]), rng.choice([100, 5000, 1_000_000])))
    dtype = rng.choice(["bf16", "f16"])
    cache = rng.choice([dtype, dtype, "e4m3"])
    page = rng.choice([1, 8, 16, 16, 24, 32, 64, 100, 128])
    layout = rng.choice(["head", "slot"])
    if op == "append":
        heads = kv_heads * group
        sequences = _between(rng, 1, 128)
        most = max(1, 60_000_000 // ((heads + 2 * kv_heads) * width * sequences))
        longest = 1 if rng.random() < 0.4 else _between(rng, 1, min(4096, most))
        return _drawn(_append("", sequences, longest, rng.choice([longest, max(0, longest // 3), 0]), heads, kv_heads,
                              width, pairs, axes, interleaved, dtype, cache, page, _between(rng, 1, 1500), layout))
    if op == "attend":
        sequences = _between(rng, 1, 128)
        most = min(131072, 250_000_000 // (sequences * kv_heads * width), 100_000_000 // (sequences * kv_heads * group))
        longest = _between(rng, 1, max(2, most))
        return _drawn(_attend("", sequences, longest, rng.choice([longest, longest // 2, 0]), kv_heads * group, kv_heads,
                              width, dtype, cache, page, layout))
    sequences = _between(rng, 1, 32)
    longest = _between(rng, 2, max(3, min(131072, 150_000_000 // (sequences * kv_heads * width))))
    budget = _between(rng, 1, max(2, int(longest * rng.uniform(0.1, 1.1))))
    sinks = min(budget, rng.choice([0, 1, 4]))
    return _drawn(_evict("", sequences, longest, rng.choice([longest, longest // 2, 0]), kv_heads, width, cache, page,
                         layout, budget, sinks, min(budget - sinks, rng.choice([0, 1, budget // 8]))))


def _drawn(case):
    del case["name"]
    return case


def _lengths(low, high, n):
    """n lengths spread over [low, high], the same for every seed; both ends are there where n allows."""
    if n == 1 or low == high:
        return [high] * n
    r = np.random.RandomState(n * 7 + high)
    inside = r.randint(low, high + 1, size=n).tolist()
    inside[0], inside[n // 2] = high, low
    return inside


def _held(case):
    """Rows the sequences hold before the call."""
    if case["op"] == "append":
        return _lengths(case["held"] // 2, case["held"], case["sequences"])
    return _lengths(case["shortest"], case["longest"], case["sequences"])


def _new(case):
    """Rows an append brings, per sequence."""
    return _lengths(case["shortest"], case["longest"], case["sequences"])


# ---- what a program has in hand ------------------------------------------------------------------
def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(_TYPES[dtype])


def _plan(case):
    """Frequencies and the axis of each pair: sections of the axes in turn, as models with several axes have them."""
    i = np.arange(case["pairs"], dtype=np.float64)
    freq = torch.tensor((10000.0 ** (-i / case["pairs"])).astype(np.float32), device="cuda")
    axis = np.minimum(np.arange(case["pairs"]) * case["axes"] // case["pairs"], case["axes"] - 1)
    return freq, torch.tensor(axis.astype(np.int32), device="cuda")


def _pool(g, case, pages):
    """keys and values [pages, page, heads, width]; "head": a page holds its rows head by head in memory."""
    h, p, d, c = case["kv_heads"], case["page"], case["width"], case["cache"]

    def rows():
        shape = (pages, h, p, d) if case["layout"] == "head" else (pages, p, h, d)
        if c == "e4m3":
            t = torch.empty(shape, device="cuda", dtype=torch.float8_e4m3fn)
            for i in range(0, pages, 4096):     # keeps the fp32 draft small
                t[i:i + 4096] = (torch.randn(t[i:i + 4096].shape, generator=g, device="cuda") * 8.0).to(t.dtype)
        else:
            t = torch.empty(shape, device="cuda", dtype=_TYPES[c]).normal_(generator=g)
        return t.permute(0, 2, 1, 3) if case["layout"] == "head" else t

    return rows(), rows()


def _tables(g, counts, page, spare=0):
    """Page tables of sequences that hold `counts` rows, the pages in shuffled order; `spare` unused pages remain."""
    need = [-(-c // page) for c in counts]
    total = sum(need)
    order = torch.randperm(total + spare, generator=g, device="cuda").to(torch.int32)
    wide = max(1, max(need))
    first = np.concatenate([[0], np.cumsum(need)[:-1]])
    at = torch.tensor(first, device="cuda")[:, None] + torch.arange(wide, device="cuda")[None]
    here = torch.arange(wide, device="cuda")[None] < torch.tensor(need, device="cuda")[:, None]
    table = torch.where(here, order[at.clamp(max=total + spare - 1)], torch.full_like(order[:1], -1))
    return table.contiguous(), order[total:], total + spare


class _State:
    """What `run` takes: plain attributes."""


def prepare(case, seed):
    s = _State()
    s.case = case
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    op = case["op"]
    if op in ("rotary", "append"):
        s.freq, s.axis = _plan(case)
        tokens = case["tokens"] if op == "rotary" else sum(_new(case))
        far = case["far"] if op == "rotary" else 100_000
        s.positions = torch.randint(0, far, (case["axes"], tokens), generator=g, device="cuda", dtype=torch.int32)
        s.q = _normal(g, (tokens, case["q_heads"], case["width"]), case["dtype"])
        s.k = _normal(g, (tokens, case["kv_heads"], case["width"]), case["dtype"])
    if op == "rotary":
        s.gq = _normal(g, s.q.shape, case["dtype"], 0.1)
        s.gk = _normal(g, s.k.shape, case["dtype"], 0.1)
        if own:
            from nv_embedding_cache_b200 import kv_cache
            s.rotary = kv_cache.RotaryPlan(s.freq, s.axis, case["axes"], interleaved=case["interleaved"])
        s.q.requires_grad_()
        s.k.requires_grad_()
        return s
    held = _held(case)
    s.lengths = torch.tensor(held, dtype=torch.int32, device="cuda")
    h, page = case["kv_heads"], case["page"]
    s.k_scale = s.v_scale = None
    if case["cache"] == "e4m3":
        s.k_scale = torch.rand(h, generator=g, device="cuda") * 0.02 + 0.01
        s.v_scale = torch.rand(h, generator=g, device="cuda") * 0.02 + 0.01
    if op == "append":
        new = _new(case)
        s.v = _normal(g, s.k.shape, case["dtype"])
        s.offsets = torch.tensor(np.concatenate([[0], np.cumsum(new)]).astype(np.int32), device="cuda")
        s.page_table, _, pages = _tables(g, [a + b for a, b in zip(held, new)], page, 3)
    elif op == "attend":
        s.q = _normal(g, (case["sequences"], case["q_heads"], case["width"]), case["dtype"])
        s.scale = 1.0 / math.sqrt(case["width"])
        s.page_table, _, pages = _tables(g, held, page, 3)
        s.longest = max(held)
    else:
        kept = [min(n, case["budget"]) for n in held]
        more = [-(-k // page) for k in kept]
        s.page_table, spare, pages = _tables(g, held, page, sum(more) + 3)
        first = np.concatenate([[0], np.cumsum(more)[:-1]])
        wide = max(1, max(more))
        at = torch.tensor(first, device="cuda")[:, None] + torch.arange(wide, device="cuda")[None]
        here = torch.arange(wide, device="cuda")[None] < torch.tensor(more, device="cuda")[:, None]
        s.new_table = torch.where(here, spare[at.clamp(max=spare.numel() - 1)], torch.full_like(spare[:1], -1)).contiguous()
        s.longest = max(held)
    s.keys, s.values = _pool(g, case, pages)
    # what decoding leaves behind: most rows drew little weight, a few a lot; equal ones (never drew any) among them
    w = torch.rand((pages, h, page), generator=g, device="cuda")
    s.weights = torch.where(w < 0.2, torch.zeros_like(w), w.pow(6) * (8.0 / max(1, max(held))))
    if own:
        from nv_embedding_cache_b200 import kv_cache
        s.cache = kv_cache.PagedKVCache(s.keys, s.values, s.weights, key_scale=s.k_scale, value_scale=s.v_scale)
        if op == "append":
            s.rotary = kv_cache.RotaryPlan(s.freq, s.axis, case["axes"], interleaved=case["interleaved"])
    return s


# ---- one pass ------------------------------------------------------------------------------------
def run(s):
    return {"rotary": _run_rotary, "append": _run_append, "attend": _run_attend, "evict": _run_evict}[s.case["op"]](s)


def _run_rotary(s):
    if own:
        from nv_embedding_cache_b200 import kv_cache
        q, k = kv_cache.rotary(s.q, s.k, s.positions, s.rotary)
    else:
        q, k = _turn(s.q.float(), s).to(s.q.dtype), _turn(s.k.float(), s).to(s.k.dtype)
    gq, gk = torch.autograd.grad((q, k), (s.q, s.k), (s.gq, s.gk))
    return {"q": q.detach(), "k": k.detach(), "gq": gq, "gk": gk}


def _run_append(s):
    if own:
        q, lengths = s.cache.append(s.k, s.v, s.page_table, s.lengths, q=s.q, offsets=s.offsets, positions=s.positions,
                                    rotary=s.rotary)
        return {"q": q, "lengths": lengths, "keys": s.keys, "values": s.values, "weights": s.weights}
    k, v = _turn(s.k.float(), s), s.v.float()
    if s.k_scale is not None:
        k = (k / s.k_scale[:, None]).clamp(-_E4M3_MAX, _E4M3_MAX)
        v = (v / s.v_scale[:, None]).clamp(-_E4M3_MAX, _E4M3_MAX)
    token = torch.arange(s.k.shape[0], device="cuda")
    b = torch.searchsorted(s.offsets[1:].contiguous(), token, right=True)
    row = s.lengths[b].long() + token - s.offsets[b].long()
    page, slot = s.page_table[b, row // s.case["page"]].long(), row % s.case["page"]
    _bits(s.keys)[page, slot] = _bits(k.to(s.keys.dtype))
    _bits(s.values)[page, slot] = _bits(v.to(s.values.dtype))
    s.weights[page, :, slot] = 0.0
    return {"q": _turn(s.q.float(), s).to(s.q.dtype), "lengths": s.lengths + (s.offsets[1:] - s.offsets[:-1]),
            "keys": s.keys, "values": s.values, "weights": s.weights}


def _run_attend(s):
    if own:
        out, lse = s.cache.attend(s.q, s.page_table, s.lengths, scale=s.scale, max_length=s.longest,
                                  accumulate_weights=True, return_lse=True)
        return {"out": out, "lse": lse, "weights": s.weights}
    n, heads, d = s.q.shape
    h = s.keys.shape[2]
    row = torch.arange(s.longest, device="cuda")
    page = s.page_table[:, row // s.case["page"]].long().clamp(min=0)
    slot = (row % s.case["page"])[None].expand_as(page)
    here = row[None] < s.lengths[:, None]
    k, v = (_bits(t)[page, slot].view(t.dtype).float().masked_fill(~here[:, :, None, None], 0.0)
            for t in (s.keys, s.values))
    q = s.q.float().view(n, h, heads // h, d)
    if s.k_scale is not None:
        k, v = k * s.k_scale[:, None], v * s.v_scale[:, None]
    x = torch.matmul(q, k.permute(0, 2, 3, 1)) * s.scale
    x = x.masked_fill(~here[:, None, None], -math.inf)
    top = x.amax(dim=-1, keepdim=True)
    e = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(dim=-1, keepdim=True)
    p = e / torch.where(total == 0, torch.ones_like(total), total)
    out = torch.matmul(p, v.permute(0, 2, 1, 3)).reshape(n, heads, d).to(s.q.dtype)
    b, at = torch.nonzero(here, as_tuple=True)
    s.weights[page[b, at], :, slot[b, at]] += p.sum(dim=2)[b, :, at]
    return {"out": out, "lse": (top + torch.log(total)).reshape(n, heads), "weights": s.weights}


def _run_evict(s):
    c = s.case
    if own:
        kept, lengths = s.cache.evict(s.page_table, s.lengths, s.new_table, c["budget"], sinks=c["sinks"],
                                      recent=c["recent"], max_length=s.longest)
        return {"kept": kept, "lengths": lengths, "keys": s.keys, "values": s.values, "weights": s.weights}
    h, size = s.keys.shape[2], c["page"]
    row = torch.arange(s.longest, device="cuda")
    page = s.page_table[:, row // size].long().clamp(min=0)
    slot = (row % size)[None].expand_as(page)
    here = row[None] < s.lengths[:, None]
    w = s.weights[page, :, slot].permute(0, 2, 1)
    must = (row[None] < c["sinks"]) | (row[None] >= s.lengths[:, None] - c["recent"])
    worth = w.nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf)
    # those that must stay first, then by weight, the rest of the padding last; equal ones stay in order
    by_weight = torch.sort(worth, dim=-1, descending=True, stable=True).indices
    group = torch.where(here, torch.where(must, 0, 1), 2)[:, None].expand(-1, h, -1)
    order = by_weight.gather(2, torch.sort(group.gather(2, by_weight), dim=-1, stable=True).indices)
    count = torch.clamp(s.lengths, max=c["budget"])
    take = min(c["budget"], s.longest)
    lanes = torch.arange(c["budget"], device="cuda")
    valid = lanes[None, None, :take] < count[:, None, None]
    kept = torch.where(valid, order[:, :, :take], torch.full_like(order[:, :, :take], s.longest))
    kept = torch.sort(kept, dim=-1).values
    kept = torch.where(valid, kept, torch.full_like(kept, -1))
    b, hh, j = torch.nonzero(valid.expand_as(kept), as_tuple=True)
    src = kept[b, hh, j]
    sp, ss = s.page_table[b, src // size].long(), src % size
    dp, ds = s.new_table[b, j // size].long(), j % size
    _bits(s.keys)[dp, ds, hh] = _bits(s.keys)[sp, ss, hh]
    _bits(s.values)[dp, ds, hh] = _bits(s.values)[sp, ss, hh]
    s.weights[dp, hh, ds] = s.weights[sp, hh, ss]
    full = torch.full((kept.shape[0], h, c["budget"]), -1, dtype=torch.int32, device="cuda")
    full[:, :, :take] = kept.to(torch.int32)
    return {"kept": full, "lengths": count, "keys": s.keys, "values": s.values, "weights": s.weights}


def _bits(t):
    """Eight-bit rows as bytes, for indexing; others as they are."""
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


def _turn(x, s):
    """Rows [tokens, heads, width] in fp32, their first 2 * pairs values turned; angles in 64 bits."""
    n = s.freq.numel()
    angle = s.positions[s.axis.long()].double() * s.freq.double()[:, None]
    cos, sin = (f(angle).float().t()[:, None] for f in (torch.cos, torch.sin))
    rest = x[..., 2 * n:]
    if s.case["interleaved"]:
        a, b = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = x[..., :n], x[..., n:2 * n]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, rest), dim=-1)


# ---- what a pass cannot do without ---------------------------------------------------------------
def work(case):
    op, d = case["op"], case["width"]
    if op == "rotary":
        rows = case["tokens"] * (case["q_heads"] + case["kv_heads"])
        return {"bytes": 4 * rows * d * _BYTES[case["dtype"]] + 2 * 4 * case["axes"] * case["tokens"],
                "flops": 2 * 3 * rows * 2 * case["pairs"]}
    h = case["kv_heads"]
    if op == "append":
        tokens = sum(_new(case))
        wide = _BYTES[case["dtype"]]
        return {"bytes": tokens * d * (2 * case["q_heads"] * wide + 2 * h * (wide + _BYTES[case["cache"]]))
                + 4 * tokens * (case["axes"] + h) + 16 * case["sequences"],
                "flops": 3 * tokens * (case["q_heads"] + h) * 2 * case["pairs"]}
    rows = sum(_held(case))
    row = 2 * d * _BYTES[case["cache"]]
    if op == "attend":
        n = case["sequences"] * case["q_heads"] * d
        return {"bytes": rows * h * (row + 8) + 2 * n * _BYTES[case["dtype"]] + 4 * case["sequences"] * case["q_heads"]
                + 4 * (rows // case["page"]), "flops": 4 * rows * case["q_heads"] * d}
    kept = sum(min(n, case["budget"]) for n in _held(case))
    return {"bytes": 4 * rows * h + kept * h * (2 * row + 8) + 4 * case["sequences"] * h * case["budget"],
            "flops": rows * h}


# ---- the definition in 64 bits -------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "append": _exact_append, "attend": _exact_attend, "evict": _exact_evict}[case["op"]](s)


def _rotation(x, positions, s, sign=1.0):
    """Complex product with e^(i angle), pair by pair, in 64 bits."""
    x = x.detach().double()
    y = x.clone()
    for i in range(s.freq.numel()):
        u, v = (2 * i, 2 * i + 1) if s.case["interleaved"] else (i, i + s.freq.numel())
        angle = sign * positions[int(s.axis[i])].double() * float(s.freq[i])
        z = torch.complex(x[:, :, u], x[:, :, v]) * torch.polar(torch.ones_like(angle), angle)[:, None]
        y[:, :, u], y[:, :, v] = z.real, z.imag
    return y


def _exact_rotary(s):
    return {"q": _rotation(s.q, s.positions, s), "k": _rotation(s.k, s.positions, s),
            "gq": _rotation(s.gq, s.positions, s, -1.0), "gk": _rotation(s.gk, s.positions, s, -1.0)}


def _exact_append(s):
    keys, values, weights = s.keys.double(), s.values.double(), s.weights.double()
    k, v = _rotation(s.k, s.positions, s), s.v.double()
    if s.k_scale is not None:
        k = (k / s.k_scale.double()[:, None]).clamp(-_E4M3_MAX, _E4M3_MAX)
        v = (v / s.v_scale.double()[:, None]).clamp(-_E4M3_MAX, _E4M3_MAX)
    size, ends = s.case["page"], s.offsets.tolist()
    for b, held in enumerate(s.lengths.tolist()):
        at = torch.arange(held, held + ends[b + 1] - ends[b], device="cuda")
        page, slot = s.page_table[b].long()[at // size], at % size
        keys[page, slot], values[page, slot] = k[ends[b]:ends[b + 1]], v[ends[b]:ends[b + 1]]
        weights[page, :, slot] = 0.0
    return {"q": _rotation(s.q, s.positions, s), "lengths": None, "keys": keys, "values": values, "weights": weights}


def _exact_attend(s):
    n, heads, d = s.q.shape
    h, size = s.keys.shape[2], s.case["page"]
    out = torch.zeros((n, heads, d), dtype=torch.float64, device="cuda")
    lse = torch.full((n, heads), -math.inf, dtype=torch.float64, device="cuda")
    weights = s.weights.double()
    for b, length in enumerate(s.lengths.tolist()):
        if not length:
            continue
        at = torch.arange(length, device="cuda")
        page, slot = s.page_table[b].long()[at // size], at % size
        for i in range(h):
            k, v = (_bits(t)[page, slot, i].view(t.dtype).double() for t in (s.keys, s.values))
            if s.k_scale is not None:
                k, v = k * s.k_scale[i].double(), v * s.v_scale[i].double()
            mine = slice(i * (heads // h), (i + 1) * (heads // h))
            x = (s.q[b, mine].double() @ k.T) * s.scale
            lse[b, mine] = torch.logsumexp(x, dim=1)
            p = torch.exp(x - lse[b, mine, None])
            out[b, mine] = p @ v
            weights[page, i, slot] += p.sum(dim=0)
    return {"out": out, "lse": lse, "weights": weights}


def _exact_evict(s):
    """Rows and weights are moved, not computed; the kept rows are whole numbers."""
    c, size = s.case, s.case["page"]
    keys, values, weights = s.keys.clone(), s.values.clone(), s.weights.clone()
    for b, length in enumerate(s.lengths.tolist()):
        count = min(length, c["budget"])
        if not count:
            continue
        at = torch.arange(length, device="cuda")
        for i in range(s.keys.shape[2]):
            w = s.weights[s.page_table[b].long()[at // size], i, at % size].double()
            w = torch.where(torch.isnan(w), torch.full_like(w, -math.inf), w)
            fixed = min(c["sinks"], count)
            late = min(c["recent"], count - fixed)
            middle = torch.argsort(w[fixed:length - late], descending=True, stable=True)[:count - fixed - late] + fixed
            kept = torch.cat((at[:fixed], torch.sort(middle).values, at[length - late:]))
            j = torch.arange(count, device="cuda")
            dp, ds = s.new_table[b].long()[j // size], j % size
            sp, ss = s.page_table[b].long()[kept // size], kept % size
            for t in (keys, values):
                _bits(t)[dp, ds, i] = _bits(t)[sp, ss, i]
            weights[dp, i, ds] = weights[sp, i, ss]
    return {"kept": None, "lengths": None, "keys": keys.double(), "values": values.double(), "weights": weights.double()}
