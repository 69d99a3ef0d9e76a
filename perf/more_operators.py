"""The operators of an attention sublayer over a paged cache as measurable
cases: block tables and slot maps from request lengths, rotary positions (and
their gradient), the same while a fused projection's keys and values are stored
into the cache's pages, and attention of a chunk of new tokens (one each while
generating) over the pages.

With ``own`` false, ``run`` computes an operator in elementary torch
operations, in 32 bits whatever the inputs' type (angles in 64), rounded once at
the end. With ``own`` true it launches the framework's operator program
(``tcacomp_amd.attention``), as a user's program does: on tensors that are
already on the GPU, into output tensors that the caller owns. The compiled
program is the handle such a program keeps, one for each set of attributes.

``listed`` holds fixed points of the ranges, ``draw`` any point of them:

  tables     1 to 4096 sequences, 0 to 2048 new tokens each, pages of 1 to 256
  rotary     1 to 16384 tokens, 1 to 64 heads of 16 to 256 features, all of
             them or a part rotated, halves or neighbours paired, f32, bf16, f16
  attention  1 to 64 sequences, 0 to 4096 new tokens each over contexts of up
             to 32768 keys, 1 to 16 key heads by groups of 1 to 16 query heads
             of 32 to 256 features, pages of 8 to 256 tokens, bf16 and f16

A cache is k, v [pages][key heads][tokens of a page][features]; queries are [tokens]
[key heads][group][features]; a sequence's last new token sees its whole cache.
"""
import functools
import math
import random

import torch

own = False

DEVICE = "cuda"
ELEMS = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # A step of 256 sequences that generate: one token each, a new page now and then.
        {"name": "table_decode_256", "op": "page_table", "s": 256, "new": 1, "mode": "same", "context": 8000, "page": 16, "pad": 0, "mix": 1},
        # Prompts of any length admitted together, in a batch padded to a captured size.
        {"name": "table_prompts_odd", "op": "page_table", "s": 37, "new": 1500, "mode": "ragged", "context": 700, "page": 24, "pad": 999, "mix": 2},
        # A large server's step: thousands of sequences, some in the middle of their prompts.
        {"name": "table_large", "op": "page_table", "s": 4096, "new": 64, "mode": "ragged", "context": 4000, "page": 64, "pad": 0, "mix": 3},
        # A training batch's queries.
        {"name": "rotary_8192", "op": "rotary", "elem": "bf16", "t": 8192, "h": 32, "d": 128, "f": 64, "interleaved": False, "inverse": False, "scale": 1.0, "far": 8192},
        # The gradient, part of a head of odd size, far positions, in f32.
        {"name": "rotary_inverse_odd", "op": "rotary", "elem": "f32", "t": 1001, "h": 9, "d": 75, "f": 20, "interleaved": True, "inverse": True, "scale": 1.0, "far": 1000000},
        # One sequence generates a token: latency.
        {"name": "cache_one_token", "op": "rotary_cache", "elem": "bf16", "t": 1, "hk": 8, "g": 4, "d": 128, "f": 64, "interleaved": False, "scale": 1.0, "page": 16, "pad": 0, "far": 8192},
        # A prompt's chunk of a model stretched to a long context, padded rows behind it.
        {"name": "cache_chunk_4000", "op": "rotary_cache", "elem": "f16", "t": 4000, "hk": 8, "g": 4, "d": 128, "f": 32, "interleaved": False, "scale": 1.25, "page": 64, "pad": 96, "far": 131072},
        # One sequence generates over a long context: the cache split over the card.
        {"name": "attend_one_token", "op": "paged_attention", "elem": "bf16", "s": 1, "new": 1, "mode": "same", "context": 16000, "hk": 8, "g": 4, "d": 128, "page": 16, "window": 0, "stats": False, "pad": 0, "mix": 4},
        # Sixty-four sequences generate together: the cache is read once.
        {"name": "attend_decode_64", "op": "paged_attention", "elem": "bf16", "s": 64, "new": 1, "mode": "same", "context": 8000, "hk": 8, "g": 4, "d": 128, "page": 16, "window": 0, "stats": False, "pad": 0, "mix": 5},
        # Two prompts at once, nothing in the cache before them.
        {"name": "attend_prompt_4096", "op": "paged_attention", "elem": "f16", "s": 2, "new": 4096, "mode": "same", "context": 0, "hk": 8, "g": 4, "d": 128, "page": 64, "window": 0, "stats": False, "pad": 0, "mix": 6},
        # Chunks of long prompts over what the cache holds of them: the largest case.
        {"name": "attend_chunk_512", "op": "paged_attention", "elem": "bf16", "s": 4, "new": 512, "mode": "same", "context": 16000, "hk": 4, "g": 8, "d": 128, "page": 32, "window": 0, "stats": False, "pad": 0, "mix": 7},
        # Odd lengths, none for some, odd pages, a sliding window, statistics kept to merge with another part.
        {"name": "attend_ragged_window", "op": "paged_attention", "elem": "f16", "s": 9, "new": 201, "mode": "ragged", "context": 3001, "hk": 5, "g": 3, "d": 64, "page": 24, "window": 1000, "stats": True, "pad": 17, "mix": 8},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(("page_table", "rotary", "rotary", "rotary_cache", "rotary_cache") + ("paged_attention",) * 5)
    mix = rng.randrange(1 << 30)
    if op == "page_table":
        s, mode = _log(rng, 1, 4096), rng.choice(("same", "ragged", "mixed"))
        return {"op": op, "s": s, "new": _log(rng, 1, min(2048, (1 << 17) // s)), "mode": mode, "context": _log(rng, 1, 8192),
                "page": _log(rng, 1, 256) if rng.random() < 0.5 else rng.choice((16, 32, 64, 128)), "pad": rng.choice((0, 0, 13)), "mix": mix}
    d = rng.choice((64, 128)) if rng.random() < 0.5 else rng.randrange(4, 33) * 8
    page = rng.choice((16, 32, 64, 128)) if rng.random() < 0.5 else _log(rng, 8, 256)
    if op != "paged_attention":
        if rng.random() < 0.25:
            d = rng.randrange(16, 257)
        f = d // 2 if rng.random() < 0.5 else rng.randrange(1, d // 2 + 1)
        case = {"op": op, "elem": rng.choice(sorted(ELEMS)), "d": d, "f": f, "interleaved": rng.random() < 0.5, "scale": rng.choice((1.0, 1.0, 1.25)), "far": _log(rng, 16, 1 << 20)}
        if op == "rotary":
            case.update(h=_log(rng, 1, 64), inverse=rng.random() < 0.5)
            width = case["h"] * d
        else:
            case.update(hk=_log(rng, 1, 16), g=_log(rng, 1, 16), page=page, pad=rng.choice((0, 0, 5)))
            width = case["hk"] * (case["g"] + 2) * d
        case["t"] = _log(rng, 1, min(16384, (1 << 25) // width))
        return case
    while True:
        s, mode = _log(rng, 1, 64), rng.choice(("same", "same", "ragged", "mixed"))
        new = 1 if rng.random() < 0.4 else _log(rng, 1, 4096)
        case = {"op": op, "elem": rng.choice(("bf16", "f16")), "s": s, "new": new, "mode": mode, "context": _log(rng, 1, 32768), "hk": _log(rng, 1, 16),
                "g": _log(rng, 1, 16), "d": d, "page": page, "window": rng.choice((0, 0, 0, _log(rng, 1, 8192))), "stats": rng.random() < 0.3,
                "pad": rng.choice((0, 0, 7)), "mix": mix}
        width = case["hk"] * d
        longest = case["context"] + new
        if s * longest * width <= 1 << 28 and s * new * longest * case["hk"] * case["g"] <= 1 << 30 and s * new * longest * width * case["g"] <= 1 << 36:
            return case


def _lengths(case):
    """Tokens that each sequence has in the cache, and new ones: by the case alone."""
    rng = random.Random(case["mix"])
    s, new = case["s"], case["new"]
    held = [rng.randint(case["context"] // 2, case["context"]) for _ in range(s)]
    if case["mode"] == "same":
        fresh = [new] * s
    elif case["mode"] == "mixed":  # one chunk beside sequences that generate
        fresh = [new] + [1] * (s - 1)
    else:  # any length, none and nothing held among them
        fresh = [rng.choice((0, 1, new, rng.randint(0, new), rng.randint(0, new))) for _ in range(s)]
        fresh[s // 2] = new
        held[s // 3] = 0
    return held, fresh


def _pages(tokens, page):
    return [-(-n // page) for n in tokens]


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _normal(gen, shape, elem):
    return torch.randn(shape, generator=gen, device=DEVICE).to(ELEMS[elem])


def _frequencies(f):
    """base^(-i / f), as a model holds them: in 32 bits."""
    return torch.tensor([10000.0 ** (-i / f) for i in range(f)], dtype=torch.float32, device=DEVICE)


def prepare(case, seed):
    """The inputs, and the output tensors that the caller owns."""
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    op = case["op"]
    empty = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=DEVICE)  # noqa: E731
    if op == "page_table":
        s, page = case["s"], case["page"]
        held, fresh = _lengths(case)
        have, need = _pages(held, page), _pages([a + b for a, b in zip(held, fresh)], page)
        total = sum(need)
        ids = torch.randperm(total + 3, generator=gen, device=DEVICE).int()
        table = torch.full((s, max(need) + 2), -1, dtype=torch.int32, device=DEVICE)
        col = torch.arange(table.shape[1], device=DEVICE)
        mine = col < _ints(have)[:, None]
        table[mine] = ids[:sum(have)]
        free, t = ids[sum(have):].contiguous(), sum(fresh) + case["pad"]
        return {"case": case, "in": [_ints(held), _ints(fresh), free, _ints([1])],
                "out": [table, empty(s + 1), empty(s), empty(t), empty(t), empty(1)]}
    e, d = case["elem"], case["d"]
    if op in ("rotary", "rotary_cache"):
        t = case["t"]
        pos = torch.randint(0, case["far"], (t,), generator=gen, device=DEVICE, dtype=torch.int32)
        freq = _frequencies(case["f"])
        if op == "rotary":
            x = _normal(gen, (t, case["h"], d), e)
            return {"case": case, "in": [x, pos, freq], "out": [torch.empty_like(x)]}
        hk, g, page, rows = case["hk"], case["g"], case["page"], t + case["pad"]
        pages = -(-t // page) + 2
        slot = torch.randperm(pages * page, generator=gen, device=DEVICE)[:t].int()
        behind = torch.full((case["pad"],), -1, dtype=torch.int32, device=DEVICE)
        x = _normal(gen, (rows, hk * (g + 2), d), e)
        k, v = (_normal(gen, (pages, hk, page, d), e) for _ in range(2))
        return {"case": case, "in": [x, torch.cat([pos, behind]), torch.cat([slot, behind]), freq],
                "out": [torch.empty((rows, hk, g, d), device=DEVICE, dtype=ELEMS[e]), k, v]}
    hk, g, page = case["hk"], case["g"], case["page"]
    held, fresh = _lengths(case)
    lens = [a + b for a, b in zip(held, fresh)]
    need = _pages(lens, page)
    total, t = sum(need), sum(fresh) + case["pad"]
    table = torch.full((case["s"], max(need) + 1), -1, dtype=torch.int32, device=DEVICE)
    col = torch.arange(table.shape[1], device=DEVICE)
    table[col < _ints(need)[:, None]] = torch.randperm(total, generator=gen, device=DEVICE).int()
    starts = [0]
    for n in fresh:
        starts.append(starts[-1] + n)
    q = _normal(gen, (t, hk, g, d), e)
    k, v = (_normal(gen, (max(total, 1), hk, page, d), e) for _ in range(2))
    outs = [torch.zeros_like(q)] + ([torch.zeros((t, hk, g), device=DEVICE)] if case["stats"] else [])
    return {"case": case, "in": [q, k, v, table, _ints(starts), _ints(lens)], "out": outs, "most": (max(fresh), max(lens))}


@functools.lru_cache(maxsize=None)
def _program(op, elem, **flags):
    from tcacomp_amd import attention, compiler

    made = {
        "page_table": lambda: attention.page_table(),
        "rotary": lambda: attention.rotary(elem, **flags),
        "rotary_cache": lambda: attention.rotary_cache(elem, **flags),
        "paged_attention": lambda: attention.paged_attention(elem, **flags),
    }[op]()
    return compiler.compile_program(made)


def run(state):
    case = state["case"]
    op, e = case["op"], case.get("elem")
    if own:
        tensors = state["in"] + state["out"]
        if op == "page_table":
            _program(op, e).launch(tensors, free_dims=(case["page"],))
        elif op == "rotary":
            _program(op, e, interleaved=case["interleaved"], inverse=case["inverse"]).launch(tensors, scalars=(case["scale"],))
        elif op == "rotary_cache":
            _program(op, e, interleaved=case["interleaved"]).launch(tensors, scalars=(case["scale"],))
        else:
            program = _program(op, e, window=bool(case["window"]), stats=case["stats"])
            program.launch(tensors, free_dims=(case["window"],) if case["window"] else (), scalars=(case["d"] ** -0.5,))
        return state["out"]
    return _plain[op](state, case, *state["in"])


def _page_table(state, case, held, new, free, first):
    table, starts, _, pos, _, _ = state["out"]
    page, columns = case["page"], table.shape[1]
    h, n = held.long(), new.long()
    have, need = (h + page - 1) // page, ((h + n + page - 1) // page).clamp(max=columns)
    take = (need - have).clamp(min=0)
    before = take.cumsum(0) - take + first.long()
    col = torch.arange(columns, device=DEVICE)
    from_free = before[:, None] + col - have[:, None]
    taken = torch.where(from_free < free.shape[0], free[from_free.clamp(0, free.shape[0] - 1)].long(), -1)
    table = torch.where((col >= have[:, None]) & (col < need[:, None]), taken, table.long())
    ends = n.cumsum(0)
    starts = torch.cat([torch.zeros_like(ends[:1]), ends])
    t = torch.arange(pos.shape[0], device=DEVICE)
    s = torch.searchsorted(ends, t, right=True).clamp(max=ends.shape[0] - 1)
    at = h[s] + t - starts[s]
    held_by = table[s, (at // page).clamp(max=columns - 1)]
    slot = torch.where((at // page < columns) & (held_by >= 0), held_by * page + at % page, -1)
    live = t < ends[-1]
    return [x.int() for x in (table, starts, h + n, torch.where(live, at, -1), torch.where(live, slot, -1), first + take.sum())]


def _turn(case, x, pos, freq):
    """x [T, heads, D] in 32 bits, turned by its positions' angles."""
    f = case["f"]
    angle = pos.double()[:, None] * freq.double()
    c, s = (case["scale"] * t.float()[:, None] for t in (angle.cos(), angle.sin()))
    if case.get("inverse"):
        s = -s
    y = x.clone()
    a, b = (slice(0, 2 * f, 2), slice(1, 2 * f, 2)) if case["interleaved"] else (slice(0, f), slice(f, 2 * f))
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def _rotary(state, case, x, pos, freq):
    return [_turn(case, x.float(), pos, freq).to(x.dtype)]


def _rotary_cache(state, case, x, pos, slot, freq):
    _, k, v = state["out"]
    hk, g, page = case["hk"], case["g"], case["page"]
    turned = _turn(case, x[:, :hk * (g + 1)].float(), pos, freq).to(x.dtype)
    t = case["t"]  # rows behind it have no slot
    at, off = slot[:t].long() // page, slot[:t].long() % page
    k[at, :, off] = turned[:t, hk * g:]
    v[at, :, off] = x[:t, hk * (g + 1):]
    return [turned[:, :hk * g].reshape(-1, hk, g, case["d"]), k, v]


def _paged_attention(state, case, q, k, v, table, starts, lens):
    hk, g, d, page = case["hk"], case["g"], case["d"], case["page"]
    new, longest = state["most"]
    s = table.shape[0]
    n = (starts[1:] - starts[:-1]).long()
    i, j = torch.arange(new, device=DEVICE), torch.arange(longest, device=DEVICE)
    rows, live = starts[:-1].long()[:, None] + i, i < n[:, None]
    pages = table[:, j // page].long()
    # [sequence, key head][...]
    queries = q[rows.clamp(max=q.shape[0] - 1)].float().permute(0, 2, 1, 3, 4).reshape(s * hk, new * g, d)
    keys = k[pages.clamp(min=0), :, j % page].float().permute(0, 2, 3, 1).reshape(s * hk, d, longest)
    values = v[pages.clamp(min=0), :, j % page].float().permute(0, 2, 1, 3).reshape(s * hk, longest, d)
    at = (lens.long() - n)[:, None] + i
    sees = (j <= at[..., None]) & (pages >= 0)[:, None]
    if case["window"]:
        sees = sees & (j > at[..., None] - case["window"])
    score = torch.matmul(queries, keys).view(s, hk, new, g, longest) * d ** -0.5
    score = torch.where(sees[:, None, :, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    y = torch.matmul(p.view(s * hk, new * g, longest), values).view(s, hk, new, g, d) / torch.where(total > 0, total, 1.0)
    out = [state["out"][0].clone()]
    out[0][rows[live]] = y.permute(0, 2, 1, 3, 4)[live].to(q.dtype)
    if case["stats"]:
        out.append(state["out"][1].clone())
        out[1][rows[live]] = (top + total.log())[..., 0].permute(0, 2, 1, 3)[live]
    return out


_plain = {"page_table": _page_table, "rotary": _rotary, "rotary_cache": _rotary_cache, "paged_attention": _paged_attention}


def work(case):
    op = case["op"]
    if op == "page_table":
        held, fresh = _lengths(case)
        have, need = _pages(held, case["page"]), _pages([a + b for a, b in zip(held, fresh)], case["page"])
        s, t, taken = case["s"], sum(fresh) + case["pad"], sum(need) - sum(have)
        return {"bytes": 4 * (2 * s + 2 * taken + 1 + 2 * s + 1 + 2 * t + 1), "flops": 4 * t + 8 * s}
    size = 4 if case["elem"] == "f32" else 2
    d = case["d"]
    if op == "rotary":
        t, h = case["t"], case["h"]
        return {"bytes": 2 * size * t * h * d + 4 * t + 4 * case["f"], "flops": 6 * t * h * case["f"]}
    hk, g = case["hk"], case["g"]
    if op == "rotary_cache":
        t = case["t"] + case["pad"]
        return {"bytes": 2 * size * t * hk * (g + 2) * d + 8 * t + 4 * case["f"], "flops": 6 * t * hk * (g + 1) * case["f"]}
    held, fresh = _lengths(case)
    seen = keys = 0
    for h, n in zip(held, fresh):
        w = case["window"] or h + n
        seen += sum(min(h + i + 1, w) for i in range(n))
        keys += min(h + n, w + n - 1) if n else 0
    t, entries = sum(fresh), -(-keys // case["page"])
    return {"bytes": size * (2 * t * hk * g * d + 2 * keys * hk * d) + 4 * (entries + 2 * case["s"] + 1) + (4 * t * hk * g if case["stats"] else 0),
            "flops": 4 * seen * hk * g * d}


def exact(case, seed):
    """The operators' definitions in 64 bits on the same inputs, a sequence at a time."""
    op = case["op"]
    state = prepare(case, seed)
    if op == "page_table":
        return None  # whole numbers
    if op in ("rotary", "rotary_cache"):
        x, pos, freq = state["in"][0], state["in"][1], state["in"][-1]
        f = case["f"]
        # a pair as a complex number, times e^(i angle)
        angle = torch.outer(pos.double(), freq.double())
        turn = torch.polar(torch.full_like(angle, case["scale"]), -angle if case.get("inverse") else angle).unsqueeze(1)
        z = x.double()
        first, second = (z[..., 0:2 * f:2], z[..., 1:2 * f:2]) if case["interleaved"] else (z[..., :f], z[..., f:2 * f])
        w = torch.complex(first.contiguous(), second.contiguous()) * turn
        pair = torch.stack([w.real, w.imag], -1 if case["interleaved"] else -2).flatten(-2)
        y = torch.cat([pair, z[..., 2 * f:]], -1)
        if op == "rotary":
            return [y]
        hk, g, page, t = case["hk"], case["g"], case["page"], case["t"]
        k, v = state["out"][1].double(), state["out"][2].double()
        slot = state["in"][2][:t].long()
        k.transpose(1, 2)[slot // page, slot % page] = y[:t, hk * g:hk * (g + 1)]
        v.transpose(1, 2)[slot // page, slot % page] = z[:t, hk * (g + 1):]
        return [y[:, :hk * g].unflatten(1, (hk, g)), k, v]
    q, k, v, table, _, _ = state["in"]
    held, fresh = _lengths(case)
    hk, d, page = case["hk"], case["d"], case["page"]
    y = state["out"][0].double()
    lse = state["out"][1].double() if case["stats"] else None
    at = 0
    for s, (h, n) in enumerate(zip(held, fresh)):
        if n == 0:
            continue
        mine = table[s, :-(-(h + n) // page)].long()
        j = torch.arange(h + n, device=DEVICE)
        i = h + torch.arange(n, device=DEVICE).unsqueeze(1)
        hidden = j > i
        if case["window"]:
            hidden |= j <= i - case["window"]
        for b in range(hk):
            keys, values = (c[mine, b].reshape(-1, d)[:h + n].double() for c in (k, v))
            z = torch.tensordot(q[at:at + n, b].double(), keys, dims=([2], [1])).mul_(1.0 / math.sqrt(d))
            z.masked_fill_(hidden.unsqueeze(1), -math.inf)
            if lse is not None:
                lse[at:at + n, b] = torch.logsumexp(z, -1)
            y[at:at + n, b] = torch.softmax(z, -1) @ values
        at += n
    return [y] + ([lse] if case["stats"] else [])
