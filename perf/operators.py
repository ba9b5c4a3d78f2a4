"""The serving operators on paged key-value caches, case by case.

Three operators that a decoder needs to read a prompt and answer it:

* append:  the keys and values of new tokens are rotated by their positions
           and written to their slots of a paged cache, the queries are
           rotated on the way (``kv_append``);
* prompt:  causal attention over packed prompts of different lengths with
           grouped heads (``prompt_attention``);
* decode:  attention of one new token per sequence over its paged cache
           (``paged_decode``).

``listed`` gives the cases, ``draw`` more of the same ranges, ``prepare`` a
case's inputs, ``run`` one pass, ``exact`` the result in 64 bits and ``work``
the bytes and operations of a pass.  While ``own`` is false ``run`` computes
the operators from elementary torch operations in 32 bits.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
MAX_POSITION = 32768       # rows of the rotation table


def listed():
    return [
        # one token of one conversation joins its cache: latency only
        dict(name="append_one", op="append", dtype="bf16", tokens=1, heads=32, kv_heads=8, dim=128,
             page=16, rot=128, interleaved=False, head_major=False, spread=0),
        # one step of a batch of 200 conversations with a few padded places,
        # interleaved pairs, only half of a narrow head rotated
        dict(name="append_step", op="append", dtype="f16", tokens=200, heads=16, kv_heads=16, dim=64,
             page=32, rot=32, interleaved=True, head_major=True, spread=5),
        # the tokens of a large prompt batch
        dict(name="append_prompts", op="append", dtype="bf16", tokens=24576, heads=32, kv_heads=8,
             dim=128, page=16, rot=128, interleaved=False, head_major=False, spread=3),
        # one conversation that has just begun: latency only
        dict(name="decode_one_short", op="decode", dtype="bf16", heads=32, kv_heads=8, dim=128,
             page=16, head_major=False, count=1, low=77, high=77, spread=0),
        # one conversation with a long document: only the cache's length to share out
        dict(name="decode_one_long", op="decode", dtype="bf16", heads=32, kv_heads=8, dim=128,
             page=64, head_major=True, count=1, low=131001, high=131001, spread=0),
        # an ordinary batch of chats of different lengths
        dict(name="decode_batch", op="decode", dtype="bf16", heads=32, kv_heads=8, dim=128,
             page=16, head_major=False, count=32, low=200, high=4000, spread=1),
        # a full server: many conversations, a few slots of the batch unused (length 0)
        dict(name="decode_full", op="decode", dtype="bf16", heads=64, kv_heads=8, dim=128,
             page=32, head_major=False, count=256, low=250, high=8192, spread=2, unused=8),
        # narrow heads that share nothing
        dict(name="decode_unshared", op="decode", dtype="f16", heads=20, kv_heads=20, dim=64,
             page=32, head_major=True, count=45, low=1, high=3001, spread=4),
        # one short question: latency only
        dict(name="prompt_short", op="prompt", dtype="bf16", heads=32, kv_heads=8, dim=128,
             causal=True, count=1, low=19, high=19, prefix=0, spread=0),
        # the prompts of several users in one pass
        dict(name="prompt_packed", op="prompt", dtype="bf16", heads=32, kv_heads=8, dim=128,
             causal=True, count=14, low=60, high=2048, prefix=0, spread=1),
        # one long document
        dict(name="prompt_long", op="prompt", dtype="bf16", heads=32, kv_heads=8, dim=128,
             causal=True, count=1, low=8192, high=8192, prefix=0, spread=0),
        # later pieces of prompts whose first parts are there already, narrow
        # heads in odd groups, one sequence without new tokens
        dict(name="prompt_pieces", op="prompt", dtype="f16", heads=15, kv_heads=5, dim=64,
             causal=True, count=7, low=100, high=1300, prefix=3000, spread=3, unused=1),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        top = most.setdefault(c["op"], {"bytes": 0, "flops": 0})
        for key in top:
            top[key] = max(top[key], w[key])
    op = rng.choice(["append", "decode", "prompt"])
    while True:
        kv_heads = rng.choice([1, 2, 3, 4, 5, 8, 12, 16])
        group = rng.choice([1, 1, 2, 3, 4, 4, 5, 6, 7, 8, 16])
        case = dict(op=op, dtype=rng.choice(["bf16", "bf16", "f16"]), heads=kv_heads * group,
                    kv_heads=kv_heads, dim=rng.choice([64, 128, 128]), spread=rng.randrange(1 << 30))
        if op == "append":
            case.update(tokens=_log_int(rng, 1, 24576), page=rng.choice([1, 8, 16, 24, 32, 64, 128]),
                        interleaved=rng.random() < 0.3, head_major=rng.random() < 0.3)
            case["rot"] = rng.choice([case["dim"], case["dim"], case["dim"] // 2])
        else:
            case.update(count=_log_int(rng, 1, 256 if op == "decode" else 48))
            top = _log_int(rng, 1, 131072 if op == "decode" else 8192)
            case.update(low=_log_int(rng, max(1, top // 64), top), high=top,
                        unused=rng.randrange(3) if case["count"] > 3 else 0)
            if op == "decode":
                case.update(page=rng.choice([1, 8, 16, 24, 32, 64, 128]), head_major=rng.random() < 0.3)
            else:
                case.update(causal=rng.random() < 0.85, prefix=rng.choice([0, 0, _log_int(rng, 1, 4096)]))
        w = work(case)
        tokens = sum(lengths_of(case)[1]) if op != "append" else case["tokens"]
        # the plain form pads a decode batch to its longest sequence
        padded = case["count"] * case["high"] if op == "decode" else tokens
        if (w["bytes"] <= most[op]["bytes"] and w["flops"] <= most[op]["flops"]
                and padded * case["kv_heads"] * case["dim"] <= 256 * 8192 * 8 * 128):
            return case


def lengths_of(case):
    """(new tokens, keys) of each sequence: fixed by the case, the same for every seed."""
    rng = random.Random(case["spread"])
    low, high, count = case["low"], case["high"], case["count"]
    new = [_log_int(rng, low, high) for _ in range(count)]
    if case["op"] == "decode":
        keys = list(new)
    else:
        keys = [n + (rng.randrange(case["prefix"] + 1) if case["prefix"] else 0) for n in new]
    for _ in range(case.get("unused", 0)):
        at = rng.randrange(count)
        new[at] = 0
        if case["op"] == "decode":
            keys[at] = 0
    return new, keys


def _pairs(case):
    """Query-key pairs that the mask leaves, over all sequences."""
    total = 0
    for n, m in zip(*lengths_of(case)):
        if case["op"] == "decode":
            total += m
        elif not case["causal"]:
            total += n * m
        else:
            total += n * (m - n) + n * (n + 1) // 2
    return total


def work(case):
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        t = case["tokens"]
        # queries, keys and values in and out, one row of the rotation table
        # for each distinct position, positions and slots
        rows = min(t, MAX_POSITION)
        return {"bytes": t * (h + 2 * hk) * d * 2 * 2 + rows * case["rot"] * 4 + t * 8,
                "flops": t * (h + hk) * case["rot"] * 3}
    new, keys = lengths_of(case)
    if case["op"] == "decode":
        pages = sum(-(-m // case["page"]) for m in keys)
        moved = sum(keys) * hk * d * 2 * 2 + len(keys) * h * d * 2 * 2 + pages * 4 + len(keys) * 4
    else:
        used = sum(m for n, m in zip(new, keys) if n)
        moved = used * hk * d * 2 * 2 + sum(new) * h * d * 2 * 2 + 8 * len(keys)
    return {"bytes": moved, "flops": 4 * _pairs(case) * h * d}


def _randn(gen, dtype, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _cache(gen, dtype, pages, case):
    """A cache [pages, page, kv_heads, dim], its memory token by token or head by head,
    that still holds what earlier requests left."""
    hk, d, page = case["kv_heads"], case["dim"], case["page"]
    if case["head_major"]:
        return torch.randn(pages, hk, page, d, generator=gen, device="cuda", dtype=dtype).transpose(1, 2)
    return torch.randn(pages, page, hk, d, generator=gen, device="cuda", dtype=dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = random.Random(seed)
    dtype = DTYPES[case["dtype"]]
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    s = {"case": case}
    if case["op"] == "append":
        t, page = case["tokens"], case["page"]
        pages = -(-t // page) + 3
        # the slices of one fused projection's output
        qkv = _randn(gen, dtype, t, h + 2 * hk, d)
        s["q"], s["k"], s["v"] = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
        s["k_cache"], s["v_cache"] = (_cache(gen, dtype, pages, case) for _ in range(2))
        # runs of following positions, as prompts and chats bring them
        positions, run = [], 0
        while len(positions) < t:
            run = min(t - len(positions), host.choice([1, 1, 3, 50, 700, 3000]))
            start = host.randrange(MAX_POSITION - run)
            positions += range(start, start + run)
        s["positions"] = torch.tensor(positions, dtype=torch.int32, device="cuda")
        order = torch.randperm(pages, generator=gen, device="cuda")
        slots = (order[:, None] * page + torch.arange(page, device="cuda")).reshape(-1)[:t].to(torch.int32)
        if t > 32:   # padded places of the batch are written nowhere
            slots[torch.rand(t, generator=gen, device="cuda") < 0.02] = -1
        s["slots"] = slots
        half = case["rot"] // 2
        freq = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        angle = torch.arange(MAX_POSITION, device="cuda", dtype=torch.float64)[:, None] * freq
        s["table"] = torch.cat([angle.cos(), angle.sin()], 1).float()
        return s
    new, keys = lengths_of(case)
    s["scale"] = d ** -0.5
    if case["op"] == "decode":
        page = case["page"]
        each = [-(-m // page) for m in keys]
        total = sum(each) + 3
        s["q"] = _randn(gen, dtype, len(keys), h, d)
        s["k_cache"], s["v_cache"] = (_cache(gen, dtype, total, case) for _ in range(2))
        order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32).cpu()
        table = torch.full((len(keys), max(1, max(each))), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(each):
            table[b, :n] = order[at:at + n]
            at += n
        s["pages"] = table.cuda()
        s["lengths"] = torch.tensor(keys, dtype=torch.int32, device="cuda")
        return s
    s["new"], s["keys"] = new, keys
    s["q"] = _randn(gen, dtype, sum(new), h, d)
    kv = _randn(gen, dtype, sum(keys), 2 * hk, d)
    s["k"], s["v"] = kv[:, :hk], kv[:, hk:]
    ends = lambda each: torch.tensor([0] + each, device="cuda").cumsum(0).to(torch.int32)  # noqa: E731
    s["offsets"], s["kv_offsets"] = ends(new), ends(keys)
    return s


def _rotate(x, table, rot, interleaved):
    """The pairs of x's first `rot` elements turned by the table's angles, in 32 bits."""
    x = x.float()
    half = rot // 2
    c, s = table[:, None, :half], table[:, None, half:]
    turned, rest = x[..., :rot], x[..., rot:]
    a, b = (turned[..., 0::2], turned[..., 1::2]) if interleaved else (turned[..., :half], turned[..., half:])
    a, b = a * c - b * s, b * c + a * s
    turned = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([turned, rest], -1)


def _plain_append(s):
    case = s["case"]
    table = s["table"][s["positions"].long()]
    dtype = s["q"].dtype
    q = _rotate(s["q"], table, case["rot"], case["interleaved"]).to(dtype)
    k = _rotate(s["k"], table, case["rot"], case["interleaved"]).to(dtype)
    kept = s["slots"] >= 0
    slot = s["slots"][kept].long()
    page, place = slot // case["page"], slot % case["page"]
    s["k_cache"][page, place] = k[kept]
    s["v_cache"][page, place] = s["v"][kept]
    return q, s["k_cache"], s["v_cache"]


def _weights(scores):
    """exp(scores - max) and its sum over the last axis; a row with nothing left gives zeros."""
    top = scores.amax(-1, keepdim=True)
    e = (scores - torch.where(top == -math.inf, 0.0, top)).exp()
    total = e.sum(-1, keepdim=True)
    return e, torch.where(total == 0, 1.0, total)


def _plain_decode(s):
    case, q = s["case"], s["q"]
    count, h, d = q.shape
    hk, page = case["kv_heads"], case["page"]
    places = torch.arange(s["pages"].shape[1] * page, device="cuda")
    at = s["pages"].long()[:, places // page].clamp(min=0), (places % page).expand(count, -1)
    k, v = s["k_cache"][at].float(), s["v_cache"][at].float()              # [count, keys, hk, d]
    scores = q.float().view(count, hk, h // hk, d) @ k.permute(0, 2, 3, 1) * s["scale"]
    seen = places < s["lengths"][:, None]
    e, total = _weights(scores.masked_fill(~seen[:, None, None], -math.inf))
    return (e @ v.transpose(1, 2) / total).reshape(count, h, d).to(q.dtype)


def _plain_prompt(s):
    case, out = s["case"], []
    hk, d = case["kv_heads"], case["dim"]
    at = key_at = 0
    # the packed sequences one after the other
    for n, m in zip(s["new"], s["keys"]):
        q = s["q"][at:at + n].float().view(n, hk, case["heads"] // hk, d).permute(1, 2, 0, 3)
        k, v = (s[x][key_at:key_at + m].float().permute(1, 2, 0)[:, None] for x in "kv")
        at, key_at = at + n, key_at + m
        if not n:
            continue
        scores = q @ k * s["scale"]
        if case["causal"]:
            later = torch.arange(m, device="cuda") > torch.arange(n, device="cuda")[:, None] + (m - n)
            scores = scores.masked_fill_(later, -math.inf)
        e, total = _weights(scores)
        out.append((e @ v.transpose(2, 3) / total).permute(2, 0, 1, 3).flatten(1, 2).to(s["q"].dtype))
    return torch.cat(out) if out else s["q"].clone()


def run(s):
    op = s["case"]["op"]
    if not own:
        return {"append": _plain_append, "decode": _plain_decode, "prompt": _plain_prompt}[op](s)
    import ktir_cpu_b200 as K
    if op == "append":
        q = K.kv_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], q=s["q"],
                        positions=s["positions"], table=s["table"], interleaved=s["case"]["interleaved"])
        return q, s["k_cache"], s["v_cache"]
    if op == "decode":
        return K.paged_decode(s["q"], s["k_cache"], s["v_cache"], s["pages"], s["lengths"], scale=s["scale"])
    return K.prompt_attention(s["q"], s["k"], s["v"], s["offsets"], kv_offsets=s["kv_offsets"],
                              causal=s["case"]["causal"], scale=s["scale"])


def _exact_turn(x, table, rot, interleaved):
    """x's pairs as complex numbers, times e^(i angle)."""
    half = rot // 2
    x = x.double()
    turn = torch.complex(table[:, :half].double(), table[:, half:].double())[:, None]
    first = list(range(0, rot, 2)) if interleaved else list(range(half))
    second = list(range(1, rot, 2)) if interleaved else list(range(half, rot))
    z = torch.complex(x[..., first], x[..., second]) * turn
    y = x.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_rows(q, k, v, scale, seen):
    """softmax(scale q k^T) v over the keys that `seen` [n, m] leaves: q [n, d], k and v [m, d]."""
    logits = torch.einsum("nd,md->nm", q, k) * scale
    logits[~seen] = -math.inf
    norm = torch.logsumexp(logits, 1)
    p = torch.exp(logits - torch.where(norm == -math.inf, 0.0, norm)[:, None])
    return torch.einsum("nm,md->nd", p, v)


def exact(case, seed):
    s = prepare(case, seed)
    hk = case["kv_heads"]
    group = case["heads"] // hk
    if case["op"] == "append":
        table = s["table"].index_select(0, s["positions"])
        q = _exact_turn(s["q"], table, case["rot"], case["interleaved"])
        k = _exact_turn(s["k"], table, case["rot"], case["interleaved"])
        k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
        pages = torch.div(s["slots"], case["page"], rounding_mode="floor").tolist()
        places = torch.remainder(s["slots"], case["page"]).tolist()
        used = [i for i, slot in enumerate(s["slots"].tolist()) if slot >= 0]
        where = (torch.tensor([pages[i] for i in used], device="cuda", dtype=torch.long),
                 torch.tensor([places[i] for i in used], device="cuda", dtype=torch.long))
        k_cache.index_put_(where, k[used])
        v_cache.index_put_(where, s["v"].double()[used])
        return q, k_cache, v_cache
    if case["op"] == "decode":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        for b, m in enumerate(lengths_of(case)[1]):
            if not m:
                continue
            own_pages = s["pages"][b, :-(-m // case["page"])].long()
            k, v = (s[x].index_select(0, own_pages).flatten(0, 1)[:m].double() for x in ("k_cache", "v_cache"))
            every = torch.ones(group, m, dtype=torch.bool, device="cuda")
            for j in range(hk):
                rows = slice(j * group, (j + 1) * group)
                out[b, rows] = _exact_rows(s["q"][b, rows].double(), k[:, j], v[:, j], s["scale"], every)
        return out
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    at = key_at = 0
    for n, m in zip(*lengths_of(case)):
        seen = torch.ones(n, m, dtype=torch.bool, device="cuda")
        if case["causal"]:
            seen = seen.tril(m - n)
        k, v = (s[x][key_at:key_at + m].double() for x in "kv")
        for i in range(case["heads"] if n else 0):
            out[at:at + n, i] = _exact_rows(s["q"][at:at + n, i].double(), k[:, i // group], v[:, i // group],
                                            s["scale"], seen)
        at, key_at = at + n, key_at + m
    return out
