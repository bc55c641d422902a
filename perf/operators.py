"""Cases and plain forms of the operators of a smaller cache: keys and values held in 4 bits, and eviction of
cached tokens by the attention weight they have gathered.

A request's keys and values live in pages; ``table[item]`` lists the pages of a request, a page holds ``page``
tokens of all kv heads.  A cache is ``[pages, 2 (keys, values), kv_heads, page, row]``.  In the engine's own types
``row`` is the head size and a head's part of a page holds

    keys    [head_dim / 8][page][8]            values  [page / 8][head_dim][8]

In 4 bits a cache is uint8 with ``row = head_dim * 17 / 32``: every 32 neighbouring dims of a key or a value are a
group of 32 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign bit, two in a byte, the even dim in the low half) and one
byte ``e`` that stands for the factor ``2 ** (e - 127)`` (255: the group is not a number).  ``e`` is the smallest
from 2 to 252 with ``max |x| <= 7 * 2 ** (e - 127)``; the codes are the nearest, ties to the even code, those
beyond 6 are 6.  A head's part of a page holds the codes, then the factors (``G = head_dim / 32`` groups):

    keys    codes [G][page][16]                factors [G][page]
    values  codes [page / 8][16][G][8]         factors [page / 8][G][8]     (byte j of 16: dims 32 G + 2 j, 2 j + 1)

The operators:

    store    q and k of a step's tokens are turned by their positions' angles in place, k and v are written
             to the tokens' places in 4 bits; the pages written to are read back in the engine's type
    attend   causal attention of a step's tokens over a 4-bit cache (optionally a window), with the
             logarithm of every row's sum of exponentials
    weigh    the softmax weight every cached key gets from the step's rows, added to what it had gathered
    evict    of every request and kv head the last ``recent`` tokens and the heaviest others, ``keep`` in all,
             are moved to other pages in their order, with their weights
"""
from __future__ import annotations

import math
import random
from types import SimpleNamespace

import torch

own = False

LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
MAX_POSITIONS = 1 << 18


# ---------------------------------------------------------------------------------------------- cases
def _case(name, op, **more):
    base = dict(name=name, op=op, dtype="bfloat16", heads=48, kv_heads=8, head_dim=128, page=64)
    base.update(more)
    return base


def listed():
    return [
        # a decode step's tokens enter the cache: one request, then a full batch
        _case("store_decode_1", "store", items=1, tokens=1, rotary_dim=64),
        _case("store_decode_64", "store", items=64, tokens=64, rotary_dim=64),
        # portions of two prompts of uneven length in one step
        _case("store_prompt_8191", "store", items=2, tokens=8191, rotary_dim=64),
        # a short chat turn of one request: nothing but latency
        _case("attend_decode_1x77", "attend", items=1, context=77, queries=1, window=0),
        # ordinary serving: uneven requests, one token each
        _case("attend_decode_8x2100", "attend", items=8, context=2100, queries=1, window=0),
        # few requests with whole books in the cache
        _case("attend_decode_4x131071", "attend", items=4, context=131071, queries=1, window=0),
        # a portion of a prompt on a long prefix
        _case("attend_portion_512_of_16384", "attend", items=1, context=16384, queries=512, window=0),
        # the weight a decode step's rows give to long caches, in 4 bits
        _case("weigh_decode_16x8200", "weigh", cache="fp4", items=16, context=8200, queries=1, window=0),
        # a prompt portion over the engine's own bfloat16 cache
        _case("weigh_portion_2048_of_6000", "weigh", cache="bfloat16", items=1, context=6000, queries=2048, window=0),
        # the float32 engine, small heads, one short request
        _case("weigh_float32_300", "weigh", cache="float32", dtype="float32", heads=12, kv_heads=2, head_dim=64,
              items=3, context=300, queries=5, window=0),
        # a batch one page over its budget, as it happens every page of decoding
        _case("evict_8x2112", "evict", cache="fp4", items=8, context=2112, keep=2048, recent=256),
        # long prompts cut to a quarter
        _case("evict_4x32768", "evict", cache="bfloat16", items=4, context=32768, keep=8192, recent=1024),
    ]


def _spread(rng, low, high):
    """Over the logarithm; odd sizes are as likely as even ones."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["store", "attend", "weigh", "evict"])
    kv_heads, ratio = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 6, 8, 16])
    head_dim = rng.choice([64, 96, 128, 128, 256])
    single = rng.random() < 0.25            # the float32 engine
    case = dict(op=op, dtype="float32" if single else "bfloat16", heads=kv_heads * ratio, kv_heads=kv_heads,
                head_dim=head_dim, page=rng.choice([32, 64, 96, 128]))
    most_heads = 15360 // head_dim          # a token's q, k and v row
    if (ratio + 2) * kv_heads > most_heads:
        case["kv_heads"] = kv_heads = max(1, most_heads // (ratio + 2))
        case["heads"] = kv_heads * ratio
    if op == "store":
        tokens = _spread(rng, 1, 2048 if single else 6000)
        case.update(items=rng.randint(1, min(tokens, 64)), tokens=tokens,
                    rotary_dim=rng.choice([0, head_dim // 2, head_dim]))
    elif op in ("attend", "weigh"):
        case.update(items=_spread(rng, 1, 16), window=rng.choice([0, 0, 0, _spread(rng, 1, 4096)]))
        if rng.random() < 0.5:
            case.update(queries=1, context=_spread(rng, 1, 2000 if single else 16384))
        else:
            case.update(queries=_spread(rng, 2, 64 if single else 512))
            case.update(context=case["queries"] + _spread(rng, 1, 800 if single else 3000), items=rng.randint(1, 2))
        if op == "weigh":
            case["cache"] = rng.choice(["fp4", case["dtype"]])
    else:
        context = _spread(rng, 2, 20000)
        keep = _spread(rng, 1, context)
        case.update(cache=rng.choice(["fp4", case["dtype"]]), items=_spread(rng, 1, 8), context=context, keep=keep,
                    recent=rng.randint(0, keep))
    return case


def _lengths(case, seed):
    """(new tokens, tokens with them) of every request of an attend, weigh or evict case: the first as long
    as the case says, the others between half and all of that.  The sizes are the case's own, not the seed's."""
    r = random.Random("%s %s" % (case["context"], case["items"]))
    context = [case["context"]] + [r.randint(max(1, case["context"] // 2), case["context"]) for _ in range(case["items"] - 1)]
    queries = case.get("queries", 1)
    fresh = [queries] + [r.randint(1, queries) for _ in range(case["items"] - 1)]
    return [min(q, c) for q, c in zip(fresh, context)], context


def _store_places(case):
    r = random.Random("%s %s" % (case["tokens"], case["items"]))
    cuts = sorted(r.sample(range(1, case["tokens"]), case["items"] - 1)) if case["items"] > 1 else []
    fresh = [b - a for a, b in zip([0] + cuts, cuts + [case["tokens"]])]
    return fresh, [r.randint(0, 4096) for _ in fresh]


def _pairs(case):
    """(row, visible key) pairs of one head."""
    q, c = _lengths(case, 0)
    w, total = case.get("window", 0), 0
    for n, m in zip(q, c):
        seen = range(m - n + 1, m + 1)
        total += sum(min(s, w) for s in seen) if w else sum(seen)
    return total


def _read_keys(case):
    """Cached tokens that some row of the step sees."""
    q, c = _lengths(case, 0)
    w = case.get("window", 0)
    return sum(min(m, w + n - 1) if w else m for n, m in zip(q, c))


def work(case):
    es = 4 if case["dtype"] == "float32" else 2
    d, h, kv, page = case["head_dim"], case["heads"], case["kv_heads"], case["page"]
    row = {"fp4": d * 17 // 32, "float32": d * 4, "bfloat16": d * 2}[case.get("cache", "fp4")]
    if case["op"] == "store":
        t = case["tokens"]
        fresh, start = _store_places(case)
        touched = sum((s + n - 1) // page - s // page + 1 for n, s in zip(fresh, start))
        moved = t * (h + 2 * kv) * d * es + t * (h + kv) * d * es * (case["rotary_dim"] > 0) + t * 2 * kv * row
        return {"bytes": moved + t * case["rotary_dim"] * 4 + touched * 2 * kv * page * (row + d * es),
                "flops": 3 * t * (h + kv) * case["rotary_dim"] + 8 * t * 2 * kv * d}
    if case["op"] == "evict":
        _, context = _lengths(case, 0)
        kept = sum(min(case["keep"], n) for n in context)
        moved = sum(context) * kv * 4 + kept * kv * (4 + 4 + 2 * 2 * row)
        if case["cache"] == "fp4":      # and the new pages are read back
            pages = case["items"] * -(-case["keep"] // page)
            moved += pages * 2 * kv * page * (row + d * es)
        return {"bytes": moved, "flops": 2 * sum(context) * kv}
    tokens, keys = sum(_lengths(case, 0)[0]), _read_keys(case)
    if case["op"] == "attend":
        return {"bytes": tokens * h * (2 * d * es + 4) + keys * kv * 2 * row, "flops": 4 * d * h * _pairs(case)}
    return {"bytes": tokens * h * (d * es + 4) + keys * kv * (row + 8), "flops": (2 * d + 2) * h * _pairs(case)}


# ---------------------------------------------------------------------------------------------- inputs
def _random(gen, *shape, scale=1.0):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32) * scale


def _kv_values(gen, pages, kv_heads, page, d, dtype):
    """Keys and values as a model's are: a few dims much larger than the others, no two tokens alike."""
    loud = torch.exp(_random(gen, 2, kv_heads, 1, d, scale=0.7))
    return (_random(gen, pages, 2, kv_heads, page, d) * loud).to(dtype)


def _quantise(x):
    """``[..., d]`` in float32 -> (codes uint8 [..., d], factors uint8 [..., d / 32])."""
    groups = x.float().reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    top = groups.abs().amax(-1)
    mantissa, exponent = torch.frexp(top)                   # top = mantissa * 2 ** exponent, mantissa in [0.5, 1)
    e = torch.where(mantissa <= 0.875, exponent - 3, exponent - 2)
    e = torch.where(top > 0, e, -125).clamp(-125, 125)
    y = torch.ldexp(groups.abs(), -e.unsqueeze(-1))
    code = ((y > 0.25).to(torch.uint8) + (y >= 0.75).to(torch.uint8) + (y > 1.25).to(torch.uint8)
            + (y >= 1.75).to(torch.uint8) + (y > 2.5).to(torch.uint8) + (y >= 3.5).to(torch.uint8) + (y > 5.0).to(torch.uint8))
    code = code + torch.signbit(groups).to(torch.uint8) * 8
    return code.reshape(x.shape), (e + 127).to(torch.uint8)


def _lay_out_fp4(codes, factors):
    """codes ``[pages, 2, kv, page, d]``, factors ``[pages, 2, kv, page, G]`` -> the cache's bytes."""
    pages, _, kv, page, d = codes.shape
    G = d // 32
    two = codes[..., 0::2] + codes[..., 1::2] * 16
    k = two[:, 0].reshape(pages, kv, page, G, 16).permute(0, 1, 3, 2, 4).reshape(pages, kv, -1)
    v = two[:, 1].reshape(pages, kv, page // 8, 8, G, 16).permute(0, 1, 2, 5, 4, 3).reshape(pages, kv, -1)
    ks = factors[:, 0].permute(0, 1, 3, 2).reshape(pages, kv, -1)
    vs = factors[:, 1].reshape(pages, kv, page // 8, 8, G).permute(0, 1, 2, 4, 3).reshape(pages, kv, -1)
    out = torch.stack([torch.cat([k, ks], -1), torch.cat([v, vs], -1)], 1)
    return out.reshape(pages, 2, kv, page, d * 17 // 32).contiguous()


def _lay_out(x):
    """``[pages, 2, kv, page, d]`` -> the same bytes in the order of the engine's own cache."""
    pages, _, kv, page, d = x.shape
    k = x[:, 0].reshape(pages, kv, page, d // 8, 8).permute(0, 1, 3, 2, 4).reshape(pages, kv, page, d)
    v = x[:, 1].reshape(pages, kv, page // 8, 8, d).permute(0, 1, 2, 4, 3).reshape(pages, kv, page, d)
    return torch.stack([k, v], 1).contiguous()


def _cache(gen, pages, case, kind, dtype):
    """Made in parts, so that the largest cache does not exist in float32 as a whole."""
    parts = []
    for first in range(0, pages, 2048):
        x = _kv_values(gen, min(2048, pages - first), case["kv_heads"], case["page"], case["head_dim"], dtype)
        parts.append(_lay_out_fp4(*_quantise(x)) if kind == "fp4" else _lay_out(x))
    return torch.cat(parts)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = getattr(torch, case["dtype"])
    h, kv, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    dev = dict(device="cuda", dtype=torch.int32)
    s = {"case": dict(case), "dtype": dtype, "kernels": {}}
    kind = case.get("cache", "fp4")
    if case["op"] == "store":
        fresh, start = _store_places(case)
        need = [-(-(a + n) // page) for n, a in zip(fresh, start)]
        pages = sum(need) + 3
        order = torch.randperm(pages, generator=gen, device="cuda", dtype=torch.int64).to(torch.int32).tolist()
        slots, touched, at = [], [], 0
        for n, a, m in zip(fresh, start, need):
            mine = order[at:at + m]
            at += m
            slots += [mine[p // page] * page + p % page for p in range(a, a + n)]
            touched += mine[a // page:]
        s["qkv"] = _random(gen, case["tokens"], (h + 2 * kv) * d).to(dtype)
        s["cache"] = _cache(gen, pages, case, "fp4", dtype)
        s["slots"], s["touched"] = torch.tensor(slots, **dev), torch.tensor(touched, **dev)
        s["positions"] = torch.tensor([p for n, a in zip(fresh, start) for p in range(a, a + n)], **dev)
        turned = case["rotary_dim"]
        if turned:
            rate = 10000.0 ** (-torch.arange(0, turned, 2, device="cuda", dtype=torch.float64) / turned)
            angle = torch.arange(max(a + n for n, a in zip(fresh, start)), device="cuda", dtype=torch.float64)[:, None] * rate
            s["angles"] = torch.cat([angle.cos(), angle.sin()], -1).float()
        # the pages read back, in the engine's own order and type
        s["read"] = torch.empty(len(touched), 2, kv, page, d, dtype=dtype, device="cuda")
        return s
    fresh, context = _lengths(case, seed)
    need = [-(-n // page) for n in context]
    evict = case["op"] == "evict"
    new = -(-case["keep"] // page) if evict else 0
    pages = sum(need) + new * len(context) + 2
    order = torch.randperm(pages, generator=gen, device="cuda", dtype=torch.int64).tolist()
    table, at = [], 0
    for m in need:
        table.append(order[at:at + m] + [-1] * (max(need) - m))
        at += m
    s["cache"] = _cache(gen, pages, case, kind, dtype)
    s["table"] = torch.tensor(table, **dev)
    s["context"] = torch.tensor(context, **dev)
    if evict:
        # most tokens get little, a few a lot, some nothing at all (their order decides then)
        w = torch.exp(_random(gen, pages, kv, page, scale=2.0))
        s["weights"] = w * (torch.rand(w.shape, generator=gen, device="cuda") > 0.3)
        s["new_table"] = torch.tensor([order[at + i * new:at + (i + 1) * new] for i in range(len(context))], **dev)
        s["new_pages"] = s["new_table"].reshape(-1).contiguous()
        s["kept"] = torch.empty(len(context), kv, case["keep"], **dev)
        s["longest"] = max(context)
        if kind == "fp4":
            s["read"] = torch.empty(new * len(context), 2, kv, page, d, dtype=dtype, device="cuda")
        return s
    tokens = sum(fresh)
    s["q"] = _random(gen, tokens, h, d, scale=0.5).to(dtype)
    row = [i for i, n in enumerate(fresh) for _ in range(n)]
    place = [c - n + j for n, c in zip(fresh, context) for j in range(n)]
    s["token_row"], s["positions"] = torch.tensor(row, **dev), torch.tensor(place, **dev)
    s["within"] = torch.tensor([j for n in fresh for j in range(n)], **dev)
    s["fresh"], s["longest"] = torch.tensor(fresh, **dev), max(context)
    s["most_fresh"] = max(fresh)
    starts = [sum(fresh[:i]) for i in range(len(fresh))]
    # what the engine's batch says about a step's requests; the first call adds its work list to `work`
    s["meta"] = SimpleNamespace(
        block_table=s["table"], token_row=s["token_row"], positions=s["positions"], page_size=page,
        item_q_start=starts, item_q_len=fresh, item_ctx_len=context,
        item_meta=torch.tensor([starts, fresh, context], **dev), work={})
    s["out"] = torch.empty(tokens, h * d, dtype=dtype, device="cuda")
    s["lse"] = torch.empty(tokens, h, dtype=torch.float32, device="cuda")
    if case["op"] == "weigh":
        s["lse"] = _attend(s, kind, logsum_only=True)
        s["previous"] = torch.rand(pages, kv, page, generator=gen, device="cuda") * 4
        s["weights"] = s["previous"].clone()
    return s


# ---------------------------------------------------------------------------------------------- plain forms
def _decode(raw, d):
    """4-bit pages ``[n, 2, kv, page, row]`` -> ``[n, 2, kv, page, d]`` in float32."""
    n, _, kv, page, _ = raw.shape
    G = d // 32
    flat = raw.reshape(n, 2, kv, -1)
    codes, factors = flat[..., :page * d // 2], flat[..., page * d // 2:]
    pair = torch.tensor([[(LEVELS[b & 7] * (-1 if b & 8 else 1)), (LEVELS[b >> 4 & 7] * (-1 if b & 128 else 1))]
                         for b in range(256)], dtype=torch.float32, device=raw.device)
    k = codes[:, 0].reshape(n, kv, G, page, 16).permute(0, 1, 3, 2, 4)
    v = codes[:, 1].reshape(n, kv, page // 8, 16, G, 8).permute(0, 1, 2, 5, 4, 3).reshape(n, kv, page, G, 16)
    kf = factors[:, 0].reshape(n, kv, G, page).permute(0, 1, 3, 2)
    vf = factors[:, 1].reshape(n, kv, page // 8, G, 8).permute(0, 1, 2, 4, 3).reshape(n, kv, page, G)
    values = pair[torch.stack([k, v], 1).int()].reshape(n, 2, kv, page, G, 32)
    f = torch.stack([kf, vf], 1)
    factor = torch.where(f == 255, float("nan"), torch.exp2(f.float() - 127))
    return (values * factor.unsqueeze(-1)).reshape(n, 2, kv, page, d)


def _undo_layout(x):
    """The engine's own pages ``[n, 2, kv, page, d]`` -> one token's dims side by side, in float32."""
    n, _, kv, page, d = x.shape
    k = x[:, 0].reshape(n, kv, d // 8, page, 8).permute(0, 1, 3, 2, 4).reshape(n, kv, page, d)
    v = x[:, 1].reshape(n, kv, page // 8, d, 8).permute(0, 1, 2, 4, 3).reshape(n, kv, page, d)
    return torch.stack([k, v], 1).float()


def _requests(s, kind, which):
    """Keys (0) or values (1) of all requests, ``[items, kv, longest, d]`` in float32; absent pages are page 0."""
    case = s["case"]
    items, width = s["table"].shape
    pages = s["cache"][s["table"].clamp(min=0).reshape(-1).long()]
    x = _decode(pages, case["head_dim"]) if kind == "fp4" else _undo_layout(pages)
    x = x[:, which].reshape(items, width, case["kv_heads"], case["page"], case["head_dim"])
    return x.permute(0, 2, 1, 3, 4).reshape(items, case["kv_heads"], width * case["page"], -1)[:, :, :s["longest"]].contiguous()


def _scores(s, kind):
    """Scaled scores ``[items, kv, ratio * most_fresh, longest]`` (-inf where masked), padded rows included."""
    case = s["case"]
    items, kv, d = s["table"].shape[0], case["kv_heads"], case["head_dim"]
    ratio, n = case["heads"] // kv, s["most_fresh"]
    q = torch.zeros(items, n, case["heads"], d, device="cuda")
    q[s["token_row"].long(), s["within"].long()] = s["q"].float()
    q = q.reshape(items, n, kv, ratio, d).permute(0, 2, 3, 1, 4).reshape(items, kv, ratio * n, d)
    score = torch.matmul(q, _requests(s, kind, 0).transpose(2, 3).contiguous()) * (1 / math.sqrt(d))
    key = torch.arange(s["longest"], device="cuda")
    place = (s["context"] - s["fresh"])[:, None] + torch.arange(n, device="cuda")      # [items, n]
    seen = key <= place[..., None]
    if case["window"]:
        seen &= key > place[..., None] - case["window"]
    seen &= (torch.arange(n, device="cuda") < s["fresh"][:, None])[..., None]
    return torch.where(seen[:, None, None], score.reshape(items, kv, ratio, n, -1), -math.inf)


def _rows(s, x):
    """``[items, kv, ratio, n, ...]`` -> the step's tokens ``[tokens, heads, ...]``."""
    x = x.flatten(1, 2).transpose(1, 2)
    return x[s["token_row"].long(), s["within"].long()]


def _attend(s, kind, logsum_only=False):
    score = _scores(s, kind)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    weight = torch.exp(score - top)
    total = weight.sum(-1, keepdim=True)
    lse = _rows(s, (torch.log(total) + top)[..., 0]).contiguous()
    if logsum_only:
        return lse
    items, kv, ratio, n, keys = score.shape
    del score
    out = torch.matmul(weight.reshape(items, kv, ratio * n, keys), _requests(s, kind, 1)).reshape(items, kv, ratio, n, -1)
    out = _rows(s, out / total)
    return [out.flatten(1).to(s["dtype"]), lse]


def _weigh(s, kind):
    case = s["case"]
    score = _scores(s, kind)
    items, kv, ratio, n, keys = score.shape
    lse = torch.full((items, n, case["heads"]), math.inf, device="cuda")
    lse[s["token_row"].long(), s["within"].long()] = s["lse"]
    lse = lse.reshape(items, n, kv, ratio).permute(0, 2, 3, 1)
    gathered = torch.exp(score - lse[..., None]).sum((2, 3))                 # [items, kv, keys]
    key = torch.arange(keys, device="cuda")
    there = key < s["context"][:, None]
    page = s["table"].clamp(min=0).long()[:, key // case["page"]]
    before = s["previous"][page, :, key % case["page"]].permute(0, 2, 1)     # [items, kv, keys]
    older = key < (s["context"] - s["fresh"])[:, None]
    total = torch.where(older[:, None], before, 0.0) + gathered
    item, at = there.nonzero(as_tuple=True)
    s["weights"][page[item, at], :, at % case["page"]] = total[item, :, at]
    return s["weights"]


def _store(s):
    case = s["case"]
    h, kv, d, page, turned = case["heads"], case["kv_heads"], case["head_dim"], case["page"], case["rotary_dim"]
    x = s["qkv"].reshape(case["tokens"], h + 2 * kv, d)
    if turned:
        angles = s["angles"][s["positions"].long()][:, None]
        cos, sin = angles[..., :turned // 2], angles[..., turned // 2:]
        a, b = x[:, :h + kv, :turned // 2].float(), x[:, :h + kv, turned // 2:turned].float()
        x = torch.cat([torch.cat([(a * cos - b * sin).to(s["dtype"]), (b * cos + a * sin).to(s["dtype"]),
                                  x[:, :h + kv, turned:]], -1), x[:, h + kv:]], 1)
    codes, factors = _quantise(x[:, h:].reshape(-1, 2, kv, d))
    which = s["touched"].long()
    place = torch.full((s["cache"].shape[0],), -1, dtype=torch.int64, device="cuda")
    place[which] = torch.arange(which.numel(), device="cuda")
    values = _decode(s["cache"][which], d)
    slot = s["slots"].long()
    level = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device="cuda")[codes.int()].reshape(*factors.shape, 32)
    values[place[slot // page], :, :, slot % page] = (level * torch.exp2(factors.float() - 127).unsqueeze(-1)).reshape(codes.shape)
    return [x.reshape(case["tokens"], -1), _lay_out(values.to(s["dtype"]))]


def _evict(s, kind):
    case = s["case"]
    page, keep, kv, d = case["page"], case["keep"], case["kv_heads"], case["head_dim"]
    items = s["table"].shape[0]
    key = torch.arange(s["longest"], device="cuda")
    at_page = s["table"].clamp(min=0).long()[:, key // page]                 # [items, longest]
    weight = s["weights"][at_page, :, key % page].permute(0, 2, 1)           # [items, kv, longest]
    length = s["context"][:, None, None]
    ranked = torch.where(key >= length - case["recent"], math.inf, weight)
    ranked = torch.where(key < length, ranked, -1.0)
    kept = torch.sort(ranked, dim=-1, descending=True, stable=True).indices[..., :keep]
    kept = torch.nn.functional.pad(kept, (0, keep - kept.shape[-1]), value=s["longest"])
    kept = torch.where(kept < length, kept, 1 << 30)
    kept = torch.sort(kept, dim=-1).values
    item, head, to = (kept < (1 << 30)).nonzero(as_tuple=True)
    source = kept[item, head, to]
    kept = torch.where(kept < (1 << 30), kept, -1).int()
    from_page, from_at = at_page[item, source], source % page
    to_page, to_at = s["new_table"].long()[item, to // page], to % page
    s["weights"][to_page, head, to_at] = s["weights"][from_page, head, from_at]
    new = s["new_pages"].long()
    place = torch.full((s["cache"].shape[0],), -1, dtype=torch.int64, device="cuda")
    place[new] = torch.arange(new.numel(), device="cuda")
    x = _decode(s["cache"], d) if kind == "fp4" else _undo_layout(s["cache"])
    moved = x[new]
    moved[place[to_page], :, head, to_at] = x[from_page, :, head, from_at]
    moved = _lay_out(moved.to(s["dtype"]))
    if kind == "fp4":
        return [kept, s["weights"], moved]
    s["cache"][new] = moved
    return [kept, s["weights"], s["cache"]]


def run(state):
    case, kind = state["case"], state["case"].get("cache", "fp4")
    if not own:
        if case["op"] == "store":
            return _store(state)
        if case["op"] == "attend":
            return _attend(state, kind)
        if case["op"] == "weigh":
            return _weigh(state, kind)
        return _evict(state, kind)
    kernels = state["kernels"].get("hip")
    if kernels is None:
        from sparseengine_amd.kernels.hip_ops import HipKernels
        kernels = state["kernels"]["hip"] = HipKernels()
    s = state
    scale = 1 / math.sqrt(case["head_dim"])
    if case["op"] == "store":
        qkv = s["qkv"].clone()      # the call turns q and k in place
        kernels.qk_norm_rope_store(qkv, s["positions"], s.get("angles"), None, None, 1e-6, case["heads"], case["kv_heads"],
                                   case["head_dim"], case["rotary_dim"], s["cache"], s["slots"], case["page"])
        kernels.unpack_cache(s["cache"], s["touched"], s["read"])
        return [qkv, s["read"]]
    if case["op"] == "attend":
        kernels.paged_attention(s["q"], s["cache"], s["meta"], s["out"], scale, case["window"], lse=s["lse"])
        return [s["out"], s["lse"]]
    if case["op"] == "weigh":
        kernels.attention_weights(s["q"], s["cache"], s["meta"], s["lse"], s["weights"], scale, case["window"],
                                  previous=s["previous"])
        return s["weights"]
    kernels.evict_tokens(s["cache"], s["weights"], s["table"], s["context"], s["new_table"], case["keep"],
                         case["recent"], s["kept"], longest=s["longest"])
    if kind == "fp4":
        kernels.unpack_cache(s["cache"], s["new_pages"], s["read"])
        return [s["kept"], s["weights"], s["read"]]
    return [s["kept"], s["weights"], s["cache"]]


# ---------------------------------------------------------------------------------------------- the definition in 64 bits
def _value_of(raw, page, d, which, off):
    """The numbers of one token of 4-bit pages ``[n, kv, page * row]``, read byte by byte, in float64."""
    G = d // 32
    dim = torch.arange(d, device=raw.device)
    byte, group = dim % 32 // 2, dim // 32
    off = off[:, None]
    if which == 0:
        code_at = (group * page + off) * 16 + byte
        factor_at = page * d // 2 + group * page + off
    else:
        code_at = ((off // 8 * 16 + byte) * G + group) * 8 + off % 8
        factor_at = page * d // 2 + (off // 8 * G + group) * 8 + off % 8
    take = lambda at: torch.gather(raw, 2, at[:, None].expand(-1, raw.shape[1], -1)).long()
    two, f = take(code_at), take(factor_at)
    code = torch.where(dim % 2 == 0, two % 16, two // 16)
    size = code % 8
    # 0, then one bit of mantissa and two of exponent
    number = torch.where(size < 2, size * 0.5, (1 + 0.5 * (size % 2).double()) * torch.pow(2.0, (size // 2 - 1).double()))
    number = torch.where(code >= 8, -number.double(), number.double()) * torch.pow(torch.tensor(2.0, dtype=torch.float64, device=raw.device), (f - 127).double())
    return torch.where(f == 255, float("nan"), number)


def _tokens_of(cache, table_row, length, case, kind, which):
    """Keys or values of one request, ``[kv, length, d]`` in float64."""
    page, d, kv = case["page"], case["head_dim"], case["kv_heads"]
    parts = []
    for first in range(0, length, 16384):
        at = torch.arange(first, min(first + 16384, length), device=cache.device)
        pages = table_row.long()[at // page]
        off = at % page
        if kind == "fp4":
            held, inverse = torch.unique(pages, return_inverse=True)
            raw = cache[held][:, which].reshape(held.numel(), kv, -1)[inverse] if at.numel() <= 256 else None
            if raw is not None:
                parts.append(_value_of(raw, page, d, which, off).transpose(0, 1))
                continue
            # whole pages at a time: the same reading for every place of a page
            raw = cache[held][:, which].reshape(held.numel(), kv, -1)
            every = [_value_of(raw, page, d, which, torch.full((held.numel(),), o, device=cache.device)) for o in range(page)]
            parts.append(torch.stack(every, 1)[inverse, off].transpose(0, 1))
        else:
            x = cache[pages][:, which].reshape(at.numel(), kv, -1).double()
            dim = torch.arange(d, device=cache.device)
            o = off[:, None]
            place = (dim // 8 * page + o) * 8 + dim % 8 if which == 0 else (o // 8 * d + dim) * 8 + o % 8
            parts.append(torch.gather(x, 2, place[:, None].expand(-1, kv, -1)).transpose(0, 1))
    return torch.cat(parts, 1)


def _nearest(x):
    """float64 ``[..., d]`` -> the numbers that 4 bits hold in its place."""
    g = x.reshape(*x.shape[:-1], -1, 32)
    top = g.abs().amax(-1, keepdim=True)
    e = torch.full_like(top, -125.0)
    # the smallest power of two from 2 ** -125 with top <= 7 * it
    safe = torch.where(top > 0, top, 1.0)
    low = torch.floor(torch.log2(safe / 7.0)) - 1
    for more in (0, 1, 2, 3):
        fits = safe <= 7.0 * torch.pow(2.0, low + more)
        e = torch.where(fits & (e == -125.0) & (top > 0), (low + more).clamp(-125, 125), e)
    unit = torch.pow(2.0, e)
    y = g.abs() / unit
    levels = torch.tensor(LEVELS, dtype=torch.float64, device=x.device)
    far = (y.unsqueeze(-1) - levels).abs()
    best = far.amin(-1, keepdim=True)
    tie = far == best
    index = torch.arange(8, device=x.device)
    even = torch.where(tie & (index % 2 == 0), index, -1).amax(-1)
    first = torch.where(tie, index, 8).amin(-1)
    chosen = torch.where(tie.sum(-1) > 1, even, first)
    return (torch.copysign(levels[chosen], g) * unit).reshape(x.shape)


def _own_order(x):
    """float64 ``[pages, 2, kv, page, d]`` -> the order of the engine's own pages."""
    return _lay_out(x)


def exact(case, seed):
    s = prepare(case, seed)
    kind, h, kv, d, page = case.get("cache", "fp4"), case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    ratio = h // kv
    if case["op"] == "store":
        x = s["qkv"].double().reshape(case["tokens"], h + 2 * kv, d)
        turned, half = case["rotary_dim"], case["rotary_dim"] // 2
        if turned:
            t = s["angles"][s["positions"].long()].double()[:, None]
            y = x.clone()
            for j in range(half):
                c, w = t[..., j], t[..., half + j]
                y[:, :h + kv, j] = x[:, :h + kv, j] * c - x[:, :h + kv, half + j] * w
                y[:, :h + kv, half + j] = x[:, :h + kv, half + j] * c + x[:, :h + kv, j] * w
            x = y
        stands = x[:, h:].to(s["dtype"]).double().reshape(-1, 2, kv, d)       # 4 bits are made of what qkv holds
        held = torch.stack([torch.stack([_value_of(s["cache"][s["touched"].long()][:, w].reshape(-1, kv, page * (d * 17 // 32)),
                                                   page, d, w, torch.full((s["touched"].numel(),), o, device="cuda"))
                                         for o in range(page)], 2) for w in (0, 1)], 1)     # [n, 2, kv, page, d]
        where = {int(p): i for i, p in enumerate(s["touched"].tolist())}
        slots = s["slots"].tolist()
        row = torch.tensor([where[p // page] for p in slots], device="cuda")
        new = torch.empty_like(stands)
        for first in range(0, len(slots), 1024):
            new[first:first + 1024] = _nearest(stands[first:first + 1024])
        held[row, :, :, s["slots"].long() % page] = new
        return [x.reshape(case["tokens"], -1), _own_order(held)]
    if case["op"] == "evict":
        kept = torch.full((case["items"], kv, case["keep"]), -1, dtype=torch.int32, device="cuda")
        weights, context = s["weights"].double(), s["context"].tolist()
        new = s["new_pages"].long()
        moved = torch.stack([_tokens_of(s["cache"], p.reshape(1), page, case, kind, w) for p in new for w in (0, 1)])
        moved = moved.reshape(new.numel(), 2, kv, page, d)
        per = s["new_table"].shape[1]
        for i, n in enumerate(context):
            at = torch.arange(n, device="cuda")
            keys, values = (_tokens_of(s["cache"], s["table"][i], n, case, kind, w) for w in (0, 1))
            mine = s["weights"].double()[s["table"][i].long()[at // page], :, at % page]      # [n, kv]
            m = min(case["keep"], n)
            for g in range(kv):
                order = sorted(range(n - min(case["recent"], n)), key=mine[:n - min(case["recent"], n), g].cpu().numpy().__neg__().__getitem__)
                late = list(range(n - min(case["recent"], n), n))[-m:] if case["recent"] else []
                chosen = torch.tensor(sorted(order[:m - len(late)] + late), device="cuda", dtype=torch.int64)
                kept[i, g, :m] = chosen.int()
                to = torch.arange(m, device="cuda")
                weights[s["new_table"][i].long()[to // page], g, to % page] = mine[chosen, g]
                moved[i * per + to // page, 0, g, to % page] = keys[g, chosen]
                moved[i * per + to // page, 1, g, to % page] = values[g, chosen]
        moved = _own_order(moved)
        if kind == "fp4":
            return [kept, weights, moved]
        cache = s["cache"].double()
        cache[new] = moved
        return [kept, weights, cache]
    scale, window = 1 / math.sqrt(d), case["window"]
    out = torch.empty(s["q"].shape[0], h, d, dtype=torch.float64, device="cuda")
    lse = torch.empty(s["q"].shape[0], h, dtype=torch.float64, device="cuda")
    weights = s["previous"].double() if case["op"] == "weigh" else None
    begin = 0
    for i, (n, m) in enumerate(zip(s["fresh"].tolist(), s["context"].tolist())):
        keys = _tokens_of(s["cache"], s["table"][i], m, case, kind, 0)
        values = _tokens_of(s["cache"], s["table"][i], m, case, kind, 1) if weights is None else None
        place, key = torch.arange(m - n, m, device="cuda")[:, None], torch.arange(m, device="cuda")
        hidden = key > place
        if window:
            hidden |= key <= place - window
        gathered = torch.zeros(kv, m, dtype=torch.float64, device="cuda")
        for head in range(h):
            q = s["q"][begin:begin + n, head].double()
            score = (q @ keys[head // ratio].t()) * scale
            score[hidden] = -math.inf
            if weights is None:
                norm = torch.logsumexp(score, -1)
                lse[begin:begin + n, head] = norm
                out[begin:begin + n, head] = torch.exp(score - norm[:, None]) @ values[head // ratio]
            else:
                gathered[head // ratio] += torch.exp(score - s["lse"][begin:begin + n, head].double()[:, None]).sum(0)
        begin += n
        if weights is not None:
            where = (s["table"][i].long()[key // page], key % page)
            before = weights[where[0], :, where[1]].t().clone()
            before[:, m - n:] = 0
            weights[where[0], :, where[1]] = (before + gathered).t()
    return weights if weights is not None else [out.flatten(1), lse]
