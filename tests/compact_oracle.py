"""Plain forms, in 64 bits and one token at a time where that is simplest, of what the cache in 4 bits and the
eviction of tokens do; they share no code with the package but the description of where a byte lies."""
from __future__ import annotations

import math
from types import SimpleNamespace

import numpy as np
import torch

LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def nearest_group(x):
    """32 numbers -> (codes, factor byte, the numbers held)."""
    x = [float(v) for v in x]
    if not all(math.isfinite(v) for v in x):
        return None, 255, [math.nan] * 32
    top = max(abs(v) for v in x)
    e = -125
    while e < 125 and top > 7.0 * 2.0 ** e:
        e += 1
    codes = []
    for v in x:
        y = abs(v) / 2.0 ** e
        far = [abs(y - level) for level in LEVELS]
        best = [i for i in range(8) if far[i] == min(far)]
        size = best[0] if len(best) == 1 else next(i for i in best if i % 2 == 0)
        codes.append(size + (8 if math.copysign(1.0, v) < 0 else 0))
    return codes, e + 127, [math.copysign(LEVELS[c % 8], v) * 2.0 ** e for c, v in zip(codes, x)]


def held(x: torch.Tensor) -> torch.Tensor:
    """What 4 bits hold of ``[..., 32 n]``, in float64."""
    flat = x.double().reshape(-1, 32)
    return torch.tensor([nearest_group(row)[2] for row in flat.tolist()], dtype=torch.float64).reshape(x.shape)


def byte_places(which, page, head_dim, off, d):
    """(byte of the code, half of that byte, byte of the factor) of dim ``d`` of the token at ``off`` in a kv head's part."""
    G, group, j = head_dim // 32, d // 32, d % 32 // 2
    if which == 0:
        return (group * page + off) * 16 + j, d % 2, page * head_dim // 2 + group * page + off
    return (((off // 8) * 16 + j) * G + group) * 8 + off % 8, d % 2, page * head_dim // 2 + (off // 8 * G + group) * 8 + off % 8


def token_of(cache, page_id, which, head, off, head_dim):
    """One token's numbers, read byte by byte from a 4-bit layer."""
    page = cache.shape[3]
    part = cache[page_id, which, head].reshape(-1).tolist()
    out = []
    for d in range(head_dim):
        code_at, half, factor_at = byte_places(which, page, head_dim, off, d)
        code = part[code_at] >> 4 if half else part[code_at] & 15
        f = part[factor_at]
        out.append(math.nan if f == 255 else LEVELS[code % 8] * (-1 if code >= 8 else 1) * 2.0 ** (f - 127))
    return out


def fill_fp4(values: torch.Tensor) -> torch.Tensor:
    """float ``[pages, 2, kv, page, d]`` of numbers that 4 bits hold exactly or not -> a 4-bit layer, byte by byte."""
    pages, _, kv, page, d = values.shape
    out = np.zeros((pages, 2, kv, page * d * 17 // 32), dtype=np.uint8)
    x = values.double().numpy()
    for p in range(pages):
        for which in range(2):
            for h in range(kv):
                for off in range(page):
                    for group in range(d // 32):
                        codes, factor, _ = nearest_group(x[p, which, h, off, 32 * group:32 * group + 32])
                        at = byte_places(which, page, d, off, 32 * group)[2]
                        out[p, which, h, at] = factor
                        for i, code in enumerate(codes or [0] * 32):
                            code_at, half, _ = byte_places(which, page, d, off, 32 * group + i)
                            out[p, which, h, code_at] |= code << (4 * half)
    return torch.from_numpy(out).reshape(pages, 2, kv, page, d * 17 // 32)


def step(ctx_lens, q_lens, page, device, rng, spare=2, window=0, stride=0):
    """A step's pages and items as the engine's batch describes them: shuffled pages, those before a window given back
    (-1), a block table with ``stride`` more columns than it needs (their entries name no page).  Returns the meta and
    the number of pages."""
    need = [-(-n // page) for n in ctx_lens]
    total = sum(need) + spare
    order = rng.permutation(total).tolist()
    table = np.full((len(ctx_lens), max(need) + stride), -1, dtype=np.int32)
    for i, m in enumerate(need):
        first = max(0, ctx_lens[i] - q_lens[i] - window + 1) // page if window else 0
        for j in range(m):
            p = order.pop()
            if j >= first:
                table[i, j] = p
    start = np.concatenate(([0], np.cumsum(q_lens)[:-1]))
    i32 = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32).to(device)
    meta = SimpleNamespace(
        block_table=i32(table), token_row=i32([r for r, n in enumerate(q_lens) for _ in range(n)]),
        positions=i32([p for n, q in zip(ctx_lens, q_lens) for p in range(n - q, n)]), page_size=page,
        item_q_start=start, item_q_len=np.asarray(q_lens), item_ctx_len=np.asarray(ctx_lens),
        item_meta=i32(np.stack([start, q_lens, ctx_lens])), work={})
    return meta, total


def attention(q, keys_of, values_of, ctx_lens, q_lens, scale, window=0):
    """float64 over the items: (out [T, heads, d], lse [T, heads], the same sum over |values|, the largest sum of
    |q| |k| a row meets).  ``keys_of(item)``: ``[ctx, kv, d]``."""
    T, H, D = q.shape
    out, lse = torch.zeros(T, H, D, dtype=torch.float64), torch.zeros(T, H, dtype=torch.float64)
    spread, size = torch.zeros_like(out), torch.zeros_like(lse)
    t = 0
    for item, (n, m) in enumerate(zip(q_lens, ctx_lens)):
        k, v = keys_of(item).double(), values_of(item).double()
        ratio = H // k.shape[1]
        for j in range(n):
            pos = m - n + j
            first = max(0, pos - window + 1) if window else 0
            for h in range(H):
                row = q[t, h].double()
                ks, vs = k[first:pos + 1, h // ratio], v[first:pos + 1, h // ratio]
                s = ks @ row * scale
                lse[t, h] = torch.logsumexp(s, 0)
                w = torch.exp(s - lse[t, h])
                out[t, h] = w @ vs
                spread[t, h] = w @ vs.abs()
                size[t, h] = (ks.abs() @ row.abs()).max() * abs(scale)
            t += 1
    return out, lse, spread, size


def weights(q, keys_of, lse, previous_of, ctx_lens, q_lens, scale, window=0):
    """Per item float64 ``[kv, ctx]``: (what a key has gathered, an upper bound of the error that float32 may make)."""
    results, t = [], 0
    for item, (n, m) in enumerate(zip(q_lens, ctx_lens)):
        k = keys_of(item).double()
        kv, D = k.shape[1], k.shape[2]
        ratio = q.shape[1] // kv
        total, bound = torch.zeros(kv, m, dtype=torch.float64), torch.zeros(kv, m, dtype=torch.float64)
        for j in range(n):
            pos = m - n + j
            first = max(0, pos - window + 1) if window else 0
            for h in range(q.shape[1]):
                row, ks = q[t, h].double(), k[first:pos + 1, h // ratio]
                s = ks @ row * scale
                w = torch.exp(s - lse[t, h].double())
                total[h // ratio, first:pos + 1] += w
                # the dot product in float: D products and sums; then scale, difference and exponential
                off = 2.0 ** -24 * ((D + 8) * (ks.abs() @ row.abs()) * abs(scale) + 4 * (s.abs() + lse[t, h].double().abs()) + 8)
                bound[h // ratio, first:pos + 1] += w * off
            t += 1
        old = previous_of(item).double()                              # [kv, ctx]
        old[:, m - n:] = 0
        total += old
        bound += 2.0 ** -24 * (n * ratio + 2) * total.abs()          # the sum over rows, in float
        results.append((total, bound))
    return results


def chosen(weight_rows, length, keep, recent):
    """Which tokens of one (request, kv head) stay, ascending: ``weight_rows`` a list of floats."""
    if length <= keep:
        return list(range(length))
    late = list(range(length - recent, length))
    nan_first = lambda i: (0.0 if math.isnan(weight_rows[i]) else 1.0, 0.0 if math.isnan(weight_rows[i]) else -weight_rows[i], i)
    early = sorted(range(length - recent), key=nan_first)[:keep - recent]
    return sorted(early + late)
