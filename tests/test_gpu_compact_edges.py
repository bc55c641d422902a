"""Calls of the cache in 4 bits, of gathered weights and of eviction at the ends of what their arguments may be, against the
plain forms of tests/compact_oracle.py (tolerances: tests/test_gpu_compact_cache.py)."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

import tests.test_gpu_compact_cache as C
from tests import backends

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def _device():
    C.DEV = backends.ACTIVE.device


@pytest.fixture
def hip():
    return backends.ACTIVE.kernels()


WIDE_WINDOWS = [  # heads, kv_heads, head_dim, page, contexts, new tokens, window: no key is older than it reaches
    (6, 1, 128, 64, [70, 5], [1, 1], 2 ** 31 - 1),
    (4, 2, 64, 32, [70, 33], [1, 3], 2 ** 31 - 1),
    (4, 1, 256, 32, [70], [1], 2 ** 31 - 64),
    (4, 1, 96, 32, [70], [2], 2 ** 31 - 1),
    (12, 1, 64, 32, [90], [40], 2 ** 31 - 1),           # more than one tile of rows
    (6, 1, 128, 64, [70], [1], 70),                     # just the context
    (6, 1, 128, 64, [70], [1], 69),
]


@pytest.mark.parametrize("kind", ["fp4", "own"])
@pytest.mark.parametrize("case", WIDE_WINDOWS)
def test_weights_under_a_window_as_long_as_everything(hip, kind, case):
    C.test_weights_of_the_cached_keys(hip, BF16, kind, *case)


@pytest.mark.parametrize("kind", ["fp4", "own"])
def test_windows_that_32_bits_do_not_hold(hip, kind):
    """A window of more tokens than an int counts is none; one below 0 is refused."""
    case = (6, 1, 64, 32, [70, 5], [1, 2])
    for window in (2 ** 31, 2 ** 32 + 5):
        if kind == "fp4":
            C.test_attention_in_4_bits(hip, BF16, *case, window)
        C.test_weights_of_the_cached_keys(hip, BF16, kind, *case, window)
        C.test_weights_of_the_cached_keys(hip, F32, kind, *case, window)
    meta, cache, q, _ = C.attention_case(kind, BF16, *case, 0)
    out, lse, weights = torch.empty(3, 6 * 64, dtype=BF16), torch.zeros(3, 6), torch.zeros(cache.shape[0], 1, 32)
    cache, q, out, lse, weights = (t.to(C.DEV) for t in (cache, q, out, lse, weights))
    with pytest.raises(ValueError, match="window"):
        hip.attention_weights(q, cache, meta, lse, weights, 0.125, -1)
    if kind == "fp4":
        with pytest.raises(ValueError, match="window"):
            hip.paged_attention(q, cache, meta, out, 0.125, -1)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind", ["fp4", "own"])
def test_weights_refuse_a_scale_that_is_not_positive(hip, kind, dtype):
    """Masked scores are the lowest there are before the scale is applied: one below 0 would make them the largest."""
    meta, cache, q, _ = C.attention_case(kind, dtype, 6, 1, 64, 32, [70], [5], 0)
    weights = torch.full((cache.shape[0], 1, 32), 9.0).to(C.DEV)
    for scale in (0.0, -0.125, float("nan")):
        with pytest.raises(ValueError, match="scale"):
            hip.attention_weights(q.to(C.DEV), cache.to(C.DEV), meta, torch.zeros(5, 6).to(C.DEV), weights, scale)
    assert (weights == 9).all()


@pytest.mark.parametrize("dtype,d", [(BF16, 64), (BF16, 96), (F32, 64)])
def test_kept_work_lists_belong_to_their_lengths(hip, dtype, d):
    """The lists that a first call leaves in ``meta.work`` are those of its lengths: calls on other ones, on a table that is
    too narrow or has too few rows, are refused as they are without a list; the same lengths in another array go on."""
    ctx, new = [70, 200], [1, 3]
    meta, cache, q, of = C.attention_case("fp4", dtype, 6, 1, d, 32, ctx, new, 0)
    cache, q = cache.to(C.DEV), q.to(C.DEV)
    out, lse = torch.empty(4, 6 * d, dtype=dtype).to(C.DEV), torch.empty(4, 6).to(C.DEV)
    attend = lambda m, rows=4: hip.paged_attention(q[:rows], cache, m, out[:rows], d ** -0.5, lse=lse[:rows])
    for turn in range(2):
        attend(meta)
        C.check_attention(out, lse, q.cpu(), of, ctx, new, d ** -0.5, 0, dtype)
        with_ = lambda **k: SimpleNamespace(**{**vars(meta), **k})
        for bad in (dict(item_ctx_len=np.asarray([70, 199])), dict(item_ctx_len=np.asarray([200, 70])), dict(item_q_len=np.asarray([2, 2])),
                    dict(block_table=meta.block_table[:, :6].contiguous()), dict(block_table=meta.block_table[:1].contiguous()),
                    dict(item_q_len=np.asarray([1]), item_ctx_len=np.asarray([70]))):
            with pytest.raises(ValueError):
                attend(with_(**bad))
        with pytest.raises(ValueError):
            attend(with_(token_row=meta.token_row[:3], positions=meta.positions[:3]), 3)
        for same in (lambda a: a.copy(), list, lambda a: a.astype(np.int32)):
            attend(with_(item_q_len=same(meta.item_q_len), item_ctx_len=same(meta.item_ctx_len)))
        C.check_attention(out, lse, q.cpu(), of, ctx, new, d ** -0.5, 0, dtype)


@pytest.mark.parametrize("d,items", [(128, 20), (256, 6), (128, 130), (256, 130)])
def test_joining_ranges(hip, d, items):
    """Ranges joined by a block per row, and from 2048 rows on by a wavefront per row."""
    from sparseengine_amd.kernels import attention_work as aw
    heads, kv, page = 2, 1, 32
    ctx = [170 + 37 * i % 130 for i in range(items)]
    meta, cache, q, of = C.attention_case("fp4", BF16, heads, kv, d, page, ctx, [1] * items, 0)
    tasks = len(aw.build_fp4_attention_work([1] * items, ctx, heads // kv, kv, 0, d).tasks)
    assert tasks == items and (tasks * kv * 16 >= 2048) == (items == 130)
    out, lse = torch.empty(items, heads * d, dtype=BF16).to(C.DEV), torch.empty(items, heads).to(C.DEV)
    hip.paged_attention(q.to(C.DEV), cache.to(C.DEV), meta, out, d ** -0.5, lse=lse)
    C.check_attention(out, lse, q, of, ctx, [1] * items, d ** -0.5, 0, BF16)


@pytest.mark.skipif(backends.ACTIVE.slow, reason="more keys than the emulated backend goes through")
@pytest.mark.parametrize("d,ctx,window,previous", [(64, [300000], 0, True), (128, [150017, 150001], 0, True), (256, [290000], 0, False),
                                                   (128, [300000, 5], 280001, True)])
def test_weights_of_more_keys_than_one_round(hip, d, ctx, window, previous):
    """Single tokens on so many cached keys that a wavefront of the 4-bit kernel asks for more of them while it works (more
    than 65536 groups of 32 keys and kv heads); the plain form in float64 on the same device."""
    heads, kv, page, scale = 16, 8, 64, d ** -0.5
    assert sum(-(-(min(c, window) if window else c) // 32) for c in ctx) * kv > 65536
    meta, pages = C.oracle.step(ctx, [1] * len(ctx), page, C.DEV, np.random.default_rng(1), window=window)
    g = torch.Generator(device=C.DEV).manual_seed(2)
    cache = torch.randint(0, 256, (pages, 2, kv, page * d * 17 // 32), dtype=torch.uint8, device=C.DEV, generator=g)
    cache[..., page * d // 2:] = torch.randint(124, 128, (pages, 2, kv, page * d // 32), dtype=torch.uint8, device=C.DEV, generator=g)
    cache = cache.view(pages, 2, kv, page, -1)
    q = torch.randn(len(ctx), heads, d, device=C.DEV, generator=g).to(BF16)
    before = torch.rand(pages, kv, page, device=C.DEV, generator=g)
    want, bound = torch.full_like(before, 9.0, dtype=torch.float64), torch.zeros_like(before, dtype=torch.float64)
    lse = torch.empty(len(ctx), heads, device=C.DEV)
    for i, n in enumerate(ctx):
        first = max(0, n - window) if window else 0
        at = torch.arange(first, n, device=C.DEV)
        where = meta.block_table[i].long()[at // page]
        for h in range(kv):
            k = C.layout.fp4_read(cache[:, :, h:h + 1].contiguous(), 0, where, at % page, torch.float64)[:, 0]
            rows = q[i, 2 * h:2 * h + 2].double()
            s = (k @ rows.t()) * scale                                                # [keys, 2]
            lse[i, 2 * h:2 * h + 2] = torch.logsumexp(s, 0).float()
            mine = lse[i, 2 * h:2 * h + 2].double()
            w = torch.exp(s - mine)
            off = 2.0 ** -24 * ((d + 8) * (k.abs() @ rows.abs().t()) * scale + 4 * (s.abs() + mine.abs()) + 8)
            total = w.sum(1)
            if previous:
                total[:-1] += before[where[:-1], h, at[:-1] % page].double()
            want[where, h, at % page] = total
            bound[where, h, at % page] = (w * off).sum(1) + 2.0 ** -24 * 4 * total
    out = torch.full_like(before, 9.0)
    hip.attention_weights(q, cache, meta, lse, out, scale, window, previous=before if previous else None)
    assert bool(((out.double() - want).abs() <= bound + 1e-30).all()), float(((out.double() - want).abs() / (bound + 1e-30)).max())


@pytest.mark.parametrize("heads,kv,d,page,ctx,new,window", [
    (6, 1, 128, 64, [300, 33, 1], [1, 1, 1], 0), (8, 2, 64, 32, [700, 90], [1, 3], 0), (4, 1, 256, 32, [300], [2], 0),
    (6, 1, 128, 32, [200, 60], [1, 5], 50)])
def test_probabilities_keep_what_their_rounding_leaves(hip, heads, kv, d, page, ctx, new, window):
    """Attention read in 4 bits: a probability goes into the value product as two bfloat16, the second half a step of the
    first at most, so that its own rounding is off by 2^-16 of the probability and the result's alone by 2^-8."""
    meta, cache, q, of = C.attention_case("fp4", BF16, heads, kv, d, page, ctx, new, window)
    out, lse = torch.empty(sum(new), heads * d, dtype=BF16).to(C.DEV), torch.empty(sum(new), heads).to(C.DEV)
    hip.paged_attention(q.to(C.DEV), cache.to(C.DEV), meta, out, d ** -0.5, window, lse=lse)
    want, _, spread, size = C.oracle.attention(q, of(0), of(1), ctx, new, d ** -0.5, window)
    relative = 2.0 ** -24 * (2 * (d + 8) * size + max(ctx) + 64)
    bound = spread * (relative[..., None] + 2.0 ** -16) + C.half_step(BF16) * want.abs()
    error = (out.cpu().double().reshape(want.shape) - want).abs()
    assert bool((error <= bound + 1e-30).all()), f"off by {float((error / (bound + 1e-30)).max()):.2f} of its bound"
