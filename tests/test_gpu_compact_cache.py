"""The cache in 4 bits (store, unpack, attention), the attention weight a key gathers, and eviction by it, against plain
forms in 64 bits (tests/compact_oracle.py).

Tolerances.  A rounding to a type is off by at most eps / 2 of the value, bfloat16 2^-8 and float32 2^-24.  What 4 bits
hold is compared exactly.  Attention in bfloat16 rounds every probability once before the value product and the
result once: |error| <= 2^-8 sum p |v| + 2^-8 |o|, beside what float32 does to scores and sums, which is the whole
error in float32: a score is a sum of D products, off by at most (D + 8) 2^-24 sum |q| |k| scale, and a relative error
of that size goes into its exponential; the sums over n keys add n 2^-24; exponential and logarithm a few 2^-24 of
their arguments."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from sparseengine_amd.cache import layout
from sparseengine_amd.kernels import hip_ops
from sparseengine_amd.kernels.hip_ops import KernelShapeError
from tests import backends
from tests import compact_oracle as oracle

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16]
DEV = "cuda"


@pytest.fixture(autouse=True)
def _device():
    global DEV
    DEV = backends.ACTIVE.device


@pytest.fixture
def hip():
    return backends.ACTIVE.kernels()


def emulator_skips(work: float, limit: float = 6e7):
    """Products of one (row, key) pair and head that the emulated backend goes through one thread at a time."""
    if backends.ACTIVE.slow and work > limit:
        pytest.skip("too large for the emulated backend")


def randn(*shape, dtype, scale=1.0, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def make_layer(kind, pages, kv, page, d, seed, dtype):
    """(a layer of random numbers on the device, which(0 keys / 1 values) -> float64 ``[pages, kv, page, d]``).  ``kind``
    fp4, or the engine's own type."""
    g = torch.Generator().manual_seed(seed)
    loud = torch.exp(torch.randn(2, kv, 1, d, generator=g))
    x = torch.randn(pages, 2, kv, page, d, generator=g) * loud
    page_at = torch.arange(pages).repeat_interleave(page)
    off_at = torch.arange(page).repeat(pages)
    tokens = lambda w: x[:, w].permute(0, 2, 1, 3).reshape(pages * page, kv, d)
    if kind == "fp4":
        cache = torch.zeros(pages, 2, kv, page, layout.fp4_row_bytes(d), dtype=torch.uint8)
        for w in (0, 1):
            layout.fp4_write(cache, w, page_at, off_at, tokens(w))
        read = lambda w: layout.fp4_read(cache, w, page_at, off_at, torch.float64)
    else:
        cache = torch.zeros(pages, 2, kv, page, d, dtype=dtype)
        layout.write_keys(cache, page_at, off_at, tokens(0).to(dtype))
        layout.write_values(cache, page_at, off_at, tokens(1).to(dtype))
        read = lambda w: (layout.read_keys, layout.read_values)[w](cache, page_at, off_at).double()
    return cache, lambda w: read(w).reshape(pages, page, kv, d)


def spoil(cache, meta, ctx_lens, page, kind):
    """Pages that no table names and slots past a request's last key hold what is not a number."""
    named = torch.zeros(cache.shape[0], dtype=torch.bool)
    table = meta.block_table.cpu()
    for item, n in enumerate(ctx_lens):
        held = table[item, :-(-n // page)]
        named[held[held >= 0].long()] = True
        beyond = torch.arange(n % page, page) if n % page else torch.arange(0)
        if beyond.numel():
            last = torch.full_like(beyond, int(held[-1]))
            if kind == "fp4":
                for w in (0, 1):
                    layout.fp4_write(cache, w, last, beyond, torch.full((beyond.numel(), cache.shape[2], cache.shape[4] * 32 // 17), float("nan")))
            else:
                nan = torch.full((beyond.numel(), cache.shape[2], cache.shape[4]), float("nan"), dtype=cache.dtype)
                layout.write_keys(cache, last, beyond, nan)
                layout.write_values(cache, last, beyond, nan)
    cache[~named] = 255 if kind == "fp4" else float("nan")


def tokens_of(layer, meta, item, n, page):
    """A request's first ``n`` tokens ``[n, kv, d]`` from ``[pages, page, kv, d]``; pages given back read as zeros."""
    table = meta.block_table[item].cpu().long()
    at = torch.arange(n)
    pages = table[at // page]
    x = layer[pages.clamp(min=0), at % page]
    x[pages < 0] = 0
    return x


# ---------------------------------------------------------------------------------------------- store and unpack
STORE = [  # tokens, heads, kv_heads, head_dim, page, rotary, pairing, norm
    (1, 4, 2, 64, 32, 32, "neox", None),
    (5, 6, 2, 128, 64, 64, "neox", "flat"),
    (19, 2, 1, 96, 32, 0, "neox", None),
    (7, 3, 3, 32, 96, 32, "interleaved", "per_head"),
    (40, 4, 1, 256, 32, 128, "neox", "flat"),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,heads,kv,d,page,rotary,pairing,norm", STORE)
def test_store_holds_what_qkv_holds(hip, dtype, tokens, heads, kv, d, page, rotary, pairing, norm):
    """The 4 bits are those of the k and v that stand in ``qkv`` afterwards, which is turned and normed as without a
    cache; skipped slots and every other byte stay."""
    rng = np.random.default_rng(tokens)
    qkv = randn(tokens, (heads + 2 * kv) * d, dtype=dtype, seed=1)
    qkv[:, heads * d:] *= torch.exp(2 * torch.randn(2 * kv * d, generator=torch.Generator().manual_seed(3)))[None].to(dtype)
    positions = torch.arange(tokens, dtype=torch.int32) * 3
    angle = torch.rand(3 * tokens, rotary // 2, generator=torch.Generator().manual_seed(2)) * 6
    table = torch.cat([angle.cos(), angle.sin()], -1).to(DEV) if rotary else None
    widths = (heads * d, kv * d) if norm == "flat" else (d, d)
    w = [None, None] if norm is None else [(1 + 0.1 * randn(n, dtype=torch.float32, seed=4)).to(dtype).to(DEV) for n in widths]
    pages = -(-tokens // page) + 2
    slots = torch.tensor(rng.permutation(pages * page)[:tokens], dtype=torch.int32)
    if tokens > 3:
        slots[2] = -1
    before = torch.randint(0, 256, (pages, 2, kv, page, layout.fp4_row_bytes(d)), dtype=torch.uint8, generator=torch.Generator().manual_seed(5))
    cache = before.clone().to(DEV)
    got, plain = qkv.clone().to(DEV), qkv.clone().to(DEV)
    kwargs = dict(pairing=pairing, per_head_norm=norm == "per_head")
    hip.qk_norm_rope_store(got, positions.to(DEV), table, *w, 1e-5, heads, kv, d, rotary, cache, slots.to(DEV), page, **kwargs)
    hip.qk_norm_rope_store(plain, positions.to(DEV), table, *w, 1e-5, heads, kv, d, rotary, None, None, page, **kwargs)
    assert torch.equal(got, plain)
    keep = slots >= 0
    where = slots[keep].long()
    stands = got.cpu()[keep, heads * d:].reshape(-1, 2, kv, d)
    after, expected = cache.cpu(), before.clone()
    for which in (0, 1):
        layout.fp4_write(expected, which, where // page, where % page, stands[:, which])
        held = oracle.held(stands[:, which])
        for i, slot in enumerate(where.tolist()[:4]):
            for h in range(kv):
                assert oracle.token_of(after, slot // page, which, h, slot % page, d) == held[i, h].tolist()
    assert torch.equal(after, expected)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,heads,kv,d,page,rotary,norm", [(3, 48, 8, 128, 64, 64, "flat"), (40, 3, 1, 64, 32, 64, None),
                                                                (130, 6, 3, 96, 32, 16, "flat"), (600, 2, 1, 32, 64, 32, None)])
def test_store_in_one_kernel_and_in_two(hip, monkeypatch, dtype, tokens, heads, kv, d, page, rotary, norm):
    """The rotation's kernel that writes 4 bits itself leaves the bytes that a kernel of its own reads back and writes,
    also for elements that are not finite."""
    emulator_skips(tokens * (heads + 2 * kv) * d, 1e6)
    rng = np.random.default_rng(tokens)
    qkv = randn(tokens, (heads + 2 * kv) * d, dtype=dtype, seed=1)
    qkv[:, heads * d:] *= torch.exp(2 * torch.randn(2 * kv * d, generator=torch.Generator().manual_seed(3)))[None].to(dtype)
    qkv[0, -1], qkv[1, -d], qkv[tokens - 1, heads * d + 1] = float("nan"), float("inf"), -float("inf")
    angle = torch.rand(tokens, rotary // 2, generator=torch.Generator().manual_seed(2)) * 6
    table = torch.cat([angle.cos(), angle.sin()], -1).to(DEV)
    w = [None, None] if norm is None else [(1 + 0.1 * randn(n * d, dtype=torch.float32, seed=4)).to(dtype).to(DEV) for n in (heads, kv)]
    pages = -(-tokens // page) + 1
    slots = torch.tensor(rng.permutation(pages * page)[:tokens], dtype=torch.int32)
    slots[2] = -1
    slots, positions = slots.to(DEV), torch.arange(tokens, dtype=torch.int32).to(DEV)
    ways = []
    for ours in (hip, type("TwoKernels", (type(hip),), dict(_writes_fp4=lambda self, *a: False))()):
        rows, cache = qkv.clone().to(DEV), torch.full((pages, 2, kv, page, layout.fp4_row_bytes(d)), 77, dtype=torch.uint8).to(DEV)
        if ours is not hip:
            monkeypatch.setattr(hip_ops, "_SHORT_WAYS", False)
        ours.qk_norm_rope_store(rows, positions, table, *w, 1e-5, heads, kv, d, rotary, cache, slots, page)
        ways.append((rows.cpu().view(torch.uint8), cache.cpu()))
    assert torch.equal(ways[0][0], ways[1][0]) and torch.equal(ways[0][1], ways[1][1])
    assert (ways[0][1] == 255).any()


def test_store_borders(hip):
    """Ties, the factor's borders, the ends of the range and what is not finite, exactly."""
    d, page = 64, 32
    edges = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 0.0, -0.0, -0.25, -5.0]
    rows = []
    for unit in (1.0, 2.0 ** 20, 2.0 ** -100, 2.0 ** -125, 2.0 ** -126, 2.0 ** 125):
        rows.append([v * unit for v in edges] + [0.0] * 19)
        rows.append([np.nextafter(np.float32(v), np.float32(9)) * unit for v in edges] + [0.0] * 19)
    rows += [[7.0] + [1.0] * 31, [np.nextafter(np.float32(7), np.float32(9))] + [1.0] * 31, [1e-45] * 32, [3.4028235e38] * 32,
             [float("inf")] + [1.0] * 31, [float("nan")] + [1.0] * 31, [0.0] * 32, [-float("inf")] * 32]
    x = torch.tensor(np.asarray(rows, dtype=np.float32))
    x = torch.nan_to_num(x, nan=float("nan"), posinf=float("inf"), neginf=-float("inf"))
    tokens = x.shape[0]
    qkv = torch.cat([torch.zeros(tokens, d), x.repeat(1, 2), x.repeat(1, 2)], 1)      # one head; k = v = the row twice
    cache = torch.zeros(2, 2, 1, page, layout.fp4_row_bytes(d), dtype=torch.uint8).to(DEV)
    slots = torch.arange(tokens, dtype=torch.int32).to(DEV)
    hip.qk_norm_rope_store(qkv.to(DEV), slots, None, None, None, 1e-6, 1, 1, d, 0, cache, slots, page)
    read = torch.empty(2, 2, 1, page, d).to(DEV)
    hip.unpack_cache(cache, torch.arange(2, dtype=torch.int32).to(DEV), read)
    held = oracle.held(x).repeat(1, 2)
    for i in range(tokens):
        for which in (0, 1):
            mine = (layout.read_keys, layout.read_values)[which](read.cpu(), torch.tensor([i // page]), torch.tensor([i % page]))[0, 0].double()
            raw = torch.tensor(oracle.token_of(cache.cpu(), i // page, which, 0, i % page, d), dtype=torch.float64)
            for seen in (mine, raw):
                assert torch.equal(torch.isnan(seen), torch.isnan(held[i]))
                assert torch.equal(torch.nan_to_num(seen), torch.nan_to_num(held[i])), (i, which, rows[i][:13])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kv,d,page", [(1, 32, 32), (3, 96, 64), (2, 128, 96), (2, 256, 32), (1, 512, 32)])
def test_unpack(hip, dtype, kv, d, page):
    cache, numbers = make_layer("fp4", 5, kv, page, d, 7, dtype)
    cache[1, 0, 0, -1] = 255      # a factor byte among others: whole groups that are not numbers
    pages = torch.tensor([3, 1, -1, 3], dtype=torch.int32)
    out = torch.full((4, 2, kv, page, d), 7.0, dtype=dtype).to(DEV)
    hip.unpack_cache(cache.to(DEV), pages.to(DEV), out)
    out = out.cpu()
    assert (out[2] == 7).all()
    every = torch.arange(page)
    for i, p in enumerate(pages.tolist()):
        if p < 0:
            continue
        at = torch.full_like(every, i)
        from_ = torch.full_like(every, p)
        for which, mine in ((0, layout.read_keys), (1, layout.read_values)):
            want = layout.fp4_read(cache, which, from_, every, torch.float64)
            got = mine(out, at, every).double()
            assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))
    assert torch.isnan(out[1].float()).any()


# ---------------------------------------------------------------------------------------------- attention
ATTEND = [  # heads, kv_heads, head_dim, page, contexts, new tokens, window
    (2, 1, 64, 32, [1], [1], 0),                           # a single key
    (6, 1, 128, 64, [1, 31, 32, 33, 64, 65], [1] * 6, 0),  # the ends of steps and pages
    (8, 2, 64, 32, [77, 5], [1, 5], 0),
    (16, 1, 128, 32, [40], [3], 0),                        # rows of several tokens in one tile
    (20, 1, 64, 64, [100, 33], [2, 1], 0),                 # more than 16 rows of one token
    (4, 4, 256, 32, [70, 1], [2, 1], 0),
    (12, 2, 128, 64, [700, 129, 64], [1, 1, 1], 0),        # split keys and a merge
    (12, 2, 128, 32, [300, 90], [1, 4], 50),               # a window: pages given back
    (2, 1, 64, 32, [200], [3], 1),                         # a window of the token itself
    (4, 2, 96, 32, [90, 20], [1, 7], 0),                   # a head size without a kernel of its own
    (4, 2, 32, 64, [65], [9], 33),
    (12, 2, 64, 32, [50, 61, 9], [40, 1, 9], 0),           # a prompt portion beside decoded tokens
    (12, 1, 128, 64, [150, 40], [70, 40], 0),
    (12, 1, 64, 32, [200, 40], [70, 1], 45),
    (16, 1, 64, 32, [600, 70], [80, 1], 0),                # rows of the same keys in several blocks
    (16, 1, 128, 32, [200], [80], 60),
]


def attention_case(kind, dtype, heads, kv, d, page, ctx, new, window, seed=0):
    rng = np.random.default_rng(seed)
    meta, pages = oracle.step(ctx, new, page, DEV, rng, window=window, stride=1)
    cache, layer = make_layer(kind, pages, kv, page, d, seed, dtype)
    numbers = (layer(0), layer(1))
    spoil(cache, meta, ctx, page, kind)
    q = randn(sum(new), heads, d, dtype=dtype, seed=seed + 1)
    of = lambda which: lambda item: tokens_of(numbers[which], meta, item, ctx[item], page)
    return meta, cache, q, of


def check_attention(out, lse, q, of, ctx, new, scale, window, dtype, visible=None):
    want, want_lse, spread, size = oracle.attention(q, of(0), of(1), ctx, new, scale, window)
    T, H, D = q.shape
    keys = max(ctx)
    relative = 2.0 ** -24 * (2 * (D + 8) * size + keys + 64)             # float32: scores, exponentials, sums
    bound = spread * (relative[..., None] + (half_step(dtype) if dtype == torch.bfloat16 else 0.0)) + half_step(dtype) * want.abs()
    error = (out.cpu().double().reshape(T, H, D) - want).abs()
    assert bool((error <= bound + 1e-30).all()), f"attention off by {float((error / (bound + 1e-30)).max()):.2f} of its bound"
    lse_error = (lse.cpu().double() - want_lse).abs()
    assert bool((lse_error <= relative + 2.0 ** -22 * want_lse.abs()).all()), float(lse_error.max())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv,d,page,ctx,new,window", ATTEND)
def test_attention_in_4_bits(hip, dtype, heads, kv, d, page, ctx, new, window):
    emulator_skips(sum(c * n for c, n in zip(ctx, new)) * heads * d)
    meta, cache, q, of = attention_case("fp4", dtype, heads, kv, d, page, ctx, new, window)
    out = torch.full((sum(new), heads * d), 9.0, dtype=dtype).to(DEV)
    lse = torch.full((sum(new), heads), 9.0).to(DEV)
    hip.paged_attention(q.to(DEV), cache.to(DEV), meta, out, d ** -0.5, window, lse=lse)
    check_attention(out, lse, q, of, ctx, new, d ** -0.5, window, dtype)
    again = torch.empty_like(out)
    hip.paged_attention(q.to(DEV), cache.to(DEV), meta, again, d ** -0.5, window)
    assert torch.equal(out, again)


@pytest.mark.parametrize("heads,kv,d,page,ctx,new,window", ATTEND[11:])
def test_attention_of_many_rows_in_unpacked_blocks(hip, monkeypatch, heads, kv, d, page, ctx, new, window):
    """Portions that the step's size alone would leave to the 4-bit kernel."""
    from sparseengine_amd.kernels import attention_work
    monkeypatch.setattr(attention_work, "FP4_BLOCK_WORK", 0)
    test_attention_in_4_bits(hip, torch.bfloat16, heads, kv, d, page, ctx, new, window)
    assert attention_work.build_fp4_attention_work(new, ctx, heads // kv, kv, window, d).block_units.size


@pytest.mark.parametrize("new,ctx", [([1, 170], [300, 4200]), ([700], [700]), ([200, 3, 40], [1200, 40, 5000]),
                                     ([90, 1], [9000, 20000]), ([1] * 70, list(range(400, 1100, 10)))])      # many rows to join
def test_portions_around_the_choice_of_a_kernel(hip, new, ctx):
    heads, kv, d, page = 12, 2, 64, 64
    emulator_skips(sum(c * n for c, n in zip(ctx, new)) * heads * d)
    meta, cache, q, of = attention_case("fp4", torch.bfloat16, heads, kv, d, page, ctx, new, 0)
    out, lse = torch.empty(sum(new), heads * d, dtype=torch.bfloat16).to(DEV), torch.empty(sum(new), heads).to(DEV)
    hip.paged_attention(q.to(DEV), cache.to(DEV), meta, out, d ** -0.5, lse=lse)
    check_attention(out, lse, q, of, ctx, new, d ** -0.5, 0, torch.bfloat16)


def test_a_step_without_tokens(hip):
    heads, kv, d, page, bf16 = 4, 2, 64, 32, torch.bfloat16
    cache = torch.zeros(2, 2, kv, page, layout.fp4_row_bytes(d), dtype=torch.uint8).to(DEV)
    i32 = lambda *shape: torch.zeros(*shape, dtype=torch.int32).to(DEV)
    meta = SimpleNamespace(block_table=i32(0, 1), token_row=i32(0), positions=i32(0), page_size=page, item_q_len=np.zeros(0, dtype=np.int32),
                           item_ctx_len=np.zeros(0, dtype=np.int32), item_meta=i32(3, 0), work={})
    qkv = torch.zeros(0, (heads + 2 * kv) * d, dtype=bf16).to(DEV)
    out, lse, weights = torch.zeros(0, heads * d, dtype=bf16).to(DEV), torch.zeros(0, heads).to(DEV), torch.ones(2, kv, page).to(DEV)
    hip.qk_norm_rope_store(qkv, i32(0), None, None, None, 1e-6, heads, kv, d, 0, cache, i32(0), page)
    hip.paged_attention(qkv[:, :heads * d].view(0, heads, d), cache, meta, out, 0.125, lse=lse)
    hip.attention_weights(qkv[:, :heads * d].view(0, heads, d), cache, meta, lse, weights, 0.125)
    hip.evict_tokens(cache, weights, i32(0, 1), i32(0), i32(0, 1), 5, 1, i32(0, kv, 5), longest=0)
    hip.unpack_cache(cache, i32(0), torch.zeros(0, 2, kv, page, d, dtype=bf16).to(DEV))
    assert not cache.any() and (weights == 1).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv,d,page,ctx,new,window", [ATTEND[i] for i in (1, 2, 6, 7, 11, 13)])
def test_logsum_of_the_engines_own_cache(hip, dtype, heads, kv, d, page, ctx, new, window):
    emulator_skips(sum(c * n for c, n in zip(ctx, new)) * heads * d)
    meta, cache, q, of = attention_case("own", dtype, heads, kv, d, page, ctx, new, window)
    out, plain = (torch.empty(sum(new), heads * d, dtype=dtype).to(DEV) for _ in range(2))
    lse = torch.full((sum(new), heads), 9.0).to(DEV)
    hip.paged_attention(q.to(DEV), cache.to(DEV), meta, plain, d ** -0.5, window)
    hip.paged_attention(q.to(DEV), cache.to(DEV), meta, out, d ** -0.5, window, lse=lse)
    assert torch.equal(out, plain)
    check_attention(out, lse, q, of, ctx, new, d ** -0.5, window, dtype)


def test_attention_strided_q_and_out(hip):
    """q as a view of a wider row, out as columns of one."""
    heads, kv, d, page, ctx, new = 4, 2, 64, 32, [50, 9], [2, 1]
    meta, cache, q, of = attention_case("fp4", torch.bfloat16, heads, kv, d, page, ctx, new, 0)
    wide = torch.full((3, heads * d + 128), float("nan"), dtype=torch.bfloat16)
    wide[:, 64:64 + heads * d] = q.reshape(3, -1)
    wide = wide.to(DEV)
    q_view = wide[:, 64:64 + heads * d].view(3, heads, d)
    out = torch.full((3, heads * d + 64), 9.0, dtype=torch.bfloat16).to(DEV)
    lse = torch.empty(3, heads).to(DEV)
    hip.paged_attention(q_view, cache.to(DEV), meta, out[:, :heads * d], d ** -0.5, lse=lse)
    check_attention(out[:, :heads * d], lse, q, of, ctx, new, d ** -0.5, 0, torch.bfloat16)
    assert (out[:, heads * d:] == 9).all()


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_token_that_is_not_a_number_is_seen_by_its_readers_only(hip, d, which):
    """Key or value of the step's third token are not numbers: rows of earlier tokens do not notice."""
    heads, kv, page, ctx, new = 3, 1, 32, [45], [5]
    meta, cache, q, of = attention_case("fp4", torch.bfloat16, heads, kv, d, page, ctx, new, 0)
    bad = 42
    layout.fp4_write(cache, which, meta.block_table[0, bad // page].cpu().long().reshape(1), torch.tensor([bad % page]),
                     torch.full((1, kv, d), float("nan")))
    out, lse = torch.empty(5, heads * d, dtype=torch.bfloat16).to(DEV), torch.empty(5, heads).to(DEV)
    hip.paged_attention(q.to(DEV), cache.to(DEV), meta, out, d ** -0.5, lse=lse)
    check_attention(out[:2], lse[:2], q[:2], lambda w: lambda i: of(w)(i)[:42], [42], [2], d ** -0.5, 0, torch.bfloat16)
    assert torch.isnan(out[2:]).all()
    assert torch.isnan(lse[2:]).all() if which == 0 else torch.isfinite(lse).all()


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("dtype,d,new,window", [(torch.bfloat16, 128, 90, 0), (torch.bfloat16, 64, 90, 20), (torch.bfloat16, 96, 90, 0),
                                                (torch.bfloat16, 160, 5, 0), (torch.float32, 64, 20, 0), (torch.bfloat16, 288, 5, 0)])
def test_a_token_that_is_not_a_number_in_unpacked_pages(hip, monkeypatch, dtype, d, new, window, which):
    """The same where attention reads unpacked pages: rows before the token, and those whose window has passed it, are as
    if it were any other; its readers are not numbers, at least in the dims of its group."""
    from sparseengine_amd.kernels import attention_work
    monkeypatch.setattr(attention_work, "FP4_BLOCK_WORK", 0)
    heads, kv, page, ctx, scale = 6, 2, 32, [130], d ** -0.5
    bad, head, group = 130 - new + 3, 1, 1           # the step's fourth token, one kv head, dims 32 to 63
    meta, cache, q, of = attention_case("fp4", dtype, heads, kv, d, page, ctx, [new], window)
    place = [meta.block_table[0, bad // page].cpu().long().reshape(1), torch.tensor([bad % page])]
    held = layout.fp4_read(cache, which, *place)
    held[0, head, 32 * group] = float("nan")
    layout.fp4_write(cache, which, *place, held)
    out, lse = torch.empty(new, heads * d, dtype=dtype).to(DEV), torch.empty(new, heads).to(DEV)
    hip.paged_attention(q.to(DEV), cache.to(DEV), meta, out, scale, window, lse=lse)
    pos = torch.arange(130 - new, 130)
    sees = (pos >= bad) & (pos - window < bad if window else True)
    readers = sees[:, None] & (torch.arange(heads) // (heads // kv) == head)[None, :]
    out, lse = out.cpu().reshape(new, heads, d), lse.cpu()
    assert torch.isnan(out[readers][:, 32 * group:32 * group + 32]).all()
    want, want_lse, spread, size = oracle.attention(q, of(0), of(1), ctx, [new], scale, window)      # the token as it was before
    bound = spread * (2.0 ** -24 * (2 * (d + 8) * size + 130 + 64)[..., None] + half_step(dtype)) + half_step(dtype) * want.abs()
    assert bool(((out.double() - want).abs() <= bound + 1e-30)[~readers].all())
    assert bool(((lse.double() - want_lse).abs() <= 2.0 ** -24 * (2 * (d + 8) * size + 130 + 64) + 2.0 ** -22 * want_lse.abs())[~readers].all())


# ---------------------------------------------------------------------------------------------- gathered weights
@pytest.mark.parametrize("kind", ["fp4", "own"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv,d,page,ctx,new,window", ATTEND)
def test_weights_of_the_cached_keys(hip, dtype, kind, heads, kv, d, page, ctx, new, window):
    emulator_skips(sum(c * n for c, n in zip(ctx, new)) * heads * d)
    meta, cache, q, of = attention_case(kind, dtype, heads, kv, d, page, ctx, new, window)
    scale = d ** -0.5
    lse = oracle.attention(q, of(0), of(1), ctx, new, scale, window)[1].float()
    pages = cache.shape[0]
    before = torch.rand(pages, kv, page, generator=torch.Generator().manual_seed(1)) * 3
    table = meta.block_table.cpu().long()

    def previous_of(item):
        at = torch.arange(ctx[item])
        return before[table[item][at // page].clamp(min=0), :, at % page].t().clone()
    results = oracle.weights(q, of(0), lse, previous_of, ctx, new, scale, window)
    out = torch.full((pages, kv, page), 9.0).to(DEV)
    hip.attention_weights(q.to(DEV), cache.to(DEV), meta, lse.to(DEV), out, scale, window, previous=before.to(DEV))
    in_place = before.clone().to(DEV)
    hip.attention_weights(q.to(DEV), cache.to(DEV), meta, lse.to(DEV), in_place, scale, window, previous=in_place)
    fresh = torch.full((pages, kv, page), 9.0).to(DEV)
    hip.attention_weights(q.to(DEV), cache.to(DEV), meta, lse.to(DEV), fresh, scale, window)
    out, in_place, fresh = out.cpu(), in_place.cpu(), fresh.cpu()
    touched = torch.zeros(pages, page, dtype=torch.bool)
    for item, (total, bound) in enumerate(results):
        first = max(0, ctx[item] - new[item] - window + 1) if window else 0
        at = torch.arange(first, ctx[item])
        where = (table[item][at // page], slice(None), at % page)
        error = (out[where].t().double() - total[:, first:]).abs()
        assert bool((error <= bound[:, first:] + 1e-30).all()), float((error / (bound[:, first:] + 1e-30)).max())
        assert torch.equal(in_place[where], out[where])
        gathered = total[:, first:].clone()
        older = ctx[item] - new[item] - first
        gathered[:, :older] -= previous_of(item).double()[:, first:first + older]
        assert bool(((fresh[where].t().double() - gathered).abs() <= bound[:, first:] + 1e-30).all())
        touched[where[0], where[2]] = True
    assert (out.permute(0, 2, 1)[~touched] == 9).all() and (fresh.permute(0, 2, 1)[~touched] == 9).all()


# ---------------------------------------------------------------------------------------------- eviction
EVICT = [  # kv_heads, head_dim, page, lengths, keep, recent
    (1, 32, 32, [1], 1, 0),
    (2, 64, 32, [40, 33, 7], 33, 8),
    (1, 128, 64, [200, 129], 64, 0),
    (3, 96, 32, [100], 40, 40),
    (2, 64, 32, [65, 64, 63, 31], 64, 1),
    (1, 64, 96, [1500, 700], 100, 13),       # more than one round of the block
    (2, 32, 64, [5000, 4097], 4000, 100),    # more than a thread's registers at the first size
    (1, 32, 128, [60000, 20000, 49153], 5000, 0),    # more than the largest size holds
]


def evict_case(kind, dtype, kv, d, page, lengths, keep, seed=0):
    rng = np.random.default_rng(seed)
    meta, pages = oracle.step(lengths, [1] * len(lengths), page, DEV, rng, stride=1)
    new = -(-keep // page)
    total = pages + new * len(lengths)
    cache, layer = make_layer(kind, total, kv, page, d, seed, dtype)
    g = torch.Generator().manual_seed(seed)
    weights = torch.rand(total, kv, page, generator=g)
    weights = torch.where(torch.rand(weights.shape, generator=g) < 0.3, torch.zeros(()), (weights * 64).round() / 64)   # many ties
    new_table = torch.arange(pages, total, dtype=torch.int32).flip(0).reshape(len(lengths), new)
    return meta, cache, layer, weights, new_table


@pytest.mark.parametrize("kind", ["fp4", "own"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kv,d,page,lengths,keep,recent", EVICT)
def test_eviction(hip, dtype, kind, kv, d, page, lengths, keep, recent):
    emulator_skips(sum(lengths) * kv * 1e4, 1e8)
    meta, cache, layer, weights, new_table = evict_case(kind, dtype, kv, d, page, lengths, keep)
    if kind == "own" and dtype == torch.float32:      # any float has a place in the order
        weights[0, 0, :4] = torch.tensor([float("inf"), float("nan"), -0.0, -1.0])
    got, got_w = cache.clone().to(DEV), weights.clone().to(DEV)
    items = len(lengths)
    kept = torch.full((items, kv, keep), 7, dtype=torch.int32).to(DEV)
    hip.evict_tokens(got, got_w, meta.block_table, torch.tensor(lengths, dtype=torch.int32).to(DEV), new_table.to(DEV), keep,
                     recent, kept, longest=max(lengths))
    got, got_w, kept = got.cpu(), got_w.cpu(), kept.cpu()
    expected, expected_w = cache.clone(), weights.clone()
    table = meta.block_table.cpu().long()
    read = (layout.read_keys, layout.read_values)
    for item, n in enumerate(lengths):
        at = torch.arange(n)
        mine = weights[table[item][at // page], :, at % page]                     # [n, kv]
        for h in range(kv):
            stay = oracle.chosen(mine[:, h].tolist(), n, keep, recent)
            assert kept[item, h].tolist() == stay + [-1] * (keep - len(stay)), (item, h)
            src, to = torch.tensor(stay), torch.arange(len(stay))
            from_page, to_page = table[item][src // page], new_table[item].long()[to // page]
            assert torch.equal(torch.nan_to_num(got_w[to_page, h, to % page], nan=-7.0), torch.nan_to_num(weights[from_page, h, src % page], nan=-7.0))
            for which in (0, 1):
                if kind == "fp4":
                    a = layout.fp4_read(got, which, to_page, to % page)[:, h]
                    b = layout.fp4_read(cache, which, from_page, src % page)[:, h]
                else:
                    a, b = read[which](got, to_page, to % page)[:, h], read[which](cache, from_page, src % page)[:, h]
                assert torch.equal(a, b), (item, h, which)
    # nothing but the kept tokens' new places has changed
    old = torch.ones(cache.shape[0], dtype=torch.bool)
    old[new_table.reshape(-1).long()] = False
    same = lambda a, b: torch.equal(a.flatten().view(torch.uint8), b.flatten().view(torch.uint8))
    assert same(got[old], cache[old]) and same(got_w[old], weights[old])
    for item, n in enumerate(lengths):
        behind = torch.arange(min(n, keep), new_table.shape[1] * page)
        if behind.numel() == 0:
            continue
        where = new_table[item].long()[behind // page]
        assert same(got_w[where, :, behind % page], weights[where, :, behind % page])
        for which in (0, 1):
            if kind == "fp4":
                assert torch.equal(layout.fp4_read(got, which, where, behind % page), layout.fp4_read(cache, which, where, behind % page))
            else:
                assert torch.equal(read[which](got, where, behind % page), read[which](cache, where, behind % page))


def test_eviction_of_equal_weights_keeps_the_first(hip):
    meta, cache, layer, weights, new_table = evict_case("own", torch.float32, 1, 32, 32, [90], 40)
    weights.fill_(0.5)
    kept = torch.empty(1, 1, 40, dtype=torch.int32).to(DEV)
    hip.evict_tokens(cache.to(DEV), weights.to(DEV), meta.block_table, torch.tensor([90], dtype=torch.int32).to(DEV),
                     new_table.to(DEV), 40, 5, kept, longest=90)
    assert kept.cpu().flatten().tolist() == list(range(35)) + list(range(85, 90))


@pytest.mark.parametrize("kind", ["fp4", "own"])
def test_eviction_from_a_table_with_pages_given_back(hip, kind):
    """Tokens whose page is gone go first; where too few others are left, a new place of one stays as it was."""
    kv, d, page, length, recent = 2, 64, 32, 200, 8
    for keep in (100, 180):                 # 40 + 96 + 64 tokens, the 64 of two middle pages gone: 136 are left
        meta, cache, layer, weights, new_table = evict_case(kind, torch.bfloat16, kv, d, page, [length], keep)
        table = meta.block_table.clone()
        table[0, 1] = table[0, 4] = -1
        gone = (torch.arange(length) // page == 1) | (torch.arange(length) // page == 4)
        got, got_w = cache.clone().to(DEV), weights.clone().to(DEV)
        kept = torch.empty(1, kv, keep, dtype=torch.int32).to(DEV)
        hip.evict_tokens(got, got_w, table, torch.tensor([length], dtype=torch.int32).to(DEV), new_table.to(DEV), keep, recent, kept,
                         longest=length)
        at, held = torch.arange(length), table.cpu().long()[0].clamp(min=0)
        for h in range(kv):
            w = weights[held[at // page], h, at % page].clone()
            w[gone] = float("-inf")          # below every weight of the case
            stay = oracle.chosen(w.tolist(), length, keep, recent)
            assert kept.cpu()[0, h].tolist() == stay
            for to, i in enumerate(stay):
                where = (new_table[0, to // page].long(), h, to % page)
                expected = weights[where] if gone[i] else weights[held[i // page], h, i % page]
                assert got_w.cpu()[where] == expected


# ---------------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_request_in_4_bits_from_store_to_eviction(hip, dtype):
    """Tokens are stored, attended to, weighed and evicted, and attention over what is left is that over the kept
    tokens: the operators one after the other, as a sparse method runs them."""
    heads, kv, d, page, n, keep, recent = 6, 2, 64, 32, 70, 40, 8
    rng = np.random.default_rng(5)
    meta, pages = oracle.step([n], [n], page, DEV, rng)
    new_pages = -(-keep // page)
    cache = torch.zeros(pages + new_pages, 2, kv, page, layout.fp4_row_bytes(d), dtype=torch.uint8).to(DEV)
    weights = torch.zeros(pages + new_pages, kv, page).to(DEV)
    qkv = randn(n, (heads + 2 * kv) * d, dtype=dtype, seed=6).to(DEV)
    at = torch.arange(n)
    slots = (meta.block_table[0].cpu()[at // page] * page + at % page).int().to(DEV)
    hip.qk_norm_rope_store(qkv, slots, None, None, None, 1e-6, heads, kv, d, 0, cache, slots, page)
    q = qkv[:, :heads * d].view(n, heads, d)
    out, lse = torch.empty(n, heads * d, dtype=dtype).to(DEV), torch.empty(n, heads).to(DEV)
    hip.paged_attention(q, cache, meta, out, d ** -0.5, lse=lse)
    k, v = (oracle.held(qkv.cpu()[:, heads * d:].reshape(n, 2, kv, d)[:, w]) for w in (0, 1))
    check_attention(out, lse, q.cpu(), lambda w: lambda i: (k, v)[w], [n], [n], d ** -0.5, 0, dtype)
    hip.attention_weights(q, cache, meta, lse, weights, d ** -0.5)
    total = weights.cpu()[meta.block_table[0].cpu().long()[at // page], :, at % page]
    assert abs(float(total.sum()) - n * heads) <= 1e-3 * n * heads      # every row gives away 1
    new_table = torch.arange(pages, pages + new_pages, dtype=torch.int32).reshape(1, -1).to(DEV)
    kept = torch.empty(1, kv, keep, dtype=torch.int32).to(DEV)
    hip.evict_tokens(cache, weights, meta.block_table, torch.tensor([n], dtype=torch.int32).to(DEV), new_table, keep, recent,
                     kept, longest=n)
    stay = [oracle.chosen(total[:, h].tolist(), n, keep, recent) for h in range(kv)]
    assert kept.cpu()[0].tolist() == stay
    left = [torch.stack([x[stay[h], h] for h in range(kv)], 1) for x in (k, v)]
    after = oracle.step([keep], [1], page, DEV, rng)[0]
    after.block_table = new_table
    out1, lse1 = torch.empty(1, heads * d, dtype=dtype).to(DEV), torch.empty(1, heads).to(DEV)
    hip.paged_attention(q[-1:], cache, after, out1, d ** -0.5, lse=lse1)
    check_attention(out1, lse1, q.cpu()[-1:], lambda w: lambda i: left[w], [keep], [1], d ** -0.5, 0, dtype)


@pytest.mark.skipif(backends.ACTIVE.name != "hip", reason="graphs and streams are the GPU's")
@pytest.mark.parametrize("graphs", [1, 2])
def test_a_captured_step_on_another_stream(hip, graphs):
    """Store, attention, weights and eviction recorded into graphs on a stream of their own, replayed in turn on new
    numbers: each replay gives what eager calls give, whichever ran between."""
    heads, kv, d, page, ctx, keep, bf16 = 12, 2, 64, 32, [200, 37, 700], 30, torch.bfloat16
    scale, items, span = d ** -0.5, len(ctx), 96       # a portion of 96 tokens beside single ones: the unpacked way too

    class Step:
        def __init__(self, seed):
            new = [1, 1, span] if seed % 2 else [1, 1, 1]
            rng = np.random.default_rng(seed)
            self.meta, self.pages = oracle.step(ctx, new, page, DEV, rng)
            fresh = -(-keep // page)
            total = self.pages + fresh * items
            self.cache, _ = make_layer("fp4", total, kv, page, d, seed, bf16)
            self.cache = self.cache.to(DEV)
            self.qkv = torch.zeros(sum(new), (heads + 2 * kv) * d, dtype=bf16).to(DEV)
            table = self.meta.block_table.cpu()
            slots = [table[i, p // page] * page + p % page for i in range(items) for p in range(ctx[i] - new[i], ctx[i])]
            self.slots = torch.tensor([int(x) for x in slots], dtype=torch.int32).to(DEV)
            angle = torch.rand(max(ctx), d // 4) * 6
            self.angles = torch.cat([angle.cos(), angle.sin()], -1).to(DEV)
            self.out, self.lse = torch.zeros(sum(new), heads * d, dtype=bf16).to(DEV), torch.zeros(sum(new), heads).to(DEV)
            self.weights = torch.zeros(total, kv, page).to(DEV)
            self.lengths = torch.tensor(ctx, dtype=torch.int32).to(DEV)
            self.new_table = torch.arange(self.pages, total, dtype=torch.int32).reshape(items, fresh).to(DEV)
            self.kept = torch.zeros(items, kv, keep, dtype=torch.int32).to(DEV)

        def run(self):
            hip.qk_norm_rope_store(self.qkv, self.meta.positions, self.angles, None, None, 1e-6, heads, kv, d, d // 2, self.cache, self.slots, page)
            hip.paged_attention(self.qkv[:, :heads * d].view(-1, heads, d), self.cache, self.meta, self.out, scale, lse=self.lse)
            hip.attention_weights(self.qkv[:, :heads * d].view(-1, heads, d), self.cache, self.meta, self.lse, self.weights, scale)
            hip.evict_tokens(self.cache, self.weights, self.meta.block_table, self.lengths, self.new_table, keep, 4, self.kept, longest=max(ctx))

        def results(self):
            return [t.clone().cpu() for t in (self.qkv, self.out, self.lse, self.weights, self.kept, self.cache)]

    steps = [Step(seed) for seed in range(1, 1 + graphs)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    recorded = []
    with torch.cuda.stream(stream):
        for s in steps:
            s.run()
    stream.synchronize()
    for s in steps:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            s.run()
        recorded.append(graph)
    for turn in range(3):
        given = [randn(*s.qkv.shape, dtype=bf16, seed=10 * turn + i) for i, s in enumerate(steps)]
        wanted = []
        for s, x in zip(steps, given):      # eager, on the default stream
            start = s.cache.clone()
            s.qkv.copy_(x)
            s.weights.zero_()
            s.run()
            wanted.append(s.results())
            s.cache.copy_(start)
        torch.cuda.synchronize()
        for s, x in zip(steps, given):
            s.qkv.copy_(x)
            s.weights.zero_()
            s.kept.zero_()
        torch.cuda.synchronize()
        for graph in recorded:
            graph.replay()
        torch.cuda.synchronize()
        for s, want in zip(steps, wanted):
            for got, expected in zip(s.results(), want):
                assert torch.equal(got.flatten().view(torch.uint8), expected.flatten().view(torch.uint8)), turn


# ---------------------------------------------------------------------------------------------- refusals
def test_refusals(hip):
    bf16 = torch.bfloat16
    meta, cache, q, of = attention_case("fp4", bf16, 4, 2, 64, 32, [50], [1], 0)
    cache, q = cache.to(DEV), q.to(DEV)
    pages = cache.shape[0]
    out, lse = torch.empty(1, 256, dtype=bf16).to(DEV), torch.empty(1, 4).to(DEV)
    attend = lambda **k: hip.paged_attention(**{**dict(q=q, cache=cache, meta=meta, out=out, scale=0.125, lse=lse), **k})
    attend()
    for bad, error in ((dict(cache=cache[..., :33].contiguous()), ValueError), (dict(scale=0.0), ValueError), (dict(scale=-1.0), ValueError),
                       (dict(lse=lse[:, :2]), ValueError), (dict(lse=lse.double()), ValueError),
                       (dict(cache=cache[:, :, :, :16].contiguous()), KernelShapeError), (dict(q=q.half()), ValueError),
                       (dict(out=out.float()), ValueError)):
        with pytest.raises(error):
            attend(**bad)
    with pytest.raises(ValueError):
        nothing = type(meta)(**{**vars(meta), "item_q_len": None})
        attend(meta=nothing)
    w = torch.zeros(pages, 2, 32).to(DEV)
    weigh = lambda **k: hip.attention_weights(**{**dict(q=q, cache=cache, meta=meta, lse=lse, out=w, scale=0.125), **k})
    weigh()
    for bad in (dict(out=w[:, :1]), dict(out=w.double()), dict(previous=w[:1]), dict(lse=lse[:, :3].contiguous()), dict(q=q.float().half())):
        with pytest.raises(ValueError):
            weigh(**bad)
    wrong = type(meta)(**{**vars(meta), "item_q_len": np.asarray([2])})
    with pytest.raises(ValueError):
        weigh(meta=wrong)
    for items in (dict(item_q_len=np.asarray([2])), dict(item_q_len=np.asarray([0])), dict(item_ctx_len=np.asarray([65])),
                  dict(item_ctx_len=np.asarray([50, 1]))):
        with pytest.raises(ValueError):
            attend(meta=type(meta)(**{**vars(meta), "block_table": meta.block_table[:, :2].contiguous(), "work": {}, **items}))
    flat = torch.zeros(cache.numel() + 8, dtype=torch.uint8).to(DEV)
    for call in (attend, weigh):
        with pytest.raises(KernelShapeError):      # a cache that begins between multiples of 16 bytes
            call(cache=flat[8:].view(cache.shape))
    short = type(meta)(**{**vars(meta), "block_table": meta.block_table[:, :1].contiguous(), "item_ctx_len": np.asarray([50])})
    with pytest.raises(ValueError):
        weigh(meta=short)
    lengths = torch.tensor([50], dtype=torch.int32).to(DEV)
    new = torch.tensor([[2]], dtype=torch.int32).to(DEV)
    kept = torch.empty(1, 2, 20, dtype=torch.int32).to(DEV)
    evict = lambda **k: hip.evict_tokens(**{**dict(cache=cache, weights=w, block_table=meta.block_table, lengths=lengths, new_table=new,
                                                   keep=20, recent=5, kept=kept, longest=50), **k})
    for bad in (dict(keep=0), dict(recent=21), dict(recent=-1), dict(kept=kept[:, :1]), dict(new_table=new[:, :0]), dict(longest=5000),
                dict(weights=w[:, :1]), dict(lengths=lengths.long()), dict(cache=cache.to(torch.int8))):
        with pytest.raises(ValueError):
            evict(**bad)
    with pytest.raises(ValueError):
        hip.unpack_cache(cache, new.flatten(), torch.empty(1, 2, 2, 32, 96, dtype=bf16).to(DEV))
    with pytest.raises(ValueError):
        hip.unpack_cache(cache, new.flatten(), torch.empty(1, 2, 2, 32, 64, dtype=torch.float16).to(DEV))
    qkv = torch.zeros(1, 8 * 64, dtype=bf16).to(DEV)
    one = torch.zeros(1, dtype=torch.int32).to(DEV)
    with pytest.raises(ValueError):
        hip.qk_norm_rope_store(qkv, one, None, None, None, 1e-6, 4, 2, 64, 0, cache, one, 64)       # another page size
    with pytest.raises(ValueError):
        hip.qk_norm_rope_store(qkv, one, None, None, None, 1e-6, 4, 2, 64, 0, cache, one.long(), 32)
