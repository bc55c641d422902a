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
