"""Calls of the cache in 4 bits, of gathered weights and of eviction at the ends of what their arguments may be, against the
plain forms of tests/compact_oracle.py (tolerances: tests/test_gpu_compact_cache.py)."""
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
