"""The bodies of tests/test_gpu_compact_edges.py on the CPU: the kernel sources built for the host, every tensor argument
next to an inaccessible page."""
import pytest
import torch

import tests.test_gpu_compact_edges as G
from tests import backends
from tests.test_emu_compact_cache import Emulated

pytestmark = pytest.mark.skipif(not backends.EmulatedBackend().available(), reason="no host compiler for the emulated kernels")


@pytest.fixture(params=["after", "before"])
def guard(request):
    return request.param


@pytest.mark.parametrize("case", G.WIDE_WINDOWS)
def test_weights_under_a_window_as_long_as_everything(guard, case):
    with Emulated(guard=guard) as hip:
        for kind in ("fp4", "own"):
            G.test_weights_under_a_window_as_long_as_everything(hip, kind, case)


def test_windows_that_32_bits_do_not_hold():
    with Emulated() as hip:
        for kind in ("fp4", "own"):
            G.test_windows_that_32_bits_do_not_hold(hip, kind)


def test_weights_refuse_a_scale_that_is_not_positive():
    with Emulated() as hip:
        for kind in ("fp4", "own"):
            for dtype in (G.BF16, G.F32):
                G.test_weights_refuse_a_scale_that_is_not_positive(hip, kind, dtype)


@pytest.mark.parametrize("dtype,d", [(G.BF16, 64), (G.BF16, 96), (G.F32, 64)])
def test_kept_work_lists_belong_to_their_lengths(guard, dtype, d):
    with Emulated(guard=guard) as hip:
        G.test_kept_work_lists_belong_to_their_lengths(hip, dtype, d)


@pytest.mark.parametrize("d,items", [(128, 20), (256, 6), (128, 130), (256, 130)])
def test_joining_ranges(d, items):
    with Emulated() as hip:
        G.test_joining_ranges(hip, d, items)


@pytest.mark.parametrize("case", [(6, 1, 128, 64, [300, 33, 1], [1, 1, 1], 0), (8, 2, 64, 32, [300, 90], [1, 3], 0), (4, 1, 256, 32, [200], [2], 0),
                                  (6, 1, 128, 32, [200, 60], [1, 5], 50)])
def test_probabilities_keep_what_their_rounding_leaves(case):
    with Emulated() as hip:
        G.test_probabilities_keep_what_their_rounding_leaves(hip, *case)
