"""The kernels of the cache in 4 bits, of gathered weights and of eviction on the CPU: the sources built for the host,
every tensor argument next to an inaccessible page (the bodies are those of tests/test_gpu_compact_cache.py, which runs
whole under ``SPARSEENGINE_AMD_TEST_BACKEND=emu pytest -m gpu``)."""
import pytest
import torch

import tests.test_gpu_compact_cache as C
from tests import backends

pytestmark = pytest.mark.skipif(not backends.EmulatedBackend().available(), reason="no host compiler for the emulated kernels")
BF16, F32 = torch.bfloat16, torch.float32


class Emulated:
    def __init__(self, **settings):
        self.backend = backends.EmulatedBackend(**settings)

    def __enter__(self):
        self.context = backends.use(self.backend)
        self.context.__enter__()
        C.DEV = "cpu"
        return self.backend.kernels()

    def __exit__(self, *exc):
        C.DEV = backends.ACTIVE.device
        return self.context.__exit__(*exc)


@pytest.fixture(params=["after", "before"])
def guard(request):
    return request.param


def test_store_and_unpack(guard):
    with Emulated(guard=guard) as hip:
        for dtype in (F32, BF16):
            for case in C.STORE:
                C.test_store_holds_what_qkv_holds(hip, dtype, *case)
            for sizes in [(1, 32, 32), (3, 96, 64), (2, 128, 96)]:
                C.test_unpack(hip, dtype, *sizes)
        C.test_store_borders(hip)


@pytest.mark.parametrize("case", range(len(C.ATTEND)))
def test_attention_and_weights(guard, case):
    if sum(c * n for c, n in zip(*C.ATTEND[case][4:6])) > 3000 and guard == "before":
        return
    with Emulated(guard=guard) as hip:
        if case < 11:
            for dtype in (F32, BF16) if case in (2, 7) else (BF16,):
                C.test_attention_in_4_bits(hip, dtype, *C.ATTEND[case])
                for kind in ("fp4", "own"):
                    C.test_weights_of_the_cached_keys(hip, dtype, kind, *C.ATTEND[case])
        elif case in (11, 13):
            C.test_attention_in_4_bits(hip, BF16, *C.ATTEND[case])
            C.test_weights_of_the_cached_keys(hip, BF16, "fp4", *C.ATTEND[case])


def test_portions_in_unpacked_blocks(guard, monkeypatch):
    with Emulated(guard=guard) as hip:
        for case in C.ATTEND[11:14]:
            C.test_attention_of_many_rows_in_unpacked_blocks(hip, monkeypatch, *case)
        C.test_a_step_without_tokens(hip)
        for which in (0, 1):
            C.test_a_token_that_is_not_a_number_in_unpacked_pages(hip, monkeypatch, BF16, 64, 90, 20, which)
            C.test_a_token_that_is_not_a_number_in_unpacked_pages(hip, monkeypatch, F32, 64, 20, 0, which)
        for kind in ("fp4", "own"):
            C.test_eviction_from_a_table_with_pages_given_back(hip, kind)


def test_which_portions_go_in_blocks():
    """The builders agree, and the rule: at least 8 tiles, and enough work in the step."""
    from sparseengine_amd.kernels import attention_work as aw
    for q, ctx, window in (([1, 40, 300], [70, 9000, 700], 0), ([64], [64], 0), ([900, 2, 30], [4000, 9, 4096], 500)):
        for block_tiles in (1, 4, 9, 1 << 30):
            a = aw.build_attention_work(q, ctx, 6, 8, window, 900, 128, 64, block_tiles)
            b = aw.build_attention_work_numpy(q, ctx, 6, 8, window, 900, 128, 64, block_tiles)
            assert all((getattr(a, f) == getattr(b, f)).all() for f in ("units", "tasks", "block_units")) and a.num_slots == b.num_slots
    blocks = lambda q, c, window=0, group=6: sorted(set(aw.build_fp4_attention_work(q, c, group, 8, window, 128).block_units[:, 0].tolist()))
    assert blocks([1, 1], [9, 100000]) == [] and blocks([128], [4096]) == [] and blocks([192], [4096]) == [0]
    assert blocks([16], [131072]) == [] and blocks([64], [32768]) == [0]
    assert blocks([512, 16, 1], [16384, 16384, 70]) == [0] and blocks([512, 32], [16384, 16384]) == [0, 1]
    assert blocks([192], [4096], window=100) == [] and blocks([512], [512]) == []
    pairs, table = aw.fp4_unpack_list([512, 16, 22], [16384, 100, 40000], 6, 128, 64, 0, True)
    assert set(pairs[:, 0].tolist()) == {0, 2} and len(pairs) == 256 + 625 and table[2, 624] == 880 and not table[1].any()


def test_eviction_and_the_operators_together(guard):
    with Emulated(guard=guard, schedule="shuffled") as hip:
        for dtype in (F32, BF16):
            for kind in ("fp4", "own"):
                for case in C.EVICT[:5]:
                    C.test_eviction(hip, dtype, kind, *case)
            C.test_a_request_in_4_bits_from_store_to_eviction(hip, dtype)
        C.test_eviction_of_equal_weights_keeps_the_first(hip)


def test_what_is_not_a_number_and_refusals(guard):
    with Emulated(guard=guard) as hip:
        for d in (64, 128, 256):
            for which in (0, 1):
                C.test_a_token_that_is_not_a_number_is_seen_by_its_readers_only(hip, d, which)
        C.test_attention_strided_q_and_out(hip)
        C.test_refusals(hip)
