"""The engine with its cache in 4 bits and with eviction, on the CPU through the kernel sources (a short version of
tests/test_gpu_compact_engine.py), and what their options refuse."""
import random

import numpy as np
import pytest
import torch

import tests.test_gpu_compact_engine as E
from sparseengine_amd import LLM, SamplingParams
from sparseengine_amd.cache.manager import CacheManager
from sparseengine_amd.cache.page_pool import OutOfPages
from sparseengine_amd.config.runtime import Config
from sparseengine_amd.engine.eviction import AccumulatedWeightMethod
from sparseengine_amd.parts.base import PagedKVRequest
from tests import backends
from tests.helpers import make_folder, random_tokens
from tests.twin_kernels import TwinKernels

emulated = pytest.mark.skipif(not backends.EmulatedBackend().available(), reason="no host compiler for the emulated kernels")


@emulated
@pytest.mark.parametrize("key,dtype,guard,lengths,new,kwargs", [
    ("C_loud", "bfloat16", "after", (33, 1), 3, {}), ("C_loud", "bfloat16", "before", (50, 1), 2, dict(blocks=True)), ("C_loud", "float32", "before", (34, 3), 2, {}),
    ("B_loud", "bfloat16", "before", (9, 35), 2, dict(max_num_batched_tokens=24))])
def test_cache_in_4_bits(tmp_path, monkeypatch, key, dtype, guard, lengths, new, kwargs):
    with backends.use(backends.EmulatedBackend(guard=guard)):
        E.check_cache_in_4_bits(tmp_path, monkeypatch, key, dtype, lengths, new, **kwargs)


@emulated
@pytest.mark.parametrize("key,dtype,guard,lengths,new,budget,recent,kwargs", [
    ("C_loud", "bfloat16", "after", (50, 20), 16, 20, 4, dict(kv_cache_dtype="fp4", max_num_batched_tokens=40)),
    ("A_loud", "float32", "before", (30, 30), 12, 17, 17, dict(kv_page_size=16, num_kvcache_slots=128, max_num_batched_tokens=16))])
def test_eviction_in_the_engine(tmp_path, key, dtype, guard, lengths, new, budget, recent, kwargs):
    with backends.use(backends.EmulatedBackend(guard=guard)):
        E.check_eviction(tmp_path, key, dtype, lengths, new, budget, recent, **kwargs)


@emulated
def test_a_budget_that_nothing_exceeds_changes_nothing(tmp_path):
    with backends.use(backends.EmulatedBackend()):
        E.check_large_budget_changes_nothing(tmp_path, "C_loud", "bfloat16", (20, 5), 3, kv_cache_dtype="fp4")


def test_options(tmp_path):
    folder = make_folder(tmp_path, "C_loud")
    make = lambda **k: Config.from_kwargs(folder, **k)
    assert make().kv_cache_dtype == "auto" and make(kv_cache_dtype="fp4").kv_page_size == 64
    for bad in (dict(kv_cache_dtype="int8"), dict(kv_cache_dtype="fp4", kv_page_size=16), dict(eviction_budget=8),
                dict(eviction_recent=2), dict(sparse_method="accumulated_weight"),
                dict(sparse_method="accumulated_weight", eviction_budget=8, eviction_recent=9)):
        with pytest.raises(ValueError):
            make(**bad)
    assert make(sparse_method="accumulated_weight", eviction_budget=9).eviction_recent == 2
    assert make(sparse_method="accumulated_weight", eviction_budget=9, eviction_recent=0).eviction_recent == 0


def manager(kv_dtype=torch.float32, window=None, head_dim=32, page=32, pages=8):
    return CacheManager({0: PagedKVRequest(2, head_dim, window, None)}, max_rows=3, max_model_len=200, page_size=page,
                        num_pages=pages, dtype=torch.float32, device="cpu", kv_dtype=kv_dtype)


def test_a_cache_of_4_bits_refuses_other_sizes():
    assert manager(torch.uint8).kv_layer(0).shape[-1] == 17      # 16 bytes of codes, one of factors
    for bad in (dict(head_dim=48), dict(page=16)):
        with pytest.raises(ValueError, match="steps of 32"):
            manager(torch.uint8, **bad)


def test_the_cache_managers_account_of_an_eviction():
    cache = manager()
    a, b = cache.admit("a"), cache.admit("b")
    cache.append([(a, 100), (b, 40)])
    with pytest.raises(OutOfPages):
        cache.begin_eviction([a, b], 33)                      # 2 + 2 fresh pages, 2 are free
    with pytest.raises(ValueError, match="holds"):
        cache.begin_eviction([b], 41)
    tables = cache.begin_eviction([a], 33)
    old = cache.groups[0].table[a, :4].tolist()
    cache.finish_eviction([a], 33, tables)
    cache.check_invariants()
    assert cache.row_len[a] == 33 and cache.row_dropped[a] == 67 and cache.groups[0].pool.free_count == 4
    assert not set(old) & set(cache.groups[0].table[a, :2].tolist())
    assert not cache.can_append([(a, 101)]) and cache.pages_needed(a, 32)[0] == 1
    with pytest.raises(ValueError, match="max_model_len"):
        cache.append([(a, 101)])                              # 67 + 33 + 101 tokens of a sequence of 200
    cache.append([(a, 100)])
    with pytest.raises(ValueError, match="max_model_len"):
        cache.append([(a, 1)])
    cache.free("a")
    assert cache.row_dropped[a] == 0
    with pytest.raises(ValueError, match="windowed"):
        manager(window=16).begin_eviction([], 4)


def test_the_method_refuses_windows_and_other_head_sizes():
    for bad in (manager(window=16), manager(head_dim=36)):
        with pytest.raises(ValueError):
            AccumulatedWeightMethod(8, 2, 4).bind(bad)
    for budget, recent in ((0, 0), (4, 5)):
        with pytest.raises(ValueError):
            AccumulatedWeightMethod(budget, recent, 4).bind(manager())
    method = AccumulatedWeightMethod(40, 2, 16)
    method.bind(manager())
    assert method.reserved_pages() == {0: 2} and method.tokens_taken(0, 500) == 40 + 32 - 1 + 16
    assert method.tokens_taken(0, 10) == 10 and method.tokens_taken(80, 300) == 16 and method.tokens_taken(80, 1) == 1
    never = AccumulatedWeightMethod(190, 2, 16)
    never.bind(manager())
    assert never.reserved_pages() == {} and np.asarray(never.weights[0].shape).tolist() == [8, 2, 32]


@pytest.mark.parametrize("seed", range(8))
def test_random_requests_under_eviction(tmp_path, seed):
    """Whatever the sizes, a cache that holds one request and its cut serves all of them: the host's account alone, on
    twins that evict nothing."""
    class Twins(TwinKernels):
        def paged_attention(self, q, cache, meta, out, scale, window=0, lse=None):
            super().paged_attention(q, cache, meta, out, scale, window)

        def attention_weights(self, *args, **kwargs):
            pass

        def evict_tokens(self, cache, weights, table, lengths, new_table, keep, recent, kept, longest):
            assert bool((lengths > keep).all()) and int(lengths.max()) == longest <= table.shape[1] * cache.shape[3]
            for old, new, n in zip(table.tolist(), new_table.tolist(), lengths.tolist()):
                assert min(old[:-(-n // cache.shape[3])] + new) >= 0 and not set(old) & set(new) and len(set(new)) == len(new)

    rng = random.Random(seed)
    page, budget, chunk, most = rng.choice([8, 16, 32]), rng.randint(1, 80), rng.choice([4, 16, 33]), rng.choice([8, 16, 64])
    one = -(-(budget + page - 1 + min(chunk, most)) // page) + -(-budget // page)      # pages of a request and of its cut
    llm = LLM(make_folder(tmp_path, "A_loud"), _kernels=Twins(), _device="cpu", dtype="float32", kv_page_size=page,
              num_kvcache_slots=page * (one + rng.randint(0, 6)), max_num_seqs_in_batch=rng.choice([2, 4, 8]), max_num_batched_tokens=most,
              engine_prefill_chunk_size=chunk, decode_reservation_tokens=rng.choice([0, 4, 64]), sparse_method="accumulated_weight",
              eviction_budget=budget, eviction_recent=rng.randint(0, budget), validate_runtime_invariants=True)
    prompts = [random_tokens(rng.randint(1, 150), 512, seed * 100 + i) for i in range(6)]
    params = [SamplingParams(temperature=0.0, max_tokens=rng.randint(1, 60), ignore_eos=True) for _ in prompts]
    out = llm.generate(prompts, params, use_tqdm=False)
    assert [len(o["token_ids"]) for o in out] == [p.max_tokens for p in params]
    E.all_free(llm)
