"""The host's account under eviction and with a cache in 4 bits: pages, reserves, memory, work lists (no kernel runs)."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from sparseengine_amd import LLM, SamplingParams
from sparseengine_amd.cache.manager import bytes_per_token
from sparseengine_amd.config.method_registry import PassThroughMethod
from sparseengine_amd.engine.runner import ModelRunner
from sparseengine_amd.parts.base import PagedKVRequest
from tests.helpers import make_folder, random_tokens
from tests.twin_kernels import TwinKernels


class Twins(TwinKernels):
    """The twins of the dense path; gathered weights and eviction do nothing."""

    def paged_attention(self, q, cache, meta, out, scale, window=0, lse=None):
        super().paged_attention(q, cache, meta, out, scale, window)

    def attention_weights(self, *args, **kwargs):
        pass

    def evict_tokens(self, *args, **kwargs):
        pass


def evicting(tmp_path, kernels=None, **kwargs):
    return LLM(make_folder(tmp_path, "A_loud"), _kernels=kernels or Twins(), _device="cpu", **{**dict(
        dtype="float32", kv_page_size=16, num_kvcache_slots=192, max_num_seqs_in_batch=4, max_num_batched_tokens=32,
        engine_prefill_chunk_size=16, sparse_method="accumulated_weight", eviction_budget=33, validate_runtime_invariants=True), **kwargs})


def greedy(n):
    return SamplingParams(temperature=0.0, max_tokens=n, ignore_eos=True)


@pytest.mark.parametrize("fails_at", [1, 2, 3])
def test_a_cut_that_fails_gives_its_pages_back(tmp_path, fails_at):
    """An error while tokens are moved: the step is undone, the fresh pages are free again, and what runs next finds the
    whole cache."""
    class Failing(Twins):
        calls = 0

        def evict_tokens(self, *args, **kwargs):
            Failing.calls += 1
            if Failing.calls == fails_at:
                raise RuntimeError("no room to move the tokens in")

    llm = evicting(tmp_path, Failing())
    prompts = [random_tokens(n, 512, n) for n in (90, 61)]
    for p in prompts:
        llm.add_request(p, greedy(20))
    with pytest.raises(RuntimeError, match="no room"):
        while not llm.is_finished():
            llm.step()
    cache = llm.runner.cache
    cache.check_invariants()
    while not llm.is_finished():
        llm.step()
    cache.check_invariants()
    assert Failing.calls > fails_at and all(g.pool.free_count == g.pool.num_pages for g in cache.groups)


@pytest.mark.parametrize("seqs", [1, 2])
def test_a_cache_of_the_engines_own_size_holds_full_requests_beside_the_reserve(tmp_path, seqs):
    """Without a number of cache slots the cache has room for so many requests of full length: the pages that eviction
    reserves come on top, and a request as long as the model allows is served."""
    most = 160
    llm = evicting(tmp_path, num_kvcache_slots=None, max_num_seqs_in_gpu=seqs, max_num_seqs_in_batch=seqs, max_model_len=most,
                   max_num_batched_tokens=most, engine_prefill_chunk_size=most, eviction_budget=100)
    prompts = [random_tokens(most - 8, 512, i) for i in range(seqs)]
    out = llm.generate(prompts, greedy(8), use_tqdm=False)
    assert [len(o["token_ids"]) for o in out] == [8] * seqs and llm.method.evictions >= seqs
    llm.runner.cache.check_invariants()


def test_can_step_leaves_the_reserved_pages_alone(tmp_path):
    """A caller that drives the runner by ``can_step``: it says no before a step would take the pages that a cut needs, and
    every request that it lets run is cut when its time comes."""
    # a request reaches its cut in 4 pages (33 + 16 tokens and a step's): two do, beside 3 pages in reserve
    runner = evicting(tmp_path, num_kvcache_slots=16 * 13).runner
    from sparseengine_amd.engine.runner import StepEntry
    reserved = runner.method.reserved_pages()[0]
    group, fed = runner.cache.groups[0], {}
    for turn in range(300):
        entries = [(name, 5) for name in ("a", "b", "c")]
        entries = [entries[turn % 3]]
        if runner.can_step(entries):
            name, n = entries[0]
            runner.step([StepEntry(name, random_tokens(n, 512, turn))])
            fed[name] = fed.get(name, 0) + n
            assert group.pool.free_count >= reserved and runner.cache.row_len[runner.cache.row_of(name)] < runner.method._limit()
        if max(fed.values()) > 150:
            break
    assert runner.method.evictions > 0
    assert not runner.can_step([("d", (group.pool.free_count - reserved) * 16 + 1)])
    assert runner.can_step([("d", (group.pool.free_count - reserved) * 16)])


@pytest.mark.parametrize("layers", [1, 2, 32])
@pytest.mark.parametrize("dtype,head_dim,direct", [(torch.bfloat16, 96, False), (torch.float32, 128, False),
                                                   (torch.bfloat16, 288, False), (torch.bfloat16, 128, True)])
def test_memory_kept_for_unpacked_pages(monkeypatch, dtype, head_dim, direct, layers):
    """The cache that the engine chooses leaves room for what attention unpacks of one layer: where a head size or type has
    no kernel that reads 4 bits, every token that the cache holds (a full decode step reads them all)."""
    free, total = 60 << 30, 64 << 30
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda device=None: (free, total))
    requests = {i: PagedKVRequest(4, head_dim, None, None) for i in range(layers)}
    runner = SimpleNamespace(kv_dtype=torch.uint8, dtype=dtype, device=torch.device("cuda"), max_model_len=4096, kv_page_size=64,
                             method=PassThroughMethod())
    tokens = ModelRunner.derive_cache_tokens(runner, requests, 1 << 20, 0.9)
    usable = free - int(0.1 * total) - (2 << 30)
    held = layers * bytes_per_token(requests[0], torch.uint8)
    unpacked = bytes_per_token(requests[0], dtype)
    at_once = 2 * 4096 if direct else tokens
    assert tokens * held + at_once * unpacked <= usable          # and no more is left unused than a token of each
    assert (tokens + 1) * held + (at_once + (not direct)) * unpacked > usable
