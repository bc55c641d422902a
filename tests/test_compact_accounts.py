"""The host's account under eviction and with a cache in 4 bits: pages, reserves, memory, work lists (no kernel runs)."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from sparseengine_amd import LLM, SamplingParams
from sparseengine_amd.cache.manager import bytes_per_token
from sparseengine_amd.config.method_registry import PassThroughMethod
from sparseengine_amd.engine.runner import ModelRunner
from sparseengine_amd.kernels import attention_work as aw
from sparseengine_amd.parts.base import PagedKVRequest
from tests import backends
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


def test_portions_of_many_prompts_unpack_no_more_than_they_may():
    """Of the items that would go in blocks the heaviest do, as far as the limit reaches; the others keep the 4-bit kernel,
    the list of pages is that of the items in blocks, and both builders agree."""
    rng = np.random.default_rng(3)
    limited = 0
    for _ in range(200):
        n = int(rng.integers(1, 12))
        ctx = rng.integers(1, 20000, n)
        q = np.minimum(rng.integers(1, 400, n), ctx)
        group, window, page = int(rng.choice([1, 6, 16])), int(rng.choice([0, 0, 3000])), int(rng.choice([32, 64, 96]))
        most = int(rng.integers(1, 80000))
        work = aw.build_fp4_attention_work(q, ctx, group, 8, window, 128, page, most)
        free = aw.build_fp4_attention_work(q, ctx, group, 8, window, 128)
        pairs, table = aw.fp4_unpack_list(q, ctx, group, 128, page, window, True, most)
        items, all_items = set(work.block_units[:, 0].tolist()), set(free.block_units[:, 0].tolist())
        assert len(pairs) * page <= most and set(pairs[:, 0].tolist()) == items and items <= all_items
        assert items | set(work.units[:, 0].tolist()) == set(range(n))
        limited += items != all_items
        held = -(-ctx // page) - (np.maximum(0, ctx - q - window + 1) // page if window else 0)
        if sum(int(held[i]) for i in all_items) * page <= most:
            assert items == all_items
        for i in all_items - items:       # what was left out would not have fitted beside those that are in
            assert (len(pairs) + int(held[i])) * page > most
        tiles = aw.fp4_block_tiles(q, ctx, group, window, page, most)
        a = aw.build_attention_work(q, ctx, group, 8, window, 900, 128, 64, tiles)
        b = aw.build_attention_work_numpy(q, ctx, group, 8, window, 900, 128, 64, tiles)
        assert all((getattr(a, f) == getattr(b, f)).all() for f in ("units", "tasks", "block_units")) and a.num_slots == b.num_slots
    assert limited > 20


def test_the_engine_limits_what_a_step_unpacks():
    """Four portions on long prefixes in one step: the batch's list of pages holds two longest prompts' tokens at most."""
    from sparseengine_amd.cache.manager import CacheManager
    from sparseengine_amd.engine.batch import BatchBuilder, StepItem
    cache = CacheManager({0: PagedKVRequest(1, 64, None, None)}, max_rows=4, max_model_len=40000, page_size=64, num_tokens=4 * 40000,
                         dtype=torch.bfloat16, device="cpu", kv_dtype=torch.uint8)
    rows = [cache.admit(i) for i in range(4)]
    cache.append([(row, 38000) for row in rows])
    builder = BatchBuilder(None, cache, torch.bfloat16, "cpu", 512, attention_shapes={0: {(16, 0)}}, most_unpacked=2 * 40000)
    fb = builder.build([StepItem(row, [1] * 64, [63]) for row in rows])
    work, (pairs, table) = fb.groups[0].work[(16, 0, "fp4")], fb.groups[0].work[("unpack", 16, 64, 64, 0, True)]
    assert pairs.shape[0] * 64 <= 80000 and len(set(pairs[:, 0].tolist())) == 2
    assert set(work.block_units[:, 0].tolist()) == set(pairs[:, 0].tolist())
    assert set(work.block_units[:, 0].tolist()) | set(work.units[:, 0].tolist()) == {0, 1, 2, 3}


def test_the_runner_limits_its_batches(tmp_path):
    llm = evicting(tmp_path, max_model_len=160)
    assert llm.runner.builder.most_unpacked == 2 * 160


def test_a_long_context_beside_many_short_ones_is_cut():
    """Where the tiles alone fill the chip, an item of more than twice the mean keys is cut all the same: no wavefront goes
    through a whole long context by itself.  Items near the mean, and short ones, stay whole."""
    longest = lambda work: int((work.units[:, 3] - work.units[:, 2]).max())
    for short, many in ((500, 100), (500, 200), (2000, 300), (70, 1000)):
        ctx = [short] * many + [131071]
        work = aw.build_fp4_attention_work([1] * len(ctx), ctx, 6, 8, 0, 128)
        mean = -(-sum(ctx) // len(ctx))
        assert longest(work) <= max(aw.FP4_WHOLE_KEYS, 2 * mean + 32, 131071 // aw.MAX_SPLITS + 32)
        assert set(work.tasks[:, 0].tolist()) == {many} or many == 100
        for item, n in ((0, short), (many, 131071)):      # every key once
            mine = work.units[work.units[:, 0] == item]
            assert mine[0, 2] == 0 and mine[-1, 3] == n and (mine[1:, 2] == mine[:-1, 3]).all()
        numpy = aw.build_attention_work_numpy([1] * len(ctx), ctx, 6, 8, 0, 1, 128, 128, 9, 2 * mean // 32 * 32)
        native = aw.build_attention_work([1] * len(ctx), ctx, 6, 8, 0, 1, 128, 128, 9, 2 * mean // 32 * 32)
        assert (numpy.units == native.units).all() and (numpy.tasks == native.tasks).all()
    rng = np.random.default_rng(0)
    near = rng.integers(4000, 8200, 160)
    assert len(aw.build_fp4_attention_work([1] * 160, near, 6, 8, 0, 128).tasks) == 0
    assert len(aw.build_fp4_attention_work([1] * 300, [20] * 299 + [160], 6, 8, 0, 128).tasks) == 0
    # a window leaves nothing long
    assert len(aw.build_fp4_attention_work([1] * 201, [500] * 200 + [131071], 6, 8, 600, 128).tasks) == 0


@pytest.mark.skipif(not backends.EmulatedBackend().available(), reason="no host compiler for the emulated kernels")
@pytest.mark.parametrize("kwargs,more", [({}, set()), (dict(kv_cache_dtype="fp4", kv_page_size=32), {"cache_fp4", "attention_fp4"}),
                                         (dict(sparse_method="accumulated_weight", eviction_budget=8), {"attention_weights", "evict"})])
def test_only_the_libraries_that_are_called_are_built(tmp_path, monkeypatch, kwargs, more):
    from sparseengine_amd.kernels import library
    asked = []
    monkeypatch.setattr(library, "ensure_built", lambda names=None, *a, **k: asked.append(set(names)))
    with backends.use(backends.EmulatedBackend()) as backend:
        LLM(make_folder(tmp_path, "C_loud"), num_kvcache_slots=128, **kwargs, **backend.llm_kwargs())
    compact = {"cache_fp4", "attention_fp4", "attention_weights", "evict"}
    assert asked[0] & compact == more and {"rope_kv", "attention_mfma", "norm"} <= asked[0]


def test_a_cache_manager_that_knows_nothing_of_eviction(tmp_path):
    """A method's own manager with the constructor and interface of the paged one, but none of what eviction and 4 bits added
    to it, serves the dense method as before."""
    from sparseengine_amd.cache.manager import CacheManager
    from sparseengine_amd.config import method_registry

    class Plain:
        def __init__(self, requests, **kwargs):
            self.paged = CacheManager(requests, **kwargs)

        def __getattr__(self, name):
            if name in ("row_dropped", "kv_dtype", "begin_eviction", "finish_eviction", "abort_eviction"):
                raise AttributeError(name)
            return getattr(self.__dict__["paged"], name)

    method_registry.register_method("plain", PassThroughMethod, "all_chunked", cache_manager_cls=Plain)
    try:
        prompts = [random_tokens(n, 512, n) for n in (20, 5)]
        make = lambda **k: evicting(tmp_path, eviction_budget=0, **k)
        out, dense = (make(sparse_method=name).generate(prompts, greedy(4), use_tqdm=False) for name in ("plain", ""))
        assert [o["token_ids"] for o in out] == [o["token_ids"] for o in dense]
    finally:
        method_registry._METHODS.pop("plain", None)
