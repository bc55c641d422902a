"""The engine with its cache in 4 bits and with the sparse method ``accumulated_weight``: every call that a step makes
of the operators behind them is checked, as it happens, against 64 bits over what the cache holds at that moment, and the
engine's own account (tokens, positions, pages) beside it."""
import numpy as np
import pytest
import torch

import tests.compact_oracle as oracle
from sparseengine_amd import LLM, SamplingParams
from sparseengine_amd.cache import layout
from sparseengine_amd.kernels import attention_work
from tests import backends
from tests.helpers import CONFIGS, make_folder, random_tokens
from tests.test_gpu_compact_cache import check_attention

pytestmark = pytest.mark.gpu


def on_host(meta):
    return type("Meta", (), dict(block_table=meta.block_table.cpu().long(), ctx=[int(n) for n in meta.item_ctx_len],
                                 new=[int(n) for n in meta.item_q_len]))


def tokens_of(cache, which, table, n, dtype=torch.float64):
    """The first ``n`` tokens of a block-table row: ``[n, kv_heads, head_dim]``."""
    page = cache.shape[3]
    at = torch.arange(n)
    if cache.dtype == torch.uint8:
        return layout.fp4_read(cache, which, table[at // page], at % page, dtype)
    return (layout.read_keys, layout.read_values)[which](cache, table[at // page], at % page).to(dtype)


def watched(kernels):
    """The kernels, with every call of the cache's operators checked against the oracle."""
    class Watched(type(kernels)):
        seen = {"store": 0, "attend": 0, "weigh": 0, "evict": 0}
        positions, lengths = [], []

        def qk_norm_rope_store(self, qkv, positions, cos_sin, q_weight, k_weight, eps, heads, kv_heads, head_dim, rotary_dim,
                               cache=None, slots=None, page_size=0, **rest):
            super().qk_norm_rope_store(qkv, positions, cos_sin, q_weight, k_weight, eps, heads, kv_heads, head_dim, rotary_dim,
                                       cache, slots, page_size, **rest)
            if cache is None:           # the rotation that a store in 4 bits begins with
                return
            self.positions.append(positions.cpu().tolist())
            if cache.dtype != torch.uint8:
                return
            self.seen["store"] += 1
            there, at = cache.cpu(), slots.cpu().long()
            # the rotated row that the kernel leaves in qkv is what goes into 4 bits
            made = qkv.cpu()[:, heads * head_dim:(heads + 2 * kv_heads) * head_dim].reshape(-1, 2, kv_heads, head_dim)
            for which in (0, 1):
                got = layout.fp4_read(there, which, at // page_size, at % page_size, torch.float64)
                assert torch.equal(got, oracle.held(made[:, which]))

        def paged_attention(self, q, cache, meta, out, scale, window=0, lse=None):
            mine = torch.empty(q.shape[0], q.shape[1], device=q.device) if lse is None else lse
            super().paged_attention(q, cache, meta, out, scale, window, lse=mine)
            self.seen["attend"] += 1
            m, there = on_host(meta), cache.cpu()
            self.lengths.append(m.ctx)
            of = lambda which: lambda i: tokens_of(there, which, m.block_table[i], m.ctx[i])
            check_attention(out, mine, q.cpu(), of, m.ctx, m.new, scale, window, q.dtype)

        def attention_weights(self, q, cache, meta, lse, out, scale, window=0, previous=None):
            before = None if previous is None else previous.cpu().clone()
            super().attention_weights(q, cache, meta, lse, out, scale, window, previous=previous)
            self.seen["weigh"] += 1
            m, there, page = on_host(meta), cache.cpu(), cache.shape[3]
            place = lambda i: (m.block_table[i][torch.arange(m.ctx[i]) // page], slice(None), torch.arange(m.ctx[i]) % page)
            found = oracle.weights(q.cpu(), lambda i: tokens_of(there, 0, m.block_table[i], m.ctx[i]), lse.cpu(),
                                   lambda i: before[place(i)].t().clone(), m.ctx, m.new, scale, window)
            for i, (total, bound) in enumerate(found):
                assert bool(((out.cpu()[place(i)].t().double() - total).abs() <= bound + 1e-30).all())

        def evict_tokens(self, cache, weights, block_table, lengths, new_table, keep, recent, kept, longest):
            old, w, table = cache.cpu().clone(), weights.cpu().clone(), block_table.cpu().long()
            super().evict_tokens(cache, weights, block_table, lengths, new_table, keep, recent, kept, longest)
            self.seen["evict"] += 1
            new, there, page = new_table.cpu().long(), cache.cpu(), cache.shape[3]
            for i, n in enumerate(lengths.cpu().tolist()):
                at = torch.arange(n)
                mine = w[table[i][at // page], :, at % page]
                for h in range(w.shape[1]):
                    stay = oracle.chosen(mine[:, h].tolist(), n, keep, recent)
                    assert kept.cpu()[i, h].tolist() == stay
                    for which in (0, 1):
                        assert torch.equal(tokens_of(there, which, new[i], keep)[:, h], tokens_of(old, which, table[i], n)[stay, h])
    got = Watched()
    got.seen, got.positions, got.lengths = dict.fromkeys(Watched.seen, 0), [], []
    return got


def engine(folder, kernels=None, **kwargs):
    there = dict(backends.ACTIVE.llm_kwargs())
    if kernels is not None:
        there["_kernels"] = kernels
    return LLM(folder, **{**dict(max_num_seqs_in_batch=4, num_kvcache_slots=512, kv_page_size=32, validate_runtime_invariants=True),
                          **kwargs}, **there)


def run(llm, prompts, new):
    return [o["token_ids"] for o in llm.generate(prompts, SamplingParams(temperature=0.0, max_tokens=new, ignore_eos=True), use_tqdm=False)]


def prompts_for(key, lengths):
    return [random_tokens(n, CONFIGS[key][0]["vocab_size"], 40 + n) for n in lengths]


def all_free(llm):
    cache = llm.runner.cache
    cache.check_invariants()
    assert all(g.pool.free_count == g.pool.num_pages for g in cache.groups) and not cache.row_dropped.any()


def check_cache_in_4_bits(tmp_path, monkeypatch, key, dtype, lengths, new, blocks=False, **kwargs):
    """``blocks``: prompts of any length go in blocks, over unpacked pages."""
    if blocks:
        monkeypatch.setattr(attention_work, "FP4_BLOCK_WORK", 0)
    folder, prompts = make_folder(tmp_path, key), prompts_for(key, lengths)
    kernels = watched(backends.ACTIVE.kernels())
    llm = engine(folder, kernels, dtype=dtype, kv_cache_dtype="fp4", **kwargs)
    out = run(llm, prompts, new)
    assert [len(o) for o in out] == [new] * len(prompts)
    layers, steps = CONFIGS[key][0]["num_hidden_layers"], kernels.seen["attend"]
    assert kernels.seen["store"] == steps >= layers * new and kernels.seen["evict"] == 0
    all_free(llm)


def check_eviction(tmp_path, key, dtype, lengths, new, budget, recent, **kwargs):
    folder, prompts = make_folder(tmp_path, key), prompts_for(key, lengths)
    kernels = watched(backends.ACTIVE.kernels())
    llm = engine(folder, kernels, dtype=dtype, sparse_method="accumulated_weight", eviction_budget=budget, eviction_recent=recent, **kwargs)
    page = llm.config.kv_page_size
    out = run(llm, prompts, new)
    assert [len(o) for o in out] == [new] * len(prompts)
    layers = CONFIGS[key][0]["num_hidden_layers"]
    assert kernels.seen["weigh"] == kernels.seen["attend"] and llm.method.evictions > 0
    assert kernels.seen["evict"] >= layers and kernels.seen["evict"] % layers == 0
    # no step begins above the limit; positions go on past it
    portion = min(llm.config.engine_prefill_chunk_size, llm.config.max_num_batched_tokens)
    assert max(max(c) for c in kernels.lengths) < budget + page + portion
    longest = max(len(p) for p in prompts) + new - 1
    assert max(max(p) for p in kernels.positions) == longest - 1
    if llm.scheduler.total_preemptions == 0:
        assert sum(sum(p) for p in kernels.positions) == layers * sum(n * (n - 1) // 2 for n in (len(p) + new - 1 for p in prompts))
    all_free(llm)
    return llm


def check_large_budget_changes_nothing(tmp_path, key, dtype, lengths, new, **kwargs):
    folder, prompts = make_folder(tmp_path, key), prompts_for(key, lengths)
    plain = engine(folder, dtype=dtype, **kwargs)
    kept = engine(folder, dtype=dtype, sparse_method="accumulated_weight", eviction_budget=max(lengths) + new, **kwargs)
    assert run(plain, prompts, new) == run(kept, prompts, new) and kept.method.evictions == 0


@pytest.mark.parametrize("key,dtype,lengths,new,kwargs", [
    ("C_loud", "bfloat16", (1, 33, 70), 5, {}),                                   # the 4-bit kernel
    ("C_loud", "bfloat16", (1, 33, 70), 5, dict(blocks=True)),                    # and its prompts in unpacked blocks
    ("C_loud", "bfloat16", (90, 8), 4, dict(max_num_batched_tokens=24)),          # portions beside decodes
    ("C_loud", "float32", (40, 3), 4, {}),                                        # unpacked, the general kernel
    ("B_loud", "bfloat16", (40, 3), 4, dict(kv_page_size=64))])                   # a head size without a kernel of its own
def test_cache_in_4_bits(tmp_path, monkeypatch, key, dtype, lengths, new, kwargs):
    check_cache_in_4_bits(tmp_path, monkeypatch, key, dtype, lengths, new, **kwargs)


@pytest.mark.parametrize("key,dtype,lengths,new,budget,recent,kwargs", [
    ("C_loud", "bfloat16", (100, 20, 70), 40, 40, 8, dict(kv_cache_dtype="fp4")),                  # cut at the prompt's end, again while decoding
    ("C_loud", "bfloat16", (100, 45), 12, 40, 8, dict(kv_page_size=16, max_num_batched_tokens=48)),  # cut between a prompt's portions
    ("B_loud", "float32", (30, 5), 30, 1, 0, dict(kv_page_size=16)),                               # one token left
    ("A_loud", "float32", (60, 60), 20, 33, 33, dict(kv_page_size=16, num_kvcache_slots=208))])    # the last tokens only; few pages
def test_eviction_in_the_engine(tmp_path, key, dtype, lengths, new, budget, recent, kwargs):
    check_eviction(tmp_path, key, dtype, lengths, new, budget, recent, **kwargs)


@pytest.mark.parametrize("dtype,kwargs", [("float32", {}), ("bfloat16", dict(kv_cache_dtype="fp4"))])
def test_a_budget_that_nothing_exceeds_changes_nothing(tmp_path, dtype, kwargs):
    check_large_budget_changes_nothing(tmp_path, "C_loud", dtype, (33, 5, 64), 8, **kwargs)


def test_more_tokens_than_the_cache_has_room_for(tmp_path):
    """Requests that would not fit whole: 160 tokens of cache for two requests of 150 tokens, each holding 33 to 64."""
    folder, prompts = make_folder(tmp_path, "A_loud"), prompts_for("A_loud", (100, 99))
    llm = engine(folder, dtype="float32", kv_page_size=16, num_kvcache_slots=192, sparse_method="accumulated_weight",
                 eviction_budget=32, max_num_batched_tokens=32)
    with pytest.raises(ValueError, match="cache"):
        run(engine(folder, dtype="float32", kv_page_size=16, num_kvcache_slots=96), prompts, 50)
    assert [len(o) for o in run(llm, prompts, 50)] == [50, 50] and llm.method.evictions > 2
    all_free(llm)


def test_the_engines_own_choice_of_how_much_cache(tmp_path):
    """Without a number of cache slots: what the memory holds, or what so many requests of full length could use."""
    folder, prompts = make_folder(tmp_path, "C_loud"), prompts_for("C_loud", (70, 9))
    kwargs = dict(dtype="bfloat16", num_kvcache_slots=None, max_num_seqs_in_gpu=4, kv_cache_dtype="fp4", gpu_memory_utilization=0.9)
    llm = engine(folder, **kwargs)
    assert llm.runner.cache.groups[0].pool.num_pages * 32 >= llm.config.max_model_len * 4 or backends.ACTIVE.name == "hip"
    evicting = engine(folder, sparse_method="accumulated_weight", eviction_budget=40, **kwargs)
    assert run(llm, prompts, 3) and run(evicting, prompts, 3) and evicting.method.evictions > 0
    all_free(llm)
    all_free(evicting)
